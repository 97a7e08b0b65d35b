"""Operators of a transformer's training step and prompt pass on one GPU: their cases, inputs and plain forms.

    attention   softmax attention over whole prompts, packed one behind the other, with grouped heads;
                ``direction`` "fwd" is the prompt pass, "train" the forward and the backward pass
    balance     balance loss of a mixture-of-experts router, pairs per expert and the gradient of the logits
    adamw       one AdamW step over a list of tensors, with moments in 32 or in 8 bits

A case is a dict of plain values; ``kind`` is one of the above and the rest are its sizes.  Where ``own`` is
false :func:`run` computes with elementary torch operations, where it is true with the library's operators.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 256     # elements that share one scale where moments are kept in 8 bits
_TOP = 448.0     # largest e4m3 value
_LEAST = 2.0 ** -100  # a block whose largest magnitude is below this is kept as zeros


def listed():
    return [
        # Three short prompts, the first a single token, on a small model: launches count.
        {"name": "attn_fwd_short", "kind": "attention", "direction": "fwd", "tokens": 41, "seqs": 3, "tail": 0,
         "heads": 4, "kv_heads": 2, "dim": 64, "causal": True, "dtype": "bf16"},
        # A batch of prompts of different lengths with a padded end: the prompt pass of a served model.
        {"name": "attn_fwd_packed", "kind": "attention", "direction": "fwd", "tokens": 8100, "seqs": 5, "tail": 92,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "dtype": "bf16"},
        # One long prompt, the heads of one of several ranks.
        {"name": "attn_fwd_long", "kind": "attention", "direction": "fwd", "tokens": 16384, "seqs": 1, "tail": 0,
         "heads": 8, "kv_heads": 2, "dim": 128, "causal": True, "dtype": "bf16"},
        # One layer's training step on one sequence of the benchmark's length.
        {"name": "attn_train_4096", "kind": "attention", "direction": "train", "tokens": 4096, "seqs": 1, "tail": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "dtype": "bf16"},
        # An encoder's training step on packed sequences: every position sees its whole sequence, odd head size.
        {"name": "attn_train_ragged", "kind": "attention", "direction": "train", "tokens": 5003, "seqs": 9, "tail": 21,
         "heads": 12, "kv_heads": 4, "dim": 80, "causal": False, "dtype": "fp16"},
        # The test suite's MoE layer.
        {"name": "balance_small", "kind": "balance", "tokens": 1000, "experts": 8, "top": 2, "masked": False,
         "dtype": "fp32"},
        # The MoE benchmark's layer: 16384 tokens of one GPU, 64 experts, top-2.
        {"name": "balance_bench", "kind": "balance", "tokens": 16384, "experts": 64, "top": 2, "masked": False,
         "dtype": "fp32"},
        # A large batch with padding over many fine-grained experts.
        {"name": "balance_large", "kind": "balance", "tokens": 200_003, "experts": 256, "top": 8, "masked": True,
         "dtype": "bf16"},
        # The norms and biases of a small model: many tiny tensors of odd sizes.
        {"name": "adamw_tiny", "kind": "adamw", "tensors": 24, "elements": 9_000, "param": "fp32", "grad": "fp32",
         "bits": 32, "copies": False},
        # The parameters of the data-parallel ResNet-50 by number and size: float32 weights and a bf16 copy.
        {"name": "adamw_resnet50", "kind": "adamw", "tensors": 161, "elements": 25_557_032, "param": "fp32",
         "grad": "bf16", "bits": 32, "copies": True},
        # The same list with 8-bit moments.
        {"name": "adamw_8bit", "kind": "adamw", "tensors": 161, "elements": 25_557_032, "param": "bf16",
         "grad": "bf16", "bits": 8, "copies": False},
        # One layer's weights of the benchmark MLP over 4 GPUs, bf16 with 8-bit moments.
        {"name": "adamw_8bit_large", "kind": "adamw", "tensors": 3, "elements": 176_160_768, "param": "bf16",
         "grad": "bf16", "bits": 8, "copies": False},
    ]


# ----------------------------------------------------------------------------------- drawn cases

def _log(rng, lo, hi):
    """A whole number between ``lo`` and ``hi``, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges, never more work than the largest listed one of its kind."""
    kind = rng.choice(["attention", "attention", "attention", "balance", "adamw", "adamw"])
    if kind == "attention":
        direction = rng.choice(["fwd", "train"])
        kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        heads = kv * group
        most = int(math.sqrt((8 * 16384 ** 2 if direction == "fwd" else 32 * 4096 ** 2) / heads))
        tokens = _log(rng, 24, min(16384, most))
        return {"kind": kind, "direction": direction, "tokens": tokens, "seqs": _log(rng, 1, max(1, min(64, tokens // 8))),
                "tail": rng.choice([0, 0, 1, 37, 200]), "heads": heads, "kv_heads": kv,
                "dim": rng.choice([16, 40, 64, 64, 72, 80, 96, 112, 128, 128, 128]), "causal": rng.random() < 0.7,
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "balance":
        experts = rng.choice([2, 5, 8, 16, 30, 64, 100, 128, 160, 256, 384])
        tokens = _log(rng, 1, min(250_000, 51_000_000 // experts))
        return {"kind": kind, "tokens": tokens, "experts": experts, "top": rng.randint(1, min(8, experts)),
                "masked": rng.random() < 0.4, "dtype": rng.choice(["fp32", "fp32", "bf16"])}
    elements = _log(rng, 300, 170_000_000)
    bits = rng.choice([8, 32])
    param = rng.choice(["bf16", "fp32"])
    if bits == 32 and elements > 60_000_000:
        elements //= 3
    return {"kind": kind, "tensors": _log(rng, 1, min(400, elements // 100)), "elements": elements, "param": param,
            "grad": rng.choice(["bf16", "fp32"]), "bits": bits, "copies": param == "fp32" and rng.random() < 0.5}


# ------------------------------------------------------------------------------- inputs

def _parts(total, count):
    """``count`` lengths of at least one that add up to ``total``: uneven, and the same for every seed."""
    rng = random.Random(total * 1009 + count)
    weights = [rng.expovariate(1.0) + 0.02 for _ in range(count)]
    scale = (total - count) / sum(weights)
    sizes = [1 + int(w * scale) for w in weights]
    sizes[sizes.index(max(sizes))] += total - sum(sizes)
    return sizes


def _lengths(case):
    sizes = _parts(case["tokens"], case["seqs"])
    if case["seqs"] >= 3:  # the first prompt is a single token
        first, sizes[0] = sizes[0], 1
        sizes[-1] += first - 1
    return sizes


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, scale, generator=gen)


def _quantize(x, keep_nonzero):
    """Blocks of 256 values as e4m3 numbers with one scale each."""
    top = x.abs().amax(1, keepdim=True)
    q = (x * torch.where(top < _LEAST, torch.zeros_like(top), _TOP / top)).to(torch.float8_e4m3fn)
    if keep_nonzero:  # a root that is not zero stays at the smallest number at least
        code = q.view(torch.uint8)
        q = torch.where((x > 0) & (code == 0), torch.ones_like(code), code).view(torch.float8_e4m3fn)
    return q, torch.where(top < _LEAST, torch.zeros_like(top), top / _TOP).squeeze(1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "attention":
        dt, n, rows = _DTYPES[case["dtype"]], case["tokens"], case["tokens"] + case["tail"]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # queries, keys and values as one projection of the tokens leaves them
        qkv = _randn(gen, rows, h + 2 * hk, d, dtype=dt)
        ends = torch.tensor([0] + _lengths(case), dtype=torch.int64).cumsum(0)
        s = {"kind": kind, "train": case["direction"] == "train", "causal": case["causal"], "n": n,
             "q": qkv[:, :h], "k": qkv[:, h:h + hk], "v": qkv[:, h + hk:], "cu": ends.to(torch.int32).cuda(),
             "out": torch.zeros(rows, h, d, dtype=dt, device="cuda"),
             "lse": torch.zeros(h, rows, dtype=torch.float32, device="cuda")}
        if s["train"]:
            s["dout"] = _randn(gen, rows, h, d, dtype=dt)
            grad = torch.zeros(rows, h + 2 * hk, d, dtype=dt, device="cuda")
            s["dq"], s["dk"], s["dv"] = grad[:, :h], grad[:, h:h + hk], grad[:, h + hk:]
        return s
    if kind == "balance":
        t, e, k = case["tokens"], case["experts"], case["top"]
        logits = _randn(gen, t, e, scale=1.5) + _randn(gen, 1, e, scale=0.7)  # some experts are preferred
        idx = logits.topk(k, 1).indices.to(torch.int32).contiguous()
        mask = None
        if case["masked"]:  # padding at the end of every run of tokens
            mask = torch.rand(t, generator=gen, device="cuda") < 0.9
        return {"kind": kind, "logits": logits.to(_DTYPES[case["dtype"]]), "idx": idx, "mask": mask, "coef": 0.01}
    sizes = _parts(case["elements"], case["tensors"])
    # parameters as views of one flat buffer, each from a block's begin on; gaps between them are zero
    begins, blocks = [], 0
    for n in sizes:
        begins.append(blocks * _BLOCK)
        blocks += -(-n // _BLOCK)
    live = torch.zeros(blocks * _BLOCK, dtype=torch.bool, device="cuda")
    views = lambda x: [x[b:b + n] for b, n in zip(begins, sizes)]  # noqa: E731
    for view in views(live):
        view.fill_(True)
    pt, gt = _DTYPES[case["param"]], _DTYPES[case["grad"]]
    flat = _randn(gen, live.numel(), dtype=pt, scale=0.02) * live
    copy = torch.zeros(live.numel(), dtype=torch.bfloat16, device="cuda") if case["copies"] else None
    s = {"kind": kind, "bits": case["bits"], "begins": begins, "flat": flat, "copy": copy, "params": views(flat),
         "grads": [_randn(gen, n, dtype=gt, scale=0.01) for n in sizes], "copies": None if copy is None else views(copy),
         "hyper": {"lr": 1e-3, "step": 100, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1, "grad_scale": 0.5}}
    # moments as after many steps, in one buffer for all tensors laid out alike
    m = _randn(gen, live.numel(), scale=0.002) * live
    r = (_randn(gen, live.numel(), scale=0.005).abs() + 1e-4) * live
    if case["bits"] == 8:
        (s["m"], s["m_scale"]), (s["r"], s["r_scale"]) = _quantize(m.view(-1, _BLOCK), False), _quantize(r.view(-1, _BLOCK), True)
        s["m"], s["r"] = s["m"].view(-1), s["r"].view(-1)
    else:
        s["m"], s["v"] = m, r * r
    if own:
        from megray_b200.ops import AdamWState

        s["state"] = AdamWState(s["params"], bits=case["bits"])
        for name in ("m", "r", "m_scale", "r_scale") if case["bits"] == 8 else ("m", "v"):
            getattr(s["state"], name).copy_(s[name])
            s[name] = getattr(s["state"], name)
    return s


# ------------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"attention": _attention, "balance": _balance, "adamw": _adamw}[state["kind"]](state)


def _run_own(s):
    from megray_b200 import ops

    if s["kind"] == "attention":
        out, lse = ops.attention(s["q"], s["k"], s["v"], s["cu"], causal=s["causal"], out=s["out"], lse=s["lse"])
        if not s["train"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = ops.attention_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, s["cu"], causal=s["causal"],
                                       dq=s["dq"], dk=s["dk"], dv=s["dv"])
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if s["kind"] == "balance":
        loss, counts, dlogits = ops.balance_loss_grad(s["logits"], s["idx"], s["coef"], mask=s["mask"])
        return {"loss": loss, "counts": counts, "dlogits": dlogits}
    ops.adamw_step(s["params"], s["grads"], s["state"], copies=s["copies"], **s["hyper"])
    return _adamw_outputs(s)


def _attention(s):
    n, cu = s["n"], s["cu"].long()
    q, k, v = s["q"][:n].float(), s["k"][:n].float(), s["v"][:n].float()
    hk, group, scale = k.shape[1], q.shape[1] // k.shape[1], 1.0 / math.sqrt(q.shape[2])
    at = torch.arange(n, device="cuda")
    seq = torch.searchsorted(cu, at, right=True)
    hidden = seq[:, None] != seq[None, :]
    if s["causal"]:
        hidden |= at[None, :] > at[:, None]
    split = lambda x: x.view(n, hk, -1, x.shape[2]).permute(1, 2, 0, 3)   # [kv heads, group, tokens, dim]  # noqa: E731
    join = lambda x: x.permute(2, 0, 1, 3).reshape(n, -1, x.shape[3])     # noqa: E731
    qg, kg, vg = split(q), split(k), split(v)
    p = torch.matmul(qg, kg.transpose(2, 3)).mul_(scale).masked_fill_(hidden, -math.inf)
    top = p.amax(3, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    p = p.div_(total)
    out = torch.matmul(p, vg)
    s["out"][:n] = join(out).to(s["out"].dtype)
    s["lse"][:, :n] = (top + total.log()).reshape(-1, n)
    if not s["train"]:
        return {"out": s["out"], "lse": s["lse"]}
    do = split(s["dout"][:n].float())
    dv = torch.matmul(p.transpose(2, 3), do).sum(1, keepdim=True)
    ds = torch.matmul(do, vg.transpose(2, 3)).sub_((out * do).sum(3, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, kg).mul_(scale)
    dk = torch.matmul(ds.transpose(2, 3), qg).sum(1, keepdim=True).mul_(scale)
    s["dq"][:n], s["dk"][:n], s["dv"][:n] = (join(x).to(s["dq"].dtype) for x in (dq, dk, dv))
    return {"out": s["out"], "lse": s["lse"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}


def _balance(s):
    x, idx = s["logits"].float(), s["idx"].long()
    t, e = x.shape
    live = torch.ones(t, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    valid = live.sum().clamp(min=1).double()
    counts = torch.zeros(e, dtype=torch.int32, device="cuda")
    counts.index_add_(0, idx.reshape(-1), live.int()[:, None].expand_as(idx).reshape(-1))
    p = (x - x.amax(1, keepdim=True)).exp_()
    p = p.div_(p.sum(1, keepdim=True)).mul_(live[:, None])
    share = counts.double() / (valid * idx.shape[1])
    loss = s["coef"] * e * (share * (p.sum(0, dtype=torch.float64) / valid)).sum()
    w = share.sub(share.mean()).mul(s["coef"] * e / valid).float()  # a constant in the shares has no gradient
    dlogits = (w - (p * w).sum(1, keepdim=True)).mul_(p)
    return {"loss": loss.float().view(1), "counts": counts, "dlogits": dlogits.to(s["logits"].dtype)}


def _adamw_outputs(s):
    if s["bits"] == 8:
        moments = {"m": s["m"], "r": s["r"], "m_scale": s["m_scale"], "r_scale": s["r_scale"]}
    else:
        moments = {"m": s["m"], "v": s["v"]}
    return {"params": s["flat"], "copies": s["copy"], **moments}


def _adamw(s):
    h = s["hyper"]
    b1, b2 = h["betas"]
    rate = h["lr"] / (1.0 - b1 ** h["step"])
    root = 1.0 / math.sqrt(1.0 - b2 ** h["step"])
    g = torch.zeros(s["m"].numel(), dtype=torch.float32, device="cuda")
    p = torch.zeros_like(g)
    at = lambda x: [x[b:b + t.numel()] for b, t in zip(s["begins"], s["params"])]  # noqa: E731
    torch._foreach_copy_(at(g), s["grads"])
    torch._foreach_copy_(at(p), s["params"])
    if s["bits"] == 8:
        m = s["m"].float().view(-1, _BLOCK) * s["m_scale"][:, None]
        v = (s["r"].float().view(-1, _BLOCK) * s["r_scale"][:, None]).square()
        m, v = m.view(-1), v.view(-1)
    else:
        m, v = s["m"], s["v"]
    g = g * h["grad_scale"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + g * g * (1.0 - b2)
    r = v.sqrt()
    p = p * (1.0 - h["lr"] * h["weight_decay"]) - m / (r * root + h["eps"]) * rate
    torch._foreach_copy_(s["params"], at(p))
    if s["copies"] is not None:
        torch._foreach_copy_(s["copies"], at(p))
    if s["bits"] == 8:
        for name, x, keep in (("m", m, False), ("r", r, True)):
            q, scale = _quantize(x.view(-1, _BLOCK), keep)
            s[name].copy_(q.view(-1))
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_outputs(s)


# ------------------------------------------------------------------------------- work

def work(case):
    """Each input read once and each result written once; products of the pairs that the mask leaves."""
    kind = case["kind"]
    if kind == "attention":
        n, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(x * (x + 1) // 2 if case["causal"] else x * x for x in _lengths(case)) * h
        fwd = 2.0 * n * d * (2 * h + 2 * hk) + 4.0 * n * h
        if case["direction"] == "fwd":
            return {"bytes": fwd, "flops": 4.0 * d * pairs}
        return {"bytes": fwd + 2.0 * n * d * (2 * h + 2 * hk), "flops": 14.0 * d * pairs}
    if kind == "balance":
        t, e, size = case["tokens"], case["experts"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": t * (2.0 * e * size + 4 * case["top"] + (1 if case["masked"] else 0)) + 4.0 * e,
                "flops": 12.0 * t * e}
    size = {"bf16": 2, "fp32": 4}
    per = 2 * size[case["param"]] + size[case["grad"]] + (2 if case["copies"] else 0)
    per += 16 if case["bits"] == 32 else 4 + 16 / _BLOCK
    return {"bytes": float(per * case["elements"]), "flops": 20.0 * case["elements"]}


# ------------------------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    """What :func:`run` returns, from the definitions in float64."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"attention": _exact_attention, "balance": _exact_balance, "adamw": _exact_adamw}[case["kind"]](case, s)


def _exact_attention(case, s):
    """Sequence by sequence and head by head; the gradients by differentiating the definition."""
    names = ("out", "lse", "dq", "dk", "dv") if s["train"] else ("out", "lse")
    got = {x: s[x].double() for x in names}
    h, hk, begin = case["heads"], case["kv_heads"], 0
    for length in _lengths(case):
        rows = slice(begin, begin + length)
        begin += length
        future = torch.ones(length, length, dtype=torch.bool, device="cuda").triu(1) if case["causal"] else None
        for i in range(h):
            j = i * hk // h
            q, k, v = (x.double().requires_grad_(s["train"]) for x in (s["q"][rows, i], s["k"][rows, j], s["v"][rows, j]))
            z = q @ k.t() / math.sqrt(case["dim"])
            if future is not None:
                z = z.masked_fill(future, -math.inf)
            lse = torch.logsumexp(z, 1)
            out = torch.softmax(z, 1) @ v
            got["out"][rows, i], got["lse"][i, rows] = out.detach(), lse.detach()
            if s["train"]:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"][rows, i].double())
                got["dq"][rows, i] = dq
                got["dk"][rows, j] += dk
                got["dv"][rows, j] += dv
    return got


def _exact_balance(case, s):
    x = s["logits"].double().requires_grad_()
    t, e = x.shape
    live = torch.ones(t, dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    valid = max(1.0, float(live.sum()))
    picked = s["idx"].long()[live > 0].reshape(-1)
    counts = torch.bincount(picked, minlength=e)
    loss = s["coef"] * e * (counts.double() / (valid * case["top"]) * (torch.softmax(x, 1) * live[:, None]).sum(0) / valid).sum()
    dlogits, = torch.autograd.grad(loss, x)
    return {"loss": loss.detach().view(1), "counts": counts.int(), "dlogits": dlogits}


def _exact_adamw(case, s):
    h, n8 = s["hyper"], case["bits"] == 8
    b1, b2 = h["betas"]
    p_all, m_all, v_all = torch.zeros(3, s["m"].numel(), dtype=torch.float64, device="cuda")
    if n8:
        per = lambda x, c: (x.double().view(-1, _BLOCK) * c.double()[:, None]).view(-1)  # noqa: E731
        m_old, v_old = per(s["m"], s["m_scale"]), per(s["r"], s["r_scale"]) ** 2
    else:
        m_old, v_old = s["m"].double(), s["v"].double()
    for b, p, g in zip(s["begins"], s["params"], s["grads"]):
        rows = slice(b, b + p.numel())
        g = g.double() * h["grad_scale"]
        m, v = b1 * m_old[rows] + (1 - b1) * g, b2 * v_old[rows] + (1 - b2) * g * g
        m_hat, v_hat = m / (1 - b1 ** h["step"]), v / (1 - b2 ** h["step"])
        p = p.double()
        p_all[rows] = p - h["lr"] * (m_hat / (v_hat.sqrt() + h["eps"]) + h["weight_decay"] * p)
        m_all[rows], v_all[rows] = m, v
    got = {"params": p_all, "copies": p_all if case["copies"] else None}
    if not n8:
        return {**got, "m": m_all, "v": v_all}
    # the 8-bit numbers themselves: a value next to a border goes either way
    top = lambda x: x.abs().view(-1, _BLOCK).amax(1) / _TOP  # noqa: E731
    return {**got, "m": None, "r": None, "m_scale": top(m_all), "r_scale": top(v_all.sqrt())}
