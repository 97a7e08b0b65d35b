"""The operators of a transformer layer together, as a training step uses them: packed attention, the expert layer
with its balance loss, AdamW over all weights; gradients against a float64 evaluation of the same layer."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LENGTHS, HEADS, KV, DIM, HIDDEN, EXPERTS, FFN, COEF = [200, 1, 183], 4, 2, 64, 256, 8, 384, 0.05
T = sum(LENGTHS)


class Layer:
    """x1 = x + attention(norm(x)); result = x1 + experts(norm(x1)); loss = mean(result^2) + balance loss."""

    def __init__(self, optimizer):
        from megray_b200.models import MoEConfig, MoELayer
        from megray_b200.ops import AdamWState

        g = torch.Generator(device="cuda").manual_seed(1)
        r = lambda *s: torch.empty(*s, device="cuda").normal_(0, 0.06, generator=g)  # noqa: E731
        self.wqkv = r((HEADS + 2 * KV) * DIM, HIDDEN).bfloat16()
        self.wo, self.wr = r(HIDDEN, HEADS * DIM).bfloat16(), r(EXPERTS, HIDDEN) * 4
        self.moe = MoELayer(MoEConfig(experts=EXPERTS, hidden=HIDDEN, ffn=FFN, tokens=T, init_std=0.06, lr=1e-3,
                                      capacity_factor=4.0, balance_coef=COEF, optimizer=optimizer))
        self.cu = torch.tensor([0] + LENGTHS, device="cuda").cumsum(0).to(torch.int32)
        self.state = AdamWState([self.wqkv, self.wo, self.wr], bits=8 if optimizer == "adamw8" else 32)

    def step(self, x, t):
        from megray_b200 import ops

        bf = dict(dtype=torch.bfloat16, device="cuda")
        n1, n2, x1 = (torch.empty(T, HIDDEN, **bf) for _ in range(3))
        inv1, inv2 = (torch.empty(T, device="cuda") for _ in range(2))
        ops.add_rmsnorm(x, n_out=n1, inv_rms=inv1)
        qkv = ops.gemm(n1, self.wqkv).view(T, HEADS + 2 * KV, DIM)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:]
        o, lse = ops.attention(q, k, v, self.cu)
        ops.add_rmsnorm(x, ops.gemm(o.view(T, -1), self.wo), x_out=x1, n_out=n2, inv_rms=inv2)
        z = self.moe.forward(n2, n2.float() @ self.wr.t())
        loss, dres = ops.mse_loss_grad(x1 + z)
        dn2, dlogits = self.moe.backward(dres)
        dn2 = (dn2.float() + dlogits @ self.wr).bfloat16()
        dwr = dlogits.t() @ n2.float()
        dx1, dx = torch.empty_like(x), torch.empty_like(x)
        ops.rmsnorm_bwd(dn2, n2, inv2, dres, dx1)
        do = ops.gemm(dx1, self.wo, b_mn=True).view(T, HEADS, DIM)
        dwo = ops.gemm(dx1, o.view(T, -1), a_mn=True, b_mn=True)
        dqkv = torch.empty_like(qkv)
        ops.attention_bwd(do, q, k, v, o, lse, self.cu, dq=dqkv[:, :HEADS], dk=dqkv[:, HEADS:HEADS + KV],
                          dv=dqkv[:, HEADS + KV:])
        dwqkv = ops.gemm(dqkv.view(T, -1), n1, a_mn=True, b_mn=True)
        ops.rmsnorm_bwd(ops.gemm(dqkv.view(T, -1), self.wqkv, b_mn=True), n1, inv1, dx1, dx)
        grads = [dwqkv, dwo, dwr]
        ops.adamw_step([self.wqkv, self.wo, self.wr], grads, self.state, 1e-3, step=t)
        self.moe.optimizer_step()
        return loss + self.moe.balance_loss, dx, grads


def reference(x, layer):
    """Loss and gradients in float64, with the experts that the layer chose."""
    leaf = lambda t: t.detach().double().clone().requires_grad_()  # noqa: E731
    x, wqkv, wo, wr, wgu, wdn = (leaf(t) for t in (x, layer.wqkv, layer.wo, layer.wr, layer.moe.w_gu, layer.moe.w_down))
    idx = layer.moe.ep.idx.long()
    norm = lambda t: t * torch.rsqrt(t.pow(2).mean(1, keepdim=True) + 1e-6)  # noqa: E731
    qkv = (norm(x) @ wqkv.t()).view(T, HEADS + 2 * KV, DIM)
    k, v = (qkv[:, a:a + KV].repeat_interleave(HEADS // KV, 1) for a in (HEADS, HEADS + KV))
    z = torch.einsum("qhd,khd->hqk", qkv[:, :HEADS], k) / math.sqrt(DIM)
    seq = torch.repeat_interleave(torch.arange(len(LENGTHS)), torch.tensor(LENGTHS)).cuda()
    at = torch.arange(T, device="cuda")
    z = z.masked_fill((seq[:, None] != seq[None, :]) | (at[None, :] > at[:, None]), -math.inf)
    o = torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v).reshape(T, -1)
    x1 = x + o @ wo.t()
    n2 = norm(x1)
    logits = n2 @ wr.t()
    gates = torch.softmax(logits.gather(1, idx), 1)
    y = torch.zeros_like(x1)
    for e in range(EXPERTS):
        token, slot = (idx == e).nonzero(as_tuple=True)
        g, u = (n2[token] @ wgu[e * 2 * FFN:(e + 1) * 2 * FFN].t()).chunk(2, 1)
        h = torch.nn.functional.silu(g) * u
        y = y.index_add(0, token, (h @ wdn[e * HIDDEN:(e + 1) * HIDDEN].t()) * gates[token, slot][:, None])
    share = torch.bincount(idx.reshape(-1), minlength=EXPERTS).double() / (2 * T)
    loss = (x1 + y).pow(2).mean() + COEF * EXPERTS * (share * torch.softmax(logits, 1).mean(0)).sum()
    return loss.detach(), torch.autograd.grad(loss, (x, wqkv, wo, wr, wgu, wdn))


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_step_matches_float64(optimizer):
    from megray_b200.ops import gemm_error_flag

    torch.manual_seed(0)
    layer = Layer(optimizer)
    x = torch.randn(T, HIDDEN, device="cuda").bfloat16()
    weights = [layer.wqkv, layer.wo, layer.wr, layer.moe.w_gu, layer.moe.w_down]
    before = [w.clone() for w in weights]
    # the reference needs the weights of before the step and the experts that it chose: one pass to choose them
    loss, dx, grads = layer.step(x, 1)
    after = [w.clone() for w in weights]
    for w, b in zip(weights, before):
        w.copy_(b)
    want_loss, want = reference(x, layer)
    torch.cuda.synchronize()
    assert int(gemm_error_flag().item()) == 0 and not layer.moe.ep.overflowed()
    assert int(layer.moe.expert_counts.sum()) == 2 * T
    # values pass through about a dozen roundings to bf16 on their way, each off by at most 2^-8 of them
    close = lambda a, b: float((a.double() - b).norm()) <= 12 * 2.0 ** -8 * float(b.norm())  # noqa: E731
    assert abs(float(loss) - float(want_loss)) <= 12 * 2.0 ** -8 * abs(float(want_loss))
    got = [dx, *grads, layer.moe.g_gu, layer.moe.g_down]
    for name, a, b in zip(("dx", "wqkv", "wo", "wr", "w_gu", "w_down"), got, want):
        assert close(a, b), name
    # the first AdamW step moves every weight by lr g / (|g| + eps), to a rounding
    for name, w, b, g in zip(("wqkv", "wo", "wr", "w_gu", "w_down"), after, before, got[1:]):
        g = g.double()
        step = b.double() - 1e-3 * g / (g.abs() + 1e-8)
        half = 2.0 ** -8 if w.dtype == torch.bfloat16 else 2.0 ** -24
        assert bool(((w.double() - step).abs() <= step.abs() * half + 1e-3 * 2.0 ** -20).all()), name


def test_more_steps_run():
    layer = Layer("adamw8")
    x = torch.randn(T, HIDDEN, device="cuda").bfloat16()
    for t in (1, 2, 3):
        loss, dx, _ = layer.step(x, t)
        assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(dx).all())
    assert layer.moe.steps == 3


def test_an_expert_layer_without_the_new_options_is_as_it_was():
    from megray_b200.models import MoEConfig, MoELayer

    cfg = MoEConfig(experts=4, hidden=256, ffn=128, tokens=200, capacity_factor=4.0)
    layer = MoELayer(cfg)
    assert layer.adamw is None
    layer.forward(torch.randn(200, 256, device="cuda").bfloat16(), torch.randn(200, 4, device="cuda"))
    layer.backward(torch.randn(200, 256, device="cuda").bfloat16())
    assert layer.balance_loss is None and layer._logits is None
    with pytest.raises(ValueError):
        MoELayer(MoEConfig(experts=4, hidden=256, ffn=128, tokens=200, optimizer="adam"))
