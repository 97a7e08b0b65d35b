"""Packed attention and its backward pass against float64: lengths around the tiles, one token, empty sequences,
grouped heads, odd head sizes, strided operands, rows behind the last sequence, refusals."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
HALF = {BF: 2.0 ** -8, HF: 2.0 ** -11}  # half a step, relative


def ends(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).cuda()


def make(lengths, heads, kv_heads, dim, dtype, tail=0, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(lengths) + tail
    r = lambda h: (torch.randn(rows, h, dim, generator=g, device="cuda") * scale).to(dtype)  # noqa: E731
    return r(heads), r(kv_heads), r(kv_heads), r(heads)


def reference(q, k, v, do, lengths, causal, scale=None):
    """out, lse, dq, dk, dv in float64 with, for each, the sum of absolute values of what was added up (the size to
    which a rounded probability or score gradient counts)."""
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    h, hk = q.shape[1], k.shape[1]
    val = {n: torch.zeros_like(t, dtype=torch.float64) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    size = {n: torch.zeros_like(t) for n, t in val.items()}
    lse = torch.full((h, q.shape[0]), math.nan, dtype=torch.float64, device=q.device)
    b = 0
    for n in lengths:
        s, b = slice(b, b + n), b + n
        for i in range(h):
            j = i * hk // h
            Q, K, V, D = (t[s, x].double() for t, x in ((q, i), (k, j), (v, j), (do, i)))
            z = Q @ K.t() * scale
            if causal:
                z = z.masked_fill(torch.ones_like(z, dtype=torch.bool).triu(1), -math.inf)
            p = torch.softmax(z, 1)
            val["out"][s, i], size["out"][s, i] = p @ V, p @ V.abs()
            lse[i, s] = torch.logsumexp(z, 1)
            dp = D @ V.t()
            delta = (D * val["out"][s, i]).sum(1, keepdim=True)
            ds = p * (dp - delta)
            val["dv"][s, j] += p.t() @ D
            size["dv"][s, j] += p.t() @ D.abs()
            val["dq"][s, i] = scale * ds @ K
            val["dk"][s, j] += scale * ds.t() @ Q
            # delta is formed from the rounded output: off by half a step of every term
            da = p * (dp.abs() + delta.abs() + (D.abs() * size["out"][s, i]).sum(1, keepdim=True))
            size["dq"][s, i] = scale * da @ K.abs()
            size["dk"][s, j] += scale * da.t() @ Q.abs()
    return val, size, lse


# A probability (or score gradient) is rounded once to the operands' type, by half a step of itself; its exponent's
# argument is off by a few float32 steps of a score, 2^-13 in all here; the result is rounded once more.
def check(got, want, size, dtype, name):
    tol = want.abs() * HALF[dtype] + size * (HALF[dtype] + 2.0 ** -13) * 1.01 + (2.0 ** -24 if dtype == HF else 0.0)
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (name, float((off / tol).nan_to_num(0.0, 9e9, 9e9).max()))


def run_and_check(lengths, heads, kv_heads, dim, dtype, causal, tail=0, backward=True, scale=None, seed=0):
    from megray_b200.ops import attention, attention_bwd, gemm_error_flag

    q, k, v, do = make(lengths, heads, kv_heads, dim, dtype, tail, seed)
    n = sum(lengths)
    for t in (q, k, v, do):
        t[n:] = float("nan")  # what lies behind the last sequence reaches nothing
    cu = ends(lengths)
    out = torch.full_like(q, 7.0)
    lse = torch.full((heads, n + tail), 7.0, device="cuda")
    attention(q, k, v, cu, causal=causal, scale=scale, out=out, lse=lse)
    val, size, lse_want = reference(q, k, v, do, lengths, causal, scale)
    torch.cuda.synchronize()
    assert int(gemm_error_flag().item()) == 0
    check(out[:n], val["out"][:n], size["out"][:n], dtype, "out")
    # scores are sums of up to 128 products, the exponent's argument a few steps off
    assert bool(((lse[:, :n].double() - lse_want[:, :n]).abs() <= 2.0 ** -14).all())
    assert bool((out[n:] == 7.0).all()) and bool((lse[:, n:] == 7.0).all())
    if not backward:
        return
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    attention_bwd(do, q, k, v, out, lse, cu, causal=causal, scale=scale, dq=grads[0], dk=grads[1], dv=grads[2])
    torch.cuda.synchronize()
    assert int(gemm_error_flag().item()) == 0
    for g, name in zip(grads, ("dq", "dk", "dv")):
        check(g[:n], val[name][:n], size[name][:n], dtype, name)
        assert bool((g[n:] == 7.0).all())


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", [[1], [2], [16], [127], [128], [129], [255], [256], [257], [384], [700]])
def test_one_sequence(lengths, causal):
    run_and_check(lengths, 2, 1, 64, BF, causal)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 80, 96, 112, 120, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_head_sizes(dim, dtype, causal):
    run_and_check([130, 1, 61], 2, 2, dim, dtype, causal, tail=3, seed=dim)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (4, 2), (6, 3), (7, 1), (8, 8), (12, 4), (16, 1)])
def test_grouped_heads(heads, kv_heads, causal):
    run_and_check([300, 77], heads, kv_heads, 64, BF, causal, tail=1)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,tail", [([0, 5, 0, 0, 130, 1, 0], 9), ([1] * 40, 0), ([3, 129, 260, 128, 17], 200),
                                          (list(range(1, 70)), 0), ([1000, 1, 513], 64)])
def test_many_sequences(lengths, tail, causal):
    run_and_check(lengths, 2, 1, 128, BF, causal, tail=tail)


@gpu
@pytest.mark.parametrize("causal,dtype,dim", [(True, BF, 128), (False, HF, 128), (True, HF, 64), (False, BF, 80)])
def test_long_sequences(causal, dtype, dim):
    run_and_check([2500, 1111], 4, 2, dim, dtype, causal, seed=5)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([1900, 1800], 8, 8), ([1000, 30], 8, 1), ([1500], 6, 2), ([64] * 30, 4, 4)])
def test_tiles_shared_and_not_shared_by_several_ctas(lengths, heads, kv_heads, causal):
    run_and_check(lengths, heads, kv_heads, 64, BF, causal, tail=5, seed=11)


@gpu
@pytest.mark.parametrize("scale", [2.0 ** -20, 0.5, 3.0])
def test_scales(scale):
    from megray_b200.ops import attention

    # a large scale makes the maximum jump from block to block, which rescales the accumulator
    lengths = [600, 200]
    q, k, v, do = make(lengths, 2, 1, 64, BF, seed=3)
    k *= torch.linspace(0.1, 1.5, sum(lengths), device="cuda").to(BF)[:, None, None]
    out, lse = attention(q, k, v, ends(lengths), causal=True, scale=scale)
    val, size, lse_want = reference(q, k, v, do, lengths, True, scale)
    # scores of up to 40 x scale, each off by 2^-20 of the sum of absolute products
    off = (q.double().abs().amax() * k.double().abs().amax() * 64 * scale * 2.0 ** -22)
    tol = val["out"].abs() * HALF[BF] + size["out"] * (HALF[BF] + 2 * float(off) + 2.0 ** -13)
    assert bool(((out.double() - val["out"]).abs() <= tol).all())
    assert bool(((lse.double() - lse_want).abs() <= 2.0 ** -14 + 2 * float(off)).all())


@gpu
def test_a_peak_in_every_block():
    """One key per block of 128 outweighs everything before it: the maximum moves in every block."""
    from megray_b200.ops import attention

    n = 1024
    q = torch.ones(n, 1, 64, device="cuda", dtype=BF)
    k = torch.zeros(n, 1, 64, device="cuda", dtype=BF)
    for b in range(8):
        k[b * 128 + 60] = 1.0 + 4 * b
    v = torch.randn(n, 1, 64, device="cuda").to(BF)
    out, lse = attention(q, k, v, causal=True)
    val, size, lse_want = reference(q, k, v, q, [n], True)
    check(out, val["out"], size["out"], BF, "out")
    assert bool(((lse.double() - lse_want).abs() <= 2.0 ** -12).all())  # scores up to 232: half steps of 2^-17


@gpu
def test_strided_operands():
    from megray_b200.ops import attention, attention_bwd

    rows, h, hk, d = 333, 4, 2, 72
    qkv = torch.randn(rows, h + 2 * hk, d, device="cuda").to(BF)
    parts = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    plain = [t.contiguous() for t in parts]
    do = torch.randn(h, rows, d, device="cuda").to(BF).transpose(0, 1)  # heads outermost
    cu = ends([200, 133])
    out, lse = attention(*parts, cu)
    out2, lse2 = attention(*plain, cu)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    grad = torch.zeros(rows, h + 2 * hk, d, device="cuda", dtype=BF)
    views = grad[:, :h], grad[:, h:h + hk], grad[:, h + hk:]
    attention_bwd(do, *parts, out, lse, cu, dq=views[0], dk=views[1], dv=views[2])
    for a, b in zip(views, attention_bwd(do.contiguous(), *plain, out2, lse2, cu)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("count", [31, 32, 33, 200, 1023, 1500])
def test_more_sequences_than_a_search_step_holds(count):
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 4, (count,), generator=g).tolist()
    lengths[count // 2] = 300
    run_and_check(lengths, 2, 1, 16, BF, True, tail=7)


@gpu
def test_rows_that_are_no_multiple_of_the_heads():
    from megray_b200.ops import attention, attention_bwd

    rows, h, d = 150, 4, 32
    store = torch.randn(rows, h * d + 8, device="cuda").to(BF)
    x = store[:, :h * d].view(rows, h, d)
    out, lse = attention(x, x, x)
    plain = x.contiguous()
    want, want_lse = attention(plain, plain, plain)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    for a, b in zip(attention_bwd(out, x, x, x, out, lse), attention_bwd(want, plain, plain, plain, want, want_lse)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("hidden", [100, 128, 200, 300])
def test_scores_of_minus_infinity(hidden):
    """Keys that give a score of -infinity to every query have no weight, also where they fill the first blocks."""
    from megray_b200.ops import attention

    n = 400
    q, k, v, _ = make([n], 1, 1, 64, BF, seed=2)
    q[..., 0] = q[..., 0].abs() + 0.5
    k[:hidden, :, 0] = float("-inf")
    out, lse = attention(q, k, v, causal=False)
    z = q[:, 0].double() @ k[hidden:, 0].double().t() / 8
    p = torch.softmax(z, 1)
    check(out[:, 0], p @ v[hidden:, 0].double(), p @ v[hidden:, 0].double().abs(), BF, "out")
    assert bool(((lse[0].double() - torch.logsumexp(z, 1)).abs() <= 2.0 ** -14).all())


@gpu
def test_other_sequences_do_not_matter():
    from megray_b200.ops import attention, attention_bwd

    lengths = [100, 200, 50]
    q, k, v, do = make(lengths, 2, 1, 64, BF)
    s = slice(100, 300)
    alone = attention(q[s], k[s], v[s])
    alone_bwd = attention_bwd(do[s], q[s], k[s], v[s], *alone)
    for t in (q, k, v, do):
        t[:100] = float("nan")
        t[300:] = float("inf")
    out, lse = attention(q, k, v, ends(lengths))
    grads = attention_bwd(do, q, k, v, out, lse, ends(lengths))
    assert torch.equal(out[s], alone[0]) and torch.equal(lse[:, s], alone[1])
    for a, b in zip(grads, alone_bwd):
        assert torch.equal(a[s], b)


@gpu
def test_gradients_against_differences():
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = (t.to(HF) for t in make([70, 9], 2, 1, 32, HF, seed=8))
    cu = ends([70, 9])
    out, lse = attention(q, k, v, cu)
    grads = attention_bwd(do, q, k, v, out, lse, cu)
    # along a direction, by the definition in float64 (the kernel's own output is too coarse to difference)
    for x, g in zip((0, 1, 2), grads):
        way = torch.randn(g.shape, device="cuda", dtype=torch.float64)
        loss = []
        for s in (1, -1):
            a = [q.double(), k.double(), v.double()]
            a[x] = a[x] + s * 2.0 ** -10 * way
            val, _, _ = reference(*a, do, [70, 9], True)
            loss.append(float((val["out"] * do.double()).sum()))
        slope = (loss[0] - loss[1]) / 2.0 ** -9
        got = float((g.double() * way).sum())
        # every gradient is off by at most 2^-9 of terms whose sum is below |g|_1 + 64
        assert abs(got - slope) <= 2.0 ** -9 * (float((g.double().abs() * way.abs()).sum()) + 64)


@gpu
def test_the_same_bits_every_time_and_from_a_graph():
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make([500, 300], 4, 2, 128, BF)
    cu = ends([500, 300])
    first = [*attention(q, k, v, cu)]
    first += attention_bwd(do, q, k, v, *first, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [*attention(q, k, v, cu)]
        got += attention_bwd(do, q, k, v, *got, cu)
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    # a graph follows the offsets: they are read on the device
    cu.copy_(ends([300, 500]))
    graph.replay()
    again = [*attention(q, k, v, cu)]
    assert torch.equal(got[0], again[0]) and not torch.equal(got[0], first[0])


@gpu
def test_two_streams_at_once():
    from megray_b200.ops import attention, attention_bwd

    sets = [make([400, 150], 4, 2, 64, BF, seed=s) for s in (1, 2)]
    cu = ends([400, 150])
    want = [[*attention(q, k, v, cu)] for q, k, v, _ in sets]
    want = [w + [*attention_bwd(do, q, k, v, *w, cu)] for w, (q, k, v, do) in zip(want, sets)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for stream, (q, k, v, do) in zip(streams, sets):
        with torch.cuda.stream(stream):
            o = [*attention(q, k, v, cu)]
            got.append(o + [*attention_bwd(do, q, k, v, *o, cu)])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_offsets_out_of_range_touch_nothing_outside():
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make([256], 1, 1, 64, BF)
    for bad in ([-5, 100, 9000], [200, 100, 50], [0, 2 ** 31 - 1, -2 ** 31], [300, 400, 500]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out, lse = attention(q, k, v, cu)
        attention_bwd(do, q, k, v, torch.zeros_like(out), torch.zeros_like(lse), cu)
    torch.cuda.synchronize()


@gpu
def test_no_rows():
    from megray_b200.ops import attention, attention_bwd

    q = torch.zeros(0, 2, 64, device="cuda", dtype=BF)
    out, lse = attention(q, q, q)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    assert all(g.shape == (0, 2, 64) for g in attention_bwd(q, q, q, q, out, lse))
    q = torch.zeros(5, 2, 64, device="cuda", dtype=BF)
    attention(q, q, q, torch.zeros(4, dtype=torch.int32, device="cuda"))  # only empty sequences
    torch.cuda.synchronize()


@gpu
def test_refusals():
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make([64], 4, 2, 64, BF)
    cu = ends([64])
    wide = torch.zeros(64, 4, 68, device="cuda", dtype=BF)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(k=k.half()), dict(k=k[:5]), dict(v=v[:, :1]), dict(k=k[:, :0], v=v[:, :0]),
                dict(k=q[:, :3], v=q[:, :3]), dict(q=wide[..., :60], k=wide[:, :2, :60], v=wide[:, :2, :60]),
                dict(q=wide[..., 4:68]), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(cu_seqlens=cu.long()),
                dict(cu_seqlens=cu[:1]), dict(cu_seqlens=cu.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                dict(scale=math.inf), dict(out=q[:5]), dict(out=q[:, :1].expand(64, 4, 64)), dict(lse=torch.zeros(4, 63, device="cuda")),
                dict(lse=torch.zeros(64, 4, device="cuda").t()), dict(q=q.cpu())):
        kw = {"q": q, "k": k, "v": v, "cu_seqlens": cu, **bad}
        with pytest.raises(ValueError):
            attention(kw.pop("q"), kw.pop("k"), kw.pop("v"), kw.pop("cu_seqlens"), **kw)
    big = torch.zeros(8, 1, 136, device="cuda", dtype=BF)
    with pytest.raises(ValueError):
        attention(big, big, big)
    out, lse = attention(q, k, v, cu)
    for same in (k, v):
        with pytest.raises(ValueError):
            attention(k, k, v, cu, out=same)
    for bad in (dict(dout=do[:5]), dict(dout=do.half()), dict(out=None), dict(lse=None), dict(lse=lse[:2]), dict(dk=q), dict(dq=k),
                dict(dq=q), dict(dq=do), dict(dk=v)):
        kw = {"dout": do, "out": out, "lse": lse, **bad}
        with pytest.raises(ValueError):
            attention_bwd(kw.pop("dout"), q, k, v, kw.pop("out"), kw.pop("lse"), cu, **kw)


@gpu
def test_results_in_one_place_are_refused():
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make([64], 2, 2, 64, BF)
    out, lse = attention(q, k, v)
    both, third = torch.empty_like(k), torch.empty_like(k)
    for grads in (dict(dk=both, dv=both), dict(dq=both, dk=both), dict(dq=both, dk=third, dv=both)):
        with pytest.raises(ValueError):
            attention_bwd(do, q, k, v, out, lse, **grads)
    attention_bwd(do, q, k, v, out, lse, dq=torch.empty_like(q), dk=both, dv=third)
    other = q.as_strided(q.shape, (64, 64 * 64, 1))  # the same memory, head by head
    with pytest.raises(ValueError):
        attention(q, k, v, out=other)


@gpu
@pytest.mark.parametrize("lens,heads,kv_heads,causal", [([1], 2, 2, True), ([200, 1, 129, 70], 4, 2, False), ([2500, 40, 1300], 16, 4, True)])
def test_the_output_may_take_the_place_of_the_queries(lens, heads, kv_heads, causal):
    from megray_b200.ops import attention

    q, k, v, _ = make(lens, heads, kv_heads, 64, BF)
    cu = ends(lens)
    want, want_lse = attention(q, k, v, cu, causal=causal)
    over = q.clone()
    got, lse = attention(over, k, v, cu, causal=causal, out=over)
    assert got is over and torch.equal(got, want) and torch.equal(lse, want_lse)


def test_cpu_tensors_are_refused():
    from megray_b200.ops import attention, attention_bwd

    q = torch.zeros(4, 2, 64, dtype=BF)
    with pytest.raises(ValueError):
        attention(q, q, q)
    with pytest.raises(ValueError):
        attention_bwd(q, q, q, q, q, torch.zeros(2, 4))


def test_bad_arguments_of_the_c_entry_are_refused_before_any_launch():
    from megray_b200 import _lib

    lib = _lib.load()
    t = _lib.AttnTensor(1024, 128, 64)
    ok = dict(cu=None, dtype=10, tokens=4, heads=2, kv_heads=1, dim=64, seqs=1, causal=1, scale=1.0, error_flag=None)
    fwd = lambda a, *ts: lib.megray_attention(a, *ts, 1024, None)  # noqa: E731
    assert fwd(None, t, t, t, t) == 6
    for bad in (dict(dtype=7), dict(tokens=-1), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(dim=60),
                dict(dim=136), dict(seqs=-1), dict(cu=1024, seqs=0), dict(cu=1025), dict(scale=0.0), dict(scale=float("nan")),
                dict(scale=float("inf"))):
        assert fwd(_lib.AttnArgs(**{**ok, **bad}), t, t, t, t) in (6, -1), bad
    a = _lib.AttnArgs(**ok)
    for bad in (_lib.AttnTensor(None, 128, 64), _lib.AttnTensor(1032, 128, 64), _lib.AttnTensor(1024, 124, 64),
                _lib.AttnTensor(1024, 128, 60), _lib.AttnTensor(1024, 0, 64), _lib.AttnTensor(1024, -128, 64), None):
        for i in range(4):
            ts = [t] * 4
            ts[i] = bad
            assert fwd(a, *ts) == -1
    assert lib.megray_attention(a, t, t, t, t, None, None) == -1
    assert lib.megray_attention_bwd(a, t, t, t, t, t, None, t, t, t, 1024, None) == -1
    assert lib.megray_attention_bwd(a, t, t, t, t, t, 1024, t, t, t, 1028, None) == -1
    assert lib.megray_attention_bwd_workspace(a) >= 4 * 8
    assert lib.megray_attention_bwd_workspace(_lib.AttnArgs(**{**ok, "dim": 60})) == 0
    assert lib.megray_attention_bwd_workspace(_lib.AttnArgs(**{**ok, "tokens": 0})) == 0
    assert lib.megray_attention_bwd(a, t, t, t, t, t, 1024, t, t, t, None, None) == -1
    assert fwd(_lib.AttnArgs(**{**ok, "tokens": 0}), t, t, t, t) == 0


@gpu
@pytest.mark.parametrize("rows,heads,kv_heads", [(60_000, 32, 8), (2000, 8, 1)])
def test_nothing_is_under_way_after_a_backward_pass_over_empty_sequences(rows, heads, kv_heads):
    """The workspace goes back to the allocator with the call: what is put in its place on the same stream stays."""
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make([], heads, kv_heads, 64, BF, tail=rows)
    cu = torch.zeros(5, dtype=torch.int32, device="cuda")
    out, lse = attention(q, k, v, cu)
    for _ in range(10):
        grads = attention_bwd(do, q, k, v, out, lse, cu)
        next_ones = [torch.full((heads, rows), 7.0, device="cuda") for _ in range(3)]
        assert all(bool((t == 7.0).all()) for t in next_ones)
        assert all(not bool(g.any()) for g in grads)
    assert not bool(out.any()) and not bool(lse.any())


@gpu
def test_rows_whose_scores_are_minus_infinity_beside_others():
    """Causal queries in front of the first key that has a weight: nothing to divide by, and the rows behind them, in
    the same warps, are as without the keys in front."""
    from megray_b200.ops import attention

    n, hidden = 400, 130
    q, k, v, _ = make([n], 1, 1, 64, BF, seed=2)
    q[..., 0] = q[..., 0].abs() + 0.5
    k[:hidden, :, 0] = float("-inf")
    out, lse = attention(q, k, v, causal=True)
    assert bool(torch.isneginf(lse[0, :hidden]).all()) and bool(torch.isnan(out[:hidden]).all())
    z = q[hidden:, 0].double() @ k[hidden:, 0].double().t() / 8
    z = z.masked_fill(torch.ones_like(z, dtype=torch.bool).triu(1), -math.inf)
    p = torch.softmax(z, 1)
    check(out[hidden:, 0], p @ v[hidden:, 0].double(), p @ v[hidden:, 0].double().abs(), BF, "out")
    assert bool(((lse[0, hidden:].double() - torch.logsumexp(z, 1)).abs() <= 2.0 ** -14).all())


@gpu
def test_scores_that_overflow_for_every_other_query():
    """The first 256 keys score -infinity for even queries; for odd ones the second block outweighs the first by far, so
    that half the rows of every warp rescale what the others have not begun."""
    from megray_b200.ops import attention

    n = 512
    q, k, v, _ = make([n], 1, 1, 64, BF, seed=4)
    q[..., :2] = k[..., :2] = 0.0
    q[::2, :, 0], k[:256, :, 0] = 2.0 ** 100, -2.0 ** 100
    q[1::2, :, 1], k[128:256, :, 1] = 8.0, 200.0
    out, lse = attention(q, k, v, causal=False)
    z = q[:, 0].double() @ k[:, 0].double().t() / 8
    z[::2, :256] = -math.inf
    p = torch.softmax(z, 1)
    check(out[:, 0], p @ v[:, 0].double(), p @ v[:, 0].double().abs(), BF, "out")
    assert bool(((lse[0].double() - torch.logsumexp(z, 1)).abs() <= 2.0 ** -12).all())  # scores up to 200


@gpu
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,size,scale", [(BF, 2.0 ** 11, None), (BF, 2.0 ** 17, None), (BF, 2.0 ** 40, 0.3), (BF, 2.0 ** 62, None),
                                              (HF, 2.0 ** 14, 2.0 ** 8)])
@pytest.mark.parametrize("first", [100, 128, 300])
def test_finite_scores_of_any_size(first, dtype, size, scale, causal, sign):
    """Scores far from zero, exact in float32: keys with the same one share a row evenly, those far below have no part in it,
    whichever come first."""
    from megray_b200.ops import attention

    n = 500
    q, k, v, _ = make([n], 2, 1, 64, dtype, seed=6)
    q[::2], q[1::2, :, 0] = 0.0, 0.0  # odd queries see ordinary scores
    q[::2, :, 0], k[:, :, 0] = size * 1.0078125, 0.0
    k[:first, :, 0] = sign * size * 1.3359375
    out, lse = attention(q, k, v, causal=causal, scale=scale)
    val, weight, want = reference(q, k, v, q, [n], causal, scale)
    off = 64 * 16.0 * (0 if scale is None else scale) * 2.0 ** -22  # ordinary scores times a large scale
    tol = val["out"].abs() * HALF[dtype] + weight["out"] * (HALF[dtype] + 2 * off + 2.0 ** -13) * 1.01 + (2.0 ** -24 if dtype == HF else 0.0)
    assert bool(((out.double() - val["out"]).abs() <= tol).all())
    assert bool(((lse.double() - want).abs() <= 2.0 ** -14 + 2 * off + want.abs() * 2.0 ** -22).all())


def test_rows_and_sequences_whose_ends_would_pass_32_bits_are_refused():
    from megray_b200 import _lib

    size = lambda rows, seqs=1: _lib.load().megray_attention_bwd_workspace(  # noqa: E731
        _lib.AttnArgs(cu=1024, dtype=10, tokens=rows, heads=1, kv_heads=1, dim=8, seqs=seqs, causal=1, scale=1.0))
    assert size(2 ** 31 - 513) >= 4 * (2 ** 31 - 513)
    assert size(2 ** 31 - 512) == 0 and size(2 ** 31 - 1) == 0 and size(8, 2 ** 31 - 1) == 0


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 1)])  # the second shares tiles between CTAs
def test_nothing_is_written_outside_whatever_the_offsets(heads, kv_heads):
    """Results in the middle of larger buffers: what lies around them, and the inputs, stay as they were."""
    from megray_b200.ops import attention, attention_bwd, gemm_error_flag

    rows, dim = 700, 64
    q, k, v, do = make([rows], heads, kv_heads, dim, BF)
    kept = [t.clone() for t in (q, k, v, do)]
    def inside(h):
        store = torch.full((rows + 512, h + 2, dim), 7.0, device="cuda", dtype=BF)
        return store, store[256:256 + rows, 1:1 + h]
    for bad in ([0, 300, 700], [-5, 100, 9000], [200, 100, 50], [0, 2 ** 31 - 1, -2 ** 31], [300, 400, 500], [900, 950, 1000],
                [700, 700, 0, 700]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        stores = [inside(h) for h in (heads, heads, kv_heads, kv_heads)]
        lse = torch.full((heads + 2, rows), 7.0, device="cuda")
        attention(q, k, v, cu, out=stores[0][1], lse=lse[1:1 + heads])
        attention_bwd(do, q, k, v, stores[0][1], lse[1:1 + heads], cu, dq=stores[1][1], dk=stores[2][1], dv=stores[3][1])
        torch.cuda.synchronize()
        assert int(gemm_error_flag().item()) == 0
        for store, view in stores:
            view.fill_(7.0)
            assert bool((store == 7.0).all()), bad
        assert bool((lse[0] == 7.0).all()) and bool((lse[-1] == 7.0).all()), bad
        assert all(torch.equal(a, b) for a, b in zip((q, k, v, do), kept)), bad


@gpu
@pytest.mark.parametrize("scale", [0.05, 0.3])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,dtype", [([300, 77], 4, 2, 64, BF), ([1000, 30], 8, 1, 64, BF), ([500], 6, 2, 80, HF)])
def test_gradients_at_other_scales(lengths, heads, kv_heads, dim, dtype, scale):
    run_and_check(lengths, heads, kv_heads, dim, dtype, True, tail=3, scale=scale, seed=21)


@gpu
@pytest.mark.parametrize("lengths,heads,kv_heads,tail", [([300, 1, 77], 4, 2, 9), ([1000, 30], 8, 1, 0), ([0, 40, 0], 2, 2, 200)])
def test_results_that_the_call_makes(lengths, heads, kv_heads, tail):
    """Without given tensors: the same results, and zeros behind the last sequence."""
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make(lengths, heads, kv_heads, 64, BF, tail, seed=5)
    n, cu = sum(lengths), ends(lengths)
    for t in (q, k, v, do):
        t[n:] = float("nan")
    torch.full((1 << 22,), float("nan"), device="cuda")  # what a fresh tensor may hold
    out, lse = attention(q, k, v, cu)
    val, size, lse_want = reference(q, k, v, do, lengths, True)
    check(out[:n], val["out"][:n], size["out"][:n], BF, "out")
    assert bool(((lse[:, :n].double() - lse_want[:, :n]).abs() <= 2.0 ** -14).all())
    assert not bool(out[n:].any()) and not bool(lse[:, n:].any())
    for g, name in zip(attention_bwd(do, q, k, v, out, lse, cu), ("dq", "dk", "dv")):
        check(g[:n], val[name][:n], size[name][:n], BF, name)
        assert not bool(g[n:].any())


@gpu
@pytest.mark.parametrize("shift", [100.0, 3000.0, 20000.0])
def test_gradients_of_scores_far_from_zero(shift):
    """The backward pass takes probabilities from the scores and lse, both of about ``shift``: a score is four sums of
    16 products, each cut or rounded to float32 (2^-23 of it), and the exponent is off by a half step of lse, of its
    product with log2 e and of the scores' factor: below 2^-20 of ``shift`` in all."""
    from megray_b200.ops import attention, attention_bwd

    q, k, v, do = make([300], 2, 1, 64, BF, seed=9)
    q[..., 0], k[..., 0] = 32.0, shift / 4 if shift < 1000 else 1024.0 * round(shift / 4096)
    out, lse = attention(q, k, v)
    val, size, lse_want = reference(q, k, v, do, [300], True)
    far = float(lse_want.abs().max())
    more = far * 2.0 ** -20
    assert bool(((lse.double() - lse_want).abs() <= 2.0 ** -14 + more).all())
    for g, name in zip((out, *attention_bwd(do, q, k, v, out, lse)), ("out", "dq", "dk", "dv")):
        tol = val[name].abs() * HALF[BF] + size[name] * (HALF[BF] + 2.0 ** -13 + 2 * more) * 1.01
        assert bool(((g.double() - val[name]).abs() <= tol).all()), name
