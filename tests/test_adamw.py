"""AdamW over a list of tensors against float64: odd sizes, tensors off the 16-byte boundary, long lists, both
moment forms, missing gradients, device-side numbers, graphs and refusals."""
import pytest
import torch

H = {"lr": 1e-2, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1, "grad_scale": 0.5}
U = 2.0 ** -24  # half a step of float32
gpu = pytest.mark.gpu


def make(sizes, pt, gt, bits, shift=0, seed=0):
    from megray_b200.ops import AdamWState

    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, dt, s: torch.empty(n + shift, device="cuda").normal_(0, s, generator=g).to(dt)[shift:]  # noqa: E731
    params, grads = [r(n, pt, 0.02) for n in sizes], [r(n, gt, 0.01) for n in sizes]
    state = AdamWState(params, bits=bits)
    return params, grads, state


def moments(state, i):
    """The float64 values of tensor i's moments and, in 8 bits, its blocks' scales."""
    b, n = state.begins[i], state.sizes[i]
    if state.bits == 32:
        return state.m[b:b + n].double(), state.v[b:b + n].double()
    per = lambda x, s: (x.float().double().view(-1, 256) * s.double()[:, None]).view(-1)[b:b + n]  # noqa: E731
    return per(state.m, state.m_scale), per(state.r, state.r_scale) ** 2


def want_step(p, g, m, v, step, h=H):
    """The formula in float64 with a bound on the float32 evaluation: every operation is off by half a step."""
    (b1, b2), lr = h["betas"], h["lr"]
    g = g.double() * h["grad_scale"]
    size_m = (b1 * m).abs() + ((1 - b1) * g).abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    d = (v / (1 - b2 ** step)).sqrt() + h["eps"]
    rate = lr / (1 - b1 ** step)
    out = p.double() * (1 - lr * h["weight_decay"]) - rate * m / d
    err_m = 6 * U * size_m          # two constants, gradient scaling, two products, a sum
    err_v = 8 * U * v               # all terms are positive
    err_p = rate * (err_m / d + 12 * U * m.abs() / d) + 4 * U * (p.double().abs() + out.abs())
    return out, m, v, err_p, err_m, err_v


def check(params, before, grads, state, old, step, h=H):
    for i, (p, p0, g) in enumerate(zip(params, before, grads)):
        if not p.numel():
            continue
        out, m, v, err_p, err_m, err_v = want_step(p0, g, *old[i], step, h)
        tol = err_p + (out.abs() + err_p) * 2.0 ** -8 if p.dtype == torch.bfloat16 else err_p
        assert bool(((p.double() - out).abs() <= tol).all()), i
        got_m, got_v = moments(state, i)
        if state.bits == 32:
            assert bool(((got_m - m).abs() <= err_m).all()) and bool(((got_v - v).abs() <= err_v).all()), i
            continue
        # e4m3: half a step is 2^-4 of a number, or 2^-10 below 2^-6, in units of the block's scale
        pad = lambda x: torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256)  # noqa: E731
        for got, x, low, err in ((got_m, m, 2.0 ** -10, err_m), (got_v.sqrt(), v.sqrt(), 2.0 ** -9, 8 * U * v.sqrt())):
            scale = pad(x).abs().amax(1, keepdim=True) / 448
            tol = torch.maximum(pad(x).abs() * 2.0 ** -4, scale * low) * (1 + 2.0 ** -10) + 2 * pad(err) + scale * 2.0 ** -14
            assert bool(((pad(got) - pad(x)).abs() <= tol).all()), i
        assert bool((got_v[v > 0] > 0).all())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_three_steps(bits, pt, gt, shift):
    from megray_b200.ops import adamw_step

    sizes = [1, 7, 8, 255, 256, 257, 0, 2047, 2048, 2049, 30_011]
    params, grads, state = make(sizes, pt, gt, bits, shift)
    copies = [torch.zeros(n + shift, dtype=torch.bfloat16, device="cuda")[shift:] for n in sizes]
    for step in (1, 2, 3):
        before, old = [p.clone() for p in params], [moments(state, i) for i in range(len(sizes))]
        adamw_step(params, grads, state, step=step, copies=copies, **H)
        check(params, before, grads, state, old, step)
        for p, c in zip(params, copies):
            assert torch.equal(p.to(torch.bfloat16), c)
        grads = [g.flip(0) * 1.5 if g.storage_offset() == 0 else g for g in grads]


@gpu
@pytest.mark.parametrize("count", [64, 65, 720, 721, 1500])
@pytest.mark.parametrize("bits", [32, 8])
def test_long_lists(count, bits):
    from megray_b200.ops import adamw_step

    sizes = [1 + (i * 37) % 700 for i in range(count)]
    params, grads, state = make(sizes, torch.float32, torch.bfloat16, bits, seed=count)
    before, old = [p.clone() for p in params], [moments(state, i) for i in range(count)]
    adamw_step(params, grads, state, step=5, **H)
    check(params, before, grads, state, old, 5)


@gpu
def test_the_split_of_the_work_changes_no_bit():
    from megray_b200.ops import AdamWState, adamw_step

    n = 256 * 40 + 3
    params, grads, state = make([n], torch.float32, torch.float32, 8)
    parts = [p.clone() for p in params[0].split(256 * 8)]
    part_state = AdamWState(parts, bits=8)
    for step in (1, 2):
        adamw_step(parts, list(grads[0].split(256 * 8)), part_state, step=step, **H)
        adamw_step(params, grads, state, step=step, **H)
    assert torch.equal(torch.cat(parts), params[0])
    assert torch.equal(state.m.view(torch.uint8), part_state.m.view(torch.uint8))
    assert torch.equal(state.r.view(torch.uint8), part_state.r.view(torch.uint8))
    assert torch.equal(state.m_scale, part_state.m_scale) and torch.equal(state.r_scale, part_state.r_scale)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_zero_missing_and_bad_gradients(bits):
    from megray_b200.ops import adamw_step

    params, grads, state = make([600, 300, 700], torch.float32, torch.float32, bits)
    grads[0].zero_()
    grads[2][300] = float("nan")  # second block
    before = [p.clone() for p in params]
    adamw_step(params, [grads[0], None, grads[2]], state, step=1, **H)
    assert torch.equal(params[1], before[1]) and float(moments(state, 1)[1].abs().sum()) == 0.0
    assert float(moments(state, 0)[0].abs().sum()) == 0.0  # zero gradients leave zero moments: only the decay acts
    torch.testing.assert_close(params[0], before[0] * (1 - H["lr"] * H["weight_decay"]), rtol=4 * U, atol=0)
    bad = torch.isnan(params[2])
    assert bad.nonzero().flatten().tolist() == [300]
    m_bad = torch.isnan(moments(state, 2)[0]).nonzero().flatten().tolist()
    assert m_bad == ([300] if bits == 32 else list(range(256, 512)))


@gpu
@pytest.mark.parametrize("reach", [40, 60])  # 60 goes past the range of the root's own iteration
def test_roots_against_float64(reach):
    """A block's scale of r is its largest root over 448: the root is at most one float32 step off (2 U of its value),
    1 / 448 and the product half a step each."""
    from megray_b200.ops import AdamWState, adamw_step

    g = torch.Generator(device="cuda").manual_seed(3)
    blocks = 20_000
    x = (1 + torch.rand(blocks, device="cuda", generator=g)) * 2.0 ** torch.randint(-reach, reach, (blocks,), device="cuda", generator=g)
    grad, param = x[:, None].expand(blocks, 256).reshape(-1).contiguous(), torch.zeros(blocks * 256, device="cuda")
    state = AdamWState([param], bits=8)
    adamw_step([param], [grad], state, 1e-3, step=1, betas=(0.9, 0.95))
    v = (x * x) * torch.tensor(1.0 - 0.95, dtype=torch.float32, device="cuda")
    want = v.double().sqrt() / 448
    assert ((state.r_scale.double() - want).abs() <= 4 * U * (1 + 1e-6) * want).all()


@gpu
def test_mixed_types_and_nothing_to_do():
    from megray_b200.ops import AdamWState, adamw_step

    params = [torch.randn(100, device="cuda"), torch.randn(300, device="cuda").bfloat16(), torch.randn(5, device="cuda")]
    grads = [torch.randn(100, device="cuda"), torch.randn(300, device="cuda").bfloat16(),
             torch.randn(5, device="cuda").bfloat16()]
    state = AdamWState(params, bits=32)
    before, old = [p.clone() for p in params], [moments(state, i) for i in range(3)]
    adamw_step(params, [None] * 3, state, step=1, **H)
    assert all(torch.equal(a, b) for a, b in zip(params, before))
    adamw_step(params, grads, state, step=1, **H)
    check(params, before, grads, state, old, 1)


@gpu
def test_a_captured_step_follows_the_numbers_on_the_device():
    from megray_b200.ops import adamw_step

    params, grads, state = make([1000, 333], torch.float32, torch.float32, 32)
    lr, step, scale = (torch.tensor([x], device="cuda") for x in (1e-2, 0.0, 0.5))
    h = {**H, "lr": lr, "grad_scale": scale}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.add_(1.0)
        adamw_step(params, grads, state, step=step, **h)
    for t in (1, 2, 3):
        before, old = [p.clone() for p in params], [moments(state, i) for i in range(2)]
        lr.fill_(1e-2 / t)
        graph.replay()
        check(params, before, grads, state, old, t, {**H, "lr": float(lr)})


@gpu
def test_another_stream():
    from megray_b200.ops import adamw_step

    params, grads, state = make([100_000], torch.bfloat16, torch.bfloat16, 8)
    before, old = [p.clone() for p in params], [moments(state, 0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adamw_step(params, grads, state, step=2, **H)
    side.synchronize()
    check(params, before, grads, state, old, 2)


@gpu
def test_refusals():
    from megray_b200.ops import AdamWState, adamw_step

    params, grads, state = make([64, 8], torch.float32, torch.float32, 32)
    before = [p.clone() for p in params]
    for bad in (dict(grads=grads[:1]), dict(grads=[grads[0], grads[1][:7]]), dict(grads=[grads[0].half(), grads[1]]),
                dict(grads=[grads[0].cpu(), grads[1]]), dict(grads=[grads[0].new_zeros(64, 2)[:, 0], grads[1]]),
                dict(params=[params[0].double(), params[1]]), dict(copies=grads), dict(copies=[grads[0].bfloat16()]),
                dict(step=0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(lr=torch.ones(1)),
                dict(lr=torch.ones(2, device="cuda")), dict(step=torch.ones(1, dtype=torch.int32, device="cuda"))):
        kw = {**H, "params": params, "grads": grads, "step": 1, **bad}
        with pytest.raises(ValueError):
            adamw_step(kw.pop("params"), kw.pop("grads"), state, kw.pop("lr"), **kw)
    with pytest.raises(ValueError):
        AdamWState(params, bits=16)
    with pytest.raises(ValueError):
        AdamWState([params[0], params[0]])
    state.m = state.m[:-1]
    with pytest.raises(ValueError):
        adamw_step(params, grads, state, step=1, **H)
    assert all(torch.equal(a, b) for a, b in zip(params, before))


def test_state_needs_cuda_tensors():
    from megray_b200.ops import AdamWState

    for params in ([], [torch.zeros(3)]):
        with pytest.raises(ValueError):
            AdamWState(params)


def test_bad_arguments_of_the_c_entry_are_refused_before_any_launch():
    from megray_b200 import _lib

    lib = _lib.load()
    rec = (_lib.C.c_uint64 * 5)(64, 64, 0, 8, 0)
    ok = dict(p_dtype=7, g_dtype=7, bits=32, m=64, v=64, step=1.0)
    assert lib.megray_adamw(rec, 0, _lib.AdamWArgs(**ok), None) == 0
    assert lib.megray_adamw(rec, 1, None, None) == 6
    for bad in (dict(p_dtype=6), dict(g_dtype=0), dict(bits=16), dict(m=None), dict(v=68), dict(bits=8)):
        assert lib.megray_adamw(rec, 1, _lib.AdamWArgs(**{**ok, **bad}), None) in (6, -1), bad
    for bad in ((0, 64, 0, 8, 0), (66, 64, 0, 8, 0), (64, 65, 0, 8, 0), (64, 64, 1, 8, 0)):
        assert lib.megray_adamw((_lib.C.c_uint64 * 5)(*bad), 1, _lib.AdamWArgs(**ok), None) == -1, bad


@gpu
def test_a_tensor_that_is_in_a_step_twice_is_refused():
    from megray_b200.ops import adamw_step

    params, grads, state = make([300, 300, 0, 0], torch.float32, torch.float32, 32)
    copies = [torch.zeros(n, dtype=torch.bfloat16, device="cuda") for n in state.sizes]
    before = params[0].clone()
    flat = torch.zeros(500, device="cuda")
    for bad in (dict(params=[params[0], params[0], *params[2:]]), dict(params=[flat[200:], flat[:300], *params[2:]]),
                dict(copies=[copies[1], copies[1], *copies[2:]]),
                dict(params=[params[0].bfloat16(), params[1], params[1][:0], params[1][:0]], copies=[copies[1], copies[1], *copies[2:]])):
        kw = {**H, "params": params, "copies": copies, "step": 1, **bad}
        with pytest.raises(ValueError):
            adamw_step(kw.pop("params"), grads, state, kw.pop("lr"), **kw)
    assert torch.equal(params[0], before) and not bool(state.m.any())
    adamw_step(params, [grads[0], grads[0], *grads[2:]], state, step=1, copies=copies, **H)  # gradients are only read
    assert not torch.equal(params[0], before)


def test_overlapping_tensors_of_a_list_are_refused_by_the_c_entry():
    from megray_b200 import _lib

    lib = _lib.load()
    # (addresses that are never read: the refusal comes before any launch)
    args = _lib.AdamWArgs(p_dtype=7, g_dtype=7, bits=32, m=64, v=64, step=1.0)
    step = lambda *recs: lib.megray_adamw((_lib.C.c_uint64 * (5 * len(recs)))(*sum(recs, ())), len(recs), args, None)  # noqa: E731
    far, near, empty = (4096, 64, 0, 100, 0), (4096 - 399 * 4, 64, 0, 400, 1), (4096, 64, 0, 0, 3)
    assert step(far, near) == -1 and step(near, far) == -1 and step(far, far) == -1
    assert step(far, (1 << 20, 64, 0, 8, 2), near) == -1 and step((1 << 20, 64, 0, 8, 2), empty, near, far) == -1
    copy = lambda p, at, n: (p, 64, at, n, 0)  # noqa: E731
    assert step(copy(1 << 20, 4096, 100), copy(1 << 21, 4096 + 198, 100)) == -1
    assert step(copy(1 << 20, 4096, 100), copy(1 << 21, 0, 8), copy(1 << 22, 4000, 100)) == -1
