"""Balance loss of the router against float64: expert counts that do and do not fill vectors and warps, masks that
leave nothing, rows of -inf, strided rows, and the sums over ranks."""
import pytest
import torch

gpu = pytest.mark.gpu


def reference(logits, idx, coef, mask=None):
    """loss, counts, gradient and a bound on the float32 evaluation of the gradient."""
    x = logits.double().requires_grad_()
    e, k = x.shape[1], idx.shape[1]
    live = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if mask is None else mask.bool()
    tv = max(1, int(live.sum()))
    pairs = idx[live].reshape(-1).long()
    counts = torch.bincount(pairs[(pairs >= 0) & (pairs < e)], minlength=e)
    z = x[live]
    empty = torch.isneginf(z).all(1)
    p = torch.softmax(z.masked_fill(empty[:, None], 0.0), 1) * (~empty)[:, None]
    loss = coef * e * (counts.double() / (k * tv) * p.sum(0) / tv).sum()
    grad = torch.autograd.grad(loss, x)[0] if live.any() else torch.zeros_like(x)
    # the exponent's argument is off by half a step of itself and of its product with log2 e, exp2 by 2^-22, and the
    # sums by a half step for each of up to ten levels: below 2^-18 of every term for arguments up to 16
    w = coef * e / tv * (counts.double() / (k * tv) - counts.double().mean() / (k * tv))
    bound = torch.zeros_like(grad)
    with torch.no_grad():
        bound[live] = p * (w.abs() + (p * w.abs()).sum(1, keepdim=True)) * 2.0 ** -18
    return loss.detach(), counts, grad, bound


def close(got, want):
    (loss, counts, d), (w_loss, w_counts, w_grad, bound) = got, want
    assert counts.dtype == torch.int32 and torch.equal(counts.long(), w_counts)
    assert abs(float(loss) - float(w_loss)) <= 2.0 ** -18 * abs(float(w_loss))
    tol = bound * (1 + 2.0 ** -8) + w_grad.abs() * 2.0 ** -8 + 2.0 ** -133 if d.dtype == torch.bfloat16 else bound + 2.0 ** -149
    assert bool(((d.double() - w_grad).abs() <= tol).all())


def make(tokens, experts, top, dtype=torch.float32, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    logits = (torch.randn(tokens, experts, generator=g, device=device) * 1.5).to(dtype)
    idx = torch.randint(0, experts, (tokens, top), generator=g, device=device, dtype=torch.int32)
    idx[:, 0] = 0 if experts == 1 else idx[:, 0] // 2  # unevenly
    return logits, idx


@gpu
@pytest.mark.parametrize("tokens", [1, 7, 1000, 20_011])
@pytest.mark.parametrize("experts", [1, 2, 5, 8, 30, 64, 100, 128, 250, 256, 1000, 1023, 1024])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(tokens, experts, dtype):
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(tokens, experts, 1 + experts % 3, dtype, seed=tokens)
    close(balance_loss_grad(logits, idx, 0.01), reference(logits, idx, 0.01))
    again = balance_loss_grad(logits, idx, 0.01)
    assert all(torch.equal(a, b) for a, b in zip(again, balance_loss_grad(logits, idx, 0.01)))


@gpu
@pytest.mark.parametrize("tokens,experts", [(600, 16), (30_000, 64)])
@pytest.mark.parametrize("live", [0.0, 0.5, 1.0])
def test_masks(tokens, experts, live):
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(tokens, experts, 2)
    mask = torch.rand(tokens, device="cuda") < live
    logits[~mask] = float("nan")  # what a masked row holds does not matter
    idx[~mask] = 2 ** 30
    clean = torch.where(mask[:, None], logits, torch.zeros_like(logits))
    close(balance_loss_grad(logits, idx, 0.1, mask=mask), reference(clean, idx, 0.1, mask))
    close(balance_loss_grad(logits, idx.long(), 0.1, mask=mask.to(torch.uint8)), reference(clean, idx, 0.1, mask))
    # adding to a gradient that is there: masked rows keep theirs
    there = torch.randn(tokens, experts, device="cuda")
    want = reference(clean, idx, 0.1, mask)
    loss, counts, d = balance_loss_grad(logits, idx, 0.1, mask=mask, dlogits=there.clone(), accumulate=True)
    assert torch.equal(d[~mask], there[~mask])
    sum_ = there.double() + want[2]
    assert bool(((d.double() - sum_).abs() <= want[3] + sum_.abs() * 2.0 ** -24).all())


@gpu
@pytest.mark.parametrize("tokens,experts", [(300, 8), (40_000, 12)])
def test_experts_that_are_ruled_out(tokens, experts):
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(tokens, experts, 2)
    logits[:, 3] = float("-inf")
    logits[5] = float("-inf")       # a row of nothing
    logits[6] = torch.finfo(torch.float32).min
    idx[7, 1], idx[8, 0] = -1, experts
    close(balance_loss_grad(logits, idx, 0.01), reference(logits, idx, 0.01))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,wide,off", [(500, 16, 24, 4), (500, 16, 17, 1), (20_000, 64, 72, 8), (20_000, 64, 65, 0)])
def test_rows_of_a_wider_matrix(tokens, experts, wide, off, dtype):
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(tokens, wide, 2, dtype)
    idx.remainder_(experts)
    logits = logits[:, off:off + experts]
    store = torch.full((tokens, wide), 7.0, device="cuda")
    d = store[:, :experts]
    close(balance_loss_grad(logits, idx, 0.02, dlogits=d), reference(logits, idx, 0.02))
    assert bool((store[:, experts:] == 7.0).all())


@gpu
def test_no_tokens():
    from megray_b200.ops import balance_loss_grad

    loss, counts, d = balance_loss_grad(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 1.0)
    assert float(loss) == 0.0 and int(counts.sum()) == 0 and d.shape == (0, 8)


@gpu
def test_gradient_against_differences():
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(64, 8, 2)
    _, _, d = balance_loss_grad(logits, idx, 1.0)
    way = torch.randn_like(logits)
    h = 2.0 ** -7
    up, down = (float(balance_loss_grad(logits + s * h * way, idx, 1.0)[0]) for s in (1, -1))
    slope = float((d.double() * way.double()).sum())
    # truncation h^2 / 6 of a third derivative below 2 |way|^3 in mean, and two losses of about 1 to 2^-18 over 2 h
    assert abs((up - down) / (2 * h) - slope) <= h * h * float(way.abs().pow(3).sum()) / 64 + 2.0 ** -18 * 2 / h


@gpu
@pytest.mark.parametrize("tokens,experts", [(500, 8), (30_000, 64)])
def test_two_captured_calls_share_nothing(tokens, experts):
    from megray_b200.ops import balance_loss_grad

    cases, graphs = [make(tokens, experts, 2, seed=s) for s in (1, 2)], []
    balance_loss_grad(*cases[0], 0.01)
    for logits, idx in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = balance_loss_grad(logits, idx, 0.01)
        graphs.append((g, out))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    for (logits, idx), (_, out) in zip(cases, graphs):
        close(out, reference(logits, idx, 0.01))


class Halves:
    """Stands in for a communicator of two ranks: what one rank gives is added to what the other gave."""

    def __init__(self, other):
        self.nranks, self.other, self.mine = 2, list(other or []), []

    def all_reduce(self, send, recv, op):
        assert op == "sum"
        self.mine.append(send.clone())
        recv.copy_(send + self.other.pop(0) if self.other else send)


@gpu
@pytest.mark.parametrize("tokens,experts", [(500, 8), (30_000, 64)])
def test_the_sums_of_two_ranks(tokens, experts):
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(tokens, experts, 2)
    cut = tokens // 3
    want = reference(logits, idx, 0.01)
    first = Halves(None)
    balance_loss_grad(logits[:cut], idx[:cut], 0.01, comm=first)
    second = Halves(first.mine)
    loss, counts, d = balance_loss_grad(logits[cut:], idx[cut:], 0.01, comm=second)
    close((loss, counts, d), (want[0], want[1], want[2][cut:], want[3][cut:]))


@pytest.mark.parametrize("n", [2, 3])
def test_records_are_added_up_over_ranks(n):
    from helpers import with_group
    from megray_b200.ops.balance import add_ranks

    experts, words = 6, 16
    parts = []
    for r in range(n):
        g = torch.Generator().manual_seed(r)
        part = torch.zeros(2 + r, words, dtype=torch.int32)
        part[:, :experts] = torch.randint(0, 64, (2 + r, experts), generator=g).float().view(torch.int32)
        part[:, experts:2 * experts + 1] = torch.randint(0, 1000, (2 + r, experts + 1), generator=g)
        parts.append(part)
    sums = sum(p[:, :experts].contiguous().view(torch.float32).sum(0) for p in parts)  # whole numbers: exact
    whole = sum(p[:, experts:2 * experts + 1].sum(0) for p in parts)
    for total in with_group(n, "shm", lambda comm, rank: add_ranks(comm, parts[rank], experts)):
        assert torch.equal(total[0, :experts].view(torch.float32), sums)
        assert torch.equal(total[0, experts:2 * experts + 1].long(), whole) and int(total[0, 2 * experts + 1:].abs().sum()) == 0


def test_cpu_tensors_are_refused():
    from megray_b200.ops import balance_loss_grad

    with pytest.raises(ValueError):
        balance_loss_grad(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32), 1.0)


@gpu
def test_refusals():
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(16, 8, 2)
    for bad in (dict(logits=logits.half()), dict(logits=logits.t()), dict(logits=logits[0]), dict(idx=idx[:5]),
                dict(idx=idx.float()), dict(idx=idx.cpu()), dict(idx=idx.t().contiguous().t()), dict(mask=torch.ones(15, device="cuda") > 0),
                dict(mask=torch.ones(16, device="cuda")), dict(accumulate=True), dict(dlogits=logits[:5]),
                dict(dlogits=logits.bfloat16()), dict(logits=torch.zeros(4, 1025, device="cuda"), idx=idx[:4])):
        kw = {"logits": logits, "idx": idx, "coef": 1.0, **bad}
        with pytest.raises(ValueError):
            balance_loss_grad(kw.pop("logits"), kw.pop("idx"), kw.pop("coef"), **kw)


def test_bad_arguments_of_the_c_entry_are_refused_before_any_launch():
    from megray_b200 import _lib

    lib = _lib.load()
    ok = dict(logits=64, idx=64, ld=8, dtype=7, idx64=0, tokens=4, experts=8, top=2)
    out = _lib.BalanceOut(64, 64, 64, 8, 7, 0, 1.0)
    assert lib.megray_balance(None, out, 64, None) == 6 and lib.megray_balance(_lib.Router(**ok), None, 64, None) == 6
    for bad in (dict(logits=None), dict(idx=None), dict(logits=66), dict(idx=66), dict(ld=7), dict(dtype=6), dict(tokens=-1),
                dict(experts=0), dict(experts=1025), dict(top=0), dict(top=65), dict(tokens=2 ** 30 + 1, experts=2)):
        r = _lib.Router(**{**ok, **bad})
        assert lib.megray_balance(r, out, 64, None) in (6, -1), bad
        assert lib.megray_balance_stats(r, 64, None) in (6, -1), bad
        assert lib.megray_balance_grad(r, 64, 1, 64, out, None) in (6, -1), bad
    r = _lib.Router(**ok)
    assert lib.megray_balance_stats(r, None, None) == -1 and lib.megray_balance_stats(r, 72, None) == -1
    for n in (0, 49):
        assert lib.megray_balance_grad(r, 64, n, 64, out, None) == -1
    assert lib.megray_balance_grad(r, None, 1, 64, out, None) == -1 and lib.megray_balance_grad(r, 64, 1, None, out, None) == -1
    assert lib.megray_balance(r, out, None, None) == -1 and lib.megray_balance(r, out, 72, None) == -1
    for bad in ((None, 64, 64, 8, 7), (64, None, 64, 8, 7), (64, 64, 66, 8, 7), (64, 64, 64, 7, 7), (64, 64, 64, 8, 10)):
        assert lib.megray_balance(r, _lib.BalanceOut(*bad, 0, 1.0), 64, None) == -1, bad


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts", [(300, 8), (700, 33), (40_000, 12), (3000, 256)])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e10, 1e12, 1e30])
def test_rows_of_large_logits(size, tokens, experts, dtype):
    """Softmax does not change with a constant added to a row: rows at +-size are as evenly spread as rows at zero, and
    single entries there take all of a row or none of it."""
    from megray_b200.ops import balance_loss_grad

    logits, idx = make(tokens, experts, 2, dtype)
    last = experts - 1
    logits[3], logits[4] = size, -size
    logits[5, last], logits[6, 1] = size, -size
    logits[7], logits[8] = -size, size
    logits[7, 2], logits[8, 2] = size, -size
    logits[9, :2], logits[9, 2:] = size, -size          # two that share a row
    logits[tokens - 1] = -size
    close(balance_loss_grad(logits, idx, 0.01), reference(logits, idx, 0.01))
