"""The packed Ulysses pass: the swap around the attention operator on CPU ranks (with the operator's definition in
its place, since it runs on a GPU only), and with the operator itself on one."""
import math

import pytest
import torch

from helpers import with_group


def plain_attention(q, k, v, cu, *, causal=True, scale=None):
    """The operator's definition for any device: zero rows behind the last prompt."""
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[1], q.shape[0], dtype=q.dtype, device=q.device)
    ends = [0, q.shape[0]] if cu is None else cu.tolist()
    for a, b in zip(ends, ends[1:]):
        z = torch.einsum("qhd,khd->hqk", q[a:b], k[a:b].repeat_interleave(group, 1)) * scale
        if causal:
            z = z.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        out[a:b] = torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v[a:b].repeat_interleave(group, 1))
        lse[:, a:b] = torch.logsumexp(z, -1)
    return out, lse


def plain_attention_bwd(dout, q, k, v, out, lse, cu, *, causal=True, scale=None):
    with torch.enable_grad():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        got, _ = plain_attention(*leaves, cu, causal=causal, scale=scale)
        return torch.autograd.grad(got, leaves, dout)


@pytest.mark.parametrize("n", [1, 2, 4])
@pytest.mark.parametrize("causal", [True, False])
def test_sharded_rows_match_the_whole_batch(n, causal, monkeypatch):
    from megray_b200.parallel import sequence_parallel as sp

    monkeypatch.setattr(sp, "attention", plain_attention)
    monkeypatch.setattr(sp, "attention_bwd", plain_attention_bwd)
    T, H, Hk, D = 12 * n, 8, 4, 6
    g = torch.Generator().manual_seed(n)
    q, k, v, do = (torch.randn(T, h, D, generator=g, dtype=torch.float64) for h in (H, Hk, Hk, H))
    cu = torch.tensor([0, 5, 6, T - 2], dtype=torch.int32)
    want, _ = plain_attention(q, k, v, cu, causal=causal, scale=0.3)
    grads = plain_attention_bwd(do, q, k, v, None, None, cu, causal=causal, scale=0.3)

    def body(comm, rank):
        s = slice(rank * T // n, (rank + 1) * T // n)
        out, saved = sp.ulysses_attention_packed(comm, *(t[s].contiguous() for t in (q, k, v)), cu, causal=causal, scale=0.3)
        return out, sp.ulysses_attention_packed_bwd(comm, do[s].contiguous(), saved)

    for rank, (out, got) in enumerate(with_group(n, "shm", body)):
        s = slice(rank * T // n, (rank + 1) * T // n)
        torch.testing.assert_close(out, want[s], rtol=1e-12, atol=1e-12)
        for a, b in zip(got, grads):
            torch.testing.assert_close(a, b[s], rtol=1e-12, atol=1e-12)


def test_cpu_tensors_reach_the_operators_refusal():
    from megray_b200.parallel.sequence_parallel import ulysses_attention_packed

    class One:
        nranks, rank = 1, 0

    with pytest.raises(ValueError):
        ulysses_attention_packed(One(), *(torch.zeros(4, 2, 8) for _ in range(3)))


@pytest.mark.gpu
def test_one_rank_on_the_gpu():
    from megray_b200.ops import attention, attention_bwd
    from megray_b200.parallel.sequence_parallel import ulysses_attention_packed, ulysses_attention_packed_bwd

    class One:
        nranks, rank = 1, 0

    q, k, v, do = (torch.randn(200, h, 64, device="cuda").bfloat16() for h in (4, 2, 2, 4))
    cu = torch.tensor([0, 70, 190], dtype=torch.int32, device="cuda")
    out, saved = ulysses_attention_packed(One(), q, k, v, cu)
    want, lse = attention(q, k, v, cu)
    assert torch.equal(out, want) and float(out[190:].abs().sum()) == 0.0
    for a, b in zip(ulysses_attention_packed_bwd(One(), do, saved), attention_bwd(do, q, k, v, want, lse, cu)):
        assert torch.equal(a, b) and float(a[190:].abs().sum()) == 0.0
