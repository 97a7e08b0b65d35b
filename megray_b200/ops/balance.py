"""Balance loss of a mixture-of-experts router with its gradient and the pairs per expert
(src/kernels/balance.cu)."""
from __future__ import annotations

import torch

from .. import _lib
from ._stream import raw_stream

_CODES = {torch.float32: 7, torch.bfloat16: 10}


def _router(logits: torch.Tensor, idx: torch.Tensor, mask):
    if logits.dim() != 2 or logits.dtype not in _CODES or not logits.is_cuda or logits.stride(1) != 1:
        raise ValueError("balance: logits is a [tokens, experts] CUDA tensor, float32 or bf16, with contiguous rows")
    (tokens, experts), index = logits.shape, logits.get_device()
    if not 1 <= experts <= 1024:
        raise ValueError("balance: 1 to 1024 experts")
    if (idx.dim() != 2 or idx.shape[0] != tokens or not 1 <= idx.shape[1] <= 64 or idx.get_device() != index or
            idx.dtype not in (torch.int32, torch.int64) or not idx.is_contiguous()):
        raise ValueError("balance: idx is a contiguous [tokens, 1..64] int32 or int64 tensor on the logits' device")
    top = idx.shape[1]
    if tokens * top >= 2 ** 31:
        raise ValueError("balance: fewer than 2^31 pairs")
    if mask is not None and (mask.shape != (tokens,) or mask.dtype not in (torch.bool, torch.uint8) or
                             mask.get_device() != index or not mask.is_contiguous()):
        raise ValueError("balance: mask is a contiguous [tokens] bool or uint8 tensor on the logits' device")
    ld = logits.stride(0) if tokens > 1 else experts
    if ld < experts:
        raise ValueError("balance: rows of the logits overlap")
    return _lib.Router(logits.data_ptr(), idx.data_ptr(), None if mask is None else mask.data_ptr(), ld,
                       _CODES[logits.dtype], 1 if idx.dtype is torch.int64 else 0, tokens, experts, top), index


def _out(logits: torch.Tensor, tokens: int, experts: int, index: int, coef: float, dlogits, accumulate: bool):
    ldd = experts
    if dlogits is None:
        if accumulate:
            raise ValueError("balance: accumulate adds to dlogits, which is not given")
        dlogits = logits.new_empty(tokens, experts)
    else:
        if (dlogits.shape != (tokens, experts) or dlogits.get_device() != index or
                dlogits.dtype not in (logits.dtype, torch.float32) or (dlogits.numel() and dlogits.stride(1) != 1) or
                (tokens > 1 and dlogits.stride(0) < experts)):
            raise ValueError("balance: dlogits has the logits' shape and device, their type or float32, and contiguous rows")
        if tokens > 1:
            ldd = dlogits.stride(0)
    loss = logits.new_empty(1, dtype=torch.float32)
    counts = logits.new_empty(experts, dtype=torch.int32)
    out = _lib.BalanceOut(loss.data_ptr(), counts.data_ptr(), dlogits.data_ptr() or None, ldd, _CODES[dlogits.dtype],
                          1 if accumulate else 0, coef)
    return out, loss, counts, dlogits


def balance_loss_grad(logits: torch.Tensor, idx: torch.Tensor, coef: float, *, mask: torch.Tensor = None,
                      dlogits: torch.Tensor = None, accumulate: bool = False, comm=None):
    """Returns (loss, counts, dlogits).

    ``logits`` [T, E] (float32 or bf16) are the router's scores, ``idx`` [T, k] the experts that each token was
    given to.  Over the tokens whose ``mask`` is not zero (all without one), Tv of them, counts[e] is the number of
    pairs on expert e (int32), p the softmax of the logits, and

        loss = coef * E * sum_e counts[e] / (k Tv) * mean_t p[t, e]

    as a 1-element float32 tensor: ``coef`` when the experts are used evenly, more otherwise.  ``dlogits`` is its
    gradient (the counts have none), in the logits' type or, when given, written into that tensor (which may be
    float32 beside bf16 logits); ``accumulate`` adds to what it holds.  A masked token has the gradient zero and its
    logits are not looked at; entries of ``idx`` outside [0, E) are not counted; a row of nothing but -inf has no
    probabilities.  Without a token that counts, loss and gradient are zero.

    With ``comm`` (a communicator of several ranks; a collective call) counts, means and Tv are taken over the tokens
    of all ranks, and ``dlogits`` is the gradient of that one loss with respect to this rank's logits."""
    if logits.is_cuda and logits.get_device() != torch.cuda.current_device():
        with torch.cuda.device(logits.device):
            return balance_loss_grad(logits, idx, coef, mask=mask, dlogits=dlogits, accumulate=accumulate, comm=comm)
    router, index = _router(logits, idx, mask)
    tokens, experts = router.tokens, router.experts
    out, loss, counts, dlogits = _out(logits, tokens, experts, index, coef, dlogits, accumulate)
    lib, stream = _lib.load(), raw_stream(index)
    room = logits.new_empty(lib.megray_balance_workspace(tokens, experts), dtype=torch.uint8)
    if comm is None or comm.nranks == 1:
        rc = lib.megray_balance(router, out, room.data_ptr(), stream)
        if rc != 0:
            raise RuntimeError(f"megray_balance failed ({rc})")
        return loss, counts, dlogits
    n, size = lib.megray_balance_partials(tokens, experts), lib.megray_balance_record(experts)
    rc = lib.megray_balance_stats(router, room.data_ptr(), stream)
    if rc != 0:
        raise RuntimeError(f"megray_balance_stats failed ({rc})")
    total = add_ranks(comm, room[:n * size].view(torch.int32).view(n, size // 4), experts)
    rc = lib.megray_balance_grad(router, total.data_ptr(), 1, room.data_ptr(), out, stream)
    if rc != 0:
        raise RuntimeError(f"megray_balance_grad failed ({rc})")
    return loss, counts, dlogits


def add_ranks(comm, part: torch.Tensor, experts: int) -> torch.Tensor:
    """One record ([1, words] int32: float sums[E], int counts[E], int tokens) from this rank's partial ones
    ([n, words]), added up over the ranks of ``comm``."""
    total = torch.zeros(1, part.shape[1], dtype=torch.int32, device=part.device)
    sums = part[:, :experts].contiguous().view(torch.float32).sum(0, dtype=torch.float64).float()
    whole = part[:, experts:2 * experts + 1].sum(0, dtype=torch.int32)
    all_sums, all_whole = torch.empty_like(sums), torch.empty_like(whole)
    comm.all_reduce(sums, all_sums, "sum")
    comm.all_reduce(whole, all_whole, "sum")
    total[0, :experts] = all_sums.view(torch.int32)
    total[0, experts:2 * experts + 1] = all_whole
    return total
