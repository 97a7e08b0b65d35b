"""Softmax attention over whole prompts and its backward pass (src/kernels/attention.cu).

Prompts lie one behind the other in the rows of ``[T, heads, D]`` tensors; ``cu_seqlens`` (int32, on the device,
``[0, L0, L0 + L1, ...]``) says where each begins.  A query sees the keys of its own prompt, with ``causal`` those up to
its own position.  Key / value heads may be fewer than query heads: query head h reads key / value head
``h * Hk // H``.  bf16 or float16, D a multiple of 8 up to 128, any strides that are multiples of 8 elements
(slices of one projection among them).  A wait inside a kernel that runs out sets the word of
:func:`megray_b200.ops.gemm_error_flag`.
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from ._stream import raw_stream
from .gemm import gemm_error_flag

_CODES = {torch.float16: 6, torch.bfloat16: 10}


def _tensor(t, rows: int, heads: int, dim: int, dtype, index: int, name: str):
    """The C view of a [T, heads, D] tensor; ValueError for anything that the kernels do not read."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index or
            t.shape != (rows, heads, dim)):
        raise ValueError(f"attention: {name} is a {(rows, heads, dim)} {dtype} tensor on the queries' device")
    row, head, one = t.stride()
    p = t.data_ptr()
    # the stride of an axis of one is never used
    if heads == 1:
        head = dim
    if rows <= 1:
        row = max(8, heads * head)
        if rows == 0:
            return _lib.AttnTensor(p or None, row, dim)
    if one != 1 or (row | head) & 7 or row <= 0 or head <= 0 or p & 15:
        raise ValueError(f"attention: {name}: innermost axis contiguous, the other strides multiples of 8 elements, "
                         "16-byte aligned")
    return _lib.AttnTensor(p, row, head)


def _output(t, rows: int, heads: int, dim: int, like: torch.Tensor, index: int, partly: bool, name: str):
    if t is None:  # what no prompt covers is zero
        t = like.new_zeros(rows, heads, dim) if partly else like.new_empty(rows, heads, dim)
    c = _tensor(t, rows, heads, dim, like.dtype, index, name)
    # token by token or head by head, every element has an address of its own
    if rows > 1 and not (c.head >= dim and c.row >= (heads - 1) * c.head + dim or
                         c.row >= dim and c.head >= (rows - 1) * c.row + dim):
        raise ValueError(f"attention: {name} overlaps itself")
    return t, c


def _problem(q, k, v, cu_seqlens, causal, scale):
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or not q.is_cuda or q.dtype not in _CODES:
        raise ValueError("attention: q is a [T, heads, D] CUDA tensor, bf16 or float16")
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("attention: k is a [T, kv heads, D] tensor")
    tokens, heads, dim = q.shape
    kv_heads, dtype, index = k.shape[1], q.dtype, q.get_device()
    if dim & 7 or not 8 <= dim <= 128 or kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("attention: D is a multiple of 8 from 8 to 128, the query heads a multiple of the key heads")
    if tokens >= 2 ** 31 - 512:
        raise ValueError("attention: fewer than 2^31 - 512 rows")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif not 0.0 < scale < math.inf:
        raise ValueError("attention: scale is positive")
    cu, seqs = None, 1
    if cu_seqlens is not None:
        if (cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or not 2 <= cu_seqlens.numel() <= 2 ** 31 - 512 or
                not cu_seqlens.is_contiguous() or cu_seqlens.get_device() != index):
            raise ValueError("attention: cu_seqlens is a contiguous int32 tensor of 2 to 2^31 - 512 entries on q's device")
        cu, seqs = cu_seqlens.data_ptr(), cu_seqlens.numel() - 1
    args = _lib.AttnArgs(cu, _CODES[dtype], tokens, heads, kv_heads, dim, seqs, 1 if causal else 0, scale,
                         gemm_error_flag(q.device).data_ptr())
    return (args, _tensor(q, tokens, heads, dim, dtype, index, "q"), _tensor(k, tokens, kv_heads, dim, dtype, index, "k"),
            _tensor(v, tokens, kv_heads, dim, dtype, index, "v"), index)


def _row_sums(t, heads: int, tokens: int, like: torch.Tensor, index: int, name: str) -> torch.Tensor:
    if t is None:
        return like.new_empty(heads, tokens, dtype=torch.float32)
    if t.dtype is not torch.float32 or t.shape != (heads, tokens) or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"attention: {name} is a contiguous [heads, T] float32 tensor on the queries' device")
    return t


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor = None, *, causal: bool = True,
              scale: float = None, out: torch.Tensor = None, lse: torch.Tensor = None):
    """Returns (out, lse): out = softmax(scale * q k^T) v in the type of ``q`` (``[T, H, D]``) and the logarithm of the
    sum of exponentials of every row (``[H, T]`` float32), which the backward pass takes and with which results
    over several sets of keys are joined.  ``scale`` defaults to 1 / sqrt(D).

    Without ``cu_seqlens`` all rows are one prompt.  Rows behind the last prompt are not looked at and keep what
    ``out`` and ``lse`` hold there (zeros in tensors made here).  ``cu_seqlens`` is read on the device: it has to
    rise from 0 to at most T; nothing outside the tensors is touched if it does not, but rows may then go
    unwritten.

    Probabilities are rounded to the type of ``v`` for the product with it, all sums are float32; values beyond 2^75 may
    overflow in them (a probability counts up to 2^32 there).  A query whose scores are all -infinity has the output NaN and the lse -infinity.  A NaN or an infinity
    in the values of a prompt may reach any row of that prompt, those of other prompts and of rows behind the last never
    do.  ``out`` may be ``q`` itself (the queries are then gone, also for the backward pass); beside that neither result may
    overlap an input or the other."""
    if isinstance(q, torch.Tensor) and q.is_cuda and q.get_device() != torch.cuda.current_device():
        with torch.cuda.device(q.device):
            return attention(q, k, v, cu_seqlens, causal=causal, scale=scale, out=out, lse=lse)
    args, cq, ck, cv, index = _problem(q, k, v, cu_seqlens, causal, scale)
    partly = cu_seqlens is not None
    out, co = _output(out, args.tokens, args.heads, args.dim, q, index, partly, "out")
    if co.p is not None and (co.p in (ck.p, cv.p) or co.p == cq.p and (co.row, co.head) != (cq.row, cq.head)):
        raise ValueError("attention: out lies where the keys or values do, or on the queries in another order")
    if lse is None and partly:
        lse = q.new_zeros(args.heads, args.tokens, dtype=torch.float32)
    lse = _row_sums(lse, args.heads, args.tokens, q, index, "lse")
    rc = _lib.load().megray_attention(args, cq, ck, cv, co, lse.data_ptr(), raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"megray_attention failed ({rc})")
    return out, lse


def attention_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                  lse: torch.Tensor, cu_seqlens: torch.Tensor = None, *, causal: bool = True, scale: float = None,
                  dq: torch.Tensor = None, dk: torch.Tensor = None, dv: torch.Tensor = None):
    """Returns (dq, dk, dv) for the gradient ``dout`` of the ``out`` that :func:`attention` returned with ``lse`` for the
    same arguments.  Gradients of key / value heads are summed over the query heads that read them.  Given tensors
    are written to (any of the strides that the inputs may have, slices of one buffer among them); rows behind the
    last prompt are left as they are (zeros in tensors made here).  They may overlap neither the inputs, which are read
    until the end, nor one another.  No atomics: the same inputs give the same bits.

    Probabilities are formed anew from the scores and ``lse`` and are off by up to ``abs(lse) * 2^-20`` of themselves: with
    scores (times scale) beyond some 1e4 gradients lose digits that the output keeps, and from 1e6 on they mean nothing.
    Probabilities and score gradients are rounded to the type of ``q`` for their products.  Float16 has steps of 2^-24
    below 6e-5 and ends at 65504: there ``dout`` is best scaled as losses are for that type, so that ``dout v`` over the
    length of a prompt is well inside."""
    if isinstance(q, torch.Tensor) and q.is_cuda and q.get_device() != torch.cuda.current_device():
        with torch.cuda.device(q.device):
            return attention_bwd(dout, q, k, v, out, lse, cu_seqlens, causal=causal, scale=scale, dq=dq, dk=dk, dv=dv)
    args, cq, ck, cv, index = _problem(q, k, v, cu_seqlens, causal, scale)
    tokens, heads, kv_heads, dim, dtype = args.tokens, args.heads, args.kv_heads, args.dim, q.dtype
    co = _tensor(out, tokens, heads, dim, dtype, index, "out")
    cd = _tensor(dout, tokens, heads, dim, dtype, index, "dout")
    if lse is None:
        raise ValueError("attention_bwd: lse is what attention returned")
    lse = _row_sums(lse, heads, tokens, q, index, "lse")
    dq, cdq = _output(dq, tokens, heads, dim, q, index, cu_seqlens is not None, "dq")
    dk, cdk = _output(dk, tokens, kv_heads, dim, q, index, cu_seqlens is not None, "dk")
    dv, cdv = _output(dv, tokens, kv_heads, dim, q, index, cu_seqlens is not None, "dv")
    if tokens and not {cdq.p, cdk.p, cdv.p}.isdisjoint((cd.p, cq.p, ck.p, cv.p, co.p)):
        raise ValueError("attention_bwd: a gradient lies where an input does")
    if tokens and len({cdq.p, cdk.p, cdv.p}) < 3:
        raise ValueError("attention_bwd: two gradients lie in one place")
    lib = _lib.load()
    room = q.new_empty(lib.megray_attention_bwd_workspace(args), dtype=torch.uint8)
    rc = lib.megray_attention_bwd(args, cd, cq, ck, cv, co, lse.data_ptr(), cdq, cdk, cdv, room.data_ptr(), raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"megray_attention_bwd failed ({rc})")
    return dq, dk, dv
