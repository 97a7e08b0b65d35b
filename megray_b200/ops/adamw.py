"""AdamW over a list of tensors (src/kernels/adamw.cu), moments in 32 or in 8 bits.

``AdamWState`` holds the moments of a list of parameters in two flat buffers; ``adamw_step`` updates all of them
in one launch (one per combination of parameter and gradient type, and per 720 tensors).  With ``bits=8`` each
block of 256 elements keeps its first moment ``m`` and the root ``r`` of its second as e4m3 numbers times a float32
scale: 2.03 instead of 8 bytes per element.  A NaN or an infinity in the gradients of a block then reaches the whole
block's moments, where 32-bit moments keep it to its element.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from .. import _lib
from ._stream import raw_stream

BLOCK = 256
_CODES = {torch.float32: 7, torch.bfloat16: 10}
_P, _G, _COPY, _N, _BLOCK_AT = range(5)  # columns of megray_adamw_tensor


# (called once per tensor: as C functions on a list, which is what a long one costs on the host)
_dtype, _numel, _device = torch.Tensor.dtype.__get__, torch.Tensor.numel, torch.Tensor.get_device
_contiguous, _address = torch.Tensor.is_contiguous, torch.Tensor.data_ptr


class AdamWState:
    """Moments of ``params`` (CUDA tensors of one device), zero at first.

    ``begins[i]`` is where tensor i starts in the flat buffers, a multiple of 256.  ``bits=32``: ``m`` and ``v`` are
    float32.  ``bits=8``: ``m`` and ``r`` are float8_e4m3fn, ``m_scale`` and ``r_scale`` hold one float32 per block; the
    moments are ``m * m_scale`` and ``(r * r_scale) ** 2``.  All of it is state: save and restore these tensors."""

    def __init__(self, params, bits: int = 32):
        params = list(params)
        if bits not in (8, 32):
            raise ValueError("AdamWState: moments are kept in 8 or in 32 bits")
        if not params or any(not p.is_cuda or p.device != params[0].device for p in params):
            raise ValueError("AdamWState: expected CUDA tensors of one device")
        places = [p.data_ptr() for p in params if p.numel()]
        if len(set(places)) < len(places):
            raise ValueError("AdamWState: a tensor is in the list twice")
        self.bits, self.device = bits, params[0].device
        self.sizes = [p.numel() for p in params]
        blocks = np.array([-(-n // BLOCK) for n in self.sizes], dtype=np.uint64)
        first = np.cumsum(blocks) - blocks
        self.begins = [int(b) * BLOCK for b in first]
        self._records = np.zeros((len(params), 5), dtype=np.uint64)
        self._records[:, _N], self._records[:, _BLOCK_AT] = self.sizes, first
        total = int(blocks.sum())
        if bits == 32:
            self.m, self.v = (torch.zeros(total * BLOCK, dtype=torch.float32, device=self.device) for _ in range(2))
        else:
            self.m, self.r = (torch.zeros(total * BLOCK, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
                              for _ in range(2))
            self.m_scale, self.r_scale = (torch.zeros(total, dtype=torch.float32, device=self.device) for _ in range(2))

    def nbytes(self) -> int:
        """Bytes of the moments."""
        names = ("m", "v") if self.bits == 32 else ("m", "r", "m_scale", "r_scale")
        return sum(getattr(self, n).numel() * getattr(self, n).element_size() for n in names)


def _number(x, device, name: str):
    """(value, address): a host number, or a float32 tensor of one element on ``device``."""
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.float32 or x.numel() != 1 or x.device != device:
            raise ValueError(f"adamw_step: {name} as a tensor is one float32 on the parameters' device")
        return 0.0, x.data_ptr()
    return float(x), None


def _buffer(t: torch.Tensor, numel: int, dtype, device, name: str) -> int:
    if t.dtype != dtype or t.numel() != numel or t.device != device or not t.is_contiguous():
        raise ValueError(f"adamw_step: the state's {name} is not the contiguous {dtype} buffer it was made as")
    return t.data_ptr()


def adamw_step(params, grads, state: AdamWState, lr, *, step, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, grad_scale=1.0, copies=None) -> None:
    """One step in place: with g = grad * grad_scale, m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
    p = p (1 - lr wd) - lr / (1 - b1^step) * m / (sqrt(v / (1 - b2^step)) + eps), all in float32.

    ``params`` are float32 or bf16, ``grads`` float32 or bf16 of the same sizes, in the order that ``state`` was made
    with; a gradient that is None leaves its tensor and moments as they are.  ``copies``, when given, are as many bf16
    tensors and receive the updated parameters rounded.  Parameters overlap neither one another nor anything else in the
    call, and copies do not either: the tensors are worked on side by side.  ``step`` counts from 1.  ``lr``, ``step`` and
    ``grad_scale`` may be float32 tensors of one element on the device: a captured graph then follows their contents,
    while host numbers are part of the capture."""
    n = len(state.sizes)
    params, grads, copies = list(params), list(grads), None if copies is None else list(copies)
    if len(params) != n or len(grads) != n or (copies is not None and len(copies) != n):
        raise ValueError("adamw_step: expected as many parameters, gradients and copies as the state was made with")
    device = state.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return adamw_step(params, grads, state, lr, step=step, betas=betas, eps=eps, weight_decay=weight_decay,
                              grad_scale=grad_scale, copies=copies)
    args = _lib.AdamWArgs(bits=state.bits, beta1=betas[0], beta2=betas[1], eps=eps, weight_decay=weight_decay)
    args.lr, args.lr_dev = _number(lr, device, "lr")
    args.step, args.step_dev = _number(step, device, "step")
    args.grad_scale, args.grad_scale_dev = _number(grad_scale, device, "grad_scale")
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or (args.step_dev is None and args.step < 1.0):
        raise ValueError("adamw_step: betas lie in [0, 1) and step counts from 1")
    total = state.begins[-1] + -(-state.sizes[-1] // BLOCK) * BLOCK
    if state.bits == 32:
        args.m = _buffer(state.m, total, torch.float32, device, "m")
        args.v = _buffer(state.v, total, torch.float32, device, "v")
    else:
        args.m = _buffer(state.m, total, torch.float8_e4m3fn, device, "m")
        args.v = _buffer(state.r, total, torch.float8_e4m3fn, device, "r")
        args.m_scale = _buffer(state.m_scale, total // BLOCK, torch.float32, device, "m_scale")
        args.v_scale = _buffer(state.r_scale, total // BLOCK, torch.float32, device, "r_scale")

    records, sizes = state._records, state.sizes
    keep = [i for i, g in enumerate(grads) if g is not None]
    if len(keep) < n:
        params, grads = [params[i] for i in keep], [grads[i] for i in keep]
        copies = [copies[i] for i in keep] if copies is not None else None
        records, sizes = records[keep], [sizes[i] for i in keep]
    records, one_kind = records.copy(), True
    for name, field, ts, types in (("parameter", _P, params, _CODES), ("gradient", _G, grads, _CODES),
                                   ("copy", _COPY, copies or [], (torch.bfloat16,))):
        if not ts:
            continue
        kinds = set(map(_dtype, ts))
        one_kind = one_kind and len(kinds) == 1
        if not kinds.issubset(types):
            raise ValueError(f"adamw_step: a {name} is {kinds}; float32 and bf16 are taken, bf16 alone for copies")
        if (list(map(_numel, ts)) != sizes or set(map(_device, ts)) != {device.index} or
                not all(map(_contiguous, ts))):
            raise ValueError(f"adamw_step: a {name} has another size than its parameter had when the state was made, "
                             "is not contiguous or lies on another device")
        records[:, field] = np.fromiter(map(_address, ts), dtype=np.uint64, count=len(ts))
    if not params:
        return
    lib, stream = _lib.load(), raw_stream(device.index)
    pairs = {(params[0].dtype, grads[0].dtype)} if one_kind else set(zip(map(_dtype, params), map(_dtype, grads)))
    if len(pairs) > 1:  # (a list of one kind is looked at by its call, before it launches anything)
        for name, field in (("parameter", _P), ("copy", _COPY)):
            places = [a for a, k in zip(records[:, field].tolist(), sizes) if a and k]
            if len(set(places)) < len(places):
                raise ValueError(f"adamw_step: a {name} is in the list twice")
    for pair in pairs:
        part = records if one_kind else records[[(p.dtype, g.dtype) == pair for p, g in zip(params, grads)]]
        args.p_dtype, args.g_dtype = _CODES[pair[0]], _CODES[pair[1]]
        rc = lib.megray_adamw(C.c_void_p(part.__array_interface__["data"][0]), len(part), args, stream)
        if rc == -1:
            raise ValueError("adamw_step: tensors of the list overlap or are not aligned to their elements")
        if rc != 0:
            raise RuntimeError(f"megray_adamw failed ({rc})")
