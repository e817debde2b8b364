"""Binding of the 8-bit block kernels (``csrc/fp8_blocks.cu``, ``csrc/gemm_fp8_tcgen05.cu``).

Operands are :class:`rwkvtune_b200.ops.fp8.Fp8Blocks` on one CUDA device; every call runs on the current stream of that
device and allocates its results there.  No sizes are refused: rows of packed matrices are padded to 16 bytes, and results
whose rows do not start on 16 bytes take a slower store inside the same kernel.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _ext, gemm_native

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_ARGTYPES = {
    "rwkv_fp8_pack": [_P, _I, _L, _P, _P, _I, _I, _I, _P],
    "rwkv_fp8_unpack": [_P, _P, _P, _I, _L, _I, _I, _I, _P],
    "rwkv_gemm_fp8_tcgen05": [_P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _P, _L, _P, _L, _P, _P, _P, _P, _I, _P, _P],
}
_NULL = contextlib.nullcontext()
_declared = False


def _call(name: str, *args) -> None:
    global _declared
    if not _declared:      # declared once: plain integers and addresses can then be passed as they are
        for fn, types in _ARGTYPES.items():
            getattr(_ext.lib(), fn).argtypes = types
        _declared = True
    _ext.call(name, *args)


def on_device(device: torch.device):
    """Context in which ``device`` is current (nothing to do when it is already)."""
    return _NULL if device.index is None or device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def pack(x: torch.Tensor, data: torch.Tensor, exponent_offset: int, rows: int) -> None:
    """``x [R, C]`` with unit inner stride -> ``data`` (values, then exponents at ``exponent_offset``)."""
    base = data.data_ptr()
    R, C = x.shape
    with on_device(x.device):
        _call("rwkv_fp8_pack", x.data_ptr(), _DTYPES[x.dtype], x.stride(0) if R > 1 else C, base, base + exponent_offset, R, C,
              rows, _ext.stream())


def unpack(p, out: torch.Tensor) -> None:
    base = p.data.data_ptr()
    with on_device(out.device):
        _call("rwkv_fp8_unpack", base, base + p.exponent_offset, out.data_ptr(), _DTYPES[out.dtype], p.C, p.R, p.C, p.rows,
              _ext.stream())


def _gemm(a, b, M: int, N: int, K: int, a_mn: int, b_mn: int, epilogue: int, out=None, residual=None, h=None, q=None) -> None:
    pa, pb = a.data.data_ptr(), b.data.data_ptr()
    ph, pq = (0 if t is None else t.data.data_ptr() for t in (h, q))
    with on_device(a.data.device):
        _call("rwkv_gemm_fp8_tcgen05", pa, pa + a.exponent_offset, a.rows, pb, pb + b.exponent_offset, M, N, K, a_mn, b_mn,
              epilogue, 0 if out is None else out.data_ptr(), N, 0 if residual is None else residual.data_ptr(),
              0 if residual is None else (residual.stride(0) if M > 1 else N), ph, 0 if h is None else ph + h.exponent_offset,
              pq, 0 if q is None else pq + q.exponent_offset, 0 if q is None else q.rows,
              gemm_native._status(a.data.device).data_ptr(), _ext.stream())


def _new(like, M: int, N: int) -> torch.Tensor:
    return torch.empty(M, N, dtype=torch.bfloat16, device=like.data.device)


def mm_nt(a, b, residual=None) -> torch.Tensor:
    """``a [M, K] @ b [N, K]^T (+ residual [M, N])`` in bf16."""
    out = _new(a, a.R, b.R)
    _gemm(a, b, a.R, b.R, a.C, 0, 0, 0 if residual is None else 1, out, residual)
    return out


def mm_nn(a, b) -> torch.Tensor:
    """``a [M, K] @ b [K, N]`` in bf16."""
    out = _new(a, a.R, b.C)
    _gemm(a, b, a.R, b.C, a.C, 0, 1, 0, out)
    return out


def mm_tn(a, b) -> torch.Tensor:
    """``a [K, M]^T @ b [K, N]`` in bf16, both in tiles."""
    out = _new(a, a.C, b.C)
    _gemm(a, b, a.C, b.C, a.R, 1, 1, 0, out)
    return out


def mm_nt_relu_sq(a, b, q) -> None:
    """``q = packed relu(a @ b^T)^2``."""
    _gemm(a, b, a.R, b.R, a.C, 0, 0, 2, q=q)


def mm_nn_relu_sq_grad(a, b, h, q) -> None:
    """``q = packed (a @ b) * 2 sqrt(h)``."""
    _gemm(a, b, a.R, b.C, a.C, 0, 1, 3, h=h, q=q)
