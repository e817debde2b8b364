"""Binding of the 8-bit block kernels (``csrc/fp8_blocks.cu``, ``csrc/gemm_fp8_tcgen05.cu``, ``csrc/gemm_fp8_decode.cu``).

An operator describes its launches as records (``csrc/fp8_steps.cuh``) and hands them over in one library call
(:func:`run`): on a small batch a foreign call with twenty arguments costs as much as a launch.  Everything runs on the
current stream of the operands' device.  No sizes are refused: rows of packed matrices are padded to 16 bytes, and results
whose rows do not start on 16 bytes take a slower store inside the same kernel.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

from . import _ext, gemm_native

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_PACK, _UNPACK, _GEMM, _DECODE = 0, 1, 2, 3
_STORE, _RESIDUAL, _RELU_SQ, _RELU_SQ_GRAD = 0, 1, 2, 3
_record = struct.Struct("=12i3q12Q").pack      # Fp8Step, field by field
_declared = False


def _status(device: torch.device) -> int:
    return gemm_native._status(device).data_ptr()


def pack(x: torch.Tensor, q) -> bytes:
    """``x [R, C]`` with unit inner stride -> ``q``."""
    at = q.address
    return _record(_PACK, q.R, q.C, 0, 0, q.rows, _DTYPES[x.dtype], 0, 0, 0, 0, 0, x.stride(0) if q.R > 1 else q.C, 0, 0,
                   x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, at, at + q.exponent_offset, 0)


def unpack(p, out: torch.Tensor) -> bytes:
    at = p.address
    return _record(_UNPACK, p.R, p.C, 0, p.rows, 0, _DTYPES[out.dtype], 0, 0, 0, 0, 0, 0, p.C, 0, 0, at, at + p.exponent_offset,
                   0, 0, out.data_ptr(), 0, 0, 0, 0, 0, 0)


def _product(a, b, M: int, N: int, K: int, a_mn: int, b_mn: int, epilogue: int, out=None, residual=None, h=None, q=None) -> bytes:
    pa, pb = a.address, b.address
    ph = pq = he = qe = qr = pr = ldr = 0
    if h is not None:
        ph = h.address
        he = ph + h.exponent_offset
    if q is not None:
        pq, qr = q.address, q.rows
        qe = pq + q.exponent_offset
    if residual is not None:
        pr, ldr = residual.data_ptr(), residual.stride(0) if M > 1 else N
    return _record(_GEMM, M, N, K, a.rows, qr, 0, a_mn, b_mn, epilogue, 0, 0, 0, N, ldr, 0, pa, pa + a.exponent_offset,
                   pb, pb + b.exponent_offset, 0 if out is None else out.data_ptr(), pr, ph, he, pq, qe, _status(a.data.device))


def mm_nt(a, b, out, residual=None) -> bytes:
    """``out [M, N] = a [M, K] @ b [N, K]^T (+ residual)``"""
    return _product(a, b, a.R, b.R, a.C, 0, 0, _STORE if residual is None else _RESIDUAL, out, residual)


def mm_nn(a, b, out) -> bytes:
    """``out [M, N] = a [M, K] @ b [K, N]``"""
    return _product(a, b, a.R, b.C, a.C, 0, 1, _STORE, out)


def mm_tn(a, b, out) -> bytes:
    """``out [M, N] = a [K, M]^T @ b [K, N]``, both in tiles"""
    return _product(a, b, a.C, b.C, a.R, 1, 1, _STORE, out)


def mm_nt_relu_sq(a, b, q) -> bytes:
    """``q = packed relu(a @ b^T)^2``"""
    return _product(a, b, a.R, b.R, a.C, 0, 0, _RELU_SQ, q=q)


def mm_nn_relu_sq_grad(a, b, h, q) -> bytes:
    """``q = packed (a @ b) * 2 sqrt(h)``"""
    return _product(a, b, a.R, b.C, a.C, 0, 1, _RELU_SQ_GRAD, h=h, q=q)


@functools.lru_cache(maxsize=None)
def decode_form(M: int, N: int, K: int, packed: bool = False) -> int:
    """How ``x [M, K]`` times a packed ``[N, K]`` weight is run while decoding: 0 not, 1 on packed tokens, 2 on bf16 tokens
    that the kernel packs itself (see ``csrc/gemm_fp8_decode.cu``)."""
    return _ext.lib().rwkv_fp8_decode_form(M, N, K, int(packed)) if M <= 128 else 0


def decode_input(x: torch.Tensor) -> torch.Tensor:
    """``x [M, K]`` with rows that start on 16 bytes."""
    if x.stride(1) == 1 and x.data_ptr() % 16 == 0 and (x.shape[0] == 1 or (x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1])):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def decode(x, b, out=None, residual=None, q=None, chained: bool = False) -> bytes:
    """``out = x @ b^T (+ residual)`` or ``q = packed relu(x @ b^T)^2`` for at most 128 rows; ``x`` is packed or bf16."""
    packed = not isinstance(x, torch.Tensor)
    pb = b.address
    M, N, K = (x.R if packed else x.shape[0]), b.R, b.C
    px, pa, ae, ldx = (0, x.address, x.address + x.exponent_offset, 0) if packed else \
        (x.data_ptr(), 0, 0, x.stride(0) if M > 1 else K)
    pq = 0 if q is None else q.address
    return _record(_DECODE, M, N, K, 1, 1, 0, 0, 0, _RELU_SQ if q is not None else _STORE if residual is None else _RESIDUAL,
                   int(chained), 0, ldx, N, 0 if residual is None else residual.stride(0) if M > 1 else N, px, pa, ae, pb,
                   pb + b.exponent_offset, 0 if out is None else out.data_ptr(), 0 if residual is None else residual.data_ptr(),
                   0, 0, pq, 0 if q is None else pq + q.exponent_offset, _status(b.data.device))


def run(device: torch.device, steps) -> None:
    """Launch ``steps`` in order on the device's current stream."""
    global _declared
    if not _declared:
        _ext.lib().rwkv_fp8_run.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p]
        _declared = True
    if device.index is not None and device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return run(device, steps)
    _ext.LAUNCH_COUNT += len(steps) - 1
    _ext.call("rwkv_fp8_run", b"".join(steps), len(steps), _ext.stream())
