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
_record = struct.Struct("=12i3q13Q").pack      # Fp8Step, field by field
_launch = None                                 # rwkv_fp8_run, bound at the first call
_status_address = {}


def _status(device: torch.device) -> int:
    """Address of the device's status word; null (no record is kept) if the first call of all is being captured into a
    graph, whose memory the word must not live in."""
    at = _status_address.get(device.index)
    if at is None:
        if device.index not in gemm_native._STATUS and torch.cuda.is_current_stream_capturing():
            return 0
        at = _status_address[device.index] = gemm_native._status(device).data_ptr()
    return at


def pack(x: torch.Tensor, q) -> bytes:
    """``x [R, C]`` with unit inner stride -> ``q``."""
    return _record(_PACK, q.R, q.C, 0, 0, q.rows, _DTYPES[x.dtype], 0, 0, 0, 0, 0, x.stride(0) if q.R > 1 else q.C, 0, 0,
                   x.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, q.address, q.exponent_address, 0, 0)


def unpack(p, out: torch.Tensor) -> bytes:
    return _record(_UNPACK, p.R, p.C, 0, p.rows, 0, _DTYPES[out.dtype], 0, 0, 0, 0, 0, 0, p.C, 0, 0, p.address,
                   p.exponent_address, 0, 0, out.data_ptr(), 0, 0, 0, 0, 0, 0, 0)


def _product(a, b, M: int, N: int, K: int, a_mn: int, b_mn: int, epilogue: int, out=None, residual=None, h=None, q=None,
             with_next: int = 0, workspace=None) -> bytes:
    ph = he = pq = qe = qr = pr = ldr = 0
    if h is not None:
        ph, he = h.address, h.exponent_address
    if q is not None:
        pq, qe, qr = q.address, q.exponent_address, q.rows
    if residual is not None:
        pr, ldr = residual.data_ptr(), residual.stride(0) if M > 1 else N
    return _record(_GEMM, M, N, K, a.rows, qr, 0, a_mn, b_mn, epilogue, 0, with_next, 0, N, ldr, 0, a.address, a.exponent_address,
                   b.address, b.exponent_address, 0 if out is None else out.data_ptr(), pr, ph, he, pq, qe,
                   0 if workspace is None else workspace.data_ptr(), _status(a.data.device))


@functools.lru_cache(maxsize=4096)         # ragged batches bring ever new sizes
def _workspace_bytes(M: int, N: int, K: int) -> int:
    fn = _ext.lib().rwkv_fp8_workspace
    fn.restype = ctypes.c_longlong
    return fn(M, N, K)


def workspace(M: int, N: int, K: int, device):
    """Room for the slices of a product of few tiles and a long contraction; ``None`` if it runs in one piece."""
    n = _workspace_bytes(M, N, K)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def mm_nt(a, b, out, residual=None, ws=None) -> bytes:
    """``out [M, N] = a [M, K] @ b [N, K]^T (+ residual)``"""
    return _product(a, b, a.R, b.R, a.C, 0, 0, _STORE if residual is None else _RESIDUAL, out, residual, workspace=ws)


def mm_nn(a, b, out, ws=None) -> bytes:
    """``out [M, N] = a [M, K] @ b [K, N]``"""
    return _product(a, b, a.R, b.C, a.C, 0, 1, _STORE, out, workspace=ws)


def mm_tn(a, b, out, with_next: bool = False, ws=None) -> bytes:
    """``out [M, N] = a [K, M]^T @ b [K, N]``, both in tiles; ``with_next``: in one launch with the next record, another of
    these (both with a workspace or neither)"""
    return _product(a, b, a.C, b.C, a.R, 1, 1, _STORE, out, with_next=int(with_next), workspace=ws)


def mm_nt_relu_sq(a, b, q) -> bytes:
    """``q = packed relu(a @ b^T)^2``"""
    return _product(a, b, a.R, b.R, a.C, 0, 0, _RELU_SQ, q=q)


def mm_nn_relu_sq_grad(a, b, h, q) -> bytes:
    """``q = packed (a @ b) * 2 sqrt(h)``"""
    return _product(a, b, a.R, b.C, a.C, 0, 1, _RELU_SQ_GRAD, h=h, q=q)


@functools.lru_cache(maxsize=4096)
def decode_form(M: int, N: int, K: int, packed: bool = False) -> int:
    """How ``x [M, K]`` times a packed ``[N, K]`` weight is run while decoding: 0 not, 1 on packed tokens, 2 on bf16 tokens
    that the kernel packs itself (see ``csrc/gemm_fp8_decode.cu``)."""
    return _ext.lib().rwkv_fp8_decode_form(M, N, K, int(packed)) if M <= 128 else 0


def chaining() -> bool:
    """True inside a chain of decode launches, during which no kernel writes weights but the packing ones, which the next
    launch waits for (``_ext.launch_chaining``)."""
    return _ext._CHAIN.on


def decode_input(x: torch.Tensor) -> torch.Tensor:
    """``x [M, K]`` with rows that start on 16 bytes."""
    if x.stride(1) == 1 and x.data_ptr() % 16 == 0 and (x.shape[0] == 1 or (x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1])):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def decode(x, b, out=None, residual=None, q=None, chained: bool = False) -> bytes:
    """``out = x @ b^T (+ residual)`` or ``q = packed relu(x @ b^T)^2`` for at most 128 rows; ``x`` is packed, or bf16 if there
    is no residual."""
    N, K = b.R, b.C
    if isinstance(x, torch.Tensor):
        M, px, pa, ae = x.shape[0], x.data_ptr(), 0, 0
        ldx = x.stride(0) if M > 1 else K
    else:
        M, px, pa, ae, ldx = x.R, 0, x.address, x.exponent_address, 0
    epilogue, po, pr, ldr, pq, qe = _STORE, 0, 0, 0, 0, 0
    if q is not None:
        epilogue, pq, qe = _RELU_SQ, q.address, q.exponent_address
    else:
        po = out.data_ptr()
        if residual is not None:
            epilogue, pr, ldr = _RESIDUAL, residual.data_ptr(), residual.stride(0) if M > 1 else N
    return _record(_DECODE, M, N, K, 1, 1, 0, 0, 0, epilogue, chained, 0, ldx, N, ldr, px, pa, ae, b.address,
                   b.exponent_address, po, pr, 0, 0, pq, qe, 0, _status(b.data.device))


def run(device: torch.device, steps) -> None:
    """Launch ``steps`` in order on the device's current stream."""
    global _launch
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return run(device, steps)
    if _launch is None:
        _launch = _ext.lib().rwkv_fp8_run
        _launch.argtypes, _launch.restype = [ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p], ctypes.c_int
    _ext.LAUNCH_COUNT += len(steps)
    status = _launch(b"".join(steps), len(steps), torch._C._cuda_getCurrentRawStream(index))
    if status:
        _ext.check(status, "rwkv_fp8_run")
