"""Operators on matrices held in 8 bits: packing, the linear map and the feed-forward half of a block.

A matrix is held as e4m3 values with a power-of-two scale for each block (:class:`Fp8Blocks`).  Two block shapes:

* tiles of 128 x 128 (``rows=128``): the scale is the same along both directions, so one packed copy is the operand of a
  product over the columns and of one over the rows.  Trainable weights use it for all three of their products.
* 128 columns of one row (``rows=1``): what a token is stored as depends on that token alone.  Products with a frozen,
  packed weight use it, so a sequence's result does not depend on what else is in the batch.

With ``P`` for packing, ``x [M, K]``, ``W [N, K]``::

    linear           y = P(x) P(W)^T      dx = P(dy) P(W)      dW = P(dy)^T P(x)
    channel mix      h = P(relu(P(x) P(Wk)^T)^2)               y = residual + h P(Wv)^T
                     p = P((P(dy) P(Wv)) * 2 sqrt(h))          dx = p P(Wk)
                     dWk = p^T P(x)       dWv = P(dy)^T h

Sums are formed in fp32 and rounded once.  The gradients are those of the products of the packed operands: packing itself
counts as the identity.  Backward keeps ``P(x)``, ``h`` and the packed weights, one byte a value, and nothing in 16 bits.

CUDA tensors run the kernels of ``csrc/fp8_blocks.cu`` and ``csrc/gemm_fp8_tcgen05.cu`` (bf16 activations; packing also
takes fp16 and fp32).  CPU tensors of any of the three types run the same definitions in plain fp32.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import reference

BLOCK = reference.FP8_BLOCK
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class Fp8Blocks:
    """A packed matrix: ``R`` rows by ``C`` columns of e4m3 values with one exponent byte per block of ``rows`` x 128.

    ``shape`` and ``dtype`` are those of the tensor it was packed from and of what :func:`unpack_fp8` returns.  ``data`` is
    one byte buffer: values row by row, each row padded to 16 bytes, then the exponents (``[ceil(R/128)][ceil(C/128)]`` for
    tiles, ``[ceil(C/128)][R padded to 16]`` for row blocks)."""

    __slots__ = ("data", "R", "C", "rows", "shape", "dtype", "exponent_offset")

    def __init__(self, data: Optional[torch.Tensor], R: int, C: int, rows: int, shape, dtype, device=None):
        self.R, self.C, self.rows, self.shape, self.dtype = R, C, rows, torch.Size(shape), dtype
        self.exponent_offset = R * (-(-C // 16) * 16)
        self.data = data if data is not None else torch.empty(self.exponent_offset + self._exponent_bytes(), dtype=torch.uint8,
                                                              device=device)

    def _exponent_bytes(self) -> int:
        return -(-self.C // BLOCK) * (-(-self.R // 16) * 16 if self.rows == 1 else -(-self.R // BLOCK))

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    @property
    def values(self) -> torch.Tensor:
        """``float8_e4m3fn [R, C]``, a view of the buffer."""
        return self.data[:self.exponent_offset].view(torch.float8_e4m3fn).view(self.R, -(-self.C // 16) * 16)[:, :self.C]

    @property
    def exponents(self) -> torch.Tensor:
        """``uint8 [ceil(R / rows), ceil(C / 128)]``, a view of the buffer: the scale of a block is ``2^(exponent - 127)``."""
        e, nb = self.data[self.exponent_offset:], -(-self.C // BLOCK)
        if self.rows == 1:
            return e.view(nb, -(-self.R // 16) * 16)[:, :self.R].t()
        return e.view(-(-self.R // BLOCK), nb)

    def to(self, device) -> "Fp8Blocks":
        data = self.data.to(device)
        return self if data is self.data else Fp8Blocks(data, self.R, self.C, self.rows, self.shape, self.dtype)

    def __repr__(self) -> str:
        return f"Fp8Blocks(shape={tuple(self.shape)}, rows={self.rows}, dtype={self.dtype}, device={self.device})"


def _native():
    from . import fp8_native

    return fp8_native


def _meta(p: Fp8Blocks):
    return p.R, p.C, p.rows, p.shape, p.dtype


def _pack2(x: torch.Tensor, rows: int, shape=None) -> Fp8Blocks:
    """Pack a matrix whose arguments have been checked."""
    R, C = x.shape
    p = Fp8Blocks(None, R, C, rows, x.shape if shape is None else shape, x.dtype, x.device)
    if R == 0:
        return p
    if x.is_cuda:
        if x.stride(1) != 1 and C > 1 or x.stride(0) < C and R > 1:
            x = x.contiguous()
        _native().pack(x, p.data, p.exponent_offset, rows)
    else:
        values, exponents = reference.fp8_pack(x, rows)
        p.values.copy_(values)
        p.exponents.copy_(exponents)
    return p


def pack_fp8(x: torch.Tensor, rows: int = BLOCK) -> Fp8Blocks:
    """Hold ``x [..., C]`` in 8 bits (leading dimensions are flattened to rows).  ``rows=1``: one scale per token and 128
    channels; ``rows=128``: one per tile of 128 x 128.  Not differentiable."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise TypeError(f"pack_fp8 takes a bfloat16, float16 or float32 tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if rows not in (1, BLOCK):
        raise ValueError(f"pack_fp8: rows is 1 or {BLOCK}, got {rows!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"pack_fp8: the last dimension must not be empty, got shape {tuple(x.shape)}")
    return _pack2(x.detach().reshape(-1, x.shape[-1]), rows, x.shape)


def unpack_fp8(p: Fp8Blocks, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``p`` stands for, in its shape and in ``dtype`` (default: the type that was packed)."""
    if not isinstance(p, Fp8Blocks):
        raise TypeError(f"unpack_fp8 takes what pack_fp8 returned, got {type(p).__name__}")
    dtype = p.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise TypeError(f"unpack_fp8: unsupported type {dtype}")
    out = torch.empty(p.shape, dtype=dtype, device=p.device)
    if p.R == 0:
        return out
    if out.is_cuda:
        _native().unpack(p, out)
    else:
        top = torch.finfo(dtype).max
        out.copy_(reference.fp8_unpack(p.values, p.exponents, p.rows).clamp(-top, top).view(p.shape))
    return out


# ------------------------------------------------------------------------------- products of packed matrices
def _f32(p: Fp8Blocks) -> torch.Tensor:
    return reference.fp8_unpack(p.values, p.exponents, p.rows)


def _mm_nt(a: Fp8Blocks, b: Fp8Blocks, dtype, residual=None) -> torch.Tensor:
    if a.data.is_cuda and a.R:
        return _native().mm_nt(a, b, residual)
    y = _f32(a) @ _f32(b).t()
    return (y if residual is None else y + residual.float()).to(dtype)


def _mm_nn(a: Fp8Blocks, b: Fp8Blocks, dtype) -> torch.Tensor:
    if a.data.is_cuda and a.R:
        return _native().mm_nn(a, b)
    return (_f32(a) @ _f32(b)).to(dtype)


def _mm_tn(a: Fp8Blocks, b: Fp8Blocks, dtype) -> torch.Tensor:
    if a.data.is_cuda and a.R:
        return _native().mm_tn(a, b)
    return (_f32(a).t() @ _f32(b)).to(dtype)


def _hidden(a: Fp8Blocks, wk: Fp8Blocks, rows: int) -> Fp8Blocks:
    """``P(relu(a wk^T)^2)``"""
    if a.data.is_cuda and a.R:
        h = Fp8Blocks(None, a.R, wk.R, rows, (a.R, wk.R), torch.bfloat16, a.device)
        _native().mm_nt_relu_sq(a, wk, h)
        return h
    return _pack2(torch.relu(_f32(a) @ _f32(wk).t()) ** 2, rows)


def _hidden_grad(d: Fp8Blocks, wv: Fp8Blocks, h: Fp8Blocks) -> Fp8Blocks:
    """``P((d wv) * 2 sqrt(h))``"""
    if d.data.is_cuda and d.R:
        p = Fp8Blocks(None, h.R, h.C, h.rows, h.shape, torch.bfloat16, d.device)
        _native().mm_nn_relu_sq_grad(d, wv, h, p)
        return p
    return _pack2((_f32(d) @ _f32(wv)) * 2 * torch.sqrt(_f32(h)), h.rows)


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    return t.reshape(-1, t.shape[-1])


class _Linear(torch.autograd.Function):
    """``x W^T`` with a trainable weight; everything in tiles."""

    @staticmethod
    def forward(ctx, x, w):
        x8, w8 = _pack2(_rows_of(x), BLOCK), _pack2(w, BLOCK)
        # each packed operand is kept only for the product that reads it
        ctx.save_for_backward(x8.data if ctx.needs_input_grad[1] else None, w8.data if ctx.needs_input_grad[0] else None)
        ctx.meta, ctx.shape, ctx.types = (_meta(x8), _meta(w8)), x.shape, (x.dtype, w.dtype)
        return _mm_nt(x8, w8, x.dtype).reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x8, w8 = (None if d is None else Fp8Blocks(d, *m) for d, m in zip(ctx.saved_tensors, ctx.meta))
        d8 = _pack2(_rows_of(dy), BLOCK)
        dx = _mm_nn(d8, w8, ctx.types[0]).reshape(ctx.shape) if ctx.needs_input_grad[0] else None
        dw = _mm_tn(d8, x8, ctx.types[1]) if ctx.needs_input_grad[1] else None
        return dx, dw


class _LinearFrozen(torch.autograd.Function):
    """``x W^T`` with a packed weight; row blocks, and a gradient for ``x`` only."""

    @staticmethod
    def forward(ctx, x, data, w8):
        ctx.save_for_backward(data)
        ctx.meta, ctx.shape = _meta(w8), x.shape
        return _linear_frozen(x, w8)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w8 = Fp8Blocks(ctx.saved_tensors[0], *ctx.meta)
        return _mm_nn(_pack2(_rows_of(dy), 1), w8, dy.dtype).reshape(ctx.shape), None, None


def _linear_frozen(x, w8):
    return _mm_nt(_pack2(_rows_of(x), 1), w8, x.dtype).reshape(*x.shape[:-1], w8.R)


def _check_activation(name: str, x, like=None) -> None:
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise TypeError(f"{name} takes a floating-point tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if x.is_cuda and x.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the 8-bit products take and return bfloat16 on CUDA, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{name}: the input needs at least one dimension")


def _check_weight(name: str, w, x, n_in: int) -> bool:
    """Shape, type and device of a weight ``[out, in]``; True when it is packed."""
    packed = isinstance(w, Fp8Blocks)
    if packed:
        if w.rows != BLOCK or len(w.shape) != 2:
            raise ValueError(f"{name}: a packed weight is a matrix packed with rows={BLOCK}, got {w!r}")
    elif not isinstance(w, torch.Tensor) or w.dtype not in _FLOATS:
        raise TypeError(f"{name}: a weight is a floating-point matrix or a packed one, got {getattr(w, 'dtype', type(w).__name__)}")
    elif w.is_cuda and w.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the 8-bit products take and return bfloat16 on CUDA, got a weight in {w.dtype}")
    if len(w.shape) != 2 or w.shape[1] != n_in or 0 in w.shape:
        raise ValueError(f"{name}: a weight [out, {n_in}] was expected, got {tuple(w.shape)}")
    if w.device != x.device:
        raise ValueError(f"{name}: input on {x.device}, weight on {w.device}")
    return packed


def fp8_linear(x: torch.Tensor, weight: Union[torch.Tensor, Fp8Blocks]) -> torch.Tensor:
    """``x @ weight^T`` as a product of 8-bit operands; ``weight [out, in]`` is a tensor (packed in the call, receives a
    gradient) or what :func:`pack_fp8` made of one (frozen: only ``x`` receives a gradient)."""
    _check_activation("fp8_linear", x)
    packed = _check_weight("fp8_linear", weight, x, x.shape[-1])
    if not packed:
        return _Linear.apply(x, weight)
    if torch.is_grad_enabled() and x.requires_grad:
        return _LinearFrozen.apply(x, weight.data, weight)
    return _linear_frozen(x, weight)


class _ChannelMix(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wk, wv, residual):
        x8, k8, v8 = _pack2(_rows_of(x), BLOCK), _pack2(wk, BLOCK), _pack2(wv, BLOCK)
        h8 = _hidden(x8, k8, BLOCK)
        need_x, need_k, need_v = ctx.needs_input_grad[:3]
        inner = need_x or need_k
        ctx.save_for_backward(x8.data if need_k else None, k8.data if need_x else None, v8.data if inner else None,
                              h8.data if inner or need_v else None)
        ctx.meta, ctx.shape, ctx.types = (_meta(x8), _meta(k8), _meta(v8), _meta(h8)), x.shape, (x.dtype, wk.dtype, wv.dtype)
        return _mm_nt(h8, v8, x.dtype, _rows_of(residual)).reshape(residual.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x8, k8, v8, h8 = (None if d is None else Fp8Blocks(d, *m) for d, m in zip(ctx.saved_tensors, ctx.meta))
        need_x, need_k, need_v, need_r = ctx.needs_input_grad
        dx = dwk = dwv = None
        if need_x or need_k or need_v:
            d8 = _pack2(_rows_of(dy), BLOCK)
        if need_x or need_k:
            p8 = _hidden_grad(d8, v8, h8)
            dx = _mm_nn(p8, k8, ctx.types[0]).reshape(ctx.shape) if need_x else None
            dwk = _mm_tn(p8, x8, ctx.types[1]) if need_k else None
        if need_v:
            dwv = _mm_tn(d8, h8, ctx.types[2])
        return dx, dwk, dwv, (dy if need_r else None)


class _ChannelMixFrozen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kdata, vdata, residual, k8, v8):
        h8 = _hidden(_pack2(_rows_of(x), 1), k8, 1)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(kdata, vdata, h8.data)
            ctx.meta, ctx.shape = (_meta(k8), _meta(v8), _meta(h8)), x.shape
        return _mm_nt(h8, v8, x.dtype, _rows_of(residual)).reshape(residual.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            k8, v8, h8 = (Fp8Blocks(d, *m) for d, m in zip(ctx.saved_tensors, ctx.meta))
            p8 = _hidden_grad(_pack2(_rows_of(dy), 1), v8, h8)
            dx = _mm_nn(p8, k8, dy.dtype).reshape(ctx.shape)
        return dx, None, None, (dy if ctx.needs_input_grad[3] else None), None, None


def fp8_channel_mix_ffn(xk: torch.Tensor, w_key: Union[torch.Tensor, Fp8Blocks], w_value: Union[torch.Tensor, Fp8Blocks],
                        residual: torch.Tensor) -> torch.Tensor:
    """``residual + relu(xk @ w_key^T)^2 @ w_value^T`` as products of 8-bit operands, the activation between the two kept in
    8 bits for backward.  Both weights are tensors (trainable) or both are packed (frozen: row blocks, gradients for ``xk``
    and ``residual`` only)."""
    name = "fp8_channel_mix_ffn"
    _check_activation(name, xk)
    packed = _check_weight(name, w_key, xk, xk.shape[-1])
    if _check_weight(name, w_value, xk, w_key.shape[0]) != packed:
        raise ValueError(f"{name}: either both weights are packed or neither is")
    if not isinstance(residual, torch.Tensor) or residual.dtype != xk.dtype or residual.device != xk.device:
        raise TypeError(f"{name}: the residual must have the input's type and device")
    if residual.shape != xk.shape[:-1] + (w_value.shape[0],):
        raise ValueError(f"{name}: a residual of shape {tuple(xk.shape[:-1]) + (w_value.shape[0],)} was expected, got "
                         f"{tuple(residual.shape)}")
    if residual.stride(-1) != 1 and residual.shape[-1] > 1:
        residual = residual.contiguous()
    if not packed:
        return _ChannelMix.apply(xk, w_key, w_value, residual)
    if torch.is_grad_enabled() and (xk.requires_grad or residual.requires_grad):
        return _ChannelMixFrozen.apply(xk, w_key.data, w_value.data, residual, w_key, w_value)
    h8 = _hidden(_pack2(_rows_of(xk), 1), w_key, 1)
    return _mm_nt(h8, w_value, xk.dtype, _rows_of(residual)).reshape(residual.shape)
