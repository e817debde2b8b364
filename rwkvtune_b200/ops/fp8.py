"""Operators on matrices held in 8 bits: packing, the linear map and the feed-forward half of a block.

A matrix is held as e4m3 values with a power-of-two scale for each block (:class:`Fp8Blocks`).  Two block shapes:

* tiles of 128 x 128 (``rows=128``): the scale is the same along both directions, so one packed copy is the operand of a
  product over the columns and of one over the rows.  Trainable weights use it for all three of their products.
* 128 columns of one row (``rows=1``): what a token is stored as depends on that token alone.  Products with a frozen,
  packed weight use it.  A token's result is then the same bit for bit in batches that run in the same way: those of at most
  128 rows, and larger ones whose contraction is cut into the same number of slices (it depends on the number of rows).
  Elsewhere the fp32 sums are taken in another order, which may round a result to its neighbour, and in the feed-forward
  half a hidden value to the next 8-bit one.

With ``P`` for packing, ``x [M, K]``, ``W [N, K]``::

    linear           y = P(x) P(W)^T      dx = P(dy) P(W)      dW = P(dy)^T P(x)
    channel mix      h = P(relu(P(x) P(Wk)^T)^2)               y = residual + h P(Wv)^T
                     p = P((P(dy) P(Wv)) * 2 sqrt(h))          dx = p P(Wk)
                     dWk = p^T P(x)       dWv = P(dy)^T h

Sums are formed in fp32 and rounded once.  The gradients are those of the products of the packed operands: packing itself
counts as the identity.  Backward keeps ``P(x)``, ``h`` and the packed weights, one byte a value, and nothing in 16 bits.

CUDA tensors run the kernels of ``csrc/fp8_blocks.cu``, ``csrc/gemm_fp8_tcgen05.cu`` and, for at most 128 rows against a
frozen weight, ``csrc/gemm_fp8_decode.cu`` (bf16 activations; packing also takes fp16 and fp32).  CPU tensors of any of the three types run
the same definitions in plain fp32.  Numbers below 2^-126 count as zero, packed and read back, on both.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _KERNELS
from . import fp8_native as native
from . import reference

BLOCK = reference.FP8_BLOCK
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _sizes(R: int, C: int, rows: int):
    """Bytes of the values and of the exponents of a packed matrix."""
    return R * (-(-C // 16) * 16), -(-C // BLOCK) * (-(-R // 16) * 16 if rows == 1 else -(-R // BLOCK))


class Fp8Blocks:
    """A packed matrix: ``R`` rows by ``C`` columns of e4m3 values with one exponent byte per block of ``rows`` x 128.

    ``shape`` and ``dtype`` are those of the tensor it was packed from and of what :func:`unpack_fp8` returns.  It lies at
    ``offset`` in the byte buffer ``data``: values row by row, each row padded to 16 bytes, then the exponents
    (``[ceil(R/128)][ceil(C/128)]`` for tiles, ``[ceil(C/128)][R padded to 16]`` for row blocks)."""

    __slots__ = ("data", "offset", "R", "C", "rows", "shape", "dtype", "exponent_offset", "address", "exponent_address")

    def __init__(self, data: torch.Tensor, offset: int, R: int, C: int, rows: int, shape=None, dtype=torch.bfloat16):
        self.data, self.offset, self.R, self.C, self.rows, self.dtype = data, offset, R, C, rows, dtype
        self.shape = (R, C) if shape is None else shape
        self.exponent_offset = R * (-(-C // 16) * 16)
        self.address = data.data_ptr() + offset
        self.exponent_address = self.address + self.exponent_offset

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return sum(_sizes(self.R, self.C, self.rows))

    @property
    def values(self) -> torch.Tensor:
        """``float8_e4m3fn [R, C]``, a view of the buffer."""
        v = self.data[self.offset:self.offset + self.exponent_offset].view(torch.float8_e4m3fn)
        return v.view(self.R, -(-self.C // 16) * 16)[:, :self.C]

    @property
    def exponents(self) -> torch.Tensor:
        """``uint8 [ceil(R / rows), ceil(C / 128)]``, a view of the buffer: the scale of a block is ``2^(exponent - 127)``."""
        e, nb = self.data[self.offset + self.exponent_offset:self.offset + self.nbytes], -(-self.C // BLOCK)
        if self.rows == 1:
            return e.view(nb, -(-self.R // 16) * 16)[:, :self.R].t()
        return e.view(-(-self.R // BLOCK), nb)

    def to(self, device) -> "Fp8Blocks":
        data = self.data.to(device)
        return self if data is self.data else Fp8Blocks(data, self.offset, self.R, self.C, self.rows, self.shape, self.dtype)

    def __reduce__(self):
        return Fp8Blocks, (self.data, self.offset, self.R, self.C, self.rows, self.shape, self.dtype)

    def __repr__(self) -> str:
        return f"Fp8Blocks(shape={tuple(self.shape)}, rows={self.rows}, dtype={self.dtype}, device={self.device})"


def _matrix(device, R: int, C: int, rows: int, shape=None, dtype=torch.bfloat16) -> Fp8Blocks:
    """An uninitialised packed matrix in a buffer of its own.  An ordinary tensor under ``torch.inference_mode`` as well: a
    packed weight is written again and kept for backward elsewhere."""
    if torch.is_inference_mode_enabled():
        with torch.inference_mode(False):
            return _matrix(device, R, C, rows, shape, dtype)
    return Fp8Blocks(torch.empty(sum(_sizes(R, C, rows)), dtype=torch.uint8, device=device), 0, R, C, rows, shape, dtype)


def _room(device, *specs):
    """Uninitialised packed matrices ``(R, C, rows)`` in one buffer; ``None`` stays ``None``."""
    total, at = 0, []
    for spec in specs:
        at.append(total)
        if spec is not None:
            total += -(-sum(_sizes(*spec)) // 128) * 128
    data = torch.empty(total, dtype=torch.uint8, device=device)
    return [None if spec is None else Fp8Blocks(data, o, *spec) for o, spec in zip(at, specs)]


class _HostRun:
    """The steps of an operator, computed one by one in plain PyTorch."""

    def __init__(self, device):
        pass

    def pack(self, x, q):
        if q.R:
            values, exponents = reference.fp8_pack(x.detach(), q.rows)
            q.values.copy_(values)
            q.exponents.copy_(exponents)

    def unpack(self, p, out):
        top = torch.finfo(out.dtype).max
        out.copy_(_f32(p).clamp(-top, top).view(out.shape))

    def nt(self, a, b, out, residual=None):
        y = _f32(a) @ _f32(b).t()
        out.copy_(y if residual is None else y + residual.float())

    def nn(self, a, b, out):
        out.copy_(_f32(a) @ _f32(b))

    def tn(self, a, b, out):
        out.copy_(_f32(a).t() @ _f32(b))

    def tn_two(self, a, b, out, c, d, out2):
        self.tn(a, b, out)
        self.tn(c, d, out2)

    def nt_frozen(self, x, w, out, hidden=None):
        x8 = _matrix(x.device, *x.shape, 1)
        self.pack(x, x8)
        self.nt(x8, w, out) if hidden is None else self.nt_relu_sq(x8, w, hidden)

    def nt_relu_sq(self, a, b, q):
        self.pack(torch.relu(_f32(a) @ _f32(b).t()) ** 2, q)

    def nn_relu_sq_grad(self, a, b, h, q):
        self.pack((_f32(a) @ _f32(b)) * 2 * torch.sqrt(_f32(h)), q)

    def go(self):
        pass


class _DeviceRun:
    """The steps of an operator, collected and launched together."""

    __slots__ = ("device", "steps", "keep")

    def __init__(self, device):
        self.device, self.steps = device, []
        self.keep = []                            # copies made on the way: their memory is not reused before the launch

    def pack(self, x, q):
        if q.R:
            s0, s1 = x.stride()
            if (s1 != 1 and q.C > 1) or (s0 < q.C and q.R > 1):
                x = x.contiguous()
                self.keep.append(x)
            self.steps.append(native.pack(x, q))

    def unpack(self, p, out):
        if p.R:
            self.steps.append(native.unpack(p, out))

    def nt(self, a, b, out, residual=None):
        if not a.R:
            return
        if a.rows == 1 and native.decode_form(a.R, b.R, b.C, True):
            # its predecessor is the step that packed `a`, which does not write the weights
            self.steps.append(native.decode(a, b, out, residual, chained=bool(self.steps)))
        else:
            ws = native.workspace(a.R, b.R, a.C, self.device)
            self.steps.append(native.mm_nt(a, b, out, residual, ws))
            self.keep.append(ws)
        self.keep.append(residual)

    def nt_frozen(self, x, w, out, hidden=None):
        """``out = P(x) w^T`` or ``hidden = P(relu(P(x) w^T)^2)`` with ``x`` packed row by row."""
        M = x.shape[0]
        if not M:
            return
        form = native.decode_form(M, w.R, w.C)
        if form == 2:
            x = native.decode_input(x)
            self.keep.append(x)
            self.steps.append(native.decode(x, w, out, q=hidden, chained=native.chaining()))
            return
        x8 = _matrix(self.device, M, w.C, 1)
        self.keep.append(x8)
        self.pack(x, x8)
        if hidden is None:
            self.nt(x8, w, out)
        elif form:
            self.steps.append(native.decode(x8, w, q=hidden, chained=True))
        else:
            self.nt_relu_sq(x8, w, hidden)

    def nn(self, a, b, out):
        if a.R:
            ws = native.workspace(a.R, b.C, a.C, self.device)
            self.steps.append(native.mm_nn(a, b, out, ws))
            self.keep.append(ws)

    def tn(self, a, b, out):
        if a.R:
            ws = native.workspace(a.C, b.C, a.R, self.device)
            self.steps.append(native.mm_tn(a, b, out, ws=ws))
            self.keep.append(ws)
        else:
            out.zero_()

    def tn_two(self, a, b, out, c, d, out2):
        """``out = a^T b`` and ``out2 = c^T d`` in one launch, where both contractions run in one piece or both in slices."""
        sizes = (a.C, b.C, a.R), (c.C, d.C, c.R)
        ws = [native.workspace(*s, self.device) for s in sizes]
        if not a.R or not c.R or (ws[0] is None) != (ws[1] is None):
            self.tn(a, b, out)
            self.tn(c, d, out2)
            return
        self.steps += [native.mm_tn(a, b, out, True, ws[0]), native.mm_tn(c, d, out2, ws=ws[1])]
        self.keep += ws

    def nt_relu_sq(self, a, b, q):
        if a.R:
            self.steps.append(native.mm_nt_relu_sq(a, b, q))

    def nn_relu_sq_grad(self, a, b, h, q):
        if a.R:
            self.steps.append(native.mm_nn_relu_sq_grad(a, b, h, q))

    def go(self):
        if self.steps:
            native.run(self.device, self.steps)


def _run_on(t: torch.Tensor):
    return (_DeviceRun if t.is_cuda and _KERNELS["fp8"] else _HostRun)(t.device)


def _f32(p: Fp8Blocks) -> torch.Tensor:
    return reference.fp8_unpack(p.values, p.exponents, p.rows)


def pack_fp8(x: torch.Tensor, rows: int = BLOCK, out: Optional[Fp8Blocks] = None) -> Fp8Blocks:
    """Hold ``x [..., C]`` in 8 bits (leading dimensions are flattened to rows).  ``rows=1``: one scale per token and 128
    channels; ``rows=128``: one per tile of 128 x 128.  ``out``: an earlier result for the same shape, type, device and
    ``rows``, written again in place (a captured graph that reads it sees the new values).  Not differentiable."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise TypeError(f"pack_fp8 takes a bfloat16, float16 or float32 tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if rows not in (1, BLOCK):
        raise ValueError(f"pack_fp8: rows is 1 or {BLOCK}, got {rows!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"pack_fp8: the last dimension must not be empty, got shape {tuple(x.shape)}")
    x2 = _rows_of(x)
    if out is None:
        p = _matrix(x.device, x2.shape[0], x2.shape[1], rows, x.shape, x.dtype)
    else:
        p = out
        if not isinstance(p, Fp8Blocks) or (tuple(p.shape), p.dtype, p.rows, p.device) != (tuple(x.shape), x.dtype, rows, x.device):
            raise ValueError(f"pack_fp8: out does not hold a {tuple(x.shape)} tensor of {x.dtype} on {x.device} with rows={rows}: {out!r}")
        torch.autograd.graph.increment_version(p.data)      # a backward pass that kept the old values is refused
    run = _run_on(x)
    run.pack(x2, p)
    run.go()
    return p


def unpack_fp8(p: Fp8Blocks, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``p`` stands for, in its shape and in ``dtype`` (default: the type that was packed)."""
    if not isinstance(p, Fp8Blocks):
        raise TypeError(f"unpack_fp8 takes what pack_fp8 returned, got {type(p).__name__}")
    dtype = p.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise TypeError(f"unpack_fp8: unsupported type {dtype}")
    out = torch.empty(p.shape, dtype=dtype, device=p.data.device)
    run = _run_on(out)
    run.unpack(p, out)
    run.go()
    return out


# ------------------------------------------------------------------------------- products of packed matrices
def _rows_of(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _meta(p: Optional[Fp8Blocks]):
    return None if p is None else (p.offset, p.R, p.C, p.rows)


class _Linear(torch.autograd.Function):
    """``x W^T`` with a trainable weight; everything in tiles."""

    @staticmethod
    def forward(ctx, x, w):
        x2 = _rows_of(x)
        (M, K), N = x2.shape, w.shape[0]
        need_x, need_w = ctx.needs_input_grad
        # a packed operand is kept for the product that reads it in backward
        x8, w8 = _room(x.device, (M, K, BLOCK) if need_w else None, (N, K, BLOCK) if need_x else None)
        kept = (x8 or w8).data if need_x or need_w else None
        ctx.save_for_backward(kept)
        ctx.meta, ctx.shape, ctx.types = (_meta(x8), _meta(w8)), x.shape, (x.dtype, w.dtype)
        if not (need_x and need_w):
            a, b = _room(x.device, None if need_w else (M, K, BLOCK), None if need_x else (N, K, BLOCK))
            x8, w8 = x8 or a, w8 or b
        # in its final shape: autograd refuses to write in place to a view made in here
        y = x.new_empty((*x.shape[:-1], N))
        run = _run_on(x)
        run.pack(x2, x8)
        run.pack(w, w8)
        run.nt(x8, w8, _rows_of(y))
        run.go()
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (data,) = ctx.saved_tensors
        x8, w8 = (None if m is None else Fp8Blocks(data, *m) for m in ctx.meta)
        d2 = _rows_of(dy)
        d8 = _matrix(dy.device, d2.shape[0], d2.shape[1], BLOCK)
        run = _run_on(dy)
        run.pack(d2, d8)
        dx = dw = None
        if w8 is not None:
            dx = torch.empty(ctx.shape, dtype=ctx.types[0], device=dy.device)
            run.nn(d8, w8, _rows_of(dx))
        if x8 is not None:
            dw = torch.empty(d8.C, x8.C, dtype=ctx.types[1], device=dy.device)
            run.tn(d8, x8, dw)
        run.go()
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
        d2 = _rows_of(dy)
        d8 = _matrix(dy.device, d2.shape[0], d2.shape[1], 1)
        dx = torch.empty(ctx.shape, dtype=dy.dtype, device=dy.device)
        run = _run_on(dy)
        run.pack(d2, d8)
        run.nn(d8, w8, _rows_of(dx))
        run.go()
        return dx, None, None


def _linear_frozen(x, w8):
    x2 = _rows_of(x)
    y = torch.empty(*x.shape[:-1], w8.R, dtype=x.dtype, device=x.device)
    run = _run_on(x)
    run.nt_frozen(x2, w8, _rows_of(y))
    run.go()
    return y


def _check_activation(name: str, x) -> None:
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise TypeError(f"{name} takes a floating-point tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if x.is_cuda and x.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the 8-bit products take and return bfloat16 on CUDA, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{name}: the input needs at least one dimension")


def _check_weight(name: str, w, x, n_in: int) -> bool:
    """Shape, type and device of a weight ``[out, in]``; True when it is packed."""
    packed = type(w) is Fp8Blocks
    if packed:
        if w.rows != BLOCK or len(w.shape) != 2:
            raise ValueError(f"{name}: a packed weight is a matrix packed with rows={BLOCK}, got {w!r}")
    elif not isinstance(w, torch.Tensor) or w.dtype not in _FLOATS:
        raise TypeError(f"{name}: a weight is a floating-point matrix or a packed one, got {getattr(w, 'dtype', type(w).__name__)}")
    elif w.is_cuda and w.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the 8-bit products take and return bfloat16 on CUDA, got a weight in {w.dtype}")
    shape = w.shape
    if len(shape) != 2 or shape[1] != n_in or not shape[0] or not n_in:
        raise ValueError(f"{name}: a weight [out, {n_in}] was expected, got {tuple(shape)}")
    if (w.data if packed else w).device != x.device:
        raise ValueError(f"{name}: input on {x.device}, weight on {w.device}")
    return packed


def _differentiated(a, b=None) -> bool:
    """True if autograd has to see the call: a gradient will be asked for, or a forward-mode level is open (whose tangents
    are refused there; a plain call would drop them)."""
    return ((torch.is_grad_enabled() and (a.requires_grad or (b is not None and b.requires_grad)))
            or forward_ad._current_level >= 0)


def fp8_linear(x: torch.Tensor, weight: Union[torch.Tensor, Fp8Blocks]) -> torch.Tensor:
    """``x @ weight^T`` as a product of 8-bit operands; ``weight [out, in]`` is a tensor (packed in the call, receives a
    gradient) or what :func:`pack_fp8` made of one (frozen: only ``x`` receives a gradient)."""
    _check_activation("fp8_linear", x)
    packed = _check_weight("fp8_linear", weight, x, x.shape[-1])
    if not packed:
        return _Linear.apply(x, weight)
    if _differentiated(x):
        return _LinearFrozen.apply(x, weight.data, weight)
    return _linear_frozen(x, weight)


class _ChannelMix(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wk, wv, residual):
        x2, dev = _rows_of(x), x.device
        (M, C), (N, H) = x2.shape, wv.shape
        need_x, need_k, need_v, _ = ctx.needs_input_grad
        specs = ((M, C, BLOCK), (H, C, BLOCK), (N, H, BLOCK), (M, H, BLOCK))
        keep = (need_k, need_x, need_x or need_k, need_x or need_k or need_v)
        ops8 = _room(dev, *(s if k else None for s, k in zip(specs, keep)))
        ctx.save_for_backward(ops8[3].data if keep[3] else None)
        ctx.meta, ctx.shape, ctx.types = [_meta(p) for p in ops8], x.shape, (x.dtype, wk.dtype, wv.dtype)
        if not all(keep):
            ops8 = [a or b for a, b in zip(ops8, _room(dev, *(None if k else s for s, k in zip(specs, keep))))]
        x8, k8, v8, h8 = ops8
        y = torch.empty(residual.shape, dtype=x.dtype, device=dev)
        run = _run_on(x)
        run.pack(x2, x8)
        run.pack(wk, k8)
        run.pack(wv, v8)
        run.nt_relu_sq(x8, k8, h8)
        run.nt(h8, v8, _rows_of(y), _rows_of(residual))
        run.go()
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (data,) = ctx.saved_tensors
        need_x, need_k, need_v, need_r = ctx.needs_input_grad
        dx = dwk = dwv = None
        if data is not None:
            x8, k8, v8, h8 = (None if m is None else Fp8Blocks(data, *m) for m in ctx.meta)
            d2, dev = _rows_of(dy), dy.device
            d8, p8 = _room(dev, (*d2.shape, BLOCK), (h8.R, h8.C, BLOCK) if need_x or need_k else None)
            run = _run_on(dy)
            run.pack(d2, d8)
            if need_x or need_k:
                run.nn_relu_sq_grad(d8, v8, h8, p8)
            if need_x:
                dx = torch.empty(ctx.shape, dtype=ctx.types[0], device=dev)
                run.nn(p8, k8, _rows_of(dx))
            if need_k:
                dwk = torch.empty(p8.C, x8.C, dtype=ctx.types[1], device=dev)
            if need_v:
                dwv = torch.empty(d8.C, h8.C, dtype=ctx.types[2], device=dev)
            if need_k and need_v:
                run.tn_two(p8, x8, dwk, d8, h8, dwv)
            elif need_k:
                run.tn(p8, x8, dwk)
            elif need_v:
                run.tn(d8, h8, dwv)
            run.go()
        return dx, dwk, dwv, (dy if need_r else None)


class _ChannelMixFrozen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kdata, vdata, residual, k8, v8):
        y, h8 = _channel_mix_frozen(x, k8, v8, residual)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(kdata, vdata, h8.data)
            ctx.meta, ctx.shape = [_meta(p) for p in (k8, v8, h8)], x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            k8, v8, h8 = (Fp8Blocks(d, *m) for d, m in zip(ctx.saved_tensors, ctx.meta))
            d2 = _rows_of(dy)
            d8, p8 = _room(dy.device, (*d2.shape, 1), (h8.R, h8.C, 1))
            dx = torch.empty(ctx.shape, dtype=dy.dtype, device=dy.device)
            run = _run_on(dy)
            run.pack(d2, d8)
            run.nn_relu_sq_grad(d8, v8, h8, p8)
            run.nn(p8, k8, _rows_of(dx))
            run.go()
        return dx, None, None, (dy if ctx.needs_input_grad[3] else None), None, None


def _channel_mix_frozen(x, k8, v8, residual):
    x2 = _rows_of(x)
    h8 = _matrix(x.device, x2.shape[0], k8.R, 1)
    y = x.new_empty(residual.shape)
    run = _run_on(x)
    run.nt_frozen(x2, k8, None, h8)
    run.nt(h8, v8, _rows_of(y), _rows_of(residual))
    run.go()
    return y, h8


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
    want = (*xk.shape[:-1], w_value.shape[0])
    if residual.shape != want:
        raise ValueError(f"{name}: a residual of shape {want} was expected, got {tuple(residual.shape)}")
    if not residual.is_contiguous() and (residual.dim() != 2 or residual.stride(1) != 1 or residual.stride(0) < residual.shape[1]):
        residual = residual.contiguous()
    if not packed:
        return _ChannelMix.apply(xk, w_key, w_value, residual)
    if _differentiated(xk, residual):
        return _ChannelMixFrozen.apply(xk, w_key.data, w_value.data, residual, w_key, w_value)
    return _channel_mix_frozen(xk, w_key, w_value, residual)[0]
