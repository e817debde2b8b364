"""8-bit blocks on the CPU: the format against its definition in 64 bits, products and gradients against formulas, refusals."""
import math

import pytest
import torch

from rwkvtune_b200 import ops

BF = torch.bfloat16
E4M3 = [i * 2.0 ** -9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 3) for e in range(-6, 9) for i in range(8)][:-1]


def oracle_pack(x, rows):
    """Values (64 bits) that packing stands for, block by block in plain Python loops over blocks."""
    R, C = x.shape
    numbers = torch.tensor(E4M3, dtype=torch.float64)
    out = torch.empty(R, C, dtype=torch.float64)
    for r in range(0, R, rows):
        for c in range(0, C, 128):
            b = x[r:r + rows, c:c + 128].double()
            if not torch.isfinite(b).all():
                out[r:r + rows, c:c + 128] = math.nan
                continue
            e = -127
            while b.abs().max().item() > 448 * 2.0 ** e:
                e += 1
            v = b / 2.0 ** e
            far = (v.abs().unsqueeze(-1) - numbers).abs()
            best = far.amin(-1, keepdim=True)
            near = far == best                                       # one entry, or two at a tie: the even one
            index = torch.arange(numbers.numel())
            pick = torch.where(near & ((index % 2 == 0) | (near.sum(-1, keepdim=True) == 1)), index, -1).amax(-1)
            out[r:r + rows, c:c + 128] = torch.copysign(numbers[pick], v) * 2.0 ** e
    return out


def sample(R, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g) * torch.exp(3 * torch.randn(R, 1, generator=g))
    x[:, ::37] *= 50
    return x.to(dtype)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 128), (3, 129), (130, 257), (128, 16), (257, 100)])
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_pack_is_the_definition(R, C, rows, dtype):
    x = sample(R, C, dtype)
    p = ops.pack_fp8(x, rows=rows)
    # the rows of the fp16 sample that overflow are non-finite blocks
    torch.testing.assert_close(ops.unpack_fp8(p, torch.float32).double(), oracle_pack(x, rows), rtol=0, atol=0, equal_nan=True)
    assert p.values.shape == (R, C) and p.exponents.shape == (-(-R // rows), -(-C // 128))
    y = ops.unpack_fp8(p)
    assert y.dtype == dtype and y.shape == x.shape


def test_borders_ties_and_signs():
    v = torch.tensor([[448.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, -17.0, 17.5, 19.0, -0.0]])   # 17, 19: ties
    p = ops.pack_fp8(v, rows=1)
    assert ops.unpack_fp8(p).tolist() == [[448.0, 2.0 ** -9, 0.0, 2.0 ** -8, -16.0, 18.0, 20.0, 0.0]]
    assert p.exponents.item() == 127
    assert ops.pack_fp8(torch.tensor([448.5]), rows=1).exponents.item() == 128
    assert ops.pack_fp8(torch.zeros(1, 4), rows=1).exponents.item() == 0


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite_blocks_become_nan_and_only_they(rows, bad):
    x = sample(130, 300, torch.float32)
    x[5, 140] = bad
    y = ops.unpack_fp8(ops.pack_fp8(x, rows=rows))
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[(slice(5, 6) if rows == 1 else slice(0, 128)), 128:256] = True
    assert torch.equal(y.isnan(), hit) and torch.isfinite(y[~hit]).all()


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_largest_finite_values_stay_finite(dtype):
    top = torch.finfo(dtype).max
    y = ops.unpack_fp8(ops.pack_fp8(torch.full((2, 130), top, dtype=dtype)))
    assert torch.equal(y, torch.full((2, 130), top, dtype=dtype))
    assert ops.unpack_fp8(ops.pack_fp8(torch.full((1, 3), 1e30)), torch.float16).tolist() == [[65504.0] * 3]


def test_shapes_leading_dimensions_and_empty():
    x = sample(6, 40, BF).view(2, 3, 40)
    p = ops.pack_fp8(x, rows=1)
    assert ops.unpack_fp8(p).shape == (2, 3, 40) and p.nbytes == 6 * 48 + 16
    assert torch.equal(ops.unpack_fp8(ops.pack_fp8(x.transpose(0, 1), rows=1)), ops.unpack_fp8(p).transpose(0, 1))
    for rows in (1, 128):
        e = ops.pack_fp8(torch.empty(0, 40), rows=rows)
        assert ops.unpack_fp8(e).shape == (0, 40) and e.exponents.shape == (0, 1)
    assert ops.unpack_fp8(ops.pack_fp8(torch.ones(7))).shape == (7,)


def test_packing_again_in_place():
    x, y = sample(6, 40, BF).view(2, 3, 40), sample(6, 40, BF, 1).view(2, 3, 40)
    for rows in (1, 128):
        p = ops.pack_fp8(x, rows=rows)
        q = ops.pack_fp8(y, rows=rows, out=p)
        assert q is p and torch.equal(ops.unpack_fp8(p), ops.unpack_fp8(ops.pack_fp8(y, rows=rows)))
        for bad in (y[:1], y.float(), y.transpose(0, 1)):
            with pytest.raises(ValueError):
                ops.pack_fp8(bad, rows=rows, out=p)
        with pytest.raises(ValueError):
            ops.pack_fp8(y, rows=129 - rows, out=p)
    with pytest.raises(ValueError):
        ops.pack_fp8(y, out=p.data)
    w = ops.pack_fp8(weights(16, 40))
    a = sample(3, 40, torch.float32).requires_grad_()
    out = ops.fp8_linear(a, w).sum()
    ops.pack_fp8(weights(16, 40, 5), out=w)
    with pytest.raises(RuntimeError):              # the forward pass saw other weights
        out.backward()


def weights(N, K, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(N, K, generator=g) - 0.5) * 2 / math.sqrt(K)


@pytest.mark.parametrize("M,K,N", [(1, 128, 16), (130, 200, 70), (5, 64, 1)])
@pytest.mark.parametrize("frozen", [False, True])
def test_linear_and_gradients_follow_the_formulas(M, K, N, frozen):
    x, w, dy = sample(M, K, torch.float32).requires_grad_(), weights(N, K), sample(M, N, torch.float32, 3)
    rows = 1 if frozen else 128
    X, W, D = oracle_pack(x.detach(), rows), oracle_pack(w, 128), oracle_pack(dy, rows)
    if frozen:
        y = ops.fp8_linear(x, ops.pack_fp8(w))
        (dx,) = torch.autograd.grad(y, [x], dy)
    else:
        w.requires_grad_()
        y = ops.fp8_linear(x, w)
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        near(dw, D.t() @ X, D.abs().t() @ X.abs(), M)
    near(y, X @ W.t(), X.abs() @ W.abs().t(), K)
    near(dx, D @ W, D.abs() @ W.abs(), N)


def near(got, want, magnitude, n, extra=0.0):
    """fp32 sums of n terms: at most n + 1 roundings of a partial sum no larger than the sum of magnitudes."""
    assert ((got.double() - want).abs() <= (n + 1) * 2.0 ** -24 * magnitude + extra + 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("frozen", [False, True])
def test_channel_mix_and_gradients_follow_the_formulas(frozen):
    M, C, H = 140, 72, 200
    x, res, dy = (sample(M, C, torch.float32, s) for s in (0, 1, 2))
    wk, wv = weights(H, C), weights(C, H, 2)
    rows = 1 if frozen else 128
    X, K, V, D = oracle_pack(x, rows), oracle_pack(wk, 128), oracle_pack(wv, 128), oracle_pack(dy, rows)
    h = torch.relu((X.float() @ K.float().t())) ** 2              # the packed activation depends on fp32 sums next to borders
    h = oracle_pack(h, rows)
    p = oracle_pack((D.float() @ V.float()) * 2 * h.float().sqrt(), rows)
    x.requires_grad_(), res.requires_grad_()
    if frozen:
        y = ops.fp8_channel_mix_ffn(x, ops.pack_fp8(wk), ops.pack_fp8(wv), res)
        dx, dr = torch.autograd.grad(y, [x, res], dy)
    else:
        wk.requires_grad_(), wv.requires_grad_()
        y = ops.fp8_channel_mix_ffn(x, wk, wv, res)
        dx, dk, dv, dr = torch.autograd.grad(y, [x, wk, wv, res], dy)
        near(dk, p.t() @ X, p.abs().t() @ X.abs(), M)
        near(dv, D.t() @ h, D.abs().t() @ h.abs(), M)
    near(y, res.double() + h @ V.t(), h.abs() @ V.abs().t() + res.double().abs(), H)
    near(dx, p @ K, p.abs() @ K.abs(), H)
    assert torch.equal(dr, dy)


def test_gradients_against_differences():
    """Along a direction u, <grad, u> against a central difference of the unpacked map in 64 bits.  The loss is quadratic
    in each input along u for the linear map, so the difference itself is exact; what is left is that packing moves every
    operand by at most 2^-4 of itself, so the two directional derivatives differ by at most ((1 + 2^-4)^2 - 1) times the
    sum of magnitudes of their terms."""
    M, K, N = 40, 64, 48
    x, w, dy, u = (sample(M, K, torch.float32).requires_grad_(), weights(N, K).requires_grad_(), sample(M, N, torch.float32, 3),
                   sample(N, K, torch.float32, 4))
    gx, gw = torch.autograd.grad(ops.fp8_linear(x, w), [x, w], dy)
    X, W, D, U = x.detach().double(), w.detach().double(), dy.double(), u.double()
    loss = lambda x_, w_: (x_ @ w_.t() * D).sum()  # noqa: E731
    slack = (1 + 2.0 ** -4) ** 2 - 1
    fd = (loss(X, W + U) - loss(X, W - U)) / 2
    # values far below a tile's largest are rounded by at most 2^-10 * 2^e, e from 448 * 2^(e - 1) < largest
    tiny = lambda t: t.abs().max() / 448 * 2 * 2.0 ** -10 * torch.ones_like(t)  # noqa: E731
    size = lambda t: t.abs() * (1 + 2.0 ** -4) + tiny(t)  # noqa: E731
    bound = ((size(D).t() @ size(X) - D.abs().t() @ X.abs()) * U.abs()).sum()
    assert abs((gw.double() * U).sum() - fd) <= bound and bound < 1e6 * slack * fd.abs().clamp(min=1)
    UX = sample(M, K, torch.float32, 5).double()
    fd = (loss(X + UX, W) - loss(X - UX, W)) / 2
    bound = ((size(D) @ size(W) - D.abs() @ W.abs()) * UX.abs()).sum()
    assert abs((gx.double() * UX).sum() - fd) <= bound


def test_only_what_needs_a_gradient_gets_one():
    x, w = sample(9, 64, torch.float32), weights(32, 64)
    for rx, rw in ((True, False), (False, True)):
        a, b = x.clone().requires_grad_(rx), w.clone().requires_grad_(rw)
        ops.fp8_linear(a, b).sum().backward()
        assert (a.grad is not None) == rx and (b.grad is not None) == rw
    assert not ops.fp8_linear(x, w).requires_grad
    wk, wv, res = weights(64, 64), weights(64, 64, 3), sample(9, 64, torch.float32, 4)
    for req in range(16):
        ts = [t.clone().requires_grad_(bool(req >> i & 1)) for i, t in enumerate((x, wk, wv, res))]
        y = ops.fp8_channel_mix_ffn(*ts)
        if req:
            y.sum().backward()
        assert [t.grad is not None for t in ts] == [bool(req >> i & 1) for i in range(4)]
    k8, v8 = ops.pack_fp8(wk), ops.pack_fp8(wv)
    for req in range(1, 4):
        a, r = x.clone().requires_grad_(bool(req & 1)), res.clone().requires_grad_(bool(req & 2))
        ops.fp8_channel_mix_ffn(a, k8, v8, r).sum().backward()
        assert (a.grad is not None, r.grad is not None) == (bool(req & 1), bool(req & 2))


def test_frozen_rows_do_not_depend_on_the_batch():
    w8 = ops.pack_fp8(weights(48, 96))
    x = sample(130, 96, torch.float32)
    # the same packed row whatever its neighbours; the library product behind the CPU form may sum in another order
    full, alone = ops.fp8_linear(x, w8), torch.cat([ops.fp8_linear(x[i:i + 1], w8) for i in range(130)])
    size = oracle_pack(x, 1).abs() @ oracle_pack(weights(48, 96), 128).abs().t()
    assert ((full - alone).double().abs() <= 2 * 97 * 2.0 ** -24 * size).all()


def test_empty_batches():
    w = weights(48, 96).requires_grad_()
    x = torch.empty(2, 0, 96, requires_grad=True)
    y = ops.fp8_linear(x, w)
    y.sum().backward()
    assert y.shape == (2, 0, 48) and x.grad.shape == x.shape and torch.equal(w.grad, torch.zeros_like(w))
    wk, wv = weights(64, 96).requires_grad_(), weights(96, 64).requires_grad_()
    out = ops.fp8_channel_mix_ffn(x, wk, wv, torch.empty(2, 0, 96))
    out.sum().backward()
    assert out.shape == (2, 0, 96) and wk.grad.abs().sum() == 0 and wv.grad.abs().sum() == 0
    assert ops.fp8_channel_mix_ffn(x.detach(), ops.pack_fp8(wk), ops.pack_fp8(wv), torch.empty(2, 0, 96)).shape == (2, 0, 96)


def test_refusals():
    x, w = torch.ones(4, 64), torch.ones(8, 64)
    with pytest.raises(TypeError):
        ops.pack_fp8(torch.ones(4, 64, dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.pack_fp8([1.0])
    with pytest.raises(TypeError):
        ops.pack_fp8(x.double())
    for rows in (0, 2, 64, None):
        with pytest.raises(ValueError):
            ops.pack_fp8(x, rows=rows)
    with pytest.raises(ValueError):
        ops.pack_fp8(torch.ones(3, 0))
    with pytest.raises(ValueError):
        ops.pack_fp8(torch.tensor(1.0))
    with pytest.raises(TypeError):
        ops.unpack_fp8(x)
    with pytest.raises(TypeError):
        ops.unpack_fp8(ops.pack_fp8(x), torch.int8)
    with pytest.raises(ValueError):
        ops.fp8_linear(x, torch.ones(8, 63))
    with pytest.raises(ValueError):
        ops.fp8_linear(x, ops.pack_fp8(w, rows=1))
    with pytest.raises(ValueError):
        ops.fp8_linear(x, ops.pack_fp8(torch.ones(2, 4, 64)))
    with pytest.raises(ValueError):
        ops.fp8_linear(x, torch.ones(0, 64))
    with pytest.raises(TypeError):
        ops.fp8_linear(x, w.int())
    with pytest.raises(TypeError):
        ops.fp8_linear(x.long(), w)
    with pytest.raises(TypeError):
        ops.fp8_linear(x, None)
    wv, res = torch.ones(64, 8), torch.ones(4, 64)
    with pytest.raises(ValueError):
        ops.fp8_channel_mix_ffn(x, w, ops.pack_fp8(wv), res)
    with pytest.raises(ValueError):
        ops.fp8_channel_mix_ffn(x, ops.pack_fp8(w), wv, res)
    with pytest.raises(ValueError):
        ops.fp8_channel_mix_ffn(x, w, torch.ones(64, 9), res)
    with pytest.raises(ValueError):
        ops.fp8_channel_mix_ffn(x, w, wv, torch.ones(64))
    with pytest.raises(TypeError):
        ops.fp8_channel_mix_ffn(x, w, wv, res.to(BF))


def test_no_second_derivative():
    x, w = torch.ones(4, 64, requires_grad=True), torch.ones(8, 64, requires_grad=True)
    (g,) = torch.autograd.grad(ops.fp8_linear(x, w).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("shape", [(64,), (4, 64), (2, 3, 64), (0, 3, 64)])
def test_result_may_be_written_in_place(shape, frozen):
    # the map is y = P(x) P(W)^T and then 2 y + 1 in place: the gradient is twice that of y itself, exactly (a power of two)
    x, w = torch.randn(shape, requires_grad=True), torch.randn(40, 64)
    weight = ops.pack_fp8(w) if frozen else w.requires_grad_()
    y = ops.fp8_linear(x, weight)
    (want,) = torch.autograd.grad(y.sum(), [x])
    z = ops.fp8_linear(x, weight)
    z.mul_(2).add_(1)
    assert torch.equal(z, y * 2 + 1)
    (got,) = torch.autograd.grad(z.sum(), [x])
    assert torch.equal(got, 2 * want)


@pytest.mark.parametrize("again", [False, True])
def test_packed_under_inference_mode(again):
    """A weight packed for serving can be packed again and trained against outside of it, and the other way round."""
    w, v, x = weights(16, 40), weights(16, 40, 5), sample(3, 40, torch.float32)
    for rows in (1, 128):
        with torch.inference_mode():
            p = ops.pack_fp8(w, rows=rows)
        with torch.inference_mode(again):
            ops.pack_fp8(v, rows=rows, out=p)
        assert torch.equal(ops.unpack_fp8(p), ops.unpack_fp8(ops.pack_fp8(v, rows=rows)))
    a = x.clone().requires_grad_()
    ops.fp8_linear(a, p).sum().backward()
    b = x.clone().requires_grad_()
    ops.fp8_linear(b, ops.pack_fp8(v)).sum().backward()
    assert torch.equal(a.grad, b.grad)
    with torch.inference_mode():
        assert torch.equal(ops.fp8_linear(x, p), ops.fp8_linear(x, ops.pack_fp8(v)))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("frozen", [False, True])
def test_forward_mode_derivatives_are_refused(frozen, grad):
    """No tangent is dropped in silence; tensors without one pass through an open level as they are."""
    import torch.autograd.forward_ad as fwd

    x, res, wk, wv = sample(4, 64, torch.float32), sample(4, 64, torch.float32, 2), weights(32, 64), weights(64, 32)
    if frozen:
        wk, wv = ops.pack_fp8(wk), ops.pack_fp8(wv)
    want = ops.fp8_linear(x, wk), ops.fp8_channel_mix_ffn(x, wk, wv, res)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        dual, dual_res = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(res, torch.ones_like(res))
        for call in (lambda: ops.fp8_linear(dual, wk), lambda: ops.fp8_channel_mix_ffn(dual, wk, wv, res),
                     lambda: ops.fp8_channel_mix_ffn(x, wk, wv, dual_res)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(ops.fp8_linear(x, wk), want[0]) and torch.equal(ops.fp8_channel_mix_ffn(x, wk, wv, res), want[1])


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_numbers_below_the_normal_ones_count_as_zero(dtype, rows):
    low = 2.0 ** -126
    x = torch.tensor([[low, -low, low / 2, -low / 2, low / 128, low * 1.5, 0.0]], dtype=dtype)
    p = ops.pack_fp8(x, rows=rows)
    assert p.exponents.item() == 0 and p.values.float().tolist() == [[2.0, -2.0, 0.0, 0.0, 0.0, 3.0, 0.0]]
    assert torch.signbit(p.values.float()).tolist() == [[False, True, False, True, False, False, False]]
    assert ops.unpack_fp8(p).tolist() == [[low, -low, 0.0, 0.0, 0.0, low * 1.5, 0.0]]
    # small against the block's largest, above 2^-126 as they are and below it once rounded down
    y = torch.tensor([[448 * 2.0 ** -126, 2.0 ** -126 * 1.0625, 2.0 ** -127 * 1.9]], dtype=torch.float32)
    q = ops.pack_fp8(y, rows=rows)
    assert q.exponents.item() == 1 and ops.unpack_fp8(q).tolist() == [[448 * 2.0 ** -126, 2.0 ** -126, 0.0]]
