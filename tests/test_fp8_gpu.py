"""8-bit block kernels: packing bit for bit against the CPU statement, products against 64-bit products of the packed
operands, gradients through the public entry points."""
import math

import pytest
import torch

from rwkvtune_b200 import ops
from rwkvtune_b200.ops import fp8, gemm_native
from rwkvtune_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def no_expired_wait():
    yield
    torch.cuda.synchronize()
    assert gemm_native.check_status() == 0


def product(name, a, b, M, N, *more):
    out = torch.full((M, N), math.nan, dtype=BF, device="cuda")
    run = fp8._run_on(a.data)
    getattr(run, name)(a, b, out, *more)
    run.go()
    return out


def packed_product(name, a, b, M, N, rows, *more):
    (q,) = fp8._room(a.device, (M, N, rows))
    run = fp8._run_on(a.data)
    getattr(run, name)(a, b, *more, q)
    run.go()
    return q


def sample(R, C, dtype=BF, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g) * torch.exp(2 * torch.randn(R, 1, generator=g))
    x[:, ::37] *= 50
    return x.clamp(-6e4, 6e4).to(dtype)


def weights(N, K, seed=1):
    g = torch.Generator().manual_seed(seed)
    return ((torch.rand(N, K, generator=g) - 0.5) * 2 / math.sqrt(K)).to(BF)


def same_bits(p, x, rows):
    values, exponents = ref.fp8_pack(x.cpu(), rows)
    assert torch.equal(p.exponents.cpu(), exponents)
    got, want = p.values.cpu().view(torch.uint8), values.view(torch.uint8)
    nan = exponents.repeat_interleave(rows, 0)[:x.shape[0]].repeat_interleave(128, 1)[:, :x.shape[1]] == 255
    assert torch.equal(got[~nan], want[~nan]) and (got[nan] & 0x7F == 0x7F).all()


# ------------------------------------------------------------------------------- packing
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 2048), (5, 130), (128, 128), (130, 257), (300, 1000), (129, 90)])
def test_pack_and_unpack(R, C, dtype, rows):
    x = sample(R, C, dtype).cuda()
    p = ops.pack_fp8(x, rows=rows)
    same_bits(p, x, rows)
    for out in (BF, torch.float16, torch.float32):
        want = ops.unpack_fp8(p.to("cpu"), out)
        assert torch.equal(ops.unpack_fp8(p, out).cpu(), want)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_pack_of_strided_and_unaligned_inputs(rows, dtype):
    base = sample(140, 410, dtype).cuda()
    for x in (base[:, 1:301], base[3:, 8:264], base[::2, 2:200], base.t(), base[:1, 5:9], base[:, ::2],
              base[0].expand(140, 410), base.view(-1)[1:1 + 139 * 410].view(139, 410)):
        same_bits(ops.pack_fp8(x, rows=rows), x.contiguous(), rows)


@pytest.mark.parametrize("rows", [1, 128])
def test_pack_of_non_finite_zero_and_extreme_blocks(rows):
    x = sample(260, 400, torch.float32)
    x[5, 140], x[200, 3], x[130, 399] = math.nan, math.inf, -math.inf
    x[128:256, 128:256] = 0
    x[256:, :128] = 3.4e38
    x[256:, 128:256] = 2.0 ** -120
    x = x.cuda()
    p = ops.pack_fp8(x, rows=rows)
    same_bits(p, x, rows)
    y = ops.unpack_fp8(p)
    torch.testing.assert_close(y.cpu(), ops.unpack_fp8(p.to("cpu")), rtol=0, atol=0, equal_nan=True)
    assert torch.isfinite(y[256:, :256]).all()


# ------------------------------------------------------------------------------- products
def values64(p):
    return ops.unpack_fp8(p, torch.float32).double()


def near(got, want, magnitude, n):
    """One rounding to bf16 (half a step: 2^-8 of the value) on top of fp32 sums: an instruction adds 32 products and the
    running sum with an error of at most 2^-22 of the largest magnitude that occurs, n / 32 instructions one after another."""
    assert got.shape == want.shape and got.dtype == BF
    tol = 2.0 ** -8 * want.abs() + (n / 32 + 1) * 2.0 ** -22 * magnitude + 1e-38
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
                          f"{got[bad][0].item()} for {want[bad][0].item()}"


SIZES = [(128, 128, 128), (256, 256, 256), (1, 128, 128), (300, 520, 384), (5, 24, 40), (257, 130, 1000), (1000, 523, 129),
         (64, 2048, 640), (700, 1024, 2048)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("rows", [1, 128])
def test_nt(M, N, K, rows):
    a, b = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(N, K).cuda())
    A, B = values64(a), values64(b)
    near(product("nt", a, b, M, N), A @ B.t(), A.abs() @ B.abs().t(), K)


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("rows", [1, 128])
def test_nt_residual(M, N, K, rows):
    a, b, c = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(N, K).cuda()), sample(M, N, seed=7).cuda()
    A, B = values64(a), values64(b)
    near(product("nt", a, b, M, N, c), c.double() + A @ B.t(), A.abs() @ B.abs().t() + c.double().abs(), K)


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("rows", [1, 128])
def test_nn(M, N, K, rows):
    a, b = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(K, N).cuda())
    A, B = values64(a), values64(b)
    near(product("nn", a, b, M, N), A @ B, A.abs() @ B.abs(), K)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_tn(M, N, K):
    a, b = ops.pack_fp8(sample(K, M).cuda()), ops.pack_fp8(sample(K, N, seed=5).cuda())
    A, B = values64(a), values64(b)
    near(product("tn", a, b, M, N), A.t() @ B, A.abs().t() @ B.abs(), K)


def packed_near(q, want, magnitude, n, rows):
    """A packed result: each value within half an e4m3 step (2^-4 of it, or 2^-10 of its block's unit) of the 64-bit one,
    plus the fp32 sums' own error; scales as the definition gives them from the 64-bit values."""
    tol_sum = (n / 32 + 1) * 2.0 ** -22 * magnitude
    top = torch.nn.functional.pad(want.abs(), (0, -want.shape[1] % 128, 0, -want.shape[0] % rows))
    top = top.unflatten(1, (-1, 128)).unflatten(0, (-1, rows)).amax(dim=(1, 3))
    assert torch.equal(q.exponents, ref.fp8_exponents(top.float()))
    unit = torch.exp2(q.exponents.double() - 127).repeat_interleave(rows, 0)[:q.R].repeat_interleave(128, 1)[:, :q.C]
    tol = 2.0 ** -4 * want.abs() + 2.0 ** -10 * unit + 2 * tol_sum + 1e-38
    assert ((values64(q) - want).abs() <= tol).all()


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("rows", [1, 128])
def test_relu_sq_packed(M, N, K, rows):
    a, b = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(N, K).cuda())
    A, B = values64(a), values64(b)
    pre, mag = A @ B.t(), A.abs() @ B.abs().t()
    packed_near(packed_product("nt_relu_sq", a, b, M, N, rows), torch.relu(pre) ** 2, 2 * pre.abs() * mag + 1e-30, K, rows)


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("rows", [1, 128])
def test_relu_sq_grad_packed(M, N, K, rows):
    d, w = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(K, N).cuda())
    h = ops.pack_fp8((torch.relu(sample(M, N, seed=3).float()) ** 2).to(BF).cuda(), rows=rows)
    D, W, slope = values64(d), values64(w), 2 * values64(h).sqrt()
    packed_near(packed_product("nn_relu_sq_grad", d, w, M, N, rows, h), (D @ W) * slope, (D.abs() @ W.abs()) * slope + 1e-30, K + 64, rows)


@pytest.mark.parametrize("N,K", [(128, 128), (40, 24), (200, 264), (2048, 2048), (640, 8192), (130, 1000), (8192, 512), (20000, 128),
                                 (40100, 136), (77000, 640), (200, 33000)])
@pytest.mark.parametrize("M", [1, 2, 16, 17, 64, 100, 128])
def test_few_rows(M, N, K):
    """The decode kernel: bf16 tokens packed inside it, packed tokens, and its three epilogues."""
    from rwkvtune_b200.ops import fp8_native as native

    x, w8 = sample(M, K).cuda(), ops.pack_fp8(weights(N, K).cuda())
    x8, res = ops.pack_fp8(x, rows=1), sample(M, N, seed=7).cuda()
    A, B = values64(x8), values64(w8)
    pre, mag = A @ B.t(), A.abs() @ B.abs().t()
    assert native.decode_form(M, N, K, True) == 1 and native.decode_form(M, N, K) == (2 if M <= 16 and K % 8 == 0 else 1)
    forms = [x8] + ([x] if native.decode_form(M, N, K) == 2 else [])
    for t in forms:
        out, out_r = (torch.full((M, N), math.nan, dtype=BF, device="cuda") for _ in range(2))
        (q,) = fp8._room(x.device, (M, N, 1))
        native.run(x.device, [native.decode(t, w8, out), native.decode(x8, w8, out_r, res), native.decode(t, w8, q=q)])
        near(out, pre, mag, K)
        near(out_r, res.double() + pre, mag + res.double().abs(), K)
        packed_near(q, torch.relu(pre) ** 2, 2 * pre.abs() * mag + 1e-30, K, 1)
    if len(forms) == 2:
        out2 = torch.empty_like(out)
        native.run(x.device, [native.decode(x8, w8, out2)])
        assert torch.equal(out, out2)


def test_few_rows_of_strided_inputs():
    w8 = ops.pack_fp8(weights(200, 256).cuda())
    base = sample(40, 600).cuda()
    for x in (base[:3, 1:257], base[:16, 8:264], base[::4, :256], base[:2, :512:2], base[0, :256].expand(5, 256), base[7, 3:259]):
        assert torch.equal(ops.fp8_linear(x, w8), ops.fp8_linear(x.contiguous().clone(), w8))


def test_weights_packed_just_before_a_chained_product():
    """Fresh weights every time: a product that fetched them before they were written would show old bytes."""
    x, res = sample(20, 512).cuda(), sample(20, 512, seed=3).cuda()
    for seed in range(6):
        wk, wv = weights(1024, 512, seed).cuda(), weights(512, 1024, seed + 50).cuda()
        torch.cuda.synchronize()
        k8, v8 = ops.pack_fp8(wk), ops.pack_fp8(wv)
        y = ops.fp8_channel_mix_ffn(x, k8, v8, res)
        torch.cuda.synchronize()
        assert torch.equal(y, ops.fp8_channel_mix_ffn(x, k8, v8, res))


def test_long_contraction_and_many_tiles():
    """More tiles than SM pairs, more scale sets than the ring holds, 8-bit scales that differ from block to block."""
    M, N, K = 2600, 2100, 5000
    for rows in (1, 128):
        a, b = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(N, K).cuda())
        A, B = values64(a), values64(b)
        near(product("nt", a, b, M, N), A @ B.t(), A.abs() @ B.abs().t(), K)
        q = packed_product("nt_relu_sq", a, b, M, N, rows)
        pre = A @ B.t()
        packed_near(q, torch.relu(pre) ** 2, 2 * pre.abs() * (A.abs() @ B.abs().t()) + 1e-30, K, rows)
    b = ops.pack_fp8(weights(M, N, 4).cuda())
    a = ops.pack_fp8(sample(M, K).cuda())
    A, B = values64(a), values64(b)
    near(product("tn", a, b, K, N), A.t() @ B, A.abs().t() @ B.abs(), M)


@pytest.mark.parametrize("first,second", [((300, 520, 384), (130, 90, 1000)), ((2048, 1024, 129), (1024, 2048, 129)),
                                          ((1, 1, 1), (4100, 2600, 700)), ((200, 300, 6000), (130, 523, 2500)), ((200, 300, 6000), (130, 523, 5000)),
                                          ((300, 300, 4000), (4100, 2600, 700))])
def test_two_products_in_one_launch(first, second):
    args, wants = [], []
    for i, (M, N, K) in enumerate((first, second)):
        a, b = ops.pack_fp8(sample(K, M, seed=i).cuda()), ops.pack_fp8(sample(K, N, seed=5 + i).cuda())
        args += [a, b, torch.full((M, N), math.nan, dtype=BF, device="cuda")]
        A, B = values64(a), values64(b)
        wants.append((A.t() @ B, A.abs().t() @ B.abs(), K))
    run = fp8._run_on(args[2])
    run.tn_two(*args)
    run.go()
    for out, want in zip(args[2::3], wants):
        near(out, *want)


@pytest.mark.parametrize("M,N,K", [(130, 200, 5000), (257, 523, 8200), (300, 64, 33000), (1000, 1024, 8192), (129, 40, 5050)])
def test_few_tiles_and_a_long_contraction(M, N, K):
    """Products whose contraction runs in slices, in all three layouts, with a residual and with rows that are not aligned."""
    from rwkvtune_b200.ops import fp8_native as native

    assert native._workspace_bytes(M, N, K) > 0
    res = sample(M, N, seed=7).cuda()
    for rows in (1, 128):
        a, b = ops.pack_fp8(sample(M, K).cuda(), rows=rows), ops.pack_fp8(weights(N, K).cuda())
        A, B = values64(a), values64(b)
        near(product("nt", a, b, M, N), A @ B.t(), A.abs() @ B.abs().t(), K)
        near(product("nt", a, b, M, N, res), res.double() + A @ B.t(), A.abs() @ B.abs().t() + res.double().abs(), K)
        b = ops.pack_fp8(weights(K, N).cuda())
        B = values64(b)
        near(product("nn", a, b, M, N), A @ B, A.abs() @ B.abs(), K)
    a, b = ops.pack_fp8(sample(K, M).cuda()), ops.pack_fp8(sample(K, N, seed=5).cuda())
    A, B = values64(a), values64(b)
    near(product("tn", a, b, M, N), A.t() @ B, A.abs().t() @ B.abs(), K)


def test_non_finite_blocks_reach_exactly_their_products():
    x, w = sample(300, 256), weights(64, 256)
    x[140, 3] = math.inf
    y = ops.fp8_linear(x.cuda(), ops.pack_fp8(w.cuda()))
    assert y[140].isnan().all() and torch.isfinite(torch.cat([y[:140], y[141:]])).all()
    y = ops.fp8_linear(x.cuda(), w.cuda())
    assert y[128:256].isnan().all() and torch.isfinite(torch.cat([y[:128], y[256:]])).all()
    out = ops.fp8_channel_mix_ffn(x.cuda(), w.cuda(), weights(256, 64).cuda(), x.cuda().nan_to_num(0, 0, 0))
    assert out[128:256].isnan().all() and torch.isfinite(out[256:]).all()
    out = ops.fp8_channel_mix_ffn(x.cuda(), ops.pack_fp8(w.cuda()), ops.pack_fp8(weights(256, 64).cuda()),
                                  x.cuda().nan_to_num(0, 0, 0))
    assert out[140].isnan().all() and torch.isfinite(torch.cat([out[:140], out[141:]])).all()


# ------------------------------------------------------------------------------- through the public entry points
@pytest.mark.parametrize("shape,N", [((1, 64), 128), ((2, 3, 200), 90), ((40, 17, 384), 523)])
@pytest.mark.parametrize("frozen", [False, True])
def test_linear_autograd(shape, N, frozen):
    K, M = shape[-1], math.prod(shape[:-1])
    rows = 1 if frozen else 128
    x = sample(M, K).view(shape).cuda().requires_grad_()
    w, dy = weights(N, K).cuda(), sample(M, N, seed=9).cuda()
    X, W, D = values64(ops.pack_fp8(x.detach().view(M, K), rows)), values64(ops.pack_fp8(w)), values64(ops.pack_fp8(dy, rows))
    y = ops.fp8_linear(x, ops.pack_fp8(w) if frozen else w.requires_grad_())
    assert y.shape == shape[:-1] + (N,) and y.is_contiguous()
    y.backward(dy.view(y.shape))
    near(y.view(M, N), X @ W.t(), X.abs() @ W.abs().t(), K)
    near(x.grad.view(M, K), D @ W, D.abs() @ W.abs(), N)
    if not frozen:
        near(w.grad, D.t() @ X, D.abs().t() @ X.abs(), M)


@pytest.mark.parametrize("M,C,H", [(1, 64, 256), (130, 192, 768), (1111, 256, 1000)])
@pytest.mark.parametrize("frozen", [False, True])
def test_channel_mix_autograd(M, C, H, frozen):
    rows = 1 if frozen else 128
    x, res = sample(M, C).cuda().requires_grad_(), sample(M, C, seed=2).cuda().requires_grad_()
    wk, wv, dy = weights(H, C).cuda(), weights(C, H, 3).cuda(), sample(M, C, seed=9).cuda()
    x8, k8, v8, d8 = ops.pack_fp8(x, rows), ops.pack_fp8(wk), ops.pack_fp8(wv), ops.pack_fp8(dy, rows)
    h8 = packed_product("nt_relu_sq", x8, k8, M, H, rows)                # these two are compared with their 64-bit values above
    p8 = packed_product("nn_relu_sq_grad", d8, v8, M, H, rows, h8)
    X, K, V, D, Hd, P = (values64(t) for t in (x8, k8, v8, d8, h8, p8))
    args = (k8, v8) if frozen else (wk.requires_grad_(), wv.requires_grad_())
    y = ops.fp8_channel_mix_ffn(x, *args, res)
    y.backward(dy)
    near(y, res.double() + Hd @ V.t(), Hd.abs() @ V.abs().t() + res.double().abs(), H)
    near(x.grad, P @ K, P.abs() @ K.abs(), H)
    assert torch.equal(res.grad, dy)
    if not frozen:
        near(wk.grad, P.t() @ X, P.abs().t() @ X.abs(), M)
        near(wv.grad, D.t() @ Hd, D.abs().t() @ Hd.abs(), M)


def test_frozen_rows_do_not_depend_on_the_batch():
    """Bit for bit among batches of at most 128 rows, and among larger ones; the two sum in different orders."""
    w8 = ops.pack_fp8(weights(384, 640).cuda())
    k8, v8 = ops.pack_fp8(weights(512, 640, 5).cuda()), ops.pack_fp8(weights(640, 512, 6).cuda())
    x, res = sample(300, 640).cuda(), sample(300, 640, seed=8).cuda()
    for f in (lambda a, r: ops.fp8_linear(a, w8), lambda a, r: ops.fp8_channel_mix_ffn(a, k8, v8, r)):
        few, many = f(x[:128], res[:128]), f(x, res)
        for i in (0, 1, 63, 127):
            assert torch.equal(f(x[i:i + 1], res[i:i + 1]), few[i:i + 1])
        assert torch.equal(f(x[:20], res[:20]), few[:20]) and torch.equal(f(x[:129], res[:129]), many[:129])


def test_same_bits_twice_and_on_other_streams():
    x, w = sample(900, 512).cuda().requires_grad_(), weights(700, 512).cuda().requires_grad_()
    dy = sample(900, 700, seed=4).cuda()

    def run():
        y = ops.fp8_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, [x, w], dy))

    first = run()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            results.append(run())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_and_replayed():
    k8, v8 = ops.pack_fp8(weights(512, 256).cuda()), ops.pack_fp8(weights(256, 512, 2).cuda())
    x, res = torch.zeros(70, 256, dtype=BF, device="cuda"), torch.zeros(70, 256, dtype=BF, device="cuda")
    with torch.no_grad():
        ops.fp8_channel_mix_ffn(x, k8, v8, res)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.fp8_channel_mix_ffn(x, k8, v8, res)
        for seed in (1, 2):
            x.copy_(sample(70, 256, seed=seed)), res.copy_(sample(70, 256, seed=seed + 10))
            graph.replay()
            assert torch.equal(out, ops.fp8_channel_mix_ffn(x, k8, v8, res))


def test_powers_of_two_pass_through():
    """Scales are powers of two: moving one from an operand to the other changes no bit, however far."""
    x, w = sample(200, 384).cuda(), weights(264, 384).cuda()
    for frozen in (False, True):
        hold = ops.pack_fp8 if frozen else (lambda t: t)
        want = ops.fp8_linear(x, hold(w))
        for e in (-90, -40, 40, 90):
            assert torch.equal(ops.fp8_linear(x * 2.0 ** e, hold(w * 2.0 ** -e)), want)
        assert torch.equal(ops.fp8_linear(x[:5] * 2.0 ** 80, hold(w * 2.0 ** -80)), ops.fp8_linear(x[:5], hold(w)))


@pytest.mark.parametrize("M", [3, 40, 300])
def test_strided_residuals_and_weights(M):
    base, x = sample(M, 700, seed=3).cuda(), sample(M, 256).cuda()
    wk, wv = weights(512, 256).cuda(), weights(256, 512, 2).cuda()
    args = ((wk, wv), (ops.pack_fp8(wk), ops.pack_fp8(wv)))
    for res in (base[:, 1:257], base[:, 8:264], base[:, ::2][:, :256], base[:1, :256].expand(M, 256), base.view(-1)[5:5 + M * 256].view(M, 256)):
        for a in args:
            assert torch.equal(ops.fp8_channel_mix_ffn(x, *a, res), ops.fp8_channel_mix_ffn(x, *a, res.contiguous().clone()))
    assert torch.equal(ops.fp8_linear(x, wk.t().contiguous().t()), ops.fp8_linear(x, wk))
    assert torch.equal(ops.fp8_linear(x.t().contiguous().t(), wk), ops.fp8_linear(x, wk))


def test_offsets_beyond_32_bits():
    R, C = 1_100_000, 2048                                    # 2.25 G values
    x = torch.zeros(R, C, dtype=BF, device="cuda")
    tail = sample(300, C).cuda()
    x[-300:], x[:300] = tail, tail
    w8 = ops.pack_fp8(weights(72, C).cuda())
    for rows in (1, 128):
        p = ops.pack_fp8(x, rows=rows)
        y = ops.unpack_fp8(p)
        off = R % 128 if rows == 128 else 0                   # the last tile is short: compare whole tiles
        want = ops.unpack_fp8(ops.pack_fp8(x[R - 300 - off - (R - 300 - off) % rows:], rows=rows))
        assert torch.equal(y[-300:], want[-300:]) and torch.equal(y[:256], ops.unpack_fp8(ops.pack_fp8(tail, rows=rows))[:256])
        del y, want
        out = product("nt", p, w8, R, 72)
        W = values64(w8)
        tail_values = ops.unpack_fp8(ops.pack_fp8(x[R - 300 - off - (R - 300 - off) % rows:], rows=rows), torch.float32).double()[-300:]
        near(out[-300:], tail_values @ W.t(), tail_values.abs() @ W.abs().t(), C)
        assert not out[300 + 128:1000].any()
        del out, p


def test_two_threads_at_once():
    import threading

    x, w = sample(150, 256).cuda(), weights(200, 256).cuda()
    w8 = ops.pack_fp8(w)
    want, errors = (ops.fp8_linear(x, w), ops.fp8_linear(x[:9], w8)), []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = ops.fp8_linear(x, w), ops.fp8_linear(x[:9], w8)
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        except Exception as exc:       # noqa: BLE001 - reported by the main thread
            errors.append(exc)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors


def test_plain_statement_on_the_gpu():
    """The family can be switched off like the others: the same operators in plain PyTorch."""
    x, w = sample(140, 256).cuda(), weights(96, 256).cuda()
    y, p = ops.fp8_linear(x, w), ops.pack_fp8(x)
    ops.set_kernel_enabled("fp8", False)
    try:
        plain, q = ops.fp8_linear(x, w), ops.pack_fp8(x)
    finally:
        ops.set_kernel_enabled("fp8", True)
    assert torch.equal(p.exponents, q.exponents) and torch.equal(ops.unpack_fp8(p), ops.unpack_fp8(q))
    X, W = values64(p), values64(ops.pack_fp8(w))
    near(plain, X @ W.t(), X.abs() @ W.abs().t(), 256)
    near(y, X @ W.t(), X.abs() @ W.abs().t(), 256)


def test_backward_captured_and_replayed():
    """A training pass as one graph: the replay follows the inputs, and leaves its own results alone."""
    x, w = torch.zeros(150, 256, dtype=BF, device="cuda").requires_grad_(), weights(200, 256).cuda().requires_grad_()
    dy = torch.zeros(150, 200, dtype=BF, device="cuda")

    def run():
        y = ops.fp8_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, [x, w], dy))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for seed in (1, 2):
        with torch.no_grad():
            x.copy_(sample(150, 256, seed=seed)), dy.copy_(sample(150, 200, seed=seed + 5))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(kept, run()))


def test_broadcast_gradients():
    x, w = sample(140, 128).cuda().requires_grad_(), weights(96, 128).cuda().requires_grad_()
    ops.fp8_linear(x, w).sum().backward()
    D, X, W = torch.ones(140, 96, dtype=torch.float64, device="cuda"), values64(ops.pack_fp8(x)), values64(ops.pack_fp8(w))
    near(x.grad, D @ W, D @ W.abs(), 96)
    near(w.grad, D.t() @ X, D.t() @ X.abs(), 140)


def test_empty_batches():
    w = weights(48, 96).cuda().requires_grad_()
    x = torch.empty(2, 0, 96, dtype=BF, device="cuda", requires_grad=True)
    y = ops.fp8_linear(x, w)
    y.sum().backward()
    assert y.shape == (2, 0, 48) and y.dtype == BF and x.grad.shape == x.shape and not w.grad.any()
    wk, wv = ops.pack_fp8(weights(64, 96).cuda()), ops.pack_fp8(weights(96, 64).cuda())
    assert ops.fp8_channel_mix_ffn(x.detach(), wk, wv, x.detach()).shape == x.shape


def test_refusals_on_cuda():
    x, w = torch.ones(4, 64, device="cuda"), torch.ones(8, 64, device="cuda")
    with pytest.raises(TypeError):
        ops.fp8_linear(x, w)
    with pytest.raises(TypeError):
        ops.fp8_linear(x.to(BF), w)
    with pytest.raises(ValueError):
        ops.fp8_linear(x.to(BF), w.to(BF).cpu())
    with pytest.raises(ValueError):
        ops.fp8_linear(x.to(BF), ops.pack_fp8(w.cpu()))
    with pytest.raises(TypeError):
        ops.pack_fp8(x.double())


@pytest.mark.parametrize("M", [1, 9, 40])
def test_weights_packed_in_and_before_a_chain_of_decode_launches(M):
    """Fresh weights every time, without a wait between packing and product: the first launch of a chain, and the one after a
    packing launch inside it, wait for everything before them."""
    from rwkvtune_b200.ops import _ext

    x, res = sample(M, 512).cuda(), sample(M, 512, seed=3).cuda()
    hold = ops.pack_fp8(weights(1024, 512).cuda()), ops.pack_fp8(weights(512, 1024).cuda())
    fresh = [(weights(1024, 512, s).cuda(), weights(512, 1024, s + 50).cuda()) for s in range(8)]
    want = [ops.fp8_channel_mix_ffn(x, ops.pack_fp8(k), ops.pack_fp8(v), res) for k, v in fresh]
    torch.cuda.synchronize()
    with torch.no_grad():
        got = []
        for k, v in fresh:
            ops.pack_fp8(k, out=hold[0]), ops.pack_fp8(v, out=hold[1])
            with _ext.launch_chaining():
                got.append(ops.fp8_channel_mix_ffn(x, *hold, res))
        with _ext.launch_chaining():
            for k, v in fresh:
                ops.pack_fp8(k, out=hold[0]), ops.pack_fp8(v, out=hold[1])
                got.append(ops.fp8_channel_mix_ffn(x, *hold, res))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want + want))


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_pack_and_unpack_next_to_the_smallest_normal_numbers(dtype, rows):
    """Blocks whose values lie around 2^-126: the CPU statement, bit for bit, signs of zeros included."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(140, 400, generator=g) * torch.exp2(torch.randint(-12, 12, (140, 400), generator=g).float())
    x = (x * 2.0 ** -100 * 2.0 ** -27).to(dtype)
    x[128:, 128:256] = (torch.randn(12, 128, generator=g) * 2.0 ** -100 * 2.0 ** -30).clamp(-2.0 ** -127, 2.0 ** -127).to(dtype)
    p = ops.pack_fp8(x.cuda(), rows=rows)
    same_bits(p, x, rows)
    for out in (BF, torch.float32):
        got, want = ops.unpack_fp8(p, out).cpu(), ops.unpack_fp8(p.to("cpu"), out)
        assert torch.equal(got, want) and torch.equal(torch.signbit(got), torch.signbit(want))
