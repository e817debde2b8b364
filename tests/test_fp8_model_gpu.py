"""The 8-bit operators as the model, the engine and the rollout generator use them on a GPU."""
import pytest
import torch

from rwkvtune_b200.engine.engine import EngineConfig, TrainEngine
from rwkvtune_b200.models import RWKV7Model, RWKVConfig
from rwkvtune_b200.ops import _ext, gemm_native
from rwkvtune_b200.parallel.bootstrap import DistContext

pytestmark = pytest.mark.gpu


def make(**kw):
    torch.manual_seed(0)
    m = RWKV7Model(RWKVConfig(n_layer=2, n_embd=256, vocab_size=1024, dim_att_lora=32, dim_gate_lora=64, dim_mv_lora=32, ctx_len=512))
    with torch.no_grad():
        for b in m.blocks:
            b.ffn.value.weight.normal_(0, 0.02)
            b.att.output.weight.normal_(0, 0.02)
    for k, v in kw.items():
        setattr(m.config, k, v)
    return m.cuda().to(torch.bfloat16)


def batch(B=2, T=272):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 1024, (B, T), generator=g).cuda() for _ in range(2)]


def run(m, **kw):
    """Loss and gradients of one model under the given settings."""
    for k, v in {"ffn_precision": "bf16", "grad_cp": 0, "grad_cp_bits": 16, **kw}.items():
        setattr(m.config, k, v)
    m.train().zero_grad(set_to_none=True)
    loss = m.loss(*batch())
    loss.backward()
    return loss.item(), {n: p.grad.float() for n, p in m.named_parameters()}


def test_training_pass_runs_the_8_bit_kernels_and_stays_near():
    """The packed operands move each feed-forward product's terms by at most 2^-4 each; a gradient's direction stays."""
    m = make()
    l16, g16 = run(m)
    before = _ext.launch_count()
    l8, g8 = run(m, ffn_precision="fp8")
    assert _ext.launch_count() > before and abs(l8 - l16) < 2 ** -4 * abs(l16)
    for name in ("blocks.0.ffn.key.weight", "blocks.1.ffn.value.weight", "emb.weight", "blocks.0.att.key.weight"):
        a, b = g8[name].flatten(), g16[name].flatten()
        assert torch.isfinite(a).all() and torch.dot(a, b) > 0.9 * a.norm() * b.norm(), name
    torch.cuda.synchronize()
    assert gemm_native.check_status() == 0


def test_checkpoints_in_8_bits():
    m = make()
    l16, g16 = run(m, grad_cp=1)
    l8, g8 = run(m, grad_cp=1, grad_cp_bits=8)
    assert l8 == l16 and torch.equal(g8["head.weight"], g16["head.weight"])
    for name in g16:
        a, b = g8[name].flatten(), g16[name].flatten()
        if b.norm() > 0:
            assert torch.isfinite(a).all() and torch.dot(a, b) > 0.9 * a.norm() * b.norm(), name


def test_a_checkpoint_takes_half_the_memory():
    from rwkvtune_b200.models.rwkv7.model import _checkpoint_block

    class Id(torch.nn.Module):
        def __init__(self, bits):
            super().__init__()
            self.config = type("C", (), {"grad_cp_bits": bits})()

    kept = {}
    for bits in (16, 8):
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        x = torch.randn(4096, 1024, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        (y,) = _checkpoint_block(lambda b, t: (t * 2,), Id(bits), x * 1.0)
        kept[bits] = torch.cuda.memory_allocated() - start
        del x, y
    assert kept[16] - kept[8] > 0.45 * 4096 * 1024 * 2


@pytest.mark.parametrize("graph", [False, True])
def test_engine_steps_with_both(graph):
    eng = TrainEngine(make(), EngineConfig(lr_init=1e-3, precision="bf16", grad_cp=1, ffn_precision="fp8", grad_cp_bits=8,
                                           cuda_graph=graph), DistContext(device=torch.device("cuda", 0)))
    ids, labels = batch()
    losses = [float(eng.train_step(ids, labels, 1e-3)) for _ in range(4)]
    assert all(v == v for v in losses) and len(set(losses)) > 1
    torch.cuda.synchronize()
    assert gemm_native.check_status() == 0


def test_captured_steps_repeat_the_eager_ones():
    got = []
    for graph in (False, True):
        eng = TrainEngine(make(), EngineConfig(lr_init=1e-3, precision="bf16", ffn_precision="fp8", cuda_graph=graph),
                          DistContext(device=torch.device("cuda", 0)))
        ids, labels = batch()
        got.append([float(eng.train_step(ids, labels, 1e-3)) for _ in range(3)])
    assert got[0] == got[1]


def test_packed_decode_steps():
    """Prefill and decoding on packed weights, eager and from the rollout generator's captured step."""
    from rwkvtune_b200.inference import GRPOBatchGenerator

    m = make().eval().pack_ffn()
    prompts = [[5, 6, 7, 8], [9, 10, 11], [12] * 6]
    outs = []
    for use_graph in (False, True):
        gen = GRPOBatchGenerator(m, None, torch.device("cuda", 0), eos_token_id=0, use_cuda_graph=use_graph)
        out = gen.generate(input_ids=prompts, max_new_tokens=12, num_generations=2, temperature=1.0, top_p=1.0, seed=3)
        outs.append(out["completion_ids"].cpu())
    assert torch.equal(outs[0], outs[1])
    torch.cuda.synchronize()
    assert gemm_native.check_status() == 0


def test_a_captured_step_follows_weights_that_are_packed_again():
    from rwkvtune_b200.inference import GRPOBatchGenerator

    m = make().eval().pack_ffn()
    gen = GRPOBatchGenerator(m, None, torch.device("cuda", 0), eos_token_id=0, use_cuda_graph=True)
    args = dict(input_ids=[[5, 6, 7, 8]] * 2, max_new_tokens=10, num_generations=1, temperature=1.0, top_p=1.0, seed=3)
    first = gen.generate(**args)["completion_ids"].cpu()
    with torch.no_grad():
        for b in m.blocks:
            b.ffn.value.weight.mul_(-3.0)
    m.pack_ffn()
    again = gen.generate(**args)["completion_ids"].cpu()
    eager = GRPOBatchGenerator(m, None, torch.device("cuda", 0), eos_token_id=0, use_cuda_graph=False).generate(**args)
    assert torch.equal(again, eager["completion_ids"].cpu()) and not torch.equal(first, again)


def test_packed_and_plain_logits_are_near():
    m, (ids, _) = make().eval(), batch()
    with torch.no_grad():
        plain = m(ids).float()
        packed = m.pack_ffn()(ids).float()
    assert (packed - plain).norm() < ((1 + 2 ** -4) ** 2 - 1) * 2 * plain.norm() and not torch.equal(packed, plain)


def ffn_calls(monkeypatch):
    """The calls of the 8-bit feed-forward half from here on: True for each one that gets packed weights."""
    from rwkvtune_b200 import ops

    calls, real = [], ops.fp8_channel_mix_ffn
    monkeypatch.setattr(ops, "fp8_channel_mix_ffn", lambda *a: calls.append(type(a[1]) is ops.Fp8Blocks) or real(*a))
    return calls


@pytest.mark.parametrize("packed", [False, True])
def test_short_recomputed_batches_run_one_function(monkeypatch, packed):
    """At most 128 tokens, where a pass without autograd would decode: both runs of a recomputed block take the same products."""
    m = make(ffn_precision="fp8", grad_cp=1).train()
    if packed:
        m.pack_ffn()
    calls = ffn_calls(monkeypatch)
    ids, labels = (t[:, :40] for t in batch())
    m.loss(ids, labels).backward()
    assert calls == [False] * 4                # two blocks, each run twice, on the trainable weights


@pytest.mark.parametrize("paths", [64, 160])
def test_rollouts_of_a_model_that_trains_in_8_bits(monkeypatch, paths):
    """More sequences than the decode products take, and fewer: neither prefill nor decoding packs a weight, and the tokens
    are those of the 16-bit model."""
    from rwkvtune_b200.inference import GRPOBatchGenerator

    m, outs = make(ffn_precision="fp8").eval(), []
    calls = ffn_calls(monkeypatch)
    for precision in ("fp8", "bf16"):
        m.config.ffn_precision = precision
        gen = GRPOBatchGenerator(m, None, torch.device("cuda", 0), eos_token_id=0, use_cuda_graph=False)
        outs.append(gen.generate(input_ids=[list(range(1, 150)), [5, 6, 7]], max_new_tokens=4, num_generations=paths // 2, temperature=1.0,
                                 top_p=1.0, seed=3)["completion_ids"].cpu())
    assert not calls and torch.equal(*outs)


def test_moving_a_packed_model_names_the_packing():
    m, (ids, _) = make().cpu().eval().pack_ffn(), batch()
    m.cuda()
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="pack_ffn"):
            m(ids)
        m.pack_ffn()(ids)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_packing_other_types_is_refused_at_once(dtype):
    from rwkvtune_b200.inference.pipeline import InferencePipeline

    m = make().to(dtype)
    with pytest.raises(ValueError, match="bfloat16"):
        m.pack_ffn()
    with pytest.raises(ValueError, match="bfloat16"):
        InferencePipeline(model=m, device="cuda", tokenizer=object(), ffn_8bit=True)


# ------------------------------------------------------------------------------- which kernels run
FORWARD = ["pack"] * 3 + ["relu_sq", "residual"]
BACKWARD = ["pack", "relu_sq_grad", "nn", "tn", "tn"]


def launched(monkeypatch):
    """Names of the 8-bit launches from here on, read from the records that go to the library."""
    import struct

    from rwkvtune_b200.ops import fp8_native

    names, real = [], fp8_native.run

    def name(record):
        kind, _, _, _, a_rows, q_rows, _, a_mn, b_mn, epilogue = struct.unpack("=10i", record[:40])
        if kind == 0:
            return "pack" if q_rows == 128 else "pack rows"
        if kind == 1:
            return "unpack rows" if a_rows == 1 else "unpack"
        product = ["tn" if a_mn else "nn" if b_mn else "nt", "residual", "relu_sq", "relu_sq_grad"][epilogue]
        return product if kind == 2 else "decode " + product

    monkeypatch.setattr(fp8_native, "run", lambda device, steps: names.extend(map(name, steps)) or real(device, steps))
    return names


def test_training_pass_launches_exactly_the_8_bit_products(monkeypatch):
    m, names = make(), launched(monkeypatch)
    l16, g16 = run(m)
    assert names == []
    l8, g8 = run(m, ffn_precision="fp8")
    assert sorted(names) == sorted(2 * (FORWARD + BACKWARD)) and names[:10] == 2 * FORWARD
    assert l8 != l16
    for i in (0, 1):
        for half in ("key", "value"):
            n = f"blocks.{i}.ffn.{half}.weight"
            assert not torch.equal(g8[n], g16[n])
    del names[:]
    run(m, ffn_precision="fp8", grad_cp=1, grad_cp_bits=8)      # each block's forward pass twice, its input packed in between
    assert sorted(names) == sorted(2 * (["pack rows"] + FORWARD + ["unpack rows"] + FORWARD + BACKWARD))
    del names[:]
    run(m, grad_cp=1, grad_cp_bits=8)
    assert sorted(names) == sorted(2 * ["pack rows", "unpack rows"])


def test_gradients_of_a_block_inside_the_model(monkeypatch):
    """What the feed-forward weights of a training step receive, against 64-bit products of the operands that the block saw."""
    from rwkvtune_b200 import ops
    from test_fp8_gpu import near, packed_product, values64

    m, seen, real = make(ffn_precision="fp8").train(), [], ops.fp8_channel_mix_ffn

    def recorded(xk, wk, wv, res):
        y = real(xk, wk, wv, res)
        entry = {"x": xk.detach().clone(), "res": res.detach().clone(), "y": y.detach().clone()}
        y.register_hook(lambda g: entry.__setitem__("dy", g.clone()))
        seen.append(entry)
        return y

    monkeypatch.setattr(ops, "fp8_channel_mix_ffn", recorded)
    m.loss(*batch()).backward()
    assert len(seen) == 2
    for block, s in zip(m.blocks, seen):
        wk, wv = block.ffn.key.weight, block.ffn.value.weight
        x, res, y, dy = (s[k].reshape(-1, s[k].shape[-1]) for k in ("x", "res", "y", "dy"))
        x8, k8, v8, d8 = (ops.pack_fp8(t.detach()) for t in (x, wk, wv, dy))
        M, H = x.shape[0], wk.shape[0]
        h8 = packed_product("nt_relu_sq", x8, k8, M, H, 128)
        p8 = packed_product("nn_relu_sq_grad", d8, v8, M, H, 128, h8)
        X, V, D, Hd, P = (values64(t) for t in (x8, v8, d8, h8, p8))
        near(y, res.double() + Hd @ V.t(), Hd.abs() @ V.abs().t() + res.double().abs(), H)
        near(wk.grad, P.t() @ X, P.abs().t() @ X.abs(), M)
        near(wv.grad, D.t() @ Hd, D.abs().t() @ Hd.abs(), M)


@pytest.mark.parametrize("graph", [False, True])
def test_engine_steps_launch_the_8_bit_products(monkeypatch, graph):
    """Per step, eager or recorded into a graph: the launches of two recomputed blocks; and losses that are not bf16's."""
    names, losses = launched(monkeypatch), {}
    for precision in ("bf16", "fp8"):
        eng = TrainEngine(make(), EngineConfig(lr_init=1e-3, precision="bf16", grad_cp=1, ffn_precision=precision, cuda_graph=graph),
                          DistContext(device=torch.device("cuda", 0)))
        ids, labels = batch()
        losses[precision] = [float(eng.train_step(ids, labels, 1e-3)) for _ in range(4)]
        # a graph is recorded in the third step and replayed in the third and the fourth
        passes = (0 if precision == "bf16" else eng.GRAPH_WARMUP_STEPS + 1 if graph else 4)
        assert sorted(names) == sorted(passes * 2 * (2 * FORWARD + BACKWARD))
        del names[:]
    assert all(a != b for a, b in zip(losses["bf16"], losses["fp8"]))


def test_packed_decode_steps_launch_the_decode_products(monkeypatch):
    from rwkvtune_b200.inference import GRPOBatchGenerator

    m = make().eval().pack_ffn()
    names = launched(monkeypatch)
    gen = GRPOBatchGenerator(m, None, torch.device("cuda", 0), eos_token_id=0, use_cuda_graph=False)
    gen.eos_ids = []
    gen.generate(input_ids=[list(range(1, 150))], max_new_tokens=3, num_generations=12, temperature=1.0, top_p=1.0, seed=3)
    # 149 prompt tokens of one sequence, then two or three steps of twelve rows
    assert names[:6] == 2 * ["pack rows", "relu_sq", "residual"]
    assert len(names) > 6 and names[6:] == len(names[6:]) // 2 * ["decode relu_sq", "decode residual"]


# ------------------------------------------------------------------------------- a token and its batch
def test_what_a_tokens_result_depends_on():
    """The 8-bit form of a token is its own; its sums are those of a dispatch form: at most 128 rows, more of them, and among
    those each number of slices of the contraction.  Within a form a row's bits stay, between forms they agree to the last
    places of an fp32 sum."""
    from rwkvtune_b200 import ops
    from rwkvtune_b200.ops import fp8_native
    from test_fp8_gpu import near, sample, values64, weights

    N, K = 1024, 8192
    w8, x = ops.pack_fp8(weights(N, K).cuda()), sample(1300, K).cuda()
    rows = (20, 128, 256, 300, 600, 1300)
    slices = {m: fp8_native._workspace_bytes(m, N, K) // (-(-m // 128) * 128 * N * 4) for m in rows[2:]}
    assert slices[256] == slices[300] and len(set(slices.values())) > 1
    full = ops.pack_fp8(x, rows=1)
    W, X = values64(w8), values64(full)
    out = {}
    for m in rows:
        p = ops.pack_fp8(x[:m], rows=1)
        assert torch.equal(p.values.view(torch.uint8), full.values[:m].view(torch.uint8)) and torch.equal(p.exponents, full.exponents[:m])
        out[m] = ops.fp8_linear(x[:m], w8)
        near(out[m], X[:m] @ W.t(), X[:m].abs() @ W.abs().t(), K)
    assert torch.equal(out[20], out[128][:20]) and torch.equal(out[256], out[300][:256])
