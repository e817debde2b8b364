"""The 8-bit operators inside the model, the engine and the trainers' settings, on the CPU."""
import copy

import pytest
import torch

from rwkvtune_b200 import ops
from rwkvtune_b200.engine.engine import EngineConfig, TrainEngine
from rwkvtune_b200.models import RWKV7Model, RWKVConfig
from rwkvtune_b200.parallel.bootstrap import DistContext
from rwkvtune_b200.peft import LoraConfig, get_peft_model
from rwkvtune_b200.training.grpo_config import GRPOConfig
from rwkvtune_b200.training.sft_config import SFTConfig


def make(**kw):
    torch.manual_seed(0)
    m = RWKV7Model(RWKVConfig(n_layer=2, n_embd=64, vocab_size=128, dim_att_lora=16, dim_gate_lora=16, dim_mv_lora=16))
    with torch.no_grad():
        for b in m.blocks:      # the value projection starts at zero, which would hide it
            b.ffn.value.weight.normal_(0, 0.05)
            b.att.output.weight.normal_(0, 0.05)
    for k, v in kw.items():
        setattr(m.config, k, v)
    return m


def batch(B=3, T=40):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 128, (B, T), generator=g)
    return ids, torch.randint(0, 128, (B, T), generator=g)


def grads(m, ids, labels):
    m.train()
    loss = m.loss(ids, labels)
    loss.backward()
    return loss.item(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


def test_the_ffn_of_a_model_in_8_bits_is_the_operator():
    m, ids = make(ffn_precision="fp8"), batch()[0]
    calls = []
    real = ops.fp8_channel_mix_ffn
    try:
        ops.fp8_channel_mix_ffn = lambda *a: calls.append(a) or real(*a)
        m(ids)
    finally:
        ops.fp8_channel_mix_ffn = real
    assert len(calls) == 2 and calls[0][1] is m.blocks[0].ffn.key.weight
    # the packed operands move every product's terms by at most (1 + 2^-4)^2 - 1: the result is another one, but near
    a, b = make()(ids), m(ids)
    assert not torch.equal(a, b) and (a - b).norm() < ((1 + 2 ** -4) ** 2 - 1) * 2 * a.norm()


def test_a_recomputed_block_sees_the_packed_input():
    """With inputs that packing leaves as they are, 8-bit checkpoints change nothing; with others the gradients are those of
    the block at the packed input."""
    m = make(grad_cp=1, grad_cp_bits=8)
    block = m.blocks[0].train()
    from rwkvtune_b200.models.rwkv7.model import _block_plain, _checkpoint_block

    x = torch.randn(2, 16, 64)
    v = torch.zeros_like(x)
    exact = ops.unpack_fp8(ops.pack_fp8(x, rows=1))
    out = {}
    for name, inp in (("packed", exact), ("given", x)):
        a = inp.clone().requires_grad_()
        y, _ = _checkpoint_block(_block_plain, block, a, v)
        dy = torch.ones_like(y)
        (out[name],) = torch.autograd.grad(y, [a], dy)
    a = exact.clone().requires_grad_()
    y, _ = _block_plain(block, a, v)
    (want,) = torch.autograd.grad(y, [a], torch.ones_like(y))
    assert torch.equal(out["packed"], want) and torch.equal(out["given"], want)


def test_checkpoints_in_8_bits_keep_the_loss_and_the_last_block():
    ids, labels = batch()
    l16, g16 = grads(make(grad_cp=1), ids, labels)
    l8, g8 = grads(make(grad_cp=1, grad_cp_bits=8), ids, labels)
    assert l8 == l16 and set(g8) == set(g16)                  # the forward pass is not rounded
    assert torch.equal(g8["head.weight"], g16["head.weight"]) and torch.equal(g8["ln_out.weight"], g16["ln_out.weight"])
    k = "blocks.0.ffn.key.weight"
    assert not torch.equal(g8[k], g16[k]) and torch.isfinite(g8[k]).all()


def test_infinite_context_chunks_with_8_bit_checkpoints():
    from rwkvtune_b200.models.rwkv7.model_infctx import as_infctx

    ids, labels = batch(2, 32)
    got = {}
    for bits in (16, 8):
        m = as_infctx(make(grad_cp=1, grad_cp_bits=bits, ffn_precision="fp8")).train()
        L, H = 2, 1
        shift, wkv = torch.zeros(L, 2, 2, 64), torch.zeros(L, 2, H, 64, 64)
        x, shift, wkv = m.forward_hidden_infctx(ids, shift, wkv, checkpoint=True)
        (x.square().mean() + wkv.square().mean()).backward()
        got[bits] = m.blocks[0].ffn.value.weight.grad
    assert got[8].abs().sum() > 0 and torch.isfinite(got[8]).all()


def test_dropout_and_8_bit_checkpoints_are_refused():
    m = get_peft_model(make(), LoraConfig(r=4, lora_alpha=8, lora_dropout=0.5))
    m.config.grad_cp, m.config.grad_cp_bits = 1, 8
    m.train()
    with pytest.raises(RuntimeError, match="dropout"):
        m.loss(*batch())


def test_packed_weights_serve_passes_without_autograd():
    m, ids = make().eval(), batch()[0]
    with torch.no_grad():
        plain = m(ids)
        m.pack_ffn()
        y = m(ids)
        state_y, st = m.forward_with_state(ids[:, :30])
        more, _ = m.forward_with_state(ids[:, 30:], st)
    ffn = m.blocks[0].ffn
    x = torch.randn(1, 5, 64)
    with torch.no_grad():
        got, _ = ffn(x, torch.ones(64), torch.zeros(64))
        (xk,), _, _ = ops.ln_shift_mix_unbound(x, torch.ones(64), torch.zeros(64), ffn.x_k, None)
        assert torch.equal(got, ops.fp8_channel_mix_ffn(xk, ops.pack_fp8(ffn.key.weight), ops.pack_fp8(ffn.value.weight), x))
    assert not torch.equal(y, plain)
    # blocks of one row: cutting the sequence in two leaves the packed operands as they are (the recurrence sums differently)
    torch.testing.assert_close(torch.cat([state_y, more], 1), y, rtol=1e-3, atol=1e-3)
    m.unpack_ffn()
    with torch.no_grad():
        assert torch.equal(m(ids), plain)


def test_stale_packed_weights_are_refused():
    m, ids = make().eval().pack_ffn(), batch()[0]
    with torch.no_grad():
        m.blocks[1].ffn.key.weight.add_(1.0)
        with pytest.raises(RuntimeError, match="pack_ffn"):
            m(ids)
        m.pack_ffn()
        m(ids)
        ops.bump_param_epoch()                     # the optimiser kernels write without a version count
        with pytest.raises(RuntimeError, match="pack_ffn"):
            m(ids)
    m.train().loss(*batch()).backward()            # training uses the weights themselves
    m.eval().pack_ffn()
    kept = m.blocks[0].ffn._packed[1][0].address
    m.pack_ffn()
    assert m.blocks[0].ffn._packed[1][0].address == kept
    m.blocks[0].ffn.key.weight = torch.nn.Parameter(m.blocks[0].ffn.key.weight.detach().clone())
    with torch.no_grad(), pytest.raises(RuntimeError, match="pack_ffn"):
        m(ids)


def test_copies_and_pickles_of_a_packed_model():
    import pickle

    m, ids = make().eval(), batch()[0]
    with torch.no_grad():
        plain, packed = m(ids), m.pack_ffn()(ids)
        for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
            assert torch.equal(other(ids), plain) and torch.equal(other.pack_ffn()(ids), packed)
        assert torch.equal(m(ids), packed)


def test_packing_wrapped_projections_is_refused():
    m = get_peft_model(make(), LoraConfig(r=4, lora_alpha=8))
    if any(not b.ffn._plain() for b in m.blocks):
        with pytest.raises(ValueError):
            m.pack_ffn()


def test_engine_trains_with_both():
    ids, labels = batch()
    eng = TrainEngine(make(), EngineConfig(lr_init=1e-3, precision="fp32", grad_cp=1, ffn_precision="fp8", grad_cp_bits=8),
                      DistContext())
    before = copy.deepcopy(eng.model.state_dict())
    out = eng.train_step(ids, labels, 1e-3) if hasattr(eng, "train_step") else None
    after = eng.model.state_dict()
    assert eng.model.config.ffn_precision == "fp8" and eng.model.config.grad_cp_bits == 8
    if out is not None:
        assert any(not torch.equal(before[k], after[k]) for k in before)


@pytest.mark.parametrize("config", [SFTConfig, GRPOConfig, EngineConfig])
def test_settings(config):
    c = config(ffn_precision="fp8", grad_cp_bits=8)
    assert (c.ffn_precision, c.grad_cp_bits) == ("fp8", 8)
    assert (config().ffn_precision, config().grad_cp_bits) == ("bf16", 16)


def test_settings_refusals():
    for kw in ({"ffn_precision": "int8"}, {"grad_cp_bits": 4}):
        with pytest.raises(ValueError):
            SFTConfig(**kw)
        with pytest.raises(ValueError):
            GRPOConfig(**kw)
        with pytest.raises(ValueError):
            TrainEngine(make(), EngineConfig(precision="fp32", **kw), DistContext())
    m = get_peft_model(make(), LoraConfig(r=4, lora_alpha=8, target_modules=["key", "value"]))
    with pytest.raises(ValueError):
        TrainEngine(m, EngineConfig(precision="fp32", ffn_precision="fp8"), DistContext())
    with pytest.raises(ValueError):
        TrainEngine(make(), EngineConfig(precision="fp32", ffn_precision="fp8", strategy="deepspeed_stage_3"), DistContext())


def test_pipeline_switch():
    from rwkvtune_b200.inference.pipeline import InferencePipeline

    pipe = InferencePipeline(model=make(), device="cpu", tokenizer=object(), ffn_8bit=True)
    assert all(b.ffn._packed is not None for b in pipe.model.blocks)


@pytest.mark.parametrize("precision", ["bf16", "fp8"])
def test_training_a_packed_model_with_recomputed_blocks(precision):
    """The first run of a recomputed block has no autograd either, but it belongs to a training pass: it takes the weights
    that the second run takes, not their packed copy."""
    ids, labels = batch()
    want = grads(make(grad_cp=1, ffn_precision=precision), ids, labels)
    got = grads(make(grad_cp=1, ffn_precision=precision).pack_ffn(), ids, labels)
    once = grads(make(ffn_precision=precision).pack_ffn(), ids, labels)
    for loss, gr in (got, once):
        assert loss == want[0] and set(gr) == set(want[1]) and all(torch.equal(gr[n], want[1][n]) for n in gr)


def test_checkpointed_passes_without_autograd_keep_nothing():
    m, ids = make(grad_cp=1, grad_cp_bits=8).train(), batch()[0]
    from rwkvtune_b200.models.rwkv7.model import _block_plain, _checkpoint_block

    real, calls = ops.pack_fp8, []
    x = torch.randn(1, 9, 64)
    try:
        ops.pack_fp8 = lambda *a, **k: calls.append(a) or real(*a, **k)
        with torch.no_grad():
            y, _ = _checkpoint_block(_block_plain, m.blocks[0], x, torch.zeros_like(x))
    finally:
        ops.pack_fp8 = real
    with torch.no_grad():
        assert not calls and torch.equal(y, _block_plain(m.blocks[0], x, torch.zeros_like(x))[0])
        packed = m.eval().pack_ffn()(ids)                 # the flag of the first run does not outlive it
        assert not torch.equal(packed, m.unpack_ffn()(ids))


def test_state_carrying_passes_without_autograd_keep_the_weights_precision():
    """Prefill and decoding of a model that trains in 8 bits: the products of the 16-bit model, whatever the length; whole
    sequences without a state run as in training."""
    from rwkvtune_b200.inference import GRPOBatchGenerator

    m, n, ids = make(ffn_precision="fp8").eval(), make().eval(), batch()[0]
    with torch.no_grad():
        states = [None, None]
        for part in (ids[:, :30], ids[:, 30:31], ids[:, 31:32]):
            (a, states[0]), (b, states[1]) = m.forward_with_state(part, states[0]), n.forward_with_state(part, states[1])
            assert torch.equal(a, b)
        assert not torch.equal(m(ids), n(ids))
        rows = torch.randn(1, 40, 64)
        (y,), (z,) = (model.blocks[0].ffn(rows, torch.ones(64), torch.zeros(64))[:1] for model in (m.train(), m.eval()))
        assert torch.equal(y, z)
    args = dict(input_ids=[[5, 6, 7]] * 3, max_new_tokens=6, num_generations=50, temperature=1.0, top_p=1.0, seed=3)
    a, b = (GRPOBatchGenerator(x, None, torch.device("cpu"), eos_token_id=0).generate(**args)["completion_ids"] for x in (m, n))
    assert torch.equal(a, b)
    # with a state and autograd (training in chunks) the 8-bit products run
    x = torch.randn(1, 5, 64, requires_grad=True)
    outs = [model.blocks[0].ffn(x, torch.ones(64), torch.zeros(64), torch.zeros(1, 64), True)[0] for model in (m, n)]
    assert not torch.equal(*outs)


def test_adapters_and_shards_that_come_after_packing():
    """A packed copy knows nothing of an adapter wrapped around the projections later, nor of panels: it is refused."""
    m, ids = make().eval().pack_ffn(), batch()[0]
    m = get_peft_model(m, LoraConfig(r=4, lora_alpha=8, target_modules=["ffn.key", "ffn.value"])).eval()
    assert not m.blocks[0].ffn._plain()
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="unpack_ffn"):
            m(ids)
        for b in m.blocks:
            b.ffn.unpack()
        m(ids)
        n = make().eval().pack_ffn()
        n.blocks[0].ffn.key._sharded = object()
        with pytest.raises(RuntimeError, match="unpack_ffn"):
            n(ids)


def test_weights_replaced_or_moved_after_packing():
    """``weight.data = other`` (what moving and casting a model do as well) counts no version."""
    for change in (lambda m: setattr(m.blocks[1].ffn.value.weight, "data", m.blocks[1].ffn.value.weight.data * 2),
                   lambda m: m.to(torch.bfloat16)):
        m, ids = make().eval().pack_ffn(), batch()[0]
        with torch.no_grad():
            m(ids)
            change(m)
            with pytest.raises(RuntimeError, match="pack_ffn"):
                m(ids)
            m.pack_ffn()
            m(ids)


def test_another_models_optimiser_leaves_a_packed_copy_valid():
    """The engine's own model is refused after a step and after loading a state; a packed model beside it is not."""
    ids, labels = batch()
    beside = [make().eval().pack_ffn(), make().eval().requires_grad_(False).pack_ffn()]
    eng = TrainEngine(make(), EngineConfig(lr_init=1e-3, precision="fp32"), DistContext())
    own = eng.model.pack_ffn()
    with torch.no_grad():
        want = [m(ids) for m in beside]
        own(ids)
    eng.train_step(ids, labels, 1e-3)
    with torch.no_grad():
        assert all(torch.equal(m(ids), w) for m, w in zip(beside, want))
        with pytest.raises(RuntimeError, match="pack_ffn"):
            own(ids)
        own.pack_ffn()(ids)
        full = [torch.ones(eng.space.numel) for _ in range(3)]
        eng.opt.load_full_state(*full, step=3)
        with pytest.raises(RuntimeError, match="pack_ffn"):
            own(ids)
        assert torch.equal(beside[0](ids), want[0])
        copied = copy.deepcopy(own).pack_ffn()                 # a copy belongs to no optimiser
        kept = copied(ids)
    eng.train_step(ids, labels, 1e-3)
    with torch.no_grad():
        assert torch.equal(copied(ids), kept)


def test_captured_steps_belong_to_the_packed_buffers(monkeypatch):
    """A generator's captured step is taken again only while the model reads the same packed memory, and keeps that memory."""
    from rwkvtune_b200.inference import grpo_batch_generator as module

    class Step:
        def __init__(self, gen, n):
            self.packed = gen._packed_buffers()

    monkeypatch.setattr(module, "_DecodeGraph", Step)
    m = make().eval()
    gen = module.GRPOBatchGenerator(m, None, torch.device("cpu"), eos_token_id=0)
    gen._graph_for(2)
    plain = gen._graph_for(4)
    assert gen._graph_for(4) is plain and plain.packed == ()
    packed = m.pack_ffn() and gen._graph_for(4)
    assert packed is not plain and len(packed.packed) == 4 and list(gen._graphs) == [4]
    m.pack_ffn()                                       # written again in place
    assert gen._graph_for(4) is packed
    m.blocks[1].ffn.unpack()
    partly = gen._graph_for(4)
    assert partly is not packed and len(partly.packed) == 2 and packed.packed[2].numel() > 0
    m.unpack_ffn()
    assert gen._graph_for(4).packed == ()
    m.pack_ffn()                                       # other memory than the first time
    assert gen._graph_for(4) is not packed
