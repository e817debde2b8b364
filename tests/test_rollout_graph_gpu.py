"""Captured decode steps of the rollout generator follow the model: its parameters after an optimiser step, and its packed
feed-forward weights."""
import pytest
import torch

from rwkvtune_b200.engine.engine import EngineConfig, TrainEngine
from rwkvtune_b200.inference import GRPOBatchGenerator
from rwkvtune_b200.models import RWKV7Model, RWKVConfig
from rwkvtune_b200.ops import gemm_native
from rwkvtune_b200.parallel.bootstrap import DistContext

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def make():
    torch.manual_seed(0)
    m = RWKV7Model(RWKVConfig(n_layer=2, n_embd=256, vocab_size=1024, dim_att_lora=32, dim_gate_lora=64, dim_mv_lora=32, ctx_len=512))
    with torch.no_grad():
        for b in m.blocks:
            b.ffn.value.weight.normal_(0, 0.02)
            b.att.output.weight.normal_(0, 0.02)
    return m.cuda().to(torch.bfloat16)


def tokens(gen):
    out = gen.generate(input_ids=[[5, 6, 7, 8], [9, 10, 11]], max_new_tokens=12, num_generations=3, temperature=1.0, top_p=1.0, seed=3)
    return out["completion_ids"].cpu()


def generators(m):
    return [GRPOBatchGenerator(m, None, DEV, eos_token_id=0, use_cuda_graph=g) for g in (True, False)]


def test_captured_steps_follow_the_optimiser():
    """The same generator before and after training steps: every parameter moves, the token-shift coefficients among them."""
    eng = TrainEngine(make(), EngineConfig(lr_init=1e-2, precision="bf16"), DistContext(device=DEV))
    captured, eager = generators(eng.model)
    ids = torch.randint(0, 1024, (2, 64), device=DEV)
    seen = []
    for _ in range(3):
        a, b = tokens(captured), tokens(eager)
        assert torch.equal(a, b)
        seen.append(a)
        with torch.no_grad():
            before = eng.model.blocks[1].att.mix_matrix().clone()
        for _ in range(3):
            eng.train_step(ids, ids, 1e-2)
        with torch.no_grad():
            assert not torch.equal(before, eng.model.blocks[1].att.mix_matrix())
    assert not torch.equal(seen[0], seen[1])
    torch.cuda.synchronize()
    assert gemm_native.check_status() == 0


def test_captured_steps_follow_packing_and_unpacking():
    m = make().eval()
    captured, eager = generators(m)
    seen = []
    for change in (lambda: None, m.pack_ffn, m.pack_ffn, m.unpack_ffn, m.pack_ffn):
        change()
        torch.cuda.empty_cache()
        a, b = tokens(captured), tokens(eager)
        assert torch.equal(a, b)
        seen.append(a)
    assert torch.equal(seen[0], seen[3]) and torch.equal(seen[1], seen[2]) and torch.equal(seen[1], seen[4])
    torch.cuda.synchronize()
    assert gemm_native.check_status() == 0
