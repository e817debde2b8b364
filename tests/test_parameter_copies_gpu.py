"""The cached fp32 copies of small parameters belong to the parameter, not to its address."""
import pytest
import torch

from rwkvtune_b200.ops import cuda_ops

pytestmark = pytest.mark.gpu


def test_a_new_parameter_at_an_old_address():
    seen = set()
    for value in (1.0, 2.0, 3.0):
        w = torch.nn.Parameter(torch.full((4096,), value, device="cuda", dtype=torch.bfloat16))
        seen.add(w.data_ptr())
        assert (cuda_ops._f32(w) == value).all()
        assert cuda_ops._f32(w) is cuda_ops._f32(w)
        del w
    assert len(seen) < 3      # the allocator did hand out an address again
