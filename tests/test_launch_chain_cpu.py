"""Host side of the launches, no GPU: chains of dependent launches belong to the thread that opened them; size caches."""
import threading

import pytest

from rwkvtune_b200.ops import _ext, fp8_native


def in_thread(fn):
    out = []
    t = threading.Thread(target=lambda: out.append(fn()))
    t.start()
    t.join()
    return out[0]


class Recorder:
    """Stands for the library: the values that each thread's chaining is set to."""

    def __init__(self):
        self.calls = []

    def rwkv_set_launch_chaining(self, on):
        self.calls.append((threading.get_ident(), on.value))
        return 0


def test_a_chain_is_its_threads_own(monkeypatch):
    fake = Recorder()
    monkeypatch.setattr(_ext, "available", lambda: True)
    monkeypatch.setattr(_ext, "lib", lambda: fake)
    monkeypatch.setattr(_ext, "CHAINING_ALLOWED", True)

    def other():
        before = _ext.chaining(), fp8_native.chaining()
        with _ext.launch_chaining():
            inside = _ext.chaining()
            with _ext.launch_chaining():           # nested: one chain
                pass
            return before, inside, _ext.chaining(), threading.get_ident()

    assert not _ext.chaining()
    with _ext.launch_chaining():
        assert _ext.chaining() and fp8_native.chaining()
        before, inside, after_nested, ident = in_thread(other)
        assert before == (False, False) and inside and after_nested
        assert _ext.chaining()
    assert not _ext.chaining() and not in_thread(_ext.chaining)
    me = threading.get_ident()
    assert fake.calls == [(me, 1), (ident, 1), (ident, 0), (me, 0)]


def test_the_library_keeps_a_chain_per_thread():
    if not _ext.available():
        pytest.skip("the native library has not been built")
    switch = _ext.lib().rwkv_set_launch_chaining
    assert switch(1) == 0
    try:
        assert in_thread(lambda: (switch(0), switch(1), switch(0))) == (0, 0, 1)
    finally:
        assert switch(0) == 1


def test_size_caches_are_bounded(monkeypatch):
    """What is remembered by size does not grow with every new length of a batch."""
    class Sizes:
        def __init__(self):
            self.rwkv_fp8_workspace = lambda m, n, k: m

        def rwkv_fp8_decode_form(self, m, n, k, packed):
            return 1

    monkeypatch.setattr(_ext, "lib", lambda fake=Sizes(): fake)
    caches = [fp8_native._workspace_bytes, fp8_native.decode_form]
    for c in caches:
        c.cache_clear()
    try:
        for m in range(1, 9000):
            assert fp8_native._workspace_bytes(m, 64, 64) == m
            assert fp8_native.decode_form(m, 64, 64) == (1 if m <= 128 else 0)
        assert all(c.cache_info().maxsize is not None and c.cache_info().currsize <= 4096 for c in caches)
    finally:
        for c in caches:
            c.cache_clear()


def test_refreshed_copies_of_parameters_restart_the_chain(monkeypatch):
    """Chained kernels read parameters before they wait; a copy that is made inside the chain has to be waited for."""
    import torch

    from rwkvtune_b200 import ops
    from rwkvtune_b200.models import RWKV7Model, RWKVConfig
    from rwkvtune_b200.ops import cuda_ops

    class Library(Recorder):
        restarts = 0

        def rwkv_restart_launch_chain(self):
            self.restarts += 1

    fake = Library()
    monkeypatch.setattr(_ext, "available", lambda: True)
    monkeypatch.setattr(_ext, "lib", lambda: fake)
    monkeypatch.setattr(_ext, "CHAINING_ALLOWED", True)
    p = torch.nn.Parameter(torch.randn(16).to(torch.bfloat16))
    att = RWKV7Model(RWKVConfig(n_layer=1, n_embd=64, vocab_size=16, dim_att_lora=16, dim_gate_lora=16, dim_mv_lora=16)).blocks[0].att
    with torch.no_grad():
        cuda_ops._f32(p), att.mix_matrix()
        assert fake.restarts == 0                       # outside of a chain there is nothing to restart
        with _ext.launch_chaining():
            for expected, touched in ((0, ()), (1, (p,)), (2, (att.x_r,)), (4, (p, att.x_k)), (4, ())):
                for t in touched:
                    t.add_(1)
                cuda_ops._f32(p), att.mix_matrix()
                assert fake.restarts == expected
            ops.bump_param_epoch()
            cuda_ops._f32(p), att.mix_matrix()
            assert fake.restarts == 6
            cuda_ops._f32(torch.nn.Parameter(torch.randn(16).to(torch.bfloat16)))
            assert fake.restarts == 7
