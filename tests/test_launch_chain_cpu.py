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
