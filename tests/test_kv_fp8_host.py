"""Host-side rules of the KV pools and what is built over them (no GPU)."""

from __future__ import annotations

import types

import torch


def test_native_executor_goes_by_the_cache_itself(monkeypatch):
    """A KV cache made after another one was dropped may get the same id: the native executor's
    descriptor, which holds the pools' addresses, is made anew."""
    import sid.model.native
    from sid.model.qwen3 import Qwen3Model

    built = []

    class Recorder:
        def __init__(self, model, kv_cache, *_):
            built.append(kv_cache.tag)

        def forward(self, *a, **kw):
            return built[-1]

    class Cache:
        def __init__(self, tag):
            self.tag = tag

        def layer(self, i):
            return torch.zeros(4, 8, 128), None

    monkeypatch.setattr(sid.model.native, "NativeQwen3", Recorder)
    model = Qwen3Model.__new__(Qwen3Model)
    model._native, model.decode_chain = None, True
    fb = types.SimpleNamespace(sample_tiles=None)
    old = Cache("old")
    assert model._native_forward(fb, old, True) == "old"
    assert model._native_forward(fb, old, True) == "old" and built == ["old"]
    was, others = id(old), []
    del old
    for _ in range(10000):
        new = Cache("new")
        if id(new) == was:
            break
        others.append(new)
    assert id(new) == was, "no object took the dropped one's place"
    assert model._native_forward(fb, new, True) == "new"
    assert model._native_forward(fb, new, True) == "new" and built == ["old", "new"]
    model.decode_chain = False
    assert model._native_forward(fb, new, True) == "new" and built == ["old", "new", "new"]
