"""What the native steps and the captured graphs keep of a cache has to change with the
cache, on the CPU: addresses alone do not tell two caches apart, since a smaller pool may
be carved from the start of a freed one."""

import contextlib
from types import SimpleNamespace

import pytest
import torch

from mu_b200.core.cache import PagedKVCache
from mu_b200.core.config import MuConfig
from mu_b200.models.base import MuModelBase

FP8 = torch.float8_e4m3fn
KINDS = [torch.bfloat16, FP8]


def _cache(blocks, dtype, bs=16, heads=2, d=64, layers=2):
    return PagedKVCache(layers, heads, d, bs, blocks, dtype, "cpu", MuConfig(enabled=False))


def _at(cache, other):
    """`cache` moved to the start of `other`'s memory."""
    for name in ("block_pool", "scales"):
        t, o = getattr(cache, name), getattr(other, name)
        if t is not None:
            setattr(cache, name, o.view(-1)[: t.numel()].view(t.shape))
    return cache


@pytest.mark.parametrize("dtype", KINDS)
def test_key_tells_pools_at_one_address_apart(dtype):
    a = _cache(12, dtype)
    key = MuModelBase.cache_key(a)
    assert key == MuModelBase.cache_key(_at(_cache(12, dtype), a))
    for other in (_cache(8, dtype), _cache(8, dtype, bs=8)):
        b = _at(other, a)
        assert b.block_pool.data_ptr() == a.block_pool.data_ptr()
        assert MuModelBase.cache_key(b) != key


class _Graph:
    """A captured graph: replays what the model did under the capture."""

    def __init__(self):
        self.steps, self.replays = [], 0

    def replay(self):
        self.replays += 1


@pytest.fixture
def graphs(monkeypatch):
    """torch.cuda's graph calls without a device."""
    stream = SimpleNamespace(wait_stream=lambda s: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _Graph)
    monkeypatch.setattr(torch.cuda, "graph", lambda g: contextlib.nullcontext())


def _graph_worker(cache):
    from mu_b200.core.config import EngineConfig
    from mu_b200.serving.step import StepPacker
    from mu_b200.serving.worker import MuWorker

    w = MuWorker(EngineConfig(), "cpu")
    w.cache, w.packer = cache, StepPacker("cpu", 16, 4, 4)
    seen = []
    w.model = SimpleNamespace(ws=SimpleNamespace(serial=1, logits=torch.zeros(4, 8)), tp_group=None,
                              ensure_workspace=lambda *a: False, cache_key=MuModelBase.cache_key,
                              forward_step=lambda batch, c: seen.append(c))
    return w, seen


def _decode(w, rid):
    seqs, errors = w.prepare([(rid, [1])], 1)
    assert not errors
    w.run_step(seqs, 1)


def test_graphs_follow_the_cache(graphs):
    """A decode step after the cache was replaced, or its blocks or scales moved, is
    captured anew; steps over an unchanged cache are replayed."""
    big = _cache(12, FP8)
    w, seen = _graph_worker(big)

    def replayed():
        n = len(seen)
        _decode(w, "a")
        assert all(c is w.cache for c in seen[n:])
        return len(seen) == n

    for cache in (big, _cache(12, torch.bfloat16), _at(_cache(8, FP8), big)):
        w.cache = cache
        assert w.allocate_request("a")
        assert not replayed() and replayed() and replayed()
    w.cache.scales = w.cache.scales.clone()
    assert not replayed() and replayed()
    w.cache.block_pool = w.cache.block_pool.clone()
    assert not replayed() and replayed()
    w.cache = big  # not what an older capture held
    assert not replayed() and replayed()


@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_native_step_follows_the_workspace(name):
    """Two growths between two steps: the second workspace may be the Python object of
    the one before the first (the interpreter reuses its place)."""
    from golden_models import load_tiny
    from mu_b200 import _lib
    from mu_b200.models.loader import build_model

    if not _lib.LIB_PATH.exists():
        pytest.skip("libmuk.so not built (run complexity-inference_b200/build.py)")
    shape, cfg, sd, _, _ = load_tiny(name)
    m = build_model(shape.arch, cfg, sd, MuConfig(enabled=True), "cpu")
    c = PagedKVCache(cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.head_dim, 16, 4,
                     torch.bfloat16, "cpu")
    m.use_cache(c)
    for n in range(64, 128, 2):
        m.ensure_workspace(n, 2, 64)
        assert m._native(c).qkv == m.ws.qkv.data_ptr()
        for more in (1, 2):
            m.ensure_workspace(n + more, 2, 64)
        assert m._native(c).qkv == m.ws.qkv.data_ptr()
