"""A worker whose cache is replaced, or moved: the step that follows has to give the bits
of a worker that had that cache from the start, natively and from captured graphs."""

import pytest
import torch

from golden_models import load_tiny
from test_fp8_model_gpu import _logits, _requests, _worker

pytestmark = pytest.mark.gpu

KINDS = ["bfloat16", "float8_e4m3"]


def _cache(w, blocks, dtype, memory=None):
    """A cache for `w`'s model; with `memory` (another cache) at the start of its memory."""
    from mu_b200.core.cache import PagedKVCache

    mc = w.model.config
    c = PagedKVCache(mc.num_hidden_layers, mc.num_key_value_heads, mc.head_dim, 16, blocks,
                     {"bfloat16": torch.bfloat16, "float8_e4m3": torch.float8_e4m3fn}[dtype],
                     str(w.device), w.cache.mu_config)
    for name in ("block_pool", "scales"):
        t = getattr(c, name)
        if memory is not None and t is not None:
            part = getattr(memory, name).view(-1)[: t.numel()].view(t.shape)
            part.copy_(t)
            setattr(c, name, part)
    return c


def _run(w, prompts, rid, n=4):
    """A prompt and n - 1 decodes of request `rid`."""
    assert w.allocate_request(rid)
    out = [_logits(w, _requests([(rid, prompts[0])], True))]
    return out + [_logits(w, _requests([(rid, [5 + i])], False)) for i in range(n - 1)]


def _pool(c):
    return [t.view(torch.uint8).cpu() for t in (c.block_pool, c.scales) if t is not None]


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_smaller_cache_in_the_memory_of_another(cuda, name, dtype):
    """The native step of a cache of 64 blocks that lies where one of 256 lay."""
    w, _, prompts, _ = _worker(name, cuda, dtype=dtype, blocks=256)
    _run(w, prompts, "a")
    big = w.cache
    w.cache = _cache(w, 64, dtype, memory=big)
    assert w.cache.block_pool.data_ptr() == big.block_pool.data_ptr()
    got = _run(w, prompts, "b")
    ref, _, _, _ = _worker(name, cuda, dtype=dtype, blocks=64)
    assert _same(got, _run(ref, prompts, "b")) and _same(_pool(w.cache), _pool(ref.cache))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_graphs_of_caches_in_turn(cuda, name, native):
    """Caches of both kinds and of two sizes in turn under one worker with graphs, each
    decode from a bucket that was captured before the swap."""
    caches = [("bfloat16", 256), ("float8_e4m3", 256), ("float8_e4m3", 64), ("bfloat16", 64)]
    w, _, prompts, _ = _worker(name, cuda, dtype=caches[0][0], graphs=True, native=native)
    live = [w.cache] + [_cache(w, n, dtype) for dtype, n in caches[1:]]
    got = [[] for _ in caches]
    for turn in range(2):
        for i, c in enumerate(live):
            w.cache = c
            got[i] += _run(w, prompts, f"r{turn}")
    for i, (dtype, n) in enumerate(caches):
        ref, _, _, _ = _worker(name, cuda, dtype=dtype, graphs=True, native=native, blocks=n)
        want = _run(ref, prompts, "r0") + _run(ref, prompts, "r1")
        assert ref.get_stats()["cuda_graphs"] and _same(got[i], want), (dtype, n)
        assert _same(_pool(live[i]), _pool(ref.cache)), (dtype, n)


@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_graphs_follow_moved_memory(cuda, name):
    """Scales, then blocks, at other addresses between two decodes of a captured bucket."""
    w, _, prompts, _ = _worker(name, cuda, graphs=True)
    ref, _, _, _ = _worker(name, cuda, graphs=True)
    assert _same(_run(w, prompts, "a"), _run(ref, prompts, "a"))
    for part in ("scales", "block_pool"):
        old = getattr(w.cache, part)
        setattr(w.cache, part, old.clone())
        old.view(torch.uint8).fill_(0x7F)
        kept = old.view(torch.uint8).clone()
        for tok in (9, 10):
            step = _requests([("a", [tok])], False)
            assert torch.equal(_logits(w, step), _logits(ref, step))
        assert torch.equal(old.view(torch.uint8), kept) and _same(_pool(w.cache), _pool(ref.cache))
