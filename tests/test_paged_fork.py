"""PagedKVCache: forked requests, compaction and the 8-bit pool, on the CPU.

The 8-bit pool's values: one rounding to e4m3 is off by at most 2^-4 of the value, or
by half of e4m3's subnormal step (2^-10) times the scale; rows that a later append
finds under a smaller scale are rounded once more."""

import pytest
import torch

from mu_b200.core.cache import PagedKVCache, create_cache
from mu_b200.core.config import CacheConfig, MuConfig

FP8 = torch.float8_e4m3fn
KINDS = [torch.bfloat16, FP8]


def _cache(dtype, blocks=16, bs=4, layers=2, heads=3, d=8):
    return PagedKVCache(layers, heads, d, bs, blocks, dtype, "cpu", MuConfig(enabled=False))


def _fill(c, rid, n, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    for layer in range(c.num_layers):
        shape = (1, n, c.num_kv_heads, c.head_dim)
        c.append(rid, layer, size * torch.randn(shape, generator=g), torch.randn(shape, generator=g))


def _content(c, rid):
    return [t.float().clone() for layer in range(c.num_layers) for t in c.get(rid, layer)]


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def _consistent(c):
    """Every block is free or held as often as block_refs says."""
    held = {}
    for t in c.request_blocks.values():
        for b in t:
            held[b] = held.get(b, 0) + 1
    assert sorted(list(held) + c.free_blocks) == list(range(c.max_num_blocks))
    assert c.block_refs == {b: n for b, n in held.items() if n > 1}


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("n", [0, 1, 3, 4, 5, 8, 11])
def test_fork(dtype, n):
    c = _cache(dtype)
    c.allocate("a")
    if n:
        _fill(c, "a", n, 1)
    assert c.fork("a", "b")
    assert c.get_seq_len("b") == n
    full = n // 4
    assert c.block_table("a")[:full] == c.block_table("b")[:full]
    if n % 4 or n == 0:
        assert c.block_table("a")[-1] != c.block_table("b")[-1]
    _consistent(c)
    before = _content(c, "a") if n else []
    if n:
        assert _same(before, _content(c, "b"))
    _fill(c, "b", 6, 2, size=50.0)  # the child's rows, of another size, leave the parent's
    if n:
        assert _same(before, _content(c, "a"))
    child = _content(c, "b")
    _fill(c, "a", 6, 3, size=0.1)
    assert _same(child, _content(c, "b"))
    _consistent(c)
    c.free("a")
    _consistent(c)
    assert _same(child, _content(c, "b"))
    c.free("b")
    assert len(c.free_blocks) == 16 and not c.block_refs


def test_fork_of_a_fork_and_many():
    c = _cache(FP8)
    c.allocate("a")
    _fill(c, "a", 9, 1)
    assert c.fork_many([("a", "b"), ("a", "c")]) and c.fork("b", "d")
    _consistent(c)
    assert c.block_refs == {b: 4 for b in c.block_table("a")[:2]}
    assert c.held_blocks("a") == 1 and c.get_stats()["used_blocks"] == 6
    want = _content(c, "a")
    for r in "bcd":
        assert _same(want, _content(c, r))
    for r in "acb":
        c.free(r)
        _consistent(c)
    assert _same(want, _content(c, "d")) and c.held_blocks("d") == 3


@pytest.mark.parametrize("pairs", [[("x", "b")], [("a", "a")], [("a", "b"), ("a", "b")],
                                   [("a", "b"), ("b", "c")],
                                   [("a", "b"), ("a", "c"), ("a", "d")]])
def test_fork_refused_changes_nothing(pairs):
    c = _cache(FP8, blocks=5)
    c.allocate("a")
    _fill(c, "a", 9, 1)  # three blocks: two are free, a third child has no room
    state = (dict(c.request_blocks), dict(c.request_pos), list(c.free_blocks), dict(c.block_refs))
    want = _content(c, "a")
    assert c.fork_many(pairs) is False
    assert state == (c.request_blocks, c.request_pos, c.free_blocks, c.block_refs)
    assert _same(want, _content(c, "a"))


def test_failed_copy_changes_nothing():
    c = _cache(FP8)
    for r in "ab":
        c.allocate(r)
        _fill(c, r, 6, 1)
    c.free("a")
    state = (dict(c.request_blocks), dict(c.request_pos), list(c.free_blocks), dict(c.block_refs))

    def fails(src, dst):
        raise RuntimeError("launch")

    c._copy_blocks = fails
    with pytest.raises(RuntimeError):
        c.fork("b", "c")
    with pytest.raises(RuntimeError):
        c.compact()
    assert state == (c.request_blocks, c.request_pos, c.free_blocks, c.block_refs)


@pytest.mark.parametrize("dtype", KINDS)
def test_compact(dtype):
    c = _cache(dtype, blocks=24)
    for i, n in enumerate((9, 3, 14, 1, 8)):
        c.allocate(f"r{i}")
        _fill(c, f"r{i}", n, i)
    c.fork("r2", "r5")
    c.free("r0")
    c.free("r3")
    want = {r: _content(c, r) for r in c.request_blocks}
    moved = c.compact()
    _consistent(c)
    live = {b for t in c.request_blocks.values() for b in t}
    assert moved > 0 and live == set(range(len(live)))
    assert c.free_blocks[-1] == len(live)  # the lowest free block is handed out next
    for r, v in want.items():
        assert _same(v, _content(c, r))
    assert c.compact() == 0
    for r in list(c.request_blocks):
        _fill(c, r, 5, 77)
    _consistent(c)
    c.clear()
    assert c.compact() == 0 and len(c.free_blocks) == 24


@pytest.mark.parametrize("steps", [[1], [16], [5, 1, 1], [16, 16], [3, 40, 1, 1, 7]])
def test_quantised_values(steps):
    """Each append's rows grow, so that blocks are rounded again under larger scales."""
    c = PagedKVCache(1, 2, 64, 16, 8, FP8, "cpu", MuConfig(enabled=False))
    c.allocate("a")
    g = torch.Generator().manual_seed(3)
    ks, vs = [], []
    for i, n in enumerate(steps):
        k = 3.0 ** i * torch.randn(1, n, 2, 64, generator=g)
        v = torch.randn(1, n, 2, 64, generator=g)
        k[:, :, 1] = 0 if i == 0 else k[:, :, 1]  # a head that starts with zeros
        c.append("a", 0, k, v)
        ks.append(k)
        vs.append(v)
    n = sum(steps)
    for want, got, scale in ((torch.cat(ks, 1), c.get("a", 0)[0], c.k_scale(0)),
                             (torch.cat(vs, 1), c.get("a", 0)[1], c.v_scale(0))):
        s = scale[c.block_table("a")].repeat_interleave(16, 0)[:n]          # [n, heads]
        assert bool((s == torch.exp2(torch.round(torch.log2(s)))).all())
        step = 2.0 ** -10 * s.double()[None, :, :, None]
        bound = torch.zeros_like(want, dtype=torch.float64)
        for _ in steps:                                                      # a rounding each
            bound += torch.maximum(2.0 ** -4 * (want.double().abs() + bound), step)
        assert bool(((got.double() - want.double()).abs() <= bound).all())


def test_quantised_non_finite():
    c = PagedKVCache(1, 2, 8, 4, 8, FP8, "cpu", MuConfig(enabled=False))
    c.allocate("a")
    x = torch.ones(1, 2, 2, 8)
    x[0, 1, 0, 3] = float("inf")
    c.append("a", 0, x, torch.ones(1, 2, 2, 8))
    c.append("a", 0, torch.ones(1, 4, 2, 8), torch.ones(1, 4, 2, 8))
    k, v = c.get("a", 0)
    assert bool(k[0, :4, 0].isnan().all()) and bool((k[0, :, 1] == 1).all())
    assert bool((k[0, 4:] == 1).all()) and bool((v == 1).all())  # the next block starts anew


def test_create_cache_kind():
    c = create_cache(CacheConfig(max_num_blocks=4, dtype="float8_e4m3"), 1, 2, 64, device="cpu")
    assert c.quantized and c.block_pool.dtype == FP8 and c.scales.shape == (1, 2, 4, 2)
    b = create_cache(CacheConfig(max_num_blocks=4, dtype="bfloat16"), 1, 2, 64, device="cpu")
    assert not b.quantized and b.scales is None and b.k_scale(0) is None
    assert c.get_stats()["memory_mb"] < b.get_stats()["memory_mb"] * 0.51
