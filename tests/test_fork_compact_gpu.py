"""Forked requests and compaction under a worker: a step after the blocks have moved has
to give the bits of a worker whose blocks stayed, natively and from captured graphs."""

import pytest
import torch

from test_fp8_model_gpu import _logits, _requests, _worker

pytestmark = pytest.mark.gpu


def _content(w, rid):
    """K and V of every layer."""
    return [t.clone() for layer in range(w.cache.num_layers) for t in w.cache.get(rid, layer)]


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float8_e4m3"])
@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_step_after_compaction(cuda, name, dtype, graphs):
    R = 4
    ws = [_worker(name, cuda, dtype=dtype, graphs=graphs)[0] for _ in range(2)]
    _, d, prompts, _ = _worker(name, cuda, dtype=dtype)
    toks = d["tokens"]
    for w in ws:
        for r in range(R):
            assert w.allocate_request(f"r{r}")
        _logits(w, _requests([(f"r{r}", prompts[r]) for r in range(R)], True))
        for r in range(R):
            assert w.fork_request(f"r{r}", f"c{r}")
        for i in range(2):  # the bucket of four is captured before the blocks move
            _logits(w, _requests([(f"c{r}", [int(toks[r, i])]) for r in range(R)], False))
        for r in range(R):
            w.free_request(f"r{r}")
    moved, stayed = ws
    before = [_content(moved, f"c{r}") for r in range(R)]
    tables = [list(moved.cache.block_table(f"c{r}")) for r in range(R)]
    live = {b for t in tables for b in t}
    assert min(live) >= len(live)                   # all of them lie above the pool's front
    assert moved.cache.compact() == len(live)
    assert {b for r in range(R) for b in moved.cache.block_table(f"c{r}")} == set(range(len(live)))
    # what lay behind the old ids is not read any more
    for t in (moved.cache.block_pool, moved.cache.scales):
        if t is not None:
            t[:, :, sorted(live)] = float("nan")
    for r in range(R):
        assert all(torch.equal(a, b) for a, b in zip(before[r], _content(moved, f"c{r}")))
    for i in range(2, 5):
        step = _requests([(f"c{r}", [int(toks[r, i])]) for r in range(R)], False)
        assert torch.equal(_logits(moved, step), _logits(stayed, step))
    for r in range(R):
        for a, b in zip(_content(moved, f"c{r}"), _content(stayed, f"c{r}")):
            assert torch.equal(a, b)
    new = _requests([("n", prompts[0])], True)       # a request in blocks that others left
    for w in ws:
        assert w.allocate_request("n")
    assert torch.equal(_logits(moved, new), _logits(stayed, new))
