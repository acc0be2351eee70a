"""The engine under a full pool when requests share blocks, on the CPU: preemption is
counted in what comes back, and a request whose blocks are all shared is preempted like
any other instead of failing."""

import pytest
import torch

import test_engine_overlap as T
from mu_b200.core.cache import PagedKVCache
from mu_b200.core.config import CacheConfig, EngineConfig, SamplingParams, SchedulerConfig
from mu_b200.core.scheduler import MuScheduler, Request, RequestStatus


def _held(c, *ids):
    """What freeing these gives back, by doing so on a copy of the bookkeeping."""
    d = PagedKVCache(1, 1, 2, 4, c.max_num_blocks, torch.float32, "cpu")
    d.free_blocks, d.block_refs = list(c.free_blocks), dict(c.block_refs)
    d.request_blocks = {r: list(t) for r, t in c.request_blocks.items()}
    d.request_pos = dict(c.request_pos)
    n = len(d.free_blocks)
    for r in ids:
        d.free(r)
    return len(d.free_blocks) - n


def test_blocks_that_come_back():
    c = PagedKVCache(1, 1, 2, 4, 32, torch.float32, "cpu")
    for r, n in (("a", 9), ("x", 5)):
        assert c.allocate(r)
        c.reserve(r, n)
    assert c.held_blocks("a", "x") == _held(c, "a", "x") == 5
    assert c.fork_many([("a", "b"), ("a", "c")])
    for ids in (["a"], ["a", "b"], ["b", "c", "a"], ["x", "b"], ["c", "a", "x", "b"], []):
        assert c.held_blocks(*ids) == _held(c, *ids), ids
    assert c.held_blocks("a", "b", "c") == 5 and c.held_blocks("none") == 0


def _running(sc, rid, status, **kw):
    q = Request(request_id=rid, **kw)
    q.status = status
    sc.running[rid] = q
    return q


def test_holders_of_shared_blocks_are_credited_together():
    """Two decodes share all of their blocks but one each: preempting both gives the
    shared ones back, and no third request has to go."""
    sc = MuScheduler(SchedulerConfig(max_batch_size=8, max_num_batched_tokens=64, max_prefill_tokens=64))
    tables = {"a": {1, 2, 3}, "b": {1, 2, 4}, "d": {5, 6}}
    for rid, gen in (("a", 9), ("b", 8), ("d", 1)):
        _running(sc, rid, RequestStatus.DECODE, num_prompt_tokens=4, num_generated_tokens=gen)
    out = sc.schedule()

    def freed_of(reqs):
        rest = set().union(*[t for r, t in tables.items() if r not in {q.request_id for q in reqs}])
        return len(set().union(*[tables[q.request_id] for q in reqs]) - rest)

    # d takes 4 blocks: a alone gives one back, a and b together four
    pre = sc.fit_blocks(out, 0, lambda r, n: 4 if r.request_id == "d" else 1,
                        lambda r: len(tables[r.request_id]), freed_of)
    assert [r.request_id for r in pre] == ["a", "b"]
    assert [r.request_id for r in out.decode_requests] == ["d"]


@pytest.mark.parametrize("overlap", [False, True])
def test_prefill_whose_blocks_are_shared_waits_for_room(overlap, monkeypatch):
    """A prompt under way, all of whose blocks a forked request shares: when its next
    piece does not fit, it is preempted and finishes once there is room."""
    from mu_b200.serving import engine as E

    monkeypatch.setattr(E, "BatchSampler", T.FakeSampler)
    ec = EngineConfig(cache=CacheConfig(block_size=4, max_num_blocks=7, max_num_seqs=4),
                      scheduler=SchedulerConfig(max_batch_size=4, max_num_batched_tokens=13,
                                                max_prefill_tokens=13, enable_chunked_prefill=True))
    w = T.FakeWorker(7)
    eng = E.StepEngine(w, ec, overlap=overlap)
    params = dict(temperature=0.0, stop_token_ids=[])
    short, long = [3, 1, 4], [(5 * i) % T.V for i in range(20)]
    got = {"r": [], "p": []}

    def step():
        for o in eng.step():
            assert o.token_id >= 0, (o.request_id, o.finish_reason)
            got[o.request_id].append(o.token_id)

    eng.add_request(short, SamplingParams(max_tokens=12, **params), "r")
    step()
    eng.add_request(long, SamplingParams(max_tokens=3, **params), "p")
    step()                                              # 12 tokens: three full blocks
    assert w.cache.get_seq_len("p") == 12
    assert w.cache.fork("p", "c") and w.cache.held_blocks("p") == 0
    assert w.allocate_request("x")                      # and the pool is full up to one block
    while len(w.cache.free_blocks) > 1:
        w.cache.reserve("x", 4)
    for _ in range(3):
        step()
    assert eng.requests["r"].num_preemptions == 0 and eng.requests["p"].num_preemptions > 0
    w.free_request("x")
    w.cache.free("c")
    for _ in range(100):
        if not eng.has_unfinished():
            break
        step()
    assert got["r"] == T.expected(short, 12, []) and got["p"] == T.expected(long, 3, [])
    assert len(w.cache.free_blocks) == 7 and not w.cache.block_refs
