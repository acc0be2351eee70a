"""The 8-bit KV cache in the models' step and the serving engine.

The attention of a step is held to 64 bits over the cache that the step itself wrote;
the native executors, the CUDA graphs and a forked or compacted cache have to give the
bits of the plain step."""

import numpy as np
import pytest
import torch

from golden_models import load_tiny
from test_fp8_cache_gpu import _attend, _near

pytestmark = pytest.mark.gpu


def _worker(name, cuda, dtype="float8_e4m3", graphs=False, native=True, max_batch=8, blocks=256):
    from mu_b200.core.config import CacheConfig, EngineConfig, MuConfig, SchedulerConfig
    from mu_b200.serving.worker import MuWorker

    shape, cfg, sd, d, prompts = load_tiny(name)
    ec = EngineConfig(model=cfg, mu=MuConfig(enabled=True),
                      cache=CacheConfig(max_seq_len=256, max_num_blocks=blocks, max_num_seqs=16,
                                        dtype=dtype),
                      scheduler=SchedulerConfig(max_batch_size=max_batch,
                                                max_num_batched_tokens=2048))
    w = MuWorker(ec, str(cuda))
    w.load_state_dict(shape.arch, cfg, sd)
    w.use_graphs, w.model.native = graphs, native
    return w, d, prompts, ec


def _requests(ids, prefill):
    from mu_b200.serving.worker import WorkerRequest

    return [WorkerRequest(r, torch.tensor([t]), is_prefill=prefill) for r, t in ids]


def _logits(w, reqs):
    outs = w.execute(reqs)
    assert all(o.error is None for o in outs), [o.error for o in outs]
    return torch.stack([o.logits.float().cpu().reshape(-1) for o in outs])


def _steps(w, prompts, toks, n=6):
    """Prompts, then decodes with one more prompt among them, then pure decodes."""
    R = len(prompts)
    for r in range(R):
        assert w.allocate_request(f"r{r}")
    out = [_logits(w, _requests([(f"r{r}", prompts[r]) for r in range(R - 1)], True))]
    out.append(_logits(w, _requests([(f"r{r}", [int(toks[r, 0])]) for r in range(R - 1)], False)
                       + _requests([(f"r{R - 1}", prompts[R - 1])], True)))
    for i in range(1, n):
        out.append(_logits(w, _requests([(f"r{r}", [int(toks[r, i])]) for r in range(R)], False)))
    return out


@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_native_step_and_graphs_equal_plain_step(cuda, name):
    from mu_b200 import _lib

    runs, pools, launches = [], [], []
    for native, graphs in ((False, False), (True, False), (True, True)):
        w, d, prompts, _ = _worker(name, cuda, graphs=graphs, native=native)
        assert w.cache.quantized and w.cache.block_pool.dtype == torch.float8_e4m3fn
        n0 = _lib.launch_count
        runs.append(_steps(w, prompts, d["tokens"]))
        launches.append(_lib.launch_count - n0)
        pools.append((w.cache.block_pool.view(torch.uint8).cpu(), w.cache.scales.cpu()))
    assert _lib.device_error() == 0
    for a, b in zip(runs[0], runs[1]):
        assert torch.equal(a, b)
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
    assert launches[0] == launches[1]
    # a graph splits the contexts for its own bound, so its sums have another order; the
    # bf16 step's tolerance against the f32 reference holds between any two such orders
    for a, b in zip(runs[0], runs[2]):
        assert float((a - b).abs().max()) <= 2e-2


@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_step_attends_to_its_layers_cache(cuda, name):
    w, d, prompts, _ = _worker(name, cuda, native=False)
    m, c = w.model, w.cache
    Hq, Hkv, D = m.config.num_attention_heads, m.config.num_key_value_heads, m.config.head_dim
    plain, seen = m.attention, []

    def attention(layer, batch, cache):
        out = plain(layer, batch, cache)
        q = m.ws.qkv[:, : Hq * D].unflatten(1, (Hq, D))
        lens, bt = batch.seq_lens.tolist(), batch.block_tables
        pcu = batch.prefill_cu.tolist()
        nd = batch.num_decode
        rows = [(b, b, b + 1) for b in range(nd)] + \
            [(nd + i, nd + pcu[i], nd + pcu[i + 1]) for i in range(batch.num_seqs - nd)]
        for b, lo, hi in rows:
            ctx = lens[b]
            limits = torch.arange(ctx - (hi - lo), ctx, device="cuda")
            want, bound = _attend(q[lo:hi], c.k_cache(layer), c.k_scale(layer), c.v_cache(layer),
                                  c.v_scale(layer), bt[b], ctx, limits, D ** -0.5, Hkv)
            _near(out[lo:hi], want, bound, f"layer {layer} sequence {b}")
            seen.append((layer, b))
        return out

    m.attention = attention
    _steps(w, prompts, d["tokens"], n=3)
    assert len({layer for layer, _ in seen}) == m.config.num_hidden_layers


def test_append_of_the_cache_equals_the_kernel(cuda):
    """PagedKVCache.append on a CPU pool and the fused append, with RoPE tables that do
    not rotate, leave the same codes and scales."""
    from mu_b200 import kernels as K
    from mu_b200.core.cache import PagedKVCache
    from mu_b200.core.config import MuConfig

    Hkv, D = 2, 64
    host = PagedKVCache(1, Hkv, D, 16, 16, torch.float8_e4m3fn, "cpu", MuConfig(enabled=False))
    dev = PagedKVCache(1, Hkv, D, 16, 16, torch.float8_e4m3fn, str(cuda), MuConfig(enabled=False))
    cos, sin = torch.ones(128, D // 2, device=cuda), torch.zeros(128, D // 2, device=cuda)
    g = torch.Generator().manual_seed(5)
    host.allocate("a")
    dev.allocate("a")
    at = 0
    for i, n in enumerate((5, 1, 1, 30, 1, 16, 7)):
        kv = (2.0 ** (i - 3) * torch.randn(n, 2 * Hkv, D, generator=g)).bfloat16()
        kv[0, 0, 0] = 448.0 if i == 2 else kv[0, 0, 0]
        host.append("a", 0, kv[None, :, :Hkv], kv[None, :, Hkv:])
        qkv = torch.cat([torch.zeros(n, D).bfloat16(), kv.reshape(n, -1)], 1).to(cuda)
        slots = torch.from_numpy(dev.reserve("a", n)).to(cuda)
        pos = torch.arange(at, at + n, dtype=torch.int32, device=cuda)
        # one query head for two KV heads is not a shape of the kernel: two query heads
        qkv = torch.cat([qkv[:, :D], qkv], 1).contiguous()
        K.rope_kv_append_fp8(qkv, pos, slots, cos, sin, 2, Hkv, D, dev.k_cache(0), dev.v_cache(0),
                             dev.k_scale(0), dev.v_scale(0))
        at += n
        k0, v0 = host.get("a", 0)
        k1, v1 = dev.get("a", 0)
        assert torch.equal(k0, k1.cpu()) and torch.equal(v0, v1.cpu()), i
        live = host.block_table("a")
        assert torch.equal(host.scales[:, :, live], dev.scales.cpu()[:, :, live])


@pytest.mark.parametrize("dtype", ["bfloat16", "float8_e4m3"])
@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_forked_request(cuda, name, dtype):
    w, d, prompts, _ = _worker(name, cuda, dtype=dtype)
    R, toks = 4, d["tokens"]
    for r in range(R):
        assert w.allocate_request(f"r{r}")
    _logits(w, _requests([(f"r{r}", prompts[r]) for r in range(R)], True))
    for r in range(R):
        assert w.fork_request(f"r{r}", f"c{r}")
    assert not w.fork_request("r0", "c0") and not w.fork_request("none", "c9")
    child = [_logits(w, _requests([(f"c{r}", [int(toks[r, i])]) for r in range(R)], False))
             for i in range(3)]
    other = _logits(w, _requests([(f"c{r}", [7]) for r in range(R)], False))
    parent = [_logits(w, _requests([(f"r{r}", [int(toks[r, i])]) for r in range(R)], False))
              for i in range(3)]
    for a, b in zip(child, parent):
        assert torch.equal(a, b)
    want = [w.cache.get(f"c{r}", 1)[0].clone() for r in range(R)]
    for r in range(R):
        w.free_request(f"r{r}")
    assert w.cache.compact() >= 0
    for r in range(R):
        assert torch.equal(want[r], w.cache.get(f"c{r}", 1)[0])
    again = _logits(w, _requests([(f"c{r}", [9]) for r in range(R)], False))
    assert bool(torch.isfinite(again).all()) and bool(torch.isfinite(other).all())
    for r in range(R):
        w.free_request(f"c{r}")
    assert len(w.cache.free_blocks) == w.cache.max_num_blocks


@pytest.mark.parametrize("blocks", [256, 30])
def test_engine_generates_the_decisive_tokens(cuda, blocks):
    """Greedy generation with the 8-bit cache, continuous batching and CUDA graphs: the
    fixture's residual stream stays close to the token's embedding (top-2 gap above 1
    at every step), and attention, whose rows alone change with the cache's rounding,
    moves its logits far less than that.  A pool of 30 blocks holds about half of the
    requests: others are preempted and prefilled again into blocks that held theirs."""
    from mu_b200.core.config import SamplingParams
    from mu_b200.serving.engine import StepEngine

    w, d, prompts, ec = _worker("llama_decisive", cuda, graphs=True, max_batch=7, blocks=blocks)
    toks = d["tokens"]
    R, n = toks.shape
    eng = StepEngine(w, ec)
    for r in range(R):
        eng.add_request(prompts[r], SamplingParams(temperature=0.0, top_k=0, top_p=1.0,
                                                   repetition_penalty=1.0, max_tokens=n), f"r{r}")
    eng.run_to_completion()
    for r in range(R):
        assert eng.requests[f"r{r}"].output_token_ids == [int(t) for t in toks[r]]
    assert w.get_stats()["cuda_graphs"] and not w.cache.block_refs
    assert len(w.cache.free_blocks) == w.cache.max_num_blocks


def test_bf16_and_8_bit_workers_share_a_model(cuda):
    """One model stepped with a cache of each kind in turn: each keeps its results."""
    w, d, prompts, _ = _worker("llama_tiny", cuda, dtype="bfloat16")
    from mu_b200.core.cache import PagedKVCache

    mc, bf16 = w.model.config, w.cache
    fp8 = PagedKVCache(mc.num_hidden_layers, mc.num_key_value_heads, mc.head_dim, 16, 256,
                       torch.float8_e4m3fn, str(cuda), w.cache.mu_config)
    got = {}
    for turn in range(2):
        for kind, cache in (("bf16", bf16), ("fp8", fp8)):
            w.cache = cache
            rid = f"{kind}{turn}"
            assert w.allocate_request(rid)
            lg = _logits(w, _requests([(rid, prompts[0])], True))
            got.setdefault(kind, []).append(lg)
    assert torch.equal(*got["bf16"]) and torch.equal(*got["fp8"])
    assert not torch.equal(got["bf16"][0], got["fp8"][0])


@pytest.mark.parametrize("name", ["llama_tiny", "deep_tiny"])
def test_native_step_follows_moved_scales(cuda, name):
    """Scales at another address beside a pool at the same one (a cache made anew)."""
    w, d, prompts, _ = _worker(name, cuda)
    for r in range(2):
        assert w.allocate_request(f"r{r}")
    reqs = [(f"r{r}", prompts[0]) for r in range(2)]
    _logits(w, _requests(reqs[:1], True))
    old = w.cache.scales
    w.cache.scales = old.clone()
    old.fill_(float("nan"))
    _logits(w, _requests(reqs[1:], True))
    assert bool(old.isnan().all())
    assert bool(torch.isfinite(_logits(w, _requests([("r0", [3]), ("r1", [3])], False))).all())


def test_shapes_that_are_not_built_are_refused(cuda):
    from mu_b200.core.cache import PagedKVCache

    w, _, _, _ = _worker("llama_tiny", cuda)
    mc = w.model.config
    for hd, bs in ((mc.head_dim, 8), (32, 16)):
        c = PagedKVCache(1, mc.num_key_value_heads, hd, bs, 4, torch.float8_e4m3fn, str(cuda))
        with pytest.raises(ValueError, match="not built"):
            w.model.use_cache(c)
