"""The 8-bit cache's decode attention at the ends of its range, as
test_fp8_prefill_extremes_gpu does it for prefill: whole sequences of a warp and
sequences whose results several runs share and join."""

import math

import pytest
import torch

from test_fp8_cache_gpu import FP8, _attend, _err, _gen, _k, _near, _quantised, _tables

pytestmark = pytest.mark.gpu

SHAPES = [(4, 1, 128), (32, 8, 128), (16, 1, 128), (4, 2, 64)]


def _decode(q, bt, lens, kc, ks, vc, vs, hq, hkv, d):
    out = torch.full_like(q, 7.0)
    ws = torch.empty(max(4, _k().decode_attn_fp8_workspace_size(len(lens), hq, d, max(lens)) // 4),
                     device="cuda")
    _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                         hq, hkv, d, max(lens), workspace=ws)
    assert _err() == 0
    return out


def _check(q, bt, lens, kc, ks, vc, vs, hq, hkv, d):
    out = _decode(q.flatten(1), bt, lens, kc, ks, vc, vs, hq, hkv, d)
    for b, ctx in enumerate(lens):
        want, bound = _attend(q[b:b + 1], kc, ks, vc, vs, bt[b], ctx,
                              torch.tensor([ctx - 1], device="cuda"), d ** -0.5, hkv)
        _near(out[b:b + 1], want, bound, f"sequence of {ctx}")


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad,loud", [(0.0, 0.6), (0.4, 0.9), (0.95, 0.1), (0.5, 0.5)])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_nan_block_below_far_larger_scores(cuda, hq, hkv, d, bad, loud, which):
    """Behind 9,000 tokens: a tenth of the blocks has scores hundreds of powers of two above
    the others, one block reads as NaN."""
    bt, nb = _tables([9000], 3)
    n = bt.shape[1]
    kc, ks = _quantised(nb, hkv, d, 71)
    vc, vs = _quantised(nb, hkv, d, 72)
    ks[bt[0, int(loud * n):int(loud * n) + n // 10].long()] *= 2.0 ** 9
    q = torch.randn(1, hq, d, device="cuda", generator=_gen(73)).bfloat16()
    _check(q, bt, [9000], kc, ks, vc, vs, hq, hkv, d)
    (ks if which == "k" else vs)[int(bt[0, int(bad * n) + 1])] = float("nan")
    assert bool(_decode(q.flatten(1), bt, [9000], kc, ks, vc, vs, hq, hkv, d).isnan().all())


@pytest.mark.parametrize("value", [0.0, 1.0])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_infinite_query(cuda, hq, hkv, d, value):
    """One key of each sequence scores inf * 0 = NaN or inf, all others -inf."""
    lens = [64] * 16
    bt, nb = _tables(lens, 5)
    kc, ks = _quantised(nb, hkv, d, 81)
    vc, vs = _quantised(nb, hkv, d, 82)
    kc = kc.float()
    kc[..., 0] = -1.0
    for b in range(16):
        kc[int(bt[b, b % 4]), :, b, 0] = value
    q = torch.randn(16, hq, d, device="cuda", generator=_gen(83)).bfloat16()
    q[:, :, 0] = math.inf
    assert bool(_decode(q.flatten(1), bt, lens, kc.to(FP8), ks, vc, vs, hq, hkv, d).isnan().all())


@pytest.mark.parametrize("ctx", [1, 100, 9040])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_tiny_query_over_zero_keys(cuda, hq, hkv, d, ctx):
    bt, nb = _tables([ctx], 7)
    kc, ks = _quantised(nb, hkv, d, 91)
    vc, vs = _quantised(nb, hkv, d, 92, spread=2.0)
    zero = bt[0, bt.shape[1] // 2:].long()
    kc.view(torch.uint8)[zero] = 0
    ks[zero] = 2.0 ** -60
    q = (2.0 ** -90 * torch.randn(1, hq, d, device="cuda", generator=_gen(93))).bfloat16()
    _check(q, bt, [ctx], kc, ks, vc, vs, hq, hkv, d)


@pytest.mark.parametrize("ctx", [100, 9040])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_values_of_both_ends_of_the_scale_range(cuda, hq, hkv, d, ctx):
    """Every other block has zero values (the smallest scale) and scores far below the
    others', whose values have the largest scale."""
    bt, nb = _tables([ctx], 8)
    kc, ks = _quantised(nb, hkv, d, 94)
    vc, vs = _quantised(nb, hkv, d, 95)
    kf = kc.float()
    kf[..., 0] = 448.0
    odd = torch.zeros(nb, dtype=torch.bool, device="cuda")
    odd[bt[0, 1::2].long()] = True
    kf[odd] = 0.0
    kf[odd, ..., 0] = -448.0
    ks[:] = 2.0 ** -3
    vs[:] = 2.0 ** 60
    vc.view(torch.uint8)[odd] = 0
    vs[odd] = 2.0 ** -60
    q = torch.randn(1, hq, d, device="cuda", generator=_gen(96)).bfloat16()
    q[:, :, 0] = 64.0
    _check(q, bt, [ctx], kf.to(FP8), ks, vc, vs, hq, hkv, d)


@pytest.mark.parametrize("size", [4, 18, 24, 26, 30, 40, 60, 100])
@pytest.mark.parametrize("ctx", [300, 9040])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_scores_of_any_size(cuda, hq, hkv, d, ctx, size):
    """Scores of about 2^6 times 2^`size`: one key of each sequence stands above all others
    and its value is the row."""
    n = 3
    bt, nb = _tables([ctx] * n, 6)
    sign = torch.where(torch.rand(d, device="cuda", generator=_gen(97)) < 0.5, -1.0, 1.0)
    vc, vs = _quantised(nb, hkv, d, 98, spread=2.0)
    ks = torch.full((nb, hkv), 2.0 ** (size // 2), device="cuda")
    for above, others in ((4.0, 0.5), (-0.5, -4.0)):
        kf = others * torch.exp2(torch.randint(-1, 1, (nb, hkv, 16, d), device="cuda", generator=_gen(99)).float()) * sign
        stars = [(4111 * b + 5) % ctx for b in range(n)]
        for b, t in enumerate(stars):
            kf[int(bt[b, t // 16]), :, t % 16] = above * sign
        q = (2.0 ** (size - size // 2) * sign).expand(n, hq, d).bfloat16().contiguous()
        out = _decode(q.flatten(1), bt, [ctx] * n, kf.to(FP8), ks, vc, vs, hq, hkv, d)
        for b, t in enumerate(stars):
            i = int(bt[b, t // 16])
            want = (vc[i, :, t % 16].float() * vs[i][:, None]).repeat_interleave(hq // hkv, 0)
            assert torch.equal(out[b].view(hq, d).float(), want), (above, b)
