"""The 8-bit cache's prefill attention at the ends of its range: blocks that read as NaN
beside keys of far larger scores, infinite queries, queries too small for f32 products,
scales at both ends of [2^-60, 2^60].  Tolerances are those of test_fp8_cache_gpu."""

import math

import pytest
import torch

from test_fp8_cache_gpu import BS, FP8, _attend, _err, _gen, _k, _near, _quantised, _tables

pytestmark = pytest.mark.gpu


def _prefill(q, bt, lens, qn, kc, ks, vc, vs, hq, hkv, d):
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    out = torch.full_like(q, 7.0)
    _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          torch.tensor(cu, dtype=torch.int32, device="cuda"), max(qn), hq, hkv, d)
    assert _err() == 0
    return out


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad,loud", [(0, 5), (3, 5), (7, 0), (5, 5)])
def test_nan_block_below_far_larger_scores(cuda, bad, loud, which):
    """The key tiles of 40 rows behind 9,000 tokens are shared out in eighths; a block of
    eighth `bad` reads as NaN, the scores of eighth `loud` are hundreds of powers of two
    above all others.  A row that sees the block is NaN all the same (0 * NaN)."""
    hq, hkv, d, past, n = 4, 1, 128, 9000, 40
    ctx = past + n
    bt, nb = _tables([ctx], 3)
    kc, ks = _quantised(nb, hkv, d, 71)
    vc, vs = _quantised(nb, hkv, d, 72)
    per = -(-(-(-ctx // 64)) // 8) * 4               # blocks of an eighth
    high = bt[0, loud * per:min((loud + 1) * per, bt.shape[1])].long()
    ks[high] *= 2.0 ** 9
    q = torch.randn(n, hq * d, device="cuda", generator=_gen(73)).bfloat16()
    want, bound = _attend(q.view(n, hq, d), kc, ks, vc, vs, bt[0], ctx,
                          past + torch.arange(n, device="cuda"), d ** -0.5, hkv)
    _near(_prefill(q, bt, [ctx], [n], kc, ks, vc, vs, hq, hkv, d), want, bound, "without NaN")
    (ks if which == "k" else vs)[int(bt[0, bad * per + 5])] = float("nan")
    assert bool(_prefill(q, bt, [ctx], [n], kc, ks, vc, vs, hq, hkv, d).isnan().all())


@pytest.mark.parametrize("past,n", [(0, 100), (9000, 40), (61, 3)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (16, 8, 128), (4, 2, 64)])
def test_tiny_query_over_zero_keys(cuda, hq, hkv, d, past, n):
    """Keys of zeros (codes 0, the smallest scale, as the append writes them) on the
    diagonal and queries of about 2^-90: scores are zero, not 0 * inf, and a row is the
    average of the values that it sees."""
    ctx = past + n
    bt, nb = _tables([ctx], 7)
    kc, ks = _quantised(nb, hkv, d, 91)
    vc, vs = _quantised(nb, hkv, d, 92, spread=2.0)
    zero = bt[0, past // BS:].long()
    kc.view(torch.uint8)[zero] = 0
    ks[zero] = 2.0 ** -60
    q = (2.0 ** -90 * torch.randn(n, hq * d, device="cuda", generator=_gen(93))).bfloat16()
    out = _prefill(q, bt, [ctx], [n], kc, ks, vc, vs, hq, hkv, d)
    want, bound = _attend(q.view(n, hq, d), kc, ks, vc, vs, bt[0], ctx,
                          past + torch.arange(n, device="cuda"), d ** -0.5, hkv)
    _near(out, want, bound, f"{past} + {n}")


@pytest.mark.parametrize("value", [0.0, 1.0])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 1, 128), (4, 2, 64)])
def test_infinite_query(cuda, hq, hkv, d, value):
    """An infinite query element against codes that are negative for every key but one of
    each sequence: that key's score is inf * 0 = NaN or inf, the others' -inf, and the
    softmax of such a row is NaN, at every place of the key in its block."""
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
    out = _prefill(q.flatten(1), bt, lens, [1] * 16, kc.to(FP8), ks, vc, vs, hq, hkv, d)
    assert bool(out.isnan().all())


@pytest.mark.parametrize("past,n", [(0, 100), (9000, 40)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (16, 8, 128), (4, 2, 64)])
def test_values_of_both_ends_of_the_scale_range(cuda, hq, hkv, d, past, n):
    """Blocks of zero values (the smallest scale) whose keys score far below the others',
    whose values have the largest: the unseen and the faint keys add nothing to the sum."""
    ctx = past + n
    bt, nb = _tables([ctx], 8)
    kc, ks = _quantised(nb, hkv, d, 94)
    vc, vs = _quantised(nb, hkv, d, 95)
    kf = kc.float()
    kf[..., 0] = 448.0                               # the score of every key: about +-448 * 8 * scale
    odd = torch.zeros(nb, dtype=torch.bool, device="cuda")
    odd[bt[0, 1::2].long()] = True
    kf[odd] = 0.0
    kf[odd, ..., 0] = -448.0
    kc = kf.to(FP8)
    ks[:] = 2.0 ** -3
    vs[:] = 2.0 ** 60
    vc.view(torch.uint8)[odd] = 0
    vs[odd] = 2.0 ** -60
    q = torch.randn(n, hq, d, device="cuda", generator=_gen(96)).bfloat16()
    q[:, :, 0] = 64.0
    out = _prefill(q.flatten(1), bt, [ctx], [n], kc, ks, vc, vs, hq, hkv, d)
    want, bound = _attend(q, kc, ks, vc, vs, bt[0], ctx, past + torch.arange(n, device="cuda"),
                          d ** -0.5, hkv)
    _near(out, want, bound, f"{past} + {n}")


@pytest.mark.parametrize("size", [4, 18, 24, 26, 30, 40, 60, 100])
@pytest.mark.parametrize("hq,hkv,d,ctx", [(4, 1, 128, 9040), (16, 8, 128, 300), (4, 2, 64, 300)])
def test_scores_of_any_size(cuda, hq, hkv, d, ctx, size):
    """Scores of about 2^6 times 2^`size`, positive and negative: one key of each sequence
    stands above all others, and its value is the row (no sum, so nothing rounds: a code
    times a power of two is a bf16 number)."""
    n = 8 if ctx < 1000 else 2
    bt, nb = _tables([ctx] * n, 6)
    sign = torch.where(torch.rand(d, device="cuda", generator=_gen(97)) < 0.5, -1.0, 1.0)
    vc, vs = _quantised(nb, hkv, d, 98, spread=2.0)
    ks = torch.full((nb, hkv), 2.0 ** (size // 2), device="cuda")
    for above, others in ((4.0, 0.5), (-0.5, -4.0)):
        kf = others * torch.exp2(torch.randint(-1, 1, (nb, hkv, BS, d), device="cuda", generator=_gen(99)).float()) * sign
        stars = [(37 * b + 5) % ctx if ctx < 1000 else 9000 - 4444 * b for b in range(n)]
        for b, t in enumerate(stars):
            kf[int(bt[b, t // BS]), :, t % BS] = above * sign
        q = (2.0 ** (size - size // 2) * sign).expand(n, hq, d).bfloat16().contiguous()
        out = _prefill(q.flatten(1), bt, [ctx] * n, [1] * n, kf.to(FP8), ks, vc, vs, hq, hkv, d)
        for b, t in enumerate(stars):
            i = int(bt[b, t // BS])
            want = (vc[i, :, t % BS].float() * vs[i][:, None]).repeat_interleave(hq // hkv, 0)
            assert torch.equal(out[b].view(hq, d).float(), want), (above, b)
