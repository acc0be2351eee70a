"""The 8-bit KV cache's kernels against plain implementations in 64 bits.

Tolerances (eps / 2 of a type is the largest relative error of one rounding to it:
bf16 2^-8, f16 2^-11, f32 2^-24, e4m3 2^-4):

* attention rows are one bf16 rounding (2^-8 of the value) of O / l, where
  - a softmax weight is rounded to f16: 2^-11 of itself, and never less than
    2^-25 of the largest weight x scale (f16's subnormal step is 2^-24),
  - its exponent carries the score's error: (D + 8) f32 roundings of the sum
    sum |q k| (products of f16 numbers are exact in f32, the sums are not; two
    multiplications by scales), and the 2^-22 relative error of exp2 with an
    argument of up to a few hundred (2^-24 x |argument| more),
  - the sums over n keys round n times (2^-23 each: the tensor core may truncate).
* codes: the kernel rounds x * 2^-e once to e4m3; x is the rotated f32 value. The
  plain form below takes the same f32 steps, so codes and scales are equal. A
  second check holds the stored values to 64 bits: 2^-4 of the value or half of
  e4m3's subnormal step (2^-10) times the scale, per rounding.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BS = 16
FP8 = torch.float8_e4m3fn


def _k():
    from mu_b200 import kernels

    return kernels


def _err():
    from mu_b200 import _lib

    return _lib.device_error()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(codes, scale):
    return codes.double() * scale.double()[..., None, None]


def _quantised(nb, hkv, d, seed, spread=0.0):
    """Blocks of normal values under power-of-two scales; `spread` varies their size."""
    g = _gen(seed)
    x = torch.randn(nb, hkv, BS, d, device="cuda", generator=g)
    x *= torch.exp2(torch.round(spread * torch.randn(nb, hkv, 1, 1, device="cuda", generator=g)))
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
    return (x / s[..., None, None]).to(FP8), s


def _tables(lens, seed, spare=3):
    per = [(n + BS - 1) // BS for n in lens]
    nb = sum(per) + spare
    ids = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).int()
    bt, at = torch.zeros(len(lens), max(per + [1]), dtype=torch.int32), 0
    for b, n in enumerate(per):
        bt[b, :n] = ids[at:at + n]
        at += n
    return bt.cuda(), nb


# ----------------------------------------------------------------------------- attention
def _attend(q, codes_k, ks, codes_v, vs, ids, ctx, limits, scale, hkv):
    """(out, bound) of rows q [R, Hq, D] of one sequence, row i seeing keys 0..limits[i]:
    64-bit attention, and how far the kernel's row may be from it."""
    R, hq, d = q.shape
    ids = ids[: (ctx + BS - 1) // BS].long()
    k = _values(codes_k[ids], ks[ids]).transpose(0, 1).reshape(hkv, -1, d)[:, :ctx]
    v = _values(codes_v[ids], vs[ids]).transpose(0, 1).reshape(hkv, -1, d)[:, :ctx]
    c = codes_v[ids].double().transpose(0, 1).reshape(hkv, -1, d)[:, :ctx].abs()
    qg = q.double().view(R, hkv, hq // hkv, d)
    w = torch.einsum("rhgd,htd->rhgt", qg, k) * scale
    size = torch.einsum("rhgd,htd->rhgt", qg.abs(), k.abs()) * scale
    seen = torch.arange(ctx, device="cuda")[None] <= limits[:, None]
    gone = ~seen[:, None, None]
    p = torch.softmax(w.masked_fill(gone, -math.inf), -1)
    out = torch.einsum("rhgt,htd->rhgd", p, v)
    mass = torch.einsum("rhgt,htd->rhgd", p, v.abs())
    worst = size.masked_fill(gone, 0).amax(-1, keepdim=True)
    rel = 2.0 ** -11 + 2 * ((d + 8) * 2.0 ** -24 * worst + 2.0 ** -21 + 2.0 ** -24 * 512) + ctx * 2.0 ** -22
    floor = 2.0 ** -25 * vs[ids].double().amax() * (c * seen.any(0)[None, :, None]).sum(1)
    bound = rel * mass + floor[None, :, None] + 2.0 ** -8 * out.abs() + 2.0 ** -120
    return out.reshape(R, hq * d), bound.reshape(R, hq * d)


def _near(got, want, bound, what):
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), what
    worst = float((off / bound).max())
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


HEADS = [(32, 8, 128), (4, 2, 64), (16, 8, 128), (8, 8, 64), (16, 1, 128), (24, 2, 64), (5, 1, 128)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode(cuda, hq, hkv, d):
    """Ragged contexts around block ends and pieces, an empty sequence, rows of wider
    tensors, dead slots that hold NaN codes, block scales that differ by powers of two."""
    lens = [1, 0, 15, 16, 17, 33, 300, 2000, 4100, 257, 512]
    B = len(lens)
    bt, nb = _tables(lens, hq + d)
    kc, ks = _quantised(nb, hkv, d, 3)
    vc, vs = _quantised(nb, hkv, d, 4, spread=3.0)
    for b, n in enumerate(lens):
        if n % BS:
            last = int(bt[b, n // BS])
            kc.view(torch.uint8)[last, :, n % BS:] = 0x7F
            vc.view(torch.uint8)[last, :, n % BS:] = 0xFF
    q = torch.randn(B, hq * d + 64, device="cuda", generator=_gen(1)).bfloat16()[:, : hq * d]
    out = torch.full((B, hq * d + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(4, _k().decode_attn_fp8_workspace_size(B, hq, d, 4100) // 4), device="cuda")
    _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, hq, hkv, d, 4100, workspace=ws)
    assert _err() == 0
    assert bool((out[:, hq * d:] == 7).all()) and bool((out[1, : hq * d] == 0).all())
    for b, n in enumerate(lens):
        if n:
            want, bound = _attend(q[b:b + 1].reshape(1, hq, d), kc, ks, vc, vs, bt[b], n, torch.tensor([n - 1], device="cuda"), d ** -0.5, hkv)
            _near(out[b:b + 1, : hq * d], want, bound, f"sequence of {n}")


@pytest.mark.parametrize("n,length", [(1, 1), (1, 37), (1, 9000), (3, 20000), (200, 700)])
def test_decode_batches(cuda, n, length):
    """From one token to long contexts, few and many sequences; two runs agree bit for bit."""
    hq, hkv, d = 32, 8, 128
    lens = [max(1, length - 7 * i) for i in range(n)]
    bt, nb = _tables(lens, n)
    kc, ks = _quantised(nb, hkv, d, 5)
    vc, vs = _quantised(nb, hkv, d, 6, spread=1.0)
    q = (3 * torch.randn(n, hq * d, device="cuda", generator=_gen(2))).bfloat16()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(4, _k().decode_attn_fp8_workspace_size(n, hq, d, length) // 4), device="cuda")
    outs = []
    for _ in range(2):
        out = torch.empty_like(q)
        _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, hq, hkv, d, length, workspace=ws)
        outs.append(out)
    assert _err() == 0 and torch.equal(outs[0], outs[1])
    for b in range(0, n, max(1, n // 9)):
        want, bound = _attend(q[b:b + 1].view(1, hq, d), kc, ks, vc, vs, bt[b], lens[b],
                              torch.tensor([lens[b] - 1], device="cuda"), d ** -0.5, hkv)
        _near(outs[0][b:b + 1], want, bound, f"sequence {b} of {lens[b]}")


@pytest.mark.parametrize("n,hq,hkv,d,length", [(2100, 4, 2, 64, 600), (70, 6, 6, 64, 900),
                                               (40, 36, 12, 128, 1500), (33, 9, 3, 128, 2000),
                                               (2048, 2, 1, 64, 300)])
def test_decode_spreads(cuda, n, hq, hkv, d, length):
    """More sequences than are cut into equal runs, head counts that leave groups of one,
    two or four heads, blocks shared by several sequences."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, length + 1, (n,), generator=g).int()
    lens[n // 2] = length
    nb = 400
    bt = torch.randint(0, nb, (n, (length + BS - 1) // BS), generator=g).int().cuda()
    kc, ks = _quantised(nb, hkv, d, 31)
    vc, vs = _quantised(nb, hkv, d, 32, spread=2.0)
    q = torch.randn(n, hq * d, device="cuda", generator=_gen(8)).bfloat16()
    out = torch.full_like(q, 7.0)
    ws = torch.empty(max(4, _k().decode_attn_fp8_workspace_size(n, hq, d, length) // 4), device="cuda")
    _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, lens.cuda(), hq, hkv, d, length, workspace=ws)
    assert _err() == 0
    for b in list(range(0, n, max(1, n // 40))) + [n // 2, n - 1]:
        ctx = int(lens[b])
        if ctx == 0:
            assert bool((out[b] == 0).all())
            continue
        want, bound = _attend(q[b:b + 1].view(1, hq, d), kc, ks, vc, vs, bt[b], ctx,
                              torch.tensor([ctx - 1], device="cuda"), d ** -0.5, hkv)
        _near(out[b:b + 1], want, bound, f"sequence {b} of {ctx}")


def test_decode_workspace_of_a_longer_bound(cuda):
    """A workspace sized for 24,016 tokens serves a launch of up to 24,000, which is cut
    into shorter runs; two streams with workspaces of their own do not disturb each other."""
    hq, hkv, d = 8, 2, 128
    lens = [24000, 5, 17000]
    bt, nb = _tables(lens, 77)
    kc, ks = _quantised(nb, hkv, d, 33)
    vc, vs = _quantised(nb, hkv, d, 34)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    size = _k().decode_attn_fp8_workspace_size(3, hq, d, 24016)
    qs = [torch.randn(3, hq * d, device="cuda", generator=_gen(i)).bfloat16() for i in (9, 10)]
    outs, wss = [torch.empty_like(q) for q in qs], [torch.empty(size // 4, device="cuda") for _ in qs]
    torch.cuda.synchronize()
    for q, out, ws, stream in zip(qs, outs, wss, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(stream):
            _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, hq, hkv, d, 24000, workspace=ws)
    torch.cuda.synchronize()
    assert _err() == 0
    for q, out in zip(qs, outs):
        for b, ctx in enumerate(lens):
            want, bound = _attend(q[b:b + 1].view(1, hq, d), kc, ks, vc, vs, bt[b], ctx,
                                  torch.tensor([ctx - 1], device="cuda"), d ** -0.5, hkv)
            _near(out[b:b + 1], want, bound, f"sequence {b}")


def test_decode_scales_and_non_finite(cuda):
    """Any positive scales, far apart; tiny and huge queries; a NaN block scale or a
    NaN query reaches its own heads and nothing else."""
    hq, hkv, d, lens = 8, 2, 128, [100, 100, 100, 100]
    bt, nb = _tables(lens, 9)
    kc, ks = _quantised(nb, hkv, d, 7)
    vc, vs = _quantised(nb, hkv, d, 8)
    vs *= torch.exp(3 * torch.randn(nb, hkv, device="cuda", generator=_gen(3)))
    ks *= 1.37
    q = torch.randn(4, hq * d, device="cuda", generator=_gen(4)).bfloat16()
    q[1] *= 2.0 ** -60
    q[2] *= 4.0
    q[2, ::3] *= 2.0 ** -20
    q[3, 5] = float("nan")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    vs[int(bt[0, 2]), 1] = float("nan")
    out = torch.empty_like(q)
    _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, hq, hkv, d, 100)
    o = out.view(4, hkv, 4, d)
    assert bool(o[0, 1].isnan().all()) and not bool(o[0, 0].isnan().any())
    assert bool(o[3, 0, 0].isnan().all()) and not bool(o[3, 0, 1:].isnan().any()) and not bool(o[3, 1].isnan().any())
    vs[int(bt[0, 2]), 1] = 1.0
    for b in (1, 2):
        want, bound = _attend(q[b:b + 1].view(1, hq, d), kc, ks, vc, vs, bt[b], 100,
                              torch.tensor([99], device="cuda"), d ** -0.5, hkv)
        _near(out[b:b + 1], want, bound, f"sequence {b}")
    assert _err() == 0


def test_decode_latches_long_contexts_and_bad_blocks(cuda):
    hq, hkv, d, lens = 32, 8, 128, [600, 100, 300, 100]
    bt, nb = _tables(lens, 17)
    kc, ks = _quantised(nb, hkv, d, 9)
    vc, vs = _quantised(nb, hkv, d, 10)
    q = torch.randn(4, hq * d, device="cuda", generator=_gen(4)).bfloat16()
    out = torch.zeros_like(q)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = torch.empty(_k().decode_attn_fp8_workspace_size(4, hq, d, 512) // 4 + 4, device="cuda")
    _k().decode_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, hq, hkv, d, 512, workspace=ws)
    assert _err() == 5 and bool((out[0] == 0).all())
    for b in (1, 2):
        want, bound = _attend(q[b:b + 1].view(1, hq, d), kc, ks, vc, vs, bt[b], lens[b],
                              torch.tensor([lens[b] - 1], device="cuda"), d ** -0.5, hkv)
        _near(out[b:b + 1], want, bound, f"sequence {b}")
    bt[3, 2] = nb  # one past the pool: read as block 0, and latched
    _k().decode_attn_fp8(q[3:], out[3:], kc, vc, ks, vs, bt[3:], sl[3:], hq, hkv, d, 112)
    assert _err() == 5


@pytest.mark.parametrize("hq,hkv,d", HEADS + [(32, 4, 128), (6, 2, 128)])
def test_prefill(cuda, hq, hkv, d):
    """Fresh prompts and continuations from one row to several tiles, an empty one between
    them, NaN codes behind the contexts, strided rows; rows behind the last sequence stay."""
    cases = [(0, 1), (0, 17), (0, 64), (5, 0), (0, 130), (20, 5), (100, 77), (700, 1), (0, 300), (1000, 140)]
    lens, qn = [p + n for p, n in cases], [n for _, n in cases]
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    T = cu[-1] + 3
    bt, nb = _tables(lens, d + hq)
    kc, ks = _quantised(nb, hkv, d, 11)
    vc, vs = _quantised(nb, hkv, d, 12, spread=2.0)
    for b, n in enumerate(lens):
        if n % BS:
            kc.view(torch.uint8)[int(bt[b, n // BS]), :, n % BS:] = 0xFF
            vc.view(torch.uint8)[int(bt[b, n // BS]), :, n % BS:] = 0x7F
    q = torch.randn(T, hq * d + 16, device="cuda", generator=_gen(2)).bfloat16()[:, : hq * d]
    out = torch.full((T, hq * d + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                          torch.tensor(cu, dtype=torch.int32, device="cuda"), max(qn), hq, hkv, d)
    assert _err() == 0
    assert bool((out[cu[-1]:] == 7).all()) and bool((out[:, hq * d:] == 7).all())
    for b, (past, n) in enumerate(cases):
        if n:
            rows = q[cu[b]:cu[b + 1]].reshape(n, hq, d)
            want, bound = _attend(rows, kc, ks, vc, vs, bt[b], lens[b],
                                  past + torch.arange(n, device="cuda"), d ** -0.5, hkv)
            _near(out[cu[b]:cu[b + 1], : hq * d], want, bound, f"{past} + {n}")


@pytest.mark.parametrize("past,n,gain", [(0, 2500, 1.0), (3000, 500, 6.0), (13, 1111, 0.01)])
def test_prefill_long(cuda, past, n, gain):
    """Long prompts and chunks, sharp and flat softmaxes, rising scores (the running maximum
    keeps moving), scales far apart; two runs agree bit for bit."""
    hq, hkv, d = 16, 4, 128
    ctx = past + n
    bt, nb = _tables([ctx], n)
    kc, ks = _quantised(nb, hkv, d, 13)
    order = torch.empty(nb, device="cuda")
    order[bt[0].long()] = torch.arange(bt.shape[1], device="cuda").float()
    ks *= torch.exp2(torch.round(order / 20).clamp_max(5))[:, None]
    vc, vs = _quantised(nb, hkv, d, 14, spread=4.0)
    q = (gain * torch.randn(n, hq * d, device="cuda", generator=_gen(5))).bfloat16()
    sl = torch.tensor([ctx], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    outs = []
    for _ in range(2):
        out = torch.empty_like(q)
        _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, cu, n, hq, hkv, d)
        outs.append(out)
    assert _err() == 0 and torch.equal(outs[0], outs[1])
    for lo in list(range(0, n, 401)) + [n - 3]:
        hi = min(lo + 5, n)
        want, bound = _attend(q[lo:hi].view(hi - lo, hq, d), kc, ks, vc, vs, bt[0], ctx,
                              past + torch.arange(lo, hi, device="cuda"), d ** -0.5, hkv)
        _near(outs[0][lo:hi], want, bound, f"rows {lo}..{hi}")


@pytest.mark.parametrize("hq,hkv,cases", [
    (4, 1, [(9000, 40), (600, 7), (1000, 1), (0, 5), (2500, 64)]),
    (2, 2, [(3844, 256), (4095, 1), (5000, 200)]),
    (16, 4, [(8000, 130), (511, 1), (1024, 64), (30000, 2)])])
def test_prefill_few_rows_long_contexts(cuda, hq, hkv, cases):
    """Launches whose key tiles are shared out over the CTAs of a cluster, each sequence
    over as many as its context is long enough for; rows that see no key of the last share;
    a NaN row and a NaN block reach nothing else; two runs agree bit for bit."""
    d = 128
    lens, qn = [p + n for p, n in cases], [n for _, n in cases]
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    bt, nb = _tables(lens, hq)
    kc, ks = _quantised(nb, hkv, d, 61, spread=1.0)
    vc, vs = _quantised(nb, hkv, d, 62, spread=3.0)
    q = torch.randn(cu[-1], hq * d, device="cuda", generator=_gen(63)).bfloat16()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    outs = []
    for _ in range(2):
        out = torch.full_like(q, 7.0)
        _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, cud, max(qn), hq, hkv, d)
        outs.append(out)
    assert _err() == 0 and torch.equal(outs[0], outs[1])
    for b, (past, n) in enumerate(cases):
        for lo in range(0, n, 64):
            hi = min(lo + 64, n)
            rows = slice(cu[b] + lo, cu[b] + hi)
            want, bound = _attend(q[rows].view(hi - lo, hq, d), kc, ks, vc, vs, bt[b], lens[b],
                                  past + torch.arange(lo, hi, device="cuda"), d ** -0.5, hkv)
            _near(outs[0][rows], want, bound, f"{past} + {n}, rows {lo}..{hi}")
    q[cu[1] - 1] = float("nan")                      # the first sequence's last row
    vs[int(bt[-1, 3])] = float("nan")                # all rows of the last one see it
    _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, cud, max(qn), hq, hkv, d)
    nan = out.isnan()
    assert bool(nan[cu[1] - 1].all()) and bool(nan[cu[-2]:].all())
    nan[cu[1] - 1] = False
    assert not bool(nan[:cu[-2]].any()) and _err() == 0


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 2, 64), (6, 2, 128), (2, 2, 64)])
def test_prefill_hidden_block_of_nan(cuda, hq, hkv, d):
    """A block whose scale is NaN reaches the rows that see a key of it and no others, also
    those whose 64-key tile holds it."""
    n, at = 200, 9                                # keys 144..159 of the tile 128..191
    bt, nb = _tables([n], 23)
    kc, ks = _quantised(nb, hkv, d, 17)
    vc, vs = _quantised(nb, hkv, d, 18)
    bad = int(bt[0, at])
    ks[bad, 0] = float("nan")
    vs[bad, 1] = float("nan")
    q = torch.randn(n, hq * d, device="cuda", generator=_gen(7)).bfloat16()
    out = torch.zeros_like(q)
    _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, torch.tensor([n], dtype=torch.int32, device="cuda"),
                          torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, hq, hkv, d)
    assert _err() == 0
    assert bool(out[16 * at:].isnan().all()) and not bool(out[:16 * at].isnan().any())
    rows = slice(130, 16 * at)
    ks[bad] = vs[bad] = 1.0
    want, bound = _attend(q[rows].view(-1, hq, d), kc, ks, vc, vs, bt[0], n,
                          torch.arange(130, 16 * at, device="cuda"), d ** -0.5, hkv)
    _near(out[rows], want, bound, "rows before the block")


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 2, 128), (8, 4, 64)])
def test_prefill_cold(cuda, hq, hkv, d):
    """Every row of prompts whose codes and scales come from memory (the L2 cache holds
    other data), each block under a scale of its own; the launch before it saw other
    scales and codes, so nothing that it left in shared memory can pass for these."""
    cases = [(0, 900), (300, 500), (0, 64), (1500, 130), (0, 1), (77, 700)]
    lens, qn = [p + n for p, n in cases], [n for _, n in cases]
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    junk = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    for turn in range(4):
        bt, nb = _tables(lens, 100 + turn)
        kc, ks = _quantised(nb, hkv, d, 40 + turn, spread=1.0 + turn)
        vc, vs = _quantised(nb, hkv, d, 50 + turn, spread=4.0 - turn)
        q = (0.2 * torch.randn(cu[-1], hq * d, device="cuda", generator=_gen(60 + turn))).bfloat16()
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out = torch.empty_like(q)
        junk.fill_(turn)
        _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, cud, max(qn), hq, hkv, d)
        assert _err() == 0
        for b, (past, n) in enumerate(cases):
            for lo in range(0, n, 128):
                hi = min(lo + 128, n)
                rows = slice(cu[b] + lo, cu[b] + hi)
                want, bound = _attend(q[rows].view(hi - lo, hq, d), kc, ks, vc, vs, bt[b], lens[b],
                                      past + torch.arange(lo, hi, device="cuda"), d ** -0.5, hkv)
                _near(out[rows], want, bound, f"turn {turn}, {past} + {n}, rows {lo}..{hi}")


def test_prefill_non_finite_and_errors(cuda):
    """A NaN block reaches only rows that see it; sequences outside the launch's sizes are
    latched and skipped, the others right."""
    hq, hkv, d = 8, 2, 128
    bt, nb = _tables([300, 300], 21)
    kc, ks = _quantised(nb, hkv, d, 15)
    vc, vs = _quantised(nb, hkv, d, 16)
    bad = int(bt[0, 10])                       # keys 160..175
    ks[bad, 0] = float("nan")
    vs[bad, 1] = float("nan")
    q = torch.randn(600, hq * d, device="cuda", generator=_gen(6)).bfloat16()
    out = torch.zeros_like(q)
    sl = torch.tensor([300, 300], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 300, 600], dtype=torch.int32, device="cuda")
    _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, sl, cu, 300, hq, hkv, d)
    assert _err() == 0
    assert not bool(out[:160].isnan().any()) and not bool(out[300:].isnan().any())
    assert bool(out[160:300].isnan().all())
    ks[bad, 0] = vs[bad, 1] = 1.0
    for lens, starts, most in (([300, 299], [0, 300, 600], 300),      # shorter than its rows
                               ([300, 300], [0, 300, 601], 301),      # rows behind the tensor
                               ([300, 9000], [0, 300, 600], 300),     # keys behind the table
                               ([300, 300], [0, 300, 600], 299)):     # more rows than max_q_len
        out.zero_()
        _k().prefill_attn_fp8(q, out, kc, vc, ks, vs, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                              torch.tensor(starts, dtype=torch.int32, device="cuda"), most, hq, hkv, d)
        assert _err() == 4
        assert bool((out[300:] == 0).all())
        if most >= 300:
            want, bound = _attend(q[200:203].view(3, hq, d), kc, ks, vc, vs, bt[0], 300,
                                  torch.arange(200, 203, device="cuda"), d ** -0.5, hkv)
            _near(out[200:203], want, bound, "the sequence beside it")


# ----------------------------------------------------------------------------- append
def _rope_tab(n, d):
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2).float() / d))
    f = torch.outer(torch.arange(n).float(), inv)
    return f.cos().cuda(), f.sin().cuda()


def _exponent(a):
    m, x = math.frexp(a)
    return -60 if a == 0 else max(-60, min(60, x - 9 + (m > 0.875)))


def _rotated(qkv, pos, cos, sin, hq, hkv, d, qn, kn, dtype):
    """q, k (rotated) and v [T, heads, D]; in f32 with the kernel's steps, or in f64."""
    x = qkv.to(dtype).view(qkv.shape[0], hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    c, s = cos[pos.long()].to(dtype)[:, None], sin[pos.long()].to(dtype)[:, None]

    def norm(t, w):
        if w is None:
            return t
        inv = 1 / (t.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
        return w.to(dtype) * (t * inv.to(dtype))

    def rope(t):
        a, b = t[..., : d // 2], t[..., d // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    return rope(norm(q, qn)), rope(norm(k, kn)), v


def _store(x, codes, scale, slots):
    """The append's definition, block by block, on CPU tensors; x [T, Hkv, D] f32."""
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        blk, run = slots[t] // BS, []
        while t < len(slots) and slots[t] >= 0 and slots[t] // BS == blk:
            run.append(t)
            t += 1
        rows = {slots[r] % BS: r for r in run}          # the last one naming a slot counts
        for h in range(x.shape[1]):
            new = torch.stack([x[r, h] for r in rows.values()])
            e = _exponent(float(new.abs().max()))
            if 0 not in rows:
                e_old = math.frexp(float(scale[blk, h]))[1] - 1
                if e > e_old:
                    codes[blk, h] = (codes[blk, h].float() * 2.0 ** (e_old - e)).to(FP8)
                e = max(e, e_old)
            for o, r in rows.items():
                codes[blk, h, o] = (x[r, h] * 2.0 ** -e).to(FP8)
            scale[blk, h] = 2.0 ** e


def _same_codes(got, want):
    """Equal numbers (+0 and -0 are one)."""
    return torch.equal(got.float(), want.float())


APPENDS = {
    # decode rows in the middle of blocks, padding rows, position 0 of a block
    "decode": lambda r: ([(17 + 16 * i + r % 16, 1) for i, r in enumerate(range(0, 90, 3))], True),
    "prompts": lambda r: ([(0, 1), (0, 16), (0, 45), (7, 9), (7, 10), (31, 70), (0, 33)], True),
    "one": lambda r: ([(5, 1)], False),
    "long": lambda r: ([(0, 700), (33, 1), (15, 1), (100, 613)], True),
}


@pytest.mark.parametrize("kind", APPENDS)
@pytest.mark.parametrize("hq,hkv,d,qk", [(32, 8, 128, False), (4, 2, 64, True), (5, 1, 128, True), (9, 9, 64, False)])
def test_append(cuda, kind, hq, hkv, d, qk):
    spans, pad = APPENDS[kind](0)
    lens = [p + n for p, n in spans]
    bt, nb = _tables(lens, d)
    pos, slots = [], []
    for b, (p, n) in enumerate(spans):
        for i in range(p, p + n):
            pos.append(i)
            slots.append(int(bt[b, i // BS]) * BS + i % BS)
        if pad and b % 2:
            pos.append(0)
            slots.append(-1)
    T = len(pos)
    g = _gen(d + hq)
    wide = torch.randn(T, (hq + 2 * hkv) * d + 24, device="cuda", generator=g)
    wide *= torch.exp(1.2 * torch.randn(T, 1, device="cuda", generator=g))
    qkv = wide.bfloat16()[:, : (hq + 2 * hkv) * d]
    qkv[:, -d:] *= (torch.arange(T, device="cuda") % 5 > 0)[:, None]        # zero rows of the last v head
    kc, ks = _quantised(nb, hkv, d, 1)
    vc, vs = _quantised(nb, hkv, d, 2)
    cos, sin = _rope_tab(max(lens) + 1, d)
    qn = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if qk else None
    kn = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if qk else None
    P, S = torch.tensor(pos, dtype=torch.int32, device="cuda"), torch.tensor(slots, dtype=torch.int32, device="cuda")
    qr, kr, vr = _rotated(qkv, P, cos, sin, hq, hkv, d, qn, kn, torch.float32)
    q64, k64, v64 = _rotated(qkv, P, cos, sin, hq, hkv, d, qn, kn, torch.float64)
    want = []
    for c, s, x in ((kc, ks, kr), (vc, vs, vr)):
        c2, s2 = c.cpu(), s.cpu()
        _store(x.cpu().contiguous(), c2, s2, slots)
        want.append((c2, s2))
    before = qkv.clone()
    q_out = torch.full((T, hq * d + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    _k().rope_kv_append_fp8(qkv, P, S, cos, sin, hq, hkv, d, kc, vc, ks, vs, qn, kn, 1e-6, q_out=q_out)
    assert _err() == 0
    assert torch.equal(qkv, before) and bool((q_out[:, hq * d:] == 7).all())
    assert torch.equal(q_out[:, : hq * d], qr.reshape(T, -1).bfloat16())
    for (c, s), (c2, s2) in zip(((kc, ks), (vc, vs)), want):
        assert torch.equal(s.cpu(), s2)
        assert _same_codes(c.cpu(), c2)
    # against 64 bits: one rounding of each new row
    off = (q_out[:, : hq * d].double() - q64.reshape(T, -1)).abs()
    near = 2.0 ** -8 * q64.reshape(T, -1).abs() + 2.0 ** -20 * q64.abs().amax()
    assert bool((off <= near).all())
    live = [t for t in range(T) if slots[t] >= 0]
    at = torch.tensor([slots[t] for t in live], device="cuda")
    for c, s, x in ((kc, ks, k64), (vc, vs, v64)):
        got = _values(c, s)[at // BS, :, at % BS]
        sc = s[at // BS].double()[..., None]
        ref = x[live]
        bound = 2.0 ** -4 * ref.abs() + 2.0 ** -10 * sc + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True)
        assert bool(((got - ref).abs() <= bound).all())
    # in place: q lands in the batch's own rows, k and v rows stay
    k2, v2, ks2, vs2 = kc.clone(), vc.clone(), ks.clone(), vs.clone()
    _k().rope_kv_append_fp8(qkv, P, S, cos, sin, hq, hkv, d, k2, v2, ks2, vs2, qn, kn)
    assert torch.equal(qkv[:, : hq * d], q_out[:, : hq * d]) and torch.equal(qkv[:, hq * d:], before[:, hq * d:])
    # the same rows again change nothing
    assert _same_codes(k2, kc) and _same_codes(v2, vc) and torch.equal(ks2, ks) and torch.equal(vs2, vs)


def test_append_borders_and_repeats(cuda):
    """Exponents at their borders, zero and tiny rows, a slot named twice, non-finite rows."""
    hq, hkv, d = 2, 1, 64
    cos, sin = torch.ones(4, d // 2, device="cuda"), torch.zeros(4, d // 2, device="cuda")
    tops = [448.0, 450.0, 447.0, 0.0, 2.0 ** -75, 1.75 * 2.0 ** 80, 3.0e38, 1.0]
    T = len(tops)
    qkv = torch.zeros(T, 4 * d, device="cuda", dtype=torch.bfloat16)
    for t, a in enumerate(tops):
        qkv[t, 2 * d + 3] = a           # k
        qkv[t, 3 * d + 9] = -a          # v
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    slots = torch.arange(T, dtype=torch.int32, device="cuda") * BS
    kc = torch.zeros(T + 1, 1, BS, d, device="cuda").to(FP8)
    vc, ks = kc.clone(), torch.full((T + 1, 1), 2.0 ** 30, device="cuda")
    vs = ks.clone()
    _k().rope_kv_append_fp8(qkv, pos, slots, cos, sin, hq, hkv, d, kc, vc, ks, vs)
    a32 = qkv[:, 2 * d + 3].float().tolist()
    assert ks[:T, 0].tolist() == vs[:T, 0].tolist() == [2.0 ** _exponent(a) for a in a32]
    assert ks[0, 0] == 1.0 and ks[1, 0] == 2.0 and ks[3, 0] == 2.0 ** -60 and ks[6, 0] == 2.0 ** 60
    for t, a in enumerate(a32):
        want = max(-448.0, min(448.0, a / float(ks[t, 0])))
        assert float(kc[t, 0, 0, 3]) == float(torch.tensor(want).to(FP8))
        assert float(vc[t, 0, 0, 9]) == -float(kc[t, 0, 0, 3])
    # 20 neighbouring rows of one block: of those naming a slot the last counts
    qkv = torch.randn(20, 4 * d, device="cuda", generator=_gen(1)).bfloat16()
    offs = [0, 1, 1, 2, 5, 5, 5, 3, 4, 0, 7, 8, 9, 10, 11, 12, 12, 13, 14, 15]
    sl = torch.tensor([T * BS + o for o in offs], dtype=torch.int32, device="cuda")
    _k().rope_kv_append_fp8(qkv, torch.zeros(20, dtype=torch.int32, device="cuda"), sl, cos, sin, hq, hkv, d,
                            kc, vc, ks, vs)
    for o, r in {o: r for r, o in enumerate(offs)}.items():
        ref = qkv[r, 3 * d:].double()
        got = _values(vc, vs)[T, 0, o]
        # a later group of rows may have grown the scale: two roundings
        assert bool(((got - ref).abs() <= 2 * 2.0 ** -4 * 1.07 * ref.abs() + 2 * 2.0 ** -10 * float(vs[T, 0])).all())
    # infinities and NaN: the block and head read NaN until the block starts anew
    row = torch.ones(1, 4 * d, device="cuda").bfloat16()
    for bad in (float("inf"), float("nan")):
        row[0, 3 * d + 1] = bad
        one = torch.zeros(1, dtype=torch.int32, device="cuda")
        _k().rope_kv_append_fp8(row, one, one + 1, cos, sin, hq, hkv, d, kc, vc, ks, vs)
        assert bool(vs[0, 0].isnan()) and not bool(ks[0, 0].isnan()) and not bool(vc.float().isnan().any())
        row[0, 3 * d + 1] = 1.0
        _k().rope_kv_append_fp8(row, one, one + 2, cos, sin, hq, hkv, d, kc, vc, ks, vs)
        assert bool(vs[0, 0].isnan())
        _k().rope_kv_append_fp8(row, one, one, cos, sin, hq, hkv, d, kc, vc, ks, vs)
        assert float(vs[0, 0]) == 2.0 ** -8
    assert _err() == 0


def test_append_latches_bad_positions_and_slots(cuda):
    hq, hkv, d = 4, 2, 64
    cos, sin = _rope_tab(8, d)
    qkv = torch.randn(4, 8 * d, device="cuda", generator=_gen(3)).bfloat16()
    kc, ks = _quantised(4, hkv, d, 1)
    vc, vs = _quantised(4, hkv, d, 2)
    k0, v0 = kc.clone(), vc.clone()
    for pos, slots in (([0, 8, 1, 2], [0, -1, -1, -1]), ([0, 1, -1, 2], [-1, -1, 16, -1]),
                       ([0, 1, 2, 3], [-1, 64, -1, -1])):
        q = qkv.clone()
        _k().rope_kv_append_fp8(q, torch.tensor(pos, dtype=torch.int32, device="cuda"),
                                torch.tensor(slots, dtype=torch.int32, device="cuda"), cos, sin, hq, hkv, d,
                                kc, vc, ks, vs)
        assert _err() == 5
    assert torch.equal(kc[2:].view(torch.uint8), k0[2:].view(torch.uint8))
    assert torch.equal(vc[2:].view(torch.uint8), v0[2:].view(torch.uint8))
    assert torch.equal(kc[1].view(torch.uint8), k0[1].view(torch.uint8))      # its position was bad


# ----------------------------------------------------------------------------- pages
@pytest.mark.parametrize("dtype", [FP8, torch.bfloat16])
@pytest.mark.parametrize("shape,n", [((3, 2, 40, 2, 16, 64), 1), ((1, 2, 1300, 1, 16, 64), 600),
                                     ((2, 2, 64, 8, 16, 128), 31), ((5, 37, 3, 16, 128), 18)])
def test_copy_pages(cuda, dtype, shape, n):
    g = _gen(n)
    pool = torch.randn(shape, device="cuda", generator=g).to(dtype)
    scales = torch.rand(shape[:-2], device="cuda", generator=g)
    ids = torch.randperm(shape[-4], generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    if n > 2:
        src[2] = src[0]            # one source, several destinations
    want, ws = pool.view(torch.uint8).clone(), scales.clone()
    dim = pool.dim() - 4
    want.index_copy_(dim, torch.tensor(dst, device="cuda"), want.index_select(dim, torch.tensor(src, device="cuda")))
    ws.index_copy_(dim, torch.tensor(dst, device="cuda"), ws.index_select(dim, torch.tensor(src, device="cuda")))
    s0 = scales.clone()
    _k().copy_pages(pool, src, dst)
    assert torch.equal(pool.view(torch.uint8), want) and torch.equal(scales, s0)
    _k().copy_pages(pool, src, dst, scales=scales)
    assert torch.equal(pool.view(torch.uint8), want) and torch.equal(scales, ws)
    _k().copy_pages(pool, [], [])


# ----------------------------------------------------------------------------- together
def _step(k, state, rows, pos, slots, ctx, bt, hq, hkv, d):
    """Append then attend, as a decode step of a layer does."""
    kc, vc, ks, vs, cos, sin, ws = state
    q = torch.empty(rows.shape[0], hq * d, device="cuda", dtype=torch.bfloat16)
    k.rope_kv_append_fp8(rows, pos, slots, cos, sin, hq, hkv, d, kc, vc, ks, vs, q_out=q)
    out = torch.empty_like(q)
    k.decode_attn_fp8(q, out, kc, vc, ks, vs, bt, ctx, hq, hkv, d, 256, workspace=ws)
    return q, out


def test_operators_together(cuda):
    """A prompt is prefilled, its request forked (the last, partly filled block copied with
    its scales), and both copies decode on their own for 20 steps, across a block's end."""
    k = _k()
    hq, hkv, d, n = 8, 2, 128, 75
    kc, vc = (torch.zeros(12, hkv, BS, d, device="cuda").to(FP8) for _ in range(2))
    pool = torch.stack([kc, vc])
    scales = torch.zeros(2, 12, hkv, device="cuda")
    kc, vc, ks, vs = pool[0], pool[1], scales[0], scales[1]
    cos, sin = _rope_tab(200, d)
    ws = torch.empty(max(4, k.decode_attn_fp8_workspace_size(2, hq, d, 256) // 4), device="cuda")
    bt = torch.zeros(2, 16, dtype=torch.int32)
    bt[0, :6] = torch.tensor([7, 2, 9, 4, 0, 11])
    bt[1, :6] = torch.tensor([7, 2, 9, 4, 5, 3])
    g = _gen(8)
    prompt = torch.randn(n, (hq + 2 * hkv) * d, device="cuda", generator=g).bfloat16()
    pos = torch.arange(n, dtype=torch.int32)
    slots = bt[0, pos.long() // BS] * BS + pos % BS
    q = torch.empty(n, hq * d, device="cuda", dtype=torch.bfloat16)
    k.rope_kv_append_fp8(prompt, pos.cuda(), slots.cuda(), cos, sin, hq, hkv, d, kc, vc, ks, vs, q_out=q)
    out = torch.empty_like(q)
    one = torch.tensor([n], dtype=torch.int32, device="cuda")
    k.prefill_attn_fp8(q, out, kc, vc, ks, vs, bt[:1].cuda(), one, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                       n, hq, hkv, d)
    want, bound = _attend(q.view(n, hq, d), kc, ks, vc, vs, bt[0].cuda(), n, torch.arange(n, device="cuda"), d ** -0.5, hkv)
    _near(out, want, bound, "prompt")
    k.copy_pages(pool, [0], [5], scales=scales)
    assert torch.equal(kc[5].view(torch.uint8), kc[0].view(torch.uint8)) and torch.equal(vs[5], vs[0])
    btd = bt.cuda()
    state = (kc, vc, ks, vs, cos, sin, ws)
    for i in range(20):
        at = n + i
        rows = torch.randn(2, (hq + 2 * hkv) * d, device="cuda", generator=g).bfloat16() * (1 + i % 4)
        p = torch.full((2,), at, dtype=torch.int32, device="cuda")
        s = (bt[:, at // BS] * BS + at % BS).cuda()
        ctx = p + 1
        q, out = _step(k, state, rows, p, s, ctx, btd, hq, hkv, d)
        for b in range(2):
            want, bound = _attend(q[b:b + 1].view(1, hq, d), kc, ks, vc, vs, btd[b], at + 1,
                                  torch.tensor([at], device="cuda"), d ** -0.5, hkv)
            _near(out[b:b + 1], want, bound, f"step {i} of copy {b}")
    assert not torch.equal(kc[5].view(torch.uint8), kc[0].view(torch.uint8))
    assert _err() == 0


def test_captured_steps_and_side_streams(cuda):
    """A captured decode step replays with new inputs in its buffers, padded rows included, and
    equals the eager one bit for bit; two captured steps with a workspace each run side by side."""
    k = _k()
    hq, hkv, d, B = 32, 8, 128, 4
    cos, sin = _rope_tab(700, d)

    def fresh(seed):
        lens = [600, 77, 1]
        bt, nb = _tables([n + BS for n in lens], seed)
        kc, ks = _quantised(nb, hkv, d, seed)
        vc, vs = _quantised(nb, hkv, d, seed + 1)
        bt = torch.cat([bt, torch.zeros(1, bt.shape[1], dtype=torch.int32, device="cuda")])  # a padding row
        pos = torch.tensor(lens + [0], dtype=torch.int32, device="cuda")
        slots = bt.gather(1, (pos.long() // BS)[:, None])[:, 0] * BS + pos % BS
        slots[3] = -1
        ctx = pos + 1
        ctx[3] = 0
        qkv = torch.randn(B, (hq + 2 * hkv) * d, device="cuda", generator=_gen(seed)).bfloat16()
        ws = torch.empty(k.decode_attn_fp8_workspace_size(B, hq, d, 624) // 4 + 4, device="cuda")
        return dict(bt=bt, kc=kc, ks=ks, vc=vc, vs=vs, pos=pos, slots=slots, ctx=ctx, qkv=qkv, ws=ws,
                    q=torch.empty(B, hq * d, device="cuda", dtype=torch.bfloat16),
                    out=torch.empty(B, hq * d, device="cuda", dtype=torch.bfloat16))

    def run(s):
        k.rope_kv_append_fp8(s["qkv"], s["pos"], s["slots"], cos, sin, hq, hkv, d, s["kc"], s["vc"], s["ks"],
                             s["vs"], q_out=s["q"])
        k.decode_attn_fp8(s["q"], s["out"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["ctx"], hq, hkv, d, 624,
                          workspace=s["ws"])

    runs, graphs, streams = [fresh(31), fresh(41)], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in runs:
        run(s)                                       # eager once, before any capture
    torch.cuda.synchronize()
    for s in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(s)
        graphs.append(graph)
    for i, s in enumerate(runs):                     # new inputs in the same buffers
        t = fresh(51 + 10 * i)
        for name in ("kc", "vc"):
            s[name].view(torch.uint8).copy_(t[name].view(torch.uint8))
        for name in ("bt", "ks", "vs", "pos", "slots", "ctx", "qkv"):
            s[name].copy_(t[name])
    torch.cuda.synchronize()
    for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for i, s in enumerate(runs):
        t = fresh(51 + 10 * i)
        run(t)
        assert torch.equal(s["out"], t["out"]) and torch.equal(s["ks"], t["ks"]) and torch.equal(s["vs"], t["vs"])
        assert torch.equal(s["kc"].view(torch.uint8), t["kc"].view(torch.uint8))
        assert torch.equal(s["vc"].view(torch.uint8), t["vc"].view(torch.uint8))
        assert bool((t["out"][3] == 0).all())
    assert _err() == 0


@pytest.mark.parametrize("hq,hkv,d,n", [(16, 8, 128, 40), (8, 8, 64, 20)])
def test_blocks_behind_32_bit_offsets(cuda, hq, hkv, d, n):
    """The last blocks of a cache of more than 2^32 bytes give the bits that the same blocks
    of a small cache give: append, decode, prefill, copies."""
    big = (1 << 32) // (hkv * BS * d) + 8
    per = (n + BS - 1) // BS
    qkv = torch.randn(n, (hq + 2 * hkv) * d, device="cuda", generator=_gen(71)).bfloat16()
    cos, sin = _rope_tab(64, d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    results = []
    for nb in (big, 8):
        kc, vc = (torch.zeros(nb, hkv, BS, d, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
        ks, vs = (torch.ones(nb, hkv, device="cuda") for _ in range(2))
        bt = torch.arange(nb - 1, nb - 1 - per, -1, dtype=torch.int32, device="cuda")[None]
        slots = bt[0].long()[pos.long() // BS] * BS + pos.long() % BS
        q = torch.empty(n, hq * d, dtype=torch.bfloat16, device="cuda")
        _k().rope_kv_append_fp8(qkv, pos, slots.int(), cos, sin, hq, hkv, d, kc, vc, ks, vs, q_out=q)
        sl = torch.tensor([n], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        dec, pre = torch.empty_like(q[:1]), torch.empty_like(q)
        _k().decode_attn_fp8(q[n - 1:], dec, kc, vc, ks, vs, bt, sl, hq, hkv, d, per * BS)
        _k().prefill_attn_fp8(q, pre, kc, vc, ks, vs, bt, sl, cu, n, hq, hkv, d)
        _k().copy_pages(kc, [nb - 1], [0], scales=ks)
        assert _err() == 0
        results.append((dec, pre, kc.view(torch.uint8)[bt[0].long()], ks[bt[0].long()],
                        vc.view(torch.uint8)[bt[0].long()], kc.view(torch.uint8)[0], ks[0]))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert bool(results[0][2].any()) and torch.equal(results[0][2][0], results[0][5])
