"""The 8-bit append over unusual steps: many rows of one block, large steps of decode rows
and prompts together.  Codes, scales and q rows have to equal the definition's, in the f32
steps of test_fp8_cache_gpu."""

import pytest
import torch

from test_fp8_cache_gpu import (BS, _err, _gen, _k, _quantised, _rope_tab, _rotated, _same_codes,
                                _store)

pytestmark = pytest.mark.gpu


def _append(pos, slots, nb, hq, hkv, d, seed=1, qk=False):
    g = _gen(seed)
    T = len(pos)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, device="cuda", generator=g)
    qkv = (qkv * torch.exp(1.5 * torch.randn(T, 1, device="cuda", generator=g))).bfloat16()
    kc, ks = _quantised(nb, hkv, d, seed + 1)
    vc, vs = _quantised(nb, hkv, d, seed + 2)
    cos, sin = _rope_tab(max(pos) + 1, d)
    w = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if qk else None
    P = torch.tensor(pos, dtype=torch.int32, device="cuda")
    S = torch.tensor(slots, dtype=torch.int32, device="cuda")
    q, k, v = _rotated(qkv, P, cos, sin, hq, hkv, d, w, w, torch.float32)
    want = []
    for c, s, x in ((kc, ks, k), (vc, vs, v)):
        c2, s2 = c.cpu(), s.cpu()
        _store(x.cpu().contiguous(), c2, s2, slots)
        want.append((c2, s2))
    _k().rope_kv_append_fp8(qkv, P, S, cos, sin, hq, hkv, d, kc, vc, ks, vs, w, w)
    assert _err() == 0
    assert torch.equal(qkv[:, : hq * d], q.reshape(T, -1).bfloat16())
    for (c, s), (c2, s2) in zip(((kc, ks), (vc, vs)), want):
        assert torch.equal(s.cpu(), s2)
        assert _same_codes(c.cpu(), c2)


RUNS = {
    "row 0 again": [*range(16), 0],
    "row 0 late": [*range(1, 16), 1, 2, 0],
    "without row 0": [*range(3, 16), *range(3, 16)],
    "one slot": [5] * 40,
    "falling": [*range(15, -1, -1), *range(15, 7, -1)],
    "long": [(7 * i) % 16 for i in range(100)],
    "exactly 32": [*range(16), *range(16)],
    "exactly 64": [(3 * i) % 16 for i in range(64)],
}


@pytest.mark.parametrize("run", RUNS)
@pytest.mark.parametrize("before,after", [(0, 0), (5, 3), (15, 1), (31, 40), (0, 1100)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (4, 1, 128), (16, 8, 128)])
def test_many_rows_of_one_block(cuda, hq, hkv, d, before, after, run):
    """More neighbouring rows than the block has, some slots named again: of the rows naming
    a slot the last counts, wherever the run lies in the step."""
    offs = RUNS[run]
    nb = 2 + (before + BS - 1) // BS + (after + BS - 1) // BS
    first = (before + BS - 1) // BS
    slots = list(range(before)) + [first * BS + o for o in offs] + \
        [(first + 1) * BS + i for i in range(after)]
    _append([i % 50 for i in range(len(slots))], slots, nb, hq, hkv, d, qk=after == 3)


@pytest.mark.parametrize("hq,hkv,d,qk", [(32, 8, 128, False), (4, 2, 64, True)])
@pytest.mark.parametrize("decode,prompts", [(700, [(0, 300), (33, 200)]), (256, [(7, 800)]),
                                            (1025, []), (1100, [(0, 1), (15, 2)]), (1024, [])])
def test_decode_rows_and_prompts_of_a_large_step(cuda, hq, hkv, d, qk, decode, prompts):
    """The engine's step: decode rows, each alone in its block, before pieces of prompts, at
    and around the size from which rows are spread in another way."""
    pos, slots, blk = [], [], 0
    for i in range(decode):
        pos.append(40 + i % 16)
        slots.append(blk * BS + (40 + i) % BS)
        blk += 1
    for past, n in prompts:
        for p in range(past, past + n):
            pos.append(p)
            slots.append((blk + p // BS) * BS + p % BS)
        blk += (past + n) // BS + 1
    _append(pos, slots, blk + 1, hq, hkv, d, seed=decode, qk=qk)
