"""Cases of the 8-bit paged KV cache: its append, the two attentions that read it and the copies of its pages.

A layer's cache is two arrays [num_blocks][num_kv_heads][16][head_dim] of e4m3 codes (K and V) and one f32 scale for each
block and head in arrays [num_blocks][num_kv_heads]; a cached value is code x scale.

Formulas (B sequences, T new tokens, Hq query heads in groups of G = Hq / Hkv, head size D):

  append    k = rope(qk_norm?(k_in)), v = v_in. For each block p and head h that gets rows R in this call: a = the largest
            finite |x| of R, e = the smallest exponent with a <= 448 2^e, held to [-60, 60]. A block whose row 0 is in R
            starts anew; any other keeps its rows: with its old exponent e0 its new one is max(e, e0) and, where that grew,
            its codes become e4m3(code 2^(e0 - e)). The new rows are e4m3(x 2^-e), the scale is 2^e. q = rope(qk_norm?(q_in)).
  decode    out[b, h] = sum_t softmax_t(scale q[b, h] . K[t]) V[t] over the first seq_lens[b] cached tokens; zeros for none.
  prefill   the same for each new row i of a sequence, which sits at position seq_lens[b] - q_len[b] + i and sees the keys
            up to and with its own.
  pages     pool[layer, k or v, dst[i]] = pool[layer, k or v, src[i]], and the same for the scales.

The codes are returned as float8 tensors, which are the numbers that the codes stand for, each with its block's scale beside
it: the cache of a user's program holds just these two arrays, so nothing is converted for the comparison.
"""

import math
import os
import random
import sys

import torch

own = False

BS = 16          # tokens of a block
E4M3 = torch.float8_e4m3fn
EXP_LO, EXP_HI = -60, 60
THETA = 500000.0
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    big = {"hq": 32, "hkv": 8, "d": 128}       # the 8B Llama shape of the benchmark
    tiny = {"hq": 4, "hkv": 2, "d": 64}        # the tiny models of the tests
    return [
        # one token of one request of a tiny model: launch latency alone
        {"name": "append 1 token tiny", "op": "append", **tiny, "rows": "decode", "n": 1, "lo": 40, "hi": 40, "qk": True, "mix": 1},
        # a decode step of the benchmark's running batch: every row lands inside a block that others have filled
        {"name": "append 256 decode rows", "op": "append", **big, "rows": "decode", "n": 256, "lo": 200, "hi": 1500, "qk": False, "mix": 2},
        # a full prefill step: ragged prompts and chunks, nearly all blocks new, QK-norm on as in the Deep models
        {"name": "append 8k prefill rows", "op": "append", **big, "rows": "prefill", "n": 11, "lo": 201, "hi": 1291, "qk": True, "mix": 3},
        # one request in its first tokens
        {"name": "decode 1 seq tiny", "op": "decode", **tiny, "n": 1, "lo": 37, "hi": 37, "mix": 4},
        # the benchmark's running batch: 256 requests of a few hundred to 1,500 tokens
        {"name": "decode 256 seqs 1.5k", "op": "decode", **big, "n": 256, "lo": 200, "hi": 1500, "mix": 5},
        # long contexts, few requests: the work of one sequence has to be spread
        {"name": "decode 32 seqs 32k", "op": "decode", **big, "n": 32, "lo": 1024, "hi": 32768, "mix": 6},
        # three short prompts of a tiny model
        {"name": "prefill 3 prompts tiny", "op": "prefill", **tiny, "n": 3, "q_lo": 5, "q_hi": 41, "past_lo": 0, "past_hi": 0, "mix": 7},
        # one fresh 4,000-token prompt, the longest of the benchmark
        {"name": "prefill 4000 fresh", "op": "prefill", **big, "n": 1, "q_lo": 4000, "q_hi": 4000, "past_lo": 0, "past_hi": 0, "mix": 8},
        # chunked prefill: pieces of prompts behind what is cached of them, 16 query heads on 8 (the Deep shape)
        {"name": "prefill 4 chunks 8k", "op": "prefill", "hq": 16, "hkv": 8, "d": 128, "n": 4, "q_lo": 300, "q_hi": 700, "past_lo": 1500, "past_hi": 8000, "mix": 9},
        # forking one request of a tiny model: its last block, two layers
        {"name": "pages fork 1 tiny", "op": "pages", "hkv": 2, "d": 64, "layers": 2, "blocks": 64, "n": 1, "bits": 8, "mix": 10},
        # forking 64 requests of the 8B shape: each last block in all 32 layers
        {"name": "pages fork 64", "op": "pages", "hkv": 8, "d": 128, "layers": 32, "blocks": 512, "n": 64, "bits": 8, "mix": 11},
        # compacting a pool: 600 scattered blocks move to the front, 16-bit cache
        {"name": "pages compact 600", "op": "pages", "hkv": 8, "d": 128, "layers": 12, "blocks": 2000, "n": 600, "bits": 16, "mix": 12},
    ]


HEADS = [(32, 8, 128), (16, 8, 128), (32, 4, 128), (16, 1, 128), (4, 4, 128), (4, 2, 64), (8, 8, 64), (16, 2, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "pages"])
    hq, hkv, d = rng.choice(HEADS)
    c = {"op": op, "hq": hq, "hkv": hkv, "d": d, "mix": rng.randrange(1 << 20)}
    if op == "append":
        if rng.random() < 0.5:
            lo = _log(rng, 1, 3000)
            return {**c, "rows": "decode", "n": _log(rng, 1, 300), "lo": lo, "hi": lo + _log(rng, 1, 2000), "qk": rng.random() < 0.5}
        lo = _log(rng, 1, 900)
        return {**c, "rows": "prefill", "n": _log(rng, 1, 9), "lo": lo, "hi": min(900, lo + _log(rng, 1, 900)), "qk": rng.random() < 0.5}
    if op == "decode":
        hi = _log(rng, 2, 32768)
        n = max(1, min(_log(rng, 1, 300), 500000 // hi))
        return {**c, "n": n, "lo": _log(rng, 1, hi), "hi": hi}
    if op == "prefill":
        q = _log(rng, 2, 2800)
        past = min(_log(rng, 1, 6000), 8000000 // q - q) if rng.random() < 0.5 else 0
        n = max(1, min(_log(rng, 1, 8), 8000000 // (q * (q + past))))
        return {**c, "n": n, "q_lo": max(1, q // 3), "q_hi": q, "past_lo": past // 3, "past_hi": past}
    layers, n = _log(rng, 1, 32), _log(rng, 1, 300)
    n = max(1, min(n, 7000 // layers))
    return {"op": op, "hkv": hkv, "d": d, "layers": layers, "blocks": 2 * n + _log(rng, 1, 200), "n": n, "bits": rng.choice([8, 16]), "mix": c["mix"]}


def _lens(c):
    """The ragged lengths of a case, made from its own numbers: (cached tokens before the call, new rows) of each sequence."""
    r = random.Random(c["mix"])
    if c["op"] == "prefill":
        q = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["n"])]
        return [(r.randint(c["past_lo"], c["past_hi"]), x) for x in q]
    if c["op"] == "append" and c["rows"] == "prefill":
        n = [r.randint(c["lo"], c["hi"]) for _ in range(c["n"])]
        return [(0 if r.random() < 0.7 else r.randint(1, 2000), x) for x in n]
    return [(r.randint(c["lo"], c["hi"]) - 1, 1) for _ in range(c["n"])]


def work(c):
    if c["op"] == "pages":
        page = c["hkv"] * BS * c["d"] * (c["bits"] // 8) + (4 * c["hkv"] if c["bits"] == 8 else 0)
        return {"bytes": 2 * c["n"] * c["layers"] * 2 * page, "flops": 0}
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    lens = _lens(c)
    rows = sum(n for _, n in lens)
    if c["op"] == "append":
        blocks = sum((p + n + BS - 1) // BS - p // BS for p, n in lens)
        moved = rows * ((hq + 2 * hkv) * d * 2 + d * 4 + 8 + hq * d * 2 + 2 * hkv * d) + blocks * 2 * hkv * 4
        return {"bytes": moved, "flops": rows * (hq + 2 * hkv) * d * 4}
    tokens = sum(p + n for p, n in lens)
    blocks = sum((p + n + BS - 1) // BS for p, n in lens)
    moved = tokens * 2 * hkv * d + blocks * (2 * hkv * 4 + 4) + rows * hq * d * 4
    seen = sum(n * p + n * (n + 1) // 2 for p, n in lens)
    return {"bytes": moved, "flops": 4 * seen * hq * d}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _blocks(nb, hkv, d, g):
    """Quantised blocks as an earlier append left them: normal values with a few strong channels, and their scales."""
    x = torch.randn(nb, hkv, BS, d, device="cuda", generator=g)
    gain = torch.exp(0.7 * torch.randn(hkv, 1, d, device="cuda", generator=g))
    x *= gain
    amax = x.abs().amax((2, 3))
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
    return (x / scale[:, :, None, None]).to(E4M3), scale


def _tables(max_pos, d):
    inv = 1.0 / (THETA ** (torch.arange(0, d, 2, device="cuda").float() / d))
    f = torch.outer(torch.arange(max_pos, device="cuda").float(), inv)
    return f.cos().contiguous(), f.sin().contiguous()


def prepare(c, seed):
    g = _gen(seed)
    if c["op"] == "pages":
        shape = (c["layers"], 2, c["blocks"], c["hkv"], BS, c["d"])
        pool = torch.randn(shape, device="cuda", generator=g).to(E4M3 if c["bits"] == 8 else torch.bfloat16)
        scales = torch.exp2(torch.randint(-9, -3, shape[:4], device="cuda", generator=g).float()) if c["bits"] == 8 else None
        ids = list(range(c["blocks"]))
        random.Random(seed).shuffle(ids)
        src, dst = ids[: c["n"]], ids[c["n"]: 2 * c["n"]]
        return {"op": "pages", "pool": pool, "scales": scales, "src": src, "dst": dst}
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    lens = _lens(c)
    ctx = [p + n for p, n in lens]
    # an append needs the blocks that its rows land in, the attentions every block of a sequence
    base = [p // BS if c["op"] == "append" else 0 for p, _ in lens]
    per = [(x + BS - 1) // BS - b for x, b in zip(ctx, base)]
    nb = sum(per) + 3
    ids = list(range(nb))
    random.Random(seed).shuffle(ids)
    bt, at = torch.zeros(len(lens), max(per), dtype=torch.int32), 0
    for b, n in enumerate(per):
        bt[b, :n] = torch.tensor(ids[at: at + n], dtype=torch.int32)
        at += n
    kc, ks = _blocks(nb, hkv, d, g)
    vc, vs = _blocks(nb, hkv, d, g)
    s = {"op": c["op"], "hq": hq, "hkv": hkv, "d": d, "kc": kc, "vc": vc, "ks": ks, "vs": vs}
    rows = sum(n for _, n in lens)
    if c["op"] == "append":
        pos = torch.cat([torch.arange(p, p + n) for p, n in lens])
        seq = torch.cat([torch.full((n,), b) for b, (_, n) in enumerate(lens)])
        slots = bt[seq, pos // BS - torch.tensor(base)[seq]].long() * BS + pos % BS
        qkv = torch.randn(rows, hq + 2 * hkv, d, device="cuda", generator=g)
        # rows of different strength, so that some new rows outgrow their block's scale and others do not
        qkv *= torch.exp(0.8 * torch.randn(rows, hq + 2 * hkv, 1, device="cuda", generator=g))
        s["qkv"] = qkv.to(torch.bfloat16).reshape(rows, -1)
        s["q"] = torch.empty(rows, hq * d, dtype=torch.bfloat16, device="cuda")
        s["pos"], s["slots"] = pos.to("cuda", torch.int32), slots.to("cuda", torch.int32)
        s["cos"], s["sin"] = _tables(max(ctx) + 1, d)
        s["qn"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if c["qk"] else None
        s["kn"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=g) if c["qk"] else None
        return s
    s["bt"], s["lens"] = bt.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda")
    s["max_len"] = max(ctx)
    s["q"] = torch.randn(rows, hq * d, device="cuda", generator=g).to(torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    if c["op"] == "decode":
        # scratch for the partial results of sequences that are worked on in pieces, as a program allocates it once
        s["ws"] = torch.empty(4 + rows * hq * min(128, max(per) // 8 + 2) * (d + 2), device="cuda")
        return s
    q_lens = [n for _, n in lens]
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    s["cu"], s["max_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda"), max(q_lens)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------
def _rope(x, cos, sin):
    """x [T, heads, D] f32, each product and sum rounded by itself."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _norm(x, w):
    """RMSNorm over the head; the factor in 64 bits, since a value next to a border of e4m3 moves with its last bits."""
    inv = (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()
    return w * (x * inv)


def _exponent(amax):
    m, x = torch.frexp(amax)                              # amax = m 2^x, m in [0.5, 1); 448 = 0.875 2^9
    e = x - 9 + (m > 0.875).int()
    return torch.where(amax > 0, e.clamp(EXP_LO, EXP_HI), torch.full_like(e, EXP_LO))


def _store(x, codes, scale, slots, nb):
    """x [T, Hkv, D] f32 into the layer's codes [NB, Hkv, 16, D] and scales, in place."""
    page, off = slots // BS, slots % BS
    amax = torch.zeros(nb, x.shape[1], device=x.device).index_reduce_(0, page, x.abs().amax(-1), "amax")
    hit = torch.zeros(nb, device=x.device).index_fill_(0, page, 1.0) > 0
    fresh = torch.zeros(nb, device=x.device).index_add_(0, page, (off == 0).float()) > 0
    e_old = torch.frexp(scale)[1] - 1
    e = _exponent(amax)
    e = torch.where(fresh[:, None], e, torch.maximum(e, e_old))
    e = torch.where(hit[:, None], e, e_old)
    shrink = torch.where(fresh[:, None], torch.zeros_like(e), e_old - e)
    codes.copy_((codes.float() * torch.exp2(shrink.float())[:, :, None, None]).to(E4M3))
    y = (x * torch.exp2(-e.float())[page][:, :, None]).to(E4M3)
    codes.view(torch.uint8)[page, :, off] = y.view(torch.uint8)
    scale.copy_(torch.exp2(e.float()))


def _plain_append(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    nb = s["kc"].shape[0]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["qn"] is not None:
        q, k = _norm(q, s["qn"]), _norm(k, s["kn"])
    pos, slots = s["pos"].long(), s["slots"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    s["q"].copy_(_rope(q, cos, sin).reshape(s["q"].shape))
    _store(_rope(k, cos, sin), s["kc"], s["ks"], slots, nb)
    _store(v, s["vc"], s["vs"], slots, nb)


def _gather(codes, scale, bt):
    """The sequences' cached values [B, Hkv, tokens, D] in f32, padded to the longest."""
    ids = bt.long()
    x = codes.view(torch.uint8)[ids].view(E4M3).float() * scale[ids][..., None, None]
    b, n, h, _, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, n * BS, d)


def _softmax(w, seen):
    w = torch.where(seen, w, torch.full_like(w, -math.inf))
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    w = torch.where(seen, w, torch.zeros_like(w))
    return w / w.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_decode(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    q = s["q"].float().view(-1, hkv, hq // hkv, d)
    w = torch.matmul(q, _gather(s["kc"], s["ks"], s["bt"]).transpose(2, 3)) * d ** -0.5
    seen = torch.arange(w.shape[-1], device=w.device) < s["lens"][:, None, None, None]
    o = torch.matmul(_softmax(w, seen), _gather(s["vc"], s["vs"], s["bt"]))
    s["out"].copy_(o.reshape(s["out"].shape))


def _plain_prefill(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    b, cu = s["lens"].numel(), s["cu"].long()
    n = cu[1:] - cu[:-1]
    row = torch.arange(s["max_q"], device="cuda")
    real = row < n[:, None]                                              # [B, max_q]
    at = (cu[:-1, None] + row).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float().view(-1, hkv, hq // hkv, d)[at]                   # [B, max_q, Hkv, G, D]
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)                  # [B, Hkv, G max_q, D]
    w = torch.matmul(q, _gather(s["kc"], s["ks"], s["bt"]).transpose(2, 3)) * d ** -0.5
    w = w.view(b, hkv, hq // hkv, s["max_q"], -1)
    pos = (s["lens"].long() - n)[:, None] + row
    seen = torch.arange(w.shape[-1], device="cuda") <= torch.where(real, pos, torch.full_like(pos, -1))[..., None]
    p = _softmax(w, seen[:, None, None]).view(b, hkv, -1, w.shape[-1])
    o = torch.matmul(p, _gather(s["vc"], s["vs"], s["bt"])).view(b, hkv, hq // hkv, s["max_q"], d)
    o = o.permute(0, 3, 1, 2, 4).reshape(b * s["max_q"], hq * d).to(torch.bfloat16)
    # rows past a sequence's end go to a row behind the last, which is dropped
    to = torch.where(real, at, torch.full_like(at, s["q"].shape[0])).reshape(-1)
    whole = torch.empty(s["q"].shape[0] + 1, hq * d, dtype=torch.bfloat16, device="cuda")
    whole[to] = o
    s["out"].copy_(whole[:-1])


def _plain_pages(s):
    src, dst = torch.tensor(s["src"], device="cuda"), torch.tensor(s["dst"], device="cuda")
    p = s["pool"].view(torch.uint8)
    p[:, :, dst] = p[:, :, src]
    if s["scales"] is not None:
        s["scales"][:, :, dst] = s["scales"][:, :, src]


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
_module = None


def _kernels():
    global _module
    if _module is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "complexity-inference_b200"))
        from mu_b200 import kernels

        _module = kernels
    return _module


def _own(s):
    k = _kernels()
    if s["op"] == "pages":
        k.copy_pages(s["pool"], s["src"], s["dst"], scales=s["scales"])
    elif s["op"] == "append":
        k.rope_kv_append_fp8(s["qkv"], s["pos"], s["slots"], s["cos"], s["sin"], s["hq"], s["hkv"], s["d"], s["kc"], s["vc"],
                             s["ks"], s["vs"], s["qn"], s["kn"], EPS, q_out=s["q"])
    elif s["op"] == "decode":
        k.decode_attn_fp8(s["q"], s["out"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["lens"], s["hq"], s["hkv"], s["d"],
                          s["max_len"], workspace=s["ws"])
    else:
        k.prefill_attn_fp8(s["q"], s["out"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"], s["lens"], s["cu"], s["max_q"],
                           s["hq"], s["hkv"], s["d"])


PLAIN = {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "pages": _plain_pages}


def run(s):
    if own:
        _own(s)
    else:
        PLAIN[s["op"]](s)
    if s["op"] == "pages":
        return {"pool": s["pool"]} if s["scales"] is None else {"pool": s["pool"], "scales": s["scales"]}
    if s["op"] == "append":
        return {"q": s["q"], "k": s["kc"], "v": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _e4m3(x):
    """The nearest number of e4m3 (ties to even), in 64 bits."""
    mag = x.abs().clamp_min(2.0 ** -40)
    step = torch.exp2(torch.floor(torch.log2(mag)).clamp_min(-6.0) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_append(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    t = s["qkv"].shape[0]
    x = s["qkv"].double().reshape(t, hq + 2 * hkv, d)
    rot = x[:, :hq + hkv]
    if s["qn"] is not None:
        w = torch.cat([s["qn"].double().expand(hq, d), s["kn"].double().expand(hkv, d)])
        rot = rot / (rot.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
    p = s["pos"].long()
    z = torch.complex(rot[..., : d // 2], rot[..., d // 2:]) * torch.complex(s["cos"].double()[p], s["sin"].double()[p])[:, None]
    rot = torch.cat([z.real, z.imag], -1)
    got = {"q": rot[:, :hq].reshape(t, -1)}
    slots = s["slots"].tolist()
    runs, i = [], 0                                       # (block, first row, last row + 1, starts anew)
    while i < t:
        j = i
        while j < t and slots[j] // BS == slots[i] // BS:
            j += 1
        runs.append((slots[i] // BS, i, j, slots[i] % BS == 0))
        i = j
    at = torch.tensor([r[0] for r in runs], device="cuda")
    anew = torch.tensor([r[3] for r in runs], device="cuda")[:, None]
    owner = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), torch.tensor([r[2] - r[1] for r in runs], device="cuda"))
    off = s["slots"].long() % BS
    for name, codes, scale, new in (("k", s["kc"], s["ks"], rot[:, hq:]), ("v", s["vc"], s["vs"], x[:, hq + hkv:])):
        c, sc = codes.double(), scale.double()
        top = torch.zeros(len(runs), hkv, device="cuda", dtype=torch.float64).scatter_reduce_(
            0, owner[:, None].expand(t, hkv), new.abs().amax(-1), "amax")
        e = torch.ceil(torch.log2(top / 448.0))
        e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(EXP_LO, EXP_HI)   # log2 may round a whole number up
        grown = torch.where(anew, torch.exp2(e), torch.maximum(torch.exp2(e), sc[at]))
        ratio = torch.where(anew | (grown == sc[at]), torch.ones_like(grown), sc[at] / grown)
        block = torch.where((ratio == 1)[..., None, None], c[at], _e4m3(c[at] * ratio[..., None, None]))
        block[owner, :, off] = _e4m3(new / grown[owner][..., None])
        c[at], sc[at] = block, grown
        got[name], got[name + "_scale"] = c, sc
    return got


def _exact_attention(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    cu = s["cu"].tolist() if "cu" in s else list(range(len(lens) + 1))
    for b, ctx in enumerate(lens):
        ids = s["bt"][b, : (ctx + BS - 1) // BS].long()
        k, v = ((c.view(torch.uint8)[ids].view(E4M3).double() * sc[ids].double()[..., None, None]).transpose(0, 1).reshape(hkv, -1, d)[:, :ctx]
                for c, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        for lo in range(cu[b], cu[b + 1], 512):
            hi = min(lo + 512, cu[b + 1])
            last = ctx - cu[b + 1] + torch.arange(lo, hi, device="cuda")      # the last key that each row sees
            gone = torch.arange(ctx, device="cuda")[None] > last[:, None]
            q = s["q"][lo:hi].double().view(hi - lo, hkv, hq // hkv, d)
            w = torch.einsum("rhgd,htd->hgrt", q, k) / math.sqrt(d)
            p = torch.softmax(w.masked_fill(gone, -math.inf), -1)
            out[lo:hi] = torch.einsum("hgrt,htd->rhgd", p, v).reshape(hi - lo, hq * d)
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if s["op"] == "append":
        return _exact_append(s)
    if s["op"] != "pages":
        return _exact_attention(s)
    move = torch.arange(c["blocks"])
    move[s["dst"]] = torch.tensor(s["src"])
    move = move.cuda()
    got = {"pool": s["pool"].float().index_select(2, move)}
    if s["scales"] is not None:
        got["scales"] = s["scales"].double().index_select(2, move)
    return got
