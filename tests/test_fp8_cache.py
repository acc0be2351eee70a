"""What the 8-bit cache's entry points refuse, checked without a GPU: the C entry
points reject a bad shape, stride, pointer or list before they touch the device,
and the Python wrappers reject wrong types, shapes and devices before they call
them."""

import ctypes

import pytest
import torch

OK = 1 << 20     # a 16-byte aligned address that is never read: every call here is refused
ODD = OK + 2
FP8 = torch.float8_e4m3fn


def _lib():
    from mu_b200 import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("libmuk.so not built (run complexity-inference_b200/build.py)")
    return _lib


def _refused(name, args, code, text):
    lib = _lib()
    rc = getattr(lib.load(), name)(*args)
    assert rc == code, (name, rc, lib.last_error())
    assert text in lib.last_error(), lib.last_error()


APPEND = dict(qkv=OK, ld=768, q=OK, ldq=512, pos=OK, slots=OK, cos=OK, sin=OK, max_pos=64, T=3,
              hq=4, hkv=1, d=128, qn=None, kn=None, eps=1e-6, k=OK, v=OK, ks=OK, vs=OK, nb=8, bs=16,
              stream=None)
DECODE = dict(q=OK, ldq=512, out=OK, ldo=512, k=OK, v=OK, ks=OK, vs=OK, bt=OK, bts=8, sl=OK, B=2,
              hq=4, hkv=1, d=128, bs=16, nb=8, scale=0.1, max_len=128, ws=None, wsb=0, stream=None)
PREFILL = dict(q=OK, ldq=512, out=OK, ldo=512, k=OK, v=OK, ks=OK, vs=OK, bt=OK, bts=8, sl=OK, cu=OK,
               B=2, rows=9, max_q=5, max_len=128, hq=4, hkv=1, d=128, bs=16, nb=8, scale=0.1,
               stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(qkv=None), -1, "null"), (dict(ks=None), -1, "null"), (dict(bs=32), -1, "block_size"),
    (dict(hq=3, hkv=2), -1, "heads"), (dict(hkv=0), -1, "heads"), (dict(d=96), -2, "head_dim"),
    (dict(d=256), -2, "head_dim"), (dict(ld=760), -1, "strides"), (dict(ld=772), -1, "strides"),
    (dict(ldq=504), -1, "strides"), (dict(nb=0), -1, "cache"), (dict(max_pos=0), -1, "cache"),
    (dict(qkv=ODD), -1, "aligned"), (dict(cos=OK + 4), -1, "aligned"), (dict(v=OK + 8), -1, "aligned")])
def test_append_refuses(change, code, text):
    _refused("muk_rope_kv_append_fp8", list({**APPEND, **change}.values()), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(sl=None), -1, "null"), (dict(vs=None), -1, "null"), (dict(bs=8), -1, "block_size"),
    (dict(hq=34, hkv=2), -1, "GQA"), (dict(hq=5, hkv=2), -1, "GQA"), (dict(d=80), -2, "head_dim"),
    (dict(ldq=514), -1, "strides"), (dict(q=ODD), -1, "strides"), (dict(k=OK + 8), -1, "strides"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=-1.0), -1, "scale"),
    (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"),
    (dict(max_len=129), -1, "block table"), (dict(max_len=0), -1, "block table"),
    (dict(B=70000), -1, "sequences"), (dict(max_len=4096, bts=256), -3, "workspace"),
    (dict(max_len=4096, bts=256, ws=OK, wsb=64), -3, "workspace"),
    (dict(max_len=4096, bts=256, ws=OK + 4, wsb=1 << 30), -3, "workspace")])
def test_decode_refuses(change, code, text):
    _refused("muk_paged_decode_attn_fp8", list({**DECODE, **change}.values()), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(cu=None), -1, "null"), (dict(bs=8), -1, "block_size"), (dict(hq=5, hkv=2), -1, "heads"),
    (dict(d=32), -2, "head_dim"), (dict(ldo=516), -1, "strides"), (dict(out=OK + 8), -1, "strides"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"),
    (dict(max_len=130), -1, "block table"), (dict(nb=0), -1, "block table"),
    (dict(B=70000), -1, "sequences"), (dict(max_q=600000), -1, "rows of a sequence"),
    (dict(hq=128, ldq=16384, ldo=16384, max_q=131072), -1, "rows of a sequence")])
def test_prefill_refuses(change, code, text):
    _refused("muk_paged_prefill_attn_fp8", list({**PREFILL, **change}.values()), code, text)


def test_decode_workspace_serves_smaller_batches():
    """What a workspace was sized for covers fewer sequences and shorter contexts, each of
    which the entry point may cut into other runs."""
    lib = _lib()

    def needs(n, length):  # as the entry point says when it has none
        rc = lib.load().muk_paged_decode_attn_fp8(*{**DECODE, "B": n, "max_len": length,
                                                    "bts": 1 << 20}.values())
        return 0 if rc != -3 else int(lib.last_error().split(" bytes")[0].split()[-1])

    def size(n, length):
        return lib.load().muk_decode_attn_fp8_workspace_size(n, DECODE["hq"], DECODE["d"], length, 16)

    lengths = [257, 300, 4096, 12000, 23999, 24000, 24001, 24016, 30000, 32768, 48000, 48001, 100000]
    for i, length in enumerate(lengths):
        for n in (1, 7, 2048, 4000):
            for shorter in lengths[: i + 1]:
                for fewer in (1, 5, 2048):
                    if fewer <= n:
                        assert 0 < needs(fewer, shorter) <= size(n, length), (n, length, fewer, shorter)


@pytest.mark.parametrize("src,dst,change,text", [
    ([1], [1], {}, "destination"), ([1, 2], [3, 3], {}, "destination"), ([1, 3], [3, 4], {}, "source"),
    ([1, 2], [2, 4], {}, "source"), ([1], [8], {}, "range"), ([-1], [2], {}, "range"),
    ([1], [2], dict(page=24), "multiples of 16"), ([1], [2], dict(pool=ODD), "multiples of 16"),
    ([1], [2], dict(plane=4 * 1024), "multiples of 16"), ([1], [2], dict(planes=0), "planes"),
    ([1], [2], dict(scales=OK, splane=8 * 6, sbytes=6), "scales"),
    ([1], [2], dict(scales=OK, splane=4 * 8, sbytes=8), "scales")])
def test_copy_refuses(src, dst, change, text):
    a = {**dict(pool=OK, plane=8 * 1024, planes=2, page=1024, scales=None, splane=0, sbytes=0, nb=8),
         **change}
    arr = ctypes.c_int32 * len(src)
    s, d = arr(*src), arr(*dst)
    _refused("muk_copy_pages", list(a.values()) + [ctypes.addressof(s), ctypes.addressof(d), len(src),
                                                   None], -1, text)


def test_nothing_to_do_is_no_error():
    lib = _lib().load()
    assert lib.muk_rope_kv_append_fp8(*{**APPEND, "T": 0}.values()) == 0
    assert lib.muk_paged_decode_attn_fp8(*{**DECODE, "B": 0}.values()) == 0
    assert lib.muk_paged_prefill_attn_fp8(*{**PREFILL, "B": 0}.values()) == 0
    assert lib.muk_paged_prefill_attn_fp8(*{**PREFILL, "max_q": 0}.values()) == 0
    assert lib.muk_copy_pages(OK, 8 * 1024, 2, 1024, None, 0, 0, 8, None, None, 0, None) == 0


def test_workspace_covers_every_smaller_batch():
    """The size for a batch covers each smaller one, and a workspace of
    [rows, heads, min(128, blocks / 8 + 2), D + 2] floats is always enough."""
    size = _lib().load().muk_decode_attn_fp8_workspace_size
    for hq, d in ((32, 128), (4, 64)):
        for length in (1, 16, 300, 2048, 5000, 32768, 131072):
            last = 0
            for n in (1, 2, 7, 64, 256):
                got = size(n, hq, d, length, 16)
                assert got >= last
                assert got <= n * hq * min(128, -(-length // 16) // 8 + 2) * (d + 2) * 4
                last = got
    assert size(0, 32, 128, 100, 16) == 0 and size(4, 32, 128, 100, 32) == 0


# ----------------------------------------------------------------------------- wrappers
def _cpu(hkv=2, d=64, nb=4):
    c = torch.zeros(nb, hkv, 16, d).to(FP8)
    s = torch.ones(nb, hkv)
    return dict(k_cache=c, v_cache=c.clone(), k_scale=s, v_scale=s.clone())


def _decode_args(**change):
    a = dict(q=torch.zeros(2, 256, dtype=torch.bfloat16), out=torch.zeros(2, 256, dtype=torch.bfloat16),
             **_cpu(), block_tables=torch.zeros(2, 4, dtype=torch.int32),
             seq_lens=torch.ones(2, dtype=torch.int32), num_q_heads=4, num_kv_heads=2, head_dim=64,
             max_seq_len=64)
    a.update(change)
    return a


@pytest.mark.parametrize("change,err", [
    (dict(q=torch.zeros(2, 256)), TypeError), (dict(q=torch.zeros(1, 256, dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros(2, 128, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(256, 2, dtype=torch.bfloat16).t()), ValueError),
    (dict(k_cache=torch.zeros(4, 2, 16, 64)), TypeError),
    (dict(k_scale=torch.ones(4, 2, dtype=torch.float64)), TypeError),
    (dict(k_scale=torch.ones(2, 4)), ValueError), (dict(num_kv_heads=4), ValueError),
    (dict(v_cache=torch.zeros(5, 2, 16, 64).to(FP8)), ValueError),
    (dict(v_cache=torch.zeros(4, 16, 2, 64).to(FP8).transpose(1, 2)), ValueError),
    (dict(block_tables=torch.zeros(2, 4)), ValueError), (dict(block_tables=torch.zeros(1, 4, dtype=torch.int32)), ValueError),
    (dict(max_seq_len=65), ValueError), (dict(seq_lens=torch.ones(2)), ValueError),
    (dict(seq_lens=torch.ones(4, dtype=torch.int32)[::2]), ValueError)])
def test_decode_wrapper_refuses(change, err):
    from mu_b200 import kernels as K

    with pytest.raises(err, match="decode_attn_fp8"):
        K.decode_attn_fp8(**_decode_args(**change))


def test_wrappers_refuse_other_devices(monkeypatch):
    from mu_b200 import kernels as K

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.decode_attn_fp8(**_decode_args())
    a = _decode_args()
    a.pop("max_seq_len")
    with pytest.raises(ValueError, match="current CUDA device"):
        K.prefill_attn_fp8(**a, cu_seqlens_q=torch.zeros(3, dtype=torch.int32), max_q_len=1)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.copy_pages(torch.zeros(4, 2, 16, 64), [0], [1])
    tab = torch.zeros(8, 32)
    with pytest.raises(ValueError, match="current CUDA device"):
        K.rope_kv_append_fp8(torch.zeros(3, 512, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32),
                             torch.zeros(3, dtype=torch.int32), tab, tab, 4, 2, 64, **_cpu())


def test_append_and_copy_wrappers_refuse():
    from mu_b200 import kernels as K

    qkv, idx = torch.zeros(3, 512, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    tab, c = torch.zeros(8, 32), _cpu()

    def append(qkv=qkv, pos=idx, slots=idx, cos=tab, sin=tab, **more):
        K.rope_kv_append_fp8(qkv, pos, slots, cos, sin, 4, 2, 64, **c, **more)

    for bad in (dict(qkv=qkv[:, :500]), dict(pos=idx[:2]), dict(slots=idx.long()),
                dict(cos=torch.zeros(8, 64)), dict(sin=torch.zeros(7, 32)),
                dict(q_norm_w=torch.ones(32)), dict(q_out=torch.zeros(2, 256, dtype=torch.bfloat16))):
        with pytest.raises(ValueError, match="rope_kv_append_fp8"):
            append(**bad)
    with pytest.raises(TypeError):
        append(qkv=qkv.float())
    pool = torch.zeros(2, 4, 2, 16, 64)
    for bad in (dict(pool=pool.transpose(0, 1)), dict(pool=pool[0, 0]), dict(dst=[1, 2]),
                dict(scales=torch.ones(2, 4))):
        with pytest.raises(ValueError, match="copy_pages"):
            K.copy_pages(**{**dict(pool=pool, src=[0], dst=[1]), **bad})
