"""More calls that the 8-bit cache's entry points refuse, on the CPU (see test_fp8_cache)."""

import pytest

from test_fp8_cache import DECODE, PREFILL, _lib, _refused


@pytest.mark.parametrize("name,args,rows", [("muk_paged_decode_attn_fp8", DECODE, "B"),
                                            ("muk_paged_prefill_attn_fp8", PREFILL, "rows")])
@pytest.mark.parametrize("stride", [0, 8, 504])
def test_overlapping_output_rows(name, args, rows, stride):
    """Rows of the output that lie over each other (a broadcast tensor) would be written by
    several blocks at once; a single row has no stride.  Query rows may be shared."""
    _refused(name, list({**args, "ldo": stride}.values()), -1, "overlap")
    lib = _lib()
    for change in ({rows: 1, "ldo": stride}, {"ldq": stride}):
        # passed over: the next refusal is the block table's
        assert getattr(lib.load(), name)(*{**args, **change, "max_len": 129}.values()) == -1
        assert "block table" in lib.last_error()
