"""Refusals of the attention entry points at the ends of what their arguments can say (no GPU needed)."""
import numpy as np
import pytest

import fusedmm_amd as fa
from test_attention_cpu import desc, rows, rows4

NOT_FINITE = [float("nan"), float("inf"), float("-inf")]


@pytest.mark.parametrize("scale", NOT_FINITE)
def test_a_scale_that_is_not_finite(capfd, scale):
    for call in (lambda d: rows(d), lambda d: rows4(d),
                 lambda d: fa.fusedMM_attn_forward(d, None, 16, 16, 16, None, 16, None, None, None, 0, stream=0),
                 lambda d: fa.fusedMM_attn_backward(d, None, None, 16, 16, 16, None, 16, None, 16, 16, 16, 16, 16, None, None, 0, stream=0)):
        assert call(desc(scale=scale)) == fa.FAIL
        assert "scale is not a finite number" in capfd.readouterr().err


def test_the_cache_does_not_read_rows_and_query_heads():
    """m, heads and the strides of q and o play no part in writing and reading a cache, whatever they hold."""
    d = desc(m=-7, heads=-1, ldq=-1, hdq=-1, ldo=-5, hdo=1 << 60, scale=float("nan"))
    assert fa.fusedMM_kv4_write(d, 0, None, None, None, None, 160, 80, stream=0) == 0
    assert fa.fusedMM_kv4_read(d, 0, None, None, 160, 80, None, None, stream=0) == 0
    lib = fa.load(32)
    assert lib.fusedMM_kv4_write(None, 0, None, None, None, None, 160, 80, None) == fa.FAIL
    assert lib.fusedMM_kv4_read(None, 0, None, None, 160, 80, None, None, None) == fa.FAIL


def test_overlap_is_decided_beyond_64_bits(capfd):
    """(heads - 1) * hdc of 2^64 bytes is not zero: 2^30 records 2^20 bytes apart under heads 2^44 apart overlap in either order."""
    d = desc(n=1 << 30, heads=(1 << 20) + 1, kv_heads=(1 << 20) + 1, d=32, dv=32)
    assert fa.fusedMM_kv4_write(d, 1, 16, 16, 16, 16, 1 << 20, 1 << 44, stream=0) == fa.FAIL
    assert "records of the cache overlap" in capfd.readouterr().err
