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


# ---- launches --------------------------------------------------------------------------------------------------------------

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include "fusedmm_attn_sizes.h"
using namespace fmm_attn;
int main(int argc, char **argv)
{
   int64_t a[16] = {0};
   for (int i = 2; i < argc; i++) a[i - 2] = atoll(argv[i]);
   switch (argv[1][0])
   {
      case 'l': printf("%d\n", launch_fits(a[0], (int)a[1])); break;
      case 'f': printf("%d\n", forward_fits({a[0], a[1], 0, (int)a[2]}, a[3], (int)a[4])); break;
      case 'b': printf("%d\n", backward_fits({1, 0, 1, 64}, {a[0], a[1], a[5], (int)a[2]}, a[3], a[4], (int)a[6])); break;
      case 'p': printf("%d\n", pack_fits(a[0])); break;
      case 'r': printf("%d\n", rows_fit(a[0], a[1], a[2], a[3])); break;
      case 'w': printf("%d\n", join_waves(a[0], a[1], a[2], (int)a[3])); break;
   }
}
"""


@pytest.fixture(scope="module")
def sizes(tmp_path_factory):
    import os
    import subprocess
    where = tmp_path_factory.mktemp("sizes")
    (where / "sizes.cc").write_text(PROGRAM)
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fusedmm_amd", "csrc")
    subprocess.check_call(["g++", "-std=c++17", "-I", csrc, str(where / "sizes.cc"), "-o", str(where / "sizes")])
    return lambda *a: int(subprocess.check_output([str(where / "sizes")] + [str(x) for x in a]))


def test_launches_hold_less_than_2_to_the_32_threads(sizes):
    assert sizes("l", 2 ** 24 - 1, 256) and not sizes("l", 2 ** 24, 256)
    assert sizes("l", 2 ** 22 - 1, 1024) and not sizes("l", 2 ** 22, 1024)
    # forward, dq: units, joins, block rows, heads, width.  2^26 - 1 rows in blocks of 64 are 2^20 units
    assert not sizes("f", 2 ** 20, 0, 64, 16, 32) and sizes("f", 2 ** 20, 0, 64, 15, 32)
    assert not sizes("f", 2 ** 22, 0, 16, 16, 32) and sizes("f", 2 ** 22, 0, 16, 15, 32)
    assert not sizes("f", 100, 2 ** 12, 64, 64, 256) and sizes("f", 100, 2 ** 12, 64, 63, 256)       # the join
    assert not sizes("f", 2 ** 31 - 1, 2 ** 31 - 1, 64, 2 ** 31 - 1, 256)
    # dk, dv: units, joins, block rows, heads, kv heads, tiles, width
    assert sizes("b", 2 ** 20, 0, 64, 15, 15, 1, 32) and not sizes("b", 2 ** 20, 0, 64, 16, 16, 1, 32)
    assert sizes("b", 2 ** 20 - 1, 0, 64, 8, 8, 1, 32)
    assert not sizes("b", 2 ** 18, 0, 64, 2 ** 24 - 2 ** 18, 1, 1, 32)                               # units + a workgroup per head
    assert not sizes("b", 100, 2 ** 12, 64, 32, 32, 1, 256) and sizes("b", 100, 2 ** 12, 64, 31, 31, 1, 256)
    assert sizes("b", 1, 0, 64, 8, 1, (2 ** 31 - 1) // 8, 32) and not sizes("b", 1, 0, 64, 8, 1, 2 ** 28, 32)
    assert sizes("p", 2 ** 23 - 1) and not sizes("p", 2 ** 23) and sizes("p", 1)
    # rows: pieces, rows, key heads * passes, heads
    assert sizes("r", 2 ** 20 - 8, 1, 16, 16) and not sizes("r", 2 ** 20, 1, 16, 16)
    assert sizes("r", 8, 2 ** 20 - 1, 1, 16) and not sizes("r", 8, 2 ** 20, 1, 16)
    # 16 waves only where the join's launch has room for them
    assert sizes("w", 10000, 8, 32, 128) == 16 and sizes("w", 300, 8, 32, 128) == 4 and sizes("w", 2 ** 40, 2 ** 17, 32, 128) == 4


@pytest.mark.parametrize("bits", [32, 64])
def test_rows_beyond_a_launch_are_refused_beforehand(capfd, bits):
    """Sizes that 2^31 workgroups held but 2^32 threads do not."""
    for change in (dict(m=1 << 20, heads=16, kv_heads=16, ldo=1024), dict(m=1 << 23, heads=32, kv_heads=1, ldo=2048), dict(m=1 << 24, heads=1, kv_heads=1)):
        d = desc(**change)
        assert fa.fusedMM_attn_rows_workspace(d, 100, index_bits=bits) == -1
        assert "too many rows" in capfd.readouterr().err
        assert rows(d, index_bits=bits) == fa.FAIL and "too many rows" in capfd.readouterr().err
    assert fa.fusedMM_attn_rows_workspace(desc(m=(1 << 20) - 8, heads=16, kv_heads=16, ldo=1024), 100, index_bits=bits) == 0


def test_inline_assembly_names_m0_where_it_writes_it():
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fusedmm_amd", "csrc")
    seen = 0
    for name in sorted(os.listdir(csrc)):
        if name.startswith("fusedmm_attn"):
            for asm in re.findall(r"asm volatile\((.*?)\);", open(os.path.join(csrc, name)).read(), re.S):
                if "s_mov_b32 m0" in asm:
                    seen += 1
                    assert asm.rstrip().endswith('"m0"'), (name, asm)
    assert seen == 2
