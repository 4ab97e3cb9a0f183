"""Sixteen-bit attention where its roundings count: bounds without a rounding of the weights and without one of the row means
(tests/attn_tight.py), weights far below the largest, score gradients outside fp16's range, large lambdas."""
import numpy as np
import pytest

import fusedmm_amd as fa
from attn_run import Case, random_pattern, transposed, window_pattern
from attn_tight import tight
from test_gpu_attention import check_backward, check_forward
from test_gpu_attention_rows import CacheCase, check_rows, ragged

pytestmark = pytest.mark.gpu


def both(c):
    import torch
    c.make_plans(True)
    c.gradients()
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    e = tight(c, do=True)
    check_forward(c, e)
    check_backward(c, e)
    return e


def cached(c):
    return tight(c, k=c.k_values, v=c.v_values, weight_type="f16")


# ---- rows over a 4-bit cache -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,dv,maps", [(8, 2, 32, 32, 1), (2, 1, 64, 96, 1), (4, 2, 32, 64, 2), (20, 1, 64, 128, 2), (3, 3, 128, 128, 1)])
def test_rows_over_the_cache_round_weights_twice(kind, heads, kv, d, dv, maps):
    import torch
    lengths = [1, 40, 700, 0, 1500]
    c = CacheCase(kind, maps, 5, 1600, heads, kv, d, dv, *ragged(lengths, 1600, seed=1), seed=2)
    e = cached(c)
    for nnz in (256, c.nnz):
        assert c.rows(nnz=nnz) == 0
        torch.cuda.synchronize()
        check_rows(c, e)


# ---- the second rounding and the exact mean --------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["bf16"])
@pytest.mark.parametrize("pattern", ["shared", "apart", "long"])
@pytest.mark.parametrize("d,dv,maps", [(32, 32, 1), (40, 24, 1), (64, 128, 2), (128, 128, 1), (16, 32, 2), (128, 256, 2)])
def test_weights_and_gradients_are_rounded_twice(kind, pattern, d, dv, maps):
    import torch
    if pattern == "shared":
        m, n, index = 100, 160, window_pattern(100, 160, 60)
    elif pattern == "apart":
        m, n, index = 90, 300, random_pattern(90, 300, 9, seed=2)
    else:
        m, n, index = 66, 1100, random_pattern(66, 1100, 9, seed=2, hub=2600)
    c = Case(kind, maps, m, n, 4, 2, d, dv, *index, seed=d + dv, spread=1.5)
    e = both(c)
    assert c.rows() == 0
    torch.cuda.synchronize()
    check_rows(c, e)
