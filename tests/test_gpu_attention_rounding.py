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


# ---- lambda ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pattern", ["shared", "apart"])
def test_large_lambdas(kind, pattern):
    """P1 - lambda P2 of some hundreds is an ordinary weight."""
    import torch
    m, n = 90, 120
    if pattern == "shared":
        index = window_pattern(m, n, 20)
    else:
        index = random_pattern(m, n, 6, seed=3)
    c = Case(kind, 2, m, n, 4, 2, 32, 64, *index, seed=4)
    c.lam = torch.tensor([100.0, -300.0, 1000.0, 0.0], device="cuda")
    c.do.view().mul_(0.125)
    e = both(c)
    assert np.abs(e["dv"]).max() > 64 and np.abs(e["o"]).max() < 65504


# ---- score gradients -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("turned", [False, True])
def test_small_gradients_over_long_rows(maps, turned):
    """Output gradients of 1e-4 over rows of 4096 columns (and over columns of 4096 rows): each score's gradient is a few of fp16's
    smallest steps, their sums are not."""
    m, n = 66, 4096
    indx, pb, pe = np.tile(np.arange(n), m), np.arange(m) * n, (np.arange(m) + 1) * n
    if turned:
        (indx, pb, pe), m, n = transposed(m, n, indx, pb, pe), n, m
    c = Case("f16", maps, m, n, 2, 1, 32, 32 * maps, indx, pb, pe, seed=1, scale=1.0)
    c.k.view().mul_(4.0)
    c.q.view().mul_(0.125)
    c.do.view().mul_(1e-4 * (4096 / 66 if turned else 1))
    both(c)


def test_large_gradients():
    """Score gradients beyond 65504 whose products with the scale are ordinary numbers."""
    c = Case("f16", 1, 80, 300, 4, 2, 32, 64, *random_pattern(80, 300, 4, seed=5, duplicates=False), seed=5, scale=1 / 64)
    c.v.view().mul_(8.0)
    c.do.view().mul_(3e3)
    e = both(c)
    dP = np.einsum("mhf,nhf->mhn", c.do.numpy(), np.repeat(c.v.numpy(), 2, axis=1))
    assert np.abs(dP).max() > 3 * 65504 and all(np.abs(e[x]).max() < 65504 for x in ("dq", "dk", "dv"))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_gradients_of_mixed_sizes(kind):
    """Rows' gradients from 1e-30 (fp16: 1e-7) to 1e3 next to each other, in one block and under one key: the running range follows."""
    rng = np.random.default_rng(0)
    c = Case(kind, 2, 130, 200, 4, 2, 32, 64, *random_pattern(130, 200, 30, seed=7), seed=7)
    import torch
    size = 10.0 ** rng.uniform(-7 if kind == "f16" else -30, 3, (130, 1, 1))
    size[::9] = 0.0
    c.do.view().mul_(torch.as_tensor(size).to(c.do.buf).to("cuda"))
    both(c)


# ---- weights far below the largest -----------------------------------------------------------------------------------------

def sink(c, depth, value):
    """Slot 0 scores `depth` log2 units above all others, and its value is zero; the others' values are `value`."""
    c.q.view().zero_()
    c.k.view().zero_()
    c.v.view().fill_(value)
    c.q.view()[..., 0] = 1.0
    c.k.view()[0, :, 0] = depth
    c.v.view()[0] = 0.0
    if c.maps == 2:
        c.q.view()[..., c.d] = 1.0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("maps", [1, 2])
def test_a_sink_leaves_the_others_their_mass(kind, maps):
    """One dominant key whose value is zero above 70000 others, each 2^-25.5 of it: the output is their mass."""
    import torch
    n = 70000
    index = (np.tile(np.arange(n), 2), np.array([0, n]), np.array([n, 2 * n]))
    c = Case(kind, maps, 2, n, 2, 1, 32, 32 * maps, *index, seed=1, scale=float(np.log(2)))
    sink(c, 25.5, 4.0)
    e = tight(c)
    mass = (n - 1) * 2.0 ** -25.5 / (1 + (n - 1) * 2.0 ** -25.5)
    if maps == 1:
        assert np.allclose(e["o"], 4 * mass, rtol=1e-6)
    c.make_plans(False)
    assert c.forward() == 0
    torch.cuda.synchronize()
    check_forward(c, e)
    for nnz in (100, c.nnz):
        c.o.view().zero_()
        assert c.rows(nnz=nnz) == 0
        torch.cuda.synchronize()
        check_rows(c, e)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_sink_in_a_cache(kind):
    import torch
    n = 60000
    index = (np.tile(np.arange(n), 2), np.array([0, n]), np.array([n, 2 * n]))


    c = Case(kind, 1, 2, n, 2, 1, 32, 32, *index, seed=1, scale=float(np.log(2)))
    sink(c, 25.5, 4.0)
    rec = fa.fusedMM_kv4_record_bytes(1, 32, 32)
    cache = torch.zeros(n * rec, dtype=torch.uint8, device="cuda")
    every = torch.arange(n, dtype=torch.int32, device="cuda")
    assert fa.fusedMM_kv4_write(c.desc, n, every, c.k.ptr, c.v.ptr, cache, rec, rec) == 0
    kx, vx = torch.empty((n, 1, 32), dtype=torch.float32, device="cuda"), torch.empty((n, 1, 32), dtype=torch.float32, device="cuda")
    c.desc.type = fa.TYPE_F32
    assert fa.fusedMM_kv4_read(c.desc, n, every, cache, rec, rec, kx, vx) == 0
    c.desc.type = fa.TYPES[kind]
    torch.cuda.synchronize()
    e = tight(c, k=kx.double().cpu().numpy(), v=vx.double().cpu().numpy(), weight_type="f16")
    assert e["o"].min() > 1e-3
    for nnz in (100, c.nnz):
        size = fa.fusedMM_attn_rows_workspace(c.desc, nnz)
        work = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        c.o.view().zero_()
        assert fa.fusedMM_attn_rows_kv4(c.desc, nnz, *c.index, c.q.ptr, cache, rec, rec, None, c.o.ptr, work, size) == 0
        torch.cuda.synchronize()
        check_rows(c, e)


# ---- the second rounding and the exact mean --------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
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


# ---- the weights' sum ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [37, 100, 300])
def test_weights_of_the_backward_pass_add_up_to_one(kind, window):
    """One value and one output gradient for all: every row's mean is 1, whatever its scores, and dlambda the number of rows.  The
    weights come from lse, which scores of 30 to 60 leave off by up to 2^-19; their sum takes that off again."""
    import torch
    m, n = 128, 500
    c = Case(kind, 2, m, n, 2, 1, 16, 16, *window_pattern(m, n, window), seed=3)
    for t in (c.q, c.v, c.do):
        t.view().zero_()
    c.q.view()[..., 0] = 1.0
    c.q.view()[..., 16] = 1.0
    c.v.view()[..., 0] = 1.0
    c.do.view()[..., 0] = 1.0
    c.k.view()[..., 0] += 120.0
    c.k.view()[..., 16] += 200.0
    c.make_plans(True)
    c.gradients()
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    # mean and sum are the same additions: their quotient is off by a reciprocal and a product (2 * 2^-24), a wave's sum by four
    # additions and dlambda by its own rounding
    assert np.abs(c.dlam.double().cpu().numpy() + m).max() <= m * 7 * 2.0 ** -24
