"""Attention over a planned pattern, forward and backward, against dense 64-bit values with derived bounds
(tests/attn_reference.py)."""
import numpy as np
import pytest

import fusedmm_amd as fa
from attn_run import Case, inside, random_pattern, transposed, window_pattern

pytestmark = pytest.mark.gpu


def check_forward(c, e):
    inside(c.o.numpy(), e["o"], e["tol"]["o"], "o")
    lse = c.lse[:-1].double().cpu().numpy().reshape(e["lse"].shape)
    inside(lse, e["lse"], e["tol"]["lse"], "lse")
    if c.maps == 2:
        inside(c.o2.numpy(), e["o2"], e["tol"]["o2"], "o2")
    assert float(c.lse[-1]) == 7.5
    assert c.o.untouched_outside() and c.o2.untouched_outside()


def check_backward(c, e):
    inside(c.dq.numpy(), e["dq"].reshape(c.m, c.heads, -1), e["tol"]["dq"].reshape(c.m, c.heads, -1), "dq")
    inside(c.dk.numpy(), e["dk"].reshape(c.n, c.kv, -1), e["tol"]["dk"].reshape(c.n, c.kv, -1), "dk")
    inside(c.dvv.numpy(), e["dv"], e["tol"]["dv"], "dv")
    if c.maps == 2:
        inside(c.dlam.double().cpu().numpy(), e["dlam"], e["tol"]["dlam"], "dlambda")
    assert c.dq.untouched_outside() and c.dk.untouched_outside() and c.dvv.untouched_outside()


def run_both(c, how="packed"):
    import torch
    c.make_plans(True)
    c.gradients(how)
    assert c.forward() == 0
    assert c.backward() == 0
    torch.cuda.synchronize()
    e = c.exact(do=True)
    check_forward(c, e)
    check_backward(c, e)


# (m, n, heads, kv, d, dv, maps): width classes, shared key heads, odd head sizes, one row, one feature
SHAPES = [
    (1, 1, 1, 1, 1, 1, 1),
    (3, 5, 2, 1, 16, 16, 1),
    (65, 64, 2, 2, 32, 32, 1),
    (130, 100, 6, 2, 40, 24, 1),
    (70, 200, 3, 3, 64, 64, 1),
    (100, 90, 4, 1, 96, 128, 1),
    (40, 70, 2, 1, 200, 256, 1),
    (2, 3, 2, 2, 16, 33, 2),
    (65, 129, 4, 2, 32, 64, 2),
    (90, 64, 6, 2, 40, 72, 2),
    (70, 70, 2, 1, 64, 128, 2),
    (64, 65, 3, 1, 77, 131, 2),
    (50, 40, 2, 1, 128, 256, 2),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_random_patterns(kind, shape):
    m, n, heads, kv, d, dv, maps = shape
    c = Case(kind, maps, m, n, heads, kv, d, dv, *random_pattern(m, n, 24, seed=m + n), seed=m)
    run_both(c)


@pytest.mark.parametrize("how", ["heads", "wide", "odd"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_layouts(kind, how):
    c = Case(kind, 2, 70, 80, 4, 2, 32, 64, *random_pattern(70, 80, 20, seed=2), seed=5, how=how)
    run_both(c, how)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("kind,maps", [("bf16", 2), ("f32", 1), ("f16", 1)])
def test_long_rows_are_split_and_joined(kind, maps, bits):
    """A hub row of several chunks among short ones; its block is several units.  Transposed, columns of many rows."""
    indx, pb, pe = random_pattern(130, 3000, 12, seed=9, hub=2600)
    c = Case(kind, maps, 130, 3000, 2, 1, 32, 32 * maps, indx, pb, pe, seed=3, bits=bits)
    run_both(c)
    t = transposed(130, 3000, indx, pb, pe)
    c = Case(kind, maps, 3000, 130, 2, 1, 32, 32 * maps, *t, seed=4, bits=bits)
    run_both(c)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_window(kind):
    c = Case(kind, 2, 300, 340, 4, 2, 32, 64, *window_pattern(300, 340, 77), seed=1)
    run_both(c)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_dense_rows(kind):
    """Every row names every column, in one order: units of several chunks of shared columns."""
    m, n = 66, 1200
    indx = np.tile(np.arange(n), m)
    c = Case(kind, 1, m, n, 1, 1, 64, 64, indx, np.arange(m) * n, (np.arange(m) + 1) * n, seed=8)
    run_both(c)


def test_large_scores():
    """Scores of some hundreds: the running maximum, not the exponent's range, decides."""
    c = Case("f32", 2, 70, 90, 2, 1, 32, 64, *random_pattern(70, 90, 30, seed=6), seed=6, spread=9.0)
    run_both(c)


def test_rows_that_name_nothing():
    """All rows empty, or all their ids masked: zeros, lse = -infinity, zero gradients; also with no columns at all."""
    import torch
    for n, indx in ((50, np.array([-1, 50, 77])), (0, np.array([0, 1, 2]))):
        m = 67
        pb, pe = np.zeros(m, np.int64), np.where(np.arange(m) % 2, 3, 0)
        c = Case("bf16", 2, m, n, 2, 1, 32, 64, indx, pb, pe, seed=1)
        c.make_plans(True)
        c.gradients()
        assert c.forward() == 0 and c.backward() == 0
        torch.cuda.synchronize()
        assert (c.o.numpy() == 0).all() and (c.o2.numpy() == 0).all()
        assert np.isneginf(c.lse[:-1].cpu().numpy()).all()
        for t in (c.dq, c.dk, c.dvv):
            assert (t.numpy() == 0).all()
        assert (c.dlam.cpu().numpy() == 0).all()


def test_no_rows():
    import torch
    c = Case("f32", 2, 0, 20, 2, 1, 32, 64, np.array([0]), np.zeros(0, np.int64), np.zeros(0, np.int64))
    c.make_plans(True)
    c.gradients()
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    assert (c.dk.numpy() == 0).all() and (c.dvv.numpy() == 0).all() and (c.dlam.cpu().numpy() == 0).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("what", ["inf", "nan"])
def test_infinities_and_nan_reach_only_the_rows_that_name_them(kind, what):
    """One key row and one value row are not finite.  Rows that do not name them have the bits they have without; rows
    that do follow the formula; so do the gradients on either side."""
    import torch
    m, n, bad = 80, 60, 17
    indx, pb, pe = random_pattern(m, n, 12, seed=4, masked=False)
    names = np.array([bad in indx[pb[i]:pe[i]] for i in range(m)])
    assert 2 < names.sum() < m - 10
    a = Case(kind, 2, m, n, 2, 1, 32, 64, indx, pb, pe, seed=2)
    b = Case(kind, 2, m, n, 2, 1, 32, 64, indx, pb, pe, seed=2)
    x = float("inf") if what == "inf" else float("nan")
    b.v.view()[bad, 0, 5] = x
    for c in (a, b):
        c.make_plans(True)
        c.gradients()
        assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    for t in ("o", "o2", "dq"):
        assert np.array_equal(getattr(a, t).numpy()[~names], getattr(b, t).numpy()[~names]), t
    got = b.o.numpy()[names]
    assert not np.isfinite(got[:, :, 5]).any()
    rest = np.arange(64) != 5
    assert np.array_equal(a.o.numpy()[names][:, :, rest], got[:, :, rest])
    # keys that no such row names
    touched = np.zeros(n, bool)
    for i in np.nonzero(names)[0]:
        touched[indx[pb[i]:pe[i]]] = True
    assert (~touched).any()
    assert np.array_equal(a.dk.numpy()[~touched], b.dk.numpy()[~touched])
    assert np.array_equal(a.dvv.numpy()[~touched], b.dvv.numpy()[~touched])
    # a key row that is not finite, and a gradient row that is not
    b.v.view().copy_(a.v.view())
    b.k.view()[bad, 0, 3] = x
    for c in (a, b):
        assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    for t in ("o", "o2", "dq"):
        assert np.array_equal(getattr(a, t).numpy()[~names], getattr(b, t).numpy()[~names]), t
    b.k.view().copy_(a.k.view())
    row = int(np.nonzero(pe - pb > 3)[0][0])
    b.do.view()[row, 1, 7] = x
    for c in (a, b):
        assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    other = np.ones(n, bool)
    other[indx[pb[row]:pe[row]]] = False
    for t in ("dk", "dvv"):
        assert np.array_equal(getattr(a, t).numpy()[other], getattr(b, t).numpy()[other]), t
    assert not np.isfinite(b.dvv.numpy()[~other][:, 0, 7]).any()
    keep = np.arange(m) != row
    assert np.array_equal(a.dq.numpy()[keep], b.dq.numpy()[keep])


def test_gradients_against_differences():
    """fp32: the directional derivative of sum(o * do) by central differences of the 64-bit formula's own operands."""
    import torch
    c = Case("f32", 2, 40, 50, 2, 1, 16, 32, *random_pattern(40, 50, 10, seed=12), seed=12)
    c.make_plans(True)
    c.gradients()
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    from attn_reference import attention, counts
    count = counts(c.m, c.n, c.indx, c.pb, c.pe)
    q, k, v = c.q.numpy().reshape(c.m, c.heads, 2, c.d), c.k.numpy().reshape(c.n, c.kv, 2, c.d), c.v.numpy()
    lam, do = c.lam.double().cpu().numpy(), c.do.numpy()
    rng = np.random.default_rng(0)
    for name, x, grad in (("q", q, c.dq), ("k", k, c.dk), ("v", v, c.dvv), ("lam", lam, None)):
        step = rng.standard_normal(x.shape)
        vals = []
        for sign in (1, -1):
            args = dict(q=q, k=k, v=v, lam=lam)
            args[name] = x + sign * 1e-5 * step
            vals.append((attention(count, args["q"], args["k"], args["v"], args["lam"], c.scale, "f32")["o"] * do).sum())
        slope = (vals[0] - vals[1]) / 2e-5
        g = c.dlam.double().cpu().numpy() if grad is None else grad.numpy().reshape(x.shape)
        # the difference quotient is exact to about 1e-10 of the terms; the gradients are fp32: 1e-5 of the sum of their sizes
        assert abs(slope - (g * step).sum()) <= 1e-5 * np.abs(g * step).sum() + 1e-8, name


def test_same_bits_again_and_with_another_plan():
    import torch
    c = Case("bf16", 2, 130, 3000, 4, 2, 32, 64, *random_pattern(130, 3000, 40, seed=9, hub=2600), seed=3)
    c.make_plans(True)
    c.gradients()
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    first = [t.buf.clone() for t in (c.o, c.o2, c.dq, c.dk, c.dvv)] + [c.lse.clone(), c.dlam.clone()]
    for again in range(2):
        if again:
            c.make_plans(True)
        c.gradients()
        assert c.forward() == 0 and c.backward() == 0
        torch.cuda.synchronize()
        for a, b in zip(first, [t.buf for t in (c.o, c.o2, c.dq, c.dk, c.dvv)] + [c.lse, c.dlam]):
            assert torch.equal(a, b)


def test_inference_call_has_the_training_call_s_bits():
    import torch
    c = Case("f16", 2, 130, 300, 4, 2, 32, 64, *random_pattern(130, 300, 40, seed=9), seed=3)
    c.make_plans(False)
    assert c.forward(save=True) == 0
    torch.cuda.synchronize()
    first = c.o.buf.clone()
    lse = c.lse.clone()
    c.o.buf.fill_(7.5)
    assert c.forward(save=False) == 0
    torch.cuda.synchronize()
    assert torch.equal(first, c.o.buf) and torch.equal(lse, c.lse)


def test_graph_capture_and_other_streams():
    """Forward and backward captured once, replayed on new operands with eager work in between; an eager run on another
    stream with a workspace of its own at the same time."""
    import torch
    c = Case("bf16", 2, 130, 700, 4, 2, 32, 64, *random_pattern(130, 700, 40, seed=9, hub=1500), seed=3)
    e = Case("bf16", 2, 130, 700, 4, 2, 32, 64, c.indx, c.pb, c.pe, seed=3)
    for x in (c, e):
        x.make_plans(True)
        x.gradients()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        assert c.forward(stream=s.cuda_stream) == 0
        assert c.backward(stream=s.cuda_stream) == 0
    other = torch.cuda.Stream()
    for turn in range(4):
        for name in ("q", "k", "v", "do"):
            t = getattr(c, name).view()
            t.copy_(torch.randn(t.shape, device="cuda"))
            getattr(e, name).view().copy_(t)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            assert e.forward(stream=other.cuda_stream) == 0
            assert e.backward(stream=other.cuda_stream) == 0
        g.replay()
        torch.cuda.synchronize()
        for name in ("o", "o2", "dq", "dk", "dvv"):
            assert torch.equal(getattr(c, name).buf, getattr(e, name).buf), (turn, name)
        assert torch.equal(c.lse, e.lse) and torch.equal(c.dlam, e.dlam)
        float(torch.randn(1000, device="cuda").sum())


def test_refusals_on_the_device():
    """Bad pointers, small workspaces, plans of other patterns and of none."""
    import torch
    c = Case("f32", 2, 130, 700, 2, 1, 32, 64, *random_pattern(130, 700, 40, seed=9, hub=1500), seed=3)
    c.make_plans(True)
    c.gradients()
    lib = fa.load(32)
    assert c.size > 0
    c.size -= 16
    assert fa.NOT_ENOUGH_MEM in (c.forward(), c.backward())      # the larger need of the two
    c.size += 16
    host = np.zeros((130, 2, 64), np.float32)
    assert fa.fusedMM_attn_forward(c.desc, c.plan, host, c.k.ptr, c.v.ptr, c.lam, c.o.ptr, None, None, c.work, c.size) == fa.FAIL
    assert fa.fusedMM_attn_forward(c.desc, c.plan, None, c.k.ptr, c.v.ptr, c.lam, c.o.ptr, None, None, c.work, c.size) == fa.FAIL
    assert fa.fusedMM_attn_forward(c.desc, c.plan, c.q.ptr, c.k.ptr, c.v.ptr, None, c.o.ptr, None, None, c.work, c.size) == fa.FAIL
    assert fa.fusedMM_attn_forward(c.desc, c.plan_t, c.q.ptr, c.k.ptr, c.v.ptr, c.lam, c.o.ptr, None, None, c.work, c.size) == fa.FAIL
    assert fa.fusedMM_attn_forward(c.desc, c.plan, c.q.ptr, c.k.ptr, c.v.ptr, c.lam, c.o.ptr, None, None, c.work.data_ptr() + 4, c.size) == fa.FAIL
    assert fa.fusedMM_attn_workspace(c.desc, c.plan_t) == -1
    with pytest.raises(OSError):          # rows of more slots than nnz says
        fa.AttnPlan(130, 700, c.nnz - 1, *c.index)
    with pytest.raises(OSError):          # pntre < pntrb
        fa.AttnPlan(130, 700, c.nnz, c.index[0], c.index[2], c.index[1])
    with pytest.raises(OSError):
        fa.AttnPlan(130, 700, c.nnz, np.zeros(4, np.int32), *c.index[1:])
    with pytest.raises(OSError):
        fa.AttnPlan(1 << 26, 700, c.nnz, *c.index)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    keep = torch.zeros(16, device="cuda")
    with torch.cuda.graph(g, stream=s):
        keep += 1
        with pytest.raises(OSError):      # a plan cannot be made inside a capture
            fa.AttnPlan(130, 700, c.nnz, *c.index, stream=s.cuda_stream)
        keep += 1
    g.replay()
    torch.cuda.synchronize()
    assert float(keep[0]) == 2.0
    assert lib.fusedMM_attn_plan_destroy(None) == 0
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    check_backward(c, c.exact(do=True))
