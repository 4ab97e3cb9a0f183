"""Infinities and NaN in attention: in blocks that are split and joined, in rows that are laid out anew, in blocks of 16 and of 64
rows, in records of a 4-bit cache; rows all of whose scores are minus infinity."""
import numpy as np
import pytest

import fusedmm_amd as fa
from attn_run import Case, inside, random_pattern, transposed, window_pattern
from test_gpu_attention_rows import CacheCase, ragged

pytestmark = pytest.mark.gpu


def pair(kind, maps, m, n, heads, kv, d, dv, index, **kw):
    return [Case(kind, maps, m, n, heads, kv, d, dv, *index, seed=2, **kw) for _ in range(2)]


def train(*cases):
    import torch
    for c in cases:
        if c.plan is None:
            c.make_plans(True)
        c.gradients()
        assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()


def pattern_of(name, m, n):
    if name == "window":
        return window_pattern(m, n, 40)
    if name == "apart":
        return random_pattern(m, n, 9, seed=4, masked=False)
    if name == "hub":           # a block of several units
        return random_pattern(m, n, 9, seed=4, masked=False, hub=1800)
    indx, pb, pe = random_pattern(n, m, 9, seed=4, masked=False, hub=1800)      # a column of many rows
    return transposed(n, m, indx, pb, pe)


@pytest.mark.parametrize("what", [float("inf"), float("nan")])
@pytest.mark.parametrize("pattern", ["window", "apart", "hub", "turned"])
@pytest.mark.parametrize("kind,d,dv,maps", [("f32", 32, 32, 1), ("f16", 64, 64, 1), ("bf16", 128, 128, 1), ("f16", 40, 72, 2), ("bf16", 21, 37, 1),
                                            ("f32", 64, 128, 2), ("bf16", 128, 256, 2)])
def test_only_the_rows_that_name_them(kind, d, dv, maps, pattern, what):
    """A value, then a key, then an output gradient that is not finite: rows and keys that are not joined to it keep their bits."""
    m, n = (90, 700) if pattern != "turned" else (700, 90)
    indx, pb, pe = pattern_of(pattern, m, n)
    a, b = pair(kind, maps, m, n, 2, 1, d, dv, (indx, pb, pe))
    named_by = [set(indx[pb[i]:pe[i]].tolist()) for i in range(m)]
    hub = int(np.argmax([len(x) for x in named_by]))
    if pattern == "hub":
        bad = sorted(named_by[hub])[7]
    else:
        times = np.bincount(indx[np.concatenate([np.arange(s, t) for s, t in zip(pb, pe)])], minlength=n)
        bad = int(np.argmax(times))
    names = np.array([bad in x for x in named_by])
    assert names.any() and not names.all()
    touched = np.zeros(n, bool)
    for i in np.nonzero(names)[0]:
        touched[list(named_by[i])] = True
    train(a)
    b.v.view()[bad, 0, dv - 3] = what
    train(b)
    for t in ("o", "dq") + (("o2",) if maps == 2 else ()):
        assert np.array_equal(getattr(a, t).numpy()[~names], getattr(b, t).numpy()[~names]), t
    got, rest = b.o.numpy()[names], np.arange(dv) != dv - 3
    assert not np.isfinite(got[:, :, dv - 3]).any()
    assert np.array_equal(a.o.numpy()[names][:, :, rest], got[:, :, rest])
    for t in ("dk", "dvv"):
        assert np.array_equal(getattr(a, t).numpy()[~touched], getattr(b, t).numpy()[~touched]), t
    b.v.view().copy_(a.v.view())
    b.k.view()[bad, 0, d - 1] = what
    train(b)
    for t in ("o", "dq"):
        assert np.array_equal(getattr(a, t).numpy()[~names], getattr(b, t).numpy()[~names]), t
    for t in ("dk", "dvv"):
        assert np.array_equal(getattr(a, t).numpy()[~touched], getattr(b, t).numpy()[~touched]), t
    b.k.view().copy_(a.k.view())
    row = hub if pattern == "hub" else int(np.nonzero(pe - pb > 1)[0][5])
    b.do.view()[row, 1, 3] = what
    train(b)
    other = np.ones(n, bool)
    other[list(named_by[row])] = False
    for t in ("dk", "dvv"):
        assert np.array_equal(getattr(a, t).numpy()[other], getattr(b, t).numpy()[other]), t
    assert not np.isfinite(b.dvv.numpy()[~other][:, 0, 3]).any()
    keep = np.arange(m) != row
    assert np.array_equal(a.dq.numpy()[keep], b.dq.numpy()[keep])


@pytest.mark.parametrize("kind,maps", [("f32", 1), ("f16", 2), ("bf16", 2)])
@pytest.mark.parametrize("pattern", ["window", "apart", "hub"])
def test_scores_of_minus_infinity_only(kind, maps, pattern):
    """A row all of whose scores are minus infinity weighs nothing: zeros and lse = -infinity as for an empty row, and no part in
    the gradients."""
    m, n = 90, 700
    indx, pb, pe = pattern_of(pattern, m, n)
    a, b = pair(kind, maps, m, n, 2, 1, 32, 32 * maps, (indx, pb, pe))
    row = int(np.argmax(pe - pb)) if pattern == "hub" else int(np.nonzero(pe - pb > 4)[0][3])
    cols = np.unique(indx[pb[row]:pe[row]])
    for c in (a, b):
        c.k.view()[cols.tolist(), 0, 5] = 1.0            # finite keys that the row's query turns into minus infinity
        if maps == 2:
            c.k.view()[cols.tolist(), 0, 32 + 5] = 1.0
    b.q.view()[row, :, 5] = float("-inf")
    if maps == 2:
        b.q.view()[row, :, 32 + 5] = float("-inf")
    a.do.view()[row] = 0.0                               # (the row gives nothing to dk and dv)
    train(a, b)
    assert (b.o.numpy()[row] == 0).all()
    lse = b.lse[:-1].view(m, 2, maps).cpu().numpy()
    assert np.isneginf(lse[row]).all() and np.isfinite(lse[[i for i in range(m) if pe[i] > pb[i] and i != row]]).all()
    assert (b.dq.numpy()[row] == 0).all()
    keep = np.arange(m) != row
    for t in ("o", "dq"):
        assert np.array_equal(getattr(a, t).numpy()[keep], getattr(b, t).numpy()[keep]), t
    near = lambda x, y: np.abs(x - y).max() <= {"f32": 2.0 ** -22, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[kind] * np.abs(x).max()
    rest = np.array([f for f in range(32 * maps) if f % 32 != 5])                 # (0 times an infinite query is NaN)
    assert near(a.dvv.numpy(), b.dvv.numpy()) and near(a.dk.numpy()[:, :, rest], b.dk.numpy()[:, :, rest])
    assert b.rows() == 0
    assert (b.o.numpy()[row] == 0).all()


# ---- records of a cache ----------------------------------------------------------------------------------------------------

class Cached(Case):
    """A Case whose keys and values were written into a 4-bit cache."""

    def __init__(self, kind, maps, m, n, heads, kv, d, dv, indx, pb, pe, seed=0):
        import torch
        super().__init__(kind, maps, m, n, heads, kv, d, dv, indx, pb, pe, seed=seed)
        self.rec = fa.fusedMM_kv4_record_bytes(maps, d, dv)
        self.cache = torch.full((n, kv, self.rec), 0xA5, dtype=torch.uint8, device="cuda")
        every = torch.arange(n, dtype=torch.int32, device="cuda")
        assert fa.fusedMM_kv4_write(self.desc, n, every, self.k.ptr, self.v.ptr, self.cache, kv * self.rec, self.rec) == 0

    def rows_again(self, stream=None, nnz=None):
        return fa.fusedMM_attn_rows_kv4(self.desc, self.nnz if nnz is None else nnz, *self.index, self.q.ptr, self.cache, self.kv * self.rec,
                                        self.rec, self.lam, self.o.ptr, self.rows_work, self.rows_size, stream=stream)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("d,dv,maps", [(32, 32, 1), (64, 64, 1), (96, 64, 1), (128, 128, 1), (32, 96, 2), (64, 128, 2), (128, 256, 2)])
@pytest.mark.parametrize("nnz", [200, None])
def test_records_that_are_not_finite(kind, d, dv, maps, nnz):
    """NaN records in slots that nobody names, slot 0 among them, which masked places read, change nothing; a NaN group of values
    reaches its 32 features of the rows that name it, a NaN group of keys all of theirs."""
    import torch
    n, heads = 1100, 4
    lengths = [60, 0, 1000, 33, 700]
    indx, pb, pe = ragged(lengths, n - 101, seed=3)                 # (a masked place in every long row)
    indx = np.where(indx == n - 101, n, np.where(indx >= 0, indx + 1, indx))      # slot 0 is named by nobody
    a, b = [Cached(kind, maps, 5, n, heads, 2, d, dv, indx, pb, pe, seed=2) for _ in range(2)]
    unused = np.setdiff1d(np.arange(n), np.concatenate([indx[pb[i]:pe[i]] for i in range(5)]))
    assert unused[0] == 0 and len(unused) > 60
    where = lambda c: c.cache
    words = (maps * d + dv) // 2
    nan = torch.tensor([0x00, 0x7E], dtype=torch.uint8, device="cuda")
    where(b)[torch.as_tensor(unused).cuda()] = 0xFF
    where(b)[torch.as_tensor(unused[:40]).cuda(), :, words:words + (maps * d + dv) // 16] = nan.repeat((maps * d + dv) // 32)
    for c in (a, b):
        assert c.rows(nnz=nnz) == 0
    torch.cuda.synchronize()
    assert np.isfinite(a.o.numpy()).all() and torch.equal(a.o.buf, b.o.buf)
    bad = int(indx[pb[3] + 2])
    names = np.array([bad in indx[pb[i]:pe[i]] for i in range(5)])
    group = dv // 32 - 1                                            # the last group of values, of the second key head
    at = words + 2 * (maps * d // 32 + group)
    keep = where(b)[bad, 1, at:at + 2].clone()
    where(b)[bad, 1, at:at + 2] = nan
    assert b.rows(nnz=nnz) == 0
    torch.cuda.synchronize()
    x, y = a.o.numpy(), b.o.numpy()
    hit = np.zeros(x.shape, bool)
    hit[names, heads // 2:, 32 * group:32 * group + 32] = True
    assert np.isnan(y[hit]).all() and np.array_equal(x[~hit], y[~hit])
    where(b)[bad, 1, at:at + 2] = keep
    where(b)[bad, 0, words:words + 2] = nan                         # a group of keys, of the first key head
    assert b.rows(nnz=nnz) == 0
    torch.cuda.synchronize()
    y = b.o.numpy()
    hit = np.zeros(x.shape, bool)
    hit[names, :heads // 2] = True
    assert np.isnan(y[hit]).all() and np.array_equal(x[~hit], y[~hit])


def test_records_that_are_not_finite_against_the_formula():
    """A saturated record (values of 32768 codes) beside NaN ones: the finite rows follow the formula."""
    import torch
    n = 300
    c = CacheCase("f16", 1, 4, n, 2, 1, 64, 64, *ragged([300, 20, 0, 3], n, seed=5, masked=False), seed=6, scale=0.01)
    bad = int(c.indx[c.pb[0] + 250])
    clean = np.array([bad not in c.indx[c.pb[i]:c.pe[i]] for i in range(4)])
    c.cache.view(n, c.rec)[bad, 64:72] = torch.tensor([0x00, 0x7E] * 4, dtype=torch.uint8, device="cuda")
    assert c.rows() == 0
    torch.cuda.synchronize()
    e = c.exact()
    inside(c.o.numpy()[clean], e["o"][clean], e["tol"]["o"][clean], "o")
    assert np.isnan(c.o.numpy()[~clean]).all()
