"""Operands for the attention tests and calls of the entry points on them.  Tensors live inside larger buffers of a
sentinel value, so that a write outside what a call may write is seen."""
import numpy as np

import fusedmm_amd as fa

TORCH = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
SENTINEL = 7.5     # exact in every type


def dtype(kind):
    import torch
    return getattr(torch, TORCH[kind])


def layout(rows, heads, width, how):
    """(ld, hd, elements, offset): packed rows, head-major, packed rows inside wider ones (16-byte aligned), the same from an
    address off 16 bytes, or rows and heads at odd places."""
    if how == "packed":
        return heads * width, width, rows * heads * width, 0
    if how == "heads":
        return width, max(rows, 1) * width, rows * heads * width, 0
    if how == "wide":
        ld = heads * width + (-(heads * width)) % 8 + 16
        return ld, width, rows * ld + 8, 8
    if how == "off":     # strides of whole 16-byte chunks, for widths that are, behind an address that is not
        ld = heads * width + 8
        return ld, width, rows * ld + 1, 1
    ld = heads * (width + 3) + 5
    return ld, width + 3, rows * ld + 1, 1


class Tensor:
    """(rows, heads, width) in a device buffer, laid out by ld and hd."""

    def __init__(self, rows, heads, width, kind, how="packed", values=None):
        import torch
        self.rows, self.heads, self.width, self.kind = rows, heads, width, kind
        self.ld, self.hd, size, self.off = layout(rows, heads, width, how)
        self.buf = torch.full((size + 64,), SENTINEL, dtype=dtype(kind), device="cuda")
        if values is not None:
            self.view().copy_(torch.as_tensor(np.ascontiguousarray(values)).to("cuda").to(dtype(kind)).reshape(rows, heads, width))

    def view(self):
        return self.buf.as_strided((self.rows, self.heads, self.width), (self.ld, self.hd, 1), self.off)

    @property
    def ptr(self):
        return self.buf.data_ptr() + self.off * self.buf.element_size()

    def numpy(self):
        return self.view().double().cpu().numpy()

    def untouched_outside(self):
        """Every element that is not part of the tensor still holds the sentinel."""
        import torch
        mask = torch.ones_like(self.buf, dtype=torch.bool)
        mask.as_strided((self.rows, self.heads, self.width), (self.ld, self.hd, 1), self.off).fill_(False)
        return bool((self.buf[mask] == SENTINEL).all())


def desc(kind, maps, m, n, heads, kv, d, dv, scale, q=None, k=None, v=None, o=None):
    s = {}
    for name, t, h, w in (("q", q, heads, maps * d), ("k", k, kv, maps * d), ("v", v, kv, dv), ("o", o, heads, dv)):
        s["ld" + name], s["hd" + name] = (t.ld, t.hd) if t is not None else (h * w, w)
    return fa.AttnDesc(type=fa.TYPES[kind], maps=maps, m=m, n=n, heads=heads, kv_heads=kv, d=d, dv=dv, scale=scale, **s)


def index_arrays(indx, pb, pe, bits):
    import torch
    it = torch.int32 if bits == 32 else torch.int64
    return [torch.as_tensor(np.asarray(a)).to(it).cuda() for a in (indx, pb, pe)]


def transposed(m, n, indx, pb, pe):
    """CSC arrays of the pattern (ids outside [0, n) left out)."""
    rows = [[] for _ in range(n)]
    for i in range(m):
        for c in indx[pb[i]:pe[i]]:
            if 0 <= c < n:
                rows[c].append(i)
    ptr = np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int64)
    return np.array([x for r in rows for x in r], np.int64), ptr[:-1], ptr[1:]


def workspace(size):
    import torch
    return torch.full((max(int(size), 16),), 0x5A, dtype=torch.uint8, device="cuda")


class Case:
    """Random operands over a pattern; runs forward, backward, rows."""

    def __init__(self, kind, maps, m, n, heads, kv, d, dv, indx, pb, pe, seed=0, how="packed", bits=32, spread=1.0, scale=None):
        import torch
        rng = np.random.default_rng(seed)
        self.kind, self.maps, self.m, self.n, self.heads, self.kv, self.d, self.dv = kind, maps, m, n, heads, kv, d, dv
        self.indx, self.pb, self.pe, self.bits = np.asarray(indx, np.int64), np.asarray(pb, np.int64), np.asarray(pe, np.int64), bits
        self.scale = float(np.float32(1.0 / np.sqrt(d) if scale is None else scale))
        self.q = Tensor(m, heads, maps * d, kind, how, spread * rng.standard_normal((m, heads, maps * d)))
        self.k = Tensor(n, kv, maps * d, kind, how, spread * rng.standard_normal((n, kv, maps * d)))
        self.v = Tensor(n, kv, dv, kind, how, rng.standard_normal((n, kv, dv)))
        self.do = Tensor(m, heads, dv, kind, how, rng.standard_normal((m, heads, dv)))
        self.o, self.o2 = Tensor(m, heads, dv, kind, how), Tensor(m, heads, dv, kind, how)
        self.lam = torch.as_tensor(rng.uniform(0.2, 0.9, heads).astype(np.float32)).cuda() if maps == 2 else None
        self.lse = torch.full((m * heads * maps + 1,), SENTINEL, dtype=torch.float32, device="cuda")
        self.desc = desc(kind, maps, m, n, heads, kv, d, dv, self.scale, self.q, self.k, self.v, self.o)
        self.index = index_arrays(self.indx, self.pb, self.pe, bits)
        self.nnz = int(np.maximum(self.pe - self.pb, 0).sum())
        self.plan = self.plan_t = None

    def make_plans(self, backward):
        self.plan = fa.AttnPlan(self.m, self.n, self.nnz, *self.index, index_bits=self.bits)
        if backward:
            t = transposed(self.m, self.n, self.indx, self.pb, self.pe)
            self.tindex = index_arrays(*t, self.bits)
            self.plan_t = fa.AttnPlan(self.n, self.m, len(t[0]), *self.tindex, index_bits=self.bits)
        size = fa.fusedMM_attn_workspace(self.desc, self.plan, self.plan_t, index_bits=self.bits)
        assert size >= 0
        self.work, self.size = workspace(size), size

    def forward(self, stream=None, save=True):
        return fa.fusedMM_attn_forward(self.desc, self.plan, self.q.ptr, self.k.ptr, self.v.ptr, self.lam, self.o.ptr,
                                       self.o2.ptr if save and self.maps == 2 else None, self.lse if save else None, self.work,
                                       self.size, stream=stream, index_bits=self.bits)

    def gradients(self, how="packed"):
        import torch
        self.dq, self.dk = Tensor(self.m, self.heads, self.maps * self.d, self.kind, how), Tensor(self.n, self.kv, self.maps * self.d, self.kind, how)
        self.dvv = Tensor(self.n, self.kv, self.dv, self.kind, how)
        self.dlam = torch.full((self.heads,), SENTINEL, dtype=torch.float32, device="cuda")

    def backward(self, stream=None):
        return fa.fusedMM_attn_backward(self.desc, self.plan, self.plan_t, self.q.ptr, self.k.ptr, self.v.ptr, self.lam, self.o.ptr,
                                        self.o2.ptr if self.maps == 2 else None, self.lse, self.do.ptr, self.dq.ptr, self.dk.ptr,
                                        self.dvv.ptr, self.dlam if self.maps == 2 else None, self.work, self.size, stream=stream,
                                        index_bits=self.bits)

    def rows(self, stream=None, nnz=None):
        nnz = self.nnz if nnz is None else nnz
        size = fa.fusedMM_attn_rows_workspace(self.desc, nnz, index_bits=self.bits)
        assert size >= 0
        self.rows_work, self.rows_size = workspace(size), size
        return self.rows_again(stream, nnz)

    def rows_again(self, stream=None, nnz=None):
        return fa.fusedMM_attn_rows(self.desc, self.nnz if nnz is None else nnz, *self.index, self.q.ptr, self.k.ptr, self.v.ptr,
                                    self.lam, self.o.ptr, self.rows_work, self.rows_size, stream=stream, index_bits=self.bits)

    def exact(self, do=False, k=None, v=None, weight_type=None):
        from attn_reference import attention, counts
        q = self.q.numpy().reshape(self.m, self.heads, self.maps, self.d)
        k = self.k.numpy() if k is None else k
        v = self.v.numpy() if v is None else v
        lam = self.lam.double().cpu().numpy() if self.maps == 2 else None
        return attention(counts(self.m, self.n, self.indx, self.pb, self.pe), q, k.reshape(self.n, self.kv, self.maps, self.d), v, lam,
                         self.scale, self.kind, self.do.numpy() if do else None, weight_type=weight_type)


def inside(got, want, tol, what):
    got, want = np.asarray(got, np.float64).reshape(want.shape), want
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - want) - tol)
    bad = ~(off <= 0)
    assert not bad.any(), "%s: %d of %d outside, first at %s: %r, exact %r, allowed %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got[tuple(np.argwhere(bad)[0])], want[tuple(np.argwhere(bad)[0])],
        np.broadcast_to(tol, want.shape)[tuple(np.argwhere(bad)[0])])


def random_pattern(m, n, degree, seed, empty=True, duplicates=True, masked=True, hub=0):
    """Rows of up to `degree` columns in any order; some empty, some columns twice, some ids outside the columns; the rows'
    slots lie apart from each other.  hub: row m // 2 has that many."""
    rng = np.random.default_rng(seed)
    indx, pb, pe = [], [], []
    for i in range(m):
        deg = int(rng.integers(0 if empty else 1, degree + 1))
        if empty and i % 11 == 3:
            deg = 0
        if hub and i == m // 2:
            deg = hub
        cols = rng.integers(0, n, deg)
        if not duplicates:
            cols = np.unique(cols)
        if masked and len(cols) > 2:
            cols[rng.integers(0, len(cols))] = rng.choice([-1, n, n + 5, -(2 ** 31)])
        pb.append(len(indx))
        indx.extend(cols.tolist())
        pe.append(len(indx))
        indx.extend([12345] * int(rng.integers(0, 3)))      # slots between the rows that belong to none
    return np.array(indx + [0], np.int64), np.array(pb, np.int64), np.array(pe, np.int64)


def window_pattern(m, n, window):
    indx, pb, pe = [], [], []
    for i in range(m):
        pos = i + n - m
        pb.append(len(indx))
        indx.extend(range(max(0, pos - window + 1), pos + 1))
        pe.append(len(indx))
    return np.array(indx, np.int64), np.array(pb, np.int64), np.array(pe, np.int64)
