"""Attention calls at the edges of what the entry points allow: signs of the scale, head sizes under a 16-byte chunk,
strides whose offsets pass 32 bits, blocks of 16 and of 64 rows, several calls at once, graphs that share a workspace."""
import numpy as np
import pytest

import fusedmm_amd as fa
from attn_run import Case, index_arrays, inside, random_pattern, transposed, window_pattern, workspace
from test_gpu_attention import check_backward, check_forward, run_both
from test_gpu_attention_rows import CacheCase, check_rows, ragged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30])
@pytest.mark.parametrize("kind,maps", [("f32", 1), ("bf16", 2)])
def test_scales(kind, maps, scale):
    """Negative scales turn the order of the scores round; zero makes every weight alike."""
    import torch
    c = Case(kind, maps, 70, 60, 4, 2, 32, 32 * maps, *random_pattern(70, 60, 30, seed=1), seed=2, scale=scale)
    run_both(c)
    e = c.exact()
    assert c.rows() == 0
    torch.cuda.synchronize()
    check_rows(c, e)
    if kind != "f32":
        r = CacheCase(kind, maps, 6, 310, 4, 2, 32, 32 * maps, *ragged([0, 1, 33, 128, 300, 2], 310, seed=1), seed=2, scale=scale)
        assert r.rows() == 0
        torch.cuda.synchronize()
        check_rows(r, r.exact())


# (d, dv, maps): shorter than a chunk of 4 or 8 elements, a chunk and a bit, one of the two short
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dv,maps", [(2, 3, 1), (3, 5, 2), (7, 1, 1), (9, 5, 2), (5, 40, 1), (17, 15, 2), (33, 31, 1), (8, 4, 1)])
@pytest.mark.parametrize("how", ["packed", "odd"])
def test_small_heads(kind, d, dv, maps, how):
    import torch
    c = Case(kind, maps, 50, 45, 4, 2, d, dv, *random_pattern(50, 45, 20, seed=d), seed=dv, how=how)
    run_both(c, how)
    assert c.rows() == 0
    torch.cuda.synchronize()
    check_rows(c, c.exact())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dv,maps", [(32, 32, 1), (64, 64, 1), (128, 128, 1), (32, 64, 2), (64, 128, 2), (48, 40, 1), (91, 117, 1), (45, 83, 2)])
@pytest.mark.parametrize("pattern", ["shared", "apart"])
def test_blocks_of_64_and_of_16_rows(kind, d, dv, maps, pattern):
    """Rows that share their columns (blocks of 64 rows) and rows that share none (blocks of 16), over several tiles."""
    m, n = 100, 1700
    if pattern == "shared":
        indx, pb, pe = window_pattern(m, n, 70)
    else:
        rng = np.random.default_rng(d)
        indx, pb, pe = rng.permutation(n)[:m * 17].astype(np.int64), np.arange(m) * 17, np.arange(m) * 17 + 17 - np.arange(m) % 3
    run_both(Case(kind, maps, m, n, 3, 3, d, dv, indx, pb, pe, seed=d + dv))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dv,maps", [(32, 32, 1), (64, 64, 1), (128, 128, 1), (64, 128, 2), (40, 24, 1), (8, 16, 2)])
@pytest.mark.parametrize("pattern", ["shared", "apart"])
def test_tensors_that_begin_off_16_bytes(kind, d, dv, maps, pattern):
    import torch
    m, n = 70, 1300
    if pattern == "shared":
        indx, pb, pe = window_pattern(m, n, 70)
    else:
        indx, pb, pe = np.random.default_rng(d).permutation(n)[:m * 18].astype(np.int64), np.arange(m) * 18, np.arange(m) * 18 + 18
    c = Case(kind, maps, m, n, 4, 2, d, dv, indx, pb, pe, seed=d + dv, how="off")
    run_both(c, "off")
    assert c.rows() == 0
    torch.cuda.synchronize()
    check_rows(c, c.exact())


def test_odd_sizes_are_captured_and_replayed():
    """Rows that are laid out anew within the call: the graph does so at every replay."""
    import torch
    c = Case("bf16", 2, 90, 120, 4, 2, 21, 37, *random_pattern(90, 120, 30, seed=1), seed=2)
    c.make_plans(True)
    c.gradients()
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        assert c.forward(stream=s.cuda_stream) == 0 and c.backward(stream=s.cuda_stream) == 0
    for _ in range(3):
        for t in (c.q, c.k, c.v, c.do):
            t.view().copy_(torch.randn(t.view().shape, device="cuda"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        e = c.exact(do=True)
        check_forward(c, e)
        check_backward(c, e)
        float(torch.randn(1000, device="cuda").sum())


def far(t, ld):
    """The tensor's values in rows `ld` elements apart."""
    import torch
    buf = torch.empty((t.rows - 1) * ld + t.heads * t.hd, dtype=t.buf.dtype, device="cuda")
    view = buf.as_strided((t.rows, t.heads, t.width), (ld, t.hd, 1))
    view.copy_(t.view())
    return buf, view


@pytest.mark.parametrize("ld", [1 << 20, (1 << 20) + 3])
def test_offsets_beyond_32_bits(ld):
    """Keys, values and their gradients 2 MiB apart, 4.6 GB of each."""
    import torch
    n = 2300
    rng = np.random.default_rng(1)
    lengths = np.array([17, 0, 900, 3, 40, 1200])
    ends = np.cumsum(lengths)
    indx = np.concatenate([np.sort(rng.permutation(n)[:x]) for x in lengths])
    indx[16], indx[-1] = n - 1, n - 1
    c = Case("bf16", 1, 6, n, 4, 2, 64, 64, indx, ends - lengths, ends, seed=1)
    run_both(c)
    e = c.exact(do=True)
    (kb, _), (vb, _) = far(c.k, ld), far(c.v, ld)
    near = (c.desc.ldk, c.desc.ldv)
    assert c.rows() == 0     # (for its workspace)
    c.o.view().zero_()
    c.desc.ldk = c.desc.ldv = ld
    assert fa.fusedMM_attn_rows(c.desc, c.nnz, *c.index, c.q.ptr, kb, vb, None, c.o.ptr, c.rows_work, c.rows_size) == 0
    torch.cuda.synchronize()
    check_rows(c, e)
    c.make_plans(True)
    c.gradients()
    assert fa.fusedMM_attn_forward(c.desc, c.plan, c.q.ptr, kb, vb, None, c.o.ptr, None, c.lse, c.work, c.size) == 0
    torch.cuda.synchronize()
    check_forward(c, e)
    dkb, dvb = torch.empty_like(kb), torch.empty_like(vb)
    assert fa.fusedMM_attn_backward(c.desc, c.plan, c.plan_t, c.q.ptr, kb, vb, None, c.o.ptr, None, c.lse, c.do.ptr, c.dq.ptr, dkb, dvb,
                                    None, c.work, c.size) == 0
    torch.cuda.synchronize()
    for near_t, b in ((c.dk, dkb), (c.dvv, dvb)):
        near_t.view().copy_(b.as_strided((n, 2, 64), (ld, near_t.hd, 1)))
    check_backward(c, e)
    c.desc.ldk, c.desc.ldv = near


def test_a_cache_beyond_32_bits():
    """Records 2 MiB apart, 4.6 GB: written, read back and attended as packed ones are."""
    import torch
    n, ldc = 2300, (1 << 21) + 16
    lengths = [17, 0, 900, 3, 40, 1200]
    c = CacheCase("bf16", 1, 6, n, 4, 2, 64, 64, *ragged(lengths, n, seed=1), seed=1)
    assert c.rows() == 0
    torch.cuda.synchronize()
    want = c.o.buf.clone()
    cache = torch.empty((n - 1) * ldc + 2 * c.hdc, dtype=torch.uint8, device="cuda")
    every = index_arrays(np.arange(n), [0], [0], 32)[0]
    assert fa.fusedMM_kv4_write(c.desc, n, every, c.k.ptr, c.v.ptr, cache, ldc, c.hdc) == 0
    c.o.buf.view(torch.int16).zero_()
    want_view = want.as_strided(c.o.view().shape, c.o.view().stride(), c.o.off)
    assert fa.fusedMM_attn_rows_kv4(c.desc, c.nnz, *c.index, c.q.ptr, cache, ldc, c.hdc, None, c.o.ptr, c.rows_work, c.rows_size) == 0
    k, v = torch.empty((n, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.empty((n, 2, 64), dtype=torch.bfloat16, device="cuda")
    k0, v0 = torch.empty_like(k), torch.empty_like(v)
    assert fa.fusedMM_kv4_read(c.desc, n, every, cache, ldc, c.hdc, k, v) == 0
    assert fa.fusedMM_kv4_read(c.desc, n, every, c.cache, c.ldc, c.hdc, k0, v0) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.o.view(), want_view) and torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("m", [257, 600])
def test_many_rows_over_the_cache(m):
    import torch
    rng = np.random.default_rng(m)
    lengths = rng.integers(0, 12, m)
    lengths[m // 3], lengths[m - 1] = 900, 700
    c = CacheCase("f16", 1, m, 1000, 2, 1, 32, 32, *ragged(lengths, 1000, seed=1), seed=2)
    assert c.rows() == 0
    torch.cuda.synchronize()
    assert c.rows_size > 0
    check_rows(c, c.exact())


@pytest.mark.parametrize("kind,maps", [("f32", 2), ("bf16", 1)])
def test_rows_of_many_pieces(kind, maps):
    """More pieces than one batch of the join, joined by four waves and, where rows are few, by sixteen."""
    import torch
    for lengths in ([150000], [9000, 1, 0, 7000, 300, 12000, 2, 5]):
        c = Case(kind, maps, len(lengths), 20000, 2, 1, 32, 32 * maps, *ragged(lengths, 20000, seed=1), seed=2)
        assert c.rows(nnz=c.nnz) == 0
        torch.cuda.synchronize()
        check_rows(c, c.exact())


def test_gradients_without_that_of_lambda():
    import torch
    c = Case("f32", 2, 40, 50, 4, 2, 16, 32, *random_pattern(40, 50, 20, seed=1), seed=2)
    run_both(c)
    want = [t.buf.clone() for t in (c.dq, c.dk, c.dvv)]
    c.gradients()
    assert fa.fusedMM_attn_backward(c.desc, c.plan, c.plan_t, c.q.ptr, c.k.ptr, c.v.ptr, c.lam, c.o.ptr, c.o2.ptr, c.lse, c.do.ptr, c.dq.ptr,
                                    c.dk.ptr, c.dvv.ptr, None, c.work, c.size) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(t.buf, w) for t, w in zip((c.dq, c.dk, c.dvv), want))
    assert (c.dlam == 7.5).all()


def test_calls_at_once():
    """A training pass, rows and rows over a cache on three streams at once, with one plan for two of the calls, have the
    bits that they have alone."""
    import torch
    c = Case("bf16", 2, 200, 700, 4, 2, 32, 64, *random_pattern(200, 700, 60, seed=9, hub=1500), seed=3)
    e = Case("bf16", 2, 200, 700, 4, 2, 32, 64, c.indx, c.pb, c.pe, seed=4)
    r = CacheCase("bf16", 2, 5, 3000, 4, 2, 32, 64, *ragged([3000, 7, 0, 2000, 900], 3000, seed=1), seed=5)
    for x in (c, e):
        x.make_plans(True)
        x.gradients()
    e.plan, e.plan_t = c.plan, c.plan_t      # one plan, two workspaces

    def passes(streams):
        s = [x.cuda_stream for x in streams]
        assert c.forward(stream=s[0]) == 0 and e.forward(stream=s[1]) == 0 and r.rows_again(stream=s[2]) == 0
        assert c.backward(stream=s[0]) == 0 and e.backward(stream=s[1]) == 0 and r.rows_again(stream=s[2]) == 0

    def results():
        torch.cuda.synchronize()
        return [t.clone() for x in (c, e) for t in (x.o.buf, x.o2.buf, x.lse, x.dq.buf, x.dk.buf, x.dvv.buf, x.dlam)] + [r.o.buf.clone()]

    assert r.rows() == 0
    alone = torch.cuda.Stream()
    passes([alone] * 3)
    want = results()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        passes(streams)
        assert all(torch.equal(a, b) for a, b in zip(results(), want))


def test_graphs_that_share_a_workspace():
    """Two captured calls with one workspace, replayed in turn on one stream."""
    import torch
    c = Case("f16", 1, 150, 700, 4, 2, 64, 64, *random_pattern(150, 700, 60, seed=9, hub=1500), seed=3)
    e = Case("f16", 1, 150, 700, 4, 2, 64, 64, c.indx, c.pb, c.pe, seed=4)
    for x in (c, e):
        run_both(x)
        x.want = [t.buf.clone() for t in (x.o, x.dq, x.dk, x.dvv)]
    e.work, e.size = c.work, c.size = workspace(max(c.size, e.size)), max(c.size, e.size)
    torch.cuda.synchronize()
    s, graphs = torch.cuda.Stream(), []
    for x in (c, e):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            assert x.forward(stream=s.cuda_stream) == 0 and x.backward(stream=s.cuda_stream) == 0
        graphs.append(g)
    for _ in range(3):
        for x in (c, e):
            for t in (x.o, x.dq, x.dk, x.dvv):
                t.view().zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x in (c, e):
            assert all(torch.equal(t.buf, w) for t, w in zip((x.o, x.dq, x.dk, x.dvv), x.want))
        float(torch.randn(1000, device="cuda").sum())
