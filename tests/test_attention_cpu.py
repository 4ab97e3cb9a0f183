"""What the attention entry points refuse before they touch a device, the record format of the 4-bit cache, and the 64-bit
reference itself."""
import ctypes as C
import os

import numpy as np
import pytest

import fusedmm_amd as fa
from attn_reference import attention, counts, quantise_group, quantise_row, record


def desc(**kw):
    d = dict(type=fa.TYPE_BF16, maps=1, m=4, n=100, heads=4, kv_heads=2, d=64, dv=64, scale=0.125, ldq=256, hdq=64, ldk=128, hdk=64,
             ldv=128, hdv=64, ldo=256, hdo=64)
    d.update(kw)
    return fa.AttnDesc(**d)


def rows(d, nnz=10, q=16, k=16, v=16, o=16, lam=None, work=None, size=0, index_bits=32):
    return fa.fusedMM_attn_rows(d, nnz, 16, 16, 16, q, k, v, lam, o, work, size, stream=0, index_bits=index_bits)


def rows4(d, nnz=10, cache=16, ldc=160, hdc=80, o=16, lam=None):
    return fa.fusedMM_attn_rows_kv4(d, nnz, 16, 16, 16, 16, cache, ldc, hdc, lam, o, None, 0, stream=0)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("change,why", [
    (dict(type=3), "element type"), (dict(maps=0), "maps"), (dict(maps=3), "maps"), (dict(m=-1), "negative size"),
    (dict(n=-1), "negative size"), (dict(kv_heads=0), "at least 1"), (dict(d=0), "at least 1"), (dict(dv=-2), "at least 1"),
    (dict(heads=5), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(ldq=-1), "stride"),
    (dict(hdk=1 << 50), "stride"), (dict(hdo=63), "rows of o overlap"), (dict(ldo=200), "rows of o overlap"),
    (dict(n=1 << 31), "2^31"), (dict(m=1 << 31, ldo=1 << 20), "too many rows"), (dict(maps=2), "null")])
def test_rows_refuse_what_does_not_fit(capfd, bits, change, why):
    assert rows(desc(**change), index_bits=bits) == fa.FAIL
    assert why in capfd.readouterr().err


def test_rows_refuse_null_pointers_and_negative_counts(capfd):
    for kw in (dict(q=None), dict(o=None), dict(k=None), dict(v=None)):
        assert rows(desc(), **kw) == fa.FAIL
        assert "null" in capfd.readouterr().err
    assert rows(desc(), nnz=-1) == fa.FAIL
    assert "negative nnz" in capfd.readouterr().err
    assert fa.load(32).fusedMM_attn_rows(None, 1, None, None, None, None, None, None, None, None, None, 0, None) == fa.FAIL
    assert fa.fusedMM_attn_rows_workspace(desc(), -1) == -1


def test_sizes_without_a_kernel():
    for change in (dict(d=257), dict(dv=257), dict(maps=2, d=129, dv=64), dict(maps=2, dv=257)):
        assert rows(desc(**change)) == fa.NO_OPT_IMPL
        assert fa.fusedMM_attn_rows_workspace(desc(**change), 10) == -1
    for change in (dict(d=256, dv=256), dict(maps=2, d=128, dv=256), dict(d=1, dv=1)):
        assert fa.fusedMM_attn_rows_workspace(desc(**change), 10) == 0


def test_workspace_of_rows():
    assert fa.fusedMM_attn_rows_workspace(desc(), 200) == 0              # nothing to cut
    need = fa.fusedMM_attn_rows_workspace(desc(), 100000)
    assert need > 0
    assert rows(desc(), nnz=100000) == fa.NOT_ENOUGH_MEM
    assert rows(desc(), nnz=100000, work=16, size=need - 1) == fa.NOT_ENOUGH_MEM
    assert rows(desc(), nnz=100000, work=24, size=need) == fa.FAIL       # alignment
    assert fa.fusedMM_attn_rows_workspace(desc(m=1000), 100000) > need


def test_no_rows_is_success_without_a_device():
    assert rows(desc(m=0), q=None, o=None) == 0
    assert rows4(desc(m=0)) == 0
    s = fa.fusedMM_kv4_write(desc(), 0, None, None, None, None, 160, 80, stream=0)
    assert s == 0


def test_plans_refuse_what_does_not_fit(capfd):
    lib = fa.load(32)
    h = C.c_void_p(5)
    for args, why in (((-1, 1, 1, 16, 16, 16), "from 0 to"), ((1, 1 << 26, 1, 16, 16, 16), "from 0 to"), ((1, 1, -1, 16, 16, 16), "negative"),
                      ((1, 1, 1, None, 16, 16), "null"), ((1, 1, 1, 16, None, 16), "null")):
        assert lib.fusedMM_attn_plan_create(*args, None, C.byref(h)) == fa.FAIL
        assert why in capfd.readouterr().err
        assert not h.value
    assert lib.fusedMM_attn_plan_create(1, 1, 1, 16, 16, 16, None, None) == fa.FAIL
    assert lib.fusedMM_attn_plan_destroy(None) == 0
    for call in (lambda: fa.fusedMM_attn_forward(desc(), None, 16, 16, 16, None, 16, None, None, None, 0, stream=0),
                 lambda: fa.fusedMM_attn_backward(desc(), None, None, 16, 16, 16, None, 16, None, 16, 16, 16, 16, 16, None, None, 0, stream=0)):
        assert call() == fa.FAIL
        assert "no plan" in capfd.readouterr().err
    assert fa.fusedMM_attn_workspace(desc(), None) == -1
    not_a_plan = np.zeros(64, np.int64)
    assert fa.fusedMM_attn_forward(desc(), not_a_plan.ctypes.data, 16, 16, 16, None, 16, None, None, None, 0, stream=0) == fa.FAIL


def test_the_cache_refuses_what_does_not_fit(capfd):
    write = lambda d, tokens=3, ldc=160, hdc=80, cache=16, slots=16: fa.fusedMM_kv4_write(d, tokens, slots, 16, 16, cache, ldc, hdc, stream=0)
    read = lambda d, tokens=3, ldc=160, hdc=80, cache=16: fa.fusedMM_kv4_read(d, tokens, 16, cache, ldc, hdc, 16, 16, stream=0)
    for call in (write, read, lambda d, **kw: rows4(d, **{k: v for k, v in kw.items() if k != "tokens"})):
        assert call(desc(d=40)) == fa.NO_OPT_IMPL
        assert call(desc(dv=48)) == fa.NO_OPT_IMPL
        assert call(desc(d=288)) == fa.NO_OPT_IMPL
        for kw in (dict(ldc=168), dict(hdc=72), dict(cache=24), dict(ldc=-160)):
            assert call(desc(), **kw) == fa.FAIL
            assert "16-byte" in capfd.readouterr().err
    for call in (write, read):
        assert call(desc(), tokens=-1) == fa.FAIL
        assert "negative" in capfd.readouterr().err
        assert call(desc(), cache=None) == fa.FAIL
        assert "null" in capfd.readouterr().err
    assert write(desc(), ldc=80) == fa.FAIL and "overlap" in capfd.readouterr().err
    assert write(desc(), tokens=(1 << 20) + 1) == fa.FAIL and "2^20" in capfd.readouterr().err
    assert read(desc(ldk=64)) == fa.FAIL and "overlap" in capfd.readouterr().err
    assert rows4(desc(type=fa.TYPE_F32)) == fa.NO_OPT_IMPL
    for sizes in (dict(maps=2, d=96, dv=160, heads=4, kv_heads=4), dict(d=160, dv=160), dict(d=256, dv=128), dict(d=32, dv=160), dict(maps=2, d=32, dv=256)):
        assert rows4(desc(ldq=1024, hdq=256, ldo=1024, hdo=256, **sizes), ldc=2048, hdc=512, lam=16) == fa.NO_OPT_IMPL


def test_record_bytes():
    lib = fa.load(64)
    assert [lib.fusedMM_kv4_record_bytes(*a) for a in ((1, 64, 64), (1, 128, 128), (2, 64, 128), (1, 32, 32), (2, 128, 256))] == [80, 144, 144, 48, 288]
    for a in ((1, 40, 64), (1, 64, 0), (3, 64, 64), (1, 288, 64), (2, 160, 64)):
        assert lib.fusedMM_kv4_record_bytes(*a) == -1


def test_no_gpu_is_a_status_code():
    """With no device to be seen, well-formed calls return FUSEDMM_FAIL_RETURN."""
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    body = ("import sys; sys.path.insert(0, %r); sys.path.insert(0, %r)\n"
            "from test_attention_cpu import desc, rows, rows4\nimport fusedmm_amd as fa, ctypes as C\n"
            "h = C.c_void_p()\n"
            "print('rc', rows(desc()), rows4(desc()), fa.fusedMM_kv4_write(desc(), 1, 16, 16, 16, 16, 160, 80, stream=0),\n"
            "      fa.load(32).fusedMM_attn_plan_create(1, 1, 1, 16, 16, 16, None, C.byref(h)))\n" % (root, os.path.join(root, "tests")))
    env = dict(os.environ, HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="", CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", body], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=120, env=env)
    assert r.returncode == 0 and "rc 1 1 1 1" in r.stdout, r.stdout + r.stderr[-2000:]


def test_quantised_values_stay_within_their_step():
    """The nearest of 16 levels: half a step off, one and a half at an end where both roundings go outwards; exact in fp16; a
    value of the cache quantises to itself."""
    rng = np.random.default_rng(0)
    for scale in (1e-5, 0.02, 1.0, 300.0, 3e4):
        for shift in (0.0, 3.0, -3.0):
            x = np.clip((rng.standard_normal(32) + shift) * scale, -32768, 32768)
            s, z, c = quantise_group(x)
            y = s * (c - z)
            assert 0 <= z <= 15 and c.min() >= 0 and c.max() <= 15
            assert np.abs(x - y).max() <= s * (1 + 1e-12)
            assert np.median(np.abs(x - y)) <= s / 2
            assert (y.astype(np.float16).astype(np.float64) == y).all()
# rounded up by less than one unit, which is 2^-20 or at most 2^-6 of the step
            step = (max(x.max(), 0) - min(x.min(), 0)) / 15
            assert step <= s <= step + max(2.0 ** -20, step * 2.0 ** -6)
    b, kx, vx = record(rng.standard_normal(64), rng.standard_normal(64))
    assert len(b) == 80 and (b[72:] == 0).all()
    again = quantise_row(kx)[2]
    assert np.abs(again - kx).max() <= 0.5 * np.abs(kx).max() / 7


def test_reference_against_a_loop():
    """The dense 64-bit reference against softmax written out edge by edge."""
    rng = np.random.default_rng(1)
    m, n, heads, kv, d, dv = 5, 6, 2, 1, 3, 4
    q, k, v, lam = rng.standard_normal((m, heads, 2, d)), rng.standard_normal((n, kv, 2, d)), rng.standard_normal((n, kv, dv)), rng.uniform(0, 1, heads)
    indx, pb, pe = np.array([0, 1, 1, 5, -1, 2, 6, 3]), np.array([0, 3, 3, 4, 5]), np.array([3, 3, 4, 8, 6])
    e = attention(counts(m, n, indx, pb, pe), q, k, v, lam, 0.7, "f32")
    for i in range(m):
        for h in range(heads):
            cols = [c for c in indx[pb[i]:pe[i]] if 0 <= c < n]
            o = np.zeros(dv)
            for p, sign in ((0, 1.0), (1, -lam[h])):
                if cols:
                    w = np.exp([0.7 * q[i, h, p] @ k[c, 0, p] for c in cols])
                    o += sign * sum(x * v[c, 0] for x, c in zip(w / w.sum(), cols))
                    assert abs(np.log(w.sum()) - e["lse"][i, h, p]) < 1e-12
            assert np.abs(o - e["o"][i, h]).max() < 1e-12


@pytest.mark.parametrize("bits,nnz,change", [
    (64, 2 ** 62, {}), (64, 2 ** 44, {}), (64, 100, dict(m=2 ** 62)), (64, 100, dict(m=2 ** 20, heads=2 ** 20, ldo=2 ** 26)),
    (32, 100, dict(m=1, heads=2 ** 31 - 1, kv_heads=2 ** 31 - 1)), (64, 2 ** 40, dict(m=1, heads=2 ** 20, kv_heads=2 ** 20))])
def test_rows_refuse_sizes_beyond_a_launch(capfd, bits, nnz, change):
    """No product of sizes wraps round into a small workspace."""
    d = desc(**change)
    assert fa.fusedMM_attn_rows_workspace(d, nnz, index_bits=bits) == -1
    assert "too many rows, slots and heads" in capfd.readouterr().err
    assert rows(d, nnz=nnz, work=16, size=2 ** 62, index_bits=bits) == fa.FAIL
    assert "too many rows, slots and heads" in capfd.readouterr().err


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 40])
def test_the_cache_refuses_slots_beyond_32_bits(capfd, n):
    d = desc(n=n)
    for call in (lambda: fa.fusedMM_kv4_write(d, 1, 16, 16, 16, 16, 160, 80, stream=0, index_bits=64),
                 lambda: fa.fusedMM_kv4_read(d, 1, 16, 16, 160, 80, 16, 16, stream=0, index_bits=64)):
        assert call() == fa.FAIL
        assert "2^31 - 1" in capfd.readouterr().err
