"""The addresses of the attention over a 4-bit cache, restated and checked on the host: every lane, word, map and size that
fusedMM_attn_rows_kv4 has a kernel for, and the sizes that it refuses (two maps of 96 with values of 160 and their like)."""
import numpy as np
import pytest

import fusedmm_amd as fa

LANE = np.arange(64)
G, I = LANE >> 4, LANE & 15


def width_class(d, dv, maps):
    return next(c for c in (32, 64, 128, 256) if d <= c and dv <= maps * c)


def sizes(refused):
    out = []
    for maps in (1, 2):
        for d in range(32, (256 if maps == 1 else 128) + 1, 32):
            for dv in range(32, 257, 32):
                dc = width_class(d, dv, maps)
                if (dc * maps == 256 and (d != dc or dv != 256)) == refused:
                    out.append((maps, d, dv, dc, d == dc and dv == dc * maps))
    return out


class Bytes:
    """How often each byte of a span of memory is read or written."""

    def __init__(self, size):
        self.count = np.zeros(size, np.int64)

    def touch(self, at, length):
        at = np.atleast_1d(at)
        assert (at >= 0).all() and (at + length <= len(self.count)).all(), (at.min(), at.max(), length, len(self.count))
        assert (at % min(length, 16) == 0).all(), "not on a multiple of its size"
        for b in range(length):
            np.add.at(self.count, at + b, 1)


def code_feature(full, words, j, g):
    return g * (words * 8) + 8 * j if full else 32 * j + 8 * g


def load_codes(mem, base, full, words, width):
    if full and words % 4 == 0:
        for j in range(words // 4):
            mem.touch(base + G[::16] * (words * 4) + 16 * j, 16)
    elif full and words == 2:
        mem.touch(base + G[::16] * 8, 8)
    else:
        for j in range(words):
            if 32 * j < width:
                mem.touch(base + 16 * j + 4 * G[::16], 4)


def load_scales(mem, base, full, words, width):
    for j in range((words + 3) // 4 if full else words):
        f = code_feature(full, words, 4 * j if full else j, G[::16])
        f = f if full else f[f < width]
        if len(f):
            mem.touch(base + f // 32 * 2, 2)


def check_record(maps, d, dv, dc, full):
    """One lane group's loads of one slot: inside the record, aligned, every code exactly once, every word at least once."""
    kw, w = maps * d, dc * maps
    rec = fa.fusedMM_kv4_record_bytes(maps, d, dv)
    mem = Bytes(rec)
    off_v, off_kw = kw // 2, (kw + dv) // 2
    off_vw = off_kw + kw // 16
    for mp in range(maps):
        load_codes(mem, mp * d // 2, full, dc // 32, d)
        load_scales(mem, off_kw + mp * d // 16, full, dc // 32, d)
    load_codes(mem, off_v, full, w // 32, dv)
    load_scales(mem, off_vw, full, w // 32, dv)
    assert (mem.count[:off_kw] == 1).all()
    assert (mem.count[off_kw:off_kw + (kw + dv) // 16] >= 1).all() and (mem.count[off_kw + (kw + dv) // 16:] == 0).all()


def check_tile(maps, d, dv, dc, full):
    """The wave's tile of values: every 16-byte chunk of its 32 rows written once; the reads of the second product inside it."""
    w = dc * maps
    rb, cr = 2 * w, 2 * w // 16
    rows_per, mask = (1, 15) if cr >= 16 else (16 // cr, cr - 1)
    twist = lambda row: (row // rows_per) & mask
    mem = Bytes(32 * rb)
    for a in (0, 1):
        for j in range(w // 32):
            f = code_feature(full, w // 32, j, G)
            mem.touch((16 * a + I) * rb + ((f // 8) ^ twist(I)) * 16, 16)
    assert (mem.count == 1).all()
    start = (4 * G + I // 4) * rb + ((((I % 4) // 2) ^ twist(4 * G + I // 4)) * 16) + (I % 2) * 8
    mem = Bytes(32 * rb)
    for t in range(w // 16):
        for half in (0, 16 * rb):
            mem.touch((start ^ (2 * t * 16)) + half, 8)
    assert (mem.count == 1).all()
    mem = Bytes(32 * rb)                                       # the sums of 16 columns, as floats
    for x in range(w // 16):
        mem.touch((I * w + 16 * x + 4 * G) * 4, 16)
    assert (mem.count == 1).all()
    for key in range(32):                                      # single elements, in the pass for values that are not finite
        f = np.arange(w)
        at = key * rb + (((f // 8) ^ twist(key)) * 16) + (f % 8) * 2
        assert (np.sort(at) == key * rb + 2 * f).all()


def check_query(maps, d, dv, dc, full, heads, kv):
    """A row's query: every chunk inside its head and map."""
    hp, group = 16 // maps, heads // kv
    for kvh in range(kv):
        for p in range(-(-group // hp)):
            hh = p * hp + I % hp
            col = hh < group
            for j in range(dc // 32):
                f = code_feature(full, dc // 32, j, G)
                live = col & (f < d)
                head, mp = kvh * group + hh, I // hp
                at = (head * maps + mp) * d + f
                assert (at[live] + 8 <= heads * maps * d).all() and (head[live] < heads).all() and (f[live] + 8 <= d).all()


def check_partial_sums(maps, dc, heads, kv, m, nnz):
    """Pieces and the sums that they leave, inside what the workspace has."""
    w, hp, group = dc * maps, 16 // maps, heads // kv
    passes = -(-group // hp)
    columns = kv * passes
    want = min(nnz, 8192 * 1024) * columns // 768
    piece = (min(max(want, 256), 8192) + 127) // 128 * 128
    if nnz <= piece or m == 0:
        return
    cap = nnz // piece + m
    rng = np.random.default_rng(nnz + m)
    cuts = np.sort(rng.integers(0, nnz + 1, m - 1))
    lengths = np.diff(np.concatenate([[0], cuts, [nnz]]))
    pieces = np.maximum(1, -(-lengths // piece))
    total = int(pieces.sum())
    assert total <= cap
    room = cap * columns * 16 * (w + 4)
    last = (((total - 1) * kv + kv - 1) * passes + passes - 1) * 16 * (w + 4) + 15 * (w + 4) + w + 1
    assert last < room
    first = np.cumsum(pieces) - pieces
    for r in np.unique(np.concatenate([[0, m - 1], rng.integers(0, m, 5)])):
        for u in range(int(pieces[r])):
            lo = u * piece if pieces[r] > 1 else 0
            hi = min(lo + piece, int(lengths[r])) if pieces[r] > 1 else int(lengths[r])
            assert first[r] + u < total and (hi > lo or lengths[r] == 0)
            for wave in range(4):
                # the place of every load of a slot, of tiles ahead too, is kept inside the piece
                at, end = lo + wave * 32, hi
                if at >= end:
                    continue
                for step in range(-(-(end - at) // 128) + 3):
                    e = at + 128 * step + (LANE & 31)
                    e = np.where(e < end, e, end - 1)
                    assert (e >= lo).all() and (e < hi).all()


@pytest.mark.parametrize("refused", [False, True])
def test_records_tiles_and_queries(refused):
    every = sizes(refused)
    assert ((2, 96, 160, 128, False) in every) == refused
    for maps, d, dv, dc, full in every:
        check_record(maps, d, dv, dc, full)
        check_tile(maps, d, dv, dc, full)
        for heads, kv in ((1, 1), (8, 2), (20, 1), (17, 1), (9, 3)):
            check_query(maps, d, dv, dc, full, heads, kv)


@pytest.mark.parametrize("maps,dc", [(1, 32), (1, 256), (2, 32), (2, 128)])
def test_partial_sums_and_slots(maps, dc):
    for heads, kv in ((1, 1), (8, 2), (20, 1), (4, 4)):
        for m in (1, 2, 6, 48):
            for nnz in (1, 255, 257, 464, 1500, 9000, 50000):
                check_partial_sums(maps, dc, heads, kv, m, nnz)


def test_what_can_be_written_and_not_attended():
    """The header's list: with one map d or dv above 128 unless both are 256, with two d above 64 or dv above 128 unless d is 128 and
    dv 256."""
    for maps, d, dv, dc, full in sizes(True):
        assert fa.fusedMM_kv4_record_bytes(maps, d, dv) > 0
        assert (d > 128 or dv > 128) if maps == 1 else (d > 64 or dv > 128)
    for maps, d, dv, dc, full in sizes(False):
        assert (d <= 128 and dv <= 128) or (d, dv) == (256, 256) if maps == 1 else (d <= 64 and dv <= 128) or (d, dv) == (128, 256)
