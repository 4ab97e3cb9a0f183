"""The attention operators over a CSR pattern: what is measured, their plain forms and their exact values.

Five operators of libfusedmm_amd (include/fusedmm_amd.h) are covered:

  train   softmax or differential attention over a sparse pattern, forward and backward (one training pass)
  forward the same, forward alone (prefill, evaluation)
  rows    the serving form: few query rows, each over its own list of cache slots
  rows4   the same over a cache that is held in 4 bits
  cache   writing keys and values into the 4-bit cache and reading them back

A pattern is a CSR matrix: row i attends the columns indx[ptr[i]:ptr[i+1]].  With maps = 2 the weights are the
difference of two softmax maps, softmax(q1 k1') - lambda_h softmax(q2 k2'), which share the values v.

The 4-bit cache holds one record of bytes for each (slot, key/value head): the codes of k (maps * d / 2 bytes), the
codes of v (dv / 2), one 16-bit word for every 32 values of k and then of v, and zeros up to a multiple of 16 bytes.
The word is an fp16 scale s whose low four mantissa bits are replaced by the zero point z; the value of code c is
s * (c - z).  Of eight consecutive codes, code e is nibble (e % 2) * 4 + e // 2 of their 32-bit word.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a few short documents packed into one training sample: launch latency counts
        dict(name="train-packed-small", op="train", type="bf16", maps=2, pattern="docs", m=192, n=192, window=192, first=0, heads=4,
             kv=2, d=32, dv=64),
        # attention over the neighbourhoods of a random graph, 128 features in four heads, single precision
        dict(name="train-graph", op="train", type="f32", maps=1, pattern="graph", m=32768, n=32768, window=16, first=0, heads=4,
             kv=4, d=32, dv=32),
        # a long sequence with a sliding window and a few tokens that everyone sees, differential, shared key heads
        dict(name="train-window-large", op="train", type="bf16", maps=2, pattern="window", m=16384, n=16384, window=256, first=16,
             heads=8, kv=4, d=64, dv=128),
        # a chunk of a prompt behind 500 earlier tokens, head sizes that are no powers of two
        dict(name="forward-odd", op="forward", type="f16", maps=2, pattern="window", m=1000, n=1500, window=300, first=0, heads=6,
             kv=2, d=40, dv=72),
        # prefill with a sliding window of 512, four query heads to a key head
        dict(name="forward-window", op="forward", type="bf16", maps=1, pattern="window", m=8192, n=8192, window=512, first=0,
             heads=8, kv=2, d=128, dv=128),
        # one new token of one sequence: latency
        dict(name="rows-one", op="rows", type="bf16", maps=2, m=1, length=4097, heads=8, kv=4, d=64, dv=128),
        # one new token each for a ragged batch, differential
        dict(name="rows-batch", op="rows", type="bf16", maps=2, m=48, length=16384, heads=16, kv=4, d=64, dv=128),
        # one new token over a short 4-bit cache, every head with keys of its own
        dict(name="rows4-one", op="rows4", type="f16", maps=1, m=1, length=1500, heads=8, kv=8, d=64, dv=64),
        # a ragged serving batch over a 4-bit cache
        dict(name="rows4-batch", op="rows4", type="bf16", maps=1, m=64, length=16384, heads=32, kv=8, d=128, dv=128),
        # two very long sequences over a 4-bit cache: the work of a row has to be split
        dict(name="rows4-long", op="rows4", type="bf16", maps=1, m=2, length=262144, heads=16, kv=2, d=128, dv=128),
        # the keys and values of one decoding step into the cache and back
        dict(name="cache-step", op="cache", type="bf16", maps=1, tokens=8, kv=8, d=128, dv=128),
        # the keys and values of a long prompt into the cache and back
        dict(name="cache-prompt", op="cache", type="bf16", maps=1, tokens=8192, kv=8, d=128, dv=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["train", "forward", "rows", "rows4", "cache"])
    kind = rng.choice(["bf16", "f16"] if op == "rows4" else ["bf16", "f16", "f32"])
    maps = rng.choice([1, 2])
    kv = rng.choice([1, 2, 3, 4])
    heads = kv * rng.choice([1, 2, 3, 4])
    if op in ("rows4", "cache"):
        d, dv = 32 * rng.randint(1, 4 // maps), 32 * rng.randint(1, 4)
    else:
        d = rng.randint(16, 64 if maps == 2 else 128)
        dv = rng.randint(16, maps * d if maps == 2 else 128)
    c = dict(op=op, type=kind, maps=maps, heads=heads, kv=kv, d=d, dv=dv)
    if op == "cache":
        del c["heads"]
        c["tokens"] = _log_int(rng, 1, 6000)
    elif op in ("rows", "rows4"):
        c["m"] = _log_int(rng, 1, 40)
        c["length"] = _log_int(rng, 1, 60000 if c["m"] < 4 else 9000)
    else:
        c["m"] = _log_int(rng, 100, 6000)
        c["n"] = c["m"] + (rng.randint(0, 900) if op == "forward" else 0)
        c["pattern"] = rng.choice(["docs", "graph", "window"])
        c["window"] = _log_int(rng, 3, 24 if c["pattern"] == "graph" else 250)
        c["first"] = rng.choice([0, 5, 16]) if c["pattern"] == "window" else 0
    return c


# ---- patterns (sizes follow from the case alone; graph edges and slots from the seed) ----------------------------------------

def _row_spans(case):
    """(columns of the prefix that everyone sees, first column of the run, length of the run) of every row."""
    m, n = case["m"], case["n"]
    i = np.arange(m, dtype=np.int64)
    if case["pattern"] == "graph":       # a fixed number of neighbours; a node here and there has none
        return np.zeros(m, np.int64), np.zeros(m, np.int64), np.where(i % 97 == 13, 0, case["window"])
    pos = i + (n - m)
    start = np.maximum(0, pos - case["window"] + 1)
    if case["pattern"] == "docs":        # documents of 23, 46, 69, ... tokens, one behind the other
        ends = 23 * np.cumsum(np.arange(1, 2 + int(math.sqrt(2 * n / 23 + 4))))
        first = np.concatenate([[0], ends])[np.searchsorted(ends, pos, side="right")]
        start = np.maximum(start, first)
    return np.minimum(case["first"], start), start, pos - start + 1


def _lengths(case):
    """Cache lengths of a serving batch, from short to the longest; one row of a larger batch is padding."""
    m = case["m"]
    n = 1 + ((case["length"] - 1) * ((np.arange(m) + 1.0) / m) ** 2).astype(np.int64)
    if m > 4:
        n[2] = 0
    return n


def _edges(case):
    if case["op"] in ("rows", "rows4"):
        return int(_lengths(case).sum())
    pre, _, run = _row_spans(case)
    return int((pre + run).sum())


PAGE = 16


def _pool(case):
    """Slots of the cache that a serving batch lives in: pages of 16 slots, a fifth of them not in use."""
    return PAGE * int(-(-_lengths(case) // PAGE).sum() * 5 // 4 + 1)


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _ptr(lengths, dev):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)])).to(dev).to(torch.int32)


def _rows_of(ptr):
    n = ptr.numel() - 1
    return torch.repeat_interleave(torch.arange(n, device=ptr.device), (ptr[1:] - ptr[:-1]).long())


def _pattern(case, gen, dev):
    pre, start, run = _row_spans(case)
    ptr = _ptr(pre + run, dev)
    row = _rows_of(ptr)
    if case["pattern"] == "graph":
        return torch.randint(0, case["n"], (row.numel(),), generator=gen, device=dev, dtype=torch.int32), ptr
    at = torch.arange(row.numel(), device=dev) - ptr.long()[row]
    p, s = torch.from_numpy(pre).to(dev)[row], torch.from_numpy(start).to(dev)[row]
    return torch.where(at < p, at, s + at - p).to(torch.int32), ptr


def _transpose(indx, ptr, n):
    """The same pattern by columns: row ids and pointers."""
    order = torch.sort(indx, stable=True)[1]
    count = torch.bincount(indx, minlength=n)
    tptr = torch.cat([torch.zeros(1, dtype=torch.int64, device=indx.device), count.cumsum(0)]).to(torch.int32)
    return _rows_of(ptr)[order].to(torch.int32), tptr


def _slots(case, gen, dev):
    """Slot lists of a serving batch: pages in any order, the last one of a sequence partly filled."""
    lens = _lengths(case)
    pages = -(-lens // PAGE)
    perm = torch.randperm(_pool(case) // PAGE, generator=gen, device=dev)
    ptr = _ptr(lens, dev)
    row = _rows_of(ptr)
    at = torch.arange(row.numel(), device=dev) - ptr.long()[row]
    base = torch.from_numpy(np.concatenate([[0], np.cumsum(pages)])[:-1]).to(dev)[row]
    return (perm[base + at // PAGE] * PAGE + at % PAGE).to(torch.int32), ptr


def record_bytes(case):
    k, v = case["maps"] * case["d"], case["dv"]
    return -(-(k // 2 + v // 2 + k // 16 + v // 16) // 16) * 16


def _fill_cache(case, n, gen, dev):
    """A cache that is in use: codes of all values, scales as keys and values of unit variance have them."""
    k, v = case["maps"] * case["d"], case["dv"]
    codes, words = (k + v) // 2, (k + v) // 32
    cache = torch.zeros((n, case["kv"], record_bytes(case)), dtype=torch.uint8, device=dev)
    cache[..., :codes] = torch.randint(0, 256, (n, case["kv"], codes), generator=gen, device=dev, dtype=torch.uint8)
    s = torch.rand((n, case["kv"], words), generator=gen, device=dev) * 0.25 + 0.125
    w = s.half().view(torch.int16).int() & 0xFFF0 | torch.randint(5, 11, s.shape, generator=gen, device=dev, dtype=torch.int32)
    cache[..., codes:codes + 2 * words] = w.to(torch.int16).view(torch.uint8).reshape(n, case["kv"], 2 * words)
    return cache


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    t = DTYPES[case["type"]]
    rand = lambda *shape: torch.randn(shape, generator=gen, device=dev).to(t)
    maps, kv, d, dv = case["maps"], case["kv"], case["d"], case["dv"]
    st = dict(case=case)
    if case["op"] == "cache":
        n = 2 * case["tokens"] + 3
        st.update(k=rand(case["tokens"], kv, maps * d), v=rand(case["tokens"], kv, dv), n=n,
                  slots=torch.randperm(n, generator=gen, device=dev)[:case["tokens"]].to(torch.int32),
                  cache=torch.zeros((n, kv, record_bytes(case)), dtype=torch.uint8, device=dev))
        return st
    serving = case["op"] in ("rows", "rows4")
    n = _pool(case) if serving else case["n"]
    indx, ptr = _slots(case, gen, dev) if serving else _pattern(case, gen, dev)
    st.update(n=n, nnz=indx.numel(), indx=indx, ptr=ptr, q=rand(case["m"], case["heads"], maps * d),
              lam=torch.rand(case["heads"], generator=gen, device=dev) * 0.6 + 0.2)
    if case["op"] == "rows4":
        st.update(cache=_fill_cache(case, n, gen, dev))
    else:
        st.update(k=rand(n, kv, maps * d), v=rand(n, kv, dv))
    if case["op"] == "train":
        st.update(do=rand(case["m"], case["heads"], dv))
        st["tindx"], st["tptr"] = _transpose(indx, ptr, n)
    if own:
        _prepare_own(st)
    return st


# ---- the framework's calls ------------------------------------------------------------------------------------------------

def _desc(st):
    import fusedmm_amd as fa
    c = st["case"]
    maps, d, dv, kv = c["maps"], c["d"], c["dv"], c["kv"]
    heads = c.get("heads", kv)
    return fa.AttnDesc(type=fa.TYPES[c["type"]], maps=maps, m=c.get("m", 0), n=st["n"], heads=heads, kv_heads=kv, d=d, dv=dv,
                       scale=1.0 / math.sqrt(d), ldq=heads * maps * d, hdq=maps * d, ldk=kv * maps * d, hdk=maps * d,
                       ldv=kv * dv, hdv=dv, ldo=heads * dv, hdo=dv)


def _prepare_own(st):
    """What a user's program keeps between calls: the plans of a training pattern, and workspace."""
    import fusedmm_amd as fa
    c, desc = st["case"], _desc(st)
    if c["op"] in ("rows", "rows4"):
        size = fa.fusedMM_attn_rows_workspace(desc, st["nnz"])
    else:
        st["plan"] = fa.AttnPlan(c["m"], st["n"], st["nnz"], st["indx"], st["ptr"][:-1], st["ptr"][1:])
        st["plan_t"] = None
        if c["op"] == "train":
            st["plan_t"] = fa.AttnPlan(st["n"], c["m"], st["nnz"], st["tindx"], st["tptr"][:-1], st["tptr"][1:])
        size = fa.fusedMM_attn_workspace(desc, st["plan"], st["plan_t"])
    st["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device=st["q"].device)


def _run_own(st):
    import fusedmm_amd as fa
    c, desc = st["case"], _desc(st)
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "cache":
        k, v, cache = st["k"], st["v"], st["cache"]
        ldc, hdc = cache.stride(0), cache.stride(1)
        rc = fa.fusedMM_kv4_write(desc, c["tokens"], st["slots"], k, v, cache, ldc, hdc, stream=stream)
        assert rc == 0, rc
        k, v = torch.empty_like(k), torch.empty_like(v)
        rc = fa.fusedMM_kv4_read(desc, c["tokens"], st["slots"], cache, ldc, hdc, k, v, stream=stream)
        assert rc == 0, rc
        return {"k": k, "v": v}
    q, work, lam = st["q"], st["work"], st["lam"] if c["maps"] == 2 else None
    o = torch.empty((c["m"], c["heads"], c["dv"]), dtype=q.dtype, device=q.device)
    if c["op"] == "rows":
        rc = fa.fusedMM_attn_rows(desc, st["nnz"], st["indx"], st["ptr"][:-1], st["ptr"][1:], q, st["k"], st["v"], lam, o,
                                  work, work.numel(), stream=stream)
    elif c["op"] == "rows4":
        cache = st["cache"]
        rc = fa.fusedMM_attn_rows_kv4(desc, st["nnz"], st["indx"], st["ptr"][:-1], st["ptr"][1:], q, cache, cache.stride(0),
                                      cache.stride(1), lam, o, work, work.numel(), stream=stream)
    elif c["op"] == "forward":
        rc = fa.fusedMM_attn_forward(desc, st["plan"], q, st["k"], st["v"], lam, o, None, None, work, work.numel(), stream=stream)
    else:
        lse = torch.empty((c["m"], c["heads"], c["maps"]), dtype=torch.float32, device=q.device)
        o2 = torch.empty_like(o) if c["maps"] == 2 else None
        rc = fa.fusedMM_attn_forward(desc, st["plan"], q, st["k"], st["v"], lam, o, o2, lse, work, work.numel(), stream=stream)
        assert rc == 0, rc
        dq, dk, dv = torch.empty_like(q), torch.empty_like(st["k"]), torch.empty_like(st["v"])
        dlam = torch.empty(c["heads"], dtype=torch.float32, device=q.device) if c["maps"] == 2 else None
        rc = fa.fusedMM_attn_backward(desc, st["plan"], st["plan_t"], q, st["k"], st["v"], lam, o, o2, lse, st["do"], dq, dk, dv,
                                      dlam, work, work.numel(), stream=stream)
        assert rc == 0, rc
        return {"o": o, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}
    assert rc == 0, rc
    return {"o": o}


# ---- the plain forms: one tensor element for each edge, head and feature -------------------------------------------------------

def _sum_by(rows, x, n):
    return torch.zeros((n,) + x.shape[1:], dtype=x.dtype, device=x.device).index_add_(0, rows, x)


def _softmax_by_row(s, row, m):
    """Softmax over the edges of each row, for every head and map; a row without edges has none."""
    idx = row.view(-1, 1, 1).expand_as(s)
    top = torch.full((m,) + s.shape[1:], -math.inf, device=s.device).scatter_reduce_(0, idx, s, "amax")
    p = torch.exp(s - top[row])
    return p / _sum_by(row, p, m)[row]


def _maps(x, case):
    return x.float().unflatten(-1, (case["maps"], case["d"]))


def _weights(st, k_edges):
    """Scores of every (edge, head, map) from the gathered keys, and their softmax."""
    c = st["case"]
    row = _rows_of(st["ptr"])
    q = _maps(st["q"], c)
    s = (q[row] * k_edges).sum(-1) * (1.0 / math.sqrt(c["d"]))
    return row, q, _softmax_by_row(s, row, c["m"])


def _sign(st):
    """(heads, maps): what each map's weights count, 1 and -lambda."""
    lam = st["lam"]
    one = torch.ones_like(lam)
    return torch.stack([one, -lam], -1) if st["case"]["maps"] == 2 else one.unsqueeze(-1)


def _by_query_head(x, case):
    return x.repeat_interleave(case["heads"] // case["kv"], dim=1)


def _unpack(codes, words):
    """Values of packed codes (..., w/2 bytes) with their words (..., w/32) in 32 bits."""
    b = codes.to(torch.int32).unflatten(-1, (-1, 4))
    nib = torch.stack([b & 15, b >> 4], -1).flatten(-2)             # the eight nibbles of a 32-bit word, low to high
    c = nib.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-3)     # code e is nibble (e % 2) * 4 + e // 2
    w = words.contiguous().view(torch.int16).int()
    s = (w & 0xFFF0).to(torch.int16).view(torch.float16).float()
    return ((c.unflatten(-1, (-1, 32)) - (w & 15).unsqueeze(-1)).float() * s.unsqueeze(-1)).flatten(-2)


def _read_records(case, rec):
    k, v = case["maps"] * case["d"], case["dv"]
    a, b, c = k // 2, (k + v) // 2, (k + v) // 2 + k // 16
    return _unpack(rec[..., :a], rec[..., b:c]), _unpack(rec[..., a:b], rec[..., c:c + v // 16])


def _quantise(x):
    """(codes, words) of the 4-bit form, groups of 32; in 64 bits, as the borders between codes need."""
    g = x.double().clamp(-32768, 32768).unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    step = (hi - lo) / 15
    grid = torch.exp2(torch.floor(torch.log2(step.clamp(min=2.0 ** -30))) - 6).clamp(min=2.0 ** -20)
    s = torch.ceil(step / grid) * grid                              # seven significant bits, rounded up
    safe = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.round(-lo / safe)
    c = (torch.round(g / safe.unsqueeze(-1)) + z.unsqueeze(-1)).clamp(0, 15)
    word = (s.to(torch.float16).view(torch.int16).int() | z.int()).to(torch.int16)
    e = c.to(torch.int32).flatten(-2).unflatten(-1, (-1, 4, 2)).transpose(-1, -2).flatten(-2).unflatten(-1, (-1, 2))
    return (e[..., 0] | e[..., 1] << 4).to(torch.uint8).flatten(-2), word.view(torch.uint8)


def _run_plain(st):
    c = st["case"]
    t = DTYPES[c["type"]]
    if c["op"] == "cache":
        (kc, kw), (vc, vw) = _quantise(st["k"]), _quantise(st["v"])
        rec = torch.cat([kc, vc, kw, vw], -1)
        st["cache"][st["slots"].long(), :, :rec.shape[-1]] = rec
        k, v = _read_records(c, st["cache"][st["slots"].long()])
        return {"k": k.to(t), "v": v.to(t)}
    col = st["indx"].long()
    if c["op"] == "rows4":
        k, v = _read_records(c, st["cache"][col])
    else:
        k, v = st["k"][col].float(), st["v"][col].float()
    k, v = _by_query_head(_maps(k, c), c), _by_query_head(v, c)
    row, q, p = _weights(st, k)
    sign = _sign(st)
    w = (p * sign).sum(-1, keepdim=True)
    o = _sum_by(row, w * v, c["m"])
    if c["op"] != "train":
        return {"o": o.to(t)}
    do = st["do"].float()[row]
    dp = (do * v).sum(-1, keepdim=True)                             # what the output's gradient gives each edge
    mean = _sum_by(row, p * dp, c["m"])
    ds = p * sign * (dp - mean[row]) * (1.0 / math.sqrt(c["d"]))
    dq = _sum_by(row, ds.unsqueeze(-1) * k, c["m"])
    share = lambda x: x.unflatten(1, (c["kv"], -1)).sum(2)           # the gradients of the heads that share keys
    dk = _sum_by(col, share(ds.unsqueeze(-1) * q[row]), st["n"])
    dv = _sum_by(col, share(w * do), st["n"])
    dlam = -mean[..., 1].sum(0) if c["maps"] == 2 else None
    return {"o": o.to(t), "dq": dq.flatten(-2).to(t), "dk": dk.flatten(-2).to(t), "dv": dv.to(t), "dlam": dlam}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    maps, kv, d, dv = case["maps"], case["kv"], case["d"], case["dv"]
    if case["op"] == "cache":
        rows = case["tokens"] * kv
        packed = (maps * d + dv) * 9 / 16
        return {"bytes": rows * (2 * (maps * d + dv) * size + 2 * packed) + 8 * case["tokens"], "flops": rows * (maps * d + dv) * 6}
    nnz, m, heads = _edges(case), case["m"], case["heads"]
    forward = 2 * nnz * heads * (maps * d + dv)
    pattern = 4 * nnz + 4 * (m + 1)
    if case["op"] == "rows4":
        return {"bytes": nnz * kv * (maps * d + dv) * 9 / 16 + m * heads * (maps * d + dv) * size + pattern, "flops": forward}
    if case["op"] == "rows":
        return {"bytes": nnz * kv * (maps * d + dv) * size + m * heads * (maps * d + dv) * size + pattern, "flops": forward}
    side_q, side_k = m * heads * (maps * d + dv) * size, case["n"] * kv * (maps * d + dv) * size
    if case["op"] == "forward":
        return {"bytes": side_q + side_k + pattern, "flops": forward}
    # training: q, k, v, the output's gradient and the pattern come in; the output and three gradients go out
    return {"bytes": 2 * side_q + 2 * side_k + pattern + 4 * nnz, "flops": 3 * forward}


# ---- exact values: dense matrices in 64 bits, a stretch of rows at a time ---------------------------------------------------------

def _exact_values(case, rec):
    """(k, v) of cache records in 64 bits, code by code."""
    k, v = case["maps"] * case["d"], case["dv"]
    n_codes = (k + v) // 2
    words = rec[..., n_codes:n_codes + (k + v) // 16].long()
    words = words[..., 0::2] + 256 * words[..., 1::2]
    out = torch.empty(rec.shape[:-1] + (k + v,), dtype=torch.float64, device=rec.device)
    for e in range(8):
        nibble = (e % 2) * 4 + e // 2
        code = (rec[..., nibble // 2:n_codes:4].long() >> (4 * (nibble % 2))) & 15
        w = words.repeat_interleave(4, dim=-1)
        exponent, fraction = (w >> 10) & 31, (w >> 4) & 63
        scale = torch.where(exponent > 0, (64 + fraction).double() * torch.exp2((exponent - 15 - 6).double()),
                            fraction.double() * 2.0 ** -20)
        out[..., e::8] = scale * (code - (w & 15)).double()
    return out[..., :k], out[..., k:]


def _exact_cache(case, x):
    """What 4 bits keep of x: seven-bit scales found by search, codes as the nearest level."""
    g = x.double().unflatten(-1, (-1, 32)).clamp(-2.0 ** 15, 2.0 ** 15)
    lo, hi = torch.clamp(g.min(-1).values, max=0.0), torch.clamp(g.max(-1).values, min=0.0)
    s = torch.full_like(lo, math.inf)
    for e in range(-20, 14):
        unit = 2.0 ** max(e - 6, -20)
        top = 128 * unit
        m = torch.ceil((hi - lo) / (15 * unit))
        ok = (m * unit <= top) & torch.isinf(s)
        s = torch.where(ok, m * unit, s)
    live = s > 0
    one = torch.where(live, s, torch.ones_like(s))
    z = torch.round(-lo / one)
    level = torch.clamp(torch.round(g / one.unsqueeze(-1)), min=-z.unsqueeze(-1), max=(15 - z).unsqueeze(-1))
    return (level * s.unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "cache":
        return {"k": _exact_cache(case, st["k"]), "v": _exact_cache(case, st["v"])}
    maps, d, dv, heads, m, n = case["maps"], case["d"], case["dv"], case["heads"], case["m"], st["n"]
    group = heads // case["kv"]
    serving = case["op"] in ("rows", "rows4")
    ptr = st["ptr"].tolist()
    if case["op"] == "rows4":
        k_all, v_all = _exact_values(case, st["cache"])
    else:
        k_all, v_all = st["k"].double(), st["v"].double()
    q_all = st["q"].double()
    dev = q_all.device
    o = torch.zeros((m, heads, dv), dtype=torch.float64, device=dev)
    train = case["op"] == "train"
    if train:
        do = st["do"].double()
        dq, dk, dvv = torch.zeros_like(q_all), torch.zeros_like(k_all), torch.zeros_like(v_all)
        dlam = torch.zeros(heads, dtype=torch.float64, device=dev)
    stretch = 1 if serving else max(1, min(m, (1 << 27) // n))
    for r0 in range(0, m, stretch):
        r1 = min(m, r0 + stretch)
        a, b = ptr[r0], ptr[r1]
        if a == b:
            continue
        cols = st["indx"][a:b].long()
        if serving:
            count = None                                            # one row, its slots are distinct
        else:
            c0, c1 = int(cols.min()), int(cols.max()) + 1           # how often each row names each column
            span = torch.tensor(ptr[r0:r1 + 1], device=dev)
            rr = torch.repeat_interleave(torch.arange(r1 - r0, device=dev), span[1:] - span[:-1])
            count = torch.zeros((r1 - r0, c1 - c0), dtype=torch.float64, device=dev)
            count.index_put_((rr, cols - c0), torch.ones(b - a, dtype=torch.float64, device=dev), accumulate=True)
            cols = slice(c0, c1)
        for h in range(heads):
            kh, vh = k_all[cols, h // group], v_all[cols, h // group]
            total, parts = 0, []
            for w in range(maps):
                sign = 1.0 if w == 0 else -st["lam"][h].double()
                s = q_all[r0:r1, h, w * d:w * d + d] @ kh[:, w * d:w * d + d].T / math.sqrt(d)
                if count is not None:
                    s = s.masked_fill(count == 0, -math.inf)
                s = s - s.amax(-1, keepdim=True).clamp(min=-1e300)
                p = torch.exp(s) if count is None else torch.exp(s) * count
                p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
                total = total + sign * p
                parts.append((sign, p))
            o[r0:r1, h] = total @ vh
            if train:
                g = do[r0:r1, h]
                dvv[cols, h // group] += total.T @ g
                dp = g @ vh.T
                for w, (sign, p) in enumerate(parts):
                    mean = (p * dp).sum(-1, keepdim=True)
                    ds = sign * p * (dp - mean) / math.sqrt(d)
                    dq[r0:r1, h, w * d:w * d + d] = ds @ kh[:, w * d:w * d + d]
                    dk[cols, h // group, w * d:w * d + d] += ds.T @ q_all[r0:r1, h, w * d:w * d + d]
                    if w == 1:
                        dlam[h] -= mean.sum()
    if train:
        return {"o": o, "dq": dq, "dk": dk, "dv": dvv, "dlam": dlam if maps == 2 else None}
    return {"o": o}
