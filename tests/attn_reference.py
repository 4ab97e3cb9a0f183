"""Attention over a CSR pattern in 64 bits, dense, with bounds on what an evaluation in the operators' types may be off by;
and the 4-bit cache format, code by code."""
import numpy as np

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}     # half a step of each type, relative
# fp16: half its smallest step.  The others have fp32's range: the hardware's exponential flushes weights below 2^-126 to
# zero, and a weight meets factors (score gradients, features) whose product stays below 2^10 in these tests.
TINY = {"f32": 2.0 ** -116, "f16": 2.0 ** -25, "bf16": 2.0 ** -116}
E32 = 2.0 ** -24


def counts(m, n, indx, pb, pe):
    """How often each row names each column; ids outside [0, n) are masked places."""
    c = np.zeros((m, n))
    for i in range(m):
        cols = indx[pb[i]:pe[i]]
        cols = cols[(cols >= 0) & (cols < n)]
        np.add.at(c[i], cols, 1.0)
    return c


def attention(count, q, k, v, lam, scale, kind, do=None, weight_type=None, bounds=True):
    """q (m, heads, maps, d), k (n, kv, maps, d), v (n, kv, dv), lam (heads,) or None; float64 copies of the operands.
    Returns dict of exact values and, under "tol", element-wise bounds of the error.

    The bounds count: products accumulated in fp32 (each of the n terms of a sum off by 2^-24 of its size per addition),
    the exponential and the fp32 row statistics (2^-20 relative covers a 1-ulp exponential, the scaling by log2 e and the
    sum), one rounding of the weights and of the scores' gradients to the tensors' type, and one of each output."""
    m, heads, maps, d = q.shape
    n, kv, dv = v.shape
    group = heads // kv
    u, uw, tiny = U[kind], U[weight_type or kind], TINY[weight_type or kind]
    if (weight_type or kind) == "f32":
        uw = 0.0
    named = count > 0
    any_row = named.any(1)
    out = dict(o=np.zeros((m, heads, dv)), o2=np.zeros((m, heads, dv)), lse=np.full((m, heads, maps), -np.inf))
    tol = dict(o=np.zeros((m, heads, dv)), o2=np.zeros((m, heads, dv)), lse=np.zeros((m, heads, maps)))
    if do is not None:
        out.update(dq=np.zeros_like(q), dk=np.zeros_like(k), dv=np.zeros_like(v), dlam=np.zeros(heads))
        tol.update(dq=np.zeros_like(q), dk=np.zeros_like(k), dv=np.zeros_like(v), dlam=np.zeros(heads))
    per_row = count.sum(1)[:, None]
    for h in range(heads):
        g = h // group
        probs, eps, o_maps, o_tols = [], [], [], []
        for p in range(maps):
            s = scale * (q[:, h, p] @ k[:, g, p].T)
            ds = abs(scale) * (np.abs(q[:, h, p]) @ np.abs(k[:, g, p]).T) * (d + 8) * E32   # fp32 accumulation of the scores
            top = np.where(named, s, -np.inf).max(1, initial=-np.inf)
            base = np.where(np.isfinite(top), top, 0.0)[:, None]
            e = np.where(named, count * np.exp(np.where(named, s - base, 0.0)), 0.0)
            tot = e.sum(1, keepdims=True)
            P = e / np.where(tot > 0, tot, 1.0)
            ds_row = np.where(named, ds + np.abs(s) * 4 * E32, 0.0).max(1, initial=0.0)[:, None]
            ep = 2 * ds_row + 2.0 ** -20 + per_row * E32            # relative error of a weight before it is rounded
            out["lse"][:, h, p] = np.where(any_row, base[:, 0] + np.log(np.where(tot[:, 0] > 0, tot[:, 0], 1.0)), -np.inf)
            tol["lse"][:, h, p] = ds_row[:, 0] + 2.0 ** -20 + np.where(any_row, np.abs(np.where(any_row, out["lse"][:, h, p], 0)) * 4 * E32, 0)
            o = P @ v[:, g]
            spread = P @ np.abs(v[:, g])
            # the weights enter the product unnormalised, at most 1, divided by a sum of at least 1/2 afterwards
            low = 2 * tiny * ((count > 0) @ np.abs(v[:, g]))
            o_maps.append(o)
            o_tols.append(spread * (ep + uw) + low)
            probs.append(P)
            eps.append(ep)
        sign = [1.0, -lam[h]] if maps == 2 else [1.0]
        o = sum(w * x for w, x in zip(sign, o_maps))
        out["o"][:, h] = o
        t = sum(abs(w) * x for w, x in zip(sign, o_tols)) + 4 * E32 * sum(np.abs(w * x) for w, x in zip(sign, o_maps))
        tol["o"][:, h] = t + u * (np.abs(o) + t) + TINY[kind]
        if maps == 2:
            out["o2"][:, h] = o_maps[1]
            tol["o2"][:, h] = o_tols[1] + u * (np.abs(o_maps[1]) + o_tols[1]) + TINY[kind]
        if do is None:
            continue
        G, aG = do[:, h], np.abs(do[:, h])
        dP = G @ v[:, g].T
        dP_err = (aG @ np.abs(v[:, g]).T) * (dv + 8) * E32
        W = sum(w * P for w, P in zip(sign, probs))
        W_err = sum(abs(w) * P * ep for w, P, ep in zip(sign, probs, eps)) + 4 * E32 * sum(abs(w) * P for w, P in zip(sign, probs))
        out["dv"][:, g] += W.T @ G
        # rounded weights; in fp16 they are multiplied by 2^10 first
        tol["dv"][:, g] += (W_err * (1 + uw) + np.abs(W) * (uw + m * E32)).T @ aG + tiny / 1024 * (named.T.astype(float) @ aG)
        for p in range(maps):
            P, w = probs[p], sign[p]
            delta = (P * dP).sum(1, keepdims=True)
            # delta comes from the rounded outputs: <do, o> (+ lambda <do, o2>)
            if maps == 1 or p == 0:
                derr = (aG * tol["o"][:, h]).sum(1, keepdims=True) + (aG * np.abs(out["o"][:, h])).sum(1, keepdims=True) * (dv + 8) * E32
                if maps == 2:
                    derr = derr + abs(lam[h]) * ((aG * tol["o2"][:, h]).sum(1, keepdims=True) + (aG * np.abs(out["o2"][:, h])).sum(1, keepdims=True) * (dv + 8) * E32)
            else:
                derr = (aG * tol["o2"][:, h]).sum(1, keepdims=True) + (aG * np.abs(out["o2"][:, h])).sum(1, keepdims=True) * (dv + 8) * E32
            dS = w * P * (dP - delta)
            dS_err = abs(w) * P * (derr + dP_err) + np.abs(dS) * (eps[p] + uw + 8 * E32) + tiny * count
            out["dq"][:, h, p] = scale * dS @ k[:, g, p]
            tol["dq"][:, h, p] = abs(scale) * ((dS_err + np.abs(dS) * n * E32) @ np.abs(k[:, g, p]))
            out["dk"][:, g, p] += scale * dS.T @ q[:, h, p]
            tol["dk"][:, g, p] += abs(scale) * ((dS_err + np.abs(dS) * m * group * E32).T @ np.abs(q[:, h, p]))
            if p == 1:
                out["dlam"][h] = -delta.sum()
                tol["dlam"][h] = (P * (np.abs(dP) * (eps[p] + (n + 8) * E32) + dP_err)).sum() + abs(delta.sum()) * 2 * E32
    if do is not None:
        for x in ("dq", "dk", "dv"):
            tol[x] = tol[x] + u * (np.abs(out[x]) + tol[x]) + TINY[kind]
    out["tol"] = tol
    return out


# ---- the 4-bit cache -------------------------------------------------------------------------------------------------------

def quantise_group(x):
    """(scale, zero point, codes) of 32 values."""
    x = np.clip(np.asarray(x, np.float64), -32768, 32768)
    if np.isnan(x).any():
        return np.nan, 0, np.zeros(32, np.int64)
    lo, hi = min(0.0, x.min()), max(0.0, x.max())
    step = (hi - lo) / 15
    if step == 0:
        return 0.0, 0, np.zeros(32, np.int64)
    unit = max(2.0 ** (np.frexp(step)[1] - 7), 2.0 ** -20)
    s = np.ceil(step / unit) * unit
    z = int(np.rint(-lo / s))
    return s, z, np.clip(np.rint(x / s) + z, 0, 15).astype(np.int64)


def quantise_row(x):
    """(code bytes, words, values) of a row whose width is a multiple of 32."""
    codes, words, values = [], [], []
    for b in range(0, len(x), 32):
        s, z, c = quantise_group(x[b:b + 32])
        w = 0x7E00 if np.isnan(s) else int(np.float16(s).view(np.uint16))
        assert np.isnan(s) or (w & 15 == 0 and float(np.float16(s)) == s)
        words.append(w | z)
        values.append(s * (c - z).astype(np.float64))
        for o in range(0, 32, 8):
            word = 0
            for e in range(8):
                word |= int(c[o + e]) << (4 * ((e % 2) * 4 + e // 2))
            codes.append(word)
    return np.array(codes, "<u4").view(np.uint8), np.array(words, "<u2").view(np.uint8), np.concatenate(values)


def record(k, v):
    """(bytes, values of k, values of v) of one record; k holds all maps."""
    kc, kw, kv = quantise_row(k)
    vc, vw, vv = quantise_row(v)
    b = np.concatenate([kc, vc, kw, vw])
    return np.concatenate([b, np.zeros(-len(b) % 16, np.uint8)]), kv, vv
