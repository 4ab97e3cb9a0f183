"""Attention over a CSR pattern in 64 bits, dense, with the bounds of an evaluation that rounds 16-bit weights twice (a rounded
value and its rounded rest) and takes the row means of the backward pass from fp32 sums.

What the bounds count, for a weight or a score's gradient x of a row or column:
  - ep: the score's fp32 accumulation, the exponential and the fp32 row statistics (2^-20 relative covers a 1-ulp
    exponential, the scaling by log2 e and the sum), and the fp32 additions of the second product, two for every weight
  - u^2 |x|: the rest that a first rounding (u, half a step) leaves is rounded in turn
  - fp16's smallest step: half of it is 2^-25, where the largest weight of the row was 2^7 when the sums' base was set
    (2^-32 of it for each named edge), and the largest gradient of a row or column is at least 2^12 (2^-37 of it)
fp32 operands follow attn_reference, whose bounds for them count nothing that is not rounded."""
import numpy as np

from attn_reference import E32, TINY, U, attention, counts

WEIGHT_LOW = {"f16": 2.0 ** -32, "bf16": 2.0 ** -116}
GRADIENT_LOW = {"f16": 2.0 ** -37, "bf16": 2.0 ** -116}


def tight(c, do=False, k=None, v=None, weight_type=None):
    """The exact values of a Case's operands, and under "tol" the bounds.  weight_type: the type of the second product's
    operands where it is not the tensors' own (rows over a 4-bit cache)."""
    q = c.q.numpy().reshape(c.m, c.heads, c.maps, c.d)
    k = (c.k.numpy() if k is None else k).reshape(c.n, c.kv, c.maps, c.d)
    v = c.v.numpy() if v is None else v
    lam = c.lam.double().cpu().numpy() if c.maps == 2 else None
    count = counts(c.m, c.n, c.indx, c.pb, c.pe)
    do = c.do.numpy() if do else None
    out = attention(count, q, k, v, lam, c.scale, c.kind, do)
    wt = weight_type or c.kind
    if wt == "f32":
        return out
    m, n, maps, d, dv, group = c.m, c.n, c.maps, c.d, c.dv, c.heads // c.kv
    u, u2, u1, low, glow = U[c.kind], U[wt] ** 2, U[wt], WEIGHT_LOW[wt], GRADIENT_LOW[wt]
    tol = out["tol"]
    for x in tol:
        if x not in ("lse",):
            tol[x] = np.zeros_like(tol[x])
    named = (count > 0).astype(float)
    length = count.sum(1)[:, None]
    uses = (count.sum(0) * group)[:, None]
    for h in range(c.heads):
        g = h // group
        sign = [1.0, -lam[h]] if maps == 2 else [1.0]
        probs, eps, o_tol = [], [], []
        for p in range(maps):
            s = c.scale * (q[:, h, p] @ k[:, g, p].T)
            ds = abs(c.scale) * (np.abs(q[:, h, p]) @ np.abs(k[:, g, p]).T) * (d + 8) * E32 + np.abs(s) * 8 * E32
            ds = np.where(named > 0, ds, 0.0).max(1, initial=0.0)[:, None]
            lse = out["lse"][:, h, p][:, None]
            P = np.where(named > 0, count * np.exp(np.where(named > 0, s, 0.0) - np.where(np.isfinite(lse), lse, 0.0)), 0.0)
            ep = 2 * ds + 2.0 ** -20 + (2 * length + 8) * E32 + np.where(np.isfinite(lse), np.abs(lse), 0.0) * 8 * E32
            probs.append(P)
            eps.append(ep)
            o_tol.append((P @ np.abs(v[:, g])) * (ep + u2) + low * (count @ np.abs(v[:, g])))
        parts = [probs[p] @ v[:, g] for p in range(maps)]
        t = sum(abs(w) * x for w, x in zip(sign, o_tol)) + 8 * E32 * sum(np.abs(w * x) for w, x in zip(sign, parts))
        tol["o"][:, h] = t + u * (np.abs(out["o"][:, h]) + t) + TINY[c.kind]
        if maps == 2:
            tol["o2"][:, h] = o_tol[1] + 8 * E32 * np.abs(parts[1]) + u * (np.abs(parts[1]) + o_tol[1]) + TINY[c.kind]
        if do is None:
            continue
        G, aG = do[:, h], np.abs(do[:, h])
        dP, dP_err = G @ v[:, g].T, (aG @ np.abs(v[:, g]).T) * (dv + 8) * E32
        W = sum(w * P for w, P in zip(sign, probs))
        W_err = sum(abs(w) * P * (ep + 4 * E32) for w, P, ep in zip(sign, probs, eps))
        tol["dv"][:, g] += (W_err + np.abs(W) * u2).T @ aG + (2 * uses * E32) * (np.abs(W).T @ aG) + \
            glow * np.abs(W).max(0, initial=0.0)[:, None] * (named.T @ aG)
        for p in range(maps):
            P, ep, w = probs[p], eps[p], sign[p]
            mean = (P * dP).sum(1, keepdims=True)
            mean_err = (P * np.abs(dP) * ep).sum(1, keepdims=True) + (P * dP_err).sum(1, keepdims=True)
            ot, oo = tol["o2"][:, h] if p else tol["o"][:, h], out["o2"][:, h] if p else out["o"][:, h]
            delta_err = (aG * (ot + np.abs(oo) * (dv + 8) * E32)).sum(1, keepdims=True)
            if maps == 2 and p == 0:
                delta_err += abs(lam[h]) * (aG * (tol["o2"][:, h] + np.abs(out["o2"][:, h]) * (dv + 8) * E32)).sum(1, keepdims=True)
            dS = w * P * (dP - mean)
            err = abs(w) * P * (mean_err + dP_err) + np.abs(dS) * (ep + u2 + 8 * E32)
            # dq: sums of P (dP - delta), and of P times what delta is off by, with weights that are rounded once
            first = err + abs(w) * P * delta_err * (ep + u2 + 8 * E32) + \
                glow * (np.abs(dS) + abs(w) * P * delta_err).max(1, initial=0.0)[:, None] * named
            tol["dq"][:, h, p] = abs(c.scale) * (first @ np.abs(k[:, g, p]) + (2 * length * E32) * (np.abs(dS) @ np.abs(k[:, g, p])) +
                                                 abs(w) * delta_err * (u1 + ep) * (P @ np.abs(k[:, g, p])))
            tol["dk"][:, g, p] += abs(c.scale) * ((err + glow * np.abs(dS).max(0, initial=0.0)[None, :] * named).T @ np.abs(q[:, h, p]) +
                                                  (2 * uses * E32) * (np.abs(dS).T @ np.abs(q[:, h, p])))
            if p == 1:
                tol["dlam"][h] = mean_err.sum() + 2 * np.abs(mean).sum() * 16 * E32
    if do is not None:
        for x in ("dq", "dk", "dv"):
            tol[x] = tol[x] + u * (np.abs(out[x]) + tol[x]) + TINY[c.kind]
    return out
