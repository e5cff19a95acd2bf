"""Windowed attention, its ring cache and the relative position bias in 64 bits, row by row from their definitions, with the
magnitudes (the same sums over absolute values) that rounding errors are measured against."""
import numpy as np


def sees(l, s, window, sinks, causal):
    return (abs(l - s) < window or s < sinks) and (not causal or s <= l)


def bucket(rel, first, bidirectional):
    dist = abs(rel) if bidirectional else max(-rel, 0)
    j = max(i for i, f in enumerate(first) if f <= dist)
    return j + (len(first) if bidirectional and rel > 0 else 0)


def attention(q, k, v, window, sinks=0, causal=True, scale=None, table=None, first=None, bidirectional=False, lengths=None, dx=None):
    """q (D, H, L, B), k (D, Hkv, S, B), v (E, Hkv, S, B) -> dict of x, dq, dk, dv, dtable and their magnitudes ('x_mag', ...)."""
    D, H, L, B = q.shape
    Hkv, S, E = k.shape[1], k.shape[2], v.shape[0]
    sc = 1.0 / (scale if scale is not None else np.sqrt(D))
    rep = H // Hkv
    out = {"x": np.zeros((E, H, L, B)), "zmax": 0.0}
    if dx is not None:
        out.update(dq=np.zeros(q.shape), dk=np.zeros(k.shape), dv=np.zeros(v.shape))
        if table is not None:
            out["dtable"] = np.zeros(table.shape)
    for n in [n for n in out if n in ("x", "dq", "dk", "dv", "dtable")]:
        out[n + "_mag"] = np.zeros(out[n].shape)
    with np.errstate(all="ignore"):
        for b in range(B):
            n = max(S, L) if lengths is None else max(0, int(lengths[b]))
            for l in range(min(L, n)):
                at = np.array([s for s in range(min(S, n)) if sees(l, s, window, sinks, causal)], dtype=int)
                if at.size == 0:
                    continue
                bk = np.array([bucket(s - l, first, bidirectional) for s in at]) if table is not None else None
                for h in range(H):
                    kk, vv, qq = k[:, h // rep, at, b], v[:, h // rep, at, b], q[:, h, l, b]
                    z = (qq @ kk) * sc
                    zm = np.abs(qq) @ np.abs(kk) * abs(sc)
                    if table is not None:
                        z, zm = z + table[h, bk], zm + np.abs(table[h, bk])
                    out["zmax"] = max(out["zmax"], float(zm[np.isfinite(zm)].max(initial=0.0)))
                    m = z.max()
                    e = np.exp(z - m)
                    p = e / e.sum()
                    out["x"][:, h, l, b], out["x_mag"][:, h, l, b] = vv @ p, np.abs(vv) @ p
                    if dx is None:
                        continue
                    g = dx[:, h, l, b]
                    dp, delta = g @ vv, g @ (vv @ p)
                    ds = p * (dp - delta)
                    dsm = p * (np.abs(g) @ np.abs(vv) + np.abs(g) @ (np.abs(vv) @ p))
                    out["dq"][:, h, l, b], out["dq_mag"][:, h, l, b] = kk @ ds * sc, np.abs(kk) @ dsm * abs(sc)
                    out["dk"][:, h // rep, at, b] += np.outer(qq, ds) * sc
                    out["dk_mag"][:, h // rep, at, b] += np.outer(np.abs(qq), dsm) * abs(sc)
                    out["dv"][:, h // rep, at, b] += np.outer(g, p)
                    out["dv_mag"][:, h // rep, at, b] += np.outer(np.abs(g), p)
                    if table is not None:
                        np.add.at(out["dtable"][h], bk, ds)
                        np.add.at(out["dtable_mag"][h], bk, dsm)
    return out


def slot(p, sinks, capacity):
    return p if p < sinks else sinks + (p - sinks) % (capacity - sinks)


def relative_bias(table, first, bidirectional, S, L, offset=0):
    bias = np.zeros((S, L, table.shape[0], 1))
    for s in range(S):
        for l in range(L):
            bias[s, l, :, 0] = table[:, bucket(s - l - offset, first, bidirectional)]
    return bias


def relative_bias_grad(delta, heads, columns, first, bidirectional, offset=0):
    """(dtable, magnitudes)"""
    g, mag = np.zeros((heads, columns)), np.zeros((heads, columns))
    S, L = delta.shape[:2]
    d = delta.reshape(S, L, heads, -1)
    for s in range(S):
        for l in range(L):
            j = bucket(s - l - offset, first, bidirectional)
            g[:, j] += d[s, l].sum(-1)
            mag[:, j] += np.abs(d[s, l]).sum(-1)
    return g, mag
