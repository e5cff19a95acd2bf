"""Windowed attention in 64 bits as whole matrices of torch, for sequences that the row-by-row oracle is too slow for, with two measures of
each output: the sum over the absolute values of its terms ('x_mag', ...) and the root of the sum of their squares ('x_rms', ...), what
independent relative errors of the terms add up to."""
import torch


def sees(Lq, S, window, sinks, causal, n, device):
    """(queries, keys) that see each other in a sequence of n tokens."""
    l, s = torch.arange(Lq, device=device)[:, None], torch.arange(S, device=device)[None, :]
    m = ((l - s).abs() < window) | (s < sinks)
    if causal:
        m &= s <= l
    return m & (l < n) & (s < n)


def buckets_of(Lq, S, first, both, device):
    rel = torch.arange(S, device=device)[None, :] - torch.arange(Lq, device=device)[:, None]
    dist = rel.abs() if both else (-rel).clamp(min=0)
    j = torch.searchsorted(torch.tensor(first, device=device), dist, right=True) - 1
    return j + len(first) * (rel > 0) if both else j


def attention(q, k, v, dx, window, sinks=0, causal=True, table=None, first=None, both=False, lengths=None, without_diagonal=None):
    """float64 Julia arrays q, dx (D, H, L, B), k, v (D, Hkv, S, B), table (H, columns) -> dict of x, dq, dk, dv, dtable and their measures.
    dtable_rms: of weights with independent relative errors that both passes share (each term times the share of its row outside the
    bucket, for the row's gradients sum to zero whatever its weights); dtable_row: of errors that a row's terms share.
    without_diagonal: key - query of pairs that dtable leaves out, for a test of the tests."""
    D, H, Lq, B = q.shape
    Hkv, S, E = k.shape[1], k.shape[2], v.shape[0]
    rep, dev, sc = H // Hkv, q.device, D ** -0.5
    z8 = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)
    out = {"zmax": 0.0, "zrms": 0.0, "pairs": 0, "x": z8(E, H, Lq, B), "dq": z8(D, H, Lq, B), "dk": z8(D, Hkv, S, B), "dv": z8(E, Hkv, S, B)}
    if table is not None:
        out["dtable"] = z8(*table.shape)
        bk = buckets_of(Lq, S, first, both, dev)
        row_of = torch.arange(Lq, device=dev)[:, None].expand(Lq, S)
        cell = (row_of * table.shape[1] + bk).flatten()                              # (row, bucket) of a pair
    for n in ("x", "dq", "dk", "dv") + (("dtable",) if table is not None else ()):
        out[n + "_mag"], out[n + "_rms"] = torch.zeros_like(out[n]), torch.zeros_like(out[n])
    if table is not None:
        out["dtable_row"] = torch.zeros_like(table)
    for b in range(B):
        m = sees(Lq, S, window, sinks, causal, max(S, Lq) if lengths is None else int(lengths[b]), dev)
        any_ = m.any(1, keepdim=True)
        for h in range(H):
            g = h // rep
            qq, kk, vv, gg = q[:, h, :, b].T, k[:, g, :, b].T, v[:, g, :, b].T, dx[:, h, :, b].T
            z, zm = qq @ kk.T * sc, qq.abs() @ kk.abs().T * sc
            if table is not None:
                z, zm = z + table[h][bk], zm + table[h].abs()[bk]
            if bool(m.any()):
                out["zmax"] = max(out["zmax"], float(zm[m].max()))
                out["zrms"] += float((z[m] ** 2).sum())
                out["pairs"] += int(m.sum())
            p = torch.where(any_, torch.softmax(torch.where(m, z, -torch.inf), 1), 0.0).nan_to_num(0.0)
            x = p @ vv
            dp, delta = gg @ vv.T, (gg * x).sum(1, keepdim=True)
            ds = torch.where(m.sum(1, keepdim=True) == 1, 0.0, p * (dp - delta))      # one key alone: exactly nothing
            dm = p * (gg.abs() @ vv.abs().T + (gg.abs() * (p @ vv.abs())).sum(1, keepdim=True))
            put = lambda n, i, val, mag, sq: (out[n][:, i, :, b].add_(val.T), out[n + "_mag"][:, i, :, b].add_(mag.T),
                                              out[n + "_rms"][:, i, :, b].add_(sq.T))
            put("x", h, x, p @ vv.abs(), p ** 2 @ vv ** 2)
            put("dq", h, ds @ kk * sc, dm @ kk.abs() * sc, ds ** 2 @ kk ** 2 * sc ** 2)
            put("dk", g, ds.T @ qq * sc, dm.T @ qq.abs() * sc, (ds ** 2).T @ qq ** 2 * sc ** 2)
            put("dv", g, p.T @ gg, p.T @ gg.abs(), (p ** 2).T @ gg ** 2)
            if table is not None:
                keep = 1.0 if without_diagonal is None else (torch.arange(S, device=dev)[None, :] - torch.arange(Lq, device=dev)[:, None] != without_diagonal)
                out["dtable"][h].index_add_(0, bk.flatten(), (ds * keep).flatten())
                out["dtable_mag"][h].index_add_(0, bk.flatten(), dm.flatten())
                rows = lambda t: z8(Lq * table.shape[1]).index_add_(0, cell, t.flatten()).view(Lq, -1)       # (row, bucket) sums
                share, own = rows(p), rows(ds ** 2)
                out["dtable_rms"][h] += (own * (1 - 2 * share) + share ** 2 * (ds ** 2).sum(1, keepdim=True)
                                         + (p ** 2).sum(1, keepdim=True) * rows(ds) ** 2).clamp(min=0).sum(0)
                out["dtable_row"][h] += (share ** 2 * ((gg * x) ** 2).sum(1, keepdim=True)).sum(0)
    out["zrms"] = (out["zrms"] / max(out["pairs"], 1)) ** 0.5
    for n in list(out):
        if n.endswith("_rms") or n.endswith("_row"):
            out[n] = out[n].sqrt()
    return out
