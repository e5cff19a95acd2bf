"""Windowed attention, its ring cache and the relative position bias: the work whose time counts.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare(case, seed)` makes what a program holds
before the call, `run(state)` is one pass (the plain form in 32 bits, or with `own = True` the public operators of luxlib_b200),
`work(case)` counts the bytes and operations that no implementation can do without, `exact(case, seed)` is what `run` returns in
64-bit arithmetic.

Four kinds of work:
  train    windowed attention (sliding window, a few first tokens that stay visible), forward + pullback
  prefill  windowed attention over a prompt, then the cache takes the keys and values that later tokens can see
  step     one new token per sequence: the cache takes its key and value, the token attends to what its window holds
  bias     a learned relative position bias by buckets, forward + pullback

Arrays are Julia arrays (first index contiguous): q (D, H, L, B), k and v (D, Hkv, L, B), the bucket table (H, buckets).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _lib():
    path = os.path.join(os.getcwd(), "lux.jl_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import luxlib_b200
    return luxlib_b200


def listed():
    return [
        # a training step of a long-context decoder layer: grouped heads, a window of 1024, four sinks, learned bias
        {"name": "train_long_bf16", "kind": "train", "dtype": "bf16", "D": 128, "H": 32, "Hkv": 8, "L": 8192, "B": 1, "window": 1024,
         "sinks": 4, "causal": True, "buckets": 32, "max_distance": 128, "ragged": False},
        # the usual heads of 64 features without sinks or bias
        {"name": "train_bf16", "kind": "train", "dtype": "bf16", "D": 64, "H": 16, "Hkv": 16, "L": 4096, "B": 2, "window": 512,
         "sinks": 0, "causal": True, "buckets": 0, "max_distance": 0, "ragged": False},
        # Lux's default element type
        {"name": "train_f32", "kind": "train", "dtype": "f32", "D": 64, "H": 8, "Hkv": 8, "L": 1024, "B": 4, "window": 256,
         "sinks": 4, "causal": True, "buckets": 32, "max_distance": 128, "ragged": False},
        # an encoder over 197 tokens that looks both ways, the class token visible to all, a padded batch
        {"name": "train_encoder_ragged_bf16", "kind": "train", "dtype": "bf16", "D": 64, "H": 12, "Hkv": 12, "L": 197, "B": 16,
         "window": 64, "sinks": 1, "causal": False, "buckets": 32, "max_distance": 128, "ragged": True},
        # a long prompt ahead of serving (the largest)
        {"name": "prefill_long_bf16", "kind": "prefill", "dtype": "bf16", "D": 128, "H": 32, "Hkv": 8, "L": 16384, "B": 1, "window": 4096,
         "sinks": 4, "causal": True, "buckets": 0, "max_distance": 0, "ragged": False, "capacity": 4100},
        # a short prompt, sizes that are no multiple of anything: latency
        {"name": "prefill_short_f32", "kind": "prefill", "dtype": "f32", "D": 80, "H": 8, "Hkv": 2, "L": 77, "B": 1, "window": 32,
         "sinks": 4, "causal": True, "buckets": 32, "max_distance": 128, "ragged": False, "capacity": 50},
        # one user's next token: latency
        {"name": "step_one_bf16", "kind": "step", "dtype": "bf16", "D": 128, "H": 32, "Hkv": 8, "B": 1, "window": 1024, "sinks": 4,
         "buckets": 0, "max_distance": 0, "capacity": 1028, "len_lo": 5000, "len_hi": 5000},
        # the next tokens of a full serving batch, caches of many ages
        {"name": "step_batch_bf16", "kind": "step", "dtype": "bf16", "D": 128, "H": 32, "Hkv": 8, "B": 32, "window": 4096, "sinks": 4,
         "buckets": 0, "max_distance": 0, "capacity": 4100, "len_lo": 1000, "len_hi": 9000},
        # a few sequences with a learned bias in Float32, odd window
        {"name": "step_bias_f32", "kind": "step", "dtype": "f32", "D": 64, "H": 12, "Hkv": 12, "B": 5, "window": 500, "sinks": 1,
         "buckets": 32, "max_distance": 128, "capacity": 777, "len_lo": 0, "len_hi": 2000},
        # the bias of an encoder's attention over 1024 tokens and its gradient from a batch of cotangents
        {"name": "bias_bf16", "kind": "bias", "dtype": "bf16", "H": 16, "S": 1024, "L": 1024, "B": 4, "buckets": 32, "max_distance": 128,
         "bidirectional": True},
        # 197 tokens: rows that are no multiple of a vector
        {"name": "bias_ragged_f32", "kind": "bias", "dtype": "f32", "H": 12, "S": 197, "L": 197, "B": 1, "buckets": 32, "max_distance": 128,
         "bidirectional": True},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """As `_log`; half of the draws are rounded to a multiple of 8."""
    v = _log(rng, lo, hi)
    return max(lo, v // 8 * 8) if rng.random() < 0.5 and v >= 16 else v


def _draw_buckets(rng):
    n = rng.choice([8, 16, 32, 32, 64])
    return {"buckets": n, "max_distance": _size(rng, n + 1, 1024)}


def draw(rng):
    kind = rng.choice(["train", "train", "prefill", "step", "step", "bias"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "bias":
        b = _draw_buckets(rng)
        H, S, L = rng.choice([1, 4, 8, 12, 16, 32]), _size(rng, 1, 2048), _size(rng, 1, 2048)
        most = int((1 << 27) / (H * S * L))
        return dict(b, kind=kind, dtype=dtype, H=H, S=S, L=L, B=max(1, min(_log(rng, 1, 16), most)), bidirectional=rng.random() < 0.5)
    hkv, rep = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 4, 8])
    c = {"kind": kind, "dtype": dtype, "D": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), "H": hkv * rep, "Hkv": hkv,
         "sinks": rng.choice([0, 0, 1, 4, rng.randint(1, 64)])}
    c.update(_draw_buckets(rng) if rng.random() < 0.5 else {"buckets": 0, "max_distance": 0})
    if kind == "step":
        c["window"] = _size(rng, 1, 8192)
        c["capacity"] = c["window"] + c["sinks"] + rng.choice([0, 0, rng.randint(1, 200)])
        most = int((1 << 30) / (4 * c["D"] * hkv * c["capacity"]))
        c["B"] = max(1, min(_log(rng, 1, 64), most))
        c["len_lo"] = rng.randint(0, c["capacity"])
        c["len_hi"] = rng.randint(c["len_lo"], 3 * c["capacity"])
        return c
    c["L"] = _size(rng, 1, 8192)
    c["window"] = _size(rng, 1, 4096)
    c["causal"] = kind == "prefill" or rng.random() < 0.7
    pairs = c["H"] * c["L"] * min(c["window"] * (1 if c["causal"] else 2) + c["sinks"], c["L"])
    most = int((3e11 if dtype == "bf16" else 3e10) / (14.0 * c["D"] * pairs))
    c["B"] = max(1, min(_log(rng, 1, 16), most))
    while c["L"] > 16 and 14.0 * c["D"] * c["H"] * c["L"] * min(c["window"] * (1 if c["causal"] else 2) + c["sinks"], c["L"]) > (3e11 if dtype == "bf16" else 3e10):
        c["L"] //= 2
    c["ragged"] = rng.random() < 0.4
    if kind == "prefill":
        c["capacity"] = c["window"] + c["sinks"] + rng.choice([0, rng.randint(1, 200)])
    return c


# ---------------------------------------------------------------------------------------------
# what the cases' numbers mean
# ---------------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens of each sequence: a step's cache before it, or a padded batch (None: all full)."""
    B = case["B"]
    if case["kind"] == "step":
        return [case["len_lo"] + (case["len_hi"] - case["len_lo"]) * b // max(B - 1, 1) for b in range(B)]
    return [case["L"] - case["L"] * b // B for b in range(B)] if case["ragged"] else None


def _slot(p, sinks, capacity):
    return p if p < sinks else sinks + (p - sinks) % (capacity - sinks)


def _visible_pairs(L, window, sinks, causal):
    """Pairs (query, key) of a sequence of L tokens that see each other."""
    n = 0
    for l in range(L):
        lo, hi = max(0, l - window + 1), (l + 1 if causal else min(L, l + window))
        n += hi - lo + min(sinks, lo)
        if not causal and sinks > hi:
            n += min(sinks, L) - hi if L > hi else 0
    return n


# ---------------------------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        t = (torch.randn(*reversed(shape), device="cuda", generator=g) * std).to(dt)
        return t.permute(*reversed(range(t.dim()))) if t.dim() > 1 else t

    st = {"case": case}
    H, B = case["H"], case["B"]
    if case["buckets"]:
        st["table"] = normal(H, case["buckets"], std=0.5)
    if case["kind"] == "bias":
        st["delta"] = normal(case["S"], case["L"], H, B)
        if own:
            st["plan"] = _lib().RelativeBuckets.make(case["buckets"], case["max_distance"], case["bidirectional"])
        return st
    D, Hkv = case["D"], case["Hkv"]
    if case["buckets"] and own:
        st["plan"] = _lib().RelativeBuckets.make(case["buckets"], case["max_distance"], _both_ways(case))
    lens = _lengths(case)
    st["lengths"] = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["kind"] == "step":
        C = case["capacity"]
        st["q"], st["k"], st["v"] = normal(D, H, B), normal(D, Hkv, B), normal(D, Hkv, B)
        st["kcache"], st["vcache"] = normal(D, Hkv, C, B), normal(D, Hkv, C, B)
        return st
    L = case["L"]
    st["q"], st["k"], st["v"] = normal(D, H, L, B), normal(D, Hkv, L, B), normal(D, Hkv, L, B)
    if case["kind"] == "train":
        st["delta"] = normal(D, H, L, B)
    else:
        C = case["capacity"]
        st["kcache"], st["vcache"] = normal(D, Hkv, C, B), normal(D, Hkv, C, B)
    return st


def _both_ways(case):
    return not case.get("causal", True)


# ---------------------------------------------------------------------------------------------
# run: the framework's operators
# ---------------------------------------------------------------------------------------------
def _run_own(st):
    L, case = _lib(), st["case"]
    table, plan = st.get("table"), st.get("plan")
    if case["kind"] == "bias":
        bias, pullback = L.rrule_relative_position_bias(table, plan, case["S"], case["L"])
        return bias, pullback(st["delta"])
    if case["kind"] == "step":
        x = L.windowed_attention_step(st["q"], st["k"], st["v"], st["kcache"], st["vcache"], st["lengths"], window=case["window"],
                                      sinks=case["sinks"], table=table, buckets=plan)
        return x, st["kcache"], st["vcache"]
    kw = dict(window=case["window"], sinks=case["sinks"], is_causal=case["causal"], table=table, buckets=plan, lengths=st["lengths"])
    if case["kind"] == "prefill":
        x = L.windowed_attention(st["q"], st["k"], st["v"], **kw)
        L.windowed_cache_fill(st["kcache"], st["vcache"], st["k"], st["v"], st["lengths"], sinks=case["sinks"])
        return x, st["kcache"], st["vcache"]
    x, pullback = L.rrule_windowed_attention(st["q"], st["k"], st["v"], **kw)
    dq, dk, dv, dtable = pullback(st["delta"])
    return (x, dq, dk, dv) + ((dtable,) if dtable is not None else ())


# ---------------------------------------------------------------------------------------------
# run: the plain form
# ---------------------------------------------------------------------------------------------
def _bucket_starts(n, max_distance):
    """The smallest distance of each of n buckets: one distance each up to n/2, then logarithmic up to max_distance. Whole
    numbers: bucket n/2 + j starts at the smallest d with (d / e)^(n-e) >= (max_distance / e)^j, e = n/2."""
    e = n // 2
    starts = list(range(e))
    d = e
    for j in range(n - e):
        while d ** (n - e) * e ** j < max_distance ** j * e ** (n - e):
            d += 1
        starts.append(d)
    return starts


def _bucket_of(rel, n, max_distance, both_ways):
    """Buckets of an integer tensor of relative positions (key - query)."""
    per_side = n // 2 if both_ways else n
    starts = torch.tensor(_bucket_starts(per_side, max_distance), device=rel.device)
    dist = rel.abs() if both_ways else (-rel).clamp(min=0)
    b = torch.searchsorted(starts, dist, right=True) - 1
    return b + per_side * (rel > 0) if both_ways else b


def _rows(t):
    """(feature, head, token, batch) Julia array -> float32 (batch, head, token, feature)."""
    return t.permute(3, 1, 2, 0).float()


def _julia(t, dt):
    return t.to(dt).permute(3, 1, 2, 0)


def _plain_attention(st, train):
    """Block by block of queries, the keys of a block's band and the sinks before it."""
    case = st["case"]
    q, k, v = _rows(st["q"]), _rows(st["k"]), _rows(st["v"])
    B, H, L, D = q.shape
    Hkv = k.shape[1]
    rep, dev = H // Hkv, q.device
    W, sinks, causal = case["window"], case["sinks"], case["causal"]
    scale = 1.0 / math.sqrt(D)
    lens = st["lengths"].long() if st["lengths"] is not None else None
    table = st["table"].float() if "table" in st else None
    x = torch.zeros_like(q)
    if train:
        g = _rows(st["delta"])
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dtable = torch.zeros_like(table) if table is not None else None
    step = 1024
    for l0 in range(0, L, step):
        l1 = min(L, l0 + step)
        lo = max(0, l0 - W + 1)
        hi = l1 if causal else max(min(L, l1 + W - 1), min(sinks, L))
        s_pos = torch.cat([torch.arange(0, min(sinks, lo), device=dev), torch.arange(lo, hi, device=dev)])
        l_pos = torch.arange(l0, l1, device=dev)
        rel = s_pos[None, :] - l_pos[:, None]
        seen = (rel.abs() < W) | (s_pos < sinks)[None, :]
        if causal:
            seen &= rel <= 0
        seen = seen[None, None]
        if lens is not None:
            seen = seen & (s_pos[None, :] < lens[:, None])[:, None, None, :] & (l_pos[None, :] < lens[:, None])[:, None, :, None]
        ks, vs = k[:, :, s_pos], v[:, :, s_pos]
        kr, vr = ks.repeat_interleave(rep, 1), vs.repeat_interleave(rep, 1)
        qb = q[:, :, l0:l1]
        z = qb @ kr.transpose(2, 3) * scale
        if table is not None:
            bk = _bucket_of(rel, case["buckets"], case["max_distance"], _both_ways(case))
            z = z + table[:, bk][None]
        z = torch.where(seen, z, -math.inf)
        m = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        x[:, :, l0:l1] = p @ vr
        if train:
            gb = g[:, :, l0:l1]
            dp = gb @ vr.transpose(2, 3)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            if dtable is not None:
                dtable.index_add_(1, bk.flatten(), ds.sum(0).flatten(1))
            dq[:, :, l0:l1] = ds @ kr * scale
            dkb, dvb = ds.transpose(2, 3) @ qb * scale, p.transpose(2, 3) @ gb
            dk.index_add_(2, s_pos, dkb.view(B, Hkv, rep, -1, D).sum(2))
            dv.index_add_(2, s_pos, dvb.view(B, Hkv, rep, -1, D).sum(2))
    dt = st["q"].dtype
    if not train:
        return (_julia(x, dt),)
    out = tuple(_julia(t, dt) for t in (x, dq, dk, dv))
    return out + ((dtable.to(dt),) if dtable is not None else ())


def _plain_fill(st):
    case = st["case"]
    L, C, sinks = case["L"], case["capacity"], case["sinks"]
    for b, n in enumerate(_lengths(case) or [L] * case["B"]):
        last = torch.arange(max(sinks, n - (C - sinks)), max(sinks, n), device="cuda")
        src = torch.cat([torch.arange(min(sinks, n), device="cuda"), last])
        dst = torch.where(src < sinks, src, sinks + (src - sinks) % (C - sinks))
        st["kcache"][:, :, dst, b] = st["k"][:, :, src, b]
        st["vcache"][:, :, dst, b] = st["v"][:, :, src, b]


def _plain_step(st):
    case = st["case"]
    C, sinks, W = case["capacity"], case["sinks"], case["window"]
    lens = st["lengths"].long()
    B, dev = case["B"], lens.device
    ring = C - sinks
    new = torch.where(lens < sinks, lens, sinks + (lens - sinks).clamp(min=0) % ring)
    idx = torch.arange(B, device=dev)
    st["kcache"].permute(3, 2, 1, 0)[idx, new] = st["k"].permute(2, 1, 0)
    st["vcache"].permute(3, 2, 1, 0)[idx, new] = st["v"].permute(2, 1, 0)
    # the position that each slot holds now: the newest one congruent to it
    slots = torch.arange(C, device=dev)[None]
    pos = torch.where(slots < sinks, slots, lens[:, None] - (lens[:, None] - slots) % ring)
    seen = (pos >= 0) & (pos <= lens[:, None]) & ((lens[:, None] - pos < W) | (pos < sinks)) & ((slots < sinks) | (pos >= sinks))
    q = st["q"].permute(2, 1, 0).float()
    k, v = st["kcache"].permute(3, 1, 2, 0).float(), st["vcache"].permute(3, 1, 2, 0).float()
    H, D, Hkv = q.shape[1], q.shape[2], k.shape[1]
    z = (q.view(B, Hkv, H // Hkv, D) @ k.transpose(2, 3)).view(B, H, C) / math.sqrt(D)
    if "table" in st:
        bk = _bucket_of((pos - lens[:, None]).clamp(max=0), case["buckets"], case["max_distance"], False)
        z = z + st["table"].float()[:, bk].transpose(0, 1)
    z = torch.where(seen[:, None], z, -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    x = (p.view(B, Hkv, H // Hkv, C) @ v).view(B, H, D)
    return x.to(st["q"].dtype).permute(2, 1, 0)


def _plain_bias(st):
    case, dt = st["case"], st["table"].dtype
    rel = torch.arange(case["S"], device="cuda")[:, None] - torch.arange(case["L"], device="cuda")[None, :]
    bk = _bucket_of(rel, case["buckets"], case["max_distance"], case["bidirectional"])
    bias = st["table"].float()[:, bk].to(dt).permute(1, 2, 0)[..., None]
    per_head = st["delta"].permute(2, 3, 0, 1).float().sum(1, dtype=torch.float64)
    dtable = torch.zeros(case["H"], case["buckets"], dtype=torch.float64, device="cuda")
    dtable.index_add_(1, bk.flatten(), per_head.flatten(1))
    return bias, dtable.to(dt)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "bias":
        return _plain_bias(state)
    if kind == "step":
        return _plain_step(state), state["kcache"], state["vcache"]
    if kind == "train":
        return _plain_attention(state, True)
    x = _plain_attention(state, False)[0]
    _plain_fill(state)
    return x, state["kcache"], state["vcache"]


# ---------------------------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------------------------
def work(case):
    es, H, B = (2 if case["dtype"] == "bf16" else 4), case["H"], case["B"]
    if case["kind"] == "bias":
        one = case["S"] * case["L"] * H
        return {"bytes": es * (one * (1 + B) + 2 * H * case["buckets"]), "flops": one * B}
    D, Hkv = case["D"], case["Hkv"]
    table = es * H * case["buckets"]
    if case["kind"] == "step":
        seen = sum(_visible_pairs_last(n + 1, case["window"], case["sinks"]) for n in _lengths(case))
        # the visible rows but the new one come from the cache; q, the new rows (read and written), x
        return {"bytes": es * (2 * D * Hkv * (seen - B) + 2 * D * H * B + 4 * D * Hkv * B) + table + 4 * B, "flops": 4 * D * H * seen}
    lens = _lengths(case) or [case["L"]] * B
    pairs = H * sum(n * _visible_pairs(m, case["window"], case["sinks"], case["causal"]) for m, n in _counted(lens))
    rows_q, rows_k = D * H * case["L"] * B, D * Hkv * case["L"] * B
    if case["kind"] == "prefill":
        kept = sum(min(n, case["capacity"]) for n in lens)
        return {"bytes": es * (2 * rows_q + 2 * rows_k + 2 * D * Hkv * kept) + table, "flops": 4 * D * pairs}
    # forward: q, k, v -> x; pullback: the cotangent -> dq, dk, dv (the arrays of the forward pass once more)
    return {"bytes": es * (2 * rows_q + 2 * rows_k + 3 * rows_q + 4 * rows_k) + 3 * table, "flops": 14 * D * pairs}


def _counted(lens):
    return [(m, lens.count(m)) for m in sorted(set(lens))]


def _visible_pairs_last(n, window, sinks):
    """Keys that the last of n tokens sees."""
    lo = max(0, n - window)
    return n - lo + min(sinks, lo)


# ---------------------------------------------------------------------------------------------
# exact
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    """From the definition, one head of one sequence at a time, in 64 bits; gradients by differentiating that."""
    st = prepare(case, seed)
    dev = "cuda"

    def bucket_table(rel, both):
        n = case["buckets"] // 2 if both else case["buckets"]
        top = int(rel.abs().max()) if rel.numel() else 0
        e, of = n // 2, []
        for d in range(top + 1):
            j = d
            if d >= e:                      # e + floor(log(d / e) / log(max / e) * (n - e)), decided in whole numbers
                j = e
                while j + 1 < n and d ** (n - e) * e ** (j + 1 - e) >= case["max_distance"] ** (j + 1 - e) * e ** (n - e):
                    j += 1
            of.append(j)
        of = torch.tensor(of, device=dev)
        if both:
            return of[rel.abs()] + torch.where(rel > 0, n, 0)
        return of[(-rel).clamp(min=0)]

    table = st["table"].double() if "table" in st else None
    if case["kind"] == "bias":
        s, l = torch.arange(case["S"], device=dev), torch.arange(case["L"], device=dev)
        bk = bucket_table(s[:, None] - l[None, :], case["bidirectional"])
        bias = torch.stack([table[h][bk] for h in range(case["H"])], 2)[..., None]
        dtable = torch.zeros_like(table)
        total = st["delta"].double().sum(3)
        for j in range(case["buckets"]):
            dtable[:, j] = (total * (bk == j)[..., None]).sum((0, 1))
        return bias, dtable

    D, H, Hkv, B, W, sinks = (case[n] for n in ("D", "H", "Hkv", "B", "window", "sinks"))
    rep, lens = H // Hkv, _lengths(case)

    def attend(q, k, v, seen, bias):
        z = (q @ k.T) / math.sqrt(D)
        if bias is not None:
            z = z + bias
        z = z.masked_fill(~seen, -math.inf)
        return torch.softmax(z, -1).masked_fill(~seen, 0.0) @ v

    if case["kind"] == "step":
        C = case["capacity"]
        kc, vc = st["kcache"].double(), st["vcache"].double()
        x = torch.zeros(D, H, B, dtype=torch.float64, device=dev)
        for b, n in enumerate(lens):
            kc[:, :, _slot(n, sinks, C), b] = st["k"][:, :, b].double()
            vc[:, :, _slot(n, sinks, C), b] = st["v"][:, :, b].double()
            pos = [p for p in range(max(0, n - W + 1), n + 1)]
            pos = [p for p in range(min(sinks, pos[0]))] + pos
            at = torch.tensor([_slot(p, sinks, C) for p in pos], device=dev)
            rel = torch.tensor(pos, device=dev) - n
            bk = bucket_table(rel, False) if table is not None else None
            for h in range(H):
                x[:, h, b] = attend(st["q"][:, h, b].double()[None], kc[:, h // rep, at, b].T, vc[:, h // rep, at, b].T,
                                    torch.ones(1, len(pos), dtype=torch.bool, device=dev), table[h][bk][None] if table is not None else None)[0]
        return x, kc, vc

    L, causal = case["L"], case["causal"]
    if 8.0 * H * B * L * L > 3e11:          # about 20 seconds
        return None
    train = case["kind"] == "train"
    pos = torch.arange(L, device=dev)
    rel = pos[None, :] - pos[:, None]
    band = (rel.abs() < W) | (pos < sinks)[None, :]
    if causal:
        band = band & (rel <= 0)
    bk = bucket_table(rel, _both_ways(case)) if table is not None else None
    x = torch.zeros(D, H, L, B, dtype=torch.float64, device=dev)
    dq, dk, dv = torch.zeros_like(x), *(torch.zeros(D, Hkv, L, B, dtype=torch.float64, device=dev) for _ in range(2))
    dtable = torch.zeros_like(table) if table is not None else None
    for b in range(B):
        n = L if lens is None else lens[b]
        for h in range(H):
            q, k, v = (st[a][:, h // (rep if a != "q" else 1), :n, b].T.double().requires_grad_(train) for a in ("q", "k", "v"))
            bias = table[h][bk[:n, :n]].requires_grad_(train) if table is not None else None
            o = attend(q, k, v, band[:n, :n], bias)
            x[:, h, :n, b] = o.detach().T
            if train:
                leaves = [q, k, v] + ([bias] if bias is not None else [])
                grads = torch.autograd.grad(o, leaves, st["delta"][:, h, :n, b].T.double())
                dq[:, h, :n, b] = grads[0].T
                dk[:, h // rep, :n, b] += grads[1].T
                dv[:, h // rep, :n, b] += grads[2].T
                if bias is not None:
                    dtable[h].index_add_(0, bk[:n, :n].flatten(), grads[3].flatten())
    if train:
        return (x, dq, dk, dv) + ((dtable,) if dtable is not None else ())
    kc, vc = st["kcache"].double(), st["vcache"].double()
    for b in range(B):
        n = L if lens is None else lens[b]
        for p in range(n):                  # in order: a later token takes an earlier one's slot
            if p < sinks or p + (case["capacity"] - sinks) >= n:
                i = _slot(p, sinks, case["capacity"])
                kc[:, :, i, b] = st["k"][:, :, p, b].double()
                vc[:, :, i, b] = st["v"][:, :, p, b].double()
    return x, kc, vc
