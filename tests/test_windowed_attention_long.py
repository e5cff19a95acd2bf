"""Windowed attention where blocks take many items in turn, where buckets of a row cancel and where the sinks' tiles are shared by blocks,
against the definition in 64 bits.

Two tolerances. Per element, that of test_windowed_attention.py with the number of terms of that output. Per output, by norm, which a lost
tile or diagonal does not pass: errors that are independent of each other add up by their squares. Root mean squares, u = 2^-24:
  a rounding to bf16 is off by half a step of 2^-8 at most and evenly spread: 2^-8 / sqrt(3) of the value. The weights (x, dv, dtable) or the
  weights and the logits' gradients (dq, dk) are rounded, and each result;
  a sum of n Float32 terms of random sign: u sqrt(n) of its value; a logit of D products therefore u sqrt(D) times its size, its weight as
  much of itself, with 16 u for the exponential, the row's sum and the products of a term; BFloat16's exponential: 2^-20;
  dx . x, which a row's logits share: 4 u sqrt(E), and for BFloat16 2^-17, for its x comes in two parts of 8 bits each.
Half as much again is allowed (the least outputs have eight entries)."""
import math

import pytest
import torch

import luxlib_b200 as L
from luxlib_b200 import _cabi
import window_reference as R
from test_windowed_attention import B6, B32, B32C, CASES, DT, U16, U32

NAMES = ("x", "dq", "dk", "dv", "dtable")


def norm_limit(dt, name, ref, D, E, n):
    r16 = U16 / math.sqrt(3) if dt == "bf16" else 0.0
    r32 = U32 * (math.sqrt(D) + 16) * (ref["zrms"] + 1) + (2.0 ** -20 if dt == "bf16" else 0.0)
    terms, value = float(ref[name + "_rms"].norm()), float(ref[name].norm())
    roundings = 2 if name in ("dq", "dk") else 1
    lim = r16 * math.sqrt(roundings * terms ** 2 + value ** 2) + r32 * terms + U32 * (math.sqrt(n) + 1) * value
    if name == "dtable":
        lim += (4 * U32 * math.sqrt(E) + (2.0 ** -17 if dt == "bf16" else 0.0)) * float(ref["dtable_row"].norm())
    return 1.5 * lim


def element_limit(dt, name, ref, D, E, n):
    rel = U32 * (2 * (D + 4) * (ref["zmax"] + 1) + 2 * E + n + 32)
    if dt == "bf16":
        rel += 2.0 ** -20 + 2.0 ** -16 + U16 * 3
    return rel * ref[name + "_mag"] + 1e-35


def close(got, ref, dt, D, E, terms, names=NAMES, where=None):
    """`where`: name -> mask of the entries that are compared."""
    for name in names:
        if name not in ref:
            continue
        g, r = got[name].double(), ref[name]
        assert g.shape == r.shape, name
        mask = torch.ones_like(r, dtype=torch.bool) if where is None or name not in where else where[name]
        err = torch.where(mask, (g - r).abs(), 0.0)
        assert torch.isfinite(err).all(), f"{name}: not finite at {(~torch.isfinite(err)).nonzero()[0].tolist()}"
        over = err > element_limit(dt, name, ref, D, E, terms[name])
        assert not over.any(), f"{name}: {int(over.sum())} entries off, first at {over.nonzero()[0].tolist()}"
        lim = norm_limit(dt, name, ref, D, E, terms[name])
        assert float(err.norm()) <= lim, f"{name}: off by {float(err.norm()):.3e}, {float(err.norm()) / lim:.2f} times the limit"


def inputs(seed, dt, D, E, H, Hkv, Lq, S, B, columns=0, device="cuda"):
    """Julia arrays of the type, and the same values in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    t = {}
    for n, (f, h, tokens) in (("q", (D, H, Lq)), ("k", (D, Hkv, S)), ("v", (E, Hkv, S)), ("dx", (E, H, Lq))):
        t[n] = torch.randn(B, tokens, h, f, generator=g).to(DT[dt]).to(device).permute(3, 2, 1, 0)
    if columns:
        t["table"] = torch.randn(columns, H, generator=g).to(DT[dt]).to(device).permute(1, 0)
    return t, {n: x.double() for n, x in t.items()}


def terms_of(H, Hkv, Lq, S, window, sinks, causal):
    keys = min(S, (1 if causal else 2) * window + sinks)
    queries = (H // Hkv) * (Lq if sinks else min(Lq, 2 * window))
    return {"x": keys, "dq": keys, "dk": queries, "dv": queries, "dtable": 64 + 127 * (keys // 32 + 2)}


def run(t, window, sinks, causal, buckets, lengths):
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kw = dict(window=window, sinks=sinks, is_causal=causal, table=t.get("table"), buckets=buckets, lengths=lens)
    x, pb = L.rrule_windowed_attention(t["q"], t["k"], t["v"], **kw)
    got = dict(zip(NAMES, (x,) + pb(t["dx"])))
    torch.cuda.synchronize()
    assert _cabi.load().lb2_poll_device_status(L.arrays.current_stream(x.device)) == _cabi.OK
    return got


def reference(d, window, sinks, causal, buckets, lengths, **kw):
    return R.attention(d["q"], d["k"], d["v"], d["dx"], window, sinks, causal, d.get("table"), buckets.first if buckets else None,
                       bool(buckets and buckets.bidirectional), lengths, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(len(v) if hasattr(v, "first") else v) for v in c))
def test_small_cases_by_norm(dt, case):
    """The shapes of test_windowed_attention.py within the limit by norm, and element by element with each output's own number of terms."""
    D, E, H, Hkv, T, S, B, window, sinks, causal, buckets, lengths = case
    t, d = inputs(40, dt, D, E, H, Hkv, T, S, B, len(buckets) if buckets else 0)
    got = run(t, window, sinks, causal, buckets, lengths)
    close(got, reference(d, window, sinks, causal, buckets, lengths), dt, D, E, terms_of(H, Hkv, T, S, window, sinks, causal))


# D, E, H, Hkv, B, L, window, sinks, causal, buckets, lengths: more tiles than twice the SMs, and no even number of them
MANY = [
    (64, 64, 32, 8, 2, 1300, 200, 5, True, B32C, None),
    (128, 128, 32, 16, 1, 1300, 200, 5, True, B32C, None),
    (64, 64, 15, 5, 6, 1100, 130, 0, False, B32, [1100, 0, 700, 1, 0, 129]),        # three heads on one, empty sequences between full ones
    (128, 128, 15, 15, 3, 1300, 300, 1, False, B32, [1300, 0, 1290]),
    (128, 128, 16, 8, 41, 70, 20, 2, False, B6, [70 - 7 * (i % 11) for i in range(41)]),   # many short sequences
    (64, 64, 16, 8, 41, 70, 20, 0, True, B6, [70 - 7 * (i % 11) for i in range(41)]),
    (96, 40, 24, 12, 3, 900, 260, 140, True, None, None),                         # sinks over more than a tile, shared by blocks
    (64, 64, 16, 4, 1, 2600, 2500, 3, True, B32C, None),                          # long items, which SMs take as they come free
    (128, 128, 16, 16, 1, 2600, 2500, 0, False, None, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(str(len(v) if hasattr(v, "__len__") else v) for v in c))
def test_blocks_that_take_many_tiles(dt, case):
    D, E, H, Hkv, B, T, window, sinks, causal, buckets, lengths = case
    t, d = inputs(41, dt, D, E, H, Hkv, T, T, B, len(buckets) if buckets else 0)
    got = run(t, window, sinks, causal, buckets, lengths)
    close(got, reference(d, window, sinks, causal, buckets, lengths), dt, D, E, terms_of(H, Hkv, T, T, window, sinks, causal))
    again = run(t, window, sinks, causal, buckets, lengths)
    assert all(torch.equal(got[n], again[n]) for n in NAMES if got[n] is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("buckets", [None, B32C], ids=["plain", "bias"])
@pytest.mark.parametrize("rising", [True, False])
def test_rows_whose_maximum_moves_from_tile_to_tile(dt, D, buckets, rising):
    """Logits that rise (or fall) by some 2^10 a tile: sums and accumulators are scaled again at every tile, or never."""
    H, Hkv, T, window, sinks = 6, 3, 700, 500, 2
    t, _ = inputs(50, dt, D, D, H, Hkv, T, T, 1, len(buckets) if buckets else 0)
    ramp = torch.linspace(0.0, 5.0, T, device="cuda")
    ramp = ramp if rising else ramp.flip(0)
    t["k"] = L.as_colmajor((t["k"].float() * 0.5 + ramp[None, None, :, None]).to(DT[dt]))
    t["q"] = L.as_colmajor((t["q"].float() * 0.5 + 60.0 / (7.0 * math.sqrt(D))).to(DT[dt]))      # times D / sqrt(D) and 5 / 700 a key
    got = run(t, window, sinks, True, buckets, None)
    ref = reference({n: x.double() for n, x in t.items()}, window, sinks, True, buckets, None)
    close(got, ref, dt, D, D, terms_of(H, Hkv, T, T, window, sinks, True))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_calls_at_once_from_threads_on_their_own_streams(dt):
    """Forward, pullback, fill and step of three threads at the same time give what they give alone."""
    import threading

    def work(t, steps):
        x, pb = L.rrule_windowed_attention(t["q"], t["k"], t["v"], window=150, sinks=3, table=t["table"], buckets=B32C)
        out = [x, *pb(t["dx"])]
        kc, vc = (L.jl_zeros((64, 4, 200, 2), DT[dt], "cuda") for _ in range(2))
        L.windowed_cache_fill(kc, vc, t["k"], t["v"], sinks=3)
        lens = torch.full((2,), 600, dtype=torch.int32, device="cuda")
        for i in range(steps):
            out.append(L.windowed_attention_step(t["q"][:, :, i], t["k"][:, :, i], t["v"][:, :, i], kc, vc, lens, window=150, sinks=3))
            lens += 1
        return out + [kc, vc]

    sets = [inputs(51 + i, dt, 64, 64, 8, 4, 600, 600, 2, len(B32C))[0] for i in range(3)]
    alone = [work(t, 5) for t in sets]
    torch.cuda.synchronize()
    results, errors = [[] for _ in sets], []

    def run_one(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(4):
                    results[i].append(work(sets[i], 5))
            stream.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run_one, args=(i,)) for i in range(3)]
    [th.start() for th in threads], [th.join() for th in threads]
    assert not errors
    for want, got in zip(alone, results):
        assert all(torch.equal(a, b) for once in got for a, b in zip(want, once))
    assert _cabi.load().lb2_poll_device_status(None) == _cabi.OK


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_padding_that_is_not_finite_with_shared_sinks_and_many_tiles(dt, D, value):
    """NaN or infinities past the lengths, in sink tiles that several blocks share and in blocks that take many tiles: as without them."""
    H, Hkv, B, T, window, sinks, lengths = 32, 8, 2, 1300, 200, 5, [1300, 1130]
    t, d = inputs(42, dt, D, D, H, Hkv, T, T, B, len(B32C))
    ref = reference(d, window, sinks, True, B32C, lengths)
    for n in ("q", "k", "v", "dx"):
        t[n][..., lengths[1]:, 1] = value
    got = run(t, window, sinks, True, B32C, lengths)
    close(got, ref, dt, D, D, terms_of(H, Hkv, T, T, window, sinks, True))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_sink_that_is_not_finite(dt, D):
    """An infinite value in a sink of one key head, NaN in a late key of another: they reach the queries that see them and nothing else."""
    H, Hkv, B, T, window, sinks = 32, 8, 2, 1300, 200, 5
    rep = H // Hkv
    t, d = inputs(43, dt, D, D, H, Hkv, T, T, B)
    ref = reference(d, window, sinks, True, None, None)
    t["v"][2, 3, 1, 0] = math.inf
    t["k"][1, 7, 1250, 1] = math.nan
    got = run(t, window, sinks, True, None, None)
    of3, of7 = slice(3 * rep, 4 * rep), slice(7 * rep, 8 * rep)
    inf = got["x"][2, of3, 1:, 0]
    assert (inf == math.inf).all()                                       # all weights are positive
    seers = R.sees(T, T, window, sinks, True, T, "cuda")[:, 1250]
    assert torch.isnan(got["x"][:, of7, seers, 1]).all() and torch.isnan(got["dq"][:, of7, seers, 1]).all()
    assert torch.isnan(got["dv"][:, 7, 1250, 1]).all() and torch.isnan(got["dk"][:, 7, 1250, 1]).all()
    where = {n: torch.ones_like(ref[n], dtype=torch.bool) for n in NAMES if n in ref}
    where["x"][2, of3, 1:, 0] = False
    where["dq"][:, of3, 1:, 0] = False                                   # dp and dx . x are infinite; weights, and with them dv, are not
    where["dk"][:, 3, :, 0] = False
    seen = R.sees(T, T, window, sinks, True, T, "cuda")[seers].any(0)
    where["x"][:, of7, seers, 1] = False
    where["dq"][:, of7, seers, 1] = False
    for n in ("dk", "dv"):
        where[n][:, 7, seen, 1] = False
    close(got, ref, dt, D, D, terms_of(H, Hkv, T, T, window, sinks, True), where=where)


# ---- the table's gradient ------------------------------------------------------------------------
# D, H, Hkv, B, L, S, window, sinks, causal, buckets, lengths: nearly all pairs of a row lie in one bucket, whose gradients cancel
F4 = lambda top: L.RelativeBuckets.make(4, top, True)
CANCEL = [
    (128, 2, 1, 5, 127, 127, 129, 0, True, F4(6), None),
    (64, 3, 1, 2, 1100, 1100, 246, 28, True, F4(10), [1100, 1]),
    (32, 6, 3, 1, 820, 445, 129, 64, True, F4(5), None),
    (80, 8, 2, 1, 300, 300, 64, 130, False, L.RelativeBuckets.make(8, 20, False), None),
    (128, 4, 4, 1, 700, 700, 500, 0, True, L.RelativeBuckets((0, 700), False), None),     # one bucket holds all: nothing
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("case", CANCEL, ids=lambda c: "-".join(str(len(v) if hasattr(v, "__len__") else v) for v in c))
def test_gradients_of_buckets_that_cancel(dt, case):
    D, H, Hkv, B, T, S, window, sinks, causal, buckets, lengths = case
    t, d = inputs(44, dt, D, D, H, Hkv, T, S, B, len(buckets))
    got = run(t, window, sinks, causal, buckets, lengths)
    close(got, reference(d, window, sinks, causal, buckets, lengths), dt, D, D, terms_of(H, Hkv, T, S, window, sinks, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("case", CANCEL, ids=lambda c: "-".join(str(len(v) if hasattr(v, "__len__") else v) for v in c))
def test_gradients_of_buckets_that_cancel_from_a_cotangent_off_its_alignment(dt, case):
    """Whichever kernels the pullback takes: with the weights of the forward pass, which the cotangent's address does not change."""
    D, H, Hkv, B, T, S, window, sinks, causal, buckets, lengths = case
    t, d = inputs(49, dt, D, D, H, Hkv, T, S, B, len(buckets))
    flat = torch.zeros(t["dx"].numel() + 1, dtype=DT[dt], device="cuda")
    dx = torch.as_strided(flat, t["dx"].shape, t["dx"].stride(), 1)
    dx.copy_(t["dx"])
    assert L.is_colmajor(dx) and dx.data_ptr() % 16
    got = run(dict(t, dx=dx), window, sinks, causal, buckets, lengths)
    close(got, reference(d, window, sinks, causal, buckets, lengths), dt, D, D, terms_of(H, Hkv, T, S, window, sinks, causal))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_a_table_gradient_without_one_diagonal_is_off_limits(dt):
    """The limit by norm is narrow enough to miss a diagonal that a kernel forgets."""
    _, d = inputs(45, dt, 64, 64, 2, 1, 300, 300, 1, len(B32C), device="cpu")
    ref = reference(d, 64, 4, True, B32C, None)
    for rel in (0, -5, -40, -63):
        less = reference(d, 64, 4, True, B32C, None, without_diagonal=rel)
        assert float((less["dtable"] - ref["dtable"]).norm()) > norm_limit(dt, "dtable", ref, 64, 64, terms_of(2, 1, 300, 300, 64, 4, True)["dtable"]), rel


# ---- single tokens -------------------------------------------------------------------------------
def step_inputs(seed, dt, D, E, H, Hkv, B, cap, columns):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*reversed(s), generator=g).to(DT[dt]).cuda().permute(*reversed(range(len(s))))
    t = {"q": r(D, H, B), "k": r(D, Hkv, B), "v": r(E, Hkv, B), "kc": r(D, Hkv, cap, B), "vc": r(E, Hkv, cap, B)}
    if columns:
        t["table"] = r(H, columns)
    return t


def slot(p, sinks, cap):
    return p if p < sinks else sinks + (p - sinks) % (cap - sinks)


def step_reference(t, lens, window, sinks, buckets):
    """x, its measures, and the caches afterwards, in 64 bits."""
    d = {n: x.double().clone() for n, x in t.items()}
    D, H, B = d["q"].shape
    E, Hkv, cap = d["vc"].shape[:3]
    out = {n: torch.zeros(E, H, B, dtype=torch.float64, device="cuda") for n in ("x", "x_mag", "x_rms")}
    out["zmax"], squares, pairs = 0.0, 0.0, 0
    for b, n in enumerate(lens):
        d["kc"][:, :, slot(n, sinks, cap), b], d["vc"][:, :, slot(n, sinks, cap), b] = d["k"][:, :, b], d["v"][:, :, b]
        pos = list(range(max(0, n - window + 1), n + 1))
        pos = list(range(min(sinks, pos[0]))) + pos
        at = torch.tensor([slot(p, sinks, cap) for p in pos], device="cuda")
        for h in range(H):
            kk, vv, qq = d["kc"][:, h * Hkv // H, at, b], d["vc"][:, h * Hkv // H, at, b], d["q"][:, h, b]
            z, zm = qq @ kk / D ** 0.5, qq.abs() @ kk.abs() / D ** 0.5
            if buckets is not None:
                bias = d["table"][h, torch.tensor([buckets.bucket(p - n) for p in pos], device="cuda")]
                z, zm = z + bias, zm + bias.abs()
            out["zmax"] = max(out["zmax"], float(zm.max()))
            squares, pairs = squares + float((z ** 2).sum()), pairs + z.numel()
            p = torch.softmax(z, 0)
            out["x"][:, h, b], out["x_mag"][:, h, b], out["x_rms"][:, h, b] = vv @ p, vv.abs() @ p, vv ** 2 @ p ** 2
    out["x_rms"], out["zrms"] = out["x_rms"].sqrt(), (squares / pairs) ** 0.5
    return out, d["kc"], d["vc"]


def step(t, lens, window, sinks, buckets):
    x = L.windowed_attention_step(t["q"], t["k"], t["v"], t["kc"], t["vc"], torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window,
                                  sinks=sinks, table=t.get("table"), buckets=buckets)
    torch.cuda.synchronize()
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 40, 24])
@pytest.mark.parametrize("rep,Hkv,window,sinks,buckets", [(3, 2, 37, 0, None), (5, 2, 60, 3, B32C), (9, 1, 200, 4, None), (12, 2, 1300, 4, B32C), (16, 1, 64, 1, None),
                                                         (20, 2, 150, 2, B32C), (33, 1, 1100, 0, None)])
def test_steps_of_many_query_heads_per_key_head(dt, D, rep, Hkv, window, sinks, buckets):
    cap = window + sinks + 5
    t = step_inputs(46, dt, D, D, rep * Hkv, Hkv, 3, cap, len(buckets) if buckets else 0)
    lens = [3 * cap + 1, window // 2, 0]
    ref, kc, vc = step_reference(t, lens, window, sinks, buckets)
    got = step(t, lens, window, sinks, buckets)
    close({"x": got}, ref, dt, D, D, {"x": window + sinks}, names=("x",))
    assert torch.equal(t["kc"].double(), kc) and torch.equal(t["vc"].double(), vc)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,rep", [(64, 2), (128, 1), (128, 12), (32, 5), (33, 2)])
@pytest.mark.parametrize("window", [21, 600])
def test_an_infinite_value_that_a_step_sees(dt, D, rep, window):
    """One infinite feature of one key: that feature of x is infinite, the others are as without it, whichever key it is."""
    sinks, cap, n = 2, window + 9, 3 * window
    clean = step_inputs(47, dt, D, D, 2 * rep, 2, 1, cap, 0)
    ref, _, _ = step_reference(clean, [n], window, sinks, None)
    seen = list(range(sinks)) + list(range(n - window + 1, n + 1))
    for p in seen if window < 100 else seen[::37] + seen[-17:]:
        t = {m: x.clone(memory_format=torch.preserve_format) for m, x in clean.items()}
        if p == n:
            t["v"][5, 1, 0] = -math.inf
        else:
            t["vc"][5, 1, slot(p, sinks, cap), 0] = -math.inf
        got = step(t, [n], window, sinks, None)
        assert (got[5, rep:] == -math.inf).all(), p
        where = torch.ones_like(ref["x"], dtype=torch.bool)
        where[5, rep:] = False
        close({"x": got}, ref, dt, D, D, {"x": window + sinks}, names=("x",), where={"x": where})


# ---- no query heads ------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_without_query_heads_the_keys_gradients_are_zero(dt):
    """Sums over nothing, not what the memory held."""
    lib = _cabi.load()
    full = lambda *s: L.jl_empty(s, DT[dt], "cuda").fill_(7.0)
    k, v, dk, dv = full(64, 2, 9, 3), full(32, 2, 9, 3), full(64, 2, 9, 3), full(32, 2, 9, 3)
    dims = _cabi.WindowDims(64, 32, 0, 2, 9, 9, 3, 4, 1, 1)
    call = lambda dk, dv: lib.lb2_window_attention_bwd(None, dk, dv, None, None, None, None, None, None, k.data_ptr(), v.data_ptr(), None, None, None, 0.125,
                                                       dims, L.arrays.dtype_code(DT[dt]), None, 0, L.arrays.current_stream(k.device))
    assert call(dk.data_ptr(), dv.data_ptr()) == _cabi.OK
    assert not dk.any() and not dv.any()
    assert call(None, dv.data_ptr()) == _cabi.BAD_ARG
    x, pb = L.rrule_windowed_attention(full(64, 0, 9, 3), k, v, window=4)
    dq, dk, dv, _ = pb(x)
    assert tuple(x.shape) == (32, 0, 9, 3) and tuple(dq.shape) == (64, 0, 9, 3) and not dk.any() and not dv.any()


def test_a_step_without_query_heads_is_refused():
    """It has no place for the token's keys and values but the cache, which it would not reach."""
    lib, one = _cabi.load(), 256
    step = lambda **kw: lib.lb2_window_attention_step(one, one, one, one, one, one, None, None, one, 0.125, _cabi.WindowDims(*dict(dict(
        head_dim=64, value_dim=64, heads=0, kv_heads=2, queries=1, keys=9, batch=3, window=4, sinks=1, causal=1), **kw).values()), 0, None)
    assert step() == _cabi.BAD_SHAPE and step(batch=0) == _cabi.OK and step(kv_heads=0) == _cabi.OK


@pytest.mark.gpu
def test_lengths_in_another_order_than_the_batch_are_refused():
    """Two batch dimensions: lengths of their shape or a vector in its order, not the transposed shape, which holds as many numbers."""
    z = lambda *s: L.jl_zeros(s, torch.float32, "cuda")
    n = lambda *s: L.jl_zeros(s, torch.int32, "cuda")
    q, c, one = z(8, 2, 4, 2, 3), z(8, 2, 5, 2, 3), z(8, 2, 2, 3)
    calls = (lambda lens: L.windowed_attention(q, q, q, window=2, lengths=lens), lambda lens: L.windowed_cache_fill(c, c.clone(), q, q, lens),
             lambda lens: L.windowed_attention_step(one, one, one, c, c.clone(), lens, window=2))
    for call in calls:
        call(n(2, 3)), call(n(6)), call(n(1, 2, 3))
        for wrong in (n(3, 2), n(6, 1)[:5], n(2, 1, 3)[:1]):
            with pytest.raises((L.DimensionMismatch, L.ArgumentError)):
                call(wrong)
    L.windowed_attention(q[..., :1], q[..., :1], q[..., :1], window=2, lengths=n(2))
    L.windowed_attention(q[..., :1, :1], q[..., :1, :1], q[..., :1, :1], window=2, lengths=torch.tensor(3, dtype=torch.int32, device="cuda"))


def test_shapes_of_lengths():
    ok = lambda shape, batch: L.ops._check_lengths(shape, batch)
    for shape, batch in (((2, 3), (2, 3)), ((6,), (2, 3)), ((), (1,)), ((1,), (1, 1)), ((4, 1), (4,)), ((0,), (0,)), ((0,), (0, 3)), ((0, 3), (0, 3))):
        ok(shape, batch)
    for shape, batch in (((3, 2), (2, 3)), ((5,), (2, 3)), ((), (2,)), ((2, 3), (6,)), ((0,), (2,)), ((3, 0), (0, 3))):
        with pytest.raises(L.DimensionMismatch):
            ok(shape, batch)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_a_bias_that_all_samples_share_where_there_are_none(dt):
    """scaled_dot_product_attention takes relative_position_bias for a batch of nothing too; its gradient is a sum over nothing."""
    table = L.jl_empty((2, len(B6)), DT[dt], "cuda").fill_(1.0)
    e = lambda n: L.jl_empty((64, 2, n, 0), DT[dt], "cuda")
    bias, pb_bias = L.rrule_relative_position_bias(table, B6, 5, 4)
    (x, _), pb = L.rrule_scaled_dot_product_attention(e(4), e(5), e(5), bias=bias)
    junk = torch.full((4096,), 7.0, device="cuda")                       # what the memory may hold
    del junk
    dbias = pb(x)[3]
    assert tuple(x.shape) == (64, 2, 4, 0) and tuple(dbias.shape) == tuple(bias.shape) and not dbias.any() and not pb_bias(dbias).any()


def test_a_prompt_in_the_memory_of_the_caches():
    """Refused unless it begins with its own cache and their samples lie alike."""
    flat = torch.arange(4000.0)
    at = lambda first, tokens, batch=1: L.arrays.jl_reshape(flat[first:first + 4 * 2 * tokens * batch], (4, 2, tokens, batch))
    check = L.ops._check_prompt_apart
    check(at(0, 9), at(1000, 9), at(0, 20), at(1000, 20))                # the prompt's first tokens are the cache
    check(at(0, 9, 2), at(1000, 9, 2), at(0, 9, 2), at(1000, 9, 2))
    check(at(0, 9), at(1000, 9), at(72, 20), at(1072, 20))               # side by side
    for kc, vc, k, v in ((at(0, 9), at(1000, 9), at(8, 20), at(2000, 20)), (at(0, 9), at(1000, 9), at(2000, 20), at(992, 20)),
                         (at(0, 9), at(1000, 9), at(1000, 9), at(2000, 9)), (at(0, 9), at(1000, 9), at(2000, 9), at(0, 9)),
                         (at(0, 9, 2), at(1000, 9, 2), at(0, 20, 2), at(2000, 20, 2))):
        with pytest.raises(L.ArgumentError, match="share memory"):
            check(kc, vc, k, v)


@pytest.mark.gpu
def test_a_cache_that_is_the_beginning_of_its_prompt():
    g = torch.Generator().manual_seed(48)
    k, v = (torch.randn(1, 23, 2, 4, generator=g).cuda().permute(3, 2, 1, 0) for _ in range(2))
    kc, vc = L.jl_zeros((4, 2, 9, 1), torch.float32, "cuda"), L.jl_zeros((4, 2, 9, 1), torch.float32, "cuda")
    L.windowed_cache_fill(kc, vc, k.clone(), v.clone(), sinks=2)
    with pytest.raises(L.ArgumentError, match="share memory"):
        L.windowed_cache_fill(k[:, :, 1:10], vc, k, v, sinks=2)
    L.windowed_cache_fill(k[:, :, :9], v[:, :, :9], k, v, sinks=2)
    assert torch.equal(k[:, :, :9], kc) and torch.equal(v[:, :, :9], vc)
