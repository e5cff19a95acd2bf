"""Windowed attention, its ring cache and the relative position bias against the definitions in 64 bits.

Tolerances, per element and relative to the same sum over absolute values (its magnitude), u = half a step of the type:
  Float32: a logit of D products is off by (D + 4) u Z at most, Z the largest magnitude of a logit; a weight p by the errors of its
  logit, of the row's log-sum and of the exponential: 2 (D + 4) u Z + 16 u; a sum over n terms adds n u, the products dx . v and dx . x
  E u each. Together u (2 (D + 4) (Z + 1) + 2 E + n + 32).
  BFloat16: those of Float32 arithmetic (the exponential to 2^-20 instead), and 2^-8 for each rounding to bf16 on the way: the weights
  and the result (x, dv); the logits' gradient and the result (dq, dk); the result alone (dtable). The x of dx . x comes in two
  parts, which leave 2^-16 of it."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import luxlib_b200 as L
from luxlib_b200 import _cabi
import window_oracle as W

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
U32, U16 = 2.0 ** -24, 2.0 ** -8


def rounded(a, dt):
    """The values a device array of that type holds, as float64."""
    return torch.from_numpy(np.ascontiguousarray(a)).to(DT[dt]).double().numpy()


def dev(a, dt):
    return L.from_numpy(a, dtype=DT[dt])


def host(t):
    return t.detach().to(torch.float64).cpu().numpy()


def bound(dt, name, mag, zmax, D, E, n):
    rel = U32 * (2 * (D + 4) * (zmax + 1) + 2 * E + n + 32)
    if dt == "bf16":
        rel += 2.0 ** -20 + 2.0 ** -16 + U16 * (1 if name == "dtable" else 2)
    return rel * mag + 1e-35


def check(got, ref, dt, names, D, E, n, rows=None):
    for name in names:
        g, r = host(got[name]), ref[name]
        assert g.shape == r.shape, name
        with np.errstate(invalid="ignore"):
            err, lim = np.abs(g - r), bound(dt, name, ref[name + "_mag"], ref["zmax"], D, E, n)
        bad = ~((err <= lim) | (np.isnan(g) & np.isnan(r)) | ((g == r) & np.isinf(g)))
        assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {g[bad][0]} instead of {r[bad][0]}, " \
                              f"{(err / np.maximum(lim, 1e-300))[bad].max():.1f} times the bound"


def make(seed, dt, D, E, H, Hkv, Lq, S, B, columns=0):
    rng = np.random.default_rng(seed)
    a = {"q": rng.standard_normal((D, H, Lq, B)), "k": rng.standard_normal((D, Hkv, S, B)), "v": rng.standard_normal((E, Hkv, S, B)),
         "dx": rng.standard_normal((E, H, Lq, B))}
    if columns:
        a["table"] = rng.standard_normal((H, columns))
    return {n: rounded(t, dt) for n, t in a.items()}


def run_case(dt, D, E, H, Hkv, Lq, S, B, window, sinks, causal, buckets=None, lengths=None, scale=None, a=None, seed=0, zmax=None):
    a = make(seed, dt, D, E, H, Hkv, Lq, S, B, len(buckets) if buckets else 0) if a is None else a
    first, both = (buckets.first, buckets.bidirectional) if buckets else (None, False)
    ref = W.attention(a["q"], a["k"], a["v"], window, sinks, causal, scale, a.get("table"), first, both, lengths, a["dx"])
    ref["zmax"] = ref["zmax"] if zmax is None else zmax
    t = {n: dev(x, dt) for n, x in a.items()}
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kw = dict(window=window, sinks=sinks, is_causal=causal, scale=scale, table=t.get("table"), buckets=buckets, lengths=lens)
    x, pb = L.rrule_windowed_attention(t["q"], t["k"], t["v"], **kw)
    dq, dk, dv, dtable = pb(t["dx"])
    assert (dtable is None) == (buckets is None)
    got = {"x": x, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}
    names = ["x", "dq", "dk", "dv"] + (["dtable"] if buckets else [])
    n = max(S, Lq) * (H // Hkv) if Hkv else 1
    check(got, ref, dt, names, D, E, n if buckets is None else n * Lq * B)
    assert torch.equal(L.windowed_attention(t["q"], t["k"], t["v"], **kw).cpu(), x.cpu()) or np.isnan(ref["x"]).any()
    assert L._cabi.load().lb2_poll_device_status(L.arrays.current_stream(x.device)) == _cabi.OK
    return got, ref


B32 = L.RelativeBuckets.make(32, 128, True)
B32C = L.RelativeBuckets.make(32, 128, False)
B6 = L.RelativeBuckets.make(6, 20, True)
B128 = L.RelativeBuckets.make(128, 300, True)
BD = L.RelativeBuckets((0, 0, 3, 3, 3, 9), False)          # starts that coincide: the earlier buckets are empty
BDB = L.RelativeBuckets((0, 0, 3, 3, 40), True)

# D, E, H, Hkv, L, S, B, window, sinks, causal, buckets, lengths
CASES = [
    (64, 64, 2, 2, 1, 1, 1, 1, 0, True, None, None),                 # one token
    (64, 64, 2, 1, 2, 2, 2, 1, 0, True, B32C, None),                 # each token sees itself alone
    (64, 64, 4, 2, 130, 130, 1, 17, 0, True, None, None),
    (64, 64, 2, 2, 257, 257, 2, 64, 4, True, B32C, None),
    (64, 64, 2, 2, 300, 300, 1, 1000, 0, True, None, None),          # a window wider than the sequence
    (64, 64, 2, 1, 290, 290, 1, 33, 150, True, B6, None),            # sinks over more than one tile
    (64, 64, 1, 1, 200, 200, 1, 5, 500, True, None, None),           # sinks past the end
    (128, 128, 4, 1, 259, 259, 1, 100, 3, True, B32C, None),
    (128, 128, 2, 2, 140, 140, 2, 50, 1, False, B32, None),          # both ways
    (64, 64, 3, 3, 197, 197, 3, 40, 1, False, B32, [197, 1, 0]),     # padded batch, an empty sequence
    (64, 64, 2, 2, 150, 150, 4, 64, 2, True, None, [-3, 149, 400, 64]),
    (64, 64, 2, 2, 200, 50, 1, 8, 0, True, None, None),              # queries past every key: rows that see nothing
    (64, 64, 2, 2, 50, 200, 1, 16, 2, True, B32C, None),             # more keys than queries
    (64, 64, 2, 2, 50, 200, 1, 16, 190, False, B32, None),
    (32, 32, 2, 2, 129, 129, 1, 128, 0, True, None, None),
    (80, 80, 4, 2, 131, 131, 1, 70, 4, True, B32C, None),
    (40, 96, 2, 2, 133, 133, 1, 31, 0, False, B128, None),           # features of keys and values differ
    (96, 40, 2, 1, 133, 133, 1, 31, 0, True, None, [100]),
    (33, 17, 2, 2, 70, 70, 2, 20, 2, True, B6, None),                # no vector of anything
    (130, 130, 2, 1, 70, 70, 1, 30, 0, True, B6, None),
    (256, 256, 2, 2, 100, 100, 1, 40, 3, False, B32, None),
    (1, 1, 1, 1, 40, 40, 1, 7, 0, True, None, None),
    (64, 64, 8, 1, 140, 140, 1, 60, 0, True, B32C, None),            # eight heads share a key head
    (128, 64, 2, 2, 385, 385, 1, 128, 128, True, B32C, [385]),       # tiles and window on the same boundaries
    (64, 64, 2, 2, 300, 300, 1, 260, 0, False, BD, None),            # one-sided buckets where keys come after the query too
    (128, 128, 2, 1, 300, 300, 1, 260, 4, False, BDB, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(len(v) if hasattr(v, "first") else v) for v in c))
def test_windowed_attention_fwd_bwd(dt, case):
    run_case(dt, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_windowed_attention_given_scale_and_large_logits(dt):
    run_case(dt, 64, 64, 2, 2, 150, 150, 1, 60, 2, True, scale=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 40, 33])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_query_does_not_see_does_not_reach_it(dt, D, value):
    """Infinities and NaN in tokens past the lengths, and in a token that only some queries see: all others are as without them."""
    a = make(3, dt, D, D, 2, 2, 200, 200, 2)
    for n in ("q", "k", "v", "dx"):
        a[n][..., 150:, 1] = value                                   # past the second sample's length
    a["k"][1, 0, 70, 0] = value
    a["v"][2, 1, 90, 0] = value
    a["dx"][0, 1, 100, 0] = value
    run_case(dt, D, D, 2, 2, 200, 200, 2, 9, 0, True, lengths=[200, 150], a=a)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 33])
def test_queries_that_see_one_key_alone_have_no_gradient_in_their_logits(dt, D):
    """Their weight is 1 whatever the logit: exactly zero, not the difference of two sums."""
    a = make(18, dt, D, D, 4, 2, 150, 150, 2, len(B6))
    t = {n: dev(x, dt) for n, x in a.items()}
    x, pb = L.rrule_windowed_attention(t["q"], t["k"], t["v"], window=1, table=t["table"], buckets=B6)
    dq, dk, dv, dtable = pb(t["dx"])
    assert np.array_equal(host(x), np.repeat(a["v"], 2, 1))
    assert not host(dq).any() and not host(dk).any() and not host(dtable).any()
    x, pb = L.rrule_windowed_attention(t["q"], t["k"][:, :, :1], t["v"][:, :, :1], window=5, sinks=1, table=t["table"], buckets=B6)
    dq, dk, dv, dtable = pb(t["dx"])
    assert not host(dq).any() and not host(dk).any() and not host(dtable).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_a_table_of_the_lowest_value_shuts_its_buckets_out(dt):
    """The type's lowest value as a bias: those keys weigh nothing; a row that sees only such keys weighs them evenly."""
    a = make(4, dt, 64, 64, 2, 2, 140, 140, 1, len(B6))
    a["table"][0, 2:] = torch.finfo(DT[dt]).min
    a["table"][1, :] = torch.finfo(DT[dt]).min
    a["q"][:, 1] = 0.0                                                # head 1: all logits are that bias
    got, ref = run_case(dt, 64, 64, 2, 2, 140, 140, 1, 30, 0, True, B6, a=a, zmax=20.0)
    assert all(np.isfinite(host(t)).all() for t in got.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_minus_infinity_in_the_table_hides_a_bucket(dt):
    a = make(5, dt, 64, 64, 1, 1, 140, 140, 1, len(B6))
    a["table"][0, 1] = -math.inf
    t = {n: dev(x, dt) for n, x in a.items()}
    x = L.windowed_attention(t["q"], t["k"], t["v"], window=30, table=t["table"], buckets=B6)
    ref = W.attention(a["q"], a["k"], a["v"], 30, 0, True, None, a["table"], B6.first, True)
    ref["zmax"] = 20.0
    check({"x": x}, ref, dt, ["x"], 64, 64, 140)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strided_inputs_other_streams_and_batch_dims(dt):
    """Views (every second token of a larger array, heads in another order of memory), two batch dimensions, another stream."""
    a = make(6, dt, 64, 64, 4, 2, 96, 96, 6)
    big = torch.zeros(2, 96, 6, 4, 64, device="cuda", dtype=DT[dt])                      # (pair, token, batch, head, feature)
    big[0] = dev(a["q"], dt).permute(2, 3, 1, 0)
    q = big[0].permute(3, 2, 0, 1)
    assert not L.is_colmajor(q)
    k, v, g = dev(a["k"], dt), dev(a["v"], dt), dev(a["dx"], dt)
    x0, pb0 = L.rrule_windowed_attention(dev(a["q"], dt), k, v, window=40, sinks=2)
    ref = [x0] + list(pb0(g))[:3]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x1, pb1 = L.rrule_windowed_attention(q, k, v, window=40, sinks=2)
        got = [x1] + list(pb1(g))[:3]
    side.synchronize()
    for r, t in zip(ref, got):
        assert torch.equal(r, t)
    five = lambda t: torch.as_strided(t, t.shape[:3] + (2, 3), t.stride()[:3] + (t.stride(3), 2 * t.stride(3)))
    x2, pb2 = L.rrule_windowed_attention(five(dev(a["q"], dt)), five(k), five(v), window=40, sinks=2)
    assert tuple(x2.shape) == (64, 4, 96, 2, 3) and torch.equal(five(x0), x2)
    for r, t in zip(ref[1:], pb2(five(g))):
        assert torch.equal(five(r), t)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_windowed_attention_is_the_same_every_time_and_in_a_graph(dt):
    a = make(7, dt, 64, 64, 4, 2, 300, 300, 2, len(B32C))
    t = {n: dev(x, dt) for n, x in a.items()}
    lens = torch.tensor([300, 123], dtype=torch.int32, device="cuda")

    def once():
        x, pb = L.rrule_windowed_attention(t["q"], t["k"], t["v"], window=70, sinks=3, table=t["table"], buckets=B32C, lengths=lens)
        return [x] + list(pb(t["dx"]))

    first = [r.clone() for r in once()]
    for _ in range(3):
        assert all(torch.equal(r, s) for r, s in zip(first, once()))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                        # two graphs, each with its own workspace, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once())
        graphs.append(g)
    for r in outs[0] + outs[1]:
        r.zero_()
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(r, s) for r, s in zip(first, o))
    t["q"].mul_(0.5)                          # new values in the same arrays
    lens.copy_(torch.tensor([40, 300], dtype=torch.int32))
    graphs[0].replay()
    assert all(torch.equal(r, s) for r, s in zip(once(), outs[0]))


@pytest.mark.gpu
def test_windowed_attention_against_differences():
    """<grad, d> against the central difference of the same Float32 operator along d: the loss is off by rel * (sum of magnitudes) on each
    side, over 2 eps; the difference itself by eps^2 / 6 times the third derivative, which the 64-bit oracle's difference also has."""
    a = make(8, "f32", 16, 16, 2, 1, 40, 40, 1, len(B6))
    kw = dict(window=12, sinks=2)
    rng = np.random.default_rng(9)
    eps = 2.0 ** -5
    t = {n: dev(x, "f32") for n, x in a.items()}
    x, pb = L.rrule_windowed_attention(t["q"], t["k"], t["v"], table=t["table"], buckets=B6, **kw)
    grads = dict(zip(("q", "k", "v", "table"), pb(t["dx"])))
    ref = W.attention(a["q"], a["k"], a["v"], 12, 2, True, None, a["table"], B6.first, True, None, a["dx"])
    for n in ("q", "k", "v", "table"):
        d = rounded(rng.standard_normal(a[n].shape), "f32")
        loss, exact = [], []
        for sign in (1, -1):
            b = dict(a, **{n: rounded(a[n] + sign * eps * d, "f32")})
            tb = {m: dev(y, "f32") for m, y in b.items()}
            y = L.windowed_attention(tb["q"], tb["k"], tb["v"], table=tb["table"], buckets=B6, **kw)
            loss.append((host(y) * a["dx"]).sum())
            o = W.attention(b["q"], b["k"], b["v"], 12, 2, True, None, b["table"], B6.first, True)
            exact.append((o["x"] * a["dx"]).sum())
        slack = bound("f32", "x", (ref["x_mag"] * np.abs(a["dx"])).sum(), 2 * ref["zmax"], 16, 16, 40) / eps
        truncation = abs((exact[0] - exact[1]) / (2 * eps) - (ref["d" + n] * d).sum())
        assert abs((loss[0] - loss[1]) / (2 * eps) - (host(grads[n]) * d).sum()) <= truncation + 2 * slack, n


def test_the_oracle_against_differences():
    rng = np.random.default_rng(10)
    D, E, H, Lq, S = 5, 4, 2, 14, 11
    a = {"q": rng.standard_normal((D, H, Lq, 2)), "k": rng.standard_normal((D, 1, S, 2)), "v": rng.standard_normal((E, 1, S, 2)),
         "table": rng.standard_normal((H, len(B6)))}
    dx = rng.standard_normal((E, H, Lq, 2))
    for causal in (True, False):
        f = lambda b, dx=None: W.attention(b["q"], b["k"], b["v"], 4, 2, causal, 1.3, b["table"], B6.first, True, [9, 14], dx)
        ref = f(a, dx)
        for n in a:
            d, eps = rng.standard_normal(a[n].shape), 1e-5
            up, down = (f(dict(a, **{n: a[n] + s * eps * d}))["x"] for s in (1, -1))
            assert abs(((up - down) * dx).sum() / (2 * eps) - (ref["d" + n] * d).sum()) < 1e-7 * np.abs(ref["d" + n + "_mag"] * d).sum()


# ---- single tokens -----------------------------------------------------------------------------
STEP_CASES = [
    # D, E, H, Hkv, B, window, sinks, capacity, buckets
    (64, 64, 4, 2, 2, 7, 0, 7, None),
    (64, 64, 4, 4, 2, 7, 3, 10, B32C),
    (128, 128, 8, 1, 1, 20, 4, 31, B32C),
    (33, 17, 2, 1, 3, 5, 2, 9, B6),
    (80, 40, 3, 3, 2, 1, 0, 1, None),
    (256, 256, 2, 2, 1, 9, 1, 10, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("case", STEP_CASES, ids=lambda c: "-".join(str(len(v) if hasattr(v, "first") else v) for v in c))
def test_steps_one_by_one_are_the_attention_over_the_sequence(dt, case):
    D, E, H, Hkv, B, window, sinks, cap, buckets = case
    T = 40
    a = make(11, dt, D, E, H, Hkv, T, T, B, len(buckets) if buckets else 0)
    t = {n: dev(x, dt) for n, x in a.items()}
    ref = W.attention(a["q"], a["k"], a["v"], window, sinks, True, None, a.get("table"), buckets.first if buckets else None,
                      bool(buckets and buckets.bidirectional))
    kc, vc = L.jl_zeros((D, Hkv, cap, B), DT[dt], "cuda"), L.jl_zeros((E, Hkv, cap, B), DT[dt], "cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    xs = []
    for i in range(T):
        xs.append(L.windowed_attention_step(t["q"][:, :, i], t["k"][:, :, i], t["v"][:, :, i], kc, vc, lens, window=window, sinks=sinks,
                                            table=t.get("table"), buckets=buckets))
        lens += 1
    check({"x": torch.stack(xs, 2)}, ref, dt, ["x"], D, E, window + sinks)
    for c, src in ((kc, a["k"]), (vc, a["v"])):
        want = np.zeros(c.shape)
        for p in range(T):
            want[:, :, W.slot(p, sinks, cap)] = src[:, :, p]
        assert np.array_equal(host(c), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_a_prompt_then_steps(dt):
    """windowed_attention over a padded batch of prompts, its keys and values into the cache, then steps: as the whole sequences at once.
    A place without a sequence stays as it is."""
    D, H, Hkv, B, window, sinks, cap, S, T = 64, 4, 2, 4, 12, 2, 17, 50, 9
    a = make(12, dt, D, D, H, Hkv, S + T, S + T, B, len(B32C))
    prompt = [50, 3, 0, 31]
    t = {n: dev(x, dt) for n, x in a.items()}
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    kw = dict(window=window, sinks=sinks, table=t["table"], buckets=B32C)
    cut = lambda n: L.as_colmajor(t[n][:, :, :S])
    x = L.windowed_attention(cut("q"), cut("k"), cut("v"), lengths=lens, **kw)
    kc, vc = (L.from_numpy(np.full((D, Hkv, cap, B), 7.0), dtype=DT[dt]) for _ in range(2))
    L.windowed_cache_fill(kc, vc, cut("k"), cut("v"), lens, sinks=sinks)
    want = np.full((D, Hkv, cap, B), 7.0)
    for b in range(B):
        for p in range(prompt[b]):
            want[:, :, W.slot(p, sinks, cap), b] = a["k"][:, :, p, b]
    assert np.array_equal(host(kc), want)
    lens[3] = -1                                                    # nobody there any more
    for b in range(B):                                              # the tokens that follow a prompt
        for n in ("q", "k", "v"):
            if b != 3:
                a[n][:, :, prompt[b]:prompt[b] + T, b] = a[n][:, :, S:S + T, b]
    ref = W.attention(a["q"], a["k"], a["v"], window, sinks, True, None, a["table"], B32C.first, False)
    before = kc[..., 3].clone()
    for i in range(T):
        tok = lambda n: L.as_colmajor(t[n][:, :, S + i])
        y = host(L.windowed_attention_step(tok("q"), tok("k"), tok("v"), kc, vc, lens, **kw))
        lens[:3] += 1
        assert not y[..., 3].any()
        for b in range(3):
            l = prompt[b] + i
            lim = bound(dt, "x", ref["x_mag"][:, :, l, b], ref["zmax"], D, D, window + sinks)
            assert (np.abs(y[..., b] - ref["x"][:, :, l, b]) <= lim).all()
    assert torch.equal(before, kc[..., 3])
    for b in range(B):
        lim = bound(dt, "x", ref["x_mag"][:, :, :prompt[b], b], ref["zmax"], D, D, window + sinks)
        if b != 3:
            assert (np.abs(host(x)[:, :, :prompt[b], b] - ref["x"][:, :, :prompt[b], b]) <= lim).all()
        assert not host(x)[:, :, prompt[b]:, b].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks,length", [(1500, 5, 4000), (700, 0, 699), (2048, 64, 100000), (3, 1, 2 ** 31 - 1)])
def test_steps_over_long_windows(dt, window, sinks, length):
    """Windows that several blocks share, and positions up to the last that lengths can hold."""
    D, H, Hkv, B, cap = 64, 4, 2, 2, window + sinks + 13
    rng = np.random.default_rng(13)
    q, k, v = (rounded(rng.standard_normal((D, h, B)), dt) for h in (H, Hkv, Hkv))
    kc, vc = (rounded(rng.standard_normal((D, Hkv, cap, B)), dt) for _ in range(2))
    table = rounded(rng.standard_normal((H, len(B32C))), dt)
    lens = [length, length // 2]
    tk, tv = dev(kc, dt), dev(vc, dt)
    x = host(L.windowed_attention_step(dev(q, dt), dev(k, dt), dev(v, dt), tk, tv, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                       window=window, sinks=sinks, table=dev(table, dt), buckets=B32C))
    for b, n in enumerate(lens):
        kc[:, :, W.slot(n, sinks, cap), b], vc[:, :, W.slot(n, sinks, cap), b] = k[..., b], v[..., b]
        pos = list(range(max(0, n - window + 1), n + 1))
        pos = [p for p in range(min(sinks, pos[0]))] + pos
        at = [W.slot(p, sinks, cap) for p in pos]
        bk = [W.bucket(p - n, B32C.first, False) for p in pos]
        for h in range(H):
            kk, vv = kc[:, h // 2, at, b], vc[:, h // 2, at, b]
            z = q[:, h, b] @ kk / 8 + table[h, bk]
            p = np.exp(z - z.max())
            p /= p.sum()
            zmax = (np.abs(q[:, h, b]) @ np.abs(kk) / 8 + np.abs(table[h, bk])).max()
            assert (np.abs(x[:, h, b] - vv @ p) <= bound(dt, "x", np.abs(vv) @ p, zmax, D, D, len(pos))).all()
    assert np.array_equal(host(tk), kc) and np.array_equal(host(tv), vc)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_steps_in_a_graph_advance_with_lengths(dt):
    D, H, Hkv, B, window, sinks, cap, T = 64, 4, 2, 2, 9, 1, 10, 25
    a = make(14, dt, D, D, H, Hkv, T, T, B)
    t = {n: dev(x, dt) for n, x in a.items()}
    kc, vc = (L.jl_zeros((D, Hkv, cap, B), DT[dt], "cuda") for _ in range(2))
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    q, k, v = (L.as_colmajor(t[n][:, :, 0]).clone(memory_format=torch.preserve_format) for n in ("q", "k", "v"))
    L.windowed_attention_step(q, k, v, kc, vc, lens, window=window, sinks=sinks)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x = L.windowed_attention_step(q, k, v, kc, vc, lens, window=window, sinks=sinks)
        lens.add_(1)
    ref = W.attention(a["q"], a["k"], a["v"], window, sinks, True)
    lens.zero_()
    for i in range(T):
        for s, n in ((q, "q"), (k, "k"), (v, "v")):
            s.copy_(t[n][:, :, i])
        g.replay()
        lim = bound(dt, "x", ref["x_mag"][:, :, i], ref["zmax"], D, D, window + sinks)
        assert (np.abs(host(x) - ref["x"][:, :, i]) <= lim).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_a_step_does_not_read_slots_that_it_does_not_see(dt):
    D, H, Hkv, B, window, sinks, cap = 64, 2, 1, 1, 5, 2, 12
    rng = np.random.default_rng(15)
    q, k, v = (dev(rng.standard_normal((D, h, B)), dt) for h in (H, Hkv, Hkv))
    kc, vc = (rng.standard_normal((D, Hkv, cap, B)) for _ in range(2))
    lens = torch.tensor([6], dtype=torch.int32, device="cuda")
    outs = []
    for fill in (0.0, math.nan):
        for c in (kc, vc):
            for s in range(cap):
                if s not in (0, 1, 2, 3, 4, 5):
                    c[:, :, s] = fill
        outs.append(L.windowed_attention_step(q, k, v, dev(kc, dt), dev(vc, dt), lens, window=window, sinks=sinks))
    assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()


# ---- relative position bias ---------------------------------------------------------------------
BIAS_CASES = [(1, 1, 1, 1, 0, B6), (197, 197, 3, 2, 0, B32), (64, 130, 2, 1, 0, B32C), (130, 64, 2, 3, 17, B32), (1, 300, 4, 1, -20, B6),
              (300, 1, 4, 1, 299, B32C), (256, 64, 1, 5, 0, B128), (513, 70, 2, 1, 0, L.RelativeBuckets((0,), False)), (90, 100, 2, 4, 3, BD), (90, 100, 2, 1, -3, BDB)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("S,Lq,H,B,offset,buckets", BIAS_CASES)
def test_relative_position_bias_fwd_bwd(dt, S, Lq, H, B, offset, buckets):
    """The bias is exact; a gradient of n terms in fp32 is off by n u of the sum of magnitudes, and rounded once."""
    rng = np.random.default_rng(16)
    table, delta = rounded(rng.standard_normal((H, len(buckets))), dt), rounded(rng.standard_normal((S, Lq, H, B)), dt)
    bias, pb = L.rrule_relative_position_bias(dev(table, dt), buckets, S, Lq, offset=offset)
    assert np.array_equal(host(bias), W.relative_bias(table, buckets.first, buckets.bidirectional, S, Lq, offset))
    g, mag = W.relative_bias_grad(delta, H, len(buckets), buckets.first, buckets.bidirectional, offset)
    got = host(pb(dev(delta, dt)))
    lim = mag * U32 * S * Lq * B + np.abs(g) * (U16 if dt == "bf16" else U32) * 1.01 + 1e-35
    assert got.shape == g.shape and (np.abs(got - g) <= lim).all()
    assert torch.equal(pb(dev(delta, dt)), pb(dev(delta, dt)))


@pytest.mark.gpu
def test_relative_position_bias_of_nothing():
    table = dev(np.ones((2, len(B6))), "f32")
    bias, pb = L.rrule_relative_position_bias(table, B6, 0, 5)
    assert tuple(bias.shape) == (0, 5, 2, 1)
    assert not host(pb(L.jl_empty((0, 5, 2, 1), torch.float32, "cuda"))).any()
    x, pb = L.rrule_windowed_attention(*(L.jl_empty((8, 2, 3, 0), torch.float32, "cuda") for _ in range(3)), window=2, table=table, buckets=B6)
    assert tuple(x.shape) == (8, 2, 3, 0) and not host(pb(x)[3]).any()
    e = lambda n: L.jl_empty((8, 2, n, 1), torch.float32, "cuda")
    x, pb = L.rrule_windowed_attention(e(4), e(0), e(0), window=2)          # no keys: rows that see nothing
    assert not host(x).any() and not host(pb(x)[0]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B", [1, 3])
def test_the_bias_in_scaled_dot_product_attention_is_the_table_in_the_window(dt, B):
    """A learned bias through scaled_dot_product_attention and back into its table, and the same through the windowed operator with a
    window over everything: equal to the definition within the roundings of each (the first rounds bias, logits, weights and their
    gradients: 3 more)."""
    D, H, S = 64, 2, 72
    a = make(17, dt, D, D, H, H, S, S, B, len(B32))
    t = {n: dev(x, dt) for n, x in a.items()}
    got, ref = run_case(dt, D, D, H, H, S, S, B, 1000, 0, False, B32, a=a)
    bias, pb_bias = L.rrule_relative_position_bias(t["table"], B32, S, S)
    (x, _), pb = L.rrule_scaled_dot_product_attention(t["q"], t["k"], t["v"], bias=bias)
    dq, dk, dv, dbias = pb(t["dx"])
    assert tuple(dbias.shape) == tuple(bias.shape)
    dtable = pb_bias(dbias)
    for name, g in (("x", x), ("dq", dq), ("dk", dk), ("dv", dv), ("dtable", dtable)):
        lim = bound(dt, name, ref[name + "_mag"], ref["zmax"], D, D, S * S * B)
        if dt == "bf16":
            lim = lim + U16 * (3 + 2 * ref["zmax"]) * ref[name + "_mag"]
        assert (np.abs(host(g) - ref[name]) <= 2 * lim).all(), name


# ---- refusals ------------------------------------------------------------------------------------
def test_buckets():
    """One distance each below n / 2, then logarithmic up to max_distance; distances on a border belong to the bucket that starts there."""
    b = L.RelativeBuckets.make(32, 128, True)
    assert b.first == (0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91) and len(b) == 32
    for buckets in (b, B32C, B6, B128):
        n = len(buckets.first)
        e, top = n // 2, {32: 128, 6: 20, 128: 300}[len(buckets)]
        for rel in range(-400, 401):
            dist = abs(rel) if buckets.bidirectional else max(-rel, 0)
            j = dist if dist < e else min(n - 1, e + int(math.log(dist / e) / math.log(top / e) * (n - e) + 1e-9))
            assert buckets.bucket(rel) == j + (n if buckets.bidirectional and rel > 0 else 0) == W.bucket(rel, buckets.first, buckets.bidirectional)
    for bad in (lambda: L.RelativeBuckets.make(31, 128), lambda: L.RelativeBuckets.make(32, 8), lambda: L.RelativeBuckets.make(0, 8),
                lambda: L.RelativeBuckets.make(200, 1000), lambda: L.RelativeBuckets((1, 2)), lambda: L.RelativeBuckets((0, 5, 3)),
                lambda: L.RelativeBuckets(()), lambda: L.RelativeBuckets((0, 2 ** 31)), lambda: L.RelativeBuckets.make(66, 128, False)):
        with pytest.raises(L.ArgumentError):
            bad()


def test_arrays_off_the_device_are_refused():
    z = lambda *s: L.jl_zeros(s, torch.float32, "cpu")
    with pytest.raises(L.ArgumentError):
        L.windowed_attention(z(8, 2, 4, 1), z(8, 2, 4, 1), z(8, 2, 4, 1), window=2)
    with pytest.raises(L.ArgumentError):
        L.windowed_attention_step(z(8, 2, 1), z(8, 2, 1), z(8, 2, 1), z(8, 2, 4, 1), z(8, 2, 4, 1), torch.zeros(1, dtype=torch.int32), window=2)
    with pytest.raises(L.ArgumentError):
        L.windowed_cache_fill(z(8, 2, 4, 1), z(8, 2, 4, 1), z(8, 2, 4, 1), z(8, 2, 4, 1))
    with pytest.raises(L.ArgumentError):
        L.relative_position_bias(z(2, 12), B6, 4, 4)


def _dims(**kw):
    base = dict(head_dim=64, value_dim=64, heads=4, kv_heads=2, queries=10, keys=10, batch=1, window=4, sinks=0, causal=1)
    base.update(kw)
    return C.byref(_cabi.WindowDims(*(base[n] for n, _ in _cabi.WindowDims._fields_)))


def _buckets(first=(0, 1, 2), count=None):
    t = _cabi.RelBuckets(len(first) if count is None else count, 0)
    t.first[:len(first)] = first
    return C.byref(t)


def test_status_codes_of_the_windowed_entry_points():
    lib = _cabi.load()
    one = 256
    fwd = lambda dims, dt=0, x=one, table=None, buckets=None, lens=None, q=one: lib.lb2_window_attention_fwd(
        x, None, None, q, one, one, table, buckets, lens, 0.125, dims, dt, None)
    assert fwd(None) == _cabi.BAD_ARG
    assert fwd(_dims(), dt=5) == _cabi.UNSUPPORTED_DTYPE
    assert fwd(_dims(window=0)) == _cabi.BAD_ARG and fwd(_dims(sinks=-1)) == _cabi.BAD_ARG
    assert fwd(_dims(heads=3)) == _cabi.BAD_SHAPE and fwd(_dims(kv_heads=0)) == _cabi.BAD_SHAPE
    assert fwd(_dims(head_dim=257)) == _cabi.BAD_SHAPE and fwd(_dims(queries=-1)) == _cabi.BAD_SHAPE
    assert fwd(_dims(), x=None) == _cabi.BAD_ARG and fwd(_dims(), q=258) == _cabi.BAD_ALIGN and fwd(_dims(), lens=2) == _cabi.BAD_ALIGN
    assert fwd(_dims(), table=one) == _cabi.BAD_ARG and fwd(_dims(), buckets=_buckets()) == _cabi.BAD_ARG
    assert fwd(_dims(), table=one, buckets=_buckets(count=65)) == _cabi.BAD_ARG
    assert fwd(_dims(), table=one, buckets=_buckets((1, 2))) == _cabi.BAD_ARG and fwd(_dims(), table=one, buckets=_buckets((0, 3, 2))) == _cabi.BAD_ARG
    assert fwd(_dims(batch=0)) == _cabi.OK and fwd(_dims(queries=0)) == _cabi.OK and fwd(_dims(heads=0, kv_heads=0)) == _cabi.OK

    bwd = lambda dims, ws=one, n=1 << 20, dq=one, dtable=None, table=None, buckets=None: lib.lb2_window_attention_bwd(
        dq, one, one, dtable, one, one, None, one, one, one, one, table, buckets, None, 0.125, dims, 0, ws, n, None)
    need = lib.lb2_window_attention_bwd_workspace_bytes(_dims(), None, 0)
    assert need >= 40 * 4
    assert bwd(_dims(), n=need - 1) == _cabi.WORKSPACE_TOO_SMALL and bwd(_dims(), ws=None, n=0) == _cabi.WORKSPACE_TOO_SMALL
    assert bwd(_dims(), ws=264) == _cabi.BAD_ALIGN and bwd(_dims(), dq=None) == _cabi.BAD_ARG
    assert bwd(_dims(), table=one, buckets=_buckets()) == _cabi.BAD_ARG           # no place for the table's gradient
    assert bwd(_dims(heads=0, kv_heads=0)) == _cabi.OK
    assert lib.lb2_window_attention_bwd_workspace_bytes(None, None, 0) == 0

    step = lambda dims, lens=one, x=one, dt=0: lib.lb2_window_attention_step(x, one, one, one, one, one, None, None, lens, 0.125, dims, dt, None)
    assert step(_dims(window=11)) == _cabi.BAD_ARG and step(_dims(window=9, sinks=2)) == _cabi.BAD_ARG and step(_dims(sinks=10)) == _cabi.BAD_ARG
    assert step(_dims(), lens=None) == _cabi.BAD_ARG and step(_dims(), x=None) == _cabi.BAD_ARG and step(_dims(window=0)) == _cabi.BAD_ARG
    assert step(_dims(), dt=9) == _cabi.UNSUPPORTED_DTYPE and step(_dims(), x=257) == _cabi.BAD_ALIGN and step(_dims(batch=0)) == _cabi.OK
    fill = lambda dims, cap, kc=one: lib.lb2_window_cache_fill(kc, one, one, one, None, cap, dims, 0, None)
    assert fill(_dims(sinks=4), 4) == _cabi.BAD_ARG and fill(_dims(), 4, None) == _cabi.BAD_ARG and fill(_dims(keys=0), 4) == _cabi.OK

    assert lib.lb2_relpos_bias_fwd(one, one, None, 4, 4, 2, 0, 0, None) == _cabi.BAD_ARG
    assert lib.lb2_relpos_bias_fwd(None, one, _buckets(), 4, 4, 2, 0, 0, None) == _cabi.BAD_ARG
    assert lib.lb2_relpos_bias_fwd(one, one, _buckets(), -1, 4, 2, 0, 0, None) == _cabi.BAD_SHAPE
    assert lib.lb2_relpos_bias_fwd(one, one, _buckets(), 4, 4, 2, 1 << 40, 0, None) == _cabi.BAD_ARG
    assert lib.lb2_relpos_bias_fwd(one, one, _buckets(), 0, 4, 2, 0, 0, None) == _cabi.OK
    assert lib.lb2_relpos_bias_bwd(one, one, _buckets(), 4, 4, 2, 1, 0, 0, None, 0, None) == _cabi.WORKSPACE_TOO_SMALL
    assert lib.lb2_relpos_bias_bwd(None, one, _buckets(), 4, 4, 2, 1, 0, 0, one, 1 << 20, None) == _cabi.BAD_ARG


def test_caches_that_overlap_are_refused():
    z = lambda *s: L.jl_zeros(s, torch.float32, "cpu")
    both = torch.zeros(3 * 8 * 2 * 4)
    cache = lambda at: L.arrays.jl_reshape(both[at:at + 64], (8, 2, 4, 1))
    for a, b in ((0, 0), (0, 32), (63, 0), (32, 16)):
        with pytest.raises(L.ArgumentError, match="share memory"):
            L.windowed_attention_step(z(8, 2, 1), z(8, 2, 1), z(8, 2, 1), cache(a), cache(b), torch.zeros(1, dtype=torch.int32), window=2)
        with pytest.raises(L.ArgumentError, match="share memory"):
            L.windowed_cache_fill(cache(a), cache(b), z(8, 2, 4, 1), z(8, 2, 4, 1))
    with pytest.raises(L.ArgumentError, match="CUDA"):                             # side by side: refused for the device alone
        L.windowed_attention_step(z(8, 2, 1), z(8, 2, 1), z(8, 2, 1), cache(0), cache(64), torch.zeros(1, dtype=torch.int32), window=2)


@pytest.mark.gpu
def test_lengths_of_every_whole_type_and_a_scale_in_an_array():
    """Int64 lengths past 2^31 are not taken modulo 2^32, fractions are refused; a scale held in an array may change between calls."""
    a = make(31, "f32", 32, 32, 2, 1, 40, 40, 3)
    q, k, v = (dev(a[n], "f32") for n in "qkv")
    run = lambda lens, scale=None: host(L.windowed_attention(q, k, v, window=9, lengths=lens, scale=scale))
    lens = lambda n, t: torch.tensor(n, dtype=t, device="cuda")
    for t in (torch.int64, torch.int16, torch.int8, torch.uint8):
        assert np.array_equal(run(lens([40, 7, 0], t)), run(lens([40, 7, 0], torch.int32))), t
    assert np.array_equal(run(lens([2 ** 32, 2 ** 31, -2 ** 40], torch.int64)), run(lens([40, 40, 0], torch.int32)))
    for t in (torch.float32, torch.bool):
        with pytest.raises(L.ArgumentError):
            run(lens([1, 1, 0], t))
        with pytest.raises(L.ArgumentError):
            L.windowed_cache_fill(L.jl_zeros((32, 1, 9, 3), torch.float32, "cuda"), L.jl_zeros((32, 1, 9, 3), torch.float32, "cuda"), k, v, lens([1, 1, 0], t))
    scale = torch.tensor(4.0)
    first = run(None, scale)
    scale.fill_(2.0)
    assert np.array_equal(first, run(None, 4.0)) and np.array_equal(run(None, scale), run(None, 2.0))


@pytest.mark.gpu
def test_refusals_of_the_operators():
    z = lambda *s, t=torch.float32: L.jl_zeros(s, t, "cuda")
    q, k = z(64, 4, 6, 1), z(64, 2, 6, 1)
    ok = dict(window=3)
    for err, call in [
        (L.LuxLibB200Error, lambda: L.windowed_attention(q, k, k, window=0)),
        (L.LuxLibB200Error, lambda: L.windowed_attention(q, k, k, window=3, sinks=-1)),
        (AssertionError, lambda: L.windowed_attention(q, z(64, 3, 6, 1), z(64, 3, 6, 1), **ok)),
        (AssertionError, lambda: L.windowed_attention(q, z(32, 2, 6, 1), k, **ok)),
        (AssertionError, lambda: L.windowed_attention(q, k, z(64, 2, 5, 1), **ok)),
        (L.DimensionMismatch, lambda: L.windowed_attention(q, z(64, 2, 6, 2), z(64, 2, 6, 2), **ok)),
        (L.DimensionMismatch, lambda: L.windowed_attention(q, k, k, lengths=torch.zeros(2, dtype=torch.int32, device="cuda"), **ok)),
        (L.DimensionMismatch, lambda: L.windowed_attention(q, k, k, table=z(4, 5), buckets=B6, **ok)),
        (L.ArgumentError, lambda: L.windowed_attention(q, k, k, table=z(4, 12), **ok)),
        (L.ArgumentError, lambda: L.windowed_attention(q, k, k, lengths=torch.zeros(1, dtype=torch.int32), **ok)),
        (L.DimensionMismatch, lambda: L.windowed_attention(z(257, 4, 6, 1), z(257, 2, 6, 1), k, **ok)),
        (L.LuxLibB200Error, lambda: L.windowed_attention(q.double(), k.double(), k.double(), **ok)),
        (L.DimensionMismatch, lambda: L.rrule_windowed_attention(q, k, k, **ok)[1](z(64, 4, 5, 1))),
        (L.DimensionMismatch, lambda: L.rrule_relative_position_bias(z(4, 12), B6, 3, 3)[1](z(3, 3, 2, 1))),
    ]:
        with pytest.raises(err):
            call()
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    tq, tk, kc = z(64, 4, 1), z(64, 2, 1), z(64, 2, 8, 1)
    for err, call in [
        (L.LuxLibB200Error, lambda: L.windowed_attention_step(tq, tk, tk, kc, kc.clone(), lens, window=9)),
        (L.LuxLibB200Error, lambda: L.windowed_attention_step(tq, tk, tk, kc, kc.clone(), lens, window=6, sinks=3)),
        (L.ArgumentError, lambda: L.windowed_attention_step(tq, tk, tk, kc, kc.bfloat16(), lens, window=4)),
        (L.ArgumentError, lambda: L.windowed_attention_step(tq, tk, tk, kc, kc.clone(), lens.long(), window=4)),
        (L.ArgumentError, lambda: L.windowed_attention_step(tq, tk, tk, kc[:, :, ::2], kc[:, :, 1::2], lens, window=4)),
        (L.ArgumentError, lambda: L.windowed_attention_step(tq, tk, tk, kc, kc, lens, window=4)),
        (L.ArgumentError, lambda: L.windowed_cache_fill(kc, kc, k, k)),
        (L.DimensionMismatch, lambda: L.windowed_attention_step(tq, tk, tk, kc, z(64, 2, 9, 1), lens, window=4)),
        (L.DimensionMismatch, lambda: L.windowed_attention_step(tq, tk, tk, z(64, 2, 8, 2), z(64, 2, 8, 2), lens, window=4)),
        (L.LuxLibB200Error, lambda: L.windowed_cache_fill(kc, kc.clone(), k, k, sinks=8)),
        (L.DimensionMismatch, lambda: L.windowed_cache_fill(z(64, 2, 8, 2), z(64, 2, 8, 2), k, k)),
    ]:
        with pytest.raises(err):
            call()
