"""Operators that programs name as custom calls, and the moves inside a paged cache, against their definitions in 64 bits.

Tolerances count roundings. u is half a step of the type, e = 2^-24. A result is rounded once (u |out|). A score is a sum of D products
(at most (D + 4) e of the sum of its absolute terms, `top`), goes through exp2 with an argument whose own rounding is at most
4 e top and whose function is good to 2^-22: a weight is off by d = (D + 8) e top + 2^-22 relative, the normaliser by as much, and
a sum over n positions by n e: 2 d + 2 n e of sum_j w_j |v_j| (`mag`). The tensor-core kernels of 16-bit data round the weights to 16
bits for the second product: u mag more, or u^2 mag where they go in two pieces."""
import numpy as np
import pytest

import b200
from b200.pages import PagedCache
from b200.shlo.builder import Builder
from oracle import interp, operators

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
E = 2.0 ** -24


def rounded(a, dt):
    a = np.asarray(a, np.float32)
    return a if dt == "f32" else a.astype(np.float16).astype(np.float32) if dt == "f16" else interp.round_bf16(a)


def put(client, a, dt):
    a = np.asarray(a)
    if dt in U:
        a = a.astype(np.float16 if dt == "f16" else np.float32)
    return client.buffer_from_host(a, dtype="bf16" if dt == "bf16" else None)


def run(client, build, arrays, dts):
    """Arguments of `build(builder, *vals)` from arrays; the results as NumPy arrays, from two calls that have to agree bit for bit."""
    b = Builder()
    outs = build(b, *[b.arg(np.shape(a), dt) for a, dt in zip(arrays, dts)])
    exe = client.compile(b.module(outs if isinstance(outs, list) else [outs]))
    bufs = [put(client, a, dt) for a, dt in zip(arrays, dts)]
    first, second = ([np.asarray(o.to_numpy()) for o in exe.execute(bufs)] for _ in range(2))
    for x, y in zip(first, second):
        np.testing.assert_array_equal(x, y)
    return first


def attention_tolerance(want, mag, top, n, D, dt, weights):
    u = U[dt]
    d = (D + 8) * E * top + 2.0 ** -22
    return u * np.abs(want) + mag * (2 * d + 2 * n * E + weights) + (2.0 ** -25 if dt == "f16" else 0.0)


def paged_case(rng, lens, H, KH, D, S, dt, new, layers=1, spare=2):
    B = len(lens)
    width = max(1, max(-(-n // S) for n in lens))
    pages = sum(-(-n // S) for n in lens) + spare
    order, table, at = rng.permutation(pages), np.full((B, width), -1, np.int32), 0
    for b, n in enumerate(lens):
        m = -(-n // S)
        table[b, :m] = order[at:at + m]
        at += m
    q = rounded(rng.standard_normal((B, H, D)), dt)
    cache = rounded(rng.standard_normal((layers, 2, pages, S, KH, D)), dt)
    fresh = rounded(rng.standard_normal((2, B, KH, D)), dt) if new else None
    return q, cache, table, np.asarray(lens, np.int32), fresh


def check_paged(client, q, cache, table, lengths, fresh, dt, **kw):
    arrays, dts = [q, cache, table, lengths], [dt, dt, "i32", "i32"]
    if fresh is not None:
        arrays.append(fresh)
        dts.append(dt)
    got = run(client, lambda b, q, c, t, n, new=None: b.paged_attention(q, c, t, n, new=new, **kw), arrays, dts)[0]
    want, mag, top = operators.paged_attention(q, cache, table, lengths, fresh, bounds=True, **kw)
    tol = attention_tolerance(want, mag, top, int(max(lengths.max(initial=0), 0)) + 1, q.shape[-1], dt, 0.0 if dt == "f32" else U[dt])
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (float(np.abs(got - want)[bad].max()), np.argwhere(bad)[:5].tolist(), int(bad.sum()))
    return got


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,KH,D,S", [(8, 1, 256, 16), (4, 4, 64, 5), (6, 2, 128, 64), (7, 1, 72, 1), (32, 2, 96, 24), (3, 3, 8, 7), (24, 1, 192, 32), (2, 1, 248, 3)])
@pytest.mark.parametrize("new", [False, True])
def test_paged_attention_heads_and_pages(client, dt, H, KH, D, S, new):
    rng = np.random.default_rng(H * D + S + new)
    check_paged(client, *paged_case(rng, [0, 1, 2, 15, 16, 17, 100, 33], H, KH, D, S, dt, new), dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (2, 1), (16, 4), (100, 0), (130, 20), (1000, 5)])
@pytest.mark.parametrize("new", [False, True])
def test_paged_attention_window_and_sinks(client, dt, window, sinks, new):
    rng = np.random.default_rng(window)
    check_paged(client, *paged_case(rng, [0, 1, 3, 16, 99, 131, 260, 700], 4, 2, 64, 8, dt, new), dt, window=window, sinks=sinks)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", [[127], [128], [129], [1023, 1], [3001, 0, 64, 2000], [40, 5000] + [17] * 37])
def test_paged_attention_split_over_the_length(client, dt, lens):
    rng = np.random.default_rng(sum(lens))
    check_paged(client, *paged_case(rng, lens, 4, 1, 64, 16, dt, True), dt)


def test_paged_attention_many_sequences(client):
    rng = np.random.default_rng(5)
    check_paged(client, *paged_case(rng, rng.integers(0, 40, 1500).tolist(), 2, 1, 8, 4, "bf16", True), "bf16")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[0] * 5, [1] * 300, [127, 0, 126, 1] * 9, [128, 0, 5] * 40, [3] * 700 + [400]])
def test_paged_attention_short_sequences(client, dt, lens):
    """Sequences that are one part each, and some beside a longer one; the token beside the cache makes 128 of 127."""
    for new in (False, True):
        rng = np.random.default_rng(len(lens) + new)
        check_paged(client, *paged_case(rng, lens, 4, 2, 64, 16, dt, new), dt)


def test_paged_attention_layer_scale_and_shared_pages(client):
    rng = np.random.default_rng(11)
    q, cache, table, lengths, fresh = paged_case(rng, [30, 45, 45], 4, 2, 64, 16, "bf16", True, layers=3)
    table[2, :2] = table[1, :2]                                    # a fork: two sequences read the same pages
    for layer in range(3):
        check_paged(client, q, cache, table, lengths, fresh, "bf16", layer=layer, scale=0.3)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_paged_attention_reads_nothing_that_is_hidden(client, dt):
    """NaN and infinities in slots behind a sequence, in pages of others, behind the window; lengths and pages out of range."""
    rng = np.random.default_rng(2)
    S, lens = 8, [21, 5, 0, 40]
    q, cache, table, lengths, fresh = paged_case(rng, lens, 4, 2, 64, S, dt, True)
    seen = np.zeros(cache.shape[2:4], bool)
    for b, n in enumerate(lens):
        for j in operators.visible(n, n, 12, 2):
            seen[table[b, j // S], j % S] = True
    cache[:, 0][:, ~seen] = np.nan
    cache[:, 1][:, ~seen] = np.inf
    check_paged(client, q, cache, table, lengths, fresh, dt, window=12, sinks=2)
    # lengths below zero and above the table's room
    check_paged(client, q, np.nan_to_num(cache, posinf=1.0), np.abs(table), np.array([-3, 1000, 2**31 - 1, -2**31], np.int32), fresh, dt)


@pytest.mark.parametrize("new", [False, True])
def test_paged_attention_leaves_out_pages_that_are_not_there(client, new):
    rng = np.random.default_rng(4)
    q, cache, table, lengths, fresh = paged_case(rng, [40, 40, 40], 4, 2, 64, 8, "bf16", new)
    table[0, 1], table[1, 3], table[2, :] = -7, cache.shape[2], 2**31 - 1
    check_paged(client, q, cache, table, lengths, fresh, "bf16")


def test_paged_attention_scores_at_the_edge(client):
    """Large scores, one position that takes all of the weight, infinities in a visible key (as the definition gives them)."""
    rng = np.random.default_rng(8)
    q, cache, table, lengths, fresh = paged_case(rng, [50, 50], 2, 1, 64, 16, "f32", False)
    check_paged(client, q * 30, cache, table, lengths, fresh, "f32")
    cache[0, 0, table[0, 0], 3, 0, :] = np.where(q[0, 0] > 0, -3e38, 3e38)          # a score of minus infinity: no weight
    got = run(client, lambda b, q, c, t, n: b.paged_attention(q, c, t, n), [q[:1, :1], cache, table[:1], lengths[:1]], ["f32", "f32", "i32", "i32"])[0]
    with np.errstate(all="ignore"):
        want = operators.paged_attention(q[:1, :1], cache, table[:1], lengths[:1])
    np.testing.assert_allclose(got, want, rtol=1e-4, atol=1e-5)
    cache[0, 0, table[0, 0], 3, 0, :] = np.nan
    got = run(client, lambda b, q, c, t, n: b.paged_attention(q, c, t, n), [q, cache, table, lengths], ["f32", "f32", "i32", "i32"])[0]
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_paged_attention_many_small_weights_beside_a_large_one(client, dt):
    """60000 positions of e^-17 each, which are 2.5e-3 of the result together, beside one whose value is zero."""
    n, S, D = 60001, 64, 64
    pages = -(-n // S)
    q, cache = np.zeros((1, 1, D)), np.zeros((1, 2, pages, S, 1, D))
    q[..., 0], cache[0, 0, 5, 3, 0, 0] = 17.0, 1.0
    cache[0, 1] = 1.0
    cache[0, 1, 5, 3] = 0.0
    table = np.arange(pages, dtype=np.int32)[None]
    check_paged(client, q, cache, table, np.array([n], np.int32), None, dt, scale=1.0)


def test_paged_attention_of_nothing(client):
    for B, W in ((0, 3), (2, 0)):
        q, cache = np.ones((B, 2, 8), np.float32), np.ones((1, 2, 0 if W == 0 else 4, 2, 1, 8), np.float32)
        args = [q, cache, np.zeros((B, W), np.int32), np.full(B, 4, np.int32)]
        got = run(client, lambda b, *a: b.paged_attention(*a), args, ["f32", "f32", "i32", "i32"])[0]
        assert got.shape == q.shape and (got == 0).all()


# ---- prompts ------------------------------------------------------------------------------------------
def check_prompt(client, q, k, v, lengths, dt, **kw):
    arrays, dts = [q, k, v] + ([lengths] if lengths is not None else []), [dt] * 3 + ["i32"]
    got = run(client, lambda b, q, k, v, n=None: b.window_attention(q, k, v, n, **kw), arrays, dts)[0]
    known = [np.where(np.isfinite(t), t, 0.0) for t in (q, k, v)]
    want, mag, top = operators.window_attention(*known, lengths, bounds=True, **kw)
    tol = attention_tolerance(want, mag, top, q.shape[1], q.shape[-1], dt, 0.0 if dt == "f32" else U[dt])
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (float(np.nanmax(np.abs(got - want)[bad])), np.argwhere(bad)[:5].tolist(), int(bad.sum()))


def prompt_case(rng, B, T, H, KH, D, dt):
    return [rounded(rng.standard_normal(s), dt) for s in ((B, T, H, D), (B, T, KH, D), (B, T, KH, D))]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,KH,D", [(2, 1, 256), (3, 3, 64), (4, 2, 128), (2, 1, 72), (1, 1, 192), (2, 2, 8), (2, 1, 248)])
@pytest.mark.parametrize("T", [1, 77, 130])
def test_window_attention_heads_and_lengths(client, dt, H, KH, D, T):
    rng = np.random.default_rng(H * D + T)
    check_prompt(client, *prompt_case(rng, 1, T, H, KH, D, dt), None, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (5, 0), (64, 1), (100, 4), (129, 130), (300, 16), (1000, 0)])
def test_window_attention_windows(client, dt, window, sinks):
    rng = np.random.default_rng(window + sinks)
    check_prompt(client, *prompt_case(rng, 1, 413, 2, 1, 64, dt), None, dt, window=window, sinks=sinks)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_window_attention_long_rows_of_tiles(client, dt, D):
    rng = np.random.default_rng(D)
    check_prompt(client, *prompt_case(rng, 1, 1100, 1, 1, D, dt), None, dt)
    check_prompt(client, *prompt_case(rng, 1, 1100, 1, 1, D, dt), None, dt, window=200, sinks=3)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_window_attention_padded_batch(client, dt):
    rng = np.random.default_rng(9)
    lengths = np.array([150, 0, 1, 64, 129, -4, 2000], np.int32)
    q, k, v = prompt_case(rng, 7, 150, 2, 1, 64, dt)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), 150)
        q[b, n:], k[b, n:], v[b, n:] = np.nan, np.inf, np.nan          # nobody reads what stands behind a sequence
    check_prompt(client, q, k, v, lengths, dt, window=70, sinks=2, scale=0.2)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,H,KH,D,window,sinks", [(1, 2, 1, 64, 0, 0), (1, 2, 1, 64, 40, 3), (1, 1, 1, 256, 150, 20), (4, 32, 8, 64, 40, 3), (4, 32, 32, 128, 0, 0), (5, 32, 32, 64, 130, 129)])
def test_window_attention_of_values_that_are_no_numbers(client, dt, B, H, KH, D, window, sinks):
    """Infinities and NaN in keys and values reach the rows that see them and no other, in all forms of the kernels (one tile of queries a
    block, two of one head, two heads)."""
    T = 300
    rng = np.random.default_rng(B * D + window)
    q, k, v = prompt_case(rng, B, T, H, KH, D, dt)
    lengths = np.array([300, 299, 131, 140, 0], np.int32)[:B]
    v[0, 130], v[:, 250, :, 3], v[:, 255], k[:, 298] = np.inf, np.nan, -np.inf, np.nan
    args, dts = [q, k, v, lengths], [dt] * 3 + ["i32"]
    got = run(client, lambda b, *a: b.window_attention(*a, window=window, sinks=sinks), args, dts)[0]
    kw = dict(lengths=lengths, window=window, sinks=sinks)
    heads = [0, 1, H - 1]
    for h in sorted(set(x for x in heads if x < H)):
        g = h // (H // KH)
        one = [q[:, :, h:h + 1], k[:, :, g:g + 1], v[:, :, g:g + 1]]
        with np.errstate(all="ignore"):
            raw = operators.window_attention(*one, **kw)
            want, mag, top = operators.window_attention(*[np.where(np.isfinite(t), t, 0.0) for t in one], bounds=True, **kw)
        fine = np.isfinite(raw)
        np.testing.assert_array_equal(np.isfinite(got[:, :, h:h + 1]), fine)
        tol = attention_tolerance(want, mag, top, T, D, dt, 0.0 if dt == "f32" else U[dt])
        assert (np.abs(got[:, :, h:h + 1] - want)[fine] <= tol[fine]).all()


# ---- log probabilities ---------------------------------------------------------------------------------
def check_probs(client, x, tokens, top, dt, cotangents=None):
    R, V = x.shape
    arrays, dts = [x, np.asarray(tokens, np.int32)], [dt, "i32"]
    if cotangents is not None:
        arrays += cotangents
        dts += ["f32"] * 3

    def build(b, x, t, *g):
        outs = b.token_log_probs(x, t, top=top)
        if g:
            total = b.add(b.add(b.mul(outs[0], g[0]), b.mul(outs[1], g[1])), b.mul(outs[2], g[2]))
            outs = outs + b.grad(b.reduce_sum(total, (0,)), [x])
        return outs
    got = run(client, build, arrays, dts)
    want = operators.token_log_probs(x, tokens, top)
    # m + log s: exponentials good to 2^-21 (argument rounding and function), sums of V terms in pairs and threads' runs (V / 256 + 16 e),
    # and the result's own rounding; the entropy's terms p (x - m) carry the same relative errors times the span of the logits that count
    finite = np.where(np.isfinite(x), x, 0.0)
    span = float(np.abs(finite).max()) * 2 + 1
    rel = 2.0 ** -21 + (V / 256 + 16) * E
    for g, w, scale in zip(got[:3], want[:3], (1.0, span, 1.0)):
        tol = scale * rel * 2 + 4 * E * (np.abs(finite).max() + np.abs(np.where(np.isfinite(w), w, 0.0)))
        same = (g == w) | (np.isnan(g) & np.isnan(w))
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(g - w) <= tol)).all(), (g, w, tol)
    if top:
        np.testing.assert_array_equal(got[4], want[4])
        with np.errstate(invalid="ignore"):
            close = np.abs(got[3] - want[3]) <= 2 * rel + 8 * E * (np.abs(finite).max() + 20)
        assert (close | (got[3] == want[3]) | (np.isnan(got[3]) & np.isnan(want[3]))).all()
    if cotangents is not None:
        dx, ref = got[-1], operators.token_log_probs_grad(x, tokens, *cotangents)
        gl, gh, gn = (np.abs(c)[:, None] for c in cotangents)
        p = np.exp(np.asarray(x, np.float64) - want[2][:, None])
        off = rel * 3 + 8 * E * (np.abs(finite).max() + 20)                 # of a probability: that of its exponent
        size = p * (gl + gn + gh * (span + 20))
        assert (np.abs(dx - ref) <= U[dt] * np.abs(ref) + size * off * 2 + 4 * E * (np.abs(ref) + size) + (2.0 ** -25 if dt == "f16" else 1e-40)).all()
    return got


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 7), (5, 255), (2, 1000), (9, 1031), (4, 30522), (1, 256000), (300, 512)])
def test_token_log_probs(client, dt, R, V):
    rng = np.random.default_rng(V + R)
    x = rounded(rng.standard_normal((R, V)) * 4, dt)
    tokens = rng.integers(0, V, R)
    tokens[::3] = -1
    tokens[1::5] = V
    check_probs(client, x, tokens, min(V, 5), dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 2, 31, 64, 128])
@pytest.mark.parametrize("V", [128, 5003, 66000])
def test_alternatives_with_equal_logits(client, dt, top, V):
    """Few distinct values: equal ones by their number; rows in order and against it; a row of one value."""
    rng = np.random.default_rng(top)
    rows = [rng.integers(0, 3, V), np.arange(V) // 7, -np.arange(V) // 5, np.zeros(V), rng.integers(0, 50, V) - 0.0, np.where(np.arange(V) % 97, -0.0, 0.0)]
    check_probs(client, rounded(np.stack(rows) / 4.0, dt), np.arange(6), top, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_token_log_probs_of_masked_vocabularies(client, dt):
    """Minus infinity, the type's lowest value, plus infinity, NaN, rows that leave one token or none."""
    rng = np.random.default_rng(1)
    V, low = 3001, {"f32": -3.4028235e38, "bf16": -3.3895314e38, "f16": -65504.0}[dt]
    x = rounded(rng.standard_normal((9, V)), dt)
    x[0, rng.random(V) < 0.9] = -np.inf
    x[1, rng.random(V) < 0.9] = low
    x[2] = -np.inf
    x[2, 1234] = 2.0
    x[3] = low
    x[4] = -np.inf
    x[5, 17] = np.inf
    x[6, 2900] = np.nan
    x[7, :10] = np.nan
    x[8, 1:] = low
    tokens = np.array([int(np.argmax(x[0])), 3, 1234, 5, 7, 17, 3, 2, 0])
    with np.errstate(invalid="ignore"):
        got = check_probs_special(client, x, tokens, 20, dt)
    assert got[0][2] == 0.0 and got[1][2] == 0.0
    assert np.isnan(got[0][[4, 5, 6, 7]]).all()


def check_probs_special(client, x, tokens, top, dt):
    got = run(client, lambda b, x, t: b.token_log_probs(x, t, top=top), [x, np.asarray(tokens, np.int32)], [dt, "i32"])
    want = operators.token_log_probs(x, tokens, top)
    np.testing.assert_array_equal(got[4], want[4])
    for g, w in zip(got[:4], want[:4]):
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        ok = ~np.isnan(w)
        np.testing.assert_allclose(g[ok], w[ok], rtol=1e-5, atol=2e-5)
    return got


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,V", [(1, 1), (7, 65), (5, 1000), (3, 30522), (2, 70001), (64, 2048)])
def test_gradient_of_token_log_probs(client, dt, R, V):
    rng = np.random.default_rng(V)
    x = rounded(rng.standard_normal((R, V)) * 3, dt)
    tokens = rng.integers(0, V, R)
    tokens[::4] = -100
    g = [rng.standard_normal(R).astype(np.float32) for _ in range(3)]
    check_probs(client, x, tokens, 0, dt, g)


@pytest.mark.parametrize("dt,R,V", [("f32", 299, 4097), ("f32", 300, 8190), ("f32", 296, 32760), ("f32", 296, 32761), ("bf16", 297, 20001), ("f16", 450, 8192)])
def test_loss_and_gradient_by_one_reading(client, dt, R, V):
    rng = np.random.default_rng(V)
    x = rounded(rng.standard_normal((R, V)) * 3, dt)
    x[5, ::3] = -np.inf
    x[6] = -np.inf
    x[6, V - 1] = 1.0
    x[7] = np.float32(-3e38) if dt == "f32" else x[7]
    tokens = rng.integers(0, V, R)
    tokens[::4], tokens[5], tokens[6] = -100, 1, V - 1
    g = [rng.standard_normal(R).astype(np.float32) for _ in range(3)]
    # (a row of the lowest value has no span: its probabilities are even, and tested as such)
    keep = np.arange(R) != 7
    got = run(client, lambda b, x, t, *g: (lambda o: o + b.grad(b.reduce_sum(b.add(b.add(b.mul(o[0], g[0]), b.mul(o[1], g[1])), b.mul(o[2], g[2])), (0,)), [x]))(
        b.token_log_probs(x, t)), [x, tokens.astype(np.int32), *g], [dt, "i32", "f32", "f32", "f32"])
    if dt == "f32":
        np.testing.assert_allclose(got[1][7], np.log(V), rtol=1e-6)
        p7 = g[2][7] - (g[0][7] if tokens[7] >= 0 else 0.0)
        np.testing.assert_allclose(np.delete(got[3][7], max(tokens[7], 0)), p7 / V, rtol=1e-4, atol=abs(g[1][7]) * 1e-5 / V + 1e-30)
    check_probs(client, x[keep], tokens[keep], 0, dt, [c[keep] for c in g])


def test_gradient_where_the_vocabulary_is_masked(client):
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((4, 999)) * 2).astype(np.float32)
    x[:, ::2] = -np.inf
    tokens = np.array([1, 3, 5, -1])
    g = [rng.standard_normal(4).astype(np.float32) for _ in range(3)]
    got = check_probs(client, x, tokens, 0, "f32", g)
    assert (got[-1][:, ::2] == 0).all()


def test_log_probs_of_no_rows(client):
    got = run(client, lambda b, x, t: b.token_log_probs(x, t, top=2), [np.zeros((0, 10), np.float32), np.zeros(0, np.int32)], ["f32", "i32"])
    assert [g.shape for g in got] == [(0,)] * 3 + [(0, 2)] * 2


# ---- moves inside a cache ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("L,P,S,KH,D,n", [(1, 3, 4, 1, 8, 1), (2, 10, 16, 2, 64, 50), (18, 6, 16, 1, 256, 3), (3, 200, 24, 3, 72, 4000), (1, 5000, 1, 1, 8, 2500)])
def test_write_pages(client, dt, L, P, S, KH, D, n):
    rng = np.random.default_rng(n)
    cache, rows = rounded(rng.standard_normal((L, 2, P, S, KH, D)), dt), rounded(rng.standard_normal((L, 2, n, KH, D)), dt)
    slots = rng.permutation(P * S)[:n].astype(np.int32)
    slots[rng.random(n) < 0.2] = -1
    buf, src = put(client, cache, dt), put(client, rows, dt)
    client.write_pages(buf, src, slots)
    np.testing.assert_array_equal(buf.to_numpy(), operators.write_pages(cache, rows, slots))
    np.testing.assert_array_equal(src.to_numpy(), rows)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("L,P,S,KH,D,n", [(1, 4, 2, 1, 8, 2), (5, 60, 16, 2, 64, 30), (2, 3000, 3, 1, 24, 1400), (1, 40, 64, 4, 128, 20)])
def test_copy_pages(client, dt, L, P, S, KH, D, n):
    rng = np.random.default_rng(n)
    cache = rounded(rng.standard_normal((L, 2, P, S, KH, D)), dt)
    # any sources, distinct destinations: chains, exchanges, pages onto themselves, one source for many
    pairs = np.stack([rng.integers(0, P, n), rng.permutation(P)[:n]], 1).astype(np.int32)
    buf = put(client, cache, dt)
    client.copy_pages(buf, pairs)
    np.testing.assert_array_equal(buf.to_numpy(), operators.copy_pages(cache, pairs))


@pytest.mark.parametrize("pairs", [[(0, 1), (1, 0)], [(i + 1, i) for i in range(999)], [(i, i + 1) for i in range(999)], [(i, (i + 1) % 1000) for i in range(1000)], [(5, 5)], []])
def test_copy_pages_chains(client, pairs):
    cache = np.arange(1000 * 16, dtype=np.float32).reshape(1, 2, 1000, 1, 1, 8)
    buf = put(client, cache, "f32")
    client.copy_pages(buf, pairs)
    np.testing.assert_array_equal(buf.to_numpy(), operators.copy_pages(cache, pairs))


def test_moves_refuse(client):
    import b200
    cache = put(client, np.zeros((2, 2, 4, 2, 1, 8)), "bf16")
    rows = put(client, np.zeros((2, 2, 3, 1, 8)), "bf16")

    def refuse(why, call):
        with pytest.raises(b200.B200Error) as e:
            call()
        assert e.value.code == b200.INVALID_ARGUMENT and why in str(e.value), str(e.value)
    refuse("two rows for one slot", lambda: client.write_pages(cache, rows, [1, 2, 1]))
    refuse("behind the cache", lambda: client.write_pages(cache, rows, [1, 2, 8]))
    refuse("rows have to be", lambda: client.write_pages(cache, rows, [1, 2]))
    refuse("rows have to be", lambda: client.write_pages(cache, put(client, np.zeros((2, 2, 3, 1, 8)), "f16"), [1, 2, 3]))
    refuse("rows have to be", lambda: client.write_pages(cache, cache, [1, 2, 3, 4]))
    refuse("two pairs", lambda: client.copy_pages(cache, [(0, 1), (2, 1)]))
    refuse("not in the cache", lambda: client.copy_pages(cache, [(0, 4)]))
    refuse("not in the cache", lambda: client.copy_pages(cache, [(-1, 0)]))
    refuse("a cache has to be", lambda: client.copy_pages(rows, [(0, 1)]))
    refuse("f32, bf16 or f16", lambda: client.copy_pages(client.buffer_from_host(np.zeros((2, 2, 4, 2, 1, 8), np.int32)), [(0, 1)]))
    refuse("multiple of 16 bytes", lambda: client.copy_pages(put(client, np.zeros((2, 2, 4, 2, 1, 4)), "bf16"), [(0, 1)]))
    client.write_pages(cache, rows, [-1, -1, -1])
    client.write_pages(cache, put(client, np.zeros((2, 2, 0, 1, 8)), "bf16"), [])
    gone = put(client, np.zeros((2, 2, 4, 2, 1, 8)), "bf16")
    gone.delete()
    refuse("deleted", lambda: client.copy_pages(gone, [(0, 1)]))


def test_moves_keep_their_place_among_executions_and_reads(client):
    """A read that was started sees the cache as it was, an execution behind the change sees it as it is."""
    rng = np.random.default_rng(0)
    shape = (1, 2, 64, 16, 8, 128)
    old = rng.standard_normal(shape).astype(np.float32)
    b = Builder()
    c = b.arg(shape, "f32")
    twice = client.compile(b.module([b.mul(c, b.full(shape, 2.0, "f32"))]))
    for _ in range(5):
        buf, rows = put(client, old, "f32"), put(client, np.ones((1, 2, 16, 8, 128)), "f32")
        before = twice.execute([buf])[0]
        host = np.empty(shape, np.float32)
        event = buf.to_host_async(host)
        client.write_pages(buf, rows, np.arange(16))
        client.copy_pages(buf, [(0, 63)])
        behind = twice.execute([buf])[0]
        event.wait()
        new = operators.copy_pages(operators.write_pages(old, np.ones((1, 2, 16, 8, 128)), np.arange(16)), [(0, 63)])
        np.testing.assert_array_equal(host, old)
        np.testing.assert_array_equal(buf.to_numpy(), new)
        np.testing.assert_array_equal(before.to_numpy(), 2 * old)
        np.testing.assert_array_equal(behind.to_numpy(), 2 * new)


def test_moves_keep_what_an_execution_reported(client):
    """Rows of an execution that gave up on a wait (test hook: a barrier nothing arrives at) make the cache's contents invalid, and rows of
    a good one written behind them do not hide it."""
    shape = (1, 2, 4, 1, 256)
    cache = client.buffer_from_host(np.zeros((1, 2, 2, 4, 1, 256), np.float32))
    b = Builder()
    x = b.arg((256, 256), "f32")
    exe = client.compile(b.module([b.reshape(b.slice(b.dot_general(x, x, ([1], [0])), (0, 0), (8, 256)), shape)]))
    arg = client.buffer_from_host(np.eye(256, dtype=np.float32))
    client.synchronize()
    client.debug_arm_wait_expiry(1000)
    bad, good = (exe.execute([arg])[0] for _ in range(2))
    client.write_pages(cache, bad, [0, 1, 2, 3])
    client.write_pages(cache, good, [4, 5, 6, 7])
    with pytest.raises(b200.B200Error, match="bounded"):
        cache.to_numpy()
    with pytest.raises(b200.B200Error):
        client.synchronize()
    other = client.buffer_from_host(np.zeros((1, 2, 2, 4, 1, 256), np.float32))
    client.write_pages(other, good, [4, 5, 6, 7])
    assert np.array_equal(other.to_numpy()[0, :, 1, :, 0], np.eye(256, dtype=np.float32)[:8].reshape(2, 4, 256))


def test_cache_of_more_than_32_bits(client):
    """The last pages of a cache with 2^31 elements and more in each plane."""
    KH, S, D, P = 8, 64, 256, 16400
    assert P * S * KH * D > 2**31
    cache = PagedCache(client, 1, P, S, KH, D)
    rng = np.random.default_rng(0)
    n = 70
    rows = rounded(rng.standard_normal((1, 2, n, KH, D)), "bf16")
    table = np.array([[P - 1, P - 2]], np.int32)
    at = np.arange(n)
    client.write_pages(cache.buffer, put(client, rows, "bf16"), table[0][at // S] * S + at % S)
    client.copy_pages(cache.buffer, [(P - 1, 3), (P - 2, P - 5)])
    q = rounded(rng.standard_normal((1, 16, D)), "bf16")
    b = Builder()
    a = [b.arg((1, 16, D), "bf16"), b.arg(cache.shape, "bf16"), b.arg((1, 2), "i32"), b.arg((1,), "i32")]
    exe = client.compile(b.module([b.paged_attention(*a)]))
    small = np.zeros((1, 2, 2, S, KH, D))
    small[0].reshape(2, 2 * S, KH, D)[:, :n] = rows[0]
    want, mag, top = operators.paged_attention(q, small, np.array([[0, 1]]), [n], bounds=True)
    for t in (table, np.array([[3, P - 5]], np.int32)):
        got = exe.execute([put(client, q, "bf16"), cache.buffer, client.buffer_from_host(t), client.buffer_from_host(np.array([n], np.int32))])[0].to_numpy()
        assert (np.abs(got - want) <= attention_tolerance(want, mag, top, n, D, "bf16", U["bf16"])).all()
    cache.buffer.delete()


# ---- inside programs -----------------------------------------------------------------------------------------
def test_operators_in_a_recorded_program_and_a_loop(client):
    """Several operators whose scratch lives in one arena, replayed with other buffers, and one in a loop body."""
    rng = np.random.default_rng(12)
    q, cache, table, lengths, _ = paged_case(rng, [700, 20, 300], 4, 2, 64, 16, "f32", False)
    b = Builder()
    a = [b.arg(q.shape, "f32"), b.arg(cache.shape, "f32"), b.arg(table.shape, "i32"), b.arg(lengths.shape, "i32")]
    outs, x = [], a[0]
    for w in (0, 300, 150, 0):
        x = b.paged_attention(x, *a[1:], window=w, sinks=2 if w else 0)
        outs.append(b.mul(x, b.full(q.shape, 2.0, "f32")))
    flat = b.reshape(x, (12, 64))
    outs += b.token_log_probs(flat, b.reshape(b.concatenate([a[3]] * 4, 0), (12,)), top=3)
    loop = b.while_([b.const(0, "i32"), a[0]], lambda s, i, v: s.compare(i, s.const(3, "i32"), "LT"),
                    lambda s, i, v: [s.add(i, s.const(1, "i32")), s.paged_attention(v, a[1], a[2], a[3])])
    text = b.module(outs + [loop[1]])
    exe = client.compile(text)
    for seed in range(3):
        q2 = np.random.default_rng(seed).standard_normal(q.shape).astype(np.float32)
        args = [q2, cache, table, lengths]
        want = interp.run_text(text, args)
        for _ in range(2):
            got = [o.to_numpy() for o in exe.execute([client.buffer_from_host(v) for v in args])]
            for g, w in zip(got, want):
                np.testing.assert_allclose(g, w, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_prompts_and_losses_in_a_recorded_program(client, dt):
    """Kernels that read arguments through tensor maps and a loss with its gradient, replayed with other buffers each time."""
    b = Builder()
    q, k, v = (b.arg((2, 150, h, 64), dt) for h in (4, 2, 2))
    n, x, t, w = b.arg((2,), "i32"), b.arg((296, 8200), dt), b.arg((296,), "i32"), b.arg((296,), "f32")
    outs, y = [], q
    for window in (0, 100, 33, 1):
        y = b.window_attention(y, k, v, n, window=window, sinks=2 if window else 0)
        outs.append(b.mul(y, b.full(y.shape, 2.0, dt)))
    lp = b.token_log_probs(x, t)[0]
    outs += [lp, *b.grad(b.reduce_sum(b.mul(lp, w), (0,)), [x])]
    exe = client.compile(b.module(outs))
    for seed in range(3):
        rng = np.random.default_rng(seed)
        arrays = [rounded(rng.standard_normal(s), dt) for s in ((2, 150, 4, 64), (2, 150, 2, 64), (2, 150, 2, 64))]
        lengths, logits = np.array([150 - seed, 77 + seed], np.int32), rounded(rng.standard_normal((296, 8200)), dt)
        tokens, weights = rng.integers(0, 8200, 296).astype(np.int32), rng.standard_normal(296).astype(np.float32)
        for _ in range(2):
            bufs = [put(client, a, dt) for a in arrays] + [client.buffer_from_host(lengths), put(client, logits, dt), client.buffer_from_host(tokens), client.buffer_from_host(weights)]
            got = [np.asarray(o.to_numpy(), np.float64) for o in exe.execute(bufs)]
            q = arrays[0]
            for i, window in enumerate((0, 100, 33, 1)):
                want, mag, top = operators.window_attention(q, *arrays[1:], lengths, window=window, sinks=2 if window else 0, bounds=True)
                assert (np.abs(got[i] / 2 - want) <= attention_tolerance(want, mag, top, 150, 64, dt, 0.0 if dt == "f32" else U[dt])).all()
                q = got[i] / 2                             # exact: what the next call read
            # a log probability: differences of numbers below 16 rounded a few times, and a sum of 8200 terms that are good to 2^-22
            assert (np.abs(got[4] - operators.token_log_probs(logits, tokens)[0]) <= 8 * 16 * E + 2.0 ** -21).all()
            want = operators.token_log_probs_grad(logits, tokens, weights, np.zeros(296), np.zeros(296))
            assert (np.abs(got[5] - want) <= U[dt] * np.abs(want) + 2.0 ** -18 * np.abs(weights)[:, None]).all()


def test_two_calls_in_flight(client):
    rng = np.random.default_rng(13)
    cases = [paged_case(rng, [900, 33], 8, 2, 64, 16, "f32", False) for _ in range(2)]
    b = Builder()
    c = cases[0]
    a = [b.arg(x.shape, dt) for x, dt in zip(c[:4], ("f32", "f32", "i32", "i32"))]
    exe = client.compile(b.module([b.paged_attention(*a)]))
    bufs = [[client.buffer_from_host(x) for x in c[:4]] for c in cases]
    outs = [exe.execute(bufs[i % 2])[0] for i in range(10)]
    for i, o in enumerate(outs):
        np.testing.assert_allclose(o.to_numpy(), operators.paged_attention(*cases[i % 2][:4]), rtol=1e-4, atol=1e-5)


# ---- maxima that grow from tile to tile ---------------------------------------------------------------------
def rising_case(rng, B, T, H, KH, D, dt, growth):
    """Scores that rise by `growth` (of the logarithm to base 2) from each 128 keys to the next, and values that fall by as much, so that every
    tile is as large a share of the result as the last, although all but it are scaled down on the way there."""
    q, k, v = prompt_case(rng, B, T, H, KH, D, dt)
    tile = np.arange(T) // 128
    q[..., 0], q[..., 1:] = 1.0, q[..., 1:] / 16
    k[..., 0] = (tile * (growth * np.log(2)))[None, :, None]
    k[..., 1:] /= 16
    most = 13 if dt == "f16" else growth * (T // 128) // 2
    v = v * 2.0 ** (most - tile * float(growth))[None, :, None, None]
    return [rounded(x, dt) for x in (q, k, v)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,H,KH,D", [(1, 2, 1, 64), (1, 1, 1, 72), (2, 2, 2, 128), (1, 2, 1, 192), (1, 2, 1, 256), (19, 8, 4, 64), (19, 8, 8, 128)])
@pytest.mark.parametrize("growth,window,sinks", [(9, 0, 0), (9, 300, 3), (5, 0, 0)])
def test_window_attention_of_rising_scores(client, dt, B, H, KH, D, growth, window, sinks):
    """One tile of queries a block (with two threads a row), two tiles of one head (19 x 8 heads, 2 tiles each), two heads: in each the outputs are
    scaled down, not to nothing, at every tile or every other one."""
    T = 250 if B > 1 and H == 8 else 384 if dt == "f16" else 700
    rng = np.random.default_rng(D + growth)
    q, k, v = rising_case(rng, B, T, H, KH, D, dt, growth)
    arrays, dts = [q, k, v], [dt] * 3
    kw = dict(window=window, sinks=sinks, scale=1.0)
    first, second = (run(client, lambda b, q, k, v: b.window_attention(q, k, v, **kw), arrays, dts)[0] for _ in range(2))
    np.testing.assert_array_equal(first, second)
    some = sorted({0, B - 1})
    want, mag, top = operators.window_attention(q[some], k[some], v[some], bounds=True, **kw)
    # (weights are in units of a maximum that is at most 2^8 below their tile's: none is small enough to lose bits beside its own rounding)
    tol = attention_tolerance(want, mag, top, T, D, dt, 0.0 if dt == "f32" else U[dt])
    bad = ~(np.abs(first[some] - want) <= tol)
    assert not bad.any(), (float(np.abs(first[some] - want)[bad].max()), np.argwhere(bad)[:5].tolist(), int(bad.sum()))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,V,top", [(1, 256000, 64), (3, 128257, 128), (40, 30522, 20)])
def test_alternatives_repeat_themselves(client, dt, R, V, top):
    """Rows of several parts: whichever thread finds an alternative, its log probability has the same bits, in each call and for equal logits."""
    rng = np.random.default_rng(V)
    x = rounded(rng.standard_normal((R, V)) * 4, dt)
    x[:, 1::2] = x[:, :V // 2 * 2:2]                                     # equal logits among the best
    b = Builder()
    a, t = b.arg(x.shape, dt), b.arg((R,), "i32")
    exe = client.compile(b.module(b.token_log_probs(a, t, top=top)))
    bufs = [put(client, x, dt), client.buffer_from_host(np.zeros(R, np.int32))]
    first = [o.to_numpy() for o in exe.execute(bufs)]
    for r in range(R):
        best = x[r, first[4][r]]
        assert (np.diff(first[3][r])[np.diff(best) == 0] == 0).all()
    for _ in range(20):
        for g, w in zip(exe.execute(bufs), first):
            np.testing.assert_array_equal(g.to_numpy(), w)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("R,V,top", [(1, 300000, 128), (2, 300000, 100), (1, 600001, 64)])
def test_alternatives_of_few_rows_of_large_vocabularies(client, dt, R, V, top):
    rng = np.random.default_rng(V + R)
    check_probs(client, rounded(rng.standard_normal((R, V)) * 4, dt), rng.integers(0, V, R), top, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,KH,D,S", [(4, 1, 64, 16), (3, 3, 128, 7), (2, 1, 72, 8), (24, 1, 192, 16), (6, 2, 256, 5)])
@pytest.mark.parametrize("lens", [[20, 3, 0], [3001, 400], [17] * 40 + [700]])
def test_paged_attention_of_values_that_are_no_numbers(client, dt, H, KH, D, S, lens):
    """Visible infinities and NaN in values and keys, the type's largest value, in the cache and beside it: what the definition makes of them, in
    the features and heads that they reach and in no others."""
    rng = np.random.default_rng(D + len(lens))
    q, cache, table, lengths, fresh = paged_case(rng, lens, H, KH, D, S, dt, True)
    values = cache[0, 1]

    def at(b, j):
        return table[b, j // S], j % S
    values[at(0, 1)][:, 3], values[at(0, 2)][:, 3] = np.inf, np.inf
    values[at(0, lens[0] - 1)][:, 5], values[at(0, 0)][:, D - 1] = -np.inf, np.nan
    values[at(0, 4)][:, 10], values[at(0, 5)][:, 10] = np.inf, -np.inf
    values[at(0, 6)][:, 11] = {"f32": 3.4028235e38, "bf16": 3.3895314e38, "f16": 65504.0}[dt]
    fresh[1, 1, :, 7], fresh[1, -1, 0, 2] = np.inf, -np.inf
    cache[0, 0][at(len(lens) - 2 if lens[-1] == 0 else len(lens) - 1, 1)][KH - 1, 9] = np.inf        # a score without a bound: to one side no weight, to the other no number
    with np.errstate(all="ignore"):
        got = run(client, lambda b, q, c, t, n, new: b.paged_attention(q, c, t, n, new=new), [q, cache, table, lengths, fresh], [dt, dt, "i32", "i32", dt])[0]
        raw = operators.paged_attention(q, cache, table, lengths, fresh)
        known = [np.where(np.isfinite(t), t, 0.0) for t in (cache, fresh)]
        _, mag, top = operators.paged_attention(q, known[0], table, lengths, known[1], bounds=True)
        tol = attention_tolerance(np.where(np.isfinite(raw), raw, 0.0), mag, top, max(lens) + 1, D, dt, 0.0 if dt == "f32" else U[dt] ** 2)
        assert np.isinf(raw).any() and np.isnan(raw).any() and np.isfinite(raw).mean() > 0.3
        np.testing.assert_array_equal(np.isnan(got), np.isnan(raw))
        np.testing.assert_array_equal(got[np.isinf(raw)], raw[np.isinf(raw)])
        fine = np.isfinite(raw)
        assert (np.abs(got - raw)[fine] <= tol[fine]).all(), float((np.abs(got - raw) - tol)[fine].max())


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,H,KH,D", [(1, 2, 1, 64), (1, 1, 1, 256), (19, 8, 4, 64), (19, 8, 8, 128)])
def test_window_attention_of_infinities_with_little_weight(client, dt, B, H, KH, D):
    """A visible infinity with e^-25 of the largest weight, which is no number of f16 any more, is an infinity all the same."""
    T = 250
    rng = np.random.default_rng(D)
    q, k, v = prompt_case(rng, B, T, H, KH, D, dt)
    q[..., 0], q[..., 1:] = 1.0, q[..., 1:] / 16
    k[..., 0], k[..., 1:] = 0.0, k[..., 1:] / 16
    k[:, 7, :, 0], k[:, 150, :, 0] = -25.0, -25.0
    v[:, 7, :, 3], v[:, 150, :, 3], v[:, 150, :, 6] = np.inf, -np.inf, -np.inf
    q, k, v = (rounded(x, dt) for x in (q, k, v))
    got = run(client, lambda b, q, k, v: b.window_attention(q, k, v, scale=1.0), [q, k, v], [dt] * 3)[0]
    some = sorted({0, B - 1})
    with np.errstate(all="ignore"):
        raw = operators.window_attention(q[some], k[some], v[some], scale=1.0)
        want, mag, top = operators.window_attention(q[some], k[some], np.where(np.isfinite(v[some]), v[some], 0.0), scale=1.0, bounds=True)
    got = got[some]
    assert (raw[:, 7:150, :, 3] == np.inf).all() and np.isnan(raw[:, 150:, :, 3]).all() and (raw[:, 150:, :, 6] == -np.inf).all()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(raw))
    np.testing.assert_array_equal(got[np.isinf(raw)], raw[np.isinf(raw)])
    fine = np.isfinite(raw)
    tol = attention_tolerance(want, mag, top, T, D, dt, 0.0 if dt == "f32" else U[dt])
    assert (np.abs(got - want)[fine] <= tol[fine]).all()


@pytest.mark.parametrize("bad_rows", [False, True])
@pytest.mark.parametrize("wait", [False, True])
def test_a_cache_is_not_marked_by_others(client, bad_rows, wait):
    """Among many executions whose rows go into a cache one gives up on a wait (test hook: a barrier nothing arrives at): the cache is invalid
    if its rows went in, however long ago, and not if they did not."""
    shape = (1, 2, 4, 1, 256)
    cache = put(client, np.zeros((1, 2, 60, 4, 1, 256)), "bf16")
    b = Builder()
    x = b.arg((256, 256), "bf16")                                         # a product in 16 bits: its executions are watched
    exe = client.compile(b.module([b.reshape(b.slice(b.dot_general(x, x, ([1], [0])), (0, 0), (8, 256)), shape)]))
    arg = put(client, np.eye(256), "bf16")
    client.synchronize()
    for i in range(60):
        if i == 7:
            client.debug_arm_wait_expiry(1000)
            bad = exe.execute([arg])[0]
            if bad_rows:
                client.write_pages(cache, bad, [28, 29, 30, 31])
        rows = exe.execute([arg])[0]
        client.write_pages(cache, rows, [4 * i, 4 * i + 1, 4 * i + 2, 4 * i + 3])
        if wait:
            rows.to_numpy()
    if bad_rows:
        for _ in range(2):
            with pytest.raises(b200.B200Error, match="bounded"):
                cache.to_numpy()
    else:
        got = cache.to_numpy()
        assert np.array_equal(got[0], np.broadcast_to(np.eye(256, dtype=np.float32)[:8].reshape(2, 1, 4, 1, 256), (2, 60, 4, 1, 256)))
    with pytest.raises(b200.B200Error):
        client.synchronize()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H", [1, 12])
@pytest.mark.parametrize("n", [2, 300])
def test_paged_attention_keeps_both_parts_of_a_weight(client, dt, H, n):
    """Two positions whose contributions nearly cancel: what is left is what the rounding of a weight to 16 bits leaves of it."""
    B, D, S = 40, 64, 16
    less = rounded(np.linspace(0.1, 2.0, B), dt)                       # the second score lies this much below the first
    pages = -(-n // S)
    table, lengths = np.arange(B * pages, dtype=np.int32).reshape(B, pages), np.full(B, n, np.int32)
    q, cache = np.zeros((B, H, D)), np.zeros((1, 2, B * pages, S, 1, D))
    q[..., 0] = 1.0
    cache[0, 0, ..., 0] = -100.0                                       # the others have no weight to speak of
    for b in range(B):
        for place, score, value in ((0, 0.0, rounded(np.exp(-less[b]), dt)), (1, -less[b], -1.0)):
            cache[0, 0, table[b, place // S], place % S, 0, 0] = score
            cache[0, 1, table[b, place // S], place % S] = value
    got = run(client, lambda b, *a: b.paged_attention(*a, scale=1.0), [q, cache, table, lengths], [dt, dt, "i32", "i32"])[0]
    want, mag, _ = operators.paged_attention(q, cache, table, lengths, scale=1.0, bounds=True)
    # (the largest score that counts is 2)
    tol = attention_tolerance(want, mag, 2.0, n, D, dt, U[dt] ** 2)
    assert (np.abs(want) > 2 * tol).any()                              # a weight in one part, whose result is zero, would not pass
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


def test_products_with_a_cache_behind_a_move(client):
    """A product may read an argument ahead of its wait for the kernel in front of it; what a move writes is there all the same."""
    D, S, P = 256, 64, 256
    shape, n = (1, 2, P, S, 1, D), P * S
    b = Builder()
    x, c = b.arg((1, D), "bf16"), b.arg(shape, "bf16")
    exe = client.compile(b.module([b.dot_general(x, c, ((1,), (5,)))]))
    one = np.zeros((1, D))
    one[0, 0] = 1.0
    first, cache = put(client, one, "bf16"), put(client, np.zeros(shape), "bf16")
    rows = [put(client, np.full((1, 2, n, 1, D), v), "bf16") for v in (1.0, 2.0)]
    slots = np.arange(n, dtype=np.int32)[::-1].copy()
    for _ in range(3):
        outs = []
        for i in range(20):
            client.write_pages(cache, rows[i % 2], slots)
            outs.append(exe.execute([first, cache])[0])
        for i, o in enumerate(outs):
            assert (o.to_numpy() == 1.0 + i % 2).all()


def test_profiles_name_operators(client):
    """The report names an operator as one, with its own name, and its launches are not counted among copies."""
    b = Builder()
    x, t = b.arg((4, 1000), "f32"), b.arg((4,), "i32")
    exe = client.compile(b.module(b.token_log_probs(x, t, top=3)))
    args = [client.buffer_from_host(np.zeros((4, 1000), np.float32)), client.buffer_from_host(np.zeros(4, np.int32))]
    client.set_profiling(True)
    try:
        exe.execute(args)
        report = client.profile_report()
    finally:
        client.set_profiling(False)
    kinds = {e["key"]: e["kind"] for e in report if "token_log_probs" in e["key"]}
    assert set(kinds.values()) == {"operator"}, report


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_operators_in_a_loop_of_unknown_length(client, dt):
    """The first call goes round by the host, later ones on the device; other arguments, other lengths."""
    rng = np.random.default_rng(3)
    q, cache, table, lengths, _ = paged_case(rng, [300, 20], 4, 2, 64, 16, dt, False)
    k, v = (rounded(rng.standard_normal((2, 40, 2, 64)), dt) for _ in range(2))
    b = Builder()
    a = [b.arg(q.shape, dt), b.arg(cache.shape, dt), b.arg(table.shape, "i32"), b.arg((2,), "i32"), b.arg((), "i32"), b.arg((2, 40, 4, 64), dt), b.arg(k.shape, dt), b.arg(k.shape, dt)]
    outs = b.while_([b.const(0, "i32"), a[0], a[5]], lambda s, i, x, y: s.compare(i, a[4], "LT"),
                    lambda s, i, x, y: [s.add(i, s.const(1, "i32")), s.paged_attention(x, a[1], a[2], a[3]), s.window_attention(y, a[6], a[7], a[3], window=9)])
    exe = client.compile(b.module(list(outs[1:])))
    prompts = rounded(rng.standard_normal((2, 40, 4, 64)), dt)
    held = [put(client, x, d) for x, d in ((q, dt), (cache, dt), (table, "i32"), (lengths, "i32"))]
    rest = [put(client, x, dt) for x in (prompts, k, v)]
    seen = {}
    for n in (3, 3, 1, 3, 2, 1, 2):
        got = [o.to_numpy() for o in exe.execute([*held, client.buffer_from_host(np.array(n, np.int32)), *rest])]
        if n in seen:
            for g, w in zip(got, seen[n]):
                np.testing.assert_array_equal(g, w)
        seen[n] = got
    want, mag, top = operators.paged_attention(q, cache, table, lengths, bounds=True)
    assert (np.abs(seen[1][0] - want) <= attention_tolerance(want, mag, top, 300, 64, dt, 0.0 if dt == "f32" else U[dt])).all()
    for n in (2, 3):                                               # each turn reads the last one's results as they are
        want, mag, top = operators.paged_attention(seen[n - 1][0], cache, table, lengths, bounds=True)
        assert (np.abs(seen[n][0] - want) <= attention_tolerance(want, mag, top, 300, 64, dt, 0.0 if dt == "f32" else U[dt])).all()
        want, mag, top = operators.window_attention(seen[n - 1][1], k, v, lengths, window=9, bounds=True)
        assert (np.abs(seen[n][1] - want) <= attention_tolerance(want, mag, top, 40, 64, dt, 0.0 if dt == "f32" else U[dt])).all()


def test_two_clients_at_once():
    """Two clients on two threads, with caches of their own. (A client is closed when nothing of it is left.)"""
    import threading
    errors = []

    def use(c, seed):
        rng = np.random.default_rng(seed)
        q, cache, table, lengths, fresh = paged_case(rng, [500, 40, 7], 8, 2, 128, 16, "bf16", True)
        x, y, z = prompt_case(rng, 1, 200, 2, 1, 64, "bf16")
        for _ in range(10):
            check_paged(c, q, cache, table, lengths, fresh, "bf16")
        buf, rows = put(c, cache, "bf16"), rounded(rng.standard_normal((1, 2, 5, 2, 128)), "bf16")
        for i in range(30):
            slots, pairs = np.arange(5) + 5 * (i % 3), [(0, 5), (5, 0)]
            c.write_pages(buf, put(c, rows, "bf16"), slots)
            c.copy_pages(buf, pairs)
            cache = operators.copy_pages(operators.write_pages(cache, rows, slots), pairs)
        np.testing.assert_array_equal(buf.to_numpy(), cache)
        check_prompt(c, x, y, z, None, "bf16")

    def work(c, seed):
        try:
            use(c, seed)
        except Exception as e:                  # handed to the test's thread
            errors.append(repr(e))
    clients = [b200.Client() for _ in range(2)]
    threads = [threading.Thread(target=work, args=(c, k)) for k, c in enumerate(clients)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=120)
    assert not errors and not any(t.is_alive() for t in threads), errors
    for c in clients:
        c.synchronize()
        c.close()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D,T", [(256, 300), (192, 257), (136, 200), (64, 300)])
def test_window_attention_repeats_itself(client, dt, D, T):
    """Several units of one tile of queries for each block (64 features: of two), tiles of keys whose products the slowest warp holds up: the same
    bits from the first call of a program and from all others, in 180 heads of 30 sequences."""
    rng = np.random.default_rng(D)
    q, k, v = prompt_case(rng, 30, T, 6, 2, D, dt)
    bufs = [put(client, x, dt) for x in (q, k, v)]
    first = None
    for window in (0, 0, 0, 150):
        b = Builder()
        exe = client.compile(b.module([b.window_attention(*[b.arg(x.shape, dt) for x in (q, k, v)], window=window)], name=f"jit_repeat_{window}"))
        outs = [np.asarray(exe.execute(bufs)[0].to_numpy()) for _ in range(8)]
        for o in outs[1:] + ([first] if first is not None and not window else []):
            np.testing.assert_array_equal(o, outs[0])
        first = outs[0] if first is None else first
        for s in (0, 17):
            want, mag, top = operators.window_attention(q[s:s + 1, :, ::5], k[s:s + 1], v[s:s + 1], window=window, bounds=True)
            assert (np.abs(outs[0][s:s + 1, :, ::5] - want) <= attention_tolerance(want, mag, top, T, D, dt, U[dt])).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 3, 300])
def test_rows_whose_scores_are_all_minus_infinity(client, dt, n):
    """They have no weight to give and are zero like rows that see nothing, whatever the values are."""
    D = 64
    q, k, v = np.ones((1, n, 2, D)), np.full((1, n, 1, D), -np.inf), np.ones((1, n, 1, D))
    v[0, 0, 0, 3], v[0, n - 1, 0, 5], v[0, n // 2, 0, 7] = np.inf, np.nan, -np.inf
    got = run(client, lambda b, q, k, v: b.window_attention(q, k, v), [q, k, v], [dt] * 3)[0]
    with np.errstate(all="ignore"):
        np.testing.assert_array_equal(got, operators.window_attention(q, k, v))
    assert (got == 0).all()
    pages = -(-n // 16)
    cache = np.zeros((1, 2, pages, 16, 1, D))
    cache[0].reshape(2, pages * 16, 1, D)[:, :n] = np.concatenate([k, v])
    got = run(client, lambda b, *a: b.paged_attention(*a), [q[:, 0], cache, np.arange(pages, dtype=np.int32)[None], np.array([n], np.int32)], [dt, dt, "i32", "i32"])[0]
    assert (got == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_attention_of_values_that_are_nan_without_infinities(client, dt):
    """NaN of values and keys reach what sees them and nothing else; there is nothing to make again."""
    rng = np.random.default_rng(14)
    q, cache, table, lengths, fresh = paged_case(rng, [700, 20, 300], 6, 2, 72, 16, dt, True)
    cache[0, 1, table[0, 3], 5, 0, 9], cache[0, 1, table[0, 40], 1, 1] = np.nan, np.nan
    cache[0, 0, table[1, 0], 7, 1, 3], fresh[1, 2, 0, 70] = np.nan, np.nan
    got = run(client, lambda b, q, c, t, n, new: b.paged_attention(q, c, t, n, new=new), [q, cache, table, lengths, fresh], [dt, dt, "i32", "i32", dt])[0]
    raw = operators.paged_attention(q, cache, table, lengths, fresh)
    want, mag, top = operators.paged_attention(q, np.nan_to_num(cache), table, lengths, np.nan_to_num(fresh), bounds=True)
    tol = attention_tolerance(want, mag, top, 701, 72, dt, 0.0 if dt == "f32" else U[dt] ** 2)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(raw))
    assert np.isnan(raw).any() and (np.abs(got - raw)[~np.isnan(raw)] <= tol[~np.isnan(raw)]).all()
    q, k, v = prompt_case(rng, 2, 200, 6, 2, 72, dt)
    v[0, 40, 0, 9], v[1, 0, 1], k[0, 150, 1, 3] = np.nan, np.nan, np.nan
    got = run(client, lambda b, q, k, v: b.window_attention(q, k, v, window=70, sinks=2), [q, k, v], [dt] * 3)[0]
    raw = operators.window_attention(q, k, v, window=70, sinks=2)
    want, mag, top = operators.window_attention(q, np.nan_to_num(k), np.nan_to_num(v), window=70, sinks=2, bounds=True)
    tol = attention_tolerance(want, mag, top, 200, 72, dt, 0.0 if dt == "f32" else U[dt])
    np.testing.assert_array_equal(np.isnan(got), np.isnan(raw))
    assert (np.abs(got - want)[~np.isnan(raw)] <= tol[~np.isnan(raw)]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_attention_of_infinite_queries(client, dt):
    """An infinite feature of a query makes scores of plus and minus infinity: of minus infinity alone, a row without weight; of both, none but
    plus infinity's, which is no number."""
    rng = np.random.default_rng(16)
    q, cache, table, lengths, _ = paged_case(rng, [300, 40], 3, 1, 64, 16, dt, False)
    cache[0, 0, ..., 5] = rounded(np.abs(cache[0, 0, ..., 5]) + 0.25, dt)
    q[0, 0, 5], q[0, 2, 5], q[1, 1, 7] = -np.inf, np.inf, np.inf
    got = run(client, lambda b, *a: b.paged_attention(*a), [q, cache, table, lengths], [dt, dt, "i32", "i32"])[0]
    with np.errstate(all="ignore"):
        raw = operators.paged_attention(q, cache, table, lengths)
    assert (raw[0, 0] == 0).all() and np.isnan(raw[0, 2]).all() and np.isnan(raw[1, 1]).all()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(raw))
    want, mag, top = operators.paged_attention(np.where(np.isfinite(q), q, 0.0), cache, table, lengths, bounds=True)
    fine = [(0, 1), (1, 0), (1, 2)]
    tol = attention_tolerance(want, mag, top, 300, 64, dt, 0.0 if dt == "f32" else U[dt] ** 2)
    assert (got[0, 0] == 0).all() and all((np.abs(got - want) <= tol)[i].all() for i in fine)
