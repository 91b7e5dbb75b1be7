"""Operators over paged caches through the device ABI against the plain float64 restatement (paged_plain.py): rotation by given positions,
append, attention and eviction, alone and in a run as a server makes it."""
import numpy as np
import pytest

from ratchet_b200 import PagedCache, RatchetCudaError, Tensor, capi, nn

from . import paged_plain as pp
from .paged_plain import BF16, F16, F32, HALF_STEP
from .test_gpu_dadezen_ops import dev, rng  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu

DTS = [F32, F16, BF16]


def up(dev, a, dt=None):
    return dev.from_numpy(np.ascontiguousarray(a), dt=dt)


def put(dev, a, dt):
    h, v = pp.encode(a, dt)
    return up(dev, h, dt), v


def get(buf):
    return pp.decode(buf.to_numpy(), buf.dt)


def device_cache(dev, c, mass=None):
    i = lambda a: up(dev, np.asarray(a, np.int32))  # noqa: E731
    m = None if mass is None else up(dev, mass.astype(np.float32))
    return PagedCache(up(dev, c.keys, c.dt), up(dev, c.values, c.dt), i(c.table), i(c.lengths), i(c.starts), m)


def close(got, want, size, dt, vmax):
    """Elementwise: the output's rounding, the rounding of every weight to the operands' type (16 bits: half a step of sum w |v|), and f32
    arithmetic: scores of up to 256 products are off by about 16 half steps of their terms' size (some 10 for the inputs here: 1e-5), which
    moves a weight by as much relative to itself, hence the sum by 2e-5 of the largest value."""
    h = HALF_STEP[dt]
    bound = h * (np.abs(want) + (size if dt != F32 else 0)) * 1.02 + 2e-5 * vmax
    return float(np.max((np.abs(got - want) - bound) / vmax)) <= 0


# ---------------------------------------------------------------------------------------- rotation
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("T,H,D,first,sections,col,halves", [
    (1, 1, 8, 0, (4,), 0, False), (5, 3, 64, 0, (32,), 8, True), (33, 2, 80, 0, (8, 16, 16), 0, True), (7, 4, 128, 16, (10, 6, 20, 4), 16, False),
    (300, 6, 96, 0, (48,), 0, False), (9, 3, 20, 3, (5,), 1, True), (9, 2, 14, 2, (2, 3), 3, False), (4, 1, 256, 64, (0, 32, 16), 0, True)])
def test_rotary_axes(dev, dt, T, H, D, first, sections, col, halves):
    g = rng(T * D + col)
    pairs = sum(sections)
    f = 10000.0 ** (-np.arange(pairs) / pairs)
    hi = f.astype(np.float32)
    freqs = up(dev, np.stack([hi, (f - hi).astype(np.float32)]))
    # far positions, negative ones, and the ends of the type
    at = g.integers(-200000, 2 ** 20, (len(sections), T)).astype(np.int32)
    at[0, 0], at[-1, -1] = 2 ** 31 - 1, -2 ** 31
    x, xv = put(dev, g.standard_normal((T, col + H * D + 8)), dt)
    got = get(dev.rotary_axes(x, H, D, freqs, up(dev, at), sections, magnitude=1.25, col=col, first=first, halves=halves))
    want = pp.rotary(xv[:, col:col + H * D].reshape(T, H, D), f, at, sections, 1.25, first, halves)
    # the output's rounding; a cosine's (two half steps of f32 and its own), times two terms of size 1.25 * 5; the table: 2^-48 of an angle of 2^31
    assert np.all(np.abs(got - want) <= HALF_STEP[dt] * np.abs(want) + 8 * 2.0 ** -24 * 1.25 * np.abs(xv).max() + 2.0 ** -16 * np.abs(xv).max())
    assert np.array_equal(np.delete(got, np.arange(first, first + 2 * pairs), 2), np.delete(xv[:, col:col + H * D].reshape(T, H, D), np.arange(first, first + 2 * pairs), 2))


def test_rotary_axes_near_positions_are_exact_to_f32(dev):
    g = rng(3)
    f = 500.0 ** (-np.arange(32) / 32)
    hi = f.astype(np.float32)
    at = np.concatenate([np.arange(50), [131071, 999983]]).astype(np.int32)[None]
    x, xv = put(dev, g.standard_normal((52, 3 * 64)), F32)
    want = pp.rotary(xv.reshape(52, 3, 64), f, at, (32,), 1.0, 0, False)
    buf = x
    got = get(dev.rotary_axes(buf, 3, 64, up(dev, np.stack([hi, (f - hi).astype(np.float32)])), up(dev, at), (32,), out=buf.view((52, 3, 64))))       # in place
    assert np.abs(got - want).max() < 6 * 2.0 ** -24 * np.abs(xv).max()


@pytest.mark.parametrize("halves", [False, True])
def test_rotary_axes_of_more_rows_than_stay_on_chip(dev, halves):
    """Rows of no whole number of 128-byte lines, a last group of tokens that is not full."""
    g = rng(11)
    T, H, D, col = 5203, 41, 80, 4
    f = 10000.0 ** (-np.arange(40) / 40)
    hi = f.astype(np.float32)
    at = g.integers(0, 2 ** 17, (2, T)).astype(np.int32)
    x, xv = put(dev, g.standard_normal((T, col + H * D)), F32)
    got = get(dev.rotary_axes(x, H, D, up(dev, np.stack([hi, (f - hi).astype(np.float32)])), up(dev, at), (24, 16), col=col, halves=halves))
    want = pp.rotary(xv[:, col:].reshape(T, H, D), f, at, (24, 16), 1.0, 0, halves)
    assert np.abs(got - want).max() < 6 * 2.0 ** -24 * np.abs(xv).max()


# ---------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("new,lengths,G,D,E,R,k_col,v_col", [
    ([1], [1], 1, 8, 8, 16, 0, 0), ([3, 0, 17, 1], [3, 9, 40, 33], 2, 24, 40, 16, 8, 16), ([40], [100], 6, 64, 64, 32, 0, 3), ([0, 0], [5, 0], 1, 16, 8, 16, 0, 0),
    ([1] * 70, list(range(1, 71)), 2, 80, 80, 64, 1, 0), ([130, 2], [130, 1024], 3, 256, 128, 1024, 0, 0)])
def test_append(dev, dt, new, lengths, G, D, E, R, k_col, v_col):
    g = rng(sum(lengths) + D)
    c = pp.Cache(g, dt, new, lengths, G, D, E, R, fill=0.5)
    T = sum(new)
    k, kv = put(dev, g.standard_normal((T + 3, k_col + G * D + 5)), dt)          # three rows belong to no sequence
    v, vv = put(dev, g.standard_normal((T + 3, v_col + G * E)), dt)
    mass = g.random((len(new), G, c.rows)) + 1
    d = device_cache(dev, c, mass)
    dev.paged_append(k, v, d, k_col=k_col, v_col=v_col)
    keys, values, want_m = pp.decode(c.keys, dt), pp.decode(c.values, dt), mass.astype(np.float32)
    for s, (n, L) in enumerate(zip(new, lengths)):
        for i in range(n):
            r, t = L - n + i, c.starts[s] + i
            p = c.table[s, r // R]
            keys[p, :, r % R] = kv[t, k_col:k_col + G * D].reshape(G, D)
            values[p, :, r % R] = vv[t, v_col:v_col + G * E].reshape(G, E)
            want_m[s, :, r] = 0
    assert np.array_equal(get(d.keys), keys) and np.array_equal(get(d.values), values) and np.array_equal(d.mass.to_numpy(), want_m)
    dev.sync()


# ---------------------------------------------------------------------------------------- attention
# new tokens, rows with them, H, G, D, E, page rows, window, first, sink
SHAPES = [
    ([1], [1], 1, 1, 8, 8, 16, 0, 0, False),
    ([1, 1, 1], [5, 128, 129], 4, 2, 64, 64, 16, 0, 0, True),
    ([3, 0, 1, 20], [3, 7, 300, 50], 6, 2, 96, 96, 32, 0, 0, False),
    ([70, 1], [200, 513], 7, 1, 80, 80, 64, 0, 0, False),
    ([129], [129], 4, 4, 128, 128, 128, 0, 0, False),
    ([300], [700], 8, 2, 128, 64, 256, 100, 4, True),
    ([1, 40], [1000, 1000], 10, 2, 64, 128, 16, 1, 0, False),
    ([1, 9], [600, 300], 16, 1, 112, 48, 32, 130, 200, False),
    ([17], [33], 3, 1, 24, 40, 16, 5, 1, True),
    ([6, 1], [260, 90], 2, 2, 256, 256, 64, 0, 0, False),
    ([33], [4100], 4, 2, 128, 128, 1024, 0, 0, False),
    ([1] * 40, [3 * i + 1 for i in range(40)], 5, 5, 64, 64, 16, 20, 2, False),
    ([2, 260], [2, 260], 130, 1, 16, 16, 16, 0, 0, False),
]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("new,lengths,H,G,D,E,R,window,first,sink", SHAPES)
def test_attention(dev, dt, new, lengths, H, G, D, E, R, window, first, sink):
    g = rng(sum(lengths) + H)
    c = pp.Cache(g, dt, new, lengths, G, D, E, R)
    T, scale = sum(new), 1.0 / np.sqrt(D)
    q, qv = put(dev, 1.5 * g.standard_normal((T, H, D)), dt)
    sk = g.standard_normal(H).astype(np.float32) if sink else None
    want, size, mass = pp.attention(c, qv, scale, sk, window, first)
    vmax = max(np.abs(v).max() for v in c.v if v.size)
    skb = up(dev, sk) if sink else None
    got = get(dev.paged_attention(q, device_cache(dev, c), scale, skb, window, first)).reshape(T, H, E)
    assert close(got, want, size, dt, vmax)
    # with the weights summed: the same outputs, and sums whose terms are off by what scores are off by (2e-5, see close)
    before = g.random((len(new), G, c.rows)).astype(np.float32)
    d = device_cache(dev, c, before)
    again = get(dev.paged_attention(q, d, scale, skb, window, first)).reshape(T, H, E)
    assert np.array_equal(again, got)
    grown = d.mass.to_numpy().astype(np.float64) - before
    for s, L in enumerate(lengths):
        assert np.all(np.abs(grown[s, :, :L] - mass[s]) <= 2e-5 * mass[s] + 4 * 2.0 ** -24 * (1 + mass[s]))
        assert np.all(grown[s, :, L:] == 0)
    dev.sync()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("H,G,D,n,L,window", [(4, 1, 64, 150, 290, 0), (2, 2, 128, 130, 130, 40), (8, 2, 80, 1, 300, 0), (3, 1, 24, 20, 40, 7)])
def test_attention_of_values_that_are_not_finite(dev, dt, H, G, D, n, L, window):
    """Infinities and NaN among the values and keys reach the tokens that see them, and no others."""
    g = rng(L + H)
    c = pp.Cache(g, dt, [n], [L], G, D, D, 16)
    q, qv = put(dev, g.standard_normal((n, H, D)), dt)
    places = [(L - 1, 0, np.inf), (L - max(1, n // 2), 1, -np.inf), (max(0, L - n - 3), 2, np.nan), (L // 3, 3, np.inf)]
    keys, values = pp.decode(c.keys, dt), pp.decode(c.values, dt)
    for r, d, x in places:
        c.v[0][r, 0, d] = values[c.table[0, r // 16], 0, r % 16, d] = x
    bad = L - 2 if n > 2 else None
    if bad is not None:                                     # a key: NaN for who sees it
        c.k[0][bad, 0, 0] = keys[c.table[0, bad // 16], 0, bad % 16, 0] = np.nan
    c.keys, c.values = pp.encode(keys, dt)[0], pp.encode(values, dt)[0]
    with np.errstate(invalid="ignore"):
        want, size, _ = pp.attention(c, qv, 0.125, None, window)
    got = get(dev.paged_attention(q, device_cache(dev, c), 0.125, window=window)).reshape(n, H, D)
    fine = np.isfinite(want)
    assert fine.any() and np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
    assert close(np.where(fine, got, 0), np.where(fine, want, 0), np.where(np.isfinite(size), size, 0), dt, 5.0)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("new,R,window", [(6, 16, 0), (40, 32, 0), (9, 64, 20)])
def test_many_short_sequences_some_with_values_that_are_not_finite(dev, dt, new, R, window):
    """Every CTA of the tensor-core kernel has many items in a row, whose query tiles leave warps without a query; infinities in every third sequence, in rows that
    some of its tokens see, have no part in its neighbours.  Which warp is ahead of which cannot be forced (test_paged.py has the order as a model)."""
    g = rng(new + R)
    S, H, G, D = 500 if new < 20 else 300, 8, 2, 64
    news = [new + s % 3 if s % 5 else 36 for s in range(S)]           # some with two query tiles
    lengths = [n + int(g.integers(0, 150)) for n in news]
    c = pp.Cache(g, dt, news, lengths, G, D, D, R)
    values = pp.decode(c.values, dt)
    for s in range(0, S, 3):
        for r, d, x in ((lengths[s] - 1, 3, np.inf), (lengths[s] - news[s] // 2, 5, np.nan)):
            c.v[s][r, s % G, d] = values[c.table[s, r // R], s % G, r % R, d] = x
    c.values = pp.encode(values, dt)[0]
    T = sum(news)
    q, qv = put(dev, g.standard_normal((T, H, D)), dt)
    want, size, _ = pp.attention(c, qv, 0.125, None, window)
    d = device_cache(dev, c)
    first = get(dev.paged_attention(q, d, 0.125, window=window)).reshape(want.shape)
    fine = np.isfinite(want)
    assert not fine.all() and np.array_equal(np.isnan(first), np.isnan(want)) and np.array_equal(np.isposinf(first), np.isposinf(want))
    assert close(np.where(fine, first, 0), np.where(fine, want, 0), np.where(np.isfinite(size), size, 0), dt, 5.0)
    for _ in range(30):
        again = get(dev.paged_attention(q, d, 0.125, window=window)).reshape(want.shape)
        assert np.array_equal(again, first, equal_nan=True)
    dev.sync()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("what", ["query", "key"])
@pytest.mark.parametrize("n,L,D,window", [(70, 300, 64, 0), (70, 300, 64, 25), (200, 200, 80, 40), (4, 60, 64, 3), (9, 40, 136, 4)])
def test_a_token_without_a_softmax_has_no_part_in_the_sums_of_rows_that_it_does_not_see(dev, dt, what, n, L, D, window):
    """A query of NaN, and one that has minus infinity for every row that it sees: the rows that it sees receive NaN, all others what the other tokens give."""
    g = rng(n + L)
    H, G = 4, 2
    at = n // 3
    c = pp.Cache(g, dt, [n], [L], G, D, D, 16)
    h, qv = pp.encode(g.standard_normal((n, H, D)), dt)
    keys = pp.decode(c.keys, dt)
    odd = np.zeros((n, G), bool)                            # tokens without a softmax in one of the group's heads
    if what == "query":
        qv[at, 3] = np.nan
        odd[at, 1] = True
    else:
        qv[:, 2:, 0] = 1.0
        for r in range(L - n + at + 1):                     # all that the token sees, and those before it
            c.k[0][r, 1, 0] = keys[c.table[0, r // 16], 1, r % 16, 0] = -np.inf
        vis = pp.seen(L, n, window, 0)
        odd[:, 1] = [not vis[i, L - n + at + 1:].any() for i in range(n)]
    q = up(dev, pp.encode(qv, dt)[0], dt)
    c.keys = pp.encode(keys, dt)[0]
    want, vis = np.zeros((G, L)), np.broadcast_to(pp.seen(L, n, window, 0), (n, L))
    for head in range(H):
        for i in range(n):
            rows = np.flatnonzero(vis[i])
            with np.errstate(invalid="ignore"):
                z = 0.125 * c.k[0][rows, head // 2] @ qv[i, head]
                w = np.exp(z - z.max())
                want[head // 2, rows] += w / w.sum()
    assert np.isnan(want).any() and np.isfinite(want).any()
    assert np.array_equal(np.isnan(want), np.stack([(odd[:, k, None] & vis).any(0) for k in range(G)]))
    d = device_cache(dev, c, np.zeros((1, G, c.rows)))
    dev.paged_attention(q, d, 0.125, window=window)
    got = d.mass.to_numpy()[0, :, :L].astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert np.all(np.abs(got - want)[fine] <= 2e-5 * want[fine] + 4 * 2.0 ** -24 * (1 + want[fine]))
    dev.sync()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("n,L,D,window", [(70, 300, 64, 25), (200, 200, 80, 40), (4, 60, 64, 3), (9, 40, 136, 4), (40, 40, 64, 0)])
def test_a_sink_beside_nothing_but_minus_infinities(dev, dt, n, L, D, window):
    """A token that has minus infinity for every row that it sees gives all its weight to the sink: its output is zero, and no row's sum grows by it."""
    g = rng(n + L + 1)
    H, G, upto = 4, 2, L - n + n // 3 + 1
    c = pp.Cache(g, dt, [n], [L], G, D, D, 16)
    q = g.standard_normal((n, H, D))
    q[:, :, 0] = 1.0
    keys = pp.decode(c.keys, dt)
    for r in range(upto):
        c.k[0][r, 1, 0] = keys[c.table[0, r // 16], 1, r % 16, 0] = -np.inf
    c.keys = pp.encode(keys, dt)[0]
    q, qv = put(dev, q, dt)
    sink = np.array([0.5, -30.0, 2.0, -1.0], np.float32)
    want, size, mass = pp.attention(c, qv, 0.125, sink, window)
    assert np.isfinite(want).all() and np.isfinite(mass[0]).all() and not want[0, 2:].any()
    d = device_cache(dev, c, np.zeros((1, G, c.rows)))
    got = get(dev.paged_attention(q, d, 0.125, up(dev, sink), window)).reshape(n, H, D)
    assert close(got, want, size, dt, 5.0) and not got[0, 2:].any()
    grown = d.mass.to_numpy()[0, :, :L].astype(np.float64)
    assert np.all(np.abs(grown - mass[0]) <= 2e-5 * mass[0] + 4 * 2.0 ** -24 * (1 + mass[0]))
    dev.sync()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,L", [(1, 131000), (8, 20008), (64, 20064)])
def test_attention_under_a_row_far_above_all_others(dev, dt, n, L):
    """A first row 17 above all others, as language models have it: the weights of the others are 2^-25 of its own, and together they are what an f16's half step
    of the output would show.  Every sequence reads the same pages, so that each CTA has whole items: a few rows each, one query tile, and two."""
    g = rng(n)
    S, H, G, D, R = 40, 16, 4, 16, 256
    c = pp.Cache(g, dt, [n], [16], G, D, D, R, spare=0)          # its rows are made below: as many as that one by one take a while
    pages = -(-L // R)
    k, v = 0.1 * g.standard_normal((pages * R, G, D)), 0.25 + 0.75 * g.random((pages * R, G, D))
    k[0], v[0] = 4.35, 0.05
    hk, k = pp.encode(k, dt)
    hv, v = pp.encode(v, dt)
    paged = lambda a: np.ascontiguousarray(a.reshape(pages, R, G, D).transpose(0, 2, 1, 3))  # noqa: E731
    c.keys, c.values, c.k, c.v, c.lengths = paged(hk), paged(hv), [k[:L]], [v[:L]], [L]
    hq, qv = pp.encode(1 + 0.01 * g.standard_normal((n, H, D)), dt)
    want, size, _ = pp.attention(c, qv, 0.25)
    assert 0.9 < np.exp(-17.4) * (L - n) * 0.625 / (want.mean() - 0.05) < 1.3 or dt == BF16
    c.table, c.lengths = np.tile(np.arange(pages, dtype=np.int32), (S, 1)), [L] * S
    c.starts = (n * np.arange(S + 1)).astype(np.int32)
    got = get(dev.paged_attention(up(dev, np.tile(hq, (S, 1, 1)), dt), device_cache(dev, c), 0.25)).reshape(S, n, H, D)
    assert all(close(got[s], want, size, dt, 1.0) for s in range(S))


@pytest.mark.parametrize("dt", DTS)
def test_single_weights_keep_their_bits(dev, dt):
    """One query of 32 heads, each with two rows of weight: row 0, and one of its own whose sum is then that one weight e^-d / (1 + e^-d).  Scores are exact.  In
    units of log 2 the exponent is off by log2 e's rounding (d log2 e < 2.9: 1.8e-7), its own (1.2e-7), and the lse's: the other weight's exponential (2^-22 of at
    most half the sum), the product's and the sum's roundings (3e-7 together), log2f's last place (4.8e-7 in f16, where the sum is 128 times as large); times
    ln 2 that is 7.5e-7 of the weight.  Its own exponential adds 2^-22."""
    H = D = 32
    c = pp.Cache(rng(1), dt, [1], [130], 1, D, D, 16)
    d = (np.arange(4 * H).reshape(4, H) + 1) / 64
    for turn in range(4):
        k = np.full((130, D), -200.0)
        k[0] = 0
        own = 3 * np.arange(H) + 5 + turn
        k[own, np.arange(H)] = -d[turn]
        keys = pp.decode(c.keys, dt)
        for r in range(130):
            keys[c.table[0, r // 16], 0, r % 16] = k[r]
        c.keys = pp.encode(keys, dt)[0]
        q = put(dev, np.eye(H)[None], dt)[0]
        cache = device_cache(dev, c, np.zeros((1, 1, c.rows)))
        dev.paged_attention(q, cache, 1.0)
        got = cache.mass.to_numpy()[0, 0].astype(np.float64)
        want = np.exp(-d[turn]) / (1 + np.exp(-d[turn]))
        assert np.abs(got[own] / want - 1).max() <= 1.0e-6
        others = np.delete(got, np.concatenate([[0], own]))
        assert not others.any() and abs(got[0] - (H - want.sum())) < 1e-5


@pytest.mark.parametrize("dt", DTS)
def test_attention_leaves_rows_of_no_sequence(dev, dt):
    g = rng(11)
    c = pp.Cache(g, dt, [3, 5], [30, 5], 2, 64, 64, 16)
    q, qv = put(dev, g.standard_normal((12, 4, 64)), dt)
    c.starts = np.array([2, 5, 10], np.int32)               # two tokens before the first sequence, two behind the last
    out = up(dev, pp.encode(np.full((12, 256), 7.0), dt)[0], dt)
    dev.paged_attention(q, device_cache(dev, c), 0.125, out=out)
    want, size, _ = pp.attention(c, qv, 0.125)
    got = get(out)
    assert np.all(got[[0, 1, 10, 11]] == 7)
    assert close(got[2:10].reshape(8, 4, 64), want[2:10], size[2:10], dt, 5.0)


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
@pytest.mark.parametrize("dt", DTS)
def test_attention_scales(dev, dt, scale):
    g = rng(5)
    c = pp.Cache(g, dt, [60, 1], [200, 77], 1, 32, 32, 16)
    q, qv = put(dev, g.standard_normal((61, 2, 32)), dt)
    want, size, _ = pp.attention(c, qv, scale)
    got = get(dev.paged_attention(q, device_cache(dev, c), scale)).reshape(61, 2, 32)
    # scores of a few hundred: f32 keeps them to 2^-24 of their terms, some 40 * 32, which is 1e-4 of a weight
    assert np.all(np.abs(got - want) <= HALF_STEP[dt] * (np.abs(want) + (size if dt != F32 else 0)) * 1.02 + 1e-3)


def test_shared_pages_and_scratch_of_the_caller(dev):
    """Two sequences over the same prompt's pages, twice on one scratch."""
    g = rng(21)
    c = pp.Cache(g, BF16, [1, 1], [64, 64], 2, 64, 64, 32)
    c.table[1] = c.table[0]
    c.k[1], c.v[1] = c.k[0], c.v[0]
    q, qv = put(dev, g.standard_normal((2, 4, 64)), BF16)
    d = device_cache(dev, c)
    scratch = dev.empty(F32, (max(1, dev.paged_attention_scratch(q, d) // 4),))
    want, size, _ = pp.attention(c, qv, 0.125)
    for _ in range(2):
        got = get(dev.paged_attention(q, d, 0.125, scratch=scratch)).reshape(2, 4, 64)
        assert close(got, want, size, BF16, 5.0)


# ---------------------------------------------------------------------------------------- eviction
EVICT = [
    ([100], 2, 24, 40, 16, 40, 4, 10), ([5, 33, 0, 300], 3, 64, 64, 32, 33, 0, 0), ([1000, 999], 1, 8, 8, 16, 1000, 1000, 0), ([700], 2, 128, 128, 64, 64, 0, 64),
    ([3000, 17, 1500], 2, 96, 64, 256, 1025, 7, 300), ([40, 41], 6, 16, 16, 16, 1, 0, 0), ([5000], 1, 256, 256, 1024, 4999, 1, 1), ([64], 70, 8, 16, 16, 9, 1, 2)]


def masses(g, S, G, rows):
    """Many ties, zeros of both signs, infinities and NaN."""
    m = np.round(g.exponential(3.0, (S, G, rows)), 0).astype(np.float32)
    m[g.random(m.shape) < 0.1] *= -1.0
    m[g.random(m.shape) < 0.02] = np.nan
    m[g.random(m.shape) < 0.01] = np.inf
    m[g.random(m.shape) < 0.01] = -np.inf
    return m


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("place", ["fresh", "same", "pages"])
@pytest.mark.parametrize("lengths,G,D,E,R,keep,first,recent", EVICT)
def test_evict(dev, dt, place, lengths, G, D, E, R, keep, first, recent):
    g = rng(sum(lengths) + keep)
    S = len(lengths)
    most = max(1, -(-min(keep, max(lengths)) // R))
    c = pp.Cache(g, dt, [0] * S, lengths, G, D, E, R, spare=S * most + 3, fill=0.25)
    mass = masses(g, S, G, c.rows)
    d = device_cache(dev, c, mass)
    new_lengths = up(dev, np.full(S, -5, np.int32))
    if place == "fresh":                                    # other arrays
        table = g.permutation(S * most + 1)[:S * most].reshape(S, most).astype(np.int32)
        blank = lambda w: up(dev, pp.encode(np.full((S * most + 1, G, R, w), 0.75), dt)[0], dt)  # noqa: E731
        into = PagedCache(blank(D), blank(E), up(dev, table), new_lengths, mass=up(dev, np.full((S, G, most * R), 9, np.float32)))
    elif place == "pages":                                  # free pages of the same arrays
        table = c.free[:S * most].reshape(S, most).astype(np.int32)
        into = PagedCache(d.keys, d.values, up(dev, table), new_lengths, mass=up(dev, np.full((S, G, most * R), 9, np.float32)))
    else:                                                   # in place
        table = c.table
        into = PagedCache(d.keys, d.values, d.table, new_lengths, mass=d.mass)
    dev.paged_evict(d, into, keep, first, recent)
    keys, values, sums = into.keys.to_numpy(), into.values.to_numpy(), into.mass.to_numpy()
    assert np.array_equal(new_lengths.to_numpy(), np.minimum(lengths, keep))
    for s, L in enumerate(lengths):
        n = min(L, keep)
        got_k, got_v = c.rows_of(keys, table, s, n), c.rows_of(values, table, s, n)
        for h in range(G):
            rows = pp.kept(mass[s, h], L, keep, first, recent)
            assert np.array_equal(got_k[:, h], c.k[s][rows, h]) and np.array_equal(got_v[:, h], c.v[s][rows, h])
            assert np.array_equal(sums[s, h, :n], mass[s, h, rows], equal_nan=True)
            if place != "same":
                assert np.all(sums[s, h, n:] == 9)
    dev.sync()


# ---------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dt,new", [(BF16, [1, 2]), (F16, [90, 40]), (F32, [3, 1])])
def test_pages_beyond_32_bits(dev, dt, new):
    """Pools of more than 2^32 bytes: rows written to, read from and moved between pages at both ends."""
    g = rng(23)
    G, D, R, lengths = 4, 128, 256, [300, 520]
    pages = 2 ** 32 // (G * R * D * (4 if dt == F32 else 2)) + 9
    keys, values = dev.empty(dt, (pages, G, R, D)), dev.empty(dt, (pages, G, R, D))
    table = np.array([[pages - 1, 3, 0], [1, pages - 2, pages - 5]], np.int32)
    c = pp.Cache(g, dt, lengths, lengths, G, D, D, R)
    k, _ = put(dev, np.concatenate([x.reshape(-1, G * D) for x in c.k]), dt)
    v, _ = put(dev, np.concatenate([x.reshape(-1, G * D) for x in c.v]), dt)
    ints = lambda a: up(dev, np.asarray(a, np.int32))  # noqa: E731
    mass = up(dev, g.random((2, G, 3 * R)).astype(np.float32))
    cache = PagedCache(keys, values, ints(table), ints(lengths), ints([0, 300, 820]), mass)
    before = mass.to_numpy()
    dev.paged_append(k, v, cache)
    assert np.all(mass.to_numpy()[0, :, :300] == 0) and np.array_equal(mass.to_numpy()[0, :, 300:], before[0, :, 300:])
    c.new, c.starts = new, np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q, qv = put(dev, g.standard_normal((sum(new), 8, D)), dt)
    want, size, sums = pp.attention(c, qv, 0.09)
    now = PagedCache(keys, values, cache.table, cache.lengths, ints(c.starts), mass)
    assert close(get(dev.paged_attention(q, now, 0.09)).reshape(want.shape), want, size, dt, 5.0)
    grown = mass.to_numpy()
    into = PagedCache(keys, values, ints([[pages - 7], [5]]), dev.zeros(capi.I32, (2,)), mass=dev.zeros(F32, (2, G, R)))
    dev.paged_evict(now, into, 200, 3, 50)
    one = dev.wrap(dt, (1, G, R, D), keys.ptr + (pages - 7) * G * R * D * (4 if dt == F32 else 2))
    got = get(one)[0]
    for h in range(G):
        assert np.allclose(grown[0, h, :300], sums[0][h], rtol=1e-4, atol=1e-6)
        assert np.array_equal(got[h, :200], c.k[0][pp.kept(grown[0, h], 300, 200, 3, 50), h])
    keys.free()
    values.free()
    dev.check(dev._lib.rcu_pool_trim(dev.handle))


def serve(dev, dt, step, evict):
    """Three sequences: prompts, then single tokens, their rows cut to 40 whenever one has more than 60; against float64 all the way."""
    g = rng(8)
    H, G, D, R, MP, keep, first, recent = 4, 2, 64, 16, 8, 40, 2, 12
    rows = MP * R
    k64, v64, m64 = [[np.zeros((0, G, D)) for _ in range(3)] for _ in range(2)] + [[np.zeros((G, 0)) for _ in range(3)]]
    for new in [[50, 20, 0], [1, 1, 33], [9, 1, 1], [1, 1, 1], [30, 0, 1], [1, 1, 60]]:
        T = sum(new)
        q, k, v = (pp.encode(g.standard_normal((T, n * D)), dt) for n in (H, G, G))
        c = pp.Cache.__new__(pp.Cache)
        c.dt, c.new, c.G, c.D, c.E, c.R = dt, new, G, D, D, R
        c.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        for s, n in enumerate(new):
            t = c.starts[s]
            k64[s] = np.concatenate([k64[s], k[1][t:t + n].reshape(n, G, D)])
            v64[s] = np.concatenate([v64[s], v[1][t:t + n].reshape(n, G, D)])
            m64[s] = np.concatenate([m64[s], np.zeros((G, n))], 1)
        c.k, c.v, c.lengths = k64, v64, [len(x) for x in k64]
        want, size, mass = pp.attention(c, q[1].reshape(T, H, D), 0.125)
        got = step(q[0].reshape(T, H, D), k[0], v[0], c.starts, np.asarray(c.lengths, np.int32))
        assert close(pp.decode(got, dt).reshape(T, H, D), want, size, dt, 5.0)
        m64 = [a + b for a, b in zip(m64, mass)]
        if max(c.lengths) > 60:
            m, lengths = evict(keep, first, recent)
            assert np.array_equal(lengths, np.minimum(c.lengths, keep))
            for s, L in enumerate(c.lengths):
                k2, v2, m2 = [], [], []
                for h in range(G):
                    at = pp.kept(m64[s][h], L, keep, first, recent)
                    assert np.allclose(m[s, h, :len(at)], m64[s][h][at], rtol=1e-4, atol=1e-6)
                    k2.append(k64[s][at, h])
                    v2.append(v64[s][at, h])
                    m2.append(m64[s][h][at])
                k64[s], v64[s], m64[s] = np.stack(k2, 1), np.stack(v2, 1), np.stack(m2)
    return rows


@pytest.mark.parametrize("dt", DTS)
def test_a_run_of_calls(dev, dt):
    G, D, R, MP = 2, 64, 16, 8
    table = up(dev, rng(1).permutation(3 * MP).reshape(3, MP).astype(np.int32))
    keys, values = dev.zeros(dt, (3 * MP, G, R, D)), dev.zeros(dt, (3 * MP, G, R, D))
    mass, cut = dev.zeros(F32, (3, G, MP * R)), dev.zeros(capi.I32, (3,))
    last = {}

    def step(q, k, v, starts, lengths):
        last["c"] = c = PagedCache(keys, values, table, up(dev, lengths), up(dev, starts), mass)
        dev.paged_append(up(dev, k, dt), up(dev, v, dt), c)
        return dev.paged_attention(up(dev, q, dt), c, 0.125).to_numpy()

    def evict(keep, first, recent):
        dev.paged_evict(last["c"], PagedCache(keys, values, table, cut, mass=mass), keep, first, recent)
        return mass.to_numpy(), cut.to_numpy()

    serve(dev, dt, step, evict)


@pytest.mark.parametrize("dt", [F16, F32])
def test_a_run_of_the_graph(dev, dt):
    """The same through the lazy graph: rows that the graph computes, nodes ordered by the lengths they hand on."""
    G, D, R, MP = 2, 64, 16, 8
    leaf = lambda a: Tensor.from_data(a, device=dev)  # noqa: E731
    host = np.float16 if dt == F16 else np.float32
    table = leaf(rng(1).permutation(3 * MP).reshape(3, MP).astype(np.int32))
    keys, values = leaf(np.zeros((3 * MP, G, R, D), host)), leaf(np.zeros((3 * MP, G, R, D), host))
    mass = leaf(np.zeros((3, G, MP * R), np.float32))
    last = {}

    def step(q, k, v, starts, lengths):
        c = nn.PagedState(keys, values, table, leaf(starts), leaf(lengths), mass)
        # keys and values through a node of the graph: a sum with zeros
        after = leaf(k).add(leaf(np.zeros_like(k))).paged_append(leaf(v), c)
        last["c"] = after
        return leaf(q).paged_attention(after, 0.125).to_numpy()

    def evict(keep, first, recent):
        lengths = last["c"].evict(nn.PagedState(keys, values, table, None, None, mass), keep, first, recent).lengths.to_numpy()
        return mass.to_numpy(), lengths

    serve(dev, dt, step, evict)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("steps", [1, 3])
def test_a_graph_whose_eviction_is_resolved_first(dev, dt, steps):
    """Append, attention with sums and eviction in place, of one step or three, all unresolved, each step's lengths from the host: the last eviction is resolved first and
    the outputs from the last to the first; outputs and weights are those of the order in which the nodes were built."""
    g = rng(19)
    H, G, D, R, MP, keep, first, recent = 4, 2, 64, 16, 8, 30, 2, 9
    leaf = lambda a, t=None: Tensor.from_data(a, device=dev, dt=t)  # noqa: E731
    table = leaf(g.permutation(3 * MP).reshape(3, MP).astype(np.int32))
    pages = pp.encode(np.zeros((3 * MP, G, R, D)), dt)[0]
    keys, values, mass = leaf(pages, dt), leaf(pages, dt), leaf(np.zeros((3, G, MP * R), np.float32))
    k64, v64, m64 = [np.zeros((0, G, D))] * 3, [np.zeros((0, G, D))] * 3, [np.zeros((G, 0))] * 3
    outs, wants = [], []
    for new in [[50, 20, 41], [9, 1, 30], [1, 33, 1]][:steps]:
        T = sum(new)
        q, k, v = (pp.encode(g.standard_normal((T, n * D)), dt) for n in (H, G, G))
        c = pp.Cache.__new__(pp.Cache)
        c.dt, c.new, c.G, c.D, c.E, c.R = dt, new, G, D, D, R
        c.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        for s, n in enumerate(new):
            rows = slice(c.starts[s], c.starts[s] + n)
            k64[s], v64[s] = np.concatenate([k64[s], k[1][rows].reshape(n, G, D)]), np.concatenate([v64[s], v[1][rows].reshape(n, G, D)])
            m64[s] = np.concatenate([m64[s], np.zeros((G, n))], 1)
        c.k, c.v, c.lengths = list(k64), list(v64), [len(x) for x in k64]
        want, size, grown = pp.attention(c, q[1].reshape(T, H, D), 0.125)
        wants.append((want, size))
        for s, L in enumerate(c.lengths):
            m = m64[s] + grown[s]
            at = [pp.kept(m[h], L, keep, first, recent) for h in range(G)]
            k64[s], v64[s] = (np.stack([x[s][at[h], h] for h in range(G)], 1) for x in (k64, v64))
            m64[s] = np.stack([m[h, at[h]] for h in range(G)])
        state = nn.PagedState(keys, values, table, leaf(c.starts), leaf(np.asarray(c.lengths, np.int32)), mass)
        after = leaf(k[0], dt).paged_append(leaf(v[0], dt), state)
        outs.append(leaf(q[0].reshape(T, H, D), dt).paged_attention(after, 0.125))
        cut = after.evict(nn.PagedState(keys, values, table, None, None, mass), keep, first, recent).lengths
        lengths = np.minimum(c.lengths, keep)
        del state, after
    assert np.array_equal(cut.to_numpy(), lengths)
    sums, got_k, got_v = mass.to_numpy(), pp.decode(keys.to_numpy(), dt), pp.decode(values.to_numpy(), dt)
    ids = table.to_numpy()
    for s, L in enumerate(lengths):
        assert np.allclose(sums[s, :, :L], m64[s], rtol=1e-4, atol=1e-6)
        for r in range(L):
            assert np.array_equal(got_k[ids[s, r // R], :, r % R], k64[s][r]) and np.array_equal(got_v[ids[s, r // R], :, r % R], v64[s][r])
    for o, (want, size) in reversed(list(zip(outs, wants))):
        assert close(pp.decode(o.to_numpy(), dt).reshape(want.shape), want, size, dt, 5.0)
    dev.sync()


def test_a_graph_that_is_a_step_ahead_keeps_no_outputs(dev):
    """Every step is built before the one ahead of it is resolved: nodes that only come before let go of one another once they have run."""
    g = rng(29)
    leaf = lambda a: Tensor.from_data(a, device=dev)  # noqa: E731
    keys, values, mass = leaf(np.zeros((40, 2, 16, 64), np.float16)), leaf(np.zeros((40, 2, 16, 64), np.float16)), leaf(np.zeros((1, 2, 640), np.float32))
    table, starts = leaf(np.arange(40, dtype=np.int32)[None]), leaf(np.array([0, 30], np.int32))
    k, q = leaf(g.standard_normal((30, 128)).astype(np.float16)), leaf(g.standard_normal((30, 4, 64)).astype(np.float16))
    waiting, used = None, []
    for step in range(20):
        after = k.paged_append(k, nn.PagedState(keys, values, table, starts, leaf(np.array([30 * (step + 1)], np.int32)), mass))
        out = q.paged_attention(after, 0.125)
        if waiting is not None:
            assert np.isfinite(waiting.to_numpy()).all()
        waiting = out
        del after, out
        dev.sync()
        used.append(dev.pool_stats()[0])
    assert len(set(used[3:])) == 1
    assert np.isfinite(waiting.to_numpy()).all()


@pytest.mark.parametrize("dt", [F16, F32])
def test_rotary_axes_of_the_graph(dev, dt):
    """Positions per token through the lazy graph, into a paged cache."""
    g = rng(6)
    T, G, D = 7, 2, 32
    f = 10000.0 ** (-np.arange(16) / 16)
    hi = f.astype(np.float32)
    at = g.integers(0, 5000, (2, T)).astype(np.int32)
    h, v = pp.encode(g.standard_normal((T, 5 + G * D)), dt)
    leaf = lambda a: Tensor.from_data(a, device=dev)  # noqa: E731
    got = leaf(h).rotary_axes(G, D, leaf(np.stack([hi, (f - hi).astype(np.float32)])), leaf(at), (6, 10), magnitude=0.5, col=5, halves=True)
    assert got.shape() == (T, G, D)
    want = pp.rotary(v[:, 5:].reshape(T, G, D), f, at, (6, 10), 0.5, 0, True)
    assert np.all(np.abs(got.to_numpy() - want) <= HALF_STEP[dt] * np.abs(want) + 1e-6)


@pytest.mark.parametrize("dt,new", [(F16, [1, 1, 1]), (BF16, [40, 3, 70]), (F32, [2, 5, 1])])
def test_a_captured_step_replayed_over_new_lengths(dt, new):
    """Append, attention with sums and eviction in one CUDA graph: replayed after the host has moved lengths, starts and rows on."""
    import torch
    from ratchet_b200 import Device
    stream = torch.cuda.Stream()
    d = Device(0, stream=stream.cuda_stream)
    g = rng(13)
    H, G, D, R, MP, T = 4, 2, 64, 16, 16, sum(new)
    table = up(d, g.permutation(3 * MP).reshape(3, MP).astype(np.int32))
    keys, values, mass = d.zeros(dt, (3 * MP, G, R, D)), d.zeros(dt, (3 * MP, G, R, D)), d.zeros(F32, (3, G, MP * R))
    starts, lengths, cut = up(d, np.zeros(4, np.int32)), up(d, np.zeros(3, np.int32)), d.zeros(capi.I32, (3,))
    rows = {n: d.zeros(dt, (T, w * D)) for n, w in (("q", H), ("k", G), ("v", G))}
    c = PagedCache(keys, values, table, lengths, starts, mass)
    into = PagedCache(keys, values, table, cut, mass=mass)
    q, out = rows["q"].view((T, H, D)), d.zeros(dt, (T, H * D))
    scratch = d.empty(F32, (max(4, d.paged_attention_scratch(q, c) // 4),))
    cutting = d.empty(F32, (max(4, d.paged_evict_scratch(c, 150) // 4),))

    def step():
        d.paged_append(rows["k"], rows["v"], c)
        d.paged_attention(q, c, 0.125, scratch=scratch, out=out)
        d.paged_evict(c, into, 150, 2, 100, scratch=cutting)

    step()                                                  # attributes are set once outside the capture
    d.sync()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
        with pytest.raises(RatchetCudaError):               # scratch from the pool would belong to others by the time of a replay
            d.paged_attention(q, c, 0.125, out=out)
    k64, v64, have, m64 = [np.zeros((0, G, D))] * 3, [np.zeros((0, G, D))] * 3, [0] * 3, [np.zeros((G, 0))] * 3
    for turn in range(4):
        order = new if turn % 2 == 0 else new[::-1]         # other lengths than those captured
        host = {n: pp.encode(g.standard_normal((T, b.shape[1])), dt) for n, b in rows.items()}
        for n, b in rows.items():
            d.h2d(b.ptr, host[n][0])
        ref = pp.Cache.__new__(pp.Cache)
        ref.dt, ref.new, ref.G, ref.D, ref.E, ref.R = dt, order, G, D, D, R
        ref.starts = np.concatenate([[0], np.cumsum(order)]).astype(np.int32)
        for s, n in enumerate(order):
            t = ref.starts[s]
            k64[s] = np.concatenate([k64[s], host["k"][1][t:t + n].reshape(n, G, D)])
            v64[s] = np.concatenate([v64[s], host["v"][1][t:t + n].reshape(n, G, D)])
            m64[s] = np.concatenate([m64[s], np.zeros((G, n))], 1)
        ref.k, ref.v, ref.lengths = k64, v64, [len(x) for x in k64]
        d.h2d(starts.ptr, ref.starts)
        d.h2d(lengths.ptr, np.asarray(ref.lengths, np.int32))
        d.sync()
        graph.replay()
        torch.cuda.synchronize()
        want, size, grown = pp.attention(ref, host["q"][1].reshape(T, H, D), 0.125)
        assert close(get(out).reshape(T, H, D), want, size, dt, 5.0), turn
        m64 = [a + b for a, b in zip(m64, grown)]
        sums = mass.to_numpy()
        assert np.array_equal(cut.to_numpy(), np.minimum(ref.lengths, 150))
        for s, L in enumerate(ref.lengths):
            kept = [pp.kept(m64[s][h], L, 150, 2, 100) for h in range(G)]
            k64[s] = np.stack([k64[s][kept[h], h] for h in range(G)], 1)
            v64[s] = np.stack([v64[s][kept[h], h] for h in range(G)], 1)
            m64[s] = np.stack([m64[s][h, kept[h]] for h in range(G)])
            assert np.allclose(sums[s, :, :len(kept[0])], m64[s], rtol=1e-4, atol=1e-6)
    del graph
    d.sync()
    d.close()


def test_two_handles_at_once(dev):
    """Calls on two streams of one device at the same time, each with its pool's scratch."""
    from ratchet_b200 import Device
    other = Device(0)
    g = rng(17)
    jobs = []
    for d, new, lengths, dt in ((dev, [1] * 6, [700] * 6, F16), (other, [200, 1], [900, 300], BF16)):
        c = pp.Cache(g, dt, new, lengths, 2, 64, 64, 32)
        q, qv = put(d, g.standard_normal((sum(new), 8, 64)), dt)
        jobs.append((d, c, device_cache(d, c, np.zeros((len(new), 2, c.rows))), q, qv, dt))
    outs = [[j[0].paged_attention(j[3], j[2], 0.125) for j in jobs] for _ in range(6)]
    for k, (d, c, _, _, qv, dt) in enumerate(jobs):
        want, size, _ = pp.attention(c, qv, 0.125)
        for o in outs:
            assert close(get(o[k]).reshape(want.shape), want, size, dt, 5.0)
    other.sync()
    for o in outs:
        o[1].free()
    for b in (jobs[1][3], jobs[1][2].keys, jobs[1][2].values, jobs[1][2].table, jobs[1][2].starts, jobs[1][2].lengths, jobs[1][2].mass):
        b.free()
    other.close()


# ---------------------------------------------------------------------------------------- refusals
def test_bad_indexes_are_reported(dev):
    g = rng(2)

    def reported(change, call):
        c = pp.Cache(g, F16, [2, 1], [20, 5], 1, 64, 64, 16, fill=0.0)
        change(c)
        call(device_cache(dev, c, np.zeros((2, 1, c.rows))))
        with pytest.raises(RatchetCudaError) as e:
            dev.sync()
        assert e.value.status == capi.ERR_BOUNDS
        dev.sync()                                          # reported once

    q, _ = put(dev, g.standard_normal((3, 2, 64)), F16)
    k, _ = put(dev, g.standard_normal((3, 64)), F16)
    attend = lambda d: dev.paged_attention(q, d, 0.1)  # noqa: E731
    append = lambda d: dev.paged_append(k, k, d)  # noqa: E731

    def setter(name, at, value):
        def change(c):
            a = np.array(getattr(c, name))
            a[at] = value
            setattr(c, name, a)
        return change

    for call in (attend, append):
        for change in (setter("starts", 1, 4), setter("starts", 2, -1), setter("starts", 0, 3), setter("lengths", 0, 33), setter("lengths", 1, -1),
                       setter("lengths", 0, 1), setter("table", (0, 1), 99), setter("table", (1, 0), -7)):
            reported(change, call)
    for change in (setter("lengths", 0, 40), setter("table", (0, 1), 1000)):
        def evict(d):
            into = PagedCache(dev.zeros(F16, (4, 1, 16, 64)), dev.zeros(F16, (4, 1, 16, 64)), up(dev, np.array([[0], [1]], np.int32)), dev.zeros(capi.I32, (2,)),
                              mass=dev.zeros(F32, (2, 1, 16)))
            dev.paged_evict(d, into, 10, 2, 8)
        reported(change, evict)


def test_refusals(dev):
    z = lambda dt, *shape: dev.zeros(dt, shape)  # noqa: E731
    I32 = capi.I32

    def cache(dt=F16, pages=4, G=2, R=16, D=64, E=64, S=2, MP=2, mass=False, **other):
        parts = {"keys": z(dt, pages, G, R, D), "values": z(dt, pages, G, R, E), "table": z(I32, S, MP), "lengths": z(I32, S), "starts": z(I32, S + 1),
                 "mass": z(F32, S, G, MP * R) if mass else None}
        parts.update(other)
        return PagedCache(**parts)

    q, k, x = z(F16, 3, 4, 64), z(F16, 3, 128), z(F16, 3, 256)
    fr, at = z(F32, 2, 32), z(I32, 1, 3)
    dev.paged_attention(q, cache(), 0.1)
    dev.paged_append(k, k, cache())
    dev.rotary_axes(x, 4, 64, fr, at, (32,))
    dev.paged_evict(cache(mass=True), cache(mass=True), 8)
    dev.sync()
    bad = [
        lambda: dev.paged_attention(z(F32, 3, 4, 64), cache(), 0.1), lambda: dev.paged_attention(z(F16, 3, 4, 32), cache(), 0.1),
        lambda: dev.paged_attention(z(F16, 3, 3, 64), cache(), 0.1), lambda: dev.paged_attention(q, cache(), 0.1, sink=z(F32, 2)),
        lambda: dev.paged_attention(q, cache(), 0.1, out=z(F16, 3, 128)), lambda: dev.paged_attention(q, cache(R=8), 0.1), lambda: dev.paged_attention(q, cache(R=24), 0.1),
        lambda: dev.paged_attention(z(F16, 3, 4, 60), cache(D=60), 0.1), lambda: dev.paged_attention(z(F16, 3, 4, 264), cache(D=264), 0.1),
        lambda: dev.paged_attention(q, cache(starts=z(I32, 2)), 0.1), lambda: dev.paged_attention(q, cache(lengths=z(I32, 3)), 0.1),
        lambda: dev.paged_attention(q, cache(lengths=z(F32, 2)), 0.1), lambda: dev.paged_attention(q, cache(starts=None), 0.1),
        lambda: dev.paged_attention(q, cache(mass=True, table=z(I32, 2, 3)), 0.1), lambda: dev.paged_attention(q, cache(values=z(F16, 5, 2, 16, 64)), 0.1),
        lambda: dev.paged_attention(q, cache(values=z(BF16, 4, 2, 16, 64)), 0.1),
        lambda: dev.paged_append(k, z(F16, 2, 128), cache()), lambda: dev.paged_append(k, k, cache(), k_col=1), lambda: dev.paged_append(z(F32, 3, 128), k, cache()),
        lambda: dev.paged_evict(cache(), cache(mass=True), 8), lambda: dev.paged_evict(cache(mass=True), cache(), 8), lambda: dev.paged_evict(cache(mass=True), cache(mass=True), 0),
        lambda: dev.paged_evict(cache(mass=True), cache(mass=True), 8, 5, 4), lambda: dev.paged_evict(cache(mass=True), cache(mass=True, MP=1), 17),
        lambda: dev.paged_evict(cache(mass=True), cache(mass=True, S=3), 8), lambda: dev.paged_evict(cache(mass=True), cache(mass=True, dt=BF16), 8),
        lambda: dev.rotary_axes(x, 4, 64, fr, at, (31,)), lambda: dev.rotary_axes(x, 4, 64, fr, at, (16, 16)), lambda: dev.rotary_axes(x, 4, 64, fr, at, (32,), col=1),
        lambda: dev.rotary_axes(x, 4, 64, fr, at, (32,), first=1), lambda: dev.rotary_axes(x, 4, 64, fr, z(I32, 1, 2), (32,)),
        lambda: dev.rotary_axes(x, 4, 64, fr, z(I32, 5, 3), (32, 0, 0, 0, 0)), lambda: dev.rotary_axes(x, 4, 64, fr, z(F32, 1, 3), (32,)),
        lambda: dev.rotary_axes(x, 2, 64, fr, at, (32,), out=dev.wrap(F16, (3, 2, 64), x.ptr)),
    ]
    m = cache(mass=True)
    bad += [lambda: dev.paged_attention(q, cache(), 0.1, out=q.view((3, 256))),
            lambda: dev.paged_evict(m, m, 8), lambda: dev.paged_evict(m, PagedCache(m.keys, m.values, m.table, m.lengths, mass=m.mass), 8),
            lambda: dev.paged_evict(m, PagedCache(m.values, m.keys, m.table, z(I32, 2), mass=m.mass), 8)]
    for f in bad:
        with pytest.raises(RatchetCudaError):
            f()
    dev.sync()


def test_scratch_that_is_too_small_is_refused(dev):
    g = rng(4)
    c = pp.Cache(g, F16, [1], [3000], 2, 64, 64, 16)
    q, _ = put(dev, g.standard_normal((1, 4, 64)), F16)
    d = device_cache(dev, c, np.zeros((1, 2, c.rows)))
    assert dev.paged_attention_scratch(q, d) > 16
    with pytest.raises(RatchetCudaError):
        dev.paged_attention(q, d, 0.1, scratch=dev.zeros(F32, (4,)))
    into = PagedCache(d.keys, d.values, d.table, dev.zeros(capi.I32, (1,)), mass=d.mass)
    with pytest.raises(RatchetCudaError):
        dev.paged_evict(d, into, 100, scratch=dev.zeros(F32, (4,)))
    dev.paged_evict(d, into, 100, scratch=dev.zeros(F32, (dev.paged_evict_scratch(d, 100) // 4,)))
    dev.sync()
