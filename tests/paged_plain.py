"""Plain float64 restatement of the operators over paged caches, and caches to test them with: pages in random order, NaN wherever a
sequence has no row, table entries behind a sequence's last page that name no page."""
import numpy as np

from ratchet_b200 import capi

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}      # a rounding is off by at most this, relative to the value


def encode(a, dt):
    """Host array of the type, and the values it holds."""
    with np.errstate(over="ignore"):
        a = np.asarray(a, np.float32)
        if dt == BF16:
            u = capi.to_bf16(a)
            return u, capi.from_bf16(u).astype(np.float64)
        h = a.astype(np.float16) if dt == F16 else a
        return h, h.astype(np.float64)


def decode(a, dt):
    return (capi.from_bf16(a) if dt == BF16 else a).astype(np.float64)


class Cache:
    """Rows k [S][L, G, D] and v [S][L, G, E] in pages, as host arrays of the type and as float64."""

    def __init__(self, g, dt, new, lengths, G, D, E, R, spare=2, fill=np.nan, std=1.0):
        self.dt, self.new, self.lengths, self.G, self.D, self.E, self.R = dt, list(new), list(lengths), G, D, E, R
        need = [-(-n // R) for n in lengths]
        pages, most = sum(need) + spare, max(1, max(need))
        ids = g.permutation(pages)
        self.table = np.full((len(lengths), most), -1, np.int32)
        self.k, self.v, at = [], [], 0
        keys = np.full((pages, G, R, D), fill, np.float32)
        values = np.full((pages, G, R, E), fill, np.float32)
        for s, (n, L) in enumerate(zip(need, lengths)):
            self.table[s, :n] = ids[at:at + n]
            at += n
            k, v = std * g.standard_normal((L, G, D)), g.standard_normal((L, G, E))
            for r in range(L):
                p = self.table[s, r // R]
                keys[p, :, r % R], values[p, :, r % R] = k[r], v[r]
            self.k.append(encode(k, dt)[1])
            self.v.append(encode(v, dt)[1])
        self.keys, self.values = encode(keys, dt)[0], encode(values, dt)[0]
        self.free = ids[at:]
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.rows = most * R

    def rows_of(self, pages, table, s, L):
        """[L, G, width] of a sequence's rows in (device) pages."""
        a = decode(pages, self.dt)
        return np.stack([a[table[s, r // self.R], :, r % self.R] for r in range(L)]) if L else np.zeros((0, self.G, a.shape[-1]))


def seen(L, n, window, first):
    """[n, L]: rows that each of a sequence's last n tokens sees."""
    r, j = np.arange(L - n, L)[:, None], np.arange(L)[None]
    return (j <= r) & ((j > r - window) | (j < first) if window else True)


def attention(cache, q, scale, sink=None, window=0, first=0):
    """(out [T, H, E], sum of weights times |v| [T, H, E], weight that every row received [S][G, L])."""
    T, H, _ = q.shape
    per = H // cache.G
    out, size, mass = np.zeros((T, H, cache.E)), np.zeros((T, H, cache.E)), []
    for s, (n, L) in enumerate(zip(cache.new, cache.lengths)):
        m = np.zeros((cache.G, L))
        t = cache.starts[s]
        vis = seen(L, n, window, first)
        for h in range(H):
            if n == 0:
                continue
            z = np.where(vis, scale * (q[t:t + n, h] @ cache.k[s][:, h // per].T), -np.inf)
            top = z.max(1, keepdims=True) if sink is None else np.maximum(z.max(1, keepdims=True), sink[h])
            w = np.exp(z - top)
            w /= w.sum(1, keepdims=True) + (0 if sink is None else np.exp(sink[h] - top))
            v = cache.v[s][:, h // per]
            with np.errstate(invalid="ignore"):
                for i in range(n):                      # what a token does not see has no part in its sum, whatever it holds
                    out[t + i, h] = w[i, vis[i]] @ v[vis[i]]
                    size[t + i, h] = w[i, vis[i]] @ np.abs(v[vis[i]])
            m[h // per] += w.sum(0)
        mass.append(m)
    return out, size, mass


def rotary(x, freqs, positions, sections, magnitude, first, halves):
    """x [T, heads, dim] turned by positions [axes, T]."""
    pairs = len(freqs)
    axis = np.repeat(np.arange(len(sections)), sections)
    a = positions.astype(np.float64)[axis].T * freqs                # [T, pairs]
    c, s = magnitude * np.cos(a)[:, None], magnitude * np.sin(a)[:, None]
    y = x.copy()
    i = first + np.arange(pairs) * (1 if halves else 2)
    j = i + (pairs if halves else 1)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def kept(mass, L, keep, first, recent):
    """Rows that an eviction keeps of L with these sums (NaN the least, of equal ones the lower)."""
    if L <= keep:
        return np.arange(L)
    middle = np.arange(first, L - recent)
    m = mass[middle].astype(np.float64)
    order = np.lexsort((middle, -np.where(np.isnan(m), -np.inf, m), np.isnan(m)))
    return np.concatenate([np.arange(first), np.sort(middle[order[:keep - first - recent]]), np.arange(L - recent, L)]).astype(int)
