"""Paged caches where no device is needed: the plain restatement that the GPU tests compare with, against brute force, and what the graph's
builders refuse."""
import ctypes as C

import numpy as np
import pytest

from . import paged_plain as pp
from .test_graph_cpu import _leaf


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


@pytest.mark.parametrize("new,lengths,window,first,sink", [([1, 4], [5, 9], 0, 0, False), ([3, 0, 7], [3, 2, 20], 4, 2, True), ([6], [6], 1, 0, True), ([2], [11], 3, 20, False)])
def test_plain_attention_by_brute_force(new, lengths, window, first, sink):
    g = rng(sum(lengths))
    c = pp.Cache(g, pp.F32, new, lengths, 2, 8, 8, 16)
    q = g.standard_normal((sum(new), 4, 8))
    sk = g.standard_normal(4) if sink else None
    out, _, mass = pp.attention(c, q, 0.3, sk, window, first)
    for s, (n, L) in enumerate(zip(new, lengths)):
        got = np.zeros((2, L))
        for i in range(n):
            r = L - n + i
            for h in range(4):
                rows = [j for j in range(r + 1) if not window or j > r - window or j < first]
                e = [np.exp(0.3 * q[c.starts[s] + i, h] @ c.k[s][j, h // 2]) for j in rows]
                total = sum(e) + (np.exp(sk[h]) if sink else 0)
                assert np.allclose(out[c.starts[s] + i, h], sum(x * c.v[s][j, h // 2] for x, j in zip(e, rows)) / total)
                for x, j in zip(e, rows):
                    got[h // 2, j] += x / total
        assert np.allclose(got, mass[s])


def test_plain_eviction_keeps_the_heaviest_and_the_lower_of_equal_ones():
    m = np.array([9, 1, 5, 5, np.nan, 5, 0, -np.inf, np.inf, 2, 3], np.float32)
    assert list(pp.kept(m, 11, 5, 1, 1)) == [0, 2, 3, 8, 10]
    assert list(pp.kept(m, 11, 11, 1, 1)) == list(range(11))
    assert list(pp.kept(m, 11, 10, 0, 0)) == [0, 1, 2, 3, 5, 6, 7, 8, 9, 10]
    assert list(pp.kept(m, 11, 3, 1, 2)) == [0, 9, 10]


def test_pages_hold_the_rows_and_nothing_else():
    c = pp.Cache(rng(1), pp.BF16, [2, 1], [33, 16], 2, 8, 16, 16)
    assert c.table.shape == (2, 3) and list(c.table[1, 1:]) == [-1, -1]
    assert np.array_equal(c.rows_of(c.keys, c.table, 0, 33), c.k[0]) and np.array_equal(c.rows_of(c.values, c.table, 1, 16), c.v[1])
    assert np.isnan(pp.decode(c.keys, c.dt)).sum() == (len(c.keys) * 16 - 49) * 2 * 8


def test_builders_refuse_what_does_not_fit():
    from ratchet_b200 import capi
    lib, F16, I32, F32 = capi.lib(), capi.F16, capi.I32, capi.F32
    leaf = lambda dt, *shape: _leaf(lib, capi, shape, dt)  # noqa: E731
    keys, values, table, starts, lengths = leaf(F16, 4, 2, 16, 64), leaf(F16, 4, 2, 16, 32), leaf(I32, 3, 2), leaf(I32, 4), leaf(I32, 3)
    mass, k, v, q = leaf(F32, 3, 2, 32), leaf(F16, 5, 130), leaf(F16, 5, 64), leaf(F16, 5, 4, 64)
    out = C.c_void_p()
    ref = C.byref(out)

    def shape():
        t = capi.rcu_tensor()
        lib.rcu_lazy_info(out, C.byref(t))
        got = t.dt, tuple(t.shape[i] for i in range(t.rank))
        lib.rcu_lazy_release(out)
        return got

    assert lib.rcu_lazy_paged_append(k, 2, v, 0, keys, values, table, starts, lengths, mass, ref) == capi.OK and shape() == (I32, (3,))
    assert lib.rcu_lazy_paged_append(k, 3, v, 0, keys, values, table, starts, lengths, None, ref) == capi.ERR_INVALID_ARG          # past the rows' end
    assert lib.rcu_lazy_paged_append(k, 0, q, 0, keys, values, table, starts, lengths, None, ref) == capi.ERR_INVALID_ARG
    assert lib.rcu_lazy_paged_append(k, 0, v, 0, keys, values, table, starts, starts, None, ref) == capi.ERR_INVALID_ARG           # four lengths of three sequences
    assert lib.rcu_lazy_paged_attention(q, keys, values, table, starts, lengths, None, None, 0, 0, 0.1, ref) == capi.OK and shape() == (F16, (5, 128))
    assert lib.rcu_lazy_paged_attention(q, values, values, table, starts, lengths, None, None, 0, 0, 0.1, ref) == capi.ERR_INVALID_ARG
    assert lib.rcu_lazy_paged_attention(None, keys, values, table, starts, lengths, None, None, 0, 0, 0.1, ref) == capi.ERR_INVALID_ARG
    # pages that a node of the graph is still to make
    made = C.c_void_p()
    assert lib.rcu_lazy_unary(8, keys, C.byref(made)) == capi.OK
    assert lib.rcu_lazy_paged_attention(q, made, values, table, starts, lengths, None, None, 0, 0, 0.1, ref) == capi.ERR_INVALID_ARG
    into = (keys, values, table, mass)
    assert lib.rcu_lazy_paged_evict(keys, values, table, lengths, mass, *into, 8, 2, 6, ref) == capi.OK and shape() == (I32, (3,))
    assert lib.rcu_lazy_paged_evict(keys, values, table, lengths, mass, *into, 8, 2, 7, ref) == capi.ERR_INVALID_ARG
    assert lib.rcu_lazy_paged_evict(keys, values, table, lengths, mass, *into, 0, 0, 0, ref) == capi.ERR_INVALID_ARG
    assert lib.rcu_lazy_paged_evict(keys, values, table, lengths, None, *into, 8, 2, 6, ref) == capi.ERR_INVALID_ARG
    freqs, at, x = leaf(F32, 2, 16), leaf(I32, 2, 5), leaf(F16, 5, 130)
    sec = lambda *s: (C.c_uint32 * len(s))(*s)  # noqa: E731
    axes = lambda col, heads, dim, first, positions, s: lib.rcu_lazy_rotary_axes(x, col, heads, dim, first, freqs, 1.0, positions, s, 0, ref)  # noqa: E731
    assert axes(2, 2, 64, 32, at, sec(10, 6)) == capi.OK and shape() == (F16, (5, 2, 64))
    assert axes(3, 2, 64, 32, at, sec(10, 6)) == capi.ERR_INVALID_ARG                  # past the rows' end
    assert axes(2, 2, 64, 33, at, sec(10, 6)) == capi.ERR_INVALID_ARG                  # past the head's
    assert axes(2, 2, 64, 0, at, sec(10, 5)) == capi.ERR_INVALID_ARG                   # a pair without an axis
    assert axes(2, 2, 64, 0, leaf(F32, 2, 5), sec(10, 6)) == capi.ERR_INVALID_ARG
    assert axes(2, 2, 64, 0, leaf(I32, 2, 4), sec(10, 6)) == capi.ERR_INVALID_ARG


def test_nodes_over_a_cache_run_in_the_order_in_which_they_were_built():
    """An eviction behind an attention whose weights it goes by, though it takes the lengths of the append before; an append behind both; not behind nodes over other
    pages, nor behind one that was released."""
    from ratchet_b200 import capi
    lib, F16, I32, F32 = capi.lib(), capi.F16, capi.I32, capi.F32
    room = iter(range(1, 1000))

    def leaf(dt, *shape):
        t = capi.describe(dt, shape, next(room) << 20)       # a place of its own: what overlaps is what the same tensor holds
        h = C.c_void_p()
        assert lib.rcu_lazy_wrap(None, C.byref(t), C.byref(h)) == capi.OK
        return h

    def order(node):
        n, ids = C.c_uint32(), (C.c_uint64 * 64)()
        assert lib.rcu_lazy_execution_order(node, ids, 64, C.byref(n)) == capi.OK
        return [ids[i] for i in range(n.value)]

    def made(call, *args):
        out = C.c_void_p()
        assert call(*args, C.byref(out)) == capi.OK
        return out

    ident = lib.rcu_lazy_id
    table, starts, lengths = leaf(I32, 3, 2), leaf(I32, 4), leaf(I32, 3)
    k, q = leaf(F16, 5, 128), leaf(F16, 5, 4, 64)
    caches = [(leaf(F16, 4, 2, 16, 64), leaf(F16, 4, 2, 16, 64), leaf(F32, 3, 2, 32)) for _ in range(2)]

    def append(c, lengths, mass=True):
        return made(lib.rcu_lazy_paged_append, k, 0, k, 0, c[0], c[1], table, starts, lengths, c[2] if mass else None)

    def attend(c, lengths, mass=True):
        return made(lib.rcu_lazy_paged_attention, q, c[0], c[1], table, starts, lengths, c[2] if mass else None, None, 0, 0, 0.1)

    def evict(c, lengths, into):
        return made(lib.rcu_lazy_paged_evict, c[0], c[1], table, lengths, c[2], into[0], into[1], table, into[2], 8, 2, 6)

    c, other = caches
    a = append(c, lengths)
    dropped = attend(c, a)
    gone = ident(dropped)
    lib.rcu_lazy_release(dropped)
    at = attend(c, a)
    plain = attend(c, a, mass=False)                         # reads pages alone
    elsewhere = append(other, lengths)
    e = evict(c, a, c)
    got = order(e)
    assert gone not in got and ident(elsewhere) not in got
    assert got[-1] == ident(e) and got.index(ident(a)) < got.index(ident(at)) and got.index(ident(a)) < got.index(ident(plain))
    # reading orders nothing: two attentions, one of them with sums, only come after the append
    assert ident(at) not in order(plain) and order(at)[-1] == ident(at)
    # a step later: an append behind the eviction and all before it, the next attention behind that; into other pages one that does not write the old ones
    a2 = append(c, e)
    at2 = attend(c, a2)
    assert [i for i in order(at2) if i in {ident(x) for x in (a, at, plain, e, a2, at2)}][-3:] == [ident(e), ident(a2), ident(at2)]
    e2 = evict(c, a2, other)
    assert {ident(at2), ident(elsewhere)} <= set(order(e2))
    # the same tensors through a view
    shape = (C.c_uint64 * 4)(4, 2, 16, 64)
    views = [made(lib.rcu_lazy_view, x, 4, shape) for x in c[:2]] + [c[2]]
    assert ident(at2) in order(evict(views, lengths, views))
    # a handle that goes away while a later node holds its node
    lib.rcu_lazy_release(at2)
    assert order(e2)[-1] == ident(e2)
    for h in (e2, a2, e, elsewhere, plain, at, a):
        lib.rcu_lazy_release(h)


# ---------------------------------------------------------------------------------------- handles
class Pool:
    """A device's part in a buffer's life."""

    def __init__(self):
        self.freed = []

    def _free(self, ptr):
        self.freed.append(ptr)


@pytest.mark.parametrize("name", ["keys", "values", "table", "lengths", "starts", "mass"])
@pytest.mark.parametrize("view", [False, True])
def test_a_cache_names_its_buffers_as_they_are(name, view):
    from ratchet_b200 import Buffer, PagedCache, RatchetCudaError, capi
    dev = Pool()
    shapes = {"keys": (4, 2, 16, 64), "values": (4, 2, 16, 64), "table": (2, 2), "lengths": (2,), "starts": (3,), "mass": (2, 2, 32)}
    types = {"keys": capi.F16, "values": capi.F16, "mass": capi.F32}
    made = {n: Buffer(dev, types.get(n, capi.I32), s, 0x1000 * (i + 1), 64, True) for i, (n, s) in enumerate(shapes.items())}
    c = PagedCache(**{n: b.view(b.shape) if view else b for n, b in made.items()})
    assert [getattr(c.struct, n).data for n in shapes] == [b.ptr for b in made.values()]
    assert c.ref is c.ref                                   # made once while nothing changes
    other = Buffer(dev, made[name].dt, made[name].shape, 0x9000, 64, True)
    kept = getattr(c, name)
    setattr(c, name, other)
    assert getattr(c.struct, name).data == 0x9000
    setattr(c, name, kept)
    assert getattr(c.struct, name).data == made[name].ptr
    c.ref
    made[name].free()
    for _ in range(2):
        with pytest.raises(RatchetCudaError):
            c.ref
    with pytest.raises(RatchetCudaError):
        c.struct
    setattr(c, name, other)
    assert getattr(c.struct, name).data == 0x9000
    with pytest.raises(RatchetCudaError):
        PagedCache(**{n: made.get(n) for n in shapes}).ref


def test_a_cache_knows_whose_view_it_has():
    """A view in the place of the buffer itself: the same address, but another's to free."""
    from ratchet_b200 import Buffer, PagedCache, RatchetCudaError, capi
    dev = Pool()
    keys, values, table, lengths = (Buffer(dev, t, s, 0x1000 * i, 64, True) for i, (t, s) in enumerate(((capi.F16, (4, 2, 16, 64)), (capi.F16, (4, 2, 16, 64)), (capi.I32, (2, 2)),
                                                                                                       (capi.I32, (2,))), 1))
    c = PagedCache(keys, values, table, lengths)
    c.ref
    c.keys = keys.view(keys.shape)
    assert c.struct.keys.data == 0x1000
    keys.free()
    with pytest.raises(RatchetCudaError):
        c.ref


def test_descriptors_say_what_their_buffers_do():
    """Calls keep a buffer's descriptor as long as its address, type and shape are the ones it has."""
    from ratchet_b200 import Buffer, PagedCache, capi
    from ratchet_b200.device import Device
    call = Device._ref                                      # what every call makes of a buffer
    b = Buffer(None, capi.F16, (4, 2, 16, 64), 0x1000, 64, False)
    rest = [Buffer(None, t, s, 0x2000, 64, False) for t, s in ((capi.F16, (4, 2, 16, 64)), (capi.I32, (2, 2)), (capi.I32, (2,)))]
    c = PagedCache(b, *rest)
    assert call(None, None) is None and call(None, b) is call(None, b) and c.ref is c.ref
    b.ptr = 0x5000
    assert call(None, b)._obj.data == 0x5000 == c.struct.keys.data
    b.shape = (8, 2, 16, 32)
    assert list(call(None, b)._obj.shape) == [8, 2, 16, 32] == list(c.struct.keys.shape)
    b.dt = capi.BF16
    assert call(None, b)._obj.dt == capi.BF16 == c.struct.keys.dt
    b.shape = [8, 2, 16, 32]
    call(None, b)
    b.shape[0] = 3
    assert call(None, b)._obj.shape[0] == 3


def test_a_cache_without_starts_and_sums():
    from ratchet_b200 import Buffer, PagedCache, capi
    b = lambda dt, *s: Buffer(None, dt, s, 0x1000, 64, False)  # noqa: E731
    c = PagedCache(b(capi.F16, 4, 2, 16, 64), b(capi.F16, 4, 2, 16, 64), b(capi.I32, 2, 2), b(capi.I32, 2))
    assert c.struct.starts.data is None and c.struct.mass.data is None and c.struct.keys.shape[1] == 2


# ---------------------------------------------------------------------------------------- notes of values that are not finite
class Meeting:
    def __init__(self, count):
        self.count, self.arrived, self.phase = count, 0, 0

    def arrive(self):
        self.arrived += 1
        if self.arrived == self.count:
            self.arrived, self.phase = 0, self.phase + 1


def group_of_warps(seed, notes, segments=40, warps=4):
    """The softmax warps of one query tile (paged_attention_tc.cu) as far as their notes go, each as far as its waits let it, in an order drawn from `seed`:
    the number of segments for which a warp read another note than what the tile's warps wrote of that segment, and whether all ended.
    notes 0: one note, which the warps take back at two further meetings where it is set."""
    import random
    r = random.Random(seed)
    bad = [[r.random() < 0.15 for _ in range(warps)] for _ in range(segments)]
    idle = [r.random() < 0.5 for _ in range(warps)]                       # warps without a query do nothing between the meetings
    note, met, wrong = [False] * max(1, notes), Meeting(warps), [0]

    def warp(w):
        phase = 0
        for i in range(segments):
            at = i % notes if notes else 0
            yield
            if bad[i][w]:
                note[at] = True
            yield
            met.arrive()
            phase += 1
            while met.phase < phase:
                yield
            if notes:
                yield
                note[(at - 1) % notes] = False
            yield
            got = note[at]
            wrong[0] += got != any(bad[i])
            if not notes and got:
                for k in range(2):
                    met.arrive()
                    phase += 1
                    while met.phase < phase:
                        yield
                    if k == 0:
                        note[0] = False
            for _ in range(0 if idle[w] else r.randrange(12)):            # sums to the output, or row by row
                yield

    running = [warp(w) for w in range(warps)]
    for _ in range(40000):
        if not running:
            return wrong[0], True
        g = r.choice(running)
        if next(g, running) is running:
            running.remove(g)
    return wrong[0], False


def test_every_warp_reads_what_its_segment_noted():
    import re
    from pathlib import Path
    source = (Path(__file__).resolve().parent.parent / "ratchet_b200" / "csrc" / "paged_attention_tc.cu").read_text()
    notes = int(re.search(r"constexpr int kNotes = (\d+);", source).group(1))
    assert re.search(r"poison\[w\]\[note == 0 \? kNotes - 1 : note - 1\] = 0;", source) and "poison[2][kNotes]" in source
    assert all(group_of_warps(seed, notes) == (0, True) for seed in range(300))
    # the model finds what fewer notes do: one read for the wrong segment, warps that wait for one another for good
    assert any(group_of_warps(seed, 2)[0] for seed in range(300))
    assert any(not group_of_warps(seed, 0)[1] for seed in range(300))
