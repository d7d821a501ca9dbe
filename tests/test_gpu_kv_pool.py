"""GPU tests of wpcg_kv_fork, wpcg_kv_compact and wpcg_kv_copy against a host pool
that goes entry by entry (pool_ref.py): random lives of sequences, with the tokens
that their pages hold followed through every copy; borders of pages, rows and
blocks; windows; pools that run out; arrays that hold anything; graphs."""
import numpy as np
import pytest

import serve_ref as R
import wpcg
from pool_ref import Pool
from serve_ref import BF16, E4M3, F32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


class Device:
    """A host pool's twin on the device."""

    def __init__(self, ctx, ref, layers=(), max_moves=None):
        self.ctx, self.ref, self.layers = ctx, ref, list(layers)
        n = ref.n_seq
        self.pool = wpcg.KvPool(ctx, ref.n_pages, ref.page, n, ref.stride)
        self.max_moves = ref.n_pages if max_moves is None else max_moves
        room = max(n, self.max_moves, 1)
        self.copies = ctx.upload(np.full(3 * room + 3, -9, np.int32))
        self.room = room
        self.result = ctx.alloc(8)
        self.args = {k: ctx.alloc(4 * max(1, n)) for k in ("parent", "keep", "grow")}
        self.push()

    def push(self):
        self.pool.refs.write(self.ref.refs)
        if self.ref.n_seq:
            self.pool.table.write(self.ref.table)
            self.pool.kv_len.write(self.ref.kv_len)

    def _copied(self, copies, result, limit):
        self.ctx.sync()
        assert tuple(self.result.read(np.int32, 2)) == result
        got = self.copies.read(np.int32, 3 * self.room + 3)
        assert np.array_equal(got[:3 * len(copies)], np.array(copies, np.int32).ravel()), (got[:30], copies[:10])
        assert (got[3 * limit:] == -9).all() or limit == self.room
        assert (got[3 * self.room:] == -9).all()
        self.same()

    def same(self):
        r = self.ref
        assert np.array_equal(self.pool.refs.read(np.int32, r.n_pages), r.refs)
        if r.n_seq:
            assert np.array_equal(self.pool.table.read(np.int32, r.table.size).reshape(r.table.shape), r.table)
            assert np.array_equal(self.pool.kv_len.read(np.int32, r.n_seq), r.kv_len)

    def fork(self, parent=None, keep=None, grow=0, window=0, sinks=0, via=None):
        kw, stream = {}, None if via is None else via.stream
        for name, v in (("parent", parent), ("keep", keep), ("grow", None if np.isscalar(grow) else grow)):
            if v is not None:
                self.args[name].write(np.asarray(v, np.int32))
                kw[name + ("_each" if name == "grow" else "")] = self.args[name]
        self.copies.write(np.full(3 * self.room + 3, -9, np.int32))
        op = wpcg.KvFork(self.ctx, self.pool, self.copies, self.result, grow=int(grow) if np.isscalar(grow) else 0,
                         window=window, sinks=sinks, **kw)
        op.workspace.write(np.full(op.workspace_bytes, 0xFF, np.uint8))
        op.run(stream)
        if self.layers:
            wpcg.KvCopy(self.ctx, self.layers, self.copies, self.result, self.ref.n_seq).run(stream)
        if via is not None:
            via.sync()
        want = self.ref.fork(parent, keep, grow, window, sinks)
        self._copied(*want, self.ref.n_seq)
        return want

    def compact(self, most=None):
        most = self.max_moves if most is None else most
        self.copies.write(np.full(3 * self.room + 3, -9, np.int32))
        op = wpcg.KvCompact(self.ctx, self.pool, self.copies, self.result, most)
        op.workspace.write(np.full(op.workspace_bytes, 0xFF, np.uint8))
        op.run()
        if self.layers:
            wpcg.KvCopy(self.ctx, self.layers, self.copies, self.result, most).run()
        want = self.ref.compact(most)
        self._copied(*want, most)
        return want


class Cache:
    """Pages of some layers on the device whose every token is told apart by its
    values, and what the host knows each sequence to hold."""

    def __init__(self, ctx, ref, n_layers, hkv, d, dtype, order):
        self.ctx, self.ref, self.dtype, self.hkv, self.d = ctx, ref, dtype, hkv, d
        if order == "head":
            self.st, strides = (hkv * ref.page * d, ref.page * d, d), None
        else:
            pad = 16
            tok = hkv * (d + pad)
            self.st = strides = (ref.page * tok + 32, d + pad, tok)
        self.elems = ref.n_pages * self.st[0]
        self.buf = [[ctx.upload(np.zeros(self.elems, R.BITS[dtype])) for _ in "kv"] for _ in range(n_layers)]
        self.layers = [wpcg.PagedKv(ctx, ref.n_pages, ref.page, hkv, d, dtype, k=k, v=v, strides=strides)
                       for k, v in self.buf]
        self.told = [[] for _ in range(ref.n_seq)]  # a number for every token
        self.next = 1

    def words(self, layer, side, number):
        """[token][head][d] bits of numbered tokens."""
        x = (np.asarray(number, np.uint64)[:, None, None] * 2654435761 + layer * 40503 + side * 977
             + np.arange(self.hkv, dtype=np.uint64)[:, None] * 131 + np.arange(self.d, dtype=np.uint64))
        return (x >> 5).astype(R.BITS[self.dtype])

    def index(self, s, tokens):
        t = np.asarray(tokens, np.int64)
        page = self.ref.table[s, t // self.ref.page].astype(np.int64)
        return ((page * self.st[0] + t % self.ref.page * self.st[2])[:, None, None]
                + np.arange(self.hkv)[:, None] * self.st[1] + np.arange(self.d))

    def check_and_write(self, parent, keep, shown=None):
        """After a call: every sequence holds what it took over; new tokens are
        written where it grew, as an append does. shown: tokens still held."""
        ref = self.ref
        old = [list(t) for t in self.told]
        host = [[b.read(R.BITS[self.dtype], self.elems) for b in kv] for kv in self.buf]
        new = []
        for s in range(ref.n_seq):
            p = s if parent is None else int(parent[s])
            has = old[p] if 0 <= p < ref.n_seq else []
            kept = has[:len(has) if keep is None else max(0, int(keep[s]))]
            grown = int(ref.kv_len[s]) - len(kept)
            self.told[s] = kept + list(range(self.next, self.next + grown))
            self.next += grown
            new.append(len(kept))
        for s in range(ref.n_seq):
            t = [i for i in range(new[s]) if shown is None or shown(s, i)]
            if t:
                at = self.index(s, t)
                for layer, kv in enumerate(host):
                    for side, x in enumerate(kv):
                        assert np.array_equal(x[at], self.words(layer, side, [self.told[s][i] for i in t])), (s, layer)
        for s in range(ref.n_seq):
            t = np.arange(new[s], len(self.told[s]))
            if len(t):
                assert (ref.refs[ref.table[s, t // ref.page]] == 1).all()  # written pages are its own
                at = self.index(s, t)
                for layer, kv in enumerate(host):
                    for side, x in enumerate(kv):
                        x[at] = self.words(layer, side, [self.told[s][i] for i in t])
        for kv, x in zip(self.buf, host):
            for b, w in zip(kv, x):
                b.write(w)


@pytest.mark.parametrize("stride", [7, 1100])
@pytest.mark.parametrize("dtype,hkv,d,page,order,n_layers", [
    (BF16, 2, 128, 16, "head", 3), (F32, 1, 64, 32, "token", 2), (E4M3, 3, 64, 16, "token", 2), (E4M3, 2, 128, 64, "head", 1),
    (F32, 2, 128, 16, "head", 2), (BF16, 1, 64, 256, "token", 70)])
def test_lives_of_sequences(ctx, dtype, hkv, d, page, order, n_layers, stride):
    """Begun, grown, forked, cut back, ended and moved together at random, with
    the tokens followed; rows short enough for one workgroup, and long ones."""
    print(f"[gpu] pool lives {dtype} {hkv}x{d} page {page} layers {n_layers}", flush=True)
    rng = np.random.default_rng(page + d + dtype)
    n = 6
    ref = Pool(40, page, n, stride)
    cache = Cache(ctx, ref, n_layers, hkv, d, dtype, order)
    dev = Device(ctx, ref, cache.layers)
    shortages = 0
    for turn in range(24 if n_layers < 10 else 8):
        if turn % 5 == 4:
            most = [None, 1, 3][turn // 5 % 3]
            dev.compact(most)
            cache.check_and_write(None, None)
            continue
        parent = rng.integers(-1, n, n) if turn % 3 == 2 else None
        keep = None if rng.random() < 0.4 else rng.integers(0, 6 * page, n)
        if keep is not None:
            has = [0 if parent is not None and parent[s] < 0 else int(ref.kv_len[s if parent is None else parent[s]])
                   for s in range(n)]
            keep = np.minimum(keep, has)
        grow = rng.integers(0, 3 * page, n)
        grow = np.minimum(grow, [7 * page - (int(ref.kv_len[s if parent is None else max(0, parent[s])]) if keep is None
                                             else int(keep[s])) for s in range(n)])
        _, result = dev.fork(parent, keep, grow)
        if result[0] < 0:
            shortages += 1
            assert dev.fork(None, None, 0)[1][0] >= 0  # all as it was
            cache.check_and_write(None, None)
        else:
            cache.check_and_write(parent, keep)
    assert shortages < 12


@pytest.mark.parametrize("keep", [0, 1, 15, 16, 17, 31, 32, 33, 47])
@pytest.mark.parametrize("grow,stride", [(0, 5), (1, 5), (2, 5), (16, 5), (17, 5), (1, 1100), (17, 1100)])
def test_many_from_one(ctx, keep, grow, stride):
    """All rows from row 0, which is not or is itself among them; the tail is
    copied for all but one, and not at all where nothing is written or it is full."""
    ref = Pool(60, 16, 9, stride)
    dev = Device(ctx, ref)
    first = np.zeros(9, np.int32)
    first[0] = 47
    dev.fork(grow=first)
    copies, _ = dev.fork(np.zeros(9, int), np.full(9, keep), grow)
    assert len(copies) == (8 if keep % 16 and grow else 0)
    dev.fork([-1, 5, 5, 5, 8, -1, 77, 1, -5], None, grow)
    dev.fork([-1] * 9)
    assert (ref.refs == 0).all() and (ref.table == -1).all()


def test_different_lengths_from_one_row(ctx):
    """One child writes into a page that another holds whole: the writer copies,
    though it comes first; without a holder the first writer keeps the page."""
    ref = Pool(30, 16, 4, 4)
    dev = Device(ctx, ref)
    dev.fork(grow=[60, 0, 0, 0])
    page = int(ref.table[0, 0])
    copies, _ = dev.fork([0, 0, 0, -1], [5, 40, 7, 0], 3)
    assert [c[2] for c in copies] == [5, 7] and {c[0] for c in copies} == {page}
    copies, _ = dev.fork([1, 1, -1, -1], [5, 9, 0, 0], 1)
    assert [c[2] for c in copies] == [9] and ref.table[0, 0] == page


def test_a_page_held_by_the_host(ctx):
    """The host's own count keeps a page from being written into and from being freed."""
    ref = Pool(20, 32, 2, 3)
    dev = Device(ctx, ref)
    dev.fork(grow=[40, 0])
    page = int(ref.table[0, 1])
    ref.refs[page] += 1
    dev.push()
    copies, _ = dev.fork(None, None, 4)
    assert copies == [(page, int(ref.table[0, 1]), 8)] and ref.refs[page] == 1
    dev.fork([-1, -1])
    assert ref.refs.sum() == 1
    copies, result = dev.compact()
    assert copies == ([(page, 0, 32)] if page else []) and result[0] == 1


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 0), (33, 5), (40, 16), (40, 17), (100, 3), (5, 200)])
@pytest.mark.parametrize("stride", [12, 1100])
def test_windows(ctx, window, sinks, stride):
    """Pages go free as the window moves on, token by token and in jumps; forked
    rows with holes; the tokens that rows see are all there."""
    ref = Pool(64, 16, 4, stride)
    cache = Cache(ctx, ref, 1, 1, 64, BF16, "head")
    dev = Device(ctx, ref, cache.layers)
    lo = [0] * 4

    def shown(s, i):  # what rows from the kept length on see
        return i > lo[s] - window or i < sinks
    rng = np.random.default_rng(window + sinks)
    for turn in range(14):
        parent = rng.integers(0, 4, 4) if turn % 4 == 3 else None
        grow = rng.integers(1, 30, 4) if turn % 2 else np.ones(4, int)
        grow = np.minimum(grow, 12 * 16 - np.array([int(ref.kv_len[s if parent is None else parent[s]]) for s in range(4)]))
        keep = [int(ref.kv_len[s if parent is None else parent[s]]) for s in range(4)]
        _, result = dev.fork(parent, None, grow, window, sinks)
        assert result[0] >= 0
        lo = keep
        cache.check_and_write(parent, None, shown)
    if window < 100 and sinks < 100:
        assert (ref.table[:, 1:3] == -1).any()


@pytest.mark.parametrize("stride", [8, 1100])
def test_running_out_and_just_enough(ctx, stride):
    """One page missing: nothing changes and none is copied; the pages that the
    call itself frees are enough for it."""
    ref = Pool(8, 16, 3, stride)
    dev = Device(ctx, ref)
    dev.fork(grow=[40, 50, 10])
    assert (ref.refs > 0).sum() == 8
    assert dev.fork(None, None, [0, 15, 0])[1] == (-1, 0)
    assert dev.fork(None, None, [8, 14, 6])[1] == (0, 0)
    assert dev.fork([0, -1, 0], [33, 0, 33], [2, 0, 2])[1] == (4, 1)
    assert dev.fork([-1] * 3, None, 42)[1] == (-1, 0)
    assert dev.fork([-1] * 3, None, [41, 32, 48])[1] == (0, 0)


@pytest.mark.parametrize("n_pages,n,stride", [(1, 1, 1), (4095, 3, 1023), (4096, 2, 1024), (4097, 2, 1025), (9000, 2100, 3),
                                              (20000, 5, 3000), (300000, 1025, 2), (8192, 64, 128), (8193, 64, 128),
                                              (2000, 65, 32), (4096, 33, 129), (3000, 32, 256), (900, 10, 512), (100, 17, 7)])
def test_sizes_of_pools(ctx, n_pages, n, stride):
    """Around the blocks of pages, of a row's entries and of sequences."""
    print(f"[gpu] pool of {n_pages} pages, {n} sequences of {stride}", flush=True)
    rng = np.random.default_rng(n_pages + n)
    ref = Pool(n_pages, 16, n, stride)
    ref.refs[rng.random(n_pages) < 0.3] = 1  # the host's
    dev = Device(ctx, ref, max_moves=n_pages)
    free = int((ref.refs == 0).sum())
    dev.fork(grow=np.minimum(rng.integers(0, max(2, 2 * 16 * free // n // 3), n), 16 * stride))
    for _ in range(3):
        parent = np.where(rng.random(n) < 0.3, rng.integers(-1, n, n), np.arange(n))
        dev.fork(parent, None, 3)
    dev.compact(min(100, n_pages))
    dev.compact()
    assert dev.compact()[1][1] == 0
    dev.fork(np.full(n, -1))


@pytest.mark.parametrize("stride", [5, 1100])
def test_arrays_that_hold_anything(ctx, stride):
    """Ids of no page, lengths that are none, parents and keeps out of range:
    nothing is touched outside the arrays, and the sequences beside them are right."""
    rng = np.random.default_rng(3)
    for turn in range(20):
        ref = Pool(50, 16, 8, stride)
        ref.table[:] = rng.integers(-4, 54, ref.table.shape)
        ref.table[rng.random(ref.table.shape) < 0.1] = 2 ** 31 - 1
        ref.kv_len[:] = rng.choice([-5, 0, 3, 16, 33, 79, 80, 81, 2 ** 31 - 1, -2 ** 31], 8)
        entries = [i for s in range(8) for i in ref._entries(s, ref._pages(ref._length(s))) if i >= 0]
        ref.refs[:] = np.bincount(entries, minlength=50)
        dev = Device(ctx, ref)
        parent = rng.choice([-2 ** 31, -1, 0, 3, 7, 8, 2 ** 31 - 1, 5], 8)
        dev.fork(parent, rng.choice([-7, 0, 5, 20, 80, 2 ** 31 - 1], 8), rng.choice([-3, 0, 1, 20, 2 ** 31 - 1], 8))
        dev.compact(int(rng.integers(0, 50)))
        dev.fork(None, None, 2 ** 31)


def test_copies_that_hold_anything(ctx):
    """Ids outside the pages and numbers of tokens that are none are passed over;
    no more than max_copies are read."""
    ref = Pool(10, 16, 1, 1)
    rng = np.random.default_rng(4)
    x = rng.integers(0, 1 << 16, 10 * 16 * 64).astype(np.uint16)
    k, v = ctx.upload(x), ctx.upload(x + 1)
    kv = wpcg.PagedKv(ctx, 10, 16, 1, 64, BF16, k=k, v=v)
    copies = np.array([[0, 5, 16], [-1, 6, 16], [1, 10, 16], [2 ** 31 - 1, 6, 3], [1, 6, -5], [2, 7, 99], [3, 8, 0], [3, 9, 7],
                       [4, 1, 16]], np.int32)
    for n, most in ((9, 8), (-3, 9), (0, 9), (2 ** 31 - 1, 8), (3, 9)):
        k.write(x)
        v.write(x + 1)
        wpcg.KvCopy(ctx, [kv], ctx.upload(copies), ctx.upload(np.array([0, n], np.int32)), most).run()
        ctx.sync()
        want = x.reshape(10, 16, 64).copy()
        for a, b, t in copies[:max(0, min(n, most))]:
            if 0 <= a < 10 and 0 <= b < 10:
                want[b, :max(0, min(t, 16))] = want[a, :max(0, min(t, 16))]
        assert np.array_equal(k.read(np.uint16, x.size), want.ravel())
        assert np.array_equal(v.read(np.uint16, x.size), want.ravel() + 1)


def test_no_sequences(ctx):
    ref = Pool(70, 16, 0, 1)
    ref.refs[[3, 50]] = 1
    dev = Device(ctx, ref)
    assert dev.fork()[1] == (68, 0)
    copies, _ = dev.compact()
    assert copies == [(50, 0, 16), (3, 1, 16)]


def test_graphs_and_streams(ctx):
    """A captured step (fork, then the copies) replayed with other parents, the
    host's own calls between; two pools' graphs in turn; another stream."""
    print("[gpu] pool graphs", flush=True)
    rng = np.random.default_rng(12)
    twins = []
    for n, pages, stride in ((6, 60, 6), (3, 30, 1100)):
        ref = Pool(pages, 16, n, stride)
        cache = Cache(ctx, ref, 2, 2, 64, BF16, "head")
        dev = Device(ctx, ref, cache.layers)
        dev.fork(grow=rng.integers(1, 40, n))
        cache.check_and_write(None, None)
        op = wpcg.KvFork(ctx, dev.pool, dev.copies, dev.result, parent=dev.args["parent"], keep=dev.args["keep"], grow=1)
        copy = wpcg.KvCopy(ctx, cache.layers, dev.copies, dev.result, n)

        def both(op=op, copy=copy):
            op.run()
            copy.run()
        twins.append((ref, cache, dev, ctx.capture(both), (op, copy)))
    for turn in range(6):
        made = []
        for ref, cache, dev, graph, _ in twins:
            parent = rng.integers(0, ref.n_seq, ref.n_seq)
            keep = np.array([rng.integers(1, int(ref.kv_len[p]) + 1) for p in parent])
            dev.args["parent"].write(parent.astype(np.int32))
            dev.args["keep"].write(keep.astype(np.int32))
            dev.copies.write(np.full(3 * dev.room + 3, -9, np.int32))
            graph.launch()
            made.append((parent, keep))
        for (ref, cache, dev, _, _), (parent, keep) in zip(twins, made):
            want = ref.fork(parent, keep, 1)
            dev._copied(*want, ref.n_seq)
            cache.check_and_write(parent, keep)
            if turn == 3:
                dev.compact()
                cache.check_and_write(None, None)
    other = wpcg.Context(0)
    ref, cache, dev = twins[0][:3]
    ctx.sync()
    dev.fork([0, 0, 1, 1, 2, 2], None, 2, via=other)
    cache.check_and_write([0, 0, 1, 1, 2, 2], None)
    other.close()
