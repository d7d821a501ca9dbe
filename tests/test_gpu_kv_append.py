"""GPU tests of wpcg_kv_append against a plain 64-bit implementation: types,
head sizes, pages' orders, far positions, rows without norm, rotation or
queries, in place, clamped and not finite 8-bit values, rows and pages that
nothing is stored for."""
import numpy as np
import pytest

import serve_ref as R
import wpcg
from serve_ref import BF16, E4M3, F32

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


def bound(want, mag, dtype):
    """fp32 arithmetic: the mean of the squares (a tree over d values, each
    step half a step), square root, division, two products and the rotation's
    two products and sum on values of at most mag, sine and cosine to 3e-7;
    then the type's own rounding (E4M3: a step of 2^-9 near 0 too)."""
    e = mag * (40 * 2.0 ** -24 + 6e-7)
    return e + (np.abs(want) + e) * R.HALF[dtype] + (2.0 ** -10 if dtype == E4M3 else 0)


def inputs(rng, rows, heads, hkv, d, dtype):
    return [R.encode(rng.standard_normal((rows, h, d)) * 3, dtype) for h in (heads, hkv, hkv)]


def near(got, want, lim):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want) - lim
    assert not (off > 0).any(), (np.nanmax(off), int((off > 0).sum()), off.size)


def magnitude(y):
    h = y.shape[-1] // 2
    m = np.hypot(y[..., :h], y[..., h:])
    return np.concatenate([m, m], -1)


@pytest.mark.parametrize("d,heads,hkv", [(128, 32, 4), (64, 14, 2), (128, 5, 5), (64, 1, 1)])
@pytest.mark.parametrize("dtype,q_dtype,cache", [(F32, F32, F32), (F32, BF16, BF16), (F32, F32, E4M3),
                                                 (BF16, BF16, E4M3), (BF16, F32, BF16)])
@pytest.mark.parametrize("order", ["head", "token"])
def test_append(ctx, d, heads, hkv, dtype, q_dtype, cache, order):
    print(f"[gpu] append {heads}/{hkv}x{d} {dtype}->{q_dtype},{cache} {order}", flush=True)
    rng = np.random.default_rng(d + heads + dtype + 10 * q_dtype + 100 * cache)
    rows, lens = [3, 1, 40, 1], [3, 30, 75, 1]
    pg = R.Paged(ctx, rng, cache, hkv, d, 32, lens, order=order, scales=cache == E4M3).upload()
    before = {n: pg.bits[n].copy() for n in "kv"}
    total = sum(rows)
    q, k, v = inputs(rng, total, heads, hkv, d, dtype)
    qn, kn = (1 + 0.2 * rng.standard_normal((2, d))).astype(np.float32)
    freq = wpcg.rope_frequencies(1e4, d)
    out = ctx.upload(np.full(total * heads * d * R.SIZE[q_dtype], 0x5A, np.uint8))
    dev = [ctx.upload(a) for a in (q, k, v, qn, kn, freq)]
    op = wpcg.KvAppend(ctx, pg.kv, pg.batch(rows), heads, dtype, q_dtype, q_norm=dev[3], k_norm=dev[4], eps=EPS,
                       frequencies=dev[5])
    op.run(*dev[:3], out)
    ctx.sync()
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(rows, lens)])
    y = R.normed_turned(R.decode(q, dtype), qn, EPS, pos, freq)
    near(R.decode(out.read(R.BITS[q_dtype], q.size).reshape(q.shape), q_dtype), y, bound(y, magnitude(y), q_dtype))
    at = 0
    touched = {n: np.zeros(pg.bits[n].size, bool) for n in "kv"}
    for name, dev_pages, x in (("k", pg.dk, R.normed_turned(R.decode(k, dtype), kn, EPS, pos, freq)),
                               ("v", pg.dv, R.decode(v, dtype))):
        bits = dev_pages.read(R.BITS[cache], pg.bits[name].size)
        at = 0
        for s, n in enumerate(rows):
            where = pg.index(s, np.arange(lens[s] - n, lens[s]))
            touched[name][where] = True
            w = x[at:at + n] / pg.scale[name][:, None]
            lim = np.clip(w, -448, 448) if cache == E4M3 else w
            near(R.decode(bits[where], cache), lim, bound(lim, magnitude(w) if name == "k" else np.abs(w), cache))
            at += n
        assert np.array_equal(bits[~touched[name]], before[name][~touched[name]])  # nothing else is written


def test_far_positions_and_exact_values_without_a_norm(ctx):
    """Positions of a hundred million: the angle needs 64 bits. Values and,
    without a rotation, keys and queries come through unchanged."""
    d, page = 64, 256
    rng = np.random.default_rng(3)
    far = 100_000_007
    blocks = -(-far // page)
    table = np.zeros((1, blocks), np.int32)
    table[0, -1] = 1
    kb, vb = ctx.alloc(2 * page * d * 4), ctx.alloc(2 * page * d * 4)
    kv = wpcg.PagedKv(ctx, 2, page, 1, d, F32, k=kb, v=vb)
    dl, dt, ds = ctx.upload(np.array([far], np.int32)), ctx.upload(table), ctx.upload(np.array([0, 3], np.int32))
    batch = wpcg.KvBatch(1, 3, dl, dt, blocks, far, max_q=3, q_start=ds)
    q, k, v = inputs(rng, 3, 2, 1, d, F32)
    freq = wpcg.rope_frequencies(1e6, d)
    dev = [ctx.upload(a) for a in (q, k, v, freq)]
    out = ctx.alloc(q.nbytes)
    wpcg.KvAppend(ctx, kv, batch, 2, F32, F32, frequencies=dev[3]).run(*dev[:3], out)
    ctx.sync()
    pos = np.arange(far - 3, far)
    y = R.normed_turned(R.decode(q, F32), None, 0, pos, freq)
    near(R.decode(out.read(np.uint32, q.size).reshape(q.shape), F32), y, bound(y, magnitude(y), F32))
    slot = pos % page
    assert np.array_equal(vb.read(np.uint32, 2 * page * d).reshape(2, page, d)[1, slot], v[:, 0])
    wpcg.KvAppend(ctx, kv, batch, 2, F32, F32).run(*dev[:3], out)
    ctx.sync()
    assert np.array_equal(out.read(np.uint32, q.size).reshape(q.shape), q)
    assert np.array_equal(kb.read(np.uint32, 2 * page * d).reshape(2, page, d)[1, slot], k[:, 0])


def test_in_place_without_queries_and_strided(ctx):
    rng = np.random.default_rng(8)
    d, heads, hkv, rows, lens = 128, 4, 2, [5, 2], [9, 2]
    width = (heads + 2 * hkv) * d + 8  # one projection's rows: q, k, v side by side
    x = R.encode(rng.standard_normal((7, width)), F32)
    freq = wpcg.rope_frequencies(1e4, d)
    fd = ctx.upload(freq)

    class At:
        def __init__(self, b, elements):
            self.ptr = b.ptr.value + 4 * elements

    outs = []
    for with_q in (True, False):
        pg = R.Paged(ctx, np.random.default_rng(1), BF16, hkv, d, 16, lens).upload()
        xd = ctx.upload(x)
        op = wpcg.KvAppend(ctx, pg.kv, pg.batch(rows), heads, F32, F32, frequencies=fd, q_stride=width, k_stride=width,
                           v_stride=width, q_out_stride=width)
        q = At(xd, 0) if with_q else None
        op.run(q, At(xd, heads * d), At(xd, (heads + hkv) * d), q)
        ctx.sync()
        got = xd.read(np.uint32, x.size).reshape(x.shape)
        assert np.array_equal(got[:, heads * d:], x[:, heads * d:])
        if with_q:
            pos = np.concatenate([np.arange(m - n, m) for n, m in zip(rows, lens)])
            y = R.normed_turned(R.decode(np.ascontiguousarray(x[:, :heads * d]), F32).reshape(7, heads, d), None, 0,
                                pos, freq)
            near(R.decode(np.ascontiguousarray(got[:, :heads * d]), F32).reshape(7, heads, d), y,
                 bound(y, magnitude(y), F32))
        else:
            assert np.array_equal(got, x)
        outs.append((pg.dk.read(np.uint16, pg.bits["k"].size), pg.dv.read(np.uint16, pg.bits["v"].size)))
    assert all(np.array_equal(a, b) for a, b in zip(*outs))


def test_e4m3_range_and_not_finite(ctx):
    """Beyond the range: its largest value; NaN stays; ties go to even."""
    rng = np.random.default_rng(5)
    d = 64
    pg = R.Paged(ctx, rng, E4M3, 1, d, 16, [1]).upload()
    v = np.zeros((1, 1, d), np.float32)
    odd = [1e9, -1e9, np.inf, -np.inf, np.nan, 448, 464, 465, 17, 19, 2.0 ** -10, 1.5 * 2.0 ** -9, 2.0 ** -11, -0.0]
    v[0, 0, :len(odd)] = odd
    k = np.ones_like(v)
    op = wpcg.KvAppend(ctx, pg.kv, pg.batch(None), 1, F32)
    op.run(None, ctx.upload(k), ctx.upload(v), None)
    ctx.sync()
    got = pg.dv.read(np.uint8, pg.bits["v"].size)[pg.index(0, [0])]
    want = R.encode(v, E4M3)
    nan = np.isnan(v)
    assert np.array_equal(got[~nan], want[~nan])
    assert np.isnan(R.decode(got[nan], E4M3)).all()


def test_rows_and_pages_that_are_none(ctx):
    rng = np.random.default_rng(6)
    d, heads = 64, 2
    lens, rows = [20, 20, 20, 1, 20], [2, 2, 2, 3, 2]
    pg = R.Paged(ctx, rng, BF16, 1, d, 16, lens).upload()
    good = pg.table.copy()
    pg.table[1, 1] = pg.n_pages
    pg.kv_len = [20, 20, 33, 1, 20]  # sequence 2 longer than max_kv; 3 has rows before its first token
    batch = pg.batch(rows, n_rows=14, max_kv=20)
    before = {n: pg.bits[n].copy() for n in "kv"}
    q, k, v = inputs(rng, 14, heads, 1, d, F32)
    out = ctx.upload(np.full(q.shape, 0x5A5A5A5A, np.uint32))
    wpcg.KvAppend(ctx, pg.kv, batch, heads, F32, F32).run(ctx.upload(q), ctx.upload(k), ctx.upload(v), out)
    ctx.sync()
    got = out.read(np.uint32, q.size).reshape(q.shape)
    for r in (0, 1, 8, 9, 10):
        assert np.array_equal(got[r], q[r]), r
    for r in (2, 3, 4, 5):
        assert np.isnan(got[r].view(np.float32)).all(), r
    for r in (6, 7, 11, 12, 13):  # before position 0, or of no sequence
        assert (got[r] == 0x5A5A5A5A).all(), r
    pg.table = good
    bits = pg.dv.read(np.uint16, pg.bits["v"].size)
    touched = np.zeros(bits.size, bool)
    for s, toks in ((0, [18, 19]), (3, [0]), (4, [18, 19])):
        touched[pg.index(s, toks)] = True
    assert np.array_equal(bits[~touched], before["v"][~touched])
    assert np.array_equal(bits[pg.index(3, [0])][0], R.encode(v[8].view(np.float32), BF16))


def test_captured(ctx):
    """A graph replayed as the sequence grows."""
    rng = np.random.default_rng(7)
    d = 64
    pg = R.Paged(ctx, rng, F32, 2, d, 16, [40]).upload()
    batch = pg.batch(None)
    q, k, v = inputs(rng, 1, 4, 2, d, F32)
    dev = [ctx.upload(a) for a in (q, k, v)]
    out = ctx.alloc(q.nbytes)
    op = wpcg.KvAppend(ctx, pg.kv, batch, 4, F32, F32)
    g = ctx.capture(lambda: op.run(*dev, out))
    for n in (1, 17, 40, 40):
        pg.d_len.write(np.array([n], np.int32))
        v = R.encode(rng.standard_normal(v.shape), F32)
        dev[2].write(v)
        g.launch()
        ctx.sync()
        got = pg.dv.read(np.uint32, pg.bits["v"].size)
        assert np.array_equal(got[pg.index(0, [n - 1])], v)
    del g


def test_other_streams(ctx):
    """Two batches of one layer's pages stored on streams of other contexts, at once."""
    rng = np.random.default_rng(10)
    d, lens = 128, [40, 25]
    pg = R.Paged(ctx, rng, BF16, 2, d, 16, lens).upload()
    others = [wpcg.Context(0) for _ in range(2)]
    runs, keep = [], []
    for s in range(2):  # all of a sequence's tokens
        q, k, v = inputs(rng, lens[s], 4, 2, d, BF16)
        dev = [ctx.upload(a) for a in (q, k, v)]
        arrays = [ctx.upload(np.array(a, np.int32)) for a in ([0, lens[s]], [lens[s]], pg.table[s])]
        batch = wpcg.KvBatch(1, lens[s], arrays[1], arrays[2], pg.table.shape[1], lens[s], max_q=lens[s],
                             q_start=arrays[0])
        runs.append((wpcg.KvAppend(ctx, pg.kv, batch, 4, BF16, BF16), dev, ctx.alloc(q.nbytes)))
        keep.append((k, v, arrays))
    for _ in range(20):
        for o, (op, dev, out) in zip(others, runs):
            op.run(*dev, out, stream=o.stream)
    for o in others:
        o.sync()
        o.close()
    for n, x in (("k", pg.dk), ("v", pg.dv)):
        got = x.read(np.uint16, pg.bits[n].size)
        for s in range(2):
            assert np.array_equal(got[pg.index(s, np.arange(lens[s]))], keep[s][0 if n == "k" else 1])


@pytest.mark.parametrize("n", [64, 65, 130, 4500])
def test_many_sequences(ctx, n):
    """A row's sequence is looked for in one, two and three steps; sequences
    without rows between, rows behind the last."""
    rng = np.random.default_rng(n)
    rows = rng.integers(0, 4, n)
    rows[0], rows[n - 1] = 0, 2
    lens = [int(r) + int(x) for r, x in zip(rows, rng.integers(0, 20, n))]
    pg = R.Paged(ctx, rng, F32, 1, 64, 16, lens).upload()
    total = int(rows.sum())
    batch = pg.batch(list(rows), n_rows=total + 3)
    k, v = (R.encode(rng.standard_normal((total + 3, 1, 64)), F32) for _ in range(2))
    op = wpcg.KvAppend(ctx, pg.kv, batch, 0, F32)
    op.run(None, ctx.upload(k), ctx.upload(v), None)
    ctx.sync()
    for name, x, dev in (("k", k, pg.dk), ("v", v, pg.dv)):
        want = pg.bits[name].copy()
        at = 0
        for s in range(n):
            r = int(rows[s])
            if r:
                want[pg.index(s, np.arange(lens[s] - r, lens[s]))] = x[at:at + r]
            at += r
        assert np.array_equal(dev.read(np.uint32, want.size), want)
