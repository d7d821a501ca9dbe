"""GPU tests of wpcg_prefix_attention against a plain 64-bit implementation of each
sequence by itself: groups of every size and prefix, types, head layouts, rows,
windows that end in either part; lengths, groups and pages that are none; loose
bounds, graphs, streams. Bounds are derived in serve_ref.attention_bound."""
import numpy as np
import pytest

import serve_ref as R
import wpcg
from serve_ref import BF16, E4M3, F32

pytestmark = pytest.mark.gpu

TYPES = [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, BF16), (F32, E4M3)]


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


class Groups:
    """A batch whose groups share: groups = [(prefix, [own tokens of each sequence])].
    loose: a length by whose bounds the prefixes would be long enough (900 MB read
    again) for sharing to be chosen. Behind the groups are `empty` sequences."""

    def __init__(self, ctx, rng, groups, dtype, hkv, d, page, order="head", width=0, empty=0):
        self.ctx, self.groups = ctx, groups
        again = max(1, sum(len(own) - 1 for _, own in groups)) * 2 * hkv * d * R.SIZE[dtype]
        self.loose = max(width * page, -(-int(900e6) // again // page) * page,
                         max(p + max(own) for p, own in groups) // page * page + page)
        width = self.loose // page
        self.size = [len(own) for _, own in groups]
        self.prefix = [p for p, _ in groups]
        lens = [p + m for p, own in groups for m in own] + [0] * empty
        self.pg = pg = R.Paged(ctx, rng, dtype, hkv, d, page, lens, order=order, scales=dtype == E4M3, width=width)
        self.start = np.cumsum([0] + self.size)
        for g, (p, own) in enumerate(groups):
            lead = self.start[g]
            for s in range(lead + 1, self.start[g + 1]):
                whole = p // page
                pg.table[s, :whole] = pg.table[lead, :whole]
                rest = np.arange(whole * page, p)
                for n in "kv":
                    pg.real[n][s][:p] = pg.real[n][lead][:p]
                    if len(rest):
                        pg.bits[n][pg.index(s, rest)] = pg.bits[n][pg.index(lead, rest)]
        pg.upload()

    def batch(self, rows, **kw):
        return self.pg.batch(rows, **{"max_kv": self.loose, **kw})

    def desc(self, max_prefix=None, start=None, prefix=None):
        self.d_start = self.ctx.upload(np.asarray(self.start if start is None else start, np.int32))
        prefix = self.prefix if prefix is None else prefix
        self.d_prefix = self.ctx.upload(np.asarray(prefix, np.int32))
        return wpcg.KvPrefix(len(prefix), self.d_start, self.d_prefix,
                             self.loose if max_prefix is None else max_prefix)


def expected(pg, q, rows, q_dtype, scale, window, sinks):
    outs, bounds = [], []
    at = 0
    for s, n in enumerate(rows):
        m = pg.kv_len[s]
        x = R.decode(q[at:at + n], q_dtype)
        o, mag, reach = R.attention(x, pg.real["k"][s], pg.real["v"][s], np.arange(m - n, m), scale, window, sinks)
        outs.append(o)
        bounds.append(R.attention_bound(o, mag, reach, pg.d, m, q_dtype))
        at += n
    return np.concatenate(outs), np.concatenate(bounds)


def check(got, want, bound):
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"NaN in rows, heads {np.argwhere(np.isnan(got).any(-1))[:40].tolist()}"
    off = np.abs(got - want) - bound
    i = np.unravel_index(np.nanargmax(off), off.shape)
    assert not (off > 0).any(), f"{(off > 0).sum()} of {off.size} off, worst {i}: {got[i]} for {want[i]} +- {bound[i]}"


def run(ctx, pg, batch, prefix, q, heads, q_dtype, scale, window=0, sinks=0, stream=None):
    rows = q.shape[0]
    out = ctx.upload(np.full(rows * heads * pg.d * R.SIZE[q_dtype], 0x5A, np.uint8))
    qd = ctx.upload(q)
    op = wpcg.PrefixAttention(ctx, pg.kv, batch, prefix, heads, q_dtype, scale=scale, window=window, sinks=sinks)
    run.workspace = op.workspace_bytes
    if op.workspace is not None:
        op.workspace.write(np.full(op.workspace_bytes, 0xFF, np.uint8))
    op.run(qd, out, stream)
    ctx.sync()
    return R.decode(out.read(R.BITS[q_dtype], rows * heads * pg.d).reshape(rows, heads, pg.d), q_dtype)


def least_window(q_dtype, dtype, hkv, d, n):
    """The fewest tokens that n sequences can read again for sharing to be chosen."""
    pays = 250e6 if q_dtype == BF16 else 700e6 if dtype == F32 else 450e6
    return -(-int(pays) // (n * 2 * hkv * d * R.SIZE[dtype]))


def one(ctx, rng, groups, q_dtype, dtype, hkv, heads, d, page, rows=1, window=0, sinks=0, order="head", null_start=False,
        empty=0):
    g = Groups(ctx, rng, groups, dtype, hkv, d, page, order, empty=empty)
    n = len(g.pg.kv_len)
    per = [rows] * (n - empty) + [0] * empty if np.isscalar(rows) else rows
    q = R.encode(rng.standard_normal((sum(per), heads, d)) * 1.5, q_dtype)
    scale = d ** -0.5
    want, bound = expected(g.pg, q, per, q_dtype, scale, window, sinks)
    # as the tight bounds have it, then shared
    check(run(ctx, g.pg, g.pg.batch(None if null_start else per), g.desc(max_prefix=max([1] + g.prefix)),
              q, heads, q_dtype, scale, window, sinks), want, bound)
    batch = g.batch(None if null_start else per)
    got = run(ctx, g.pg, batch, g.desc(), q, heads, q_dtype, scale, window, sinks)
    check(got, want, bound)
    plain = wpcg.PagedAttention(ctx, g.pg.kv, batch, heads, q_dtype, scale=scale, window=window, sinks=sinks)
    few = max(per) * heads // hkv <= 32 and n <= 512 and len(groups) <= 256 and n > len(groups)
    if window:  # what a window lets be read again
        few &= window + sinks + max(per) >= least_window(q_dtype, dtype, hkv, d, n - len(groups))
    assert (run.workspace != plain.workspace_bytes) == few
    return g, batch, q, got, want, bound


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("d,heads,hkv", [(128, 8, 2), (64, 14, 2), (64, 3, 3), (128, 20, 1), (128, 32, 1), (128, 32, 4)])
def test_one_row_each(ctx, q_dtype, dtype, d, heads, hkv):
    """Groups of 4, 7, 1, 20, 32 and 8 query heads; of 2 to 40 sequences and of one;
    prefixes of none, of parts of pages and of several chunks."""
    print(f"[gpu] prefix {q_dtype}/{dtype} {heads}/{hkv}x{d}", flush=True)
    rng = np.random.default_rng(d + heads + 10 * q_dtype + dtype)
    groups = [(300, [1, 2, 40, 33, 7]), (64, [5, 5]), (17, [100]), (0, [3, 90]), (1, [1, 1, 1]), (129, list(range(1, 41))),
              (16, [31, 32, 64])]
    one(ctx, rng, groups, q_dtype, dtype, hkv, heads, d, 16)
    one(ctx, rng, groups, q_dtype, dtype, hkv, heads, d, 16, null_start=True)


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 5, 8])
def test_drafts(ctx, q_dtype, dtype, rows):
    """Several rows a sequence, ragged, one of them without any; prefixes that end
    within the rows' own positions."""
    print(f"[gpu] prefix drafts {q_dtype}/{dtype} rows {rows}", flush=True)
    rng = np.random.default_rng(rows + 10 * q_dtype + dtype)
    groups = [(200, [rows, rows + 1, 50, 90]), (33, [60, 8, 8]), (500, [20] * 9)]
    per = [max(1, rows - i % 3) for i in range(16)]
    per[5] = 0
    one(ctx, rng, groups, q_dtype, dtype, 2, 8, 128, 32, rows=per, order="token")
    # rows that begin before the prefix ends
    one(ctx, rng, [(100, [1, 2, 0, 3]), (64, [0, 0])], q_dtype, dtype, 2, 8, 128, 16, rows=rows)


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 3), (33, 16), (64, 70), (100, 4), (150, 0), (400, 10), (5000, 4), (40, 250)])
def test_windows(ctx, q_dtype, dtype, window, sinks):
    """Windows that leave nothing of the prefix, some of it or all; sinks in it, up
    to its end and beyond."""
    print(f"[gpu] prefix window {q_dtype}/{dtype} {window} {sinks}", flush=True)
    rng = np.random.default_rng(window + sinks + 10 * q_dtype + dtype)
    groups = [(200, [3, 40, 130, 90]), (37, [120, 3, 8]), (300, [20] * 5), (10, [400, 5])]
    one(ctx, rng, groups, q_dtype, dtype, 2, 8, 64, 16, rows=3, window=window, sinks=sinks)


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("more,sinks", [(0, 0), (1, 3), (17, 16), (30, 70), (100, 4), (0, 330), (3000, 5)])
def test_windows_over_shared_prefixes(ctx, q_dtype, dtype, more, sinks):
    """The same with windows wide enough, by a batch's bounds, for sharing to be
    chosen: 512 sequences, most of them empty."""
    print(f"[gpu] prefix shared window {q_dtype}/{dtype} {more} {sinks}", flush=True)
    rng = np.random.default_rng(more + sinks + 10 * q_dtype + dtype)
    w = least_window(q_dtype, dtype, 16, 128, 512 - 4)
    groups = [(w + 50, [3, 40, 130, 90]), (37, [120, 3, 8]), (w + 150, [20] * 5), (10, [w + 200, 5])]
    # (one() says that the call shares)
    one(ctx, rng, groups, q_dtype, dtype, 16, 32, 128, 16, rows=3, window=w + more, sinks=sinks, empty=512 - 14)


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
def test_long_prefixes(ctx, q_dtype, dtype):
    """Several chunks and workgroups a prefix, own tokens of several too; the same
    call gives the same bits."""
    print(f"[gpu] prefix long {q_dtype}/{dtype}", flush=True)
    rng = np.random.default_rng(3 + 10 * q_dtype + dtype)
    groups = [(5000, [700, 3, 1500]), (900, [40, 1]), (2050, [9] * 12)]
    g, batch, q, got, _, _ = one(ctx, rng, groups, q_dtype, dtype, 2, 4, 128, 64)
    again = run(ctx, g.pg, batch, g.desc(), q, 4, q_dtype, 128 ** -0.5)
    assert np.array_equal(got.view(np.uint64), again.view(np.uint64))


@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, F32), (F32, E4M3)])
def test_bounds_that_are_loose(ctx, q_dtype, dtype):
    """More rows, tokens and prefix by the bounds than there are; rows of no
    sequence as they were."""
    rng = np.random.default_rng(4 + dtype)
    g = Groups(ctx, rng, [(150, [4, 30, 9]), (20, [8, 8])], dtype, 2, 64, 16)
    q = R.encode(rng.standard_normal((5 + 20, 6, 64)), q_dtype)
    batch = g.batch([1] * 5, n_rows=25, max_q=3)
    got = run(ctx, g.pg, batch, g.desc(), q, 6, q_dtype, 0.2)
    check(got[:5], *expected(g.pg, q[:5], [1] * 5, q_dtype, 0.2, 0, 0))
    assert (got[5:] == R.decode(np.full(1, 0x5A5A if q_dtype == BF16 else 0x5A5A5A5A, R.BITS[q_dtype]), q_dtype)[0]).all()


@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, BF16)])
def test_groups_that_are_none(ctx, q_dtype, dtype):
    """Groups whose numbers are out of bounds share nothing, a bound below the
    prefix cuts it short, and there may be no groups at all."""
    rng = np.random.default_rng(5)
    g = Groups(ctx, rng, [(150, [4, 30, 9]), (70, [8, 8]), (33, [1, 2])], dtype, 2, 64, 16)
    q = R.encode(rng.standard_normal((7, 8, 64)), q_dtype)
    batch = g.batch([1] * 7)
    want = expected(g.pg, q, [1] * 7, q_dtype, 0.125, 0, 0)
    for start, prefix, most in (([0, 3, 5, 7], [-5, 70, -2 ** 31], g.loose), ([0, 3, 5, 7], [150, 70, 33], 60),
                                ([0, 3, 5, 7], [150, 70, 33], 0), ([-1, 3, 5, 7], [150, 70, 33], g.loose),
                                ([0, 3, 5, 8], [150, 70, 33], g.loose), ([0, 3, 5, 2 ** 31 - 1], [150, 70, 33], g.loose),
                                ([0, 3, 3, 5, 7], [150, 9, 70, 33], g.loose), ([1, 3, 4, 6], [150, 70, 0], g.loose),
                                ([3, 5], [70], g.loose)):
        check(run(ctx, g.pg, batch, g.desc(max_prefix=most, start=start, prefix=prefix), q, 8, q_dtype, 0.125), *want)
    none = wpcg.KvPrefix(0, None, None, 100)
    check(run(ctx, g.pg, batch, none, q, 8, q_dtype, 0.125), *want)


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
def test_lengths_and_pages_that_are_none(ctx, q_dtype, dtype):
    """A length that is none, the first sequence's too; a page of the prefix that
    is none reaches its group alone, one of a sequence's own that one alone."""
    print(f"[gpu] prefix bad {q_dtype}/{dtype}", flush=True)
    rng = np.random.default_rng(6 + dtype)
    g, batch, q, _, want, bound = one(ctx, rng, [(150, [4, 30, 9]), (200, [8, 40, 20]), (33, [1, 2])], q_dtype, dtype, 2, 8, 64, 16)
    pg, prefix = g.pg, g.desc()

    def again(lens, table):
        pg.d_len.write(np.asarray(lens, np.int32))
        pg.d_table.write(table)
        return run(ctx, pg, batch, prefix, q, 8, q_dtype, 0.125)
    for bad in (-1, g.loose + 1, 2 ** 31 - 1, -2 ** 31):
        for s in (0, 4):
            got = again([bad if i == s else m for i, m in enumerate(pg.kv_len)], pg.table)
            assert np.isnan(got[s]).all()
            rest = [i for i in range(8) if i != s]
            check(got[rest], want[rest], bound[rest])
    table = pg.table.copy()
    table[3:6, 2] = [pg.n_pages, -1, 2 ** 31 - 1]
    got = again(pg.kv_len, table)
    assert np.isnan(got[3:6]).all()
    check(got[[0, 1, 2, 6, 7]], want[[0, 1, 2, 6, 7]], bound[[0, 1, 2, 6, 7]])
    table = pg.table.copy()
    table[1, 11] = -5
    got = again(pg.kv_len, table)
    assert np.isnan(got[1]).all()
    check(got[[0, 2, 3, 4, 5, 6, 7]], want[[0, 2, 3, 4, 5, 6, 7]], bound[[0, 2, 3, 4, 5, 6, 7]])


@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, F32), (F32, BF16)])
def test_values_that_are_not_finite(ctx, q_dtype, dtype):
    """NaN and infinities at tokens that a window hides from some rows reach those
    that see them alone."""
    rng = np.random.default_rng(7 + dtype)
    # (the batch's other sequences are empty: enough of them for a window to share)
    w = least_window(q_dtype, dtype, 8, 128, 510)
    g = Groups(ctx, rng, [(w + 30, [3, 60, 90]), (64, [5, 80])], dtype, 8, 128, 16, empty=507)
    pg = g.pg
    q = R.encode(rng.standard_normal((5, 16, 128)), q_dtype)
    batch = g.batch([1] * 5 + [0] * 507)
    want, bound = expected(pg, q, [1] * 5, q_dtype, 0.125, w, 2)
    plain = wpcg.PagedAttention(ctx, pg.kv, batch, 16, q_dtype, scale=0.125, window=w, sinks=2).workspace_bytes
    words = {F32: (0x7F800000, 0xFF800000, 0x7FC00000), BF16: (0x7F80, 0xFF80, 0x7FC0)}[dtype]
    # the row of sequence 0 sees the prefix from its 33rd token on, those of 1 and 2 from the 90th and the 120th
    for word in words:
        for n in "kv":
            x = pg.bits[n].copy()
            x[pg.index(0, [60])] = word
            (pg.dk if n == "k" else pg.dv).write(x)
            got = run(ctx, pg, batch, g.desc(), q, 16, q_dtype, 0.125, w, 2)
            print(f"[gpu] prefix with {word:#x} in {n}", flush=True)
            assert run.workspace != plain
            check(got[1:], want[1:], bound[1:])
            assert not (np.abs(got[0] - want[0]) <= bound[0]).all()
            (pg.dk if n == "k" else pg.dv).write(pg.bits[n])


def test_prompts_are_plain(ctx):
    """More than 32 rows times heads: the same bits as wpcg_paged_attention."""
    rng = np.random.default_rng(8)
    g = Groups(ctx, rng, [(90, [40, 40]), (33, [50, 70])], BF16, 2, 128, 16)
    rows = [40, 30, 50, 1]
    q = R.encode(rng.standard_normal((121, 8, 128)), BF16)
    batch = g.pg.batch(rows)
    got = run(ctx, g.pg, batch, g.desc(), q, 8, BF16, 0.1)
    check(got, *expected(g.pg, q, rows, BF16, 0.1, 0, 0))
    op = wpcg.PagedAttention(ctx, g.pg.kv, batch, 8, BF16, scale=0.1)
    out = ctx.alloc(q.nbytes)
    op.run(ctx.upload(q), out)
    ctx.sync()
    assert np.array_equal(R.decode(out.read(np.uint16, q.size).reshape(q.shape), BF16), got)


def test_many_sequences(ctx):
    """Groups laid out over more sequences than a workgroup has threads, and more
    groups than a wave looks through at once."""
    rng = np.random.default_rng(9)
    groups = [(int(rng.integers(0, 90)), [int(x) for x in rng.integers(1, 40, rng.integers(1, 9))]) for _ in range(150)]
    one(ctx, rng, groups[:100], BF16, BF16, 1, 4, 64, 16)
    one(ctx, rng, [(int(rng.integers(0, 90)), [1, 20]) for _ in range(256)], BF16, E4M3, 1, 4, 64, 16)
    one(ctx, rng, [(40, [2] * 512)], BF16, E4M3, 1, 4, 64, 16)
    one(ctx, rng, [(200, [1 + i % 30 for i in range(511)])], F32, BF16, 1, 2, 64, 16)
    one(ctx, rng, groups, F32, F32, 1, 4, 64, 16)  # more than are shared
    one(ctx, rng, [(40, [2] * 513)], BF16, BF16, 1, 4, 64, 16)


@pytest.mark.parametrize("heads,hkv", [(4, 1), (3, 3), (10, 5), (8, 1)])
def test_costs_that_are_rounded(ctx, heads, hkv):
    """Prefixes of 1 to 12 tiles in few items, several groups behind each other."""
    rng = np.random.default_rng(heads)
    for most in (3, 6, 12):
        groups = [(int(rng.integers(1, 32 * most)), [int(x) for x in rng.integers(1, 60, rng.integers(2, 5))]) for _ in range(12)]
        one(ctx, rng, groups, BF16, BF16, hkv, heads, 64, 16)


def test_graphs_and_streams(ctx):
    """Two captured calls in turn whose lengths, groups and queries change between
    the replays, and the same bits from another stream."""
    print("[gpu] prefix graphs", flush=True)
    rng = np.random.default_rng(10)
    made = []
    for groups, dtype in (([(400, [60] * 7), (90, [60] * 3)], BF16), ([(64, [40] * 4)], F32)):
        g = Groups(ctx, rng, groups, dtype, 2, 128, 16)
        n = len(g.pg.kv_len)
        batch, prefix = g.batch([1] * n), g.desc()
        q, out = ctx.alloc(n * 8 * 128 * R.SIZE[dtype]), ctx.alloc(n * 8 * 128 * R.SIZE[dtype])
        op = wpcg.PrefixAttention(ctx, g.pg.kv, batch, prefix, 8, dtype, scale=0.1)
        made.append((g, dtype, n, q, out, ctx.capture(lambda op=op, q=q, out=out: op.run(q, out)), op, batch))
    whole = [list(m[0].pg.kv_len) for m in made]
    for turn in range(5):
        xs = []
        for (g, dtype, n, q, out, graph, _, _), lens in zip(made, whole):
            g.pg.kv_len = [m - int(rng.integers(0, 59 if dtype == BF16 else 39)) for m in lens]
            g.pg.d_len.write(np.array(g.pg.kv_len, np.int32))
            g.d_prefix.write(np.array([p - turn for p in g.prefix], np.int32))
            x = R.encode(rng.standard_normal((n, 8, 128)), dtype)
            q.write(x)
            xs.append(x)
            graph.launch()
        ctx.sync()
        for (g, dtype, n, _, out, _, _, _), x in zip(made, xs):
            got = R.decode(out.read(R.BITS[dtype], x.size).reshape(x.shape), dtype)
            real = {k: [v[:m] for v, m in zip(g.pg.real[k], g.pg.kv_len)] for k in "kv"}
            outs = [R.attention(R.decode(x[s:s + 1], dtype), real["k"][s], real["v"][s], [g.pg.kv_len[s] - 1], 0.1, 0, 0)
                    for s in range(n)]
            bound = np.concatenate([R.attention_bound(*o, 128, g.pg.kv_len[s], dtype) for s, o in enumerate(outs)])
            check(got, np.concatenate([o[0] for o in outs]), bound)
    other = wpcg.Context(0)
    g, dtype, n, q, out, graph, op, _ = made[0]
    first = out.read(R.BITS[dtype], n * 8 * 128)
    out.write(np.zeros_like(first))
    op.run(q, out, other.stream)
    other.sync()
    assert np.array_equal(out.read(R.BITS[dtype], n * 8 * 128), first)
    other.close()


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("sinks", [0, 20])
def test_windows_that_left_the_first_sequence_ahead(ctx, q_dtype, dtype, sinks):
    """A group's first sequence is further on than others, or has ended: pages behind
    its window, which others still see, are no longer in its row of the table, nor
    are any behind theirs in the others'. Ids of no page there, and ids of pages that hold
    something else."""
    print(f"[gpu] prefix window, first ahead {q_dtype}/{dtype} sinks {sinks}", flush=True)
    rng = np.random.default_rng(100 + sinks + 10 * q_dtype + dtype)
    w = least_window(q_dtype, dtype, 16, 128, 512 - 5) + 5
    # longest first; ended first; ended and longest; shortest first; rows that begin before the prefix ends
    groups = [(w + 90, [w + 300, 3, 40, w + 130]), (w + 40, [0, 70, 3]), (2 * w + 100, [200, 20, 20, 130]),
              (300, [9, w + 20]), (150, [w + 60, 0, 2 * w])]
    live = sum(len(own) for _, own in groups)
    g = Groups(ctx, rng, groups, dtype, 16, 128, 16, empty=512 - live)
    pg = g.pg
    per = [3] * live + [0] * (512 - live)
    per[4], pg.kv_len[4] = 0, 0
    for n in "kv":
        pg.real[n][4] = pg.real[n][4][:0]
    # sequence 14's only rows lie before its group's prefix ends
    pg.kv_len[14] = 60
    for n in "kv":
        pg.real[n][14] = pg.real[n][14][:60]
    q = R.encode(rng.standard_normal((sum(per), 32, 128)) * 1.5, q_dtype)
    batch = g.batch(per)
    want, bound = expected(pg, q, per, q_dtype, 128 ** -0.5, w, sinks)
    plain = wpcg.PagedAttention(ctx, pg.kv, batch, 32, q_dtype, scale=128 ** -0.5, window=w, sinks=sinks).workspace_bytes
    whole = pg.table.copy()
    for gone in (-1, 2 ** 31 - 1, pg.n_pages, "others"):
        table = whole.copy()
        for s in range(live):
            pages = -(-pg.kv_len[s] // 16)
            lo = pg.kv_len[s] - per[s] - w + 1  # the first token that its rows see
            for j in range(table.shape[1]):
                seen = j < pages and per[s] and (16 * (j + 1) > lo or 16 * j < sinks)
                if not seen:
                    table[s, j] = int(rng.integers(0, pg.n_pages)) if gone == "others" else gone
        pg.d_table.write(table)
        got = run(ctx, pg, batch, g.desc(), q, 32, q_dtype, 128 ** -0.5, w, sinks)
        assert run.workspace != plain  # it shares
        check(got, want, bound)


@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, E4M3)])
def test_windows_whose_pages_a_fork_gave_back(ctx, q_dtype, dtype):
    """The same with the tables that wpcg_kv_fork leaves, in steps of uneven numbers of
    tokens a sequence."""
    print(f"[gpu] prefix window after forks {q_dtype}/{dtype}", flush=True)
    rng = np.random.default_rng(200 + dtype)
    w = least_window(q_dtype, dtype, 16, 128, 512 - 2) + 3
    groups = [(w + 90, [5, 3, 40, 1]), (2 * w, [1, 1, 1])]
    live = 7
    g = Groups(ctx, rng, groups, dtype, 16, 128, 16, empty=512 - live)
    pg = g.pg
    stride = pg.table.shape[1]
    pg.table[:, :] = np.where(np.arange(stride) < -(-np.array(pg.kv_len)[:, None] // 16), pg.table, -1)
    refs = np.bincount(pg.table[pg.table >= 0], minlength=pg.n_pages).astype(np.int32)
    pool = wpcg.KvPool(ctx, pg.n_pages, 16, 512, stride, refs=ctx.upload(refs), table=ctx.upload(pg.table),
                       kv_len=ctx.upload(np.array(pg.kv_len, np.int32)))
    copies, result, grow = ctx.alloc(12 * 512), ctx.alloc(8), ctx.alloc(4 * 512)
    fork = wpcg.KvFork(ctx, pool, copies, result, grow_each=grow, window=w)
    copy = wpcg.KvCopy(ctx, [pg.kv], copies, result, 512)
    gone = 0
    for turn in range(5):
        # the first sequence is ahead of the others
        more = np.zeros(512, np.int32)
        more[:live] = [3, 1, 2, 1, 3, 1, 2] if turn else [w + 60, 1, 1, 2, w // 2, 1, 1]
        per = [min(3, int(m)) for m in more]
        grow.write(more)
        fork.run()
        copy.run()
        ctx.sync()
        assert result.read(np.int32, 2)[0] >= 0
        pg.table = pool.table.read(np.int32, 512 * stride).reshape(512, stride)
        for n, buf in (("k", pg.dk), ("v", pg.dv)):
            pg.bits[n] = buf.read(R.BITS[dtype], pg.bits[n].size).reshape(pg.bits[n].shape)
        for s in range(live):
            m = int(more[s])
            new = np.arange(pg.kv_len[s], pg.kv_len[s] + m)
            for n in "kv":
                x = R.encode(rng.standard_normal((m, 16, 128)), dtype)
                pg.bits[n][pg.index(s, new)] = x
                pg.real[n][s] = np.concatenate([pg.real[n][s], R.decode(x, dtype) * pg.scale[n][:, None].astype(np.float64)])
            pg.kv_len[s] += m
        pg.dk.write(pg.bits["k"])
        pg.dv.write(pg.bits["v"])
        gone += int((pg.table[0] == -1)[:5].sum())
        q = R.encode(rng.standard_normal((sum(per), 32, 128)) * 1.5, q_dtype)
        batch = g.batch(per)
        want, bound = expected(pg, q, per, q_dtype, 0.1, w, 0)
        check(run(ctx, pg, batch, g.desc(), q, 32, q_dtype, 0.1, w, 0), want, bound)
        plain = wpcg.PagedAttention(ctx, pg.kv, batch, 32, q_dtype, scale=0.1, window=w)
        assert run.workspace != plain.workspace_bytes
    assert gone > 0


@pytest.mark.parametrize("start", [[0, 12, -2 ** 31], [0, 2 ** 31 - 1, -2 ** 31, 12], [3, -2 ** 31, 0, 12], [-2 ** 31, 0, 2 - 2 ** 31, 12]])
@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, F32)])
def test_group_starts_that_are_the_least_number(ctx, q_dtype, dtype, start):
    """Groups that end two and fewer above the least number, where a difference of the two overflows."""
    print(f"[gpu] prefix least starts {q_dtype}/{dtype} {start}", flush=True)
    rng = np.random.default_rng(320 + dtype)
    g = Groups(ctx, rng, [(90, list(range(1, 13)))], dtype, 2, 64, 16)
    q = R.encode(rng.standard_normal((12, 8, 64)) * 1.5, q_dtype)
    want = expected(g.pg, q, [1] * 12, q_dtype, 0.125, 0, 0)
    prefix = g.desc(start=start, prefix=[90] * (len(start) - 1))
    check(run(ctx, g.pg, g.batch([1] * 12), prefix, q, 8, q_dtype, 0.125), *want)
    assert run.workspace != wpcg.PagedAttention(ctx, g.pg.kv, g.batch([1] * 12), 8, q_dtype, scale=0.125).workspace_bytes


@pytest.mark.parametrize("start", [[512 if i % 2 else 4 * i for i in range(129)], [0, 512, 256, 512, 512], [0, 512] * 9 + [0],
                                   [0, 100, 50, 512], [100, 0, 512],
                                   [5, 512, 5, 2 ** 30, 7]])
@pytest.mark.parametrize("q_dtype,dtype", [(BF16, BF16), (F32, BF16)])
def test_group_starts_that_fall(ctx, q_dtype, dtype, start):
    """Groups that lie over each other or end before they begin: the outputs are those of
    the sequences all the same."""
    print(f"[gpu] prefix falling starts {q_dtype}/{dtype} {start[:5]}", flush=True)
    rng = np.random.default_rng(300 + dtype)
    g = Groups(ctx, rng, [(100, [1 + i % 20 for i in range(512)])], dtype, 2, 64, 16)
    q = R.encode(rng.standard_normal((512, 8, 64)) * 1.5, q_dtype)
    want = expected(g.pg, q, [1] * 512, q_dtype, 0.125, 0, 0)
    batch = g.batch([1] * 512)
    prefix = g.desc(start=start, prefix=[100] * (len(start) - 1))
    check(run(ctx, g.pg, batch, prefix, q, 8, q_dtype, 0.125), *want)
    assert run.workspace != wpcg.PagedAttention(ctx, g.pg.kv, batch, 8, q_dtype, scale=0.125).workspace_bytes


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
def test_first_sequences_without_rows(ctx, q_dtype, dtype):
    """Sequences of a step that have no rows, at their groups' begin: ended ones, and
    ones whose rows of the table hold anything, as no row sees their pages."""
    print(f"[gpu] prefix first without rows {q_dtype}/{dtype}", flush=True)
    rng = np.random.default_rng(400 + dtype)
    groups = [(150, [4, 30, 9]), (200, [8, 40, 20, 1]), (70, [8, 8, 5]), (33, [1, 2])]
    g = Groups(ctx, rng, groups, dtype, 2, 64, 16)
    pg = g.pg
    per = [0, 2, 2, 0, 0, 1, 2, 0, 2, 2, 0, 0]
    pg.kv_len[3] = 0
    for n in "kv":
        pg.real[n][3] = pg.real[n][3][:0]
    whole = pg.table.copy()
    for s in (0, 4, 7, 10, 11):
        pg.table[s] = rng.integers(0, pg.n_pages, pg.table.shape[1]) if s != 4 else -1
    pg.table[7] = 2 ** 31 - 1
    q = R.encode(rng.standard_normal((sum(per), 8, 64)) * 1.5, q_dtype)
    batch = g.batch(per)
    want = expected(pg, q, per, q_dtype, 0.125, 0, 0)
    check(run(ctx, pg, batch, g.desc(), q, 8, q_dtype, 0.125), *want)
    assert run.workspace != wpcg.PagedAttention(ctx, pg.kv, batch, 8, q_dtype, scale=0.125).workspace_bytes
    # a length that is none in their place, and with their own pages
    pg.table = whole
    for bad in (-1, 2 ** 31 - 1):
        batch = g.batch(per)
        pg.d_len.write(np.array([bad if i in (0, 7) else m for i, m in enumerate(pg.kv_len)], np.int32))
        check(run(ctx, pg, batch, g.desc(), q, 8, q_dtype, 0.125), *want)


def test_errors_of_other_calls(ctx):
    """A refused allocation before them is not reported by calls that work."""
    rng = np.random.default_rng(500)
    g = Groups(ctx, rng, [(150, [4, 30, 9])], BF16, 2, 64, 16)
    q = ctx.upload(R.encode(rng.standard_normal((3, 8, 64)), BF16))
    out, ints, flt = ctx.alloc(3 * 8 * 64 * 2), ctx.upload(np.zeros(64, np.int32)), ctx.alloc(4096)
    batch = g.batch([1] * 3)
    shared = wpcg.PrefixAttention(ctx, g.pg.kv, batch, g.desc(), 8, BF16)
    plain = wpcg.PagedAttention(ctx, g.pg.kv, batch, 8, BF16)
    assert shared.workspace_bytes != plain.workspace_bytes
    prompt = wpcg.PagedAttention(ctx, g.pg.kv, g.batch([40] * 3, n_rows=120), 8, BF16)  # (many rows; not run)
    assert prompt.workspace_bytes >= 0
    many_q = ctx.upload(R.encode(rng.standard_normal((120, 8, 64)), BF16))
    many_out = ctx.alloc(120 * 8 * 64 * 2)
    pool = wpcg.KvPool(ctx, 20, 16, 3, 4)
    copies, result = ctx.alloc(400), ctx.alloc(8)
    k = ctx.upload(R.encode(rng.standard_normal((3, 2, 64)), BF16))
    scratch = wpcg.PagedKv(ctx, 20, 16, 2, 64, BF16)
    room = wpcg.KvBatch(3, 3, pool.kv_len, pool.table, 4, 64)
    score = wpcg.LogProbs(ctx, 2, 100, top=3)
    logits = ctx.upload(rng.standard_normal((2, 100)).astype(np.float32))
    u = ctx.upload(np.full(8, 0.5, np.float32))
    draft = wpcg.DraftVerify(ctx, 1, 2, 2, 100)
    ids = ctx.alloc(400)
    calls = {"fork": lambda: wpcg.KvFork(ctx, pool, copies, result, grow=5).run(),
             "large fork": lambda: wpcg.KvFork(ctx, wpcg.KvPool(ctx, 20, 16, 70, 4), ctx.alloc(1024), result).run(),
             "compact": lambda: wpcg.KvCompact(ctx, pool, copies, result, 5).run(),
             "copy": lambda: wpcg.KvCopy(ctx, [scratch], copies, result, 3).run(),
             "append": lambda: wpcg.KvAppend(ctx, scratch, room, 8, BF16).run(None, k, k, None),
             "shared": lambda: shared.run(q, out), "plain": lambda: plain.run(q, out),
             "prompt": lambda: prompt.run(many_q, many_out), "score": lambda: score.run(logits, ints, flt, top_ids=ids),
             "draft": lambda: draft.run(logits, ints, u, u, flt, out)}
    for name, call in calls.items():
        with pytest.raises(wpcg.WpcgError):
            ctx.alloc(1 << 50)
        print(f"[gpu] after a refused allocation: {name}", flush=True)
        call()
        ctx.sync()


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("sinks", [0, 40, 500])
def test_windows_that_have_left_the_prefix(ctx, q_dtype, dtype, sinks):
    """Groups none of whose rows, or of whose later ones, see a token of the prefix but
    for the sinks; the prefixes' pages are others' by now. Prefixes that end inside tiles
    and pages, and at their borders."""
    print(f"[gpu] prefix window beyond {q_dtype}/{dtype} sinks {sinks}", flush=True)
    rng = np.random.default_rng(600 + sinks + 10 * q_dtype + dtype)
    w = least_window(q_dtype, dtype, 16, 128, 512 - 6) + 5
    groups = [(361, [w + 90, w + 50, w + 70]), (64, [w + 1, w + 200]), (100, [w + 70, 5, w]), (17, [w + 39, w + 80]), (128, [w, w - 1]),
              (360, [w + 300, w + 31])]
    live = sum(len(own) for _, own in groups)
    g = Groups(ctx, rng, groups, dtype, 16, 128, 32, empty=512 - live)
    pg = g.pg
    per = [1] * live + [0] * (512 - live)
    q = R.encode(rng.standard_normal((live, 32, 128)) * 1.5, q_dtype)
    lo = np.array(pg.kv_len) - w  # the first token in the row's window
    first = np.arange(pg.table.shape[1])[None] * 32
    seen = (first < np.array(pg.kv_len)[:, None]) & ((first + 32 > lo[:, None]) | (first < sinks))
    pg.table = np.where(seen, pg.table, -1).astype(np.int32)
    batch = g.batch(per)
    want, bound = expected(pg, q, per, q_dtype, 0.1, w, sinks)
    plain = wpcg.PagedAttention(ctx, pg.kv, batch, 32, q_dtype, scale=0.1, window=w, sinks=sinks).workspace_bytes
    check(run(ctx, pg, batch, g.desc(), q, 32, q_dtype, 0.1, w, sinks), want, bound)
    assert run.workspace != plain


@pytest.mark.parametrize("window", [False, True])
def test_captured_calls_whose_first_sequences_change(ctx, window):
    """One captured call: which sequence of a group has rows, or is furthest on, and what
    the tables hold for the others, changes between the replays."""
    print(f"[gpu] prefix captured, window {window}", flush=True)
    rng = np.random.default_rng(700)
    w = least_window(BF16, BF16, 16, 128, 512 - 2) + 5 if window else 0
    g = Groups(ctx, rng, [(w + 90, [w + 300] * 4), (200, [w + 200] * 3)], BF16, 16, 128, 16, empty=505)
    pg = g.pg
    whole = {"table": pg.table.copy(), "real": pg.real}
    batch, prefix = g.batch([1] * 7 + [0] * 505), g.desc()
    lens, table, start = pg.d_len, pg.d_table, pg.d_start
    q, out = ctx.alloc(7 * 32 * 128 * 2), ctx.alloc(7 * 32 * 128 * 2)
    op = wpcg.PrefixAttention(ctx, pg.kv, batch, prefix, 32, BF16, scale=0.1, window=w)
    assert op.workspace_bytes != wpcg.PagedAttention(ctx, pg.kv, batch, 32, BF16, scale=0.1, window=w).workspace_bytes
    graph = ctx.capture(lambda: op.run(q, out))
    for turn in range(6):
        per = [1] * 7 + [0] * 505
        per[turn % 4] = per[4 + turn % 3] = 0  # the first one of both groups in turn 0
        n = [int(m - rng.integers(0, 150)) for m in (w + 90 + w + 300,) * 4 + (200 + w + 200,) * 3] + [0] * 505
        pg.kv_len, pg.real = n, {k: [x[:m] for x, m in zip(whole["real"][k], n)] for k in "kv"}
        lo = np.where(np.array(per) > 0, np.array(n) - w if window else 0, 2 ** 30)
        first = np.arange(pg.table.shape[1])[None] * 16
        seen = (first < np.array(n)[:, None]) & (first + 16 > lo[:, None])
        table.write(np.where(seen, whole["table"], turn % 2 * (2 ** 31 - 1) - 1).astype(np.int32))
        lens.write(np.array(n, np.int32))
        start.write(np.cumsum([0] + per).astype(np.int32))
        x = R.encode(rng.standard_normal((5, 32, 128)) * 1.5, BF16)
        q.write(np.concatenate([x, x[:2]]))
        graph.launch()
        ctx.sync()
        got = R.decode(out.read(np.uint16, 5 * 32 * 128).reshape(5, 32, 128), BF16)
        check(got, *expected(pg, x, per, BF16, 0.1, w, 0))
