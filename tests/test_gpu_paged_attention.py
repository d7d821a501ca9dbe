"""GPU tests of wpcg_paged_attention against a plain 64-bit implementation:
one to many rows a sequence, every pair of types, head layouts, lengths from
none to split ones, windows and sinks, page orders and strides; what a row does
not see (NaN, infinities, ids of no page) does not reach it; bad pages and
lengths; graphs, streams. Bounds are derived in serve_ref.attention_bound."""
import numpy as np
import pytest

import serve_ref as R
import wpcg
from serve_ref import BF16, E4M3, F32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


def expected(pg, q, rows, heads, q_dtype, scale, window, sinks):
    """(outputs, bounds) [row][head][d] from the stored values."""
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
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want) - bound
    i = np.unravel_index(np.nanargmax(off), off.shape)
    assert not (off > 0).any(), f"{(off > 0).sum()} of {off.size} off, worst {i}: {got[i]} for {want[i]} +- {bound[i]}"


def run(ctx, pg, batch, q, heads, q_dtype, scale, window=0, sinks=0, fill=0x5A, stream=None):
    """Output rows as values; rows that nothing is written to keep the fill."""
    rows = q.shape[0]
    out = ctx.upload(np.full(rows * heads * pg.d * R.SIZE[q_dtype], fill, np.uint8))
    qd = ctx.upload(q)
    op = wpcg.PagedAttention(ctx, pg.kv, batch, heads, q_dtype, scale=scale, window=window, sinks=sinks)
    if op.workspace is not None:  # the workspace may hold anything
        op.workspace.write(np.full(op.workspace_bytes, 0xFF, np.uint8))
    op.run(qd, out, stream)
    ctx.sync()
    bits = out.read(R.BITS[q_dtype], rows * heads * pg.d).reshape(rows, heads, pg.d)
    return R.decode(bits, q_dtype), op


TYPES = [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, BF16), (F32, E4M3)]
LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 0, 257]


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("d,heads,hkv", [(128, 8, 2), (64, 14, 2), (64, 3, 3), (128, 20, 1), (128, 32, 1)])
def test_one_row_every_length(ctx, q_dtype, dtype, d, heads, hkv):
    """Groups of 4, 7, 1, 20 and 32 query heads (the last in the kernel for
    many rows); a length of none gives zeros."""
    print(f"[gpu] one row: {q_dtype}/{dtype} {heads}/{hkv}x{d}", flush=True)
    rng = np.random.default_rng(d + heads + 100 * q_dtype + dtype)
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, LENGTHS, scales=dtype == E4M3).upload()
    q = R.encode(rng.standard_normal((len(LENGTHS), heads, d)) * 1.5, q_dtype)
    scale = d ** -0.5
    got, _ = run(ctx, pg, pg.batch(None), q, heads, q_dtype, scale)
    check(got, *expected(pg, q, [1] * len(LENGTHS), heads, q_dtype, scale, 0, 0))


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 3), (33, 16), (50, 40), (1000, 4), (7, 300)])
def test_few_rows_windows(ctx, q_dtype, dtype, window, sinks):
    """Three rows a sequence (drafts): causal among themselves, windows that
    end inside tiles, sinks that meet the window and that exceed the length."""
    print(f"[gpu] few rows: {q_dtype}/{dtype} window {window} sinks {sinks}", flush=True)
    rng = np.random.default_rng(window * 7 + sinks + q_dtype + 10 * dtype)
    lens = [3, 5, 20, 50, 64, 97, 150, 258]
    pg = R.Paged(ctx, rng, dtype, 2, 128, 32, lens, order="token", scales=dtype == E4M3).upload()
    q = R.encode(rng.standard_normal((3 * len(lens), 8, 128)) * 1.5, q_dtype)
    got, _ = run(ctx, pg, pg.batch([3] * len(lens)), q, 8, q_dtype, 0.1, window, sinks)
    check(got, *expected(pg, q, [3] * len(lens), 8, q_dtype, 0.1, window, sinks))


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("d,heads,hkv,window,sinks", [(128, 8, 2, 0, 0), (64, 7, 1, 0, 0), (128, 4, 4, 40, 5),
                                                      (64, 4, 2, 64, 0), (128, 16, 1, 100, 70)])
def test_many_rows(ctx, q_dtype, dtype, d, heads, hkv, window, sinks):
    """Ragged prompts, with and without cached tokens before them, and a
    sequence with more rows than tokens (its first rows see nothing)."""
    print(f"[gpu] many rows: {q_dtype}/{dtype} {heads}/{hkv}x{d} window {window} sinks {sinks}", flush=True)
    rng = np.random.default_rng(d + heads + window + q_dtype + 10 * dtype)
    rows, lens = [70, 1, 133, 40, 9], [70, 200, 190, 167, 5]
    pg = R.Paged(ctx, rng, dtype, hkv, d, 64, lens, scales=dtype == E4M3).upload()
    q = R.encode(rng.standard_normal((sum(rows), heads, d)) * 1.5, q_dtype)
    scale = d ** -0.5
    got, _ = run(ctx, pg, pg.batch(rows), q, heads, q_dtype, scale, window, sinks)
    check(got, *expected(pg, q, rows, heads, q_dtype, scale, window, sinks))


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("rows,lens,heads,hkv,window", [([1, 1], [5000, 37], 4, 2, 0), ([2, 2], [3001, 1], 8, 2, 700),
                                                        ([40, 3], [2500, 3], 8, 2, 0), ([65], [4000], 4, 1, 900)])
def test_split_and_joined(ctx, q_dtype, dtype, rows, lens, heads, hkv, window):
    """Sequences split over workgroups, beside ones too short for a second
    part; the same call gives the same bits."""
    print(f"[gpu] split: {q_dtype}/{dtype} rows {rows} lens {lens}", flush=True)
    rng = np.random.default_rng(sum(lens) + q_dtype + 10 * dtype)
    pg = R.Paged(ctx, rng, dtype, hkv, 128, 16, lens, scales=dtype == E4M3).upload()
    q = R.encode(rng.standard_normal((sum(rows), heads, 128)) * 1.5, q_dtype)
    b = pg.batch(rows)
    got, op = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, 4)
    assert op.workspace_bytes > 0 or 0 < window < 5000  # (a short window is not worth a second part)
    check(got, *expected(pg, q, rows, heads, q_dtype, 0.09, window, 4))
    again, _ = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, 4)
    assert np.array_equal(got.view(np.uint64), again.view(np.uint64))


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("singles,prompts,lens,heads,hkv,window", [
    (5, [70, 9, 8, 0, 33], (1, 400), 8, 2, 0), (70, [200, 5], (20, 300), 8, 2, 60), (150, [300], (1, 90), 4, 4, 0),
    (3, [90], (2000, 6000), 8, 2, 0), (6, [20, 150, 1], (10, 700), 20, 1, 0), (4, [40], (10, 700), 64, 1, 0)])
@pytest.mark.parametrize("max_kv", [None, 6500, 1000000])
def test_prompts_among_single_tokens(ctx, q_dtype, dtype, singles, prompts, lens, heads, hkv, window, max_kv):
    """A batch's short and long row ranges are two kernels' work where it may be
    long: around the border (32 columns: 8 rows of 4 heads and 9), more sequences than a wave
    looks through at once, long sequences of few rows beside a prompt, groups
    of 20 and of 64 heads (none of its rows is the few-row kernel's); a bad
    length and a bad page in either part, rows of no sequence as they were."""
    print(f"[gpu] mixed: {q_dtype}/{dtype} {singles} + {prompts} {heads}/{hkv} window {window}", flush=True)
    rng = np.random.default_rng(singles + heads + q_dtype + 10 * dtype)
    rows = [1] * singles + prompts
    order = rng.permutation(len(rows))
    rows = [rows[i] for i in order]
    kv = [int(x) + r for x, r in zip(rng.integers(*lens, len(rows)), rows)]
    pg = R.Paged(ctx, rng, dtype, hkv, 64, 16, kv, scales=dtype == E4M3, width=(max_kv or 0) // 16 + 1).upload()
    n = sum(rows)
    q = R.encode(rng.standard_normal((n + 7, heads, 64)) * 1.5, q_dtype)
    batch = pg.batch(rows, n_rows=n + 7, max_kv=max_kv)
    want, bound = expected(pg, q[:n], rows, heads, q_dtype, 0.125, window, 9)
    got, op = run(ctx, pg, batch, q, heads, q_dtype, 0.125, window, 9)
    fill = R.decode(np.full(1, 0x5A5A if q_dtype == BF16 else 0x5A5A5A5A, R.BITS[q_dtype]), q_dtype)[0]
    check(got[:n], want, bound)
    assert (got[n:] == fill).all()
    at = np.cumsum([0] + rows)
    one, many = rows.index(1), int(np.argmax(rows))
    pg.table[many, kv[many] // 16 - 1] = -3  # the prompt's last whole page, which its last row sees
    pg.d_table.write(pg.table)
    pg.d_len.write(np.array([-1 if s == one else m for s, m in enumerate(kv)], np.int32))
    got, _ = run(ctx, pg, batch, q, heads, q_dtype, 0.125, window, 9)
    assert np.isnan(got[at[one]]).all() and np.isnan(got[at[many + 1] - 1]).all()
    for s in range(len(rows)):
        if s not in (one, many) and rows[s]:
            part = slice(at[s], at[s + 1])
            check(got[part], want[part], bound[part])


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("rows,heads,hkv,d,window", [(1, 8, 2, 128, 0), (1, 4, 4, 64, 0), (5, 8, 2, 128, 0),
                                                     (3, 7, 1, 64, 2000), (2, 8, 2, 128, 40000)])
def test_tiles_dealt_out(ctx, q_dtype, dtype, rows, heads, hkv, d, window):
    """Sequences that may be long by the call's bounds (a million tokens) have
    their tiles dealt out evenly, whatever their lengths are: some of several
    workgroups, some many to one, some of no token or fewer than rows."""
    print(f"[gpu] dealt: {q_dtype}/{dtype} rows {rows} {heads}/{hkv}x{d} window {window}", flush=True)
    rng = np.random.default_rng(rows + heads + d + q_dtype + 10 * dtype)
    lens = [3000, 5, 0, 517, 1024, 33, 2100, rows, 512, 511, 1, 1500, 16, 640, 2, 900, 64, 100, 31, 32, 260, 700, 4, 48]
    n = len(lens)
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, lens, scales=dtype == E4M3, width=62500).upload()
    nr = [rows] * n
    nr[4], nr[9] = 1, max(1, rows - 1)
    q = R.encode(rng.standard_normal((sum(nr), heads, d)) * 1.5, q_dtype)
    b = pg.batch(nr, max_kv=1000000, max_q=rows)
    got, op = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, 20)
    assert op.workspace_bytes > 0
    want, bound = expected(pg, q, nr, heads, q_dtype, 0.09, window, 20)
    check(got, want, bound)
    again, _ = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, 20)
    assert np.array_equal(got.view(np.uint64), again.view(np.uint64))
    # a page that is none in one sequence, a length that is none in another
    pg.table[0, 100] = pg.n_pages + 1
    pg.d_table.write(pg.table)
    pg.d_len.write(np.array(lens[:3] + [-1] + lens[4:], np.int32))
    got, _ = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, 20)
    at = np.cumsum([0] + nr)
    if window != 2000:  # (which hides the page)
        assert np.isnan(got[:at[1]]).all()
    assert np.isnan(got[at[3]:at[4]]).all()
    check(got[at[1]:at[3]], want[at[1]:at[3]], bound[at[1]:at[3]])
    check(got[at[4]:], want[at[4]:], bound[at[4]:])


@pytest.mark.parametrize("n,rows", [(700, 1), (2048, 2), (2049, 1)])
def test_more_sequences_than_threads(ctx, n, rows):
    """Dealt out over several rounds of a workgroup's threads; one sequence more
    than that takes, each with workgroups of its own again."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 40, n)]
    lens[5], lens[n - 1] = 900, 1300
    pg = R.Paged(ctx, rng, BF16, 1, 64, 16, lens, width=6250).upload()
    q = R.encode(rng.standard_normal((n * rows, 2, 64)), BF16)
    got, op = run(ctx, pg, pg.batch([rows] * n, max_kv=100000), q, 2, BF16, 0.125)
    assert (op.workspace_bytes > 0) == (n <= 2048)
    check(got, *expected(pg, q, [rows] * n, 2, BF16, 0.125, 0, 0))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("d,heads,hkv,window,sinks", [(64, 8, 2, 0, 0), (128, 8, 2, 0, 0), (128, 20, 4, 0, 0),
                                                      (64, 8, 2, 2500, 3), (128, 8, 2, 2300, 70)])
def test_long_prompts(ctx, dtype, d, heads, hkv, window, sinks):
    """Batches that may hold long prompts with blocks enough for every CU take 256
    columns a workgroup, two halves of it in turns: sequences of none, one, two,
    three and many tiles, of rows for a part of a workgroup and for several, one
    whose last token's values are not finite (twice in a row of tiles), a bad
    length, a bad page; the same call gives the same bits."""
    print(f"[gpu] long prompts: {dtype} {heads}/{hkv}x{d} window {window}", flush=True)
    rng = np.random.default_rng(d + heads + window + dtype)
    n = 300 // hkv
    rows = [1] * n
    kv = [int(x) for x in rng.integers(1, 9, n)]
    for s, (r, m) in {3: (100, 100), 4: (70, 2600), 10: (33, 64), 11: (90, 129), 20: (130, 192), 21: (100, 193),
                      30: (40, 500), 31: (9, 64), 40: (64, 65), 50: (20, 5), 60: (110, 900)}.items():
        rows[s], kv[s] = r, m
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, kv, scales=dtype == E4M3, width=170)
    # not finite: the last rows alone see them, the others' are masked
    for at in (450, 499):
        x = pg.real["v"][30][at] / pg.scale["v"][:, None]  # as stored
        x[0, 7], x[0, 9] = np.nan, (np.nan if dtype == E4M3 else -np.inf)
        pg.put("v", 30, R.encode(x, dtype)[None], [at])
    pg.upload()
    total = sum(rows)
    q = R.encode(rng.standard_normal((total + 3, heads, d)) * 1.5, BF16)
    batch = pg.batch(rows, n_rows=total + 3, max_kv=2700, max_q=256)
    got, _ = run(ctx, pg, batch, q, heads, BF16, 0.1, window, sinks)
    want, bound = expected(pg, q[:total], rows, heads, BF16, 0.1, window, sinks)
    at = np.cumsum([0] + rows)
    group = heads // hkv
    odd = got[at[30]:at[31], :group][..., [7, 9]]
    first = np.array([max(0, t - (500 - 40)) for t in (450, 499)])  # row from which a token is seen
    assert np.isfinite(odd[:first[0]]).all() and not np.isfinite(odd[first[0]:]).any()
    got[at[30] + first[0]:at[31], :group, [7, 9]] = want[at[30] + first[0]:at[31], :group, [7, 9]]
    check(got[:total], want, bound)
    fill = R.decode(np.full(1, 0x5A5A, np.uint16), BF16)[0]
    assert (got[total:] == fill).all()
    again, _ = run(ctx, pg, batch, q, heads, BF16, 0.1, window, sinks)
    again[at[30] + first[0]:at[31], :group, [7, 9]] = want[at[30] + first[0]:at[31], :group, [7, 9]]
    assert np.array_equal(got.view(np.uint64), again.view(np.uint64))
    pg.table[60, 40] = pg.n_pages
    pg.d_table.write(pg.table)
    pg.d_len.write(np.array([2701 if s == 20 else m for s, m in enumerate(kv)], np.int32))
    bad, _ = run(ctx, pg, batch, q, heads, BF16, 0.1, window, sinks)
    assert np.isnan(bad[at[20]:at[21]]).all() and np.isnan(bad[at[61] - 1]).all()
    for s in range(n):
        if s not in (20, 30, 60):
            assert np.array_equal(bad[at[s]:at[s + 1]], got[at[s]:at[s + 1]])


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 30])
def test_infinite_values_reach_only_rows_that_see_them(ctx, q_dtype, dtype, rows):
    """The last token's values hold NaN (and infinities where the type has
    them): rows before it are as if they were not there, its own row has them."""
    print(f"[gpu] not finite: {q_dtype}/{dtype} rows {rows}", flush=True)
    rng = np.random.default_rng(rows + dtype)
    n = 75
    pg = R.Paged(ctx, rng, dtype, 1, 64, 16, [n])
    odd = [np.nan] if dtype == E4M3 else [np.inf, -np.inf, np.nan]
    last = pg.real["v"][0][n - 1, 0].copy()
    for i, x in enumerate(odd):
        last[5 + 17 * i] = x
    words = R.encode(last, dtype)
    pg.put("v", 0, words[None, None], [n - 1])
    pg.upload()
    q = R.encode(rng.standard_normal((rows, 4, 64)), q_dtype)
    got, _ = run(ctx, pg, pg.batch([rows]), q, 4, q_dtype, 0.125)
    want, bound = expected(pg, q, [rows], 4, q_dtype, 0.125, 0, 0)
    check(got[:-1], want[:-1], bound[:-1])
    clean = np.isfinite(last)
    check(got[-1][:, clean], want[-1][:, clean], bound[-1][:, clean])
    for i, x in enumerate(odd):
        assert np.array_equal(got[-1][:, 5 + 17 * i], np.full(4, x), equal_nan=True)


@pytest.mark.parametrize("rows", [1, 40])
def test_bad_pages_lengths_and_row_ranges(ctx, rows):
    """NaN for sequences with an id of no page or an impossible length, others
    as they should be; rows of no sequence stay as they were. Ids of pages that
    no row sees are not looked at."""
    print(f"[gpu] bad pages, rows {rows}", flush=True)
    rng = np.random.default_rng(rows)
    lens = [300] * 6
    pg = R.Paged(ctx, rng, BF16, 2, 128, 16, lens).upload()
    pg.table[1, 18] = pg.n_pages       # one past the last
    pg.table[2, 3] = -1                # in the window's gap below, seen without it
    pg.kv_len[3] = 301                 # above max_kv
    pg.kv_len[4] = -5
    nr = [rows] * 6
    batch = pg.batch(nr, n_rows=6 * rows + 5, max_kv=300)
    pg.kv_len = lens
    q = R.encode(rng.standard_normal((6 * rows + 5, 4, 128)), BF16)
    for window in (0, 100):
        got, _ = run(ctx, pg, batch, q, 4, BF16, 0.1, window, 16)
        want, bound = expected(pg, q, nr, 4, BF16, 0.1, window, 16)
        ok = [0, 5] + ([2] if window else [])
        for s in range(6):
            part = slice(s * rows, (s + 1) * rows)
            if s in ok:
                check(got[part], want[part], bound[part])
            elif s != 2:
                assert np.isnan(got[part]).all(), s
        if not window:
            assert np.isnan(got[2 * rows:3 * rows]).all()
        fill = R.decode(np.full(1, 0x5A5A, np.uint16), BF16)[0]
        assert (got[6 * rows:] == fill).all()
    # row ranges out of order or beyond the rows: left out
    start = np.cumsum([0] + nr).astype(np.int32)
    start[4] = 6 * rows + 6
    pg.d_start.write(start)
    got, _ = run(ctx, pg, batch, q, 4, BF16, 0.1, 100, 16)
    assert (got[3 * rows:4 * rows] == fill).all() and (got[4 * rows:5 * rows] == fill).all()
    check(got[:rows], want[:rows], bound[:rows])


@pytest.mark.parametrize("rows", [1, 50])
def test_strided_rows_leave_the_gaps(ctx, rows):
    """q and out as slices of wider rows."""
    rng = np.random.default_rng(9)
    lens = [90, 130]
    pg = R.Paged(ctx, rng, BF16, 2, 64, 128, lens, order="token").upload()
    heads, width = 6, 6 * 64 + 72
    n = 2 * rows
    q = R.encode(rng.standard_normal((n, width)), F32)
    qd, out = ctx.upload(q), ctx.upload(np.full((n, width), 0x5A5A5A5A, np.uint32))
    op = wpcg.PagedAttention(ctx, pg.kv, pg.batch([rows] * 2), heads, F32, scale=0.2, q_stride=width, out_stride=width)
    op.run(qd, out)
    ctx.sync()
    bits = out.read(np.uint32, n * width).reshape(n, width)
    assert (bits[:, heads * 64:] == 0x5A5A5A5A).all()
    x = np.ascontiguousarray(q[:, :heads * 64]).reshape(n, heads, 64)
    check(R.decode(np.ascontiguousarray(bits[:, :heads * 64]), F32).reshape(n, heads, 64),
          *expected(pg, x, [rows] * 2, heads, F32, 0.2, 0, 0))


@pytest.mark.parametrize("rows", [1, 60])
def test_pages_beyond_32_bit_offsets(ctx, rows):
    """A cache of 5 GiB keys and as many values, the sequence's pages at its
    far end."""
    print(f"[gpu] far pages, rows {rows}", flush=True)
    rng = np.random.default_rng(4)
    hkv, d, page = 2, 128, 16
    elems = hkv * page * d
    total = (5 << 30) // (2 * elems)
    pg = R.Paged(ctx, rng, BF16, hkv, d, page, [100], spare=0)
    near = {n: pg.bits[n] for n in "kv"}
    big = [ctx.alloc(total * elems * 2) for _ in range(2)]
    first = total - pg.n_pages
    for b, n in zip(big, "kv"):
        wpcg.check(wpcg.lib.wpcg_memcpy_h2d(ctx.h, b.ptr.value + first * elems * 2, near[n].ctypes.data,
                                            near[n].nbytes))
    pg.kv = wpcg.PagedKv(ctx, total, page, hkv, d, BF16, k=big[0], v=big[1])
    keep = pg.table.copy()
    pg.table[0, :7] += first
    batch = pg.batch([rows])
    pg.table = keep
    q = R.encode(rng.standard_normal((rows, 8, d)), BF16)
    got, _ = run(ctx, pg, batch, q, 8, BF16, 0.09)
    check(got, *expected(pg, q, [rows], 8, BF16, 0.09, 0, 0))
    for b in big:
        b.free()


@pytest.mark.parametrize("rows", [1, 40])
def test_captured_graph_follows_the_lengths(ctx, rows):
    """One graph, replayed while the lengths change on the device, with other
    calls (and another operator object with its own workspace) between."""
    print(f"[gpu] graph, rows {rows}", flush=True)
    rng = np.random.default_rng(rows + 1)
    full = [900, 1500]
    pg = R.Paged(ctx, rng, BF16, 2, 128, 16, full).upload()
    batch = pg.batch([rows] * 2)
    q = R.encode(rng.standard_normal((2 * rows, 8, 128)), F32)
    qd = ctx.upload(q)
    outs = [ctx.alloc(q.nbytes) for _ in range(2)]
    ops = [wpcg.PagedAttention(ctx, pg.kv, batch, 8, F32, scale=0.09) for _ in range(2)]
    assert ops[0].workspace_bytes > 0
    g = ctx.capture(lambda: ops[0].run(qd, outs[0]))
    g2 = ctx.capture(lambda: ops[1].run(qd, outs[1]))
    for lens in ([900, 1500], [rows, 777], [450, rows + 1], [900, 1500]):
        pg.d_len.write(np.array(lens, np.int32))
        outs[0].write(np.full(q.size, 0xFFFFFFFF, np.uint32))
        g.launch()
        g2.launch()
        g.launch()
        ctx.sync()
        pg.kv_len = lens
        kept = pg.real
        pg.real = {n: [x[:m] for x, m in zip(kept[n], lens)] for n in "kv"}
        want, bound = expected(pg, q, [rows] * 2, 8, F32, 0.09, 0, 0)
        pg.real = kept
        bits = [o.read(np.uint32, q.size).reshape(q.shape) for o in outs]
        assert np.array_equal(bits[0], bits[1])
        check(R.decode(bits[0], F32), want, bound)
    del g, g2


@pytest.mark.parametrize("max_kv", [1200, 60000])
def test_captured_graph_follows_the_row_ranges(ctx, max_kv):
    """One graph of a batch that both kernels may have parts of (the longer
    bound), replayed while sequences change from one new row to a prompt and
    back, with eager calls of another object between."""
    print(f"[gpu] graph of mixed rows, bound {max_kv}", flush=True)
    rng = np.random.default_rng(max_kv)
    full = [700, 90, 1100, 300, 64, 33]
    pg = R.Paged(ctx, rng, BF16, 2, 128, 16, full, width=max_kv // 16).upload()
    total = 320
    batch = pg.batch([1] * 6, n_rows=total, max_kv=max_kv, max_q=250)
    q = R.encode(rng.standard_normal((total, 8, 128)), BF16)
    qd = ctx.upload(q)
    outs = [ctx.alloc(q.nbytes) for _ in range(2)]
    ops = [wpcg.PagedAttention(ctx, pg.kv, batch, 8, BF16, scale=0.09) for _ in range(2)]
    g = ctx.capture(lambda: ops[0].run(qd, outs[0]))
    kept = pg.real
    for rows, lens in (([1, 90, 1, 200, 8, 9], full), ([250, 1, 0, 1, 64, 1], [250, 2, 0, 300, 64, 33]),
                       ([1] * 6, full), ([9, 9, 9, 9, 9, 9], [700, 90, 1100, 300, 64, 5]),
                       ([1, 90, 1, 200, 8, 9], full)):
        pg.d_len.write(np.array(lens, np.int32))
        pg.d_start.write(np.cumsum([0] + rows).astype(np.int32))
        for o in outs:
            o.write(np.full(q.size, 0xFFFF, np.uint16))
        g.launch()
        ops[1].run(qd, outs[1])
        g.launch()
        ctx.sync()
        pg.kv_len = lens
        pg.real = {n: [x[:m] for x, m in zip(kept[n], lens)] for n in "kv"}
        n = sum(rows)
        want, bound = expected(pg, q[:n], rows, 8, BF16, 0.09, 0, 0)
        pg.real = kept
        bits = [o.read(np.uint16, q.size).reshape(q.shape) for o in outs]
        assert np.array_equal(bits[0], bits[1]) and (bits[0][n:] == 0xFFFF).all()
        check(R.decode(bits[0][:n], BF16), want, bound)
    del g


def test_other_streams(ctx):
    """Calls of two objects on streams of other contexts, at once."""
    rng = np.random.default_rng(12)
    pg = R.Paged(ctx, rng, E4M3, 2, 64, 32, [2000, 1000], scales=True).upload()
    batch = pg.batch(None)
    q = R.encode(rng.standard_normal((2, 6, 64)), F32)
    qd = ctx.upload(q)
    want, bound = expected(pg, q, [1, 1], 6, F32, 0.125, 0, 0)
    others = [wpcg.Context(0) for _ in range(2)]
    ops = [wpcg.PagedAttention(ctx, pg.kv, batch, 6, F32, scale=0.125) for _ in others]
    outs = [ctx.alloc(q.nbytes) for _ in others]
    for _ in range(20):
        for o, op, out in zip(others, ops, outs):
            op.run(qd, out, o.stream)
    for o, out in zip(others, outs):
        o.sync()
        check(R.decode(out.read(np.uint32, q.size).reshape(q.shape), F32), want, bound)
        o.close()


def test_nothing_to_do(ctx):
    rng = np.random.default_rng(1)
    pg = R.Paged(ctx, rng, BF16, 1, 64, 16, [10]).upload()
    batch = pg.batch(None)
    q = ctx.upload(R.encode(rng.standard_normal((1, 1, 64)), BF16))
    for n_seq, n_rows in ((0, 0), (0, 1)):
        b = wpcg.KvBatch(n_seq, n_rows, batch.kv_len, batch.table, 2, 10)
        op = wpcg.PagedAttention(ctx, pg.kv, b, 1, BF16)
        op.run(q, q)
    # a batch that has room for tokens and holds none
    pg.d_len.write(np.zeros(1, np.int32))
    got, _ = run(ctx, pg, batch, R.encode(rng.standard_normal((1, 1, 64)), BF16), 1, BF16, 0.125)
    assert (got == 0).all()


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("rows,lens,max_q,n_rows,heads,hkv,d", [([60], [9000], 64, 3000, 8, 2, 128),
                                                                ([40, 0, 33, 1], [5000, 9, 3000, 2], 48, 900, 14, 2, 64)])
def test_rows_far_below_their_bound(ctx, q_dtype, dtype, rows, lens, max_q, n_rows, heads, hkv, d):
    """A batch that is split, n_rows a much looser bound than max_q of each
    sequence: the parts are the sequences' own, the rows behind stay as they were."""
    print(f"[gpu] loose rows: {q_dtype}/{dtype} rows {rows} of {n_rows}", flush=True)
    rng = np.random.default_rng(n_rows + q_dtype + 10 * dtype)
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, lens, scales=dtype == E4M3).upload()
    n = sum(rows)
    q = np.zeros((n_rows, heads, d), R.BITS[q_dtype])
    q[:n] = R.encode(rng.standard_normal((n, heads, d)) * 1.5, q_dtype)
    b = pg.batch(rows, n_rows=n_rows, max_q=max_q)
    got, op = run(ctx, pg, b, q, heads, q_dtype, 0.09)
    part = len(rows) * max_q * heads * (d + 2) * 4
    assert op.workspace_bytes >= 2 * part and op.workspace_bytes % part == 0
    check(got[:n], *expected(pg, q[:n], rows, heads, q_dtype, 0.09, 0, 0))
    fill = R.decode(np.full(1, 0x5A5A if q_dtype == BF16 else 0x5A5A5A5A, R.BITS[q_dtype]), q_dtype)[0]
    assert (got[n:] == fill).all()


def expected_rows(pg, q, rows, picked, q_dtype, scale, window, sinks):
    """As `expected`, for the picked rows of every sequence alone."""
    outs, bounds, at = [], [], 0
    for s, n in enumerate(rows):
        m, i = pg.kv_len[s], picked[s]
        o, mag, reach = R.attention(R.decode(q[at + i], q_dtype), pg.real["k"][s], pg.real["v"][s], m - n + i, scale,
                                    window, sinks)
        outs.append(o)
        bounds.append(R.attention_bound(o, mag, reach, pg.d, m, q_dtype))
        at += n
    return np.concatenate(outs), np.concatenate(bounds)


# Prompts of 256 columns a workgroup, a workgroup for every column block: whole
# (128 tiles, two look-ups of pages) and in parts that are joined, with and
# without a window. parts: of each (row, query head).
WIDE = [(64, [2050], [16384], 0, 0, 3), (128, [2050], [16384], 0, 0, 3), (64, [2050], [8192], 0, 0, 0),
        (128, [1100, 1000], [12000, 4000], 5000, 70, 3), (128, [1000, 3, 900], [12000, 12000, 7001], 5000, 70, 2)]


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("d,rows,lens,window,sinks,parts", WIDE)
def test_prompts_far_behind_in_a_sequence(ctx, dtype, d, rows, lens, window, sinks, parts):
    """Some rows of every sequence against 64 bits; the same call gives the same
    bits; a page that is none reaches the rows that see it and no other sequence."""
    print(f"[gpu] far prompts: {dtype} {d} rows {rows} lens {lens} window {window}", flush=True)
    rng = np.random.default_rng(d + sum(rows) + window + dtype)
    heads, hkv = 32, 8
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, lens, scales=dtype == E4M3).upload()
    n = sum(rows)
    q = R.encode(rng.standard_normal((n, heads, d)) * 1.5, BF16)
    b = pg.batch(rows)
    got, op = run(ctx, pg, b, q, heads, BF16, 0.1, window, sinks)
    # 256 columns: with 128 the parts would be others
    assert op.workspace_bytes == parts * n * heads * (d + 2) * 4
    at = np.cumsum([0] + rows)
    picked = [np.unique([0, r - 1, *rng.integers(0, r, 8 // len(rows))]) for r in rows]
    want, bound = expected_rows(pg, q, rows, picked, BF16, 0.1, window, sinks)
    check(np.concatenate([got[a + i] for a, i in zip(at, picked)]), want, bound)
    again, _ = run(ctx, pg, b, q, heads, BF16, 0.1, window, sinks)
    assert np.array_equal(got.view(np.uint64), again.view(np.uint64))
    t = lens[0] - rows[0] // 2  # a token of the first sequence's later rows
    pg.table[0, t // 16] = pg.n_pages + 9
    pg.d_table.write(pg.table)
    bad, _ = run(ctx, pg, b, q, heads, BF16, 0.1, window, sinks)
    first = t // 16 * 16 - (lens[0] - rows[0])  # the first row that sees the page
    assert np.isnan(bad[first + 16:at[1]]).all()
    assert np.array_equal(bad[at[1]:].view(np.uint64), got[at[1]:].view(np.uint64))
    whole = first // 64 * 64  # (column blocks of 64 rows)
    assert np.array_equal(bad[:whole].view(np.uint64), got[:whole].view(np.uint64))


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
@pytest.mark.parametrize("rows,heads", [(2, 8), (5, 16)])
def test_tiles_dealt_out_behind_a_window(ctx, q_dtype, dtype, rows, heads):
    """Tiles dealt out by lists that leave a gap between sinks and window: the
    lists are those of a sequence's rows together, sequences longer and shorter
    than the window, sinks that meet it; ids of pages in the gap are anything."""
    window, sinks = (12000, 6000)[dtype != E4M3], 300
    print(f"[gpu] dealt, window: {q_dtype}/{dtype} rows {rows} heads {heads}", flush=True)
    rng = np.random.default_rng(rows + q_dtype + 10 * dtype)
    n, hkv, d = 130, 4, 128
    lens = [int(x) + rows for x in rng.integers(0, 40, n)]
    lens[3], lens[70], lens[71], lens[100], lens[129] = 2 * window + 77, window + 1, 0, window + 310, window - 5
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, lens, scales=dtype == E4M3, width=2500)
    gap = (lens[3] - window) // 32  # a page in the gap's middle
    pg.upload()
    nr = [rows] * n
    nr[50], nr[100] = 0, 1
    q = R.encode(rng.standard_normal((sum(nr), heads, d)) * 1.5, q_dtype)
    b = pg.batch(nr, max_kv=40000, max_q=rows)
    keep = pg.table[3, gap]
    pg.table[3, gap] = -3
    pg.d_table.write(pg.table)
    pg.table[3, gap] = keep
    got, op = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, sinks)
    cols = 32 if rows * heads // hkv > 16 and dtype != F32 else 16
    assert op.workspace_bytes == 512 * cols * (d + 2) * 4 + 256 * 20
    want, bound = expected(pg, q, nr, heads, q_dtype, 0.09, window, sinks)
    check(got, want, bound)
    at = np.cumsum([0] + nr)
    pg.table[3, (lens[3] - 100) // 16] = pg.n_pages
    pg.d_table.write(pg.table)
    bad, _ = run(ctx, pg, b, q, heads, q_dtype, 0.09, window, sinks)
    assert np.isnan(bad[at[3]:at[4]]).all()
    assert np.array_equal(np.delete(bad, range(at[3], at[4]), 0), np.delete(got, range(at[3], at[4]), 0))


# Bounds of one batch for each way that a call's work is laid out: n_seq, n_rows,
# max_q, max_kv, heads, hkv, d, q_dtype, dtype, window, sinks.
LAYOUTS = [
    (1, 5, 8, 1317, 2, 1, 64, F32, E4M3, 0, 0), (2, 24, 6, 1569, 4, 1, 64, F32, BF16, 0, 4),    # 16 and 32 columns in parts
    (4, 24, 3, 40000, 64, 8, 64, F32, BF16, 0, 4),                                              # dealt out, 32 columns
    (3, 54, 9, 531, 8, 1, 64, BF16, E4M3, 0, 0), (1, 12, 6, 585, 8, 1, 64, F32, BF16, 0, 0),    # parts under a loose n_rows
    (5, 49, 98, 669, 7, 1, 64, F32, E4M3, 0, 0), (6, 8, 9, 783, 128, 2, 64, BF16, BF16, 0, 4),  # blocks looked for, in parts
    (34, 68, 1, 8724, 512, 8, 64, BF16, E4M3, 0, 4), (59, 60, 35, 8139, 5, 5, 64, BF16, BF16, 0, 4),  # 256 columns in parts
    (76, 81, 121, 7439, 28, 4, 64, BF16, E4M3, 0, 0), (76, 81, 121, 7439, 28, 4, 64, BF16, BF16, 6000, 100),  # ... looked for
    (64, 71, 58, 3544, 8, 8, 64, BF16, E4M3, 0, 4),                                             # 256 columns, a grid, whole
    (7, 8, 90, 9851, 28, 4, 128, F32, F32, 0, 0), (52, 86, 6, 7451, 14, 2, 64, F32, E4M3, 0, 4),  # from here on, few rows and
    (95, 98, 5, 1834, 14, 2, 128, F32, BF16, 0, 4), (7, 30, 27, 20000, 32, 4, 64, BF16, BF16, 0, 4),  # many in two parts
    (46, 80, 115, 3658, 8, 4, 128, BF16, BF16, 0, 4), (67, 70, 46, 1083, 8, 2, 128, F32, F32, 0, 0),
    (9, 1611, 5695, 5695, 28, 4, 64, BF16, E4M3, 0, 4), (64, 70, 8, 4153, 100, 5, 64, F32, E4M3, 0, 0),
    (87, 271, 7, 8682, 80, 4, 128, BF16, BF16, 0, 0), (89, 850, 65, 6249, 16, 4, 128, BF16, E4M3, 0, 4),
    (86, 162, 21, 6564, 56, 8, 64, BF16, E4M3, 0, 0), (86, 162, 21, 6564, 56, 8, 64, BF16, BF16, 5000, 90),
    (416, 418, 17, 5317, 40, 5, 64, BF16, BF16, 0, 0)]


@pytest.mark.parametrize("n_seq,n_rows,max_q,max_kv,heads,hkv,d,q_dtype,dtype,window,sinks", LAYOUTS)
def test_layouts(ctx, n_seq, n_rows, max_q, max_kv, heads, hkv, d, q_dtype, dtype, window, sinks):
    """Ragged batches within the bounds, of which every way to lay a call out
    over the chip is chosen for one: one sequence of the bound's length, the
    others of any, some empty, some without rows, rows of no sequence."""
    print(f"[gpu] layout: {n_seq} {n_rows} {max_q} {max_kv} {heads}/{hkv}x{d} {q_dtype}/{dtype}", flush=True)
    rng = np.random.default_rng(n_seq + n_rows + heads + d + q_dtype + 10 * dtype + window)
    left, rows = n_rows, []
    for s in range(n_seq):  # a few long row ranges, the others short
        most = min(max_q, max(0, left - (n_seq - s) // 2))
        rows.append(int(rng.integers(1, max(1, most) + 1) if rng.random() < max(0.25, 5 / n_seq) else rng.integers(0, 2)))
        rows[-1] = min(most, rows[-1])
        left -= rows[-1]
    # lengths: few long ones, for the references' sake, the rows at their ends
    lens = [min(max_kv, r + int(max_kv ** rng.random()) - 1) if rng.random() < 0.9 else 0 for r in rows]
    lens[int(np.argmax(rows))] = max_kv
    pg = R.Paged(ctx, rng, dtype, hkv, d, 16, lens, scales=dtype == E4M3).upload()
    n = sum(rows)
    q = np.zeros((n_rows, heads, d), R.BITS[q_dtype])
    q[:n] = R.encode(rng.standard_normal((n, heads, d)) * 1.5, q_dtype)
    got, _ = run(ctx, pg, pg.batch(rows, n_rows=n_rows, max_kv=max_kv, max_q=max_q), q, heads, q_dtype, 0.1, window, sinks)
    # the rows of the longest sequence by samples
    picked = [np.arange(r) if r * m < 20000 else np.unique([0, r - 1, *rng.integers(0, r, 6)]) for r, m in zip(rows, lens)]
    at = np.cumsum([0] + rows)
    want, bound = expected_rows(pg, q[:n], rows, picked, q_dtype, 0.1, window, sinks)
    check(np.concatenate([got[a + i] for a, i in zip(at, picked)]), want, bound)
    fill = R.decode(np.full(1, 0x5A5A if q_dtype == BF16 else 0x5A5A5A5A, R.BITS[q_dtype]), q_dtype)[0]
    assert (got[n:] == fill).all()


@pytest.mark.parametrize("q_dtype,dtype", TYPES)
def test_one_row_each_of_a_wide_group_in_parts(ctx, q_dtype, dtype):
    """Groups of 40 query heads (the kernel for many rows), no row starts, more
    rows than sequences: the parts are one row's of each sequence."""
    print(f"[gpu] wide group, loose rows: {q_dtype}/{dtype}", flush=True)
    rng = np.random.default_rng(q_dtype + 10 * dtype)
    lens = [3000, 1, 700, 0, 64]
    pg = R.Paged(ctx, rng, dtype, 2, 64, 16, lens, scales=dtype == E4M3).upload()
    q = R.encode(rng.standard_normal((9, 80, 64)) * 1.5, q_dtype)
    got, op = run(ctx, pg, pg.batch(None, n_rows=9), q, 80, q_dtype, 0.12)
    part = 5 * 80 * 66 * 4
    assert op.workspace_bytes >= 2 * part and op.workspace_bytes % part == 0
    check(got[:5], *expected(pg, q[:5], [1] * 5, 80, q_dtype, 0.12, 0, 0))
    fill = R.decode(np.full(1, 0x5A5A if q_dtype == BF16 else 0x5A5A5A5A, R.BITS[q_dtype]), q_dtype)[0]
    assert (got[5:] == fill).all()
