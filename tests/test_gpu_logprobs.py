"""GPU tests of wpcg_logprobs against a plain 64-bit implementation: sizes around
its chunks and segments, both types, strides, temperatures from greedy to infinite,
masked rows, ties of every extent, what is not finite; missing outputs, streams,
graphs. Bounds are derived in logprob_ref.row."""
import numpy as np
import pytest

import logprob_ref as P
import serve_ref as R
import wpcg
from serve_ref import BF16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


def run(ctx, bits, dtype, tokens, top, temperature=None, vocab=None, offset=0, stream=None, skip=()):
    """bits [rows][stride], of which vocab are the logits; offset: elements before the first row."""
    n, stride = bits.shape
    vocab = vocab or stride
    room = ctx.upload(np.concatenate([np.zeros(offset, bits.dtype), bits.ravel()]))

    class At:
        ptr = room.ptr.value + offset * bits.dtype.itemsize
    t = None if temperature is None else ctx.upload(np.asarray(temperature, np.float32))
    op = wpcg.LogProbs(ctx, n, vocab, top=top, dtype=dtype, temperature=t, logits_stride=0 if stride == vocab else stride)
    op.workspace.write(np.full(op.workspace_bytes, 0xFF, np.uint8))
    fill = {"logprob": (np.float32, (n,)), "entropy": (np.float32, (n,)), "rank": (np.int32, (n,)),
            "top_ids": (np.int32, (n, top)), "top_logprob": (np.float32, (n, top))}
    out = {k: ctx.upload(np.full(max(1, int(np.prod(s))) + 3, 77, d)) for k, (d, s) in fill.items()}
    op.run(At, ctx.upload(np.asarray(tokens, np.int32)), stream=stream, **{k: b for k, b in out.items() if k not in skip})
    ctx.sync()
    got = {}
    for k, (d, s) in fill.items():
        a = out[k].read(d, int(np.prod(s)) + 3)
        assert (a[int(np.prod(s)):] == 77).all()
        got[k] = a[:int(np.prod(s))].reshape(s)
    return got


def check(got, x, tokens, top, temperature=None):
    for i in range(len(x)):
        want = P.row(x[i], int(tokens[i]), top, 1.0 if temperature is None else float(temperature[i]))
        where = f"row {i} of {x.shape}"
        assert got["rank"][i] == want["rank"], where
        assert np.array_equal(got["top_ids"][i], want["ids"]), (where, got["top_ids"][i], want["ids"])
        if want["lp"] is None:
            assert np.isnan(got["logprob"][i]) and np.isnan(got["entropy"][i]) and np.isnan(got["top_logprob"][i]).all(), where
            continue
        for a, b, tol in ((got["logprob"][i], want["lp"], want["lp_tol"]), (got["entropy"][i], want["h"], want["h_tol"])):
            assert a == b or abs(a - b) <= tol, (where, a, b, tol)
        a, b = got["top_logprob"][i].astype(np.float64), want["best"]
        with np.errstate(invalid="ignore"):
            same = (a == b) | (np.abs(np.where(np.isfinite(b), a - b, np.inf)) <= want["best_tol"])
        assert same.all(), (where, a[~same], b[~same])


def logits(rng, n, v, dtype, width=2.0):
    bits = R.encode(rng.standard_normal((n, v)) * width, dtype)
    return bits, R.decode(bits, dtype)


SIZES = [1, 2, 63, 64, 65, 255, 256, 257, 1000, 2047, 2048, 2049, 4096, 8191, 8193, 32003, 151936]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", SIZES)
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_sizes(ctx, dtype, v, top):
    """More entries asked for than there are ids among them."""
    print(f"[gpu] logprobs {dtype} vocab {v} top {top}", flush=True)
    rng = np.random.default_rng(v + top)
    n = 3 if v > 10000 else 9
    bits, x = logits(rng, n, v, dtype)
    tokens = rng.integers(0, v, n)
    tokens[0], tokens[-1] = v - 1, 0
    got = run(ctx, bits, dtype, tokens, top)
    check(got, x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top", [1, 24, 25, 64])
def test_segments_that_do_not_fit_in_registers(ctx, dtype, top):
    rng = np.random.default_rng(170001 + top)
    bits, x = logits(rng, 2, 170001, dtype)
    tokens = rng.integers(0, 170001, 2)
    check(run(ctx, bits, dtype, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_rows(ctx, dtype):
    """Many rounds of workgroups."""
    rng = np.random.default_rng(8300)
    bits, x = logits(rng, 8300, 501, dtype)
    tokens = rng.integers(0, 501, 8300)
    got = run(ctx, bits, dtype, tokens, 3)
    some = np.append(np.arange(0, 8300, 13), 8299)
    check({k: a[some] for k, a in got.items()}, x[some], tokens[some], 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [1e-3, 0.1, 0.5, 1.0, 3.0, 5.0, 8.0, 20.0])
def test_flat_and_peaked(ctx, dtype, width):
    """Sums of nearly all ids, of some, and of hardly more than the maximum; the
    likeliest ids' log probabilities among them."""
    rng = np.random.default_rng(int(width * 1000))
    bits, x = logits(rng, 12, 4500, dtype, width)
    tokens = np.argsort(-x, -1)[np.arange(12), [0, 0, 0, 0, 1, 1, 2, 3, 10, 100, 1000, 4000]]
    check(run(ctx, bits, dtype, tokens, 5), x, tokens, 5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("stride,offset", [(5008, 0), (5001, 0), (5008, 1), (5003, 3)])
def test_strides_and_alignment(ctx, dtype, stride, offset):
    """Rows on 16 bytes and off them; what lies between them is not looked at."""
    rng = np.random.default_rng(stride + offset)
    v = 5000
    bits, x = logits(rng, 6, stride, dtype)
    bits[:, v:] = R.NAN_BITS[dtype]
    tokens = rng.integers(0, v, 6)
    check(run(ctx, bits, dtype, tokens, 7, vocab=v, offset=offset), x[:, :v], tokens, 7)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_temperatures(ctx, dtype):
    rng = np.random.default_rng(5)
    temp = np.array([1.0, 0.5, 0.7, 1.3, 3.0, 0.01, 100.0, np.inf, 0.0, -1.0, np.nan, 1e-30, 1e-45, 1e30], np.float32)
    n, v = len(temp), 3000
    bits, x = logits(rng, n, v, dtype)
    tokens = rng.integers(0, v, n)
    tokens[::2] = [int(np.argmax(r)) for r in x[::2]]
    check(run(ctx, bits, dtype, tokens, 9, temp), x, tokens, 9, temp)
    x[:, 1::3] = -np.inf  # masked ids: alike at +inf are only the others
    bits = R.encode(x, dtype)
    check(run(ctx, bits, dtype, tokens, 9, temp), R.decode(bits, dtype), tokens, 9, temp)


def test_confident_rows_keep_their_digits(ctx):
    """One id holds nearly everything: log p of 1 - s is -s, for s down to 1e-30."""
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((12, 5000)) * 0.1).astype(np.float32)
    tops = rng.integers(0, 5000, 12)
    x[np.arange(12), tops] = np.linspace(8, 80, 12).astype(np.float32)
    got = run(ctx, x.view(np.uint32), F32, tops, 2)
    check(got, x.astype(np.float64), tops, 2)
    assert (got["logprob"] < 0).all() and (got["logprob"][-1] > -1e-25).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_ties(ctx, dtype, top):
    """Equal logits in every number: all, two values, in one segment, across
    chunks, zeros of both signs, and a few ids above many equal ones."""
    print(f"[gpu] ties {dtype} top {top}", flush=True)
    rng = np.random.default_rng(top)
    v = 20000
    x = np.zeros((9, v))
    x[1] = rng.integers(0, 2, v)
    x[2] = -1.0
    x[2, 7000:7064] = 3.0
    x[3] = rng.integers(0, 40, v) / 8.0
    x[4] = np.where(rng.random(v) < 0.5, 0.0, -0.0)
    x[5, rng.integers(0, v, 15)] = 1.0
    x[6] = -np.inf
    x[6, 17::1000] = 2.0
    x[7] = np.repeat(rng.permutation(v // 50), 50) / 4.0
    x[8] = np.sort(rng.standard_normal(v))  # rising: the best all in the last segment
    bits = R.encode(x, dtype)
    x = R.decode(bits, dtype)
    tokens = np.array([v - 1, 5, 7063, 100, 19999, 3, 18017, 9000, v - 1])
    check(run(ctx, bits, dtype, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v,top", [(20001, 1), (40000, 20), (40000, 64), (170001, 20)])
def test_many_alike(ctx, dtype, v, top):
    """More equal candidates than can be sorted: rows masked by the type's lowest
    value but for a few ids (none, fewer and more than are asked for), neighbouring
    values in every number, and a value above, between and below many equal ones."""
    rng = np.random.default_rng(v + top)
    low = -3.4028234663852886e38 if dtype == F32 else -3.3895313892515355e38
    x = np.full((11, v), low)
    for i, n in enumerate((0, 1, top - 1, top, top + 1, 300)):
        x[i, rng.permutation(v)[:n]] = rng.standard_normal(n) * 3
    step = 2.0 ** (-23 if dtype == F32 else -7)
    x[6] = 1 + step * rng.integers(0, 6, v)
    x[7] = 1 + step * rng.integers(0, 2, v) * (np.arange(v) > v // 2)
    x[8] = np.where(rng.random(v) < 0.01, 2.0, 1.0)
    x[9] = np.where(np.arange(v) % 3 == 0, -1.0, np.where(np.arange(v) % 3 == 1, -1.0 - step, -1.0 - 2 * step))
    x[10] = np.where(rng.random(v) < 0.5, -np.inf, -5.0)
    bits = R.encode(x, dtype)
    x = R.decode(bits, dtype)
    tokens = np.array([0, v - 1] + [int(i) for i in rng.integers(0, v, 9)])
    check(run(ctx, bits, dtype, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_is_not_finite(ctx, dtype):
    """Masked rows and rows that are no distribution; the rows beside them stay
    right; lowest values of the type as masks."""
    rng = np.random.default_rng(8)
    v, n = 6000, 13
    _, x = logits(rng, n, v, dtype)
    low = -3.4028235e38 if dtype == F32 else -3.3895314e38
    x[0, :] = -np.inf
    x[1, 1:] = -np.inf
    x[2, 10] = np.nan
    x[3, 5999] = np.inf
    x[4, [3, 4000]] = np.inf
    x[5, rng.random(v) < 0.99] = -np.inf
    x[6, 2048:] = -np.inf
    x[7, rng.random(v) < 0.9] = low
    x[8, :] = np.nan
    x[9, :] = low
    x[10, :4096] = -np.inf
    x[11, :] = np.inf
    bits = R.encode(x, dtype)
    if dtype == BF16:
        bits = np.where(np.isinf(x), np.where(x > 0, 0x7F80, 0xFF80), bits).astype(np.uint16)
    x = R.decode(bits, dtype)
    tokens = np.array([0, 0, 10, 5999, 4, 77, 5000, 4, 9, 3, 5000, 2, 12])
    check(run(ctx, bits, dtype, tokens, 20), x, tokens, 20)
    greedy = np.zeros(n, np.float32)
    tokens[2] = np.nanargmax(x[2])
    tokens[3], tokens[4] = 5999, 3
    check(run(ctx, bits, dtype, tokens, 20, greedy), x, tokens, 20, greedy)


def test_tokens_outside(ctx):
    rng = np.random.default_rng(9)
    bits, x = logits(rng, 5, 700, F32)
    x[4, 699] = np.inf  # equal to what an absent token is compared with
    bits = x.astype(np.float32).view(np.uint32)
    tokens = np.array([-1, 700, 2 ** 31 - 1, -2 ** 31, 701])
    got = run(ctx, bits, F32, tokens, 3)
    assert (got["logprob"][:4] == -np.inf).all() and (got["rank"] == 0).all() and np.isnan(got["logprob"][4])
    assert np.isfinite(got["entropy"][:4]).all()


def test_missing_outputs(ctx):
    """Each output alone; without them nothing is written, and tokens may be missing."""
    rng = np.random.default_rng(10)
    bits, x = logits(rng, 4, 3000, F32)
    tokens = rng.integers(0, 3000, 4)
    names = ["logprob", "entropy", "rank", "top_ids", "top_logprob"]
    whole = run(ctx, bits, F32, tokens, 5)
    for one in names:
        got = run(ctx, bits, F32, tokens, 5, skip=[n for n in names if n != one])
        assert np.array_equal(got[one], whole[one])
        assert all((got[n] == 77).all() for n in names if n != one)
    op = wpcg.LogProbs(ctx, 4, 3000)
    d, h = ctx.upload(bits), ctx.alloc(16)
    op.run(d, entropy=h)
    ctx.sync()
    assert np.array_equal(h.read(np.float32, 4), whole["entropy"])
    with pytest.raises(wpcg.WpcgError, match="null"):
        op.run(d, rank=h)


def test_many_rows_streams_and_graphs(ctx):
    """More rows than workgroups are resident; the same bits from another stream
    and from replays of a graph whose inputs change, two graphs in turn."""
    print("[gpu] logprobs graphs", flush=True)
    rng = np.random.default_rng(11)
    n, v = 700, 4000
    bits, x = logits(rng, n, v, BF16)
    tokens = rng.integers(0, v, n)
    first = run(ctx, bits, BF16, tokens, 10)
    some = np.r_[0:5, 300:305, 695:700]
    check({k: a[some] for k, a in first.items()}, x[some], tokens[some], 10)
    other = wpcg.Context(0)
    again = run(ctx, bits, BF16, tokens, 10, stream=other.stream)
    other.sync()
    assert all(np.array_equal(first[k], again[k]) for k in first)

    def build(rows):
        d = {"x": ctx.alloc(rows * v * 2), "t": ctx.alloc(4 * rows), "lp": ctx.alloc(4 * rows), "ids": ctx.alloc(40 * rows)}
        op = wpcg.LogProbs(ctx, rows, v, top=10, dtype=BF16)
        return d, ctx.capture(lambda: op.run(d["x"], d["t"], logprob=d["lp"], top_ids=d["ids"])), op
    graphs = [build(33), build(5)]
    for turn in range(4):
        for (d, g, _), rows in zip(graphs, (33, 5)):
            at = 40 * turn
            d["x"].write(bits[at:at + rows])
            d["t"].write(tokens[at:at + rows].astype(np.int32))
            g.launch()
        ctx.sync()
        for (d, _, _), rows in zip(graphs, (33, 5)):
            at = 40 * turn
            assert np.array_equal(d["lp"].read(np.float32, rows), first["logprob"][at:at + rows])
            assert np.array_equal(d["ids"].read(np.int32, 10 * rows).reshape(rows, 10), first["top_ids"][at:at + rows])
    other.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [257, 300, 1000, 4096, 32003])
@pytest.mark.parametrize("top", [20, 64])
def test_ties_at_the_border(ctx, dtype, v, top):
    """The last of the best ids is one of many equal ones, zeros and powers of two among
    them, with none, a few and nearly enough above, and any number below: more
    candidates than can be sorted, in fewer segments than ids are asked for."""
    print(f"[gpu] ties at the border {dtype} {v} top {top}", flush=True)
    rng = np.random.default_rng(v + top + dtype)
    low = -3.4028234663852886e38 if dtype == F32 else -3.3895313892515355e38
    rows, tokens = [], []
    for tie in (0.0, 2.0, 1.0, -0.5):
        for below in ("spread", low, -1e4, -np.inf):
            for above, more in ((0, 10), (3, 90), (top - 1, 40)):
                x = tie - 1 - np.abs(rng.standard_normal(v)) if below == "spread" else np.full(v, below)
                n = top + more
                at = int(rng.integers(0, v - n + 1))
                x[at:at + n] = tie
                x[at + rng.permutation(n)[:above]] = tie + 1 + rng.integers(0, 4, above) / 4
                rows.append(x)
                tokens.append(at + n - 1)
    # rounded values in every number, and masks that leave 300 neighbours
    rows += [np.round(rng.standard_normal(v) * w) / 4 for w in (1, 4, 16)]
    x = np.full(v, -np.inf)
    at = int(rng.integers(0, max(1, v - 300)))
    x[at:at + 300] = np.round(rng.standard_normal(len(x[at:at + 300])) * 4) / 4
    rows.append(x)
    bits = R.encode(np.array(rows), dtype)
    if dtype == BF16:
        bits = np.where(np.isneginf(rows), 0xFF80, bits).astype(np.uint16)
    tokens += [int(i) for i in rng.integers(0, v, 4)]
    x = R.decode(bits, dtype)
    check(run(ctx, bits, dtype, np.array(tokens), top), x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v,top", [(32000, 20), (151936, 20), (151936, 64), (170016, 24)])
def test_ties_at_the_border_of_segments(ctx, dtype, v, top):
    """The same among the segments of 64 ids: more segments than can be sorted, the
    K-th best maximum at zero or two, in few of the groups that they are looked at in."""
    print(f"[gpu] ties of segments {dtype} {v} top {top}", flush=True)
    rng = np.random.default_rng(v + top + dtype)
    rows = []
    for tie in (0.0, 2.0, 1.0):
        for groups in ((5,), (5, 6, 40)):
            x = np.full(v, -1e4)
            segs = [s for s in range(v // 64) if s % 64 in groups]
            for s in segs:
                x[64 * s + rng.integers(0, 64, 2)] = tie
            for s in rng.permutation(segs)[:3]:
                x[64 * s + 7] = tie + 1
            rows.append(x)
    x = np.full(v, -1e4)  # ten above neighbouring zeros
    x[v // 2:v // 2 + 30 + top] = 0.0
    x[v // 2 + rng.permutation(30)[:10]] = rng.standard_normal(10) ** 2 + 0.25
    rows.append(x)
    bits = R.encode(np.array(rows), dtype)
    tokens = [int(i) for i in rng.integers(0, v, len(rows))]
    check(run(ctx, bits, dtype, np.array(tokens), top), R.decode(bits, dtype), tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_as_wide_as_the_type(ctx, dtype):
    """Differences beyond the type's range: at +inf all finite logits are alike, at
    temperatures of their size they are told apart; differences of the least numbers at
    the least temperatures."""
    rng = np.random.default_rng(12)
    v = 5000
    most = 3.4028234663852886e38 if dtype == F32 else 3.3895313892515355e38
    temp = np.array([np.inf, np.inf, np.inf, 1e38, 3.4e38, 2e37, 1e35, 1.0, 1e6, 1e-38, 1e-45, 3e-45, 1e-40], np.float32)
    x = rng.uniform(-1, 1, (len(temp), v)) * most
    x[1, ::2] = -np.inf
    x[2] = rng.standard_normal(v)
    x[2, ::3] = -most
    x[2, 17] = most
    x[7, 100:] = -most  # a mask beneath ordinary logits
    x[7, :100] = rng.standard_normal(100)
    x[8] = rng.standard_normal(v) * 1e6
    least = 2.0 ** (-149 if dtype == F32 else -133)
    x[9:] = rng.integers(-5, 6, (4, v)) * least
    x[9] = rng.integers(-5, 6, v) * 2.0 ** -127
    bits = R.encode(x, dtype)
    x = R.decode(bits, dtype)
    tokens = rng.integers(0, v, len(temp))
    tokens[3:7] = [int(np.argmax(r)) for r in x[3:7]]
    check(run(ctx, bits, dtype, tokens, 9, temp), x, tokens, 9, temp)
