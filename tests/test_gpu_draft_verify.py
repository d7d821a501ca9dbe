"""GPU tests of wpcg_draft_verify against a plain 64-bit implementation:
accepted counts and every token equal. Probabilities in the operator are fp64
to 1e-12, so that a decision can differ only where a number falls that close
to a border; the inputs are seeded and do not."""
import numpy as np
import pytest

import serve_ref as R
import wpcg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


def case(rng, drafts, vocab, agree=0.4, temperature=None):
    """Logits, a drafter that is near the target, its drafts, and the numbers."""
    rows = [k + 1 for k in drafts]
    n = sum(rows)
    base = rng.standard_normal((n, vocab)) * 2.5
    logits = (base + agree * rng.standard_normal((n, vocab))).astype(np.float32)
    x = base + agree * rng.standard_normal((n, vocab))
    p = np.exp(x - x.max(-1, keepdims=True))
    probs = (p / p.sum(-1, keepdims=True)).astype(np.float32)
    tokens = rng.integers(0, vocab, n).astype(np.uint32)
    for r in range(n - 1):
        tokens[r + 1] = min(vocab - 1, np.searchsorted(np.cumsum(probs[r].astype(np.float64)), rng.random()))
    return {"rows": rows, "logits": logits, "probs": probs, "tokens": tokens,
            "u": rng.random(n, dtype=np.float32), "u_next": rng.random(len(rows), dtype=np.float32),
            "t": np.full(len(rows), 1.0, np.float32) if temperature is None else np.asarray(temperature, np.float32)}


def want(c, with_probs=True):
    acc, out, at = [], [], 0
    for s, n in enumerate(c["rows"]):
        r = slice(at, at + n)
        a, o = R.verify(c["logits"][r], c["probs"][r] if with_probs else None, c["tokens"][r], c["u"][r],
                        c["u_next"][s], c["t"][s])
        acc.append(a)
        out.append(o)
        at += n
    return np.array(acc, np.int32), np.concatenate(out)


def run(ctx, c, with_probs=True, ragged=True, extra=0, start=None, temperature=True, op=None, pad=0):
    n, vocab = c["logits"].shape
    wide = vocab + pad

    def rows(x):
        y = np.full((n + extra, wide), np.nan, np.float32)
        y[:n, :vocab] = x
        return ctx.upload(y)

    q = ctx.upload((np.cumsum([0] + c["rows"]) if start is None else np.asarray(start)).astype(np.int32))
    lg, pr = rows(c["logits"]), rows(c["probs"]) if with_probs else None
    tk, u, un, t = (ctx.upload(np.concatenate([c[k], np.zeros(extra, c[k].dtype)]) if k in ("tokens", "u") else c[k])
                    for k in ("tokens", "u", "u_next", "t"))
    acc, out = ctx.upload(np.full(len(c["rows"]), 77, np.int32)), ctx.upload(np.full(n + extra, 99, np.int32))
    op = wpcg.DraftVerify(ctx, len(c["rows"]), n + extra, max(c["rows"]), vocab, q_start=q if ragged else None,
                          temperature=t if temperature else None, logits_stride=wide if pad else 0,
                          draft_stride=wide if pad else 0)
    op.workspace.write(np.full(op.workspace_bytes, 0xFF, np.uint8))
    op.run(lg, tk, u, un, acc, out, draft_probs=pr)
    ctx.sync()
    return acc.read(np.int32, len(c["rows"])), out.read(np.int32, n + extra)


@pytest.mark.parametrize("vocab", [1, 2, 63, 256, 1000, 2048, 2049, 9001, 151936])
@pytest.mark.parametrize("with_probs", [True, False])
def test_ragged_sequences(ctx, vocab, with_probs):
    print(f"[gpu] verify vocab {vocab} probs {with_probs}", flush=True)
    rng = np.random.default_rng(vocab)
    drafts = [4, 0, 1, 7, 2, 3] if vocab > 100000 else [4, 0, 1, 63, 2, 3, 5, 5, 5, 5]
    t = [1.0, 0.7, 0.0, 1.3, 0.05, -1.0, 0.9, 2.0, 30.0, 1.0][:len(drafts)]
    c = case(rng, drafts, vocab, temperature=t)
    c["tokens"][c["logits"].shape[0] // 2] = vocab + 5  # an id outside the vocabulary
    acc, out = run(ctx, c, with_probs)
    wa, wo = want(c, with_probs)
    assert np.array_equal(acc, wa) and np.array_equal(out, wo)
    assert vocab < 1000 or not with_probs or 0 < acc.sum() < sum(drafts)


def test_many_sequences_uniform_rows(ctx):
    """Enough rows for the longer chunks, no q_start, wider rows, no temperatures."""
    rng = np.random.default_rng(2)
    c = case(rng, [3] * 300, 2000)
    acc, out = run(ctx, c, ragged=False, temperature=False, pad=13)
    wa, wo = want(c)
    assert np.array_equal(acc, wa) and np.array_equal(out, wo)
    assert len(set(acc.tolist())) == 4


def test_many_ragged_sequences(ctx):
    """More sequences than are looked at in one step."""
    rng = np.random.default_rng(10)
    c = case(rng, [int(x) for x in rng.integers(0, 5, 700)], 400)
    acc, out = run(ctx, c, extra=5)
    wa, wo = want(c)
    assert np.array_equal(acc, wa) and np.array_equal(out[:len(wo)], wo) and (out[len(wo):] == 99).all()
    assert set(acc.tolist()) == {0, 1, 2, 3, 4}


def test_drafter_equal_to_the_target(ctx):
    """p = q to fp32: nearly every draft stands, and where one does not, the
    rest of p - q is rounding, compared in 64 bits."""
    rng = np.random.default_rng(3)
    c = case(rng, [5] * 40, 4000, agree=0.0)
    c["u"][:] = np.nextafter(np.float32(1), np.float32(0))
    acc, out = run(ctx, c)
    wa, wo = want(c)
    assert np.array_equal(acc, wa) and np.array_equal(out, wo)
    assert 0 < acc.sum() < 200


def test_masked_ties_and_rows_without_weight(ctx):
    rng = np.random.default_rng(4)
    c = case(rng, [2] * 8, 700, temperature=[1, 1, 0, 1, 1, 0, 0, 1])
    lg = c["logits"]
    lg[0:3, 100:] = -np.inf          # masked ids
    lg[3:6] = -3.4028235e38          # the type's lowest value everywhere: uniform
    lg[6:9] = np.round(lg[6:9])      # ties: the lowest id
    c["tokens"][7] = np.flatnonzero(lg[6] == lg[6].max())[0]
    lg[9] = -np.inf                  # no weight
    lg[12, 5] = np.nan
    lg[15] = -np.inf                 # greedy, no weight
    lg[18:21, ::2] = np.nan          # greedy over what is a number
    c["probs"][21] = 0               # a drafter's row that is none: p - q is p
    c["u"][:] = 0.01
    c["u_next"][:] = [0, 0.999, 0.5, 0.5, 0.5, 0.5, 0.5, 0.3]
    acc, out = run(ctx, c)
    wa, wo = want(c)
    assert np.array_equal(acc, wa) and np.array_equal(out, wo)
    assert (acc[3], out[9]) == (0, -1) and (acc[4], out[12]) == (0, -1) and (acc[5], out[15]) == (0, -1)


def test_low_temperatures_and_large_logits(ctx):
    """(x - max) / T is taken as a difference first: logits around 300 at
    temperatures down to the smallest float."""
    rng = np.random.default_rng(8)
    c = case(rng, [3] * 7, 3001, temperature=[1, 1e-3, 1e-6, 1e-12, 1e-20, 1e-38, 1e-45])
    c["logits"] += np.float32(300)
    lg = c["logits"]
    lg[4:8, 1000:1006] = lg[4:8].max(-1, keepdims=True) + np.float32(0.001) * np.arange(6, dtype=np.float32)
    lg[8:12, 500] = lg[8:12, 77] = lg[8:12].max(-1) + 1  # equal ones share the weight at any temperature
    lg[16:20, 2999] = lg[16:20, 5] = lg[16:20].max(-1) + 1
    for s in range(1, 7):  # drafts that are likely there
        c["tokens"][4 * s + 1:4 * s + 3] = lg[4 * s:4 * s + 2].argmax(-1)
    acc, out = run(ctx, c)
    wa, wo = want(c)
    assert np.array_equal(acc, wa) and np.array_equal(out, wo)
    assert acc[1:].min() >= 1


def test_bounds_of_u_next(ctx):
    """0 takes the first id with weight, the largest float below 1 the last ones."""
    rng = np.random.default_rng(5)
    c = case(rng, [0] * 4, 5000)
    c["logits"][:, :50] = -np.inf
    c["logits"][:, 4990:] = -np.inf
    c["u_next"][:] = [0, np.nextafter(np.float32(1), np.float32(0)), 0.5, 1e-30]
    acc, out = run(ctx, c)
    wa, wo = want(c)
    assert np.array_equal(out, wo) and out[0] == 50 and out[3] == 50


def test_row_ranges_that_are_none(ctx):
    """accepted -1 and no output for them; rows of no sequence stay as they were."""
    rng = np.random.default_rng(6)
    c = case(rng, [2] * 4, 300)
    wa, wo = want(c)
    acc, out = run(ctx, c, extra=3)
    assert np.array_equal(acc, wa) and np.array_equal(out, np.concatenate([wo, [99] * 3]))
    for start, bad in (([0, 3, 3, 9, 12], [1, 2]), ([0, 3, 6, 9, 16], [3]), ([-1, 3, 6, 9, 12], [0])):
        acc, out = run(ctx, c, extra=3, start=start)
        for s in range(4):
            if s in bad:
                assert acc[s] == -1
            else:
                assert acc[s] == wa[s] and np.array_equal(out[3 * s:3 * s + 3], wo[3 * s:3 * s + 3])
        assert (out[12:] == 99).all()


def test_captured(ctx):
    """One graph, replayed over new logits and numbers in the same buffers."""
    rng = np.random.default_rng(7)
    cs = [case(rng, [3, 1, 2], 5000, temperature=[1, 0, 0.8]) for _ in range(3)]
    n = 9
    dev = {k: ctx.upload(cs[0][k]) for k in ("logits", "probs", "tokens", "u", "u_next", "t")}
    q = ctx.upload(np.cumsum([0] + cs[0]["rows"]).astype(np.int32))
    acc, out = ctx.alloc(12), ctx.alloc(4 * n)
    op = wpcg.DraftVerify(ctx, 3, n, 4, 5000, q_start=q, temperature=dev["t"])
    g = ctx.capture(lambda: op.run(dev["logits"], dev["tokens"], dev["u"], dev["u_next"], acc, out,
                                   draft_probs=dev["probs"]))
    for c in cs + cs[:1]:
        for k, b in dev.items():
            b.write(c[k])
        g.launch()
        ctx.sync()
        wa, wo = want(c)
        assert np.array_equal(acc.read(np.int32, 3), wa) and np.array_equal(out.read(np.int32, n), wo)
    del g


def test_other_streams(ctx):
    """Calls of two objects on streams of other contexts, at once."""
    rng = np.random.default_rng(9)
    c = case(rng, [4, 2, 3], 30000)
    wa, wo = want(c)
    dev = {k: ctx.upload(c[k]) for k in ("logits", "probs", "tokens", "u", "u_next", "t")}
    q = ctx.upload(np.cumsum([0] + c["rows"]).astype(np.int32))
    others = [wpcg.Context(0) for _ in range(2)]
    n = len(wo)
    ops = [wpcg.DraftVerify(ctx, 3, n, 5, 30000, q_start=q, temperature=dev["t"]) for _ in others]
    accs, outs = ([ctx.alloc(4 * m) for _ in others] for m in (3, n))
    for _ in range(20):
        for o, op, acc, out in zip(others, ops, accs, outs):
            op.run(dev["logits"], dev["tokens"], dev["u"], dev["u_next"], acc, out, draft_probs=dev["probs"],
                   stream=o.stream)
    for o, acc, out in zip(others, accs, outs):
        o.sync()
        assert np.array_equal(acc.read(np.int32, 3), wa) and np.array_equal(out.read(np.int32, n), wo)
        o.close()


def test_infinite_temperature(ctx):
    """softmax(logits / inf): every id whose logit is above -inf alike, and no
    mark for greedy; sequences at other temperatures beside it."""
    rng = np.random.default_rng(11)
    inf = np.float32(np.inf)
    for vocab in (7, 3000, 20011):
        for with_probs in (True, False):
            c = case(rng, [3, 0, 5, 2, 1, 4, 0, 2], vocab, temperature=[inf, inf, inf, 0, 1, inf, inf, inf])
            c["u"][:4] = 0.5 / vocab  # below every p / q: drafts that were chosen outright pass too
            acc, out = run(ctx, c, with_probs)
            wa, wo = want(c, with_probs)
            assert np.array_equal(acc, wa) and np.array_equal(out, wo), (vocab, with_probs)
            assert acc[0] == 3


def test_infinite_temperature_over_masked_ids(ctx):
    """Ids at -inf have no weight at any temperature, all others one and the
    same; rows of no weight, NaN or +inf accept nothing."""
    rng = np.random.default_rng(12)
    vocab, n = 5000, 12
    c = case(rng, [0] * n + [1, 1], vocab, temperature=[np.inf] * (n + 2))
    lg = c["logits"]
    lg[:] *= 1e30
    open_ids = [np.sort(rng.choice(vocab, int(k), replace=False)) for k in rng.integers(1, vocab, n + 2)]
    open_ids[0], open_ids[1] = np.array([4321]), np.arange(vocab)
    for r in range(n + 2):
        row = r if r <= n else n + 2
        keep = lg[row, open_ids[r]]
        lg[row] = -np.inf
        lg[row, open_ids[r]] = keep
    lg[9], lg[10, 3], lg[11, 3] = -np.inf, np.nan, np.inf
    # the drafts, chosen outright: an open id (probability 1 / k), a masked one
    k = len(open_ids[n])
    c["tokens"][n + 1], c["u"][n] = open_ids[n][k // 2], 0.9 / k
    c["tokens"][n + 3], c["u"][n + 2] = np.setdiff1d(np.arange(vocab), open_ids[n + 1])[0], 0
    acc, out = run(ctx, c, with_probs=False)
    for r in range(9):
        ids = open_ids[r]
        at = float(c["u_next"][r]) * len(ids)
        assert abs(at - round(at)) > 1e-6 and out[r] == ids[int(at)], r
    assert (out[9:12] == -1).all() and (acc[9:12] == 0).all()
    assert acc[n] == 1 and out[n] == c["tokens"][n + 1]
    ids = open_ids[n + 1]
    assert acc[n + 1] == 0 and out[n + 2] == ids[int(float(c["u_next"][n + 1]) * len(ids))] and out[n + 3] == -1


@pytest.mark.parametrize("vocab,block,second", [(2048, 1000, 1024), (4096, 1500, 2048 + 300), (26 * 2048, 5 * 2048 + 11, 13 * 2048),
                                                (600 * 2048, 3 * 2048, 333 * 2048)])
@pytest.mark.parametrize("rest", [False, True])
def test_the_drawn_id_has_weight(ctx, vocab, block, second, rest):
    """Two equal blocks of weights and u_next at 1/2: the running sum meets the
    mark where the first block ends, to rounding that depends on its order. Ids
    without weight between the blocks (masked, or with p below q) are never
    drawn: the last id of the first block or the first one of the second is."""
    rng = np.random.default_rng(vocab + rest)
    n = max(24, min(400, (1 << 23) // vocab))
    rows = [2] * n if rest else [1] * n
    total = sum(rows)
    at = np.arange(0, total, rows[0])  # the rows that the next tokens come from
    lg = np.full((total, vocab), 0.0 if rest else -np.inf, np.float32)
    x = (rng.standard_normal((n, block)) * 3).astype(np.float32)
    lg[at, :block] = lg[at, second:second + block] = x
    probs = np.ones((total, vocab), np.float32)
    probs[:, :block] = probs[:, second:second + block] = 0
    c = {"rows": rows, "logits": lg, "probs": probs, "tokens": np.full(total, vocab - 1, np.uint32),
         "u": np.full(total, np.nextafter(np.float32(1), np.float32(0))), "u_next": np.full(n, 0.5, np.float32),
         "t": np.full(n, 1, np.float32)}
    acc, out = run(ctx, c, with_probs=rest)
    assert (acc == 0).all()
    assert set(out[at].tolist()) <= {block - 1, second}


def test_one_workspace_for_calls_in_a_row(ctx):
    """Calls over other data one behind the other, without a wait between: the
    parts and counts that a call leaves are none of the next one's."""
    rng = np.random.default_rng(13)
    cs = [case(rng, [4, 1, 0, 3] * 6, 21000, agree=1.5) for _ in range(5)]
    n, k = len(cs[0]["tokens"]), len(cs[0]["rows"])
    q = ctx.upload(np.cumsum([0] + cs[0]["rows"]).astype(np.int32))
    op = wpcg.DraftVerify(ctx, k, n, 5, 21000, q_start=q)
    dev = [{x: ctx.upload(c[x]) for x in ("logits", "probs", "tokens", "u", "u_next")} for c in cs]
    order = [i for _ in range(4) for i in rng.permutation(5)]
    outs = [(ctx.alloc(4 * k), ctx.alloc(4 * n)) for _ in order]
    for i, (acc, out) in zip(order, outs):
        d = dev[i]
        op.run(d["logits"], d["tokens"], d["u"], d["u_next"], acc, out, draft_probs=d["probs"])
    ctx.sync()
    right = [want(c) for c in cs]
    for i, (acc, out) in zip(order, outs):
        assert np.array_equal(acc.read(np.int32, k), right[i][0]) and np.array_equal(out.read(np.int32, n), right[i][1])
    assert min(min(a) for a, _ in right) == 0  # (drafts that fall: the parts are of use)
