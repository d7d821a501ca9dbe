"""GPU tests of the operators behind several answers to one prompt as a server uses
them together: prompts written to pages that the device hands out, forked into
beams, steps whose attention reads a prompt once for its beams, log probabilities
that choose the next beams, pages given back and moved together on the way. Every
beam's logits are compared with the framework's own model in EXACT mode fed its
tokens one by one; and wpcg_model_score with its formulas in 64 bits.

Tolerance of the logits: as for the batched-serving operators (5e-5 of the logit
range), those of the scores are logprob_ref's."""
import numpy as np
import pytest

import logprob_ref as L
import wpcg
from pool_ref import Pool
from test_gpu_serve_step import DENSE, MOE, TOL, WIDE_HEADS, Server, model, tensors_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


def check_scores(got, logits, targets, top, temperature, tag):
    """got: {name: array}; every row of logits against 64 bits."""
    for i, x in enumerate(logits):
        w = L.row(x, -1 if targets is None else int(targets[i]), top, temperature)
        assert np.array_equal(got["top_ids"][i], w["ids"]), f"{tag} row {i}"
        assert abs(got["entropy"][i] - w["h"]) <= w["h_tol"], f"{tag} row {i}"
        some = w["best"] > -np.inf
        assert np.array_equal(got["top_logprob"][i] > -np.inf, some)
        assert (np.abs(got["top_logprob"][i][some] - w["best"][some]) <= w["best_tol"][some]).all(), f"{tag} row {i}"
        if targets is not None:
            assert got["rank"][i] == w["rank"], f"{tag} row {i}"
            lp = got["logprob"][i]
            assert lp == w["lp"] or abs(lp - w["lp"]) <= w["lp_tol"], f"{tag} row {i}: {lp} {w['lp']}"


class Branches(Server):
    """A server whose rows are groups of `width` beams, one group a prompt, and whose
    pages are a pool's. loose: tokens by the bounds, enough for shared prefixes to
    be chosen, or few."""

    def __init__(self, ctx, cfg, t, groups, width, pages, loose, rng):
        super().__init__(ctx, cfg, t, groups * width, rng)
        n, page = self.n_seq, self.PAGE
        self.groups, self.width, self.bound = groups, width, loose // page * page
        self.pool = wpcg.KvPool(ctx, pages, page, n, loose // page, kv_len=self.kv_len)
        self.kv_len.write(np.zeros(n, np.int32))
        self.twin = Pool(pages, page, n, loose // page)
        for y in self.layers:
            y["kv"] = wpcg.PagedKv(ctx, pages, page, self.hk, cfg["head_dim"], wpcg.DTYPE_F32)
        self.copies, self.result = ctx.alloc(12 * max(n, pages)), ctx.alloc(8)
        self.parent, self.grow = ctx.alloc(4 * n), ctx.alloc(4 * n)
        self.group_start = ctx.upload((np.arange(groups + 1) * width).astype(np.int32))
        self.prefix_len = ctx.upload(np.zeros(groups, np.int32))
        kvs = [y["kv"] for y in self.layers]
        self.fork = wpcg.KvFork(ctx, self.pool, self.copies, self.result, parent=self.parent, grow_each=self.grow)
        self.compact = wpcg.KvCompact(ctx, self.pool, self.copies, self.result, pages)
        self.copy = {m: wpcg.KvCopy(ctx, kvs, self.copies, self.result, m) for m in (n, pages)}

    def branch(self, parent, grow):
        """Rows continue their parents' and take grow tokens more each."""
        self.parent.write(np.asarray(parent, np.int32))
        self.grow.write(np.asarray(grow, np.int32))
        self.fork.run()
        self.copy[self.n_seq].run()
        self.twin.fork(parent, None, grow)
        self.same()

    def together(self):
        self.compact.run()
        self.copy[self.twin.n_pages].run()
        moved = self.twin.compact(self.twin.n_pages)[0]
        self.same()
        return len(moved)

    def same(self):
        self.ctx.sync()
        t = self.twin
        assert np.array_equal(self.pool.refs.read(np.int32, t.n_pages), t.refs)
        assert np.array_equal(self.pool.table.read(np.int32, t.table.size).reshape(t.table.shape), t.table)
        assert np.array_equal(self.kv_len.read(np.int32, t.n_seq), t.kv_len)

    def between(self, l, rows, max_q):
        y, b = self.layers[l], self.buf
        if (l, max_q) not in self.ops:
            batch = wpcg.KvBatch(self.n_seq, self.ROWS, self.kv_len, self.pool.table, self.bound // self.PAGE,
                                 self.bound, max_q=max_q, q_start=self.q_start)
            append = wpcg.KvAppend(self.ctx, y["kv"], batch, self.hq, q_norm=y["qn"], k_norm=y["kn"],
                                   eps=self.cfg["eps"], frequencies=self.freq)
            prefix = wpcg.KvPrefix(self.groups, self.group_start, self.prefix_len, self.bound)
            attend = wpcg.PrefixAttention(self.ctx, y["kv"], batch, prefix, self.hq) if max_q <= 2 else \
                wpcg.PagedAttention(self.ctx, y["kv"], batch, self.hq)

            def run():
                append.run(b["q"], b["k"], b["v"], b["q"])
                attend.run(b["q"], b["a"])
            # (lengths, groups and pages are read on the device: one capture for all steps)
            self.ops[(l, max_q)] = (self.ctx.capture(run), append, attend, prefix, batch)
        self.ops[(l, max_q)][0].launch()
        y["o_proj"].gemm_dev(b["a"], rows, b["o"], wpcg.DTYPE_F32_SPLIT)
        self.ctx.sync()
        return b["o"].read(np.float32, rows * self.cfg["hidden"]).reshape(rows, -1)

    def step(self, new):
        rows = [len(n) for n in new]
        self.len = self.twin.kv_len - np.array(rows, np.int32)  # the fork has counted them
        return super().step(new)


@pytest.mark.parametrize("name,cfg,seed,loose", [("heads of 64, shared", DENSE, 31, 1 << 18),
                                                 ("heads of 128, shared", WIDE_HEADS, 32, 1 << 17),
                                                 ("heads of 64, apart", DENSE, 33, 96)])
def test_beams_over_pages(ctx, name, cfg, seed, loose):
    print(f"[gpu] beams {name}", flush=True)
    rng = np.random.default_rng(seed)
    t = tensors_of(cfg, seed)
    m = model(ctx, cfg, t, wpcg.MODE_EXACT)
    G, W, V = 2, 4, cfg["vocab"]
    n = G * W
    srv = Branches(ctx, cfg, t, G, W, 60, loose, rng)
    prompts = [rng.integers(0, V, k).tolist() for k in (41, 16)]
    told = [list(p) for p in prompts for _ in range(W)]

    def check(lg, rows):
        for s, x in zip(rows, lg):
            m.reset()
            for tok in told[s]:
                exp, _ = m.forward_token(int(tok))
            err = np.max(np.abs(x - exp)) / (exp.max() - exp.min())
            assert err <= TOL, f"{name}: row {s} after {len(told[s])} tokens: {err:.2e} of range"

    # the prompts, each in its group's first row, read by one step
    first = [g * W for g in range(G)]
    grow = [len(prompts[s // W]) if s in first else 0 for s in range(n)]
    srv.branch(np.arange(n), grow)
    lg = srv.step([prompts[s // W] if s in first else [] for s in range(n)])
    last = lg[np.cumsum([len(p) for p in prompts]) - 1]
    check(last, first)
    srv.prefix_len.write(np.array([len(p) for p in prompts], np.int32))
    score = np.zeros(n)
    out = {"logprob": np.float32, "entropy": np.float32, "rank": np.int32, "top_ids": np.int32, "top_logprob": np.float32}
    dev = {k: ctx.alloc(4 * n * (W if k.startswith("top") else 1)) for k in out}
    prompt_op, step_op = wpcg.LogProbs(ctx, G, V, top=W), wpcg.LogProbs(ctx, n, V, top=W)

    def best(op, lg, targets=None):
        at = ctx.upload(lg)
        to = None if targets is None else ctx.upload(np.asarray(targets, np.int32))
        kw = {k: v for k, v in dev.items() if targets is not None or k not in ("logprob", "rank")}
        op.run(at, to, **kw)
        ctx.sync()
        got = {k: dev[k].read(out[k], len(lg) * (W if k.startswith("top") else 1)) for k in kw}
        got = {k: v.reshape(len(lg), -1) if k.startswith("top") else v for k, v in got.items()}
        check_scores(got, lg, targets, W, 1.0, name)
        return got["top_ids"], got["top_logprob"]

    ids, lps = best(prompt_op, last)
    parent = [s // W * W for s in range(n)]
    nxt = ids.reshape(n)
    score = lps.reshape(n).astype(np.float64)
    moved = changed = 0
    for turn in range(20):
        srv.branch(parent, [1] * n)
        told = [told[p] + [int(nxt[s])] for s, p in enumerate(parent)]
        lg = srv.step([[int(i)] for i in nxt])
        rows = list(range(n)) if turn % 5 in (0, 4) else [turn % n]
        check(lg[rows], rows)
        ids, lps = best(step_op, lg, nxt)
        parent, nxt = [], []
        for g in range(G):
            all_ = (score[g * W:g * W + W, None] + lps[g * W:g * W + W]).ravel()
            pick = np.argsort(-all_, kind="stable")[:W]
            # (answers stay apart as a sampler would have them: every third turn each row goes on)
            if turn % 3 == 2:
                pick = np.arange(W) * W
            parent += [g * W + int(i) // W for i in pick]
            nxt += [int(ids[g * W + i // W, i % W]) for i in pick]
            score[g * W:g * W + W] = all_[pick]
        nxt = np.array(nxt)
        changed += parent != list(range(n))
        if turn % 6 == 5:
            moved += srv.together()
    assert changed >= 5
    # the second prompt's answers end; the first one's best row goes on alone
    keep = np.zeros(n, np.int32)
    srv.branch([0] + [-1] * (n - 1), keep)
    assert (srv.twin.refs > 0).sum() == -(-(41 + 20) // srv.PAGE)
    moved += srv.together()
    assert moved > 0 and srv.twin.refs[:4].min() == 1 and srv.twin.refs[4:].max() == 0
    srv.branch(np.arange(n), [2] + [0] * (n - 1))
    new = rng.integers(0, V, 2).tolist()
    lg = srv.step([new] + [[]] * (n - 1))
    for i in range(2):
        told[0] = told[0] + [new[i]]
        check(lg[i:i + 1], [0])
    m.close()


@pytest.mark.parametrize("name,cfg,mode,seed", [("dense-fast", DENSE, wpcg.MODE_FAST, 41),
                                                ("dense-exact", DENSE, wpcg.MODE_EXACT, 42),
                                                ("moe-fast", MOE, wpcg.MODE_FAST, 43)])
def test_model_score(ctx, name, cfg, mode, seed):
    print(f"[gpu] score {name}", flush=True)
    rng = np.random.default_rng(seed)
    V = cfg["vocab"]
    m = model(ctx, cfg, tensors_of(cfg, seed), mode)
    m.prefill(rng.integers(0, V, 20).astype(np.uint32))
    for n, top, temp in ((5, 3, 1.0), (1, 64, 0.7), (64, 0, 1.0), (2, 1, 3.0), (9, 20, 0.0)):
        tokens = rng.integers(0, V, n).astype(np.uint32)
        targets = np.append(tokens[1:].astype(np.int32), rng.integers(0, V))
        _, lg = m.verify(tokens, want_logits=True)
        m.set_position(20)
        got = m.score(tokens, targets, temperature=temp, top=top)
        assert m.position() == 20 + n
        check_scores(got, lg, targets, top, temp, f"{name} {n}")
        # the places are as steps leave them
        l1 = m.forward_token(3)[0]
        m.set_position(20)
        m.verify(tokens)
        l2 = m.forward_token(3)[0]
        assert np.array_equal(l1, l2)
        m.set_position(20)
        bare = m.score(tokens, top=top, temperature=temp)
        assert set(bare) == {"entropy", "top_ids", "top_logprob"}
        assert all(np.array_equal(bare[k], got[k]) for k in bare)
        m.set_position(20)
    # an answer in turns has the score of the answer
    answer = rng.integers(0, V, 31).astype(np.uint32)
    targets = np.append(answer[1:].astype(np.int32), -1)
    whole = m.score(answer, targets)
    assert whole["logprob"][30] == -np.inf and whole["rank"][30] == 0
    m.set_position(20)
    parts = [m.score(answer[a:b], targets[a:b])["logprob"] for a, b in ((0, 10), (10, 11), (11, 31))]
    m.set_position(20)
    _, lg = m.verify(answer, want_logits=True)
    m.set_position(20)
    # logits of either are off by TOL of the range, and ln Z by as much as they
    off = np.abs(np.concatenate(parts)[:30] - whole["logprob"][:30])
    assert (off <= 4 * TOL * (lg.max(-1) - lg.min(-1))[:30]).all(), off.max()
    for bad, text in ((lambda: m.score(answer[:0]), "1..64"), (lambda: m.score(np.zeros(65)), "1..64"),
                      (lambda: m.score(np.array([1, V])), "out of range"), (lambda: m.score(answer, top=65), "top")):
        with pytest.raises(wpcg.WpcgError, match=text):
            bad()
    with pytest.raises(ValueError, match="targets"):
        m.score(answer, targets[:5])
    assert m.position() == 20
    m.verify(np.zeros(60, np.uint32))
    with pytest.raises(wpcg.WpcgError, match="full"):
        m.score(np.zeros(17))
    assert m.position() == 80
    m.close()
