"""GPU tests of the batched-serving operators as a server uses them together:
several sequences of a dense model share steps (prompts, single tokens,
drafts), their projections one batched GEMM each, with the append and the
attention between them and the sampled verification behind the head. Every
row's logits are compared with the framework's own model in EXACT mode fed
the same tokens one by one (which is bit-identical to the oracle), and
wpcg_model_verify_sampled with its rule in 64 bits.

Tolerance: the batched GEMMs carry x as two bf16 terms as the model's prefill
does, and the pages are F32, so the steps may be off by what the prefill may
(5e-5 of the logit range)."""
import numpy as np
import pytest

import serve_ref as R
import wpcg
from wpcg import synth

pytestmark = pytest.mark.gpu

TOL = 5e-5
DENSE = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, inter=512, vocab=1000,
             n_experts=0, top_k=0, moe_inter=0, norm_topk=1, tied=1, max_pos=96, eps=1e-6, rope_theta=1e6)
WIDE_HEADS = dict(DENSE, hidden=384, n_heads=16, n_kv_heads=2, head_dim=128, vocab=900)
MOE = dict(DENSE, inter=0, n_experts=16, top_k=4, moe_inter=128, tied=0)


@pytest.fixture(scope="module")
def ctx():
    c = wpcg.Context(0)
    yield c
    c.close()


def tensors_of(cfg, seed):
    t = dict(synth.model_tensors(cfg, 4, seed, wpcg.encode))
    rng = np.random.default_rng(seed + 1)
    for name, w in t.items():
        if name.endswith("norm.weight"):
            t[name] = (0.6 + 0.8 * rng.random(w.size)).astype(np.float32)
    return t


def model(ctx, cfg, tensors, mode):
    m = wpcg.Model(ctx, 4, wpcg.ModelConfig(**cfg))
    for name, w in tensors.items():
        m.set_tensor(name, w)
    m.set_mode(mode)
    return m


def norm(x, w, eps):
    y = x.astype(np.float64)
    return (y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w).astype(np.float32)


class Server:
    """A dense model over pages: each step takes each sequence's new tokens."""
    PAGE, WIDTH, ROWS = 16, 6, 64

    def __init__(self, ctx, cfg, t, n_seq, rng):
        self.ctx, self.cfg, self.t, self.n_seq = ctx, cfg, t, n_seq
        h, d = cfg["hidden"], cfg["head_dim"]
        self.hq, self.hk = cfg["n_heads"], cfg["n_kv_heads"]
        qd, kd, inter = self.hq * d, self.hk * d, cfg["inter"]

        def lin(name, out, inp):
            return wpcg.WpcLinear.from_blocks(ctx, 4, t[name], out, inp)
        self.embed = lin("model.embed_tokens.weight", cfg["vocab"], h)
        self.freq = ctx.upload(wpcg.rope_frequencies(cfg["rope_theta"], d))
        self.kv_len = ctx.alloc(4 * n_seq)
        pages = n_seq * self.WIDTH + 2
        self.table = ctx.upload(rng.permutation(pages)[:n_seq * self.WIDTH].astype(np.int32))
        self.q_start = ctx.alloc(4 * (n_seq + 1))
        self.layers = []
        for l in range(cfg["n_layers"]):
            p = f"model.layers.{l}."
            y = {n: lin(p + n + ".weight", *s) for n, s in {
                "self_attn.q_proj": (qd, h), "self_attn.k_proj": (kd, h), "self_attn.v_proj": (kd, h),
                "self_attn.o_proj": (h, qd), "mlp.gate_proj": (inter, h), "mlp.up_proj": (inter, h),
                "mlp.down_proj": (h, inter)}.items()}
            y = {n.split(".")[1]: v for n, v in y.items()}
            y["qn"], y["kn"] = (ctx.upload(t[p + f"self_attn.{c}_norm.weight"]) for c in "qk")
            y["n1"], y["n2"] = t[p + "input_layernorm.weight"], t[p + "post_attention_layernorm.weight"]
            y["kv"] = wpcg.PagedKv(ctx, pages, self.PAGE, self.hk, d, wpcg.DTYPE_F32)
            self.layers.append(y)
        self.buf = {n: ctx.alloc(4 * self.ROWS * w) for n, w in
                    {"q": qd, "k": kd, "v": kd, "a": qd, "o": h}.items()}
        self.len = np.zeros(n_seq, np.int32)
        self.ops, self.graphs = {}, {}

    def between(self, l, rows, max_q):
        """Append, attention and o_proj of a layer, as one captured graph where
        every sequence has one row."""
        y, b = self.layers[l], self.buf
        key = (l, max_q)
        if key not in self.ops:
            batch = wpcg.KvBatch(self.n_seq, self.ROWS, self.kv_len, self.table, self.WIDTH,
                                 self.PAGE * self.WIDTH, max_q=max_q, q_start=self.q_start)
            self.ops[key] = (
                wpcg.KvAppend(self.ctx, y["kv"], batch, self.hq, q_norm=y["qn"], k_norm=y["kn"],
                              eps=self.cfg["eps"], frequencies=self.freq),
                wpcg.PagedAttention(self.ctx, y["kv"], batch, self.hq))

        def run():
            append, attend = self.ops[key]
            append.run(b["q"], b["k"], b["v"], b["q"])
            attend.run(b["q"], b["a"])
            y["o_proj"].gemm_dev(b["a"], rows, b["o"], wpcg.DTYPE_F32_SPLIT)
        if max_q == 1 and rows == self.n_seq:
            if l not in self.graphs:
                self.graphs[l] = self.ctx.capture(run)
            self.graphs[l].launch()
        else:
            run()
        self.ctx.sync()
        return b["o"].read(np.float32, rows * self.cfg["hidden"]).reshape(rows, -1)

    def step(self, new):
        """new: token ids per sequence; logits of all their rows."""
        rows = [len(n) for n in new]
        self.len += rows
        self.kv_len.write(self.len)
        self.q_start.write(np.cumsum([0] + rows).astype(np.int32))
        x = np.stack([self.embed.embed(int(t)) for n in new for t in n])
        for l, y in enumerate(self.layers):
            xn = norm(x, y["n1"], self.cfg["eps"])
            for n in "qkv":
                self.buf[n].write(y[n + "_proj"].gemm(xn, wpcg.DTYPE_F32_SPLIT))
            x = x + self.between(l, sum(rows), max(rows))
            xn = norm(x, y["n2"], self.cfg["eps"])
            g, u = (y[n].gemm(xn, wpcg.DTYPE_F32_SPLIT) for n in ("gate_proj", "up_proj"))
            act = wpcg.silu_mul(self.ctx, g.ravel(), u.ravel()).reshape(g.shape)
            x = x + y["down_proj"].gemm(act, wpcg.DTYPE_F32_SPLIT)
        return self.embed.gemm(norm(x, self.t["model.norm.weight"], self.cfg["eps"]), wpcg.DTYPE_F32_SPLIT)


def greedy(lg):
    return int(np.argmax(lg))


@pytest.mark.parametrize("name,cfg,seed", [("heads of 64", DENSE, 11), ("heads of 128", WIDE_HEADS, 12)])
def test_steps_of_several_sequences_match_the_model(ctx, name, cfg, seed):
    print(f"[gpu] serving {name}", flush=True)
    rng = np.random.default_rng(seed)
    t = tensors_of(cfg, seed)
    m = model(ctx, cfg, t, wpcg.MODE_EXACT)
    srv = Server(ctx, cfg, t, 3, rng)
    told = [[], [], []]      # the tokens that each sequence was fed and kept
    V = cfg["vocab"]

    def check(lg, new):
        at = 0
        for s, n in enumerate(new):
            m.reset()
            for tok in told[s]:
                m.forward_token(tok)
            for i, tok in enumerate(n):
                exp, _ = m.forward_token(int(tok))
                err = np.max(np.abs(lg[at + i] - exp)) / (exp.max() - exp.min())
                assert err <= TOL, f"{name}: sequence {s} row {i}: {err:.2e} of range"
            at += len(n)

    def step(new):
        lg = srv.step(new)
        check(lg, new)
        for s, n in enumerate(new):
            told[s] += [int(i) for i in n]
        ends = np.cumsum([len(n) for n in new]) - 1
        return lg, [greedy(lg[e]) for e in ends]

    _, nxt = step([rng.integers(0, V, n) for n in (5, 40, 17)])
    for _ in range(3):  # single tokens: one captured graph a layer, replayed
        _, nxt = step([[n] for n in nxt])
    # drafts: sequence 0 three drawn evenly, 1 none, 2 a right and a wrong one, greedily
    m.reset()
    for tok in told[2]:
        m.forward_token(tok)
    _, right = m.forward_token(nxt[2])
    new = [[nxt[0]] + [int(i) for i in rng.integers(0, V, 3)], [nxt[1]], [nxt[2], right, (right + 1) % V]]
    rows = [len(n) for n in new]
    lg = srv.step(new)
    check(lg, new)
    u, u_next = rng.random(sum(rows), dtype=np.float32), rng.random(3, dtype=np.float32)
    temp = np.array([1.0, 0.7, 0.0], np.float32)
    probs = np.full((sum(rows), V), 1.0 / V, np.float32)
    tokens = np.concatenate(new).astype(np.uint32)
    acc, out = ctx.alloc(12), ctx.alloc(4 * sum(rows))
    op = wpcg.DraftVerify(ctx, 3, sum(rows), max(rows), V, q_start=srv.q_start, temperature=ctx.upload(temp))
    op.run(ctx.upload(lg), ctx.upload(tokens), ctx.upload(u), ctx.upload(u_next), acc, out,
           draft_probs=ctx.upload(probs))
    ctx.sync()
    acc, out = acc.read(np.int32, 3), out.read(np.int32, sum(rows))
    at = np.cumsum([0] + rows)
    last = []
    for s in range(3):
        r = slice(at[s], at[s + 1])
        a, o = R.verify(lg[r], probs[r], tokens[r], u[r], u_next[s], temp[s])
        assert acc[s] == a and np.array_equal(out[r], o)
        last.append(int(o[a]))
        told[s] += [int(i) for i in new[s][:1 + a]]
        srv.len[s] -= rows[s] - 1 - a  # the rejected drafts' places are written anew
    assert acc[2] == 1
    for _ in range(2):
        _, last = step([[n] for n in last])
    m.close()


@pytest.mark.parametrize("name,cfg,mode,seed", [("dense-fast", DENSE, wpcg.MODE_FAST, 21),
                                                ("dense-exact", DENSE, wpcg.MODE_EXACT, 22),
                                                ("moe-fast", MOE, wpcg.MODE_FAST, 23)])
def test_model_verify_sampled(ctx, name, cfg, mode, seed):
    print(f"[gpu] sampled verification {name}", flush=True)
    rng = np.random.default_rng(seed)
    V = cfg["vocab"]
    m = model(ctx, cfg, tensors_of(cfg, seed), mode)
    m.prefill(rng.integers(0, V, 20).astype(np.uint32))
    seen = set()
    for n in (5, 1, 64, 2, 8):
        for kind in ("even", "near", "chosen", "greedy", "nan"):
            tokens = rng.integers(0, V, n).astype(np.uint32)
            u, u_next = rng.random(n - 1, dtype=np.float32), float(rng.random(dtype=np.float32))
            temp = 0.0 if kind == "greedy" else 0.8
            ids, lg = m.verify(tokens, want_logits=True)
            m.set_position(20)
            probs = None
            if kind in ("even", "greedy"):
                probs = np.full((n - 1, V), 1.0 / V, np.float32)
            elif kind in ("near", "nan"):
                x = lg[:n - 1].astype(np.float64) + 0.3 * rng.standard_normal((n - 1, V))
                probs = np.exp(x - x.max(-1, keepdims=True))
                probs = (probs / probs.sum(-1, keepdims=True)).astype(np.float32)
                if kind == "nan" and n > 2:
                    probs[1] = np.nan
            if kind == "chosen":  # certain to pass now and then: u at 0
                u[:n // 2] = 0
            if kind == "greedy":
                tokens[1:1 + n // 2] = ids[:len(tokens[1:1 + n // 2])]
                ids, lg = m.verify(tokens, want_logits=True)
                m.set_position(20)
            got, out = m.verify_sampled(tokens, u, u_next, draft_probs=probs, temperature=temp)
            full = None if probs is None else np.vstack([probs, np.zeros((1, V), np.float32)])
            if kind == "nan" and n > 2:
                a, o = R.verify(lg[:2], full[:2], tokens[:2], u, u_next, temp)
                if a == 1:  # the second draft's row of probabilities is NaN: rejected, the next token from p
                    o = R.verify(lg[1:2], None, tokens[1:2], u, u_next, temp)[1]
                    o = np.concatenate([tokens[1:2].astype(np.int32), o])
                o = np.concatenate([o, np.full(n - 2, -1, np.int32)])
            else:
                a, o = R.verify(lg, full, tokens, u, u_next, temp)
            assert got == a and np.array_equal(out, o), f"{name} {kind} {n}: {got} {out} vs {a} {o}"
            seen.add(min(got, 2))
            assert m.position() == 20 + n
            # the kept tokens' places are good: the next step equals a fresh run
            m.set_position(20 + 1 + got)
            l1 = m.forward_token(int(out[got]))[0]
            m.set_position(20)
            for tok in tokens[:1 + got]:
                m.forward_token(int(tok))
            l2 = m.forward_token(int(out[got]))[0]
            assert np.max(np.abs(l1 - l2)) <= TOL * (l2.max() - l2.min())
            m.set_position(20)
    assert seen == {0, 1, 2}
    tok, u2 = np.arange(3, dtype=np.uint32), [0.5, 0.5]
    for bad in (lambda: m.verify_sampled(tok[:0], [], 0.5), lambda: m.verify_sampled(tok, [0.5, 1.0], 0.5),
                lambda: m.verify_sampled(tok, [0.5, np.nan], 0.5), lambda: m.verify_sampled(tok, u2, -0.1),
                lambda: m.verify_sampled(np.array([1, V, 2]), u2, 0.5),
                lambda: m.verify_sampled(np.zeros(65), np.zeros(64), 0.5)):
        with pytest.raises(wpcg.WpcgError):
            bad()
    with pytest.raises(ValueError):
        m.verify_sampled(tok, [0.5], 0.5)
    assert m.position() == 20
    m.verify(np.zeros(60, np.uint32))
    with pytest.raises(wpcg.WpcgError, match="full"):
        m.verify_sampled(np.zeros(17), np.zeros(16), 0.5)
    m.close()


def test_model_verify_sampled_at_infinite_temperature(ctx):
    """All ids alike: drafts chosen outright stand while u is below 1 / vocab."""
    m = model(ctx, DENSE, tensors_of(DENSE, 24), wpcg.MODE_FAST)
    V = DENSE["vocab"]
    m.prefill(np.arange(9, dtype=np.uint32))
    for u, kept in (([0.5 / V, 0.0005, 0.0011], 2), ([0.5, 0, 0], 0), ([0, 0, 0], 3)):
        got, out = m.verify_sampled(np.array([3, 500, 1, 999]), u, 0.2505, temperature=np.inf)
        m.set_position(9)
        assert got == kept and out[:kept].tolist() == [500, 1, 999][:kept] and (out[kept + 1:] == -1).all()
        # running sums of 1000 ones, of 999 without the rejected draft (500: behind the mark; 999)
        assert out[kept] == 250
    m.close()
