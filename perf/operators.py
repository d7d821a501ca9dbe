"""The operators of batched serving over a paged key-value cache, and what their speed is measured on.

A serving step of several sequences does, in every layer, between the projections
that wpcg_linear_gemm runs:

  append   the new rows' queries and keys take the head norm and the rotation,
           keys and values go into the sequences' pages
  attend   each new row's attention over its sequence's pages: one row a
           sequence (decode), a few (drafts being verified) or many (prompts),
           causal, with a sliding window and first tokens that stay visible
           where the model has them

and, at the end of a speculative step,

  verify   drafted tokens accepted or rejected against the target's
           probabilities from given random numbers

Every case is one call. `own` chooses between the operators' plain form in torch
and the library's kernels. Head counts are those of the Qwen2.5-0.5B (14 / 2 of
64), Qwen3-4B (32 / 8 of 128) and Qwen3-30B-A3B (32 / 4 of 128) shapes that
bench.py and the tests run.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6
E4M3_MAX = 448.0
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}
# (query heads, key-value heads, head size)
HEADS = {"0.5b": (14, 2, 64), "4b": (32, 8, 128), "30b": (32, 4, 128)}


def listed():
    return [
        # one decode step of 64 sequences: their new tokens' q, k and v
        {"name": "append-decode-64", "kind": "append", "heads": "30b", "n_seq": 64, "rows": 1, "cached": 2000,
         "page": 16, "in": "f32", "q": "bf16", "cache": "bf16"},
        # three prompts, ragged, into an 8-bit cache
        {"name": "append-prompts", "kind": "append", "heads": "4b", "n_seq": 3, "rows": 2000, "cached": 70,
         "page": 64, "in": "f32", "q": "bf16", "cache": "e4m3"},
        # a small model's single sequence in full precision: latency
        {"name": "decode-one-short", "kind": "attend", "heads": "0.5b", "n_seq": 1, "rows": 1, "kv": 300, "window": 0,
         "sinks": 0, "page": 16, "q": "f32", "cache": "f32"},
        # a full decode batch, ragged lengths
        {"name": "decode-64", "kind": "attend", "heads": "30b", "n_seq": 64, "rows": 1, "kv": 4096, "window": 0,
         "sinks": 0, "page": 16, "q": "bf16", "cache": "bf16"},
        # one sequence deep in a long document, 8-bit cache
        {"name": "decode-131072", "kind": "attend", "heads": "4b", "n_seq": 1, "rows": 1, "kv": 131072, "window": 0,
         "sinks": 0, "page": 64, "q": "f32", "cache": "e4m3"},
        # streaming decode: a window of the last tokens and four sinks
        {"name": "decode-window-32", "kind": "attend", "heads": "4b", "n_seq": 32, "rows": 1, "kv": 12000,
         "window": 1024, "sinks": 4, "page": 32, "q": "f32", "cache": "bf16"},
        # the last token and four drafts of 16 sequences
        {"name": "attend-drafts-16x5", "kind": "attend", "heads": "4b", "n_seq": 16, "rows": 5, "kv": 6000,
         "window": 0, "sinks": 0, "page": 16, "q": "f32", "cache": "bf16"},
        # a long prompt
        {"name": "prompt-4096", "kind": "attend", "heads": "4b", "n_seq": 1, "rows": 4096, "kv": 4096, "window": 0,
         "sinks": 0, "page": 16, "q": "bf16", "cache": "bf16"},
        # two ragged prompts of a model with a window, 8-bit cache
        {"name": "prompt-window", "kind": "attend", "heads": "30b", "n_seq": 2, "rows": 5000, "kv": 6001,
         "window": 1024, "sinks": 4, "page": 32, "q": "bf16", "cache": "e4m3"},
        # the rest of a prompt behind cached tokens, in full precision
        {"name": "prompt-f32", "kind": "attend", "heads": "30b", "n_seq": 1, "rows": 777, "kv": 1300, "window": 0,
         "sinks": 0, "page": 16, "q": "f32", "cache": "f32"},
        # four drafts of one sequence: latency
        {"name": "verify-one", "kind": "verify", "n_seq": 1, "drafts": 4, "vocab": 151936},
        # a batch of sequences, up to five drafts each, some of them greedy
        {"name": "verify-64", "kind": "verify", "n_seq": 64, "drafts": 5, "vocab": 151936},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "attend", "verify"])
    heads = rng.choice(sorted(HEADS))
    if kind == "append":
        n = _log_int(rng, 1, 64)
        return {"kind": kind, "heads": heads, "n_seq": n, "rows": _log_int(rng, 1, max(1, 4000 // n)),
                "cached": rng.choice([0, _log_int(rng, 1, 2000)]), "page": rng.choice([16, 32, 64, 128]),
                "in": rng.choice(["f32", "f32", "bf16"]), "q": rng.choice(["f32", "bf16"]),
                "cache": rng.choice(["f32", "bf16", "e4m3"])}
    if kind == "verify":
        return {"kind": kind, "n_seq": _log_int(rng, 1, 64), "drafts": rng.randint(1, 5),
                "vocab": rng.choice([151936, 32768, _log_int(rng, 50, 151936)])}
    q = rng.choice(["f32", "bf16"])
    cache = rng.choice(["bf16", "e4m3"] + (["f32"] if q == "f32" else []))
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    c = {"kind": kind, "heads": heads, "window": window, "sinks": rng.choice([0, 1, 4, 20]) if window else 0,
         "page": rng.choice([16, 32, 64, 128]), "q": q, "cache": cache}
    form = rng.choice(["decode", "decode", "drafts", "prompt"])
    if form == "prompt":
        c.update(n_seq=rng.randint(1, 3), rows=_log_int(rng, 64, 4096))
        c["kv"] = c["rows"] + rng.choice([0, _log_int(rng, 1, 2048)])
    else:
        n = _log_int(rng, 1, 64)
        c.update(n_seq=n, rows=1 if form == "decode" else rng.randint(2, 8))
        c["kv"] = c["rows"] + _log_int(rng, 1, min(100000, 200000 // n))
    top = work(listed()[7])["flops"], work(listed()[4])["bytes"]
    while work(c)["flops"] > top[0] or work(c)["bytes"] > top[1]:  # no dearer than the largest listed ones
        c["rows"] = max(1, c["rows"] * 3 // 4)
        c["kv"] = max(c["rows"], c["kv"] * 3 // 4)
    return c


# ---- inputs ------------------------------------------------------------------

def _spread(n, lo, hi):
    """n whole numbers from hi down, spread over lo .. hi: a ragged batch."""
    return [hi] + [lo + int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(1, n)]


def _lengths(case):
    """(new rows, cached and new tokens) of each sequence."""
    n, r = case["n_seq"], case["rows"]
    rows = _spread(n, max(1, r // 4), r) if r > 8 else [r] * n
    if case["kind"] == "append":
        return rows, [a + b for a, b in zip(rows, _spread(n, case["cached"] // 8, case["cached"]))]
    return rows, [max(a, b) for a, b in zip(rows, _spread(n, max(r, case["kv"] // 8), case["kv"]))]


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _as_cache(x, kind):
    """Values as a cache of that type holds them (8 bits: clamped to its range)."""
    return (x.clamp(-E4M3_MAX, E4M3_MAX) if kind == "e4m3" else x).to(KINDS[kind])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(rows):
    return [0] + np.cumsum(rows).tolist()


def _paged(case, g):
    """The pages of a ragged batch, and the table that says whose they are."""
    h, hkv, d = HEADS[case["heads"]]
    rows, kv = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in kv]
    pool = sum(need) + 8
    order = torch.randperm(pool, generator=g, device="cuda").cpu().numpy().astype(np.int32)
    table = np.full((len(kv), max(need)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"kind": case["kind"], "h": h, "hkv": hkv, "d": d, "n": len(rows), "rows": sum(rows), "max_q": max(rows),
         "max_kv": max(kv), "page": page, "cache": case["cache"], "q_start": _ints(_starts(rows)), "kv_len": _ints(kv),
         "table": torch.from_numpy(table).cuda()}
    for name in ("k", "v"):
        x = torch.empty(pool, hkv, page, d, dtype=KINDS[case["cache"]], device="cuda")
        for i in range(0, pool, 4096):
            x[i:i + 4096] = _as_cache(_rand(g, min(4096, pool - i), hkv, page, d) * (1.0 if name == "k" else 0.5),
                                      case["cache"])
        s[name + "_pages"] = x
    # the scales that an 8-bit cache is kept with: a power of two or not, per head
    for name in ("k", "v"):
        sc = 0.02 + 0.03 * torch.rand(hkv, generator=g, device="cuda")
        s[name + "_scale"] = sc if case["cache"] == "e4m3" else torch.ones(hkv, device="cuda")
        if case["cache"] == "e4m3":
            x = s[name + "_pages"]
            for i in range(0, pool, 4096):
                x[i:i + 4096] = _as_cache(x[i:i + 4096].float() / sc[:, None, None], "e4m3")
    return s


def _frequencies(d):
    return THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "verify":
        s = _verify_state(case, g)
    else:
        s = _paged(case, g)
        h, hkv, d, r = s["h"], s["hkv"], s["d"], s["rows"]
        s["q_out"] = torch.zeros(r, h, d, dtype=KINDS[case["q"]], device="cuda")
        if case["kind"] == "append":
            t = KINDS[case["in"]]
            # as the projections leave them: a few channels are larger than the rest
            hot = 1.0 + 4.0 * (torch.rand(d, generator=g, device="cuda") > 0.97)
            s["q"], s["k"] = (_rand(g, r, h, d) * hot).to(t), (_rand(g, r, hkv, d) * hot).to(t)
            s["v"] = (_rand(g, r, hkv, d) * 0.7).to(t)
            s["q_norm"], s["k_norm"] = 1.0 + 0.1 * _rand(g, d), 1.0 + 0.1 * _rand(g, d)
            s["freq"] = _frequencies(d)
        else:
            s["q"] = (_rand(g, r, h, d) * 1.5).to(KINDS[case["q"]])
            s["window"], s["sinks"], s["scale"] = case["window"], case["sinks"], 1.0 / math.sqrt(d)
    if own:
        s["call"] = _own_call(case, s)
    torch.cuda.synchronize()
    return s


def _verify_state(case, g):
    n, v = case["n_seq"], case["vocab"]
    drafts = [case["drafts"] - (i % 3 == 2 and case["drafts"] > 1) for i in range(n)]
    rows = sum(drafts) + n
    # a drafter that mostly agrees with its target
    both = _rand(g, rows, v) * 2.5
    logits = both + 0.5 * _rand(g, rows, v)
    probs = torch.softmax(both + 0.5 * _rand(g, rows, v), dim=-1)
    del both
    drawn = torch.multinomial(probs, 1, generator=g)[:, 0].to(torch.int32)
    tokens = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), drawn[:-1]])  # row i+1 is fed row i's draft
    temperature = torch.tensor([0.0 if i % 7 == 3 else 0.7 + 0.1 * (i % 5) for i in range(n)], device="cuda")
    return {"kind": "verify", "n": n, "rows": rows, "max_rows": max(drafts) + 1, "vocab": v, "logits": logits,
            "probs": probs, "tokens": tokens, "temperature": temperature,
            "q_start": _ints(_starts([k + 1 for k in drafts])),
            "u": torch.rand(rows, generator=g, device="cuda"), "u_next": torch.rand(n, generator=g, device="cuda"),
            "accepted": _ints([0] * n), "out": _ints([0] * rows)}


# ---- the library's calls -------------------------------------------------------

_CTX = []


class _Dev:
    """A torch tensor as the library's device buffer."""

    def __init__(self, t):
        import ctypes
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr())


def _own_call(case, s):
    """The library's objects over the state's buffers, as a program keeps them, and the call."""
    sys.path.insert(0, os.path.join(os.getcwd(), "wpc-engine_amd"))
    import wpcg
    if not _CTX:
        _CTX.append(wpcg.Context(0))
    ctx = _CTX[0]
    types = {torch.float32: wpcg.DTYPE_F32, torch.bfloat16: wpcg.DTYPE_BF16, torch.float8_e4m3fn: wpcg.DTYPE_E4M3}
    b = {k: _Dev(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
    if s["kind"] == "verify":
        op = wpcg.DraftVerify(ctx, s["n"], s["rows"], s["max_rows"], s["vocab"], q_start=b["q_start"],
                              temperature=b["temperature"])
        return lambda: op.run(b["logits"], b["tokens"], b["u"], b["u_next"], b["accepted"], b["out"],
                              draft_probs=b["probs"])
    scales = {"k_scale": b["k_scale"], "v_scale": b["v_scale"]} if s["cache"] == "e4m3" else {}
    kv = wpcg.PagedKv(ctx, s["k_pages"].shape[0], s["page"], s["hkv"], s["d"], types[s["k_pages"].dtype],
                      k=b["k_pages"], v=b["v_pages"], **scales)
    batch = wpcg.KvBatch(s["n"], s["rows"], b["kv_len"], b["table"], s["table"].shape[1], s["max_kv"],
                         max_q=s["max_q"], q_start=b["q_start"])
    if s["kind"] == "append":
        op = wpcg.KvAppend(ctx, kv, batch, s["h"], types[s["q"].dtype], types[s["q_out"].dtype], q_norm=b["q_norm"],
                           k_norm=b["k_norm"], eps=EPS, frequencies=b["freq"])
        return lambda: op.run(b["q"], b["k"], b["v"], b["q_out"])
    op = wpcg.PagedAttention(ctx, kv, batch, s["h"], types[s["q"].dtype], scale=s["scale"], window=s["window"],
                             sinks=s["sinks"])
    return lambda: op.run(b["q"], b["q_out"])


# ---- a pass --------------------------------------------------------------------

def _outputs(s):
    if s["kind"] == "append":
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["kind"] == "attend":
        return s["q_out"]
    return {"accepted": s["accepted"], "tokens": s["out"]}


def run(s):
    if own:
        s["call"]()
    elif s["kind"] == "append":
        _append(s)
    elif s["kind"] == "attend":
        _attend(s)
    else:
        _verify(s)
    return _outputs(s)


def _of_rows(s):
    """(sequence, place in the sequence's new rows, position) of every row."""
    start, kv = s["q_start"].long(), s["kv_len"].long()
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), r, right=True)
    i = r - start[seq]
    return seq, i, kv[seq] - (start[seq + 1] - start[seq]) + i


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rotated(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _append(s):
    seq, _, pos = _of_rows(s)
    angle = pos.double()[:, None, None] * s["freq"]  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    s["q_out"].copy_(_rotated(_normed(s["q"], s["q_norm"]), cos, sin))
    k = _rotated(_normed(s["k"], s["k_norm"]), cos, sin) / s["k_scale"][:, None]
    v = s["v"].float() / s["v_scale"][:, None]
    page = s["table"].long()[seq, pos // s["page"]]
    for x, pages in ((k, s["k_pages"]), (v, s["v_pages"])):
        x = _as_cache(x, s["cache"])
        if s["cache"] == "e4m3":
            x, pages = x.view(torch.uint8), pages.view(torch.uint8)
        pages[page, :, pos % s["page"]] = x


def _gathered(pages, table, scale):
    """Each sequence's keys or values in the order of positions, [sequence][head][position][size], in 32 bits."""
    n, blocks = table.shape
    x = pages[table.clamp(min=0).long()].float() * scale[:, None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(n, pages.shape[1], blocks * pages.shape[2], pages.shape[3])


def _attend(s):
    n, hkv, d, most = s["n"], s["hkv"], s["d"], s["max_q"]
    group = s["h"] // hkv
    k = _gathered(s["k_pages"], s["table"], s["k_scale"])
    v = _gathered(s["v_pages"], s["table"], s["v_scale"])
    seq, i, pos = _of_rows(s)
    q = torch.zeros(n, hkv, group, most, d, device="cuda")
    q[seq, :, :, i] = s["q"].float().view(-1, hkv, group, d)
    at = torch.full((n, most), -1, device="cuda")
    at[seq, i] = pos
    j = torch.arange(k.shape[2], device="cuda")
    seen = j <= at[:, :, None]
    if s["window"]:
        seen &= (j > at[:, :, None] - s["window"]) | (j < s["sinks"])
    seen = seen[:, None, None]
    v = torch.where(j[:, None] < s["kv_len"][:, None, None, None], v, 0.0)
    scores = torch.matmul(q.view(n, hkv, group * most, d), k.transpose(2, 3).contiguous()) * s["scale"]
    scores = scores.view(n, hkv, group, most, -1).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(seen.any(-1, keepdim=True), top, 0.0))
    del scores
    o = torch.matmul(e.view(n, hkv, group * most, -1), v).view(n, hkv, group, most, d)
    o = torch.where(seen.any(-1, keepdim=True), o / e.sum(-1, keepdim=True), 0.0)
    s["q_out"].copy_(o[seq, :, :, i].reshape(s["rows"], s["h"], d))


def _verify(s):
    n, rows = s["n"], s["rows"]
    start = s["q_start"].long()
    drafts = start[1:] - start[:-1] - 1
    seq = torch.searchsorted(start[1:].contiguous(), torch.arange(rows, device="cuda"), right=True)
    greedy = s["temperature"] == 0
    # the target's probabilities, in 64 bits: decisions fall next to borders
    p = torch.softmax(s["logits"].double() / torch.where(greedy, 1.0, s["temperature"]).double()[seq, None], dim=-1)
    best = s["logits"].argmax(-1)
    place = torch.arange(s["max_rows"] - 1, device="cuda")
    row = (start[:-1, None] + place).clamp(max=rows - 2 if rows > 1 else 0)
    draft = s["tokens"].long()[row + 1]
    ok = s["u"].double()[row] * s["probs"].double()[row, draft] < p[row, draft]
    ok = torch.where(greedy[:, None], best[row] == draft, ok) & (place < drafts[:, None])
    accepted = ok.long().cumprod(-1).sum(-1)
    at = start[:-1] + accepted
    target = p[at]
    rest = (target - torch.where((accepted < drafts)[:, None], s["probs"][at].double(), 0.0)).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, target)
    cdf = rest.cumsum(-1)
    over = cdf > (s["u_next"].double() * cdf[:, -1])[:, None]
    # where the rounding of the sums leaves none, the last token with any weight
    last = s["vocab"] - 1 - (rest > 0).int().flip(-1).argmax(-1)
    token = torch.where(over.any(-1), over.int().argmax(-1), last)
    token = torch.where(greedy, best[at], token)
    i = torch.arange(rows, device="cuda") - start[seq]
    fed = torch.cat([s["tokens"][1:], s["tokens"][:1]]).long()  # the draft that follows each row
    s["out"].copy_(torch.where(i < accepted[seq], fed, torch.where(i == accepted[seq], token[seq], -1)))
    s["accepted"].copy_(accepted)


# ---- what a pass cannot do without ---------------------------------------------

def _keys(first, last, window, sinks):
    """(keys that rows at positions first .. last see together, pairs of a row and a key)"""
    if not window:
        return last + 1, sum(p + 1 for p in range(first, last + 1))
    lo = max(0, first - window + 1)
    return last + 1 - lo + min(sinks, lo), sum(
        min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(first, last + 1))


def work(case):
    if case["kind"] == "verify":
        n, v = case["n_seq"], case["vocab"]
        rows = sum(case["drafts"] - (i % 3 == 2 and case["drafts"] > 1) + 1 for i in range(n))
        # every row's logits, and one row of the drafter's probabilities a sequence
        return {"bytes": 4 * v * (rows + n) + 20 * rows, "flops": 4 * v * rows}
    h, hkv, d = HEADS[case["heads"]]
    rows, kv = _lengths(case)
    if case["kind"] == "append":
        r = sum(rows)
        values = r * (h + 2 * hkv) * d
        return {"bytes": values * SIZE[case["in"]] + r * h * d * SIZE[case["q"]] + r * 2 * hkv * d * SIZE[case["cache"]],
                "flops": 8 * values}
    keys, pairs = (sum(x) for x in zip(*(_keys(b - a, b - 1, case["window"], case["sinks"])
                                         for a, b in zip(rows, kv))))
    return {"bytes": keys * 2 * hkv * d * SIZE[case["cache"]] + sum(rows) * 2 * h * d * SIZE[case["q"]]
            + 4 * keys // case["page"], "flops": 4 * d * h * pairs}


# ---- the same in 64 bits, sequence by sequence ----------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    start, n = s["q_start"].tolist(), s["n"]
    if case["kind"] == "verify":
        return _exact_verify(s, start)
    kv, table = s["kv_len"].tolist(), s["table"].tolist()
    page, group = s["page"], s["h"] // s["hkv"]
    ks, vs = s["k_scale"].double(), s["v_scale"].double()
    if case["kind"] == "append":
        out = {"q": torch.zeros_like(s["q_out"], dtype=torch.float64),
               "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        half = s["d"] // 2
        top = E4M3_MAX if case["cache"] == "e4m3" else math.inf
        for i in range(n):
            a, b = start[i], start[i + 1]
            pos = np.arange(kv[i] - (b - a), kv[i])
            turn = torch.polar(torch.ones(b - a, half, dtype=torch.float64, device="cuda"),
                               torch.from_numpy(pos[:, None] * s["freq"].cpu().numpy()).cuda())[:, None]

            def turned(x, w):
                x = x[a:b].double()
                x = x / (x.pow(2).sum(-1, keepdim=True) / s["d"] + EPS).sqrt() * w.double()
                z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
                return torch.cat([z.real, z.imag], -1)

            out["q"][a:b] = turned(s["q"], s["q_norm"])
            where = torch.tensor([table[i][p // page] for p in pos], device="cuda")
            slot = torch.from_numpy(pos % page).cuda()
            out["k_pages"][where, :, slot] = (turned(s["k"], s["k_norm"]) / ks[:, None]).clamp(-top, top)
            out["v_pages"][where, :, slot] = (s["v"][a:b].double() / vs[:, None]).clamp(-top, top)
        return out
    out = torch.zeros_like(s["q_out"], dtype=torch.float64)
    for i in range(n):
        a, b, m = start[i], start[i + 1], kv[i]
        ids = torch.tensor(table[i][:-(-m // page)], device="cuda", dtype=torch.long)
        p = torch.arange(m - (b - a), m, device="cuda")[:, None]
        t = torch.arange(m, device="cuda")[None]
        hidden = t > p
        if s["window"]:
            hidden = hidden | ((p - t >= s["window"]) & (t >= s["sinks"]))
        for h in range(s["hkv"]):
            k = s["k_pages"][ids, h].double().reshape(-1, s["d"])[:m] * ks[h]
            v = s["v_pages"][ids, h].double().reshape(-1, s["d"])[:m] * vs[h]
            for e in range(h * group, (h + 1) * group):
                x = s["q"][a:b, e].double() @ k.T.contiguous() * s["scale"]
                out[a:b, e] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
    return out


def _exact_verify(s, start):
    accepted, tokens = [], []
    fed, t = s["tokens"].tolist(), s["temperature"].tolist()
    u, un = s["u"].double().tolist(), s["u_next"].double().tolist()
    for i in range(s["n"]):
        a, b = start[i], start[i + 1]
        x = s["logits"][a:b].double()
        if t[i] == 0:
            p = torch.zeros_like(x)
            p[torch.arange(b - a), s["logits"][a:b].argmax(-1)] = 1.0
        else:
            x = x / float(s["temperature"][i].double())
            p = (x - torch.logsumexp(x, -1, keepdim=True)).exp()
        q = s["probs"][a:b].double()
        k = 0
        while k < b - a - 1:
            d = fed[a + k + 1]
            if not u[a + k] * float(q[k, d]) < float(p[k, d]):
                break
            k += 1
        w = p[k] if k == b - a - 1 else (p[k] - q[k]).clamp(min=0)
        w = w if float(w.sum()) > 0 else p[k]
        w = w.cpu().numpy()
        c = np.cumsum(w)
        j = int(np.searchsorted(c, un[i] * c[-1], side="right"))
        j = j if j < len(w) else int(np.flatnonzero(w > 0)[-1])
        accepted.append(k)
        tokens += fed[a + 1:a + 1 + k] + [j] + [-1] * (b - a - 1 - k)
    return {"accepted": _ints(accepted), "tokens": _ints(tokens)}
