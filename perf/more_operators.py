"""The operators behind several answers to one prompt, and what their speed is measured on.

A server that samples n answers, searches with beams or takes rejected drafts back
works on sequences that share pages of keys and values:

  fork     rows of the page table become continuations of other rows: whole pages
           shared, the page that is written next copied, dropped ones free again,
           fresh ones handed out; then the copies, in every layer
  compact  pages in use moved together after sequences have ended, in every layer
  attend   attention of a batch in groups whose sequences share a long prefix: its
           keys and values are read once for the group
  score    log probabilities of given tokens, their rank, the distribution's entropy
           and its top alternatives, from rows of logits

`own` chooses between the operators' plain form in torch and the library's kernels.
Head and layer counts are those of the Qwen2.5-0.5B (14 / 2 heads of 64, 24 layers),
Qwen3-4B (32 / 8 of 128, 36) and Qwen3-30B-A3B (32 / 4 of 128, 48) shapes that
bench.py and the tests run.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}
# (query heads, key-value heads, head size, layers)
HEADS = {"0.5b": (14, 2, 64, 24), "4b": (32, 8, 128, 36), "30b": (32, 4, 128, 48)}


def listed():
    return [
        # a step of beam search: 8 requests of 4 beams of a small model, latency
        {"name": "fork-beams-8x4", "kind": "fork", "form": "beams", "heads": "0.5b", "n_seq": 32, "width": 4,
         "len": 601, "grow": 1, "page": 16, "cache": "bf16"},
        # 64 answers begun from one prompt: 63 copies of its last page in every layer
        {"name": "fork-samples-64", "kind": "fork", "form": "samples", "heads": "30b", "n_seq": 64, "width": 64,
         "len": 2012, "grow": 1, "page": 16, "cache": "bf16"},
        # half of the sequences have ended: the others' pages move together
        {"name": "compact-pool", "kind": "compact", "heads": "4b", "n_seq": 40, "len": 800, "page": 32, "cache": "e4m3"},
        # four answers to a short prompt in full precision: latency
        {"name": "prefix-4-short", "kind": "attend", "heads": "0.5b", "groups": 1, "width": 4, "rows": 1, "prefix": 700,
         "own": 60, "window": 0, "sinks": 0, "page": 16, "q": "f32", "cache": "f32"},
        # a decode step of 64 answers to one long prompt
        {"name": "prefix-64", "kind": "attend", "heads": "30b", "groups": 1, "width": 64, "rows": 1, "prefix": 8192,
         "own": 1000, "window": 0, "sinks": 0, "page": 16, "q": "bf16", "cache": "bf16"},
        # six prompts with up to 16 answers each, 8-bit cache
        {"name": "prefix-6x16", "kind": "attend", "heads": "4b", "groups": 6, "width": 16, "rows": 1, "prefix": 4000,
         "own": 500, "window": 0, "sinks": 0, "page": 32, "q": "bf16", "cache": "e4m3"},
        # 16 answers, each with the last token and four drafts
        {"name": "prefix-drafts-16x5", "kind": "attend", "heads": "4b", "groups": 1, "width": 16, "rows": 5,
         "prefix": 6000, "own": 300, "window": 0, "sinks": 0, "page": 16, "q": "f32", "cache": "bf16"},
        # 32 questions about one document, 8-bit cache
        {"name": "prefix-65536", "kind": "attend", "heads": "4b", "groups": 1, "width": 32, "rows": 1, "prefix": 65536,
         "own": 200, "window": 0, "sinks": 0, "page": 64, "q": "f32", "cache": "e4m3"},
        # one step's token with its 20 best alternatives: latency
        {"name": "score-one", "kind": "score", "rows": 1, "vocab": 151936, "top": 20, "type": "f32", "temp": False},
        # a decode batch at the temperatures that it is sampled at
        {"name": "score-64", "kind": "score", "rows": 64, "vocab": 151936, "top": 5, "type": "f32", "temp": True},
        # answers scored by a reference model: every token's log probability and entropy
        {"name": "score-1500", "kind": "score", "rows": 1500, "vocab": 151936, "top": 0, "type": "f32", "temp": False},
        # a beam search's candidates over a smaller vocabulary, 16-bit logits
        {"name": "score-bf16", "kind": "score", "rows": 777, "vocab": 32003, "top": 50, "type": "bf16", "temp": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["fork", "compact", "attend", "attend", "attend", "score", "score"])
    if kind == "score":
        c = {"kind": kind, "rows": _log_int(rng, 1, 1500), "vocab": rng.choice([151936, _log_int(rng, 500, 151936)]),
             "top": rng.choice([0, 1, 5, 20, rng.randint(1, 64)]), "type": rng.choice(["f32", "f32", "bf16"]),
             "temp": rng.random() < 0.5}
        return c
    heads = rng.choice(sorted(HEADS))
    c = {"kind": kind, "heads": heads, "page": rng.choice([16, 32, 64])}
    if kind == "fork":
        form = rng.choice(["beams", "samples", "drafts"])
        width = rng.randint(2, 8) if form == "beams" else _log_int(rng, 2, 64)
        groups = _log_int(rng, 1, max(1, 64 // width))
        c.update(form=form, n_seq=groups * width, width=width, len=_log_int(rng, 20, 2000),
                 grow=rng.randint(2, 8) if form == "drafts" else 1, cache=rng.choice(["bf16", "e4m3", "f32"]))
        while _pool_bytes(c) > 1 << 30:
            c["len"] = max(20, c["len"] * 3 // 4)
            if c["len"] == 20:
                c["heads"] = "0.5b"
        return c
    if kind == "compact":
        c.update(n_seq=_log_int(rng, 2, 64), len=_log_int(rng, 50, 2000), cache=rng.choice(["bf16", "e4m3"]))
        while _pool_bytes(c) > 1 << 30:
            c["len"] = c["len"] * 3 // 4
        return c
    q = rng.choice(["f32", "bf16"])
    window = rng.choice([0, 0, 0, _log_int(rng, 64, 8192)])
    width = _log_int(rng, 2, 64)
    c.update(groups=_log_int(rng, 1, max(1, 96 // width)), width=width, rows=rng.choice([1, 1, 1, rng.randint(2, 5)]),
             prefix=_log_int(rng, 100, 65536), own=_log_int(rng, 10, 1500), window=window,
             sinks=rng.choice([0, 1, 4, 20]) if window else 0, q=q,
             cache=rng.choice(["bf16", "e4m3"] + (["f32"] if q == "f32" else [])))
    most = [work(x) for x in listed() if x["kind"] == "attend"]
    most = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while work(c)["flops"] > most[0] or work(c)["bytes"] > most[1]:  # no dearer than the largest listed ones
        c["prefix"], c["own"] = max(20, c["prefix"] * 3 // 4), max(10, c["own"] * 3 // 4)
        if c["prefix"] == 20:
            c["groups"] = max(1, c["groups"] - 1)
    return c


# ---- inputs ------------------------------------------------------------------

def _spread(n, lo, hi):
    """n whole numbers from hi down, spread over lo .. hi: a ragged batch."""
    return [hi] + [lo + int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(1, n)]


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _as_cache(x, kind):
    """Values as a cache of that type holds them (8 bits: clamped to its range)."""
    return (x.clamp(-E4M3_MAX, E4M3_MAX) if kind == "e4m3" else x).to(KINDS[kind])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(case, g, layers, pool):
    """[layers][2][pool][heads][page][size] of values; the keys' and values' scale per head."""
    _, hkv, d, _ = HEADS[case["heads"]]
    x = torch.empty(layers * 2 * pool, hkv, case["page"], d, dtype=KINDS[case["cache"]], device="cuda")
    step = max(1, (1 << 24) // (hkv * case["page"] * d))
    for i in range(0, len(x), step):
        x[i:i + step] = _as_cache(_rand(g, min(step, len(x) - i), hkv, case["page"], d), case["cache"])
    return x.view(layers, 2, pool, hkv, case["page"], d)


def _shares(case):
    """The sequences before a call on the pool: what each keeps and which one it goes on from; how many of its
    first pages it shares with its group's first sequence. The same for every seed, so that the work is known."""
    rng = random.Random(1000 * case["n_seq"] + case["len"])
    n, page = case["n_seq"], case["page"]
    lens, keep, parent, shared = [], [], [], []
    if case["kind"] == "compact":
        lens = _spread(n, max(1, case["len"] // 8), case["len"])
        return lens, lens, [-1 if i % 2 == 0 else i for i in range(n)], [0] * n
    of_group = _spread(n // case["width"], max(1, case["len"] // 2), case["len"])
    for i in range(n):
        group, place = divmod(i, case["width"])
        m = of_group[group]
        keep.append(m)
        if case["form"] == "beams":
            parent.append(group * case["width"] + rng.randrange(case["width"]))
            lens.append(m)
            shared.append(m * 3 // 4 // page if place else 0)
        elif case["form"] == "samples":
            parent.append(group * case["width"])
            lens.append(m if place == 0 else 0)
            shared.append(0)
        else:  # drafts: some of the tokens that the last call made room for are taken back
            parent.append(i)
            lens.append(m + case["grow"] - 1)
            keep[i] = m + rng.randrange(case["grow"])
            shared.append(m * 3 // 4 // page if place else 0)
    return lens, keep, parent, shared


def _pool_pages(case):
    lens, keep, _, shared = _shares(case)
    page = case["page"]
    need = sum(-(-m // page) - k for m, k in zip(lens, shared))
    if case["kind"] == "compact":
        return need + need // 4 + 4
    # room for the call's fresh pages while the old ones are still held
    return need + sum(-(-(k + case["grow"]) // page) - k // page for k in keep) + need // 8 + 4


def _pool_bytes(case):
    _, hkv, d, layers = HEADS[case["heads"]]
    return _pool_pages(case) * layers * 2 * hkv * case["page"] * d * SIZE[case["cache"]]


def _pool_state(case, g):
    _, _, _, layers = HEADS[case["heads"]]
    lens, keep, parent, shared = _shares(case)
    page, n, pool = case["page"], case["n_seq"], _pool_pages(case)
    grow = case.get("grow", 0)
    stride = max(-(-(max(a, b + grow)) // page) for a, b in zip(lens, keep)) + 1
    order = torch.randperm(pool, generator=g, device="cuda").cpu().numpy().astype(np.int32)
    table = np.full((n, stride), -1, np.int32)
    at = 0
    for i in range(n):
        m, k = -(-lens[i] // page), shared[i]
        if k:
            table[i, :k] = table[i - i % case["width"], :k]
        table[i, k:m] = order[at:at + m - k]
        at += m - k
    if case["kind"] == "compact":  # every second sequence has ended
        for i in range(n):
            if parent[i] < 0:
                table[i], lens[i] = -1, 0
    refs = np.bincount(table[table >= 0], minlength=pool).astype(np.int32)
    most = int((refs > 0).sum()) if case["kind"] == "compact" else n  # copies
    # counts, table and lengths lie side by side: what a repeated call starts from is one array
    book = torch.from_numpy(np.concatenate([refs, table.ravel(), np.array(lens, np.int32)])).cuda()
    s = {"kind": case["kind"], "n": n, "page": page, "pool": pool, "stride": stride, "grow": grow, "layers": layers,
         "most": most, "book": book, "first": book.clone(), "refs": book[:pool],
         "table": book[pool:pool + n * stride].view(n, stride), "kv_len": book[pool + n * stride:],
         "parent": _ints(parent), "keep": _ints(keep), "pages": _pages(case, g, layers, pool),
         "copies": _ints([0] * (3 * most)).view(most, 3), "result": _ints([0, 0])}
    return s


def _rows_of(case):
    """(sequences of each group, prefix of each group, own tokens of each sequence)"""
    width = _spread(case["groups"], max(1, case["width"] // 2), case["width"])
    prefix = _spread(case["groups"], max(1, case["prefix"] // 4), case["prefix"])
    n = sum(width)
    return width, prefix, [max(case["rows"], x) for x in _spread(n, max(1, case["own"] // 8), case["own"])]


def _attend_state(case, g):
    h, hkv, d, _ = HEADS[case["heads"]]
    page = case["page"]
    width, prefix, mine = _rows_of(case)
    n = len(mine)
    group = [i for i, w in enumerate(width) for _ in range(w)]
    kv = [prefix[group[i]] + mine[i] for i in range(n)]
    whole = [p // page for p in prefix]  # pages that a group shares
    need = sum(whole) + sum(-(-m // page) - whole[group[i]] for i, m in enumerate(kv))
    pool = need + 8
    order = torch.randperm(pool, generator=g, device="cuda").cpu().numpy().astype(np.int32)
    table = np.full((n, max(-(-m // page) for m in kv)), -1, np.int32)
    at, tails = 0, []
    for i in range(n):
        k, m = whole[group[i]], -(-kv[i] // page)
        if i == 0 or group[i] != group[i - 1]:
            lead = i
            table[i, :k] = order[at:at + k]
            at += k
        table[i, :k] = table[lead, :k]
        table[i, k:m] = order[at:at + m - k]
        at += m - k
        if i != lead and prefix[group[i]] % page:
            tails.append((int(table[lead, k]), int(table[i, k]), prefix[group[i]] % page))
    pages = _pages(case, g, 1, pool)[0]
    s = {"kind": "attend", "h": h, "hkv": hkv, "d": d, "n": n, "q_rows": case["rows"], "rows": n * case["rows"],
         "page": page, "cache": case["cache"], "groups": len(width), "max_kv": max(kv), "max_prefix": max(prefix),
         "width": max(width), "max_own": max(mine), "window": case["window"], "sinks": case["sinks"],
         "scale": 1.0 / math.sqrt(d), "k_pages": pages[0], "v_pages": pages[1], "kv_len": _ints(kv),
         "table": torch.from_numpy(table).cuda(), "q_start": _ints(list(range(0, n * case["rows"] + 1, case["rows"]))),
         "group_start": _ints([0] + np.cumsum(width).tolist()), "prefix": _ints(prefix)}
    for a, b, t in tails:  # the first tokens of a forked page are copies
        for x in (s["k_pages"], s["v_pages"]):
            x[b, :, :t] = x[a, :, :t]
    for name in ("k", "v"):
        sc = 0.5 + torch.rand(hkv, generator=g, device="cuda")
        s[name + "_scale"] = sc if case["cache"] == "e4m3" else torch.ones(hkv, device="cuda")
    s["q"] = (_rand(g, s["rows"], h, d) * 1.5).to(KINDS[case["q"]])
    s["out"] = torch.zeros(s["rows"], h, d, dtype=KINDS[case["q"]], device="cuda")
    return s


def _score_state(case, g):
    n, v = case["rows"], case["vocab"]
    x = torch.empty(n, v, dtype=KINDS[case["type"]], device="cuda")
    tokens = torch.empty(n, dtype=torch.int64, device="cuda")
    for i in range(0, n, 256):
        part = _rand(g, min(256, n - i), v) * 2.0
        # a few likely ids a row, as a model leaves them
        likely = torch.randint(0, v, (len(part), 6), generator=g, device="cuda")
        part.scatter_add_(1, likely, 4.0 + 4.0 * torch.rand(len(part), 6, generator=g, device="cuda"))
        # every eighth row is held to a grammar: most ids are masked
        bound = torch.arange(i, i + len(part), device="cuda") % 8 == 7
        part.masked_fill_(bound[:, None] & (torch.rand(part.shape, generator=g, device="cuda") < 0.7), -math.inf)
        x[i:i + len(part)] = part
        noise = -torch.log(-torch.log(torch.rand(part.shape, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
        tokens[i:i + len(part)] = (x[i:i + len(part)].float() + noise).argmax(-1)
    temp = torch.tensor([0.6 + 0.1 * (i % 7) for i in range(n)], device="cuda")
    k = case["top"]
    return {"kind": "score", "rows": n, "vocab": v, "top": k, "logits": x, "tokens": tokens.to(torch.int32),
            "temperature": temp if case["temp"] else None, "logprob": torch.zeros(n, device="cuda"),
            "entropy": torch.zeros(n, device="cuda"), "rank": _ints([0] * n),
            "top_ids": torch.zeros(n, k, dtype=torch.int32, device="cuda"), "top_logprob": torch.zeros(n, k, device="cuda")}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"score": _score_state, "attend": _attend_state}.get(case["kind"], _pool_state)(case, g)
    if own:
        s["call"] = _own_call(s)
    torch.cuda.synchronize()
    return s


# ---- the library's calls -------------------------------------------------------

_CTX = []


class _Dev:
    """A torch tensor as the library's device buffer."""

    def __init__(self, t):
        import ctypes
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr())


def _own_call(s):
    """The library's objects over the state's buffers, as a program keeps them, and the call."""
    sys.path.insert(0, os.path.join(os.getcwd(), "wpc-engine_amd"))
    import wpcg
    if not _CTX:
        _CTX.append(wpcg.Context(0))
    ctx = _CTX[0]
    types = {torch.float32: wpcg.DTYPE_F32, torch.bfloat16: wpcg.DTYPE_BF16, torch.float8_e4m3fn: wpcg.DTYPE_E4M3}
    b = {k: _Dev(t) for k, t in s.items() if isinstance(t, torch.Tensor) and t.numel()}
    if s["kind"] == "score":
        op = wpcg.LogProbs(ctx, s["rows"], s["vocab"], top=s["top"], dtype=types[s["logits"].dtype],
                           temperature=b.get("temperature"))
        return lambda: op.run(b["logits"], b["tokens"], b["logprob"], entropy=b["entropy"], rank=b["rank"],
                              top_ids=b.get("top_ids"), top_logprob=b.get("top_logprob"))
    if s["kind"] == "attend":
        scales = {"k_scale": b["k_scale"], "v_scale": b["v_scale"]} if s["cache"] == "e4m3" else {}
        kv = wpcg.PagedKv(ctx, s["k_pages"].shape[0], s["page"], s["hkv"], s["d"], types[s["k_pages"].dtype],
                          k=b["k_pages"], v=b["v_pages"], **scales)
        batch = wpcg.KvBatch(s["n"], s["rows"], b["kv_len"], b["table"], s["table"].shape[1], s["max_kv"],
                             max_q=s["q_rows"], q_start=b["q_start"])
        prefix = wpcg.KvPrefix(s["groups"], b["group_start"], b["prefix"], s["max_prefix"])
        op = wpcg.PrefixAttention(ctx, kv, batch, prefix, s["h"], types[s["q"].dtype], scale=s["scale"],
                                  window=s["window"], sinks=s["sinks"])
        return lambda: op.run(b["q"], b["out"])
    pages = s["pages"]
    layers = [wpcg.PagedKv(ctx, s["pool"], s["page"], pages.shape[3], pages.shape[5], types[pages.dtype],
                           k=_Dev(pages[i, 0]), v=_Dev(pages[i, 1])) for i in range(s["layers"])]
    pool = wpcg.KvPool(ctx, s["pool"], s["page"], s["n"], s["stride"], b["refs"], b["table"], b["kv_len"])
    copy = wpcg.KvCopy(ctx, layers, b["copies"], b["result"], s["most"])
    if s["kind"] == "fork":
        fork = wpcg.KvFork(ctx, pool, b["copies"], b["result"], parent=b["parent"], keep=b["keep"], grow=s["grow"])

        def call():
            fork.run()
            copy.run()
        return call
    compact = wpcg.KvCompact(ctx, pool, b["copies"], b["result"], s["most"])
    stream = torch.cuda.ExternalStream(ctx.stream.value)

    def call():
        with torch.cuda.stream(stream):
            s["book"].copy_(s["first"])
        compact.run()
        copy.run()
    return call


# ---- a pass --------------------------------------------------------------------

def _outputs(s):
    names = {"score": ["logprob", "entropy", "rank", "top_ids", "top_logprob"], "attend": ["out"]}
    return {k: s[k] for k in names.get(s["kind"], ["refs", "table", "kv_len", "copies", "result", "pages"])}


def run(s):
    if own:
        s["call"]()
    elif s["kind"] == "score":
        _score(s)
    elif s["kind"] == "attend":
        _attend(s)
    elif s["kind"] == "fork":
        _fork(s)
    else:
        s["book"].copy_(s["first"])  # a pool once compacted leaves nothing to do
        _compact(s)
    return _outputs(s)


def _bump(counts, ids, by, where):
    """counts[ids] += by where it holds; the others count nowhere."""
    more = torch.zeros(len(counts) + 1, dtype=counts.dtype, device="cuda")
    more.index_add_(0, torch.where(where, ids, len(counts)).reshape(-1).long(),
                    torch.full((ids.numel(),), by, dtype=counts.dtype, device="cuda"))
    counts += more[:-1]


def _listed_ids(mask):
    """Ids where mask holds, in rising order, then ids behind the end."""
    n = len(mask)
    rank = mask.long().cumsum(0) - 1
    ids = torch.full((n + 1,), n, dtype=torch.long, device="cuda")
    ids.scatter_(0, torch.where(mask, rank, n), torch.arange(n, device="cuda"))
    return ids[:n], mask.long().sum()


def _fork(s):
    """A call that runs out of pages changes nothing, but the states here have enough."""
    n, page, pool, stride = s["n"], s["page"], s["pool"], s["stride"]
    refs, table, kv_len = s["refs"], s["table"], s["kv_len"]
    seq, j = torch.arange(n, device="cuda"), torch.arange(stride, device="cuda")
    parent = s["parent"].long()
    keep = torch.where(parent >= 0, torch.minimum(s["keep"], kv_len[parent.clamp(min=0)]), 0).long()
    size = torch.minimum(keep + s["grow"], torch.tensor(stride * page, device="cuda"))
    held = (j < ((kv_len + page - 1) // page)[:, None]) & (table >= 0)
    kept = torch.where(j < ((keep + page - 1) // page)[:, None], table[parent.clamp(min=0)], -1)
    _bump(refs, table, -1, held)
    _bump(refs, kept, 1, kept >= 0)
    # who writes into a page that is begun: the first of them keeps it if no one else has it
    tail = kept.gather(1, (keep // page).clamp(max=stride - 1)[:, None])[:, 0].long()
    writes = (keep % page > 0) & (size > keep) & (tail >= 0)
    at = torch.where(writes, tail, pool)
    writers = torch.zeros(pool + 1, dtype=torch.long, device="cuda").index_add_(0, at, torch.ones_like(at))
    first = torch.full((pool + 1,), n, dtype=torch.long, device="cuda").scatter_reduce_(0, at, seq, "amin")
    copy = writes & ((refs[tail.clamp(min=0)] > writers[at]) | (first[at] != seq))
    _bump(refs, tail, -1, copy)
    # fresh pages: the lowest free ones, sequence by sequence
    from_page = torch.where(copy, keep // page, (keep + page - 1) // page)
    fresh = (size + page - 1) // page - from_page
    end = fresh.cumsum(0)
    free, n_free = _listed_ids(refs == 0)
    wants = (j >= from_page[:, None]) & (j < ((size + page - 1) // page)[:, None])
    rank = (end - fresh)[:, None] + j - from_page[:, None]
    new = free[torch.where(wants, rank, 0)].int()
    table.copy_(torch.where(wants, new, kept))
    _bump(refs, table, 1, wants)
    kv_len.copy_(size)
    place = torch.where(copy, copy.long().cumsum(0) - 1, n)
    rows = torch.cat([s["copies"], s["copies"][:1]])
    dst = table.gather(1, (keep // page).clamp(max=stride - 1)[:, None])[:, 0]
    rows[place] = torch.where(copy[:, None], torch.stack([tail.int(), dst, (keep % page).int()], 1), 0)
    s["copies"].copy_(rows[:n])
    s["result"].copy_(torch.stack([n_free - end[-1], copy.long().sum()]))
    _copy_pages(s)


def _compact(s):
    pool, most = s["pool"], s["most"]
    refs, table = s["refs"], s["table"]
    free, n_free = _listed_ids(refs == 0)
    down, n_used = _listed_ids(refs.flip(0) != 0)
    used = pool - 1 - down  # the highest first; -1 where there are no more
    moves = ((free < used) & (torch.arange(pool, device="cuda") < most)).cumprod(0).bool()
    to = torch.arange(pool + 1, device="cuda")
    to.scatter_(0, torch.where(moves, used, pool), free)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), -1))
    counts = torch.zeros(pool + 1, dtype=refs.dtype, device="cuda")
    counts.scatter_(0, torch.where(refs != 0, to[:pool], pool), refs)
    refs.copy_(counts[:pool])
    n = moves.long().sum()
    whole = torch.full((pool,), s["page"], dtype=torch.long, device="cuda")
    s["copies"].copy_(torch.where(moves[:most, None], torch.stack([used, free, whole], 1)[:most], s["copies"]))
    s["result"].copy_(torch.stack([torch.where(refs != 0, torch.arange(1, pool + 1, device="cuda"), 0).max(), n]))
    _copy_pages(s)


def _copy_pages(s):
    k = torch.arange(s["most"], device="cuda")
    some = s["result"][1] > 0
    rows = s["copies"][torch.where(k < s["result"][1], k, 0)].long()  # behind the last one the first again
    src = torch.where(some, rows[:, 0], 0)
    dst, t = torch.where(some, rows[:, 1], src), torch.where(some, rows[:, 2], 0)
    pages = s["pages"].view(torch.uint8) if s["pages"].element_size() == 1 else s["pages"]
    old = pages[:, :, dst]
    taken = torch.arange(s["page"], device="cuda") < t[:, None]
    pages[:, :, dst] = torch.where(taken[:, None, :, None], pages[:, :, src], old)


def _gathered(pages, table, scale):
    """Keys or values in the order of positions, [row of table][head][position][size], in 32 bits."""
    n, blocks = table.shape
    x = pages[table.clamp(min=0).long()].float() * scale[:, None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(n, pages.shape[1], blocks * pages.shape[2], pages.shape[3])


def _part(q, k, v, seen, scale):
    """Maximum, sum and unnormalised output of softmax(scale q K^T) V over the seen keys; q [n][kv head][row][size]."""
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    x = x.masked_fill(~seen[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    return m, e.sum(-1, keepdim=True), torch.matmul(e, v)


def _attend(s):
    n, h, hkv, d, r = s["n"], s["h"], s["hkv"], s["d"], s["q_rows"]
    group, page, width = h // hkv, s["page"], s["width"]
    start, prefix, kv = s["group_start"].long(), s["prefix"].long(), s["kv_len"].long()
    seq = torch.arange(n, device="cuda")
    of = torch.searchsorted(start[1:].contiguous(), seq, right=True)
    place = seq - start[of]
    pos = (kv[:, None] - r + torch.arange(r, device="cuda"))  # [sequence][row]
    q = s["q"].float().view(n, r, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * r, d)

    def seen(at, token, lo, hi):
        ok = (token <= at) & (token >= lo) & (token < hi)
        if s["window"]:
            ok = ok & ((token > at - s["window"]) | (token < s["sinks"]))
        return ok

    # the prefix, once for all of a group's sequences
    blocks = -(-s["max_prefix"] // page)
    lead = s["table"][start[:-1], :blocks]
    token = torch.arange(blocks * page, device="cuda")
    qg = torch.zeros(s["groups"], hkv, width, group * r, d, device="cuda")
    qg[of, :, place] = q
    at = torch.full((s["groups"], width, r), -1, device="cuda")
    at[of, place] = pos
    at = at[:, :, None].expand(-1, -1, group, -1).reshape(s["groups"], -1, 1)
    m, l, o = _part(qg.view(s["groups"], hkv, -1, d), _gathered(s["k_pages"], lead, s["k_scale"]),
                    _gathered(s["v_pages"], lead, s["v_scale"]),
                    seen(at, token, 0, prefix[:, None, None]), s["scale"])
    m, l, o = (x.view(s["groups"], hkv, width, group * r, -1)[of, :, place] for x in (m, l, o))
    # their own tokens
    first = (prefix // page)[of]
    j = first[:, None] + torch.arange(-(-(s["max_own"] + page) // page), device="cuda")
    mine = s["table"].gather(1, j.clamp(max=s["table"].shape[1] - 1))
    token = (j[:, :, None] * page + torch.arange(page, device="cuda")).view(n, 1, -1)
    at = pos[:, None].expand(-1, group, -1).reshape(n, -1, 1)
    v = _gathered(s["v_pages"], mine, s["v_scale"])
    v = torch.where((token < kv[:, None, None]).view(n, 1, -1, 1), v, 0.0)
    m2, l2, o2 = _part(q, _gathered(s["k_pages"], mine, s["k_scale"]), v,
                       seen(at, token, prefix[of][:, None, None], kv[:, None, None]), s["scale"])
    top = torch.maximum(m, m2)
    a, b = torch.exp(m - top), torch.exp(m2 - top)
    out = (o * a + o2 * b) / (l * a + l2 * b)
    s["out"].copy_(out.view(n, hkv, group, r, d).permute(0, 3, 1, 2, 4).reshape(s["rows"], h, d))


def _score(s):
    n, v, k = s["rows"], s["vocab"], s["top"]
    x = s["logits"].float()
    tokens = s["tokens"].long()[:, None]
    rate = 1.0 if s["temperature"] is None else (1.0 / s["temperature"])[:, None]
    x_t = x.gather(1, tokens)
    ids = torch.arange(v, device="cuda")
    s["rank"].copy_(1 + ((x > x_t) | ((x == x_t) & (ids < tokens))).sum(-1))
    top = x.amax(-1, keepdim=True)
    t = (x - top) * rate
    e = torch.exp(t)
    z = e.sum(-1, keepdim=True)
    log_z = torch.log(z)
    s["logprob"].copy_(((x_t - top) * rate - log_z)[:, 0])
    s["entropy"].copy_((log_z - (e * torch.where(e > 0, t, 0.0)).sum(-1, keepdim=True) / z)[:, 0])
    if k:
        # unique keys: the value's order, then the lower id
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 31) + (v - 1 - ids)
        best = v - 1 - (key.topk(k, dim=-1, sorted=True).values & ((1 << 31) - 1))
        s["top_ids"].copy_(best)
        s["top_logprob"].copy_((x.gather(1, best) - top) * rate - log_z)


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    if case["kind"] == "score":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * SIZE[case["type"]] + n * (16 + 8 * case["top"]), "flops": 4 * n * v}
    h, hkv, d, layers = HEADS[case["heads"]]
    if case["kind"] == "attend":
        width, prefix, mine = _rows_of(case)
        r, window, sinks = case["rows"], case["window"], case["sinks"]
        keys = pairs = at = 0
        for w, p in zip(width, prefix):
            lo = p  # the group's first prefix token that some row's window reaches
            for m in mine[at:at + w]:
                first = p + m - r
                for i in range(r):
                    pairs += min(first + i + 1, window + sinks) if window else first + i + 1
                lo = min(lo, max(0, first - window + 1) if window else 0)
                keys += min(m, window + r) if window else m
            keys += p - lo + min(sinks, lo)
            at += w
        return {"bytes": keys * 2 * hkv * d * SIZE[case["cache"]] + len(mine) * r * 2 * h * d * SIZE[case["q"]]
                + 4 * keys // case["page"], "flops": 4 * d * h * pairs}
    lens, keep, parent, _ = _shares(case)
    page, unit = case["page"], 2 * hkv * d * SIZE[case["cache"]] * layers  # bytes of a token
    if case["kind"] == "compact":
        used = sum(-(-m // page) for m, p in zip(lens, parent) if p >= 0)
        pool = _pool_pages(case)
        moved = used * (pool - used) // pool  # the used pages lie anywhere in the pool
        return {"bytes": 2 * moved * page * unit + 4 * pool + 8 * used, "flops": used}
    seen, tokens = set(), 0
    for m, p in zip(keep, parent):  # of the rows that go on from one, all but one copy its last tokens
        if p in seen:
            tokens += m % page
        seen.add(p)
    entries = sum(-(-(m + case["grow"]) // page) for m in keep)
    return {"bytes": 2 * tokens * unit + 12 * entries, "flops": entries}


# ---- the same apart from that, in 64 bits and row by row -------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "score":
        return _exact_score(s)
    if case["kind"] == "attend":
        return _exact_attend(s)
    book = {k: s[k].cpu().numpy().copy() for k in ("refs", "table", "kv_len", "copies", "result")}
    moves = (_exact_fork if case["kind"] == "fork" else _exact_compact)(case, s, book)
    pages = s["pages"].clone()
    raw = pages.view(torch.uint8) if pages.element_size() == 1 else pages
    for a, b, t in moves:
        raw[:, :, b, :, :t] = raw[:, :, a, :, :t]
    book["pages"] = pages.double()
    return book


def _exact_fork(case, s, book):
    """The rows one by one, on the host."""
    page, refs, table, kv_len = s["page"], book["refs"], book["table"], book["kv_len"]
    old = [[int(p) for p in row[:-(-int(m) // page)]] for row, m in zip(table, kv_len)]
    keep, parent = s["keep"].tolist(), s["parent"].tolist()
    rows = [old[p][:-(-k // page)] for p, k in zip(parent, keep)]
    for row, by in [(r, -1) for r in old] + [(r, 1) for r in rows]:
        for p in row:
            refs[p] += by
    writers = {}
    for i, k in enumerate(keep):
        if k % page:
            writers.setdefault(rows[i][-1], []).append(i)
    copied = [i for p, w in writers.items() for x, i in enumerate(w) if x > 0 or refs[p] > len(w)]
    lost = {i: rows[i].pop() for i in sorted(copied)}
    free = []
    for p in lost.values():
        refs[p] -= 1
    free = iter([p for p in range(len(refs)) if refs[p] == 0])
    moves = []
    for i, k in enumerate(keep):
        while len(rows[i]) * page < k + s["grow"]:
            p = next(free)
            refs[p] += 1
            rows[i].append(p)
        if i in lost:
            moves.append((lost[i], rows[i][k // page], k % page))
        table[i] = -1
        table[i, :len(rows[i])] = rows[i]
        kv_len[i] = k + s["grow"]
    book["copies"][:len(moves)] = np.array(moves, np.int32).reshape(-1, 3)
    book["result"][:] = (refs == 0).sum(), len(moves)
    return moves


def _exact_compact(case, s, book):
    refs, table = book["refs"], book["table"]
    lo, hi, moves = 0, len(refs) - 1, []
    while True:
        while lo < len(refs) and refs[lo]:
            lo += 1
        while hi >= 0 and not refs[hi]:
            hi -= 1
        if lo >= hi or len(moves) == s["most"]:
            break
        refs[lo], refs[hi] = refs[hi], 0
        table[table == hi] = lo
        moves.append((hi, lo, s["page"]))
    book["copies"][:len(moves)] = np.array(moves, np.int32).reshape(-1, 3)
    book["result"][:] = hi + 1, len(moves)
    return moves


def _exact_attend(s):
    out = torch.zeros_like(s["out"], dtype=torch.float64)
    kv, table, r, page = s["kv_len"].tolist(), s["table"].tolist(), s["q_rows"], s["page"]
    group = s["h"] // s["hkv"]
    for i in range(s["n"]):
        m = kv[i]
        ids = torch.tensor(table[i][:-(-m // page)], device="cuda", dtype=torch.long)
        p = torch.arange(m - r, m, device="cuda")[:, None]
        t = torch.arange(m, device="cuda")[None]
        hidden = t > p
        if s["window"]:
            hidden = hidden | ((p - t >= s["window"]) & (t >= s["sinks"]))
        for h in range(s["hkv"]):
            k = s["k_pages"][ids, h].double().reshape(-1, s["d"])[:m] * s["k_scale"][h].double()
            v = s["v_pages"][ids, h].double().reshape(-1, s["d"])[:m] * s["v_scale"][h].double()
            for e in range(h * group, (h + 1) * group):
                x = s["q"][i * r:(i + 1) * r, e].double() @ k.T.contiguous() * s["scale"]
                out[i * r:(i + 1) * r, e] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
    return {"out": out}


def _exact_score(s):
    n, k = s["rows"], s["top"]
    lp, ent = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    rank, ids, best = np.zeros(n, np.int32), np.zeros((n, k), np.int32), np.zeros((n, k))
    tokens = s["tokens"].tolist()
    for i in range(n):
        row = s["logits"][i].double()
        t = 1.0 if s["temperature"] is None else float(s["temperature"][i].double())
        p = row / t - torch.logsumexp(row / t, -1)
        lp[i] = p[tokens[i]]
        ent[i] = torch.special.entr(torch.exp(p)).sum()
        order = torch.argsort(row, descending=True, stable=True)
        rank[i] = int((order == tokens[i]).nonzero()) + 1
        ids[i], best[i] = order[:k].cpu().numpy(), p[order[:k]].cpu().numpy()
    return {"logprob": lp, "entropy": ent, "rank": rank, "top_ids": ids, "top_logprob": best}
