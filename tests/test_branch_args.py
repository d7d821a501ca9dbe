"""CPU tests of what the operators behind several answers to one prompt refuse:
every argument check comes back as a status code before anything reaches a GPU,
and a call whose arguments are right ends at the missing context. Workspace
queries need no GPU."""
import ctypes as C

import pytest

import wpcg
from wpcg import E_ARG, E_SHAPE, E_UNSUPPORTED, OK

F32, BF16, SPLIT, E4M3 = 0, 1, 2, 3
AT = 1 << 20  # an aligned address that nothing here follows
SCORE, SCORE_WS = (getattr(wpcg.lib, n) for n in ("wpcg_logprobs", "wpcg_logprobs_workspace"))


def ref(x):
    return None if x is None else C.byref(x)


def refused(rc, code, text):
    assert rc == code and text in wpcg.last_error(), (rc, wpcg.last_error())


# ---- log probabilities ---------------------------------------------------------
def scores(**kw):
    a = dict(n_rows=5, vocab=1000, top=4, dtype=F32, logits=AT, logits_stride=0, temperature=AT, tokens=AT, logprob=AT,
             entropy=AT, rank=AT, top_ids=AT, top_logprob=AT)
    a.update(kw)
    return wpcg._Logprob(**a)


def score(d, ws=AT, n=1 << 40):
    return SCORE(None, ref(d), ws, n, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=E4M3), E_ARG, "F32 or BF16"), (dict(dtype=SPLIT), E_ARG, "F32 or BF16"), (dict(vocab=0), E_ARG, "vocab"),
    (dict(vocab=(1 << 30) + 1), E_ARG, "vocab"), (dict(top=65), E_ARG, "top"), (dict(n_rows=1 << 31), E_ARG, "bounds"),
    (dict(logits_stride=999), E_SHAPE, "shorter"), (dict(logits_stride=1 << 41), E_ARG, "too large"),
    (dict(logits=None), E_ARG, "null"), (dict(tokens=None), E_ARG, "null"),
    (dict(tokens=None, logprob=None), E_ARG, "null"), (dict(tokens=None, rank=None), E_ARG, "null"),
    (dict(logits=AT + 2), E_ARG, "aligned"), (dict(dtype=BF16, logits=AT + 1), E_ARG, "aligned"),
    (dict(n_rows=1 << 24), E_UNSUPPORTED, "workgroups"), (dict(n_rows=1 << 15, vocab=1 << 25), E_UNSUPPORTED, "workgroups"),
])
def test_scores(kw, code, text):
    refused(score(scores(**kw)), code, text)


def test_right_scores_end_at_the_context():
    for d in (scores(), scores(tokens=None, logprob=None, rank=None), scores(top=64), scores(top=0, top_ids=None),
              scores(dtype=BF16, logits=AT + 2, logits_stride=1001), scores(n_rows=0, logits=None), scores(vocab=1 << 30)):
        refused(score(d), E_ARG, "null context")
    refused(score(None), E_ARG, "null")


def test_model_scores():
    call = wpcg.lib.wpcg_model_score
    refused(call(None, AT, 4, AT, 1.0, 0, AT, None, None, None, None), E_ARG, "null")


def test_score_workspace():
    n = C.c_uint64(7)
    assert SCORE_WS(ref(scores()), C.byref(n)) == OK and n.value == 5 * 20 + 12 + 5 * 32 * 4
    refused(score(scores(), n=n.value - 1), E_ARG, "bytes of workspace")
    refused(score(scores(), ws=None, n=0), E_ARG, "bytes of workspace")
    refused(score(scores(), ws=AT + 4), E_ARG, "aligned")
    assert SCORE_WS(ref(scores(top=0)), C.byref(n)) == OK and n.value == 112
    assert SCORE_WS(ref(scores(top=65)), C.byref(n)) == E_ARG and n.value == 0
    assert SCORE_WS(ref(scores()), None) == E_ARG and SCORE_WS(None, C.byref(n)) == E_ARG


# ---- pages ---------------------------------------------------------------------
FORK, FORK_WS, COMPACT, COMPACT_WS, COPY = (getattr(wpcg.lib, "wpcg_kv_" + n) for n in (
    "fork", "fork_workspace", "compact", "compact_workspace", "copy"))


def pool(**kw):
    a = dict(n_pages=100, page_size=16, n_seq=4, table_stride=20, refs=AT, table=AT, kv_len=AT)
    a.update(kw)
    return wpcg._KvPool(**a)


def change(**kw):
    a = dict(parent=AT, keep=AT, grow_each=AT, copies=AT, result=AT)
    a.update(kw)
    return wpcg._KvChange(**a)


def pages(**kw):
    a = dict(k=AT, v=AT, dtype=BF16, n_pages=10, page_size=16, n_kv_heads=2, head_dim=128)
    a.update(kw)
    return wpcg._KvPages(**a)


def fork(p, c, ws=AT, n=1 << 40):
    return FORK(None, ref(p), ref(c), ws, n, None)


def compact(p, most=5, copies=AT, result=AT, ws=AT, n=1 << 40):
    return COMPACT(None, ref(p), most, copies, result, ws, n, None)


def copy(layers, copies=AT, n=AT, most=5):
    return COPY(None, (wpcg._KvPages * len(layers))(*layers), len(layers), copies, n, most, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(page_size=8), E_SHAPE, "page_size"), (dict(page_size=48), E_SHAPE, "page_size"), (dict(n_pages=0), E_ARG, "n_pages"),
    (dict(n_pages=(1 << 26) + 1), E_ARG, "n_pages"), (dict(table_stride=0), E_ARG, "table"),
    (dict(n_seq=1 << 16, table_stride=1 << 15), E_ARG, "table"), (dict(table_stride=1 << 27), E_ARG, "table"),
    (dict(n_seq=(1 << 30) + 1), E_ARG, "table"), (dict(n_seq=1 << 22, table_stride=1), E_UNSUPPORTED, "workgroups"),
    (dict(refs=None), E_ARG, "null"), (dict(table=None), E_ARG, "null"), (dict(kv_len=None), E_ARG, "null"),
])
def test_pools(kw, code, text):
    refused(fork(pool(**kw), change()), code, text)
    refused(compact(pool(**kw)), code, text)


def test_changes():
    refused(fork(None, change()), E_ARG, "null")
    refused(fork(pool(), None), E_ARG, "null")
    for kw in (dict(copies=None), dict(result=None)):
        refused(fork(pool(), change(**kw)), E_ARG, "null")
        refused(compact(pool(), **kw), E_ARG, "null")
    for p, c in ((pool(), change()), (pool(), change(parent=None, keep=None, grow_each=None, grow=1 << 31, window=1 << 31)),
                 (pool(n_seq=0, table=None, kv_len=None), change(copies=None)), (pool(n_pages=1 << 26), change())):
        refused(fork(p, c), E_ARG, "null context")
    refused(compact(pool(), most=0, copies=None), E_ARG, "null context")
    refused(compact(pool(n_seq=0, table=None, kv_len=None)), E_ARG, "null context")


@pytest.mark.parametrize("query,call,words", [(FORK_WS, lambda *a: fork(pool(), change(), *a), 2 * 100 + 4 * 12 + 4 + 4 * 20 + 4 + 4),
                                              (COMPACT_WS, lambda *a: compact(pool(), 5, AT, AT, *a), 3 * 100 + 4 + 4)])
def test_pool_workspaces(query, call, words):
    n = C.c_uint64()
    assert query(ref(pool()), C.byref(n)) == OK and n.value == 4 * words
    refused(call(AT, n.value - 1), E_ARG, "bytes of workspace")
    refused(call(None, 0), E_ARG, "bytes of workspace")
    refused(call(AT + 8, n.value), E_ARG, "aligned")
    refused(call(AT, n.value), E_ARG, "null context")
    assert query(ref(pool(n_pages=0)), C.byref(n)) == E_ARG and n.value == 0
    assert query(ref(pool()), None) == E_ARG and query(None, C.byref(n)) == E_ARG


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=SPLIT), E_ARG, "F32, BF16 or E4M3"), (dict(head_dim=96), E_UNSUPPORTED, "head_dim"),
    (dict(page_size=8), E_SHAPE, "page_size"), (dict(k=None), E_ARG, "null"), (dict(v=AT + 8), E_ARG, "aligned"),
    (dict(n_pages=11), E_SHAPE, "different"), (dict(dtype=F32), E_SHAPE, "different"), (dict(n_kv_heads=4), E_SHAPE, "different"),
    (dict(head_dim=64), E_SHAPE, "different"), (dict(page_size=32), E_SHAPE, "different"),
    (dict(page_stride=4096, head_stride=128, token_stride=256), E_SHAPE, "different"),
])
def test_layers(kw, code, text):
    refused(copy([pages(), pages(**kw)]), code, text)


def test_copies():
    # the packed order in other words is the same geometry
    refused(copy([pages(), pages(page_stride=4096, head_stride=2048, token_stride=128)]), E_ARG, "null context")
    refused(copy([pages()] * 200), E_ARG, "null context")
    refused(copy([]), E_ARG, "null context")
    refused(copy([pages()], most=0, copies=None, n=None), E_ARG, "null context")
    refused(copy([pages()], copies=None), E_ARG, "null")
    refused(copy([pages()], n=None), E_ARG, "null")
    refused(copy([pages()], most=(1 << 26) + 1), E_ARG, "max_copies")
    refused(COPY(None, None, 1, AT, AT, 1, None), E_ARG, "null")
    refused(COPY(None, None, 65537, AT, AT, 1, None), E_ARG, "null")


# ---- attention over shared prefixes ----------------------------------------------
ATTEND, ATTEND_WS = wpcg.lib.wpcg_prefix_attention, wpcg.lib.wpcg_prefix_attention_workspace


def batch(**kw):
    a = dict(n_seq=3, n_rows=5, max_q=3, max_kv=60, table_stride=4, q_start=AT, kv_len=AT, table=AT)
    a.update(kw)
    return wpcg._KvBatch(**a)


def prefix(**kw):
    a = dict(n_groups=2, max_prefix=50, group_start=AT, prefix_len=AT)
    a.update(kw)
    return wpcg._KvPrefix(**a)


def attention(**kw):
    a = dict(q=AT, out=AT, dtype=BF16, n_heads=8, scale=0.1)
    a.update(kw)
    return wpcg._Attention(**a)


def attend(kv, b, x, a, ws=AT, n=1 << 40):
    return ATTEND(None, ref(kv), ref(b), ref(x), ref(a), ws, n, None)


def attend_ws(kv, b, x, a):
    n = C.c_uint64(7)
    rc = ATTEND_WS(ref(kv), ref(b), ref(x), ref(a), C.byref(n))
    return n.value if rc == OK else rc


def test_right_prefixes_end_at_the_context():
    for x in (prefix(), prefix(n_groups=0, group_start=None, prefix_len=None), prefix(n_groups=3), prefix(n_groups=50),
              prefix(max_prefix=0), prefix(max_prefix=1 << 30)):
        for b in (batch(), batch(q_start=None, max_q=1), batch(n_seq=0), batch(n_rows=0), batch(max_q=5, n_rows=9)):
            refused(attend(pages(), b, x, attention()), E_ARG, "null context")


@pytest.mark.parametrize("kv,b,x,a,code,text", [
    (None, {}, {}, {}, E_ARG, "null"), ({}, None, {}, {}, E_ARG, "null"), ({}, {}, None, {}, E_ARG, "null"),
    ({}, {}, {}, None, E_ARG, "null"), ({}, {}, dict(group_start=None), {}, E_ARG, "null"),
    ({}, {}, dict(prefix_len=None), {}, E_ARG, "null"), ({}, {}, dict(n_groups=(1 << 30) + 1), {}, E_ARG, "prefix bounds"),
    ({}, {}, dict(max_prefix=(1 << 30) + 1), {}, E_ARG, "prefix bounds"), (dict(head_dim=96), {}, {}, {}, E_UNSUPPORTED, "head_dim"),
    (dict(k=None), {}, {}, {}, E_ARG, "null"), ({}, dict(table_stride=3), {}, {}, E_SHAPE, "table"),
    ({}, dict(q_start=None), {}, {}, E_ARG, "q_start"), ({}, {}, {}, dict(scale=0.0), E_ARG, "scale"),
    ({}, {}, {}, dict(n_heads=9), E_SHAPE, "n_heads"), ({}, {}, {}, dict(out=AT + 2), E_ARG, "aligned"),
    ({}, {}, {}, dict(q=None), E_ARG, "null"), ({}, {}, {}, dict(q_stride=8), E_SHAPE, "shorter"),
    (dict(dtype=F32), {}, {}, {}, E_UNSUPPORTED, "BF16 queries"), ({}, dict(kv_len=None), {}, {}, E_ARG, "null"),
])
def test_prefix_refusals(kv, b, x, a, code, text):
    made = [None if kw is None else f(**kw) for f, kw in ((pages, kv), (batch, b), (prefix, x), (attention, a))]
    refused(attend(*made), code, text)


def test_prefix_workspace():
    # sharing pays where many bytes would be read again
    b, x = batch(n_seq=64, n_rows=64, max_q=1, max_kv=10000, table_stride=1000), prefix(n_groups=1, max_prefix=9000)
    n = attend_ws(pages(), b, x, attention())
    assert n > 0 and n % 4 == 0
    refused(attend(pages(), b, x, attention(), n=n - 1), E_ARG, "bytes of workspace")
    refused(attend(pages(), b, x, attention(), ws=None, n=0), E_ARG, "bytes of workspace")
    refused(attend(pages(), b, x, attention(), ws=AT + 4), E_ARG, "aligned")
    refused(attend(pages(), b, x, attention(), n=n), E_ARG, "null context")
    # without sharing that of the plain call
    plain = C.c_uint64()
    assert wpcg.lib.wpcg_paged_attention_workspace(ref(pages()), ref(b), ref(attention()), C.byref(plain)) == OK
    for y in (prefix(n_groups=0), prefix(max_prefix=0), prefix(n_groups=64, max_prefix=9000), prefix(n_groups=1, max_prefix=500)):
        assert attend_ws(pages(), b, y, attention()) == plain.value
    # a window reads no more again than it sees
    assert attend_ws(pages(), b, x, attention(window=8000, sinks=10)) == n
    narrow = attention(window=700, sinks=10)
    assert wpcg.lib.wpcg_paged_attention_workspace(ref(pages()), ref(b), ref(narrow), C.byref(plain)) == OK
    assert attend_ws(pages(), b, x, narrow) == plain.value
    assert ATTEND_WS(ref(pages()), ref(batch()), ref(prefix()), ref(attention()), None) == E_ARG
    # the parts' places hold whatever the bounds allow, loose rows too
    assert attend_ws(pages(), batch(n_seq=64, n_rows=1 << 20, max_q=1, max_kv=10000, table_stride=1000), x, attention()) == n


def test_prefixes_of_too_many_rows_and_heads_are_plain():
    """Outputs for 2^32 threads of one launch: the plain call, which takes them."""
    plain = C.c_uint64()
    for n_kv, heads, rows in ((2048, 65536, 512), (65536, 65536, 512 * 32)):
        kv = pages(n_kv_heads=n_kv)
        b = batch(n_seq=512, n_rows=rows, max_q=rows // 512, max_kv=64, table_stride=4)
        rc = wpcg.lib.wpcg_paged_attention_workspace(ref(kv), ref(b), ref(attention(n_heads=heads)), C.byref(plain))
        n = attend_ws(kv, b, prefix(n_groups=1, max_prefix=64), attention(n_heads=heads))
        if rc != OK:
            assert n == rc == E_UNSUPPORTED
            continue
        assert n == plain.value
    # a row less of each is shared
    kv, b = pages(n_kv_heads=2048), batch(n_seq=511, n_rows=511, max_q=1, max_kv=64, table_stride=4)
    assert wpcg.lib.wpcg_paged_attention_workspace(ref(kv), ref(b), ref(attention(n_heads=65536)), C.byref(plain)) == OK
    assert attend_ws(kv, b, prefix(n_groups=1, max_prefix=64), attention(n_heads=65536)) != plain.value
