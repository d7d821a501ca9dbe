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


def test_score_workspace():
    n = C.c_uint64(7)
    assert SCORE_WS(ref(scores()), C.byref(n)) == OK and n.value == 5 * 20 + 12 + 5 * 32 * 4
    refused(score(scores(), n=n.value - 1), E_ARG, "bytes of workspace")
    refused(score(scores(), ws=None, n=0), E_ARG, "bytes of workspace")
    refused(score(scores(), ws=AT + 4), E_ARG, "aligned")
    assert SCORE_WS(ref(scores(top=0)), C.byref(n)) == OK and n.value == 112
    assert SCORE_WS(ref(scores(top=65)), C.byref(n)) == E_ARG and n.value == 0
    assert SCORE_WS(ref(scores()), None) == E_ARG and SCORE_WS(None, C.byref(n)) == E_ARG
