"""CPU tests of what the operators of batched serving refuse: every argument
check comes back as a status code before anything reaches a GPU, and a call
whose arguments are right ends at the missing context. Workspace queries need
no GPU at all."""
import ctypes as C

import numpy as np
import pytest

import wpcg
from wpcg import E_ARG, E_SHAPE, E_UNSUPPORTED, OK

F32, BF16, SPLIT, E4M3 = 0, 1, 2, 3
AT = 1 << 20  # an aligned address that nothing here follows
# the library's functions by C name; the classes call the same ones
APPEND, ATTEND, VERIFY = (getattr(wpcg.lib, n) for n in ("wpcg_kv_append", "wpcg_paged_attention", "wpcg_draft_verify"))


def pages(**kw):
    a = dict(k=AT, v=AT, dtype=BF16, n_pages=10, page_size=16, n_kv_heads=2, head_dim=128, page_stride=0, head_stride=0,
             token_stride=0, k_scale=None, v_scale=None)
    a.update(kw)
    return wpcg._KvPages(**a)


def batch(**kw):
    a = dict(n_seq=3, n_rows=5, max_q=3, max_kv=60, table_stride=4, q_start=AT, kv_len=AT, table=AT)
    a.update(kw)
    return wpcg._KvBatch(**a)


def rows(**kw):
    a = dict(q=AT, k=AT, v=AT, dtype=F32, q_out_dtype=BF16, n_heads=8, q_out=2 * AT, eps=1e-6)
    a.update(kw)
    return wpcg._KvRows(**a)


def attention(**kw):
    a = dict(q=AT, out=AT, dtype=BF16, n_heads=8, scale=0.1)
    a.update(kw)
    return wpcg._Attention(**a)


def draft(**kw):
    a = dict(n_seq=2, n_rows=6, max_rows=4, vocab=1000, q_start=AT, logits=AT, draft_probs=AT, tokens=AT, u=AT,
             u_next=AT, temperature=AT, accepted=AT, out=AT)
    a.update(kw)
    return wpcg._Draft(**a)


def ref(x):
    return None if x is None else C.byref(x)


def append(kv, b, r):
    return APPEND(None, ref(kv), ref(b), ref(r), None)


def attend(kv, b, a, ws=AT, n=1 << 40):
    return ATTEND(None, ref(kv), ref(b), ref(a), ws, n, None)


def verify(d, ws=AT, n=1 << 40):
    return VERIFY(None, ref(d), ws, n, None)


def refused(rc, code, text):
    assert rc == code and text in wpcg.last_error(), (rc, wpcg.last_error())


def test_right_arguments_end_at_the_context():
    for rc in (append(pages(), batch(), rows()), attend(pages(), batch(), attention()), verify(draft())):
        refused(rc, E_ARG, "null context")


BAD_PAGES = [
    (dict(dtype=SPLIT), E_ARG, "F32, BF16 or E4M3"), (dict(dtype=9), E_ARG, "F32, BF16 or E4M3"),
    (dict(head_dim=96), E_UNSUPPORTED, "head_dim"), (dict(head_dim=256), E_UNSUPPORTED, "head_dim"),
    (dict(page_size=8), E_SHAPE, "page_size"), (dict(page_size=48), E_SHAPE, "page_size"),
    (dict(page_size=512), E_SHAPE, "page_size"), (dict(n_pages=0), E_ARG, "n_pages"),
    (dict(n_kv_heads=0), E_ARG, "n_kv_heads"), (dict(k_scale=AT), E_ARG, "scales"), (dict(v_scale=AT), E_ARG, "scales"),
    (dict(page_stride=1 << 20, head_stride=2048, token_stride=100), E_SHAPE, "shorter"),
    (dict(page_stride=1 << 20, head_stride=2048), E_SHAPE, "shorter"),
    (dict(page_stride=1 << 20, head_stride=2048, token_stride=132), E_SHAPE, "16 bytes"),
    (dict(page_stride=1 << 45, head_stride=2048, token_stride=128), E_ARG, "too large"),
    # 16 tokens of a page 2^31 bytes apart in all: places in a page are 32-bit offsets
    (dict(page_stride=1 << 32, head_stride=128, token_stride=1 << 26), E_ARG, "too large"),
    (dict(k=None), E_ARG, "null"), (dict(v=None), E_ARG, "null"), (dict(k=AT + 8), E_ARG, "aligned"),
]


@pytest.mark.parametrize("kw,code,text", BAD_PAGES)
def test_pages(kw, code, text):
    refused(append(pages(**kw), batch(), rows()), code, text)
    refused(attend(pages(**kw), batch(), attention()), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_seq=1 << 31), E_ARG, "bounds"), (dict(max_kv=1 << 31), E_ARG, "bounds"), (dict(max_q=0), E_ARG, "max_q"),
    (dict(q_start=None), E_ARG, "q_start"), (dict(q_start=None, max_q=1, n_rows=2), E_ARG, "q_start"),
    (dict(table_stride=3), E_SHAPE, "table"), (dict(kv_len=None), E_ARG, "null"), (dict(table=None), E_ARG, "null"),
])
def test_batches(kw, code, text):
    refused(append(pages(), batch(**kw), rows()), code, text)
    refused(attend(pages(), batch(**kw), attention()), code, text)


def test_model_verification():
    a = np.zeros(4, np.uint32)
    n = C.c_uint32()
    at = a.ctypes.data_as(C.c_void_p)
    refused(wpcg.lib.wpcg_model_verify_sampled(None, at, 4, None, at, 0.5, 1.0, C.byref(n), at), E_ARG, "null")


def test_null_descriptions():
    for rc in (append(None, batch(), rows()), append(pages(), None, rows()), append(pages(), batch(), None),
               attend(None, batch(), attention()), attend(pages(), None, attention()), attend(pages(), batch(), None),
               verify(None)):
        refused(rc, E_ARG, "null")


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=E4M3), E_ARG, "F32 or BF16"), (dict(q_out_dtype=SPLIT), E_ARG, "F32 or BF16"),
    (dict(n_heads=0), E_SHAPE, "n_heads"), (dict(n_heads=7), E_SHAPE, "n_heads"),
    (dict(q_stride=1000), E_SHAPE, "shorter"), (dict(k_stride=255), E_SHAPE, "shorter"),
    (dict(v_stride=257), E_SHAPE, "16 bytes"), (dict(q_out_stride=1028), E_SHAPE, "16 bytes"),
    (dict(q=None), E_ARG, "null"), (dict(q_out=None), E_ARG, "null"), (dict(k=None), E_ARG, "null"),
    (dict(v=None), E_ARG, "null"), (dict(q=AT + 4), E_ARG, "aligned"), (dict(q_norm=AT + 4), E_ARG, "aligned"),
    (dict(q_norm=AT, eps=-1.0), E_ARG, "eps"), (dict(q_norm=AT, eps=float("nan")), E_ARG, "eps"),
    (dict(q_out=AT), E_ARG, "q_out"), (dict(q_out=AT, q_out_dtype=F32, q_out_stride=1028), E_ARG, "q_out"),
])
def test_append_rows(kw, code, text):
    refused(append(pages(), batch(), rows(**kw)), code, text)


def test_append_without_queries_and_in_place():
    for r in (rows(q=None, q_out=None, n_heads=0, q_out_dtype=77), rows(q_out=AT, q_out_dtype=F32)):
        refused(append(pages(), batch(), r), E_ARG, "null context")


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=E4M3), E_ARG, "F32 or BF16"), (dict(n_heads=9), E_SHAPE, "n_heads"), (dict(scale=0.0), E_ARG, "scale"),
    (dict(scale=-1.0), E_ARG, "scale"), (dict(scale=float("nan")), E_ARG, "scale"),
    (dict(scale=float("inf")), E_ARG, "scale"), (dict(q_stride=8), E_SHAPE, "shorter"),
    (dict(out_stride=1025), E_SHAPE, "16 bytes"), (dict(q=None), E_ARG, "null"), (dict(out=None), E_ARG, "null"),
    (dict(out=AT + 2), E_ARG, "aligned"),
])
def test_attention_rows(kw, code, text):
    refused(attend(pages(), batch(), attention(**kw)), code, text)


def test_types_that_do_not_go_together():
    refused(attend(pages(dtype=F32), batch(), attention()), E_UNSUPPORTED, "BF16 queries")
    refused(attend(pages(dtype=F32), batch(), attention(dtype=F32)), E_ARG, "null context")


def test_too_many_workgroups():
    refused(attend(pages(), batch(n_seq=1 << 20, n_rows=1 << 30, max_q=1 << 20), attention()), E_UNSUPPORTED, "workgroups")
    refused(append(pages(n_kv_heads=64), batch(n_rows=1 << 30), rows(n_heads=64)), E_UNSUPPORTED, "workgroups")
    refused(verify(draft(n_rows=1 << 25, vocab=1 << 20)), E_UNSUPPORTED, "workgroups")
    # a launch's threads have to fit 32 bits: 256 a workgroup, one for a row or chunk
    refused(append(pages(), batch(n_rows=1 << 24), rows()), E_UNSUPPORTED, "workgroups")
    refused(append(pages(), batch(n_rows=(1 << 24) - 1), rows()), E_ARG, "null context")
    refused(verify(draft(n_rows=1 << 24)), E_UNSUPPORTED, "workgroups")
    refused(attend(pages(), batch(n_seq=1 << 22, n_rows=1 << 22, max_q=1), attention()), E_UNSUPPORTED, "workgroups")
    refused(attend(pages(), batch(n_seq=1 << 21, n_rows=1 << 21, max_q=1), attention()), E_ARG, "null context")


def workspace(kv, b, a):
    n = C.c_uint64(7)
    assert wpcg.lib.wpcg_paged_attention_workspace(ref(kv), ref(b), ref(a), C.byref(n)) == OK
    return n.value


def test_attention_workspace():
    """None for short sequences, a state of every column or row and head for each
    part; too small a one, none or an unaligned one is refused."""
    assert workspace(pages(), batch(), attention()) == 0
    long = batch(max_kv=100000, table_stride=6250)
    n, part = workspace(pages(), long, attention()), 3 * 2 * 16 * 130 * 4
    assert n > 0 and n % part == 0
    refused(attend(pages(), long, attention(), n=n - 1), E_ARG, "bytes of workspace")
    refused(attend(pages(), long, attention(), ws=None, n=0), E_ARG, "bytes of workspace")
    refused(attend(pages(), long, attention(), ws=AT + 4, n=n), E_ARG, "aligned")
    refused(attend(pages(), long, attention(), n=n), E_ARG, "null context")
    # many sequences that may be long: the same whatever the lengths are
    many = [batch(max_kv=k, table_stride=k // 16, n_rows=n, n_seq=n, max_q=1) for k, n in ((100000, 200), (200000, 300))]
    assert len({workspace(pages(), b, attention()) for b in many}) == 1
    # a window bounds what there is to share
    assert workspace(pages(), long, attention(window=64)) == 0
    rows = batch(max_kv=100000, table_stride=6250, n_seq=1, n_rows=40, max_q=40)
    n, part = workspace(pages(), rows, attention()), 40 * 8 * 130 * 4
    assert n > 0 and n % part == 0
    refused(attend(pages(), rows, attention(), n=n - 1), E_ARG, "bytes of workspace")
    assert wpcg.lib.wpcg_paged_attention_workspace(ref(pages()), ref(batch()), ref(attention()), None) == E_ARG


@pytest.mark.parametrize("kw,code,text", [
    (dict(vocab=0), E_ARG, "vocab"), (dict(vocab=(1 << 30) + 1), E_ARG, "vocab"), (dict(max_rows=0), E_ARG, "max_rows"),
    (dict(max_rows=65), E_ARG, "max_rows"), (dict(q_start=None), E_ARG, "q_start"),
    (dict(logits_stride=999), E_SHAPE, "shorter"), (dict(draft_stride=1), E_SHAPE, "shorter"),
    (dict(logits=None), E_ARG, "null"), (dict(tokens=None), E_ARG, "null"), (dict(u=None), E_ARG, "null"),
    (dict(u_next=None), E_ARG, "null"), (dict(accepted=None), E_ARG, "null"), (dict(out=None), E_ARG, "null"),
])
def test_drafts(kw, code, text):
    refused(verify(draft(**kw)), code, text)


def test_draft_workspace():
    n = C.c_uint64()
    assert wpcg.lib.wpcg_draft_verify_workspace(ref(draft()), C.byref(n)) == OK and n.value > 0
    refused(verify(draft(), n=n.value - 1), E_ARG, "bytes of workspace")
    refused(verify(draft(), ws=AT + 4, n=n.value), E_ARG, "aligned")
    refused(verify(draft(draft_probs=None, temperature=None)), E_ARG, "null context")
    refused(verify(draft(q_start=None, n_rows=8)), E_ARG, "null context")


def test_nothing_to_do_still_checks():
    refused(append(pages(), batch(n_seq=0), rows()), E_ARG, "null context")
    refused(attend(pages(), batch(n_seq=0), attention(scale=0)), E_ARG, "scale")
    refused(verify(draft(n_seq=0)), E_ARG, "null context")


def test_frequencies():
    f = wpcg.rope_frequencies(1e6, 128)
    assert f.dtype == np.float64 and f.shape == (64,)
    assert f[0] == 1.0 and np.allclose(f[63], 1e6 ** (-126 / 128), rtol=1e-14)


def test_workspace_under_loose_bounds():
    """n_rows may be far above what the sequences can have: parts are of max_q
    rows each then, and in any case of at most 2048 workgroups of 128 columns."""
    def of(n_seq, n_rows, max_q, max_kv, heads, hkv, q=BF16, c=BF16, d=128, window=0):
        kv = pages(n_kv_heads=hkv, head_dim=d, dtype=c)
        b = batch(n_seq=n_seq, n_rows=n_rows, max_q=max_q, max_kv=max_kv, table_stride=max_kv // 16 + 1)
        n = C.c_uint64(7)
        a = attention(dtype=q, n_heads=heads, window=window)
        rc = wpcg.lib.wpcg_paged_attention_workspace(ref(kv), ref(b), ref(a), C.byref(n))
        assert rc == OK or (rc == E_UNSUPPORTED and "workgroups" in wpcg.last_error() and n.value == 0)
        return n.value
    for n_seq, max_q, max_kv, heads, hkv in ((1, 64, 131072, 32, 4), (8, 64, 4096, 32, 8), (3, 40, 60000, 8, 2)):
        tight = of(n_seq, n_seq * max_q, max_q, max_kv, heads, hkv)
        assert 0 < tight <= 2048 * 128 * 130 * 4
        for n_rows in (n_seq * max_q + 1, 4000, 32768, 1 << 22):
            assert of(n_seq, n_rows, max_q, max_kv, heads, hkv) == tight
    rng = np.random.default_rng(1)
    for _ in range(3000):
        n_seq, n_rows, max_q, max_kv, window = (int(2 ** x) for x in rng.random(5) * [12, 22, 16, 20, 16])
        hkv, group = int(rng.choice([1, 2, 4, 5, 8])), int(rng.choice([1, 2, 4, 7, 20, 64]))
        q, c = [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, BF16)][int(rng.integers(4))]
        d, window = int(rng.choice([64, 128])), window * int(rng.integers(2))
        n = of(n_seq, n_rows, max_q, max_kv, hkv * group, hkv, q, c, d, window)
        assert n <= 2048 * 128 * (d + 2) * 4, (n_seq, n_rows, max_q, max_kv, hkv, group, q, c, d, window, n)


@pytest.mark.parametrize("scale,taken", [(2.0 ** 127, True), (2.3e38, True), (2.4e38, False), (3.4028235e38, False),
                                         (1e-45, True)])
def test_scales_at_the_ends_of_fp32(scale, taken):
    """The kernels multiply by scale * log2 e in fp32."""
    rc = attend(pages(), batch(), attention(scale=scale))
    refused(rc, E_ARG, "null context" if taken else "scale")


def test_plans_by_their_workspace():
    """The parts that windowed batches are split in (none of them is too short
    for a second one), in 128 and 256 columns a workgroup; and tiles dealt out
    over 256 workgroups, with the table of ends behind their parts."""
    def of(n_seq, n_rows, max_q, max_kv, heads, hkv, d, q, c, window, sinks):
        kv = pages(n_kv_heads=hkv, head_dim=d, dtype=c)
        b = batch(n_seq=n_seq, n_rows=n_rows, max_q=max_q, max_kv=max_kv, table_stride=max_kv // 16 + 1)
        return workspace(kv, b, attention(dtype=q, n_heads=heads, window=window, sinks=sinks))
    for q, c in ((BF16, BF16), (BF16, E4M3), (F32, F32), (F32, BF16), (F32, E4M3)):
        assert of(2, 4, 2, 3001, 8, 2, 128, q, c, 700, 4) == 3 * 2 * 2 * 16 * 130 * 4
        assert of(1, 65, 65, 4000, 4, 1, 128, q, c, 900, 4) == 6 * 65 * 4 * 130 * 4
        window = 12000 if c == E4M3 else 6000
        assert of(130, 260, 2, 40000, 8, 4, 128, q, c, window, 300) == 2 * 256 * 16 * 130 * 4 + 256 * 20
        wide = 32 if c != F32 else 16
        assert of(130, 650, 5, 40000, 16, 4, 128, q, c, window, 300) == 2 * 256 * wide * 130 * 4 + 256 * 20
    for c in (BF16, E4M3):
        for d, rows, lens, window, sinks, parts in (
                (64, [2050], [16384], 0, 0, 3), (128, [2050], [16384], 0, 0, 3), (64, [2050], [8192], 0, 0, 0),
                (128, [1100, 1000], [12000, 4000], 5000, 70, 3), (128, [1000, 3, 900], [12000, 12000, 7001], 5000, 70, 2)):
            n = sum(rows)
            assert of(len(rows), n, max(rows), max(lens), 32, 8, d, BF16, c, window, sinks) == parts * n * 32 * (d + 2) * 4
