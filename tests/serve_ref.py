"""Plain 64-bit implementations of the operators of batched serving, and the
inputs their tests share: pages, tables, number formats."""
import ctypes as C

import numpy as np

import wpcg

F32, BF16, E4M3 = wpcg.DTYPE_F32, wpcg.DTYPE_BF16, wpcg.DTYPE_E4M3
SIZE = {F32: 4, BF16: 2, E4M3: 1}
BITS = {F32: np.uint32, BF16: np.uint16, E4M3: np.uint8}
# half a step, relative: the most that one rounding moves a value by
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, E4M3: 2.0 ** -4}


def _e4m3_table():
    b = np.arange(256)
    e, f = (b >> 3) & 15, b & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


E4M3_VALUES = _e4m3_table()


def encode(x, dtype):
    """float values to the bits of a type, to nearest, ties to even; E4M3
    clamped to +-448."""
    x = np.asarray(x, np.float64)
    if dtype == F32:
        return x.astype(np.float32).view(np.uint32)
    if dtype == BF16:
        u = x.astype(np.float32).view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(x), np.uint16(0x7FC0), r)
    pos = E4M3_VALUES[:127]
    a = np.minimum(np.abs(x), 448.0)
    hi = np.searchsorted(pos, np.nan_to_num(a)).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = np.abs(a - pos[lo]), np.abs(pos[hi] - a)
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    r = pick | np.where(np.signbit(x), 128, 0)
    return np.where(np.isnan(x), 127, r).astype(np.uint8)


def decode(bits, dtype):
    if dtype == F32:
        return bits.view(np.float32).astype(np.float64)
    if dtype == BF16:
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return E4M3_VALUES[bits]


NAN_BITS = {F32: 0x7FC00000, BF16: 0x7FC0, E4M3: 0x7F}


class Paged:
    """Pages of a ragged batch in host memory, every place that no token holds
    NaN, and the device objects over them. order: "head" packs [page][head]
    [token][dim], "token" [page][token][head][dim] with some padding."""

    def __init__(self, ctx, rng, dtype, hkv, d, page, kv_len, order="head", scales=False, spare=3, values=True, width=0):
        self.ctx, self.dtype, self.hkv, self.d, self.page = ctx, dtype, hkv, d, page
        self.kv_len = list(kv_len)
        need = [-(-n // page) for n in self.kv_len]
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(need), max(max(need) + 1, 2, width)), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        if order == "head":
            self.strides, self.page_elems = None, hkv * page * d
            self._st = (hkv * page * d, page * d, d)
        else:
            pad = 16  # elements between heads, a multiple of 16 bytes in every type
            tok = hkv * (d + pad) + pad
            self._st = (page * tok + 2 * pad, d + pad, tok)
            self.strides, self.page_elems = self._st, self._st[0]
        self.bits = {}
        self.scale = {n: (0.05 + rng.random(hkv)).astype(np.float32) if scales else np.ones(hkv, np.float32)
                      for n in "kv"}
        for n in "kv":
            self.bits[n] = np.full(self.n_pages * self.page_elems, NAN_BITS[dtype], BITS[dtype])
        # what the tokens hold: [sequence] -> [token][head][d], as stored
        self.real = {n: [] for n in "kv"}
        for n in "kv":
            for s, m in enumerate(self.kv_len):
                x = rng.standard_normal((m, hkv, d)) * (1.0 if n == "k" else 0.7)
                w = encode(x if values else x * 0, dtype)
                self.put(n, s, w)
                self.real[n].append(decode(w, dtype) * self.scale[n][:, None].astype(np.float64))

    def index(self, s, tokens):
        """Places [token][head][d] of a sequence's tokens in the page arrays."""
        t = np.asarray(tokens, np.int64)
        base = self.table[s, t // self.page].astype(np.int64) * self._st[0] + t % self.page * self._st[2]
        return (base[:, None, None] + np.arange(self.hkv)[None, :, None] * self._st[1]
                + np.arange(self.d)[None, None])

    def put(self, n, s, words, tokens=None):
        m = len(words)
        if m:
            self.bits[n][self.index(s, np.arange(m) if tokens is None else tokens)] = words

    def upload(self):
        self.dk, self.dv = self.ctx.upload(self.bits["k"]), self.ctx.upload(self.bits["v"])
        sc = {}
        if self.dtype == E4M3:
            sc = {"k_scale": self.ctx.upload(self.scale["k"]), "v_scale": self.ctx.upload(self.scale["v"])}
        self.kv = wpcg.PagedKv(self.ctx, self.n_pages, self.page, self.hkv, self.d, self.dtype, k=self.dk, v=self.dv,
                               strides=self.strides, **sc)
        return self

    def batch(self, rows, n_rows=None, max_kv=None, max_q=None):
        """rows: new rows per sequence, or None (one each, without q_start)."""
        self.d_len, self.d_table = (self.ctx.upload(np.array(a, np.int32)) for a in (self.kv_len, self.table))
        self.d_start = None
        n = len(self.kv_len)
        if rows is not None:
            self.d_start = self.ctx.upload(np.cumsum([0] + list(rows)).astype(np.int32))
        total = n if rows is None else sum(rows)
        return wpcg.KvBatch(n, n_rows or total, self.d_len, self.d_table, self.table.shape[1],
                            max(self.kv_len) if max_kv is None else max_kv,
                            max_q=max_q or (1 if rows is None else max(rows)), q_start=self.d_start)


def attention(q, k, v, positions, scale, window, sinks):
    """q [rows][heads][d], k and v [tokens][kv heads][d], real values in 64
    bits: outputs, and for each the sums that bound a rounded computation:
    sum p |v| and the largest scale * sum |q k|."""
    r, h, d = q.shape
    m, hkv = k.shape[:2]
    out, mag = np.zeros((r, h, d)), np.zeros((r, h, d))
    reach = np.zeros((r, h, 1))
    t = np.arange(m)
    for i in range(r):
        p = positions[i]
        see = t <= p
        if window:
            see &= (t > p - window) | (t < sinks)
        if not see.any():
            continue
        for e in range(h):
            kk, vv = k[see, e // (h // hkv)], v[see, e // (h // hkv)]
            x = kk @ q[i, e] * scale
            reach[i, e] = (np.abs(kk) @ np.abs(q[i, e])).max() * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, e], mag[i, e] = w @ vv, w @ np.abs(vv)
    return out, mag, reach


def attention_bound(out, mag, reach, d, tokens, q_dtype):
    """How far a computation in the operator's own arithmetic can be off.
    Scores are sums of d products in fp32 (each of the d + 2 steps half a step
    of the magnitude sum, the factor scale * log2 e another): an error of
    (d + 4) 2^-24 reach in the exponent, twice (the term and the sum of terms).
    Terms are 2^x to 2^-22 (hardware exponential and its argument's rounding,
    |x| < 64 * 2^-24 included), their products with the values are added in
    fp32 over the tokens and the parts a long sequence is split in. BF16
    queries round terms (half a step each) and everything rounds its output."""
    eps = 2.0 ** -24
    e = 2 * (d + 4) * eps * reach + 2 * 2.0 ** -20 + (tokens + 80) * eps
    if q_dtype == BF16:
        return mag * (e + HALF[BF16]) * 1.01 + np.abs(out) * HALF[BF16]
    return mag * e + np.abs(out) * HALF[F32]


def normed_turned(x, w, eps, positions, freq):
    """[rows][heads][d] in 64 bits: head norm, then the rotation."""
    y = np.asarray(x, np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    if freq is not None:
        a = np.asarray(positions, np.float64)[:, None, None] * freq
        h = y.shape[-1] // 2
        lo, hi = y[..., :h], y[..., h:]
        y = np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)
    return y


def verify(logits, probs, tokens, u, u_next, temperature):
    """One sequence in 64 bits: (accepted, tokens of its rows)."""
    n, vocab = logits.shape
    x = logits.astype(np.float64)
    out = np.full(n, -1, np.int32)

    def target(i):
        if not (x[i] > -np.inf).any() or np.isnan(x[i]).any() or np.isposinf(x[i]).any():
            return None
        e = np.exp((x[i] - x[i].max()) / float(np.float32(temperature)))
        return e / e.sum()

    k = 0
    if not temperature > 0:
        def best(i):
            m = np.nanmax(np.where(np.isnan(x[i]), -np.inf, x[i]))
            return int(np.flatnonzero(x[i] == m)[0]) if m > -np.inf else -1
        while k + 1 < n and best(k) >= 0 and tokens[k + 1] == best(k):
            k += 1
        nxt = best(k)
    else:
        while k + 1 < n:
            p, d = target(k), int(tokens[k + 1])
            if p is None or d >= vocab:
                break
            q = 1.0 if probs is None else float(probs[k, d])
            if not float(u[k]) * q < p[d]:
                break
            k += 1
        p = target(k)
        if p is None:
            nxt = -1
        else:
            w = p
            if k + 1 < n:
                if probs is None:
                    q = (np.arange(vocab) == int(tokens[k + 1])).astype(np.float64)
                else:
                    q = probs[k].astype(np.float64)
                w = np.maximum(p - q, 0)
                w = w if w.sum() > 0 else p
            c = np.cumsum(w)
            j = int(np.searchsorted(c, float(u_next) * c[-1], side="right"))
            nxt = j if j < vocab else int(np.flatnonzero(w > 0)[-1])
    out[:k] = tokens[1:k + 1]
    out[k] = nxt
    return k, out
