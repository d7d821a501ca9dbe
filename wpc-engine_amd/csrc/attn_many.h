// The pieces of the attention of many rows (attn_many.hip has the layout and the
// measurements): tiles of keys and values on their way to LDS, columns of queries,
// masks, the softmax's terms, outputs.
#pragma once
#include "paged.h"

namespace wpcg {
namespace many {

constexpr int TILE = ATTN_MANY_TILE;

template <int D, int CT, bool QF32>
struct Shape {
    static constexpr int NQ = QF32 ? 3 : 1;         // bf16 terms of q and of the softmax's terms
    static constexpr int NK = CT == CT_F32 ? 3 : 1;  // of keys and values
    static constexpr int NBUF = NK == 1 ? 2 : 1;     // tiles in LDS
    static constexpr int CW = CT == CT_F32 ? 4 : 8;  // dimensions of a value load
    static constexpr int NCH = D / CW;
    static constexpr int KEYS = TILE * (D + 8), VALUES = TILE * D;  // bf16 elements of one term of a tile in LDS
    static constexpr int KT = 16 * (D / 8) / 64;     // key pieces of a lane and tile
    static constexpr int VT = (4 * NCH + 63) / 64;   // value pieces (4 tokens) of a lane and tile
};

// A tile on its way: what one lane carries of the 16 tokens that its wave
// brings in, keys and values (BOTH) or one of them.
template <int D, int CT, bool BOTH>
struct Carried {
    using S = Shape<D, CT, true>;
    static constexpr int KW = 8 * ct_size<CT>() / 4, VW = S::CW * ct_size<CT>() / 4;  // words
    static constexpr int KN = S::KT * KW, VN = S::VT * 4 * VW;
    uint32_t w[BOTH ? KN + VN : KN > VN ? KN : VN];
    __device__ __forceinline__ uint32_t& k(int i, int y) { return w[i * KW + y]; }
    __device__ __forceinline__ uint32_t& v(int i, int x, int y) { return w[(BOTH ? KN : 0) + (i * 4 + x) * VW + y]; }
};
template <int W>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* base, uint32_t at)  // base: uniform
{
    const uint8_t* p = base + at;
    if constexpr (W >= 4) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const pu32x4 x = *(const pu32x4*)(p + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; j++) w[i + j] = x[j];
        }
    } else {
        static_assert(W == 2, "8 bytes");
        const pu32x2 x = *(const pu32x2*)p;
        w[0] = x[0];
        w[1] = x[1];
    }
}

// Whether a word of a cache holds a value that is not finite.
template <int CT>
__device__ __forceinline__ bool word_odd(uint32_t w)
{
    if constexpr (CT == CT_F32) return (w & 0x7f800000u) == 0x7f800000u;
    else if constexpr (CT == CT_BF16) return bf16_odd(w);
    else return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;  // NaN alone: 0x7f
}

// Place of the 16-byte piece (dimensions 8c .. 8c+7, token t) of a tile's keys:
// rows of D + 8 elements, an odd number of pieces, so that sixteen tokens'
// pieces lie in different banks, and every read is one base and a constant.
template <int D>
__device__ __forceinline__ int key_at(int c, int t) { return t * (D + 8) + c * 8; }
// Place of slot (h, p) of 16-token group j of its values: the eight tokens
// 16j + 4h + 0..3 and 16j + 8 + 4h + 0..3 of dimension CW * (p % NCH) + p / NCH.
template <int D>
__device__ __forceinline__ int value_at(int j, int h, int p)
{
    return ((j * (D / 32) + p / 32) * 64 + h * 32 + p % 32) * 8;
}

// What brings tiles from the pages to LDS, in registers on the way: of four
// waves, wave w the tokens 16 w .. 16 w + 15, of eight the first four their
// values and the others their keys. Their places in the pages are looked up 64
// tiles at a time, a tile a lane; where no row sees them page 0 is read
// unlooked at.
template <int D, int CT, int WAVES>
struct Stage {
    using S = Shape<D, CT, true>;
    static constexpr int ES = ct_size<CT>(), CW = S::CW, NCH = S::NCH, NK = S::NK;
    using C = Carried<D, CT, WAVES == 4>;
    C in;
    SeenTiles<TILE> seen;  // of the block's columns
    int v0, v1;            // its tiles
    int all_hi, all_lo;    // tokens that every column sees
    const uint8_t *kp, *vp;
    const int32_t* table;
    uint64_t page_bytes;
    uint32_t token_bytes;  // a page's tokens span less than 2^31 bytes
    uint32_t n_pages;
    int page_shift, page_size;
    int lane, wave;     // wave: which 16 tokens
    bool keys, values;  // what this wave brings
    uint32_t place_lo = 0, place_hi = 0;
    uint32_t offset[4];  // of eight waves: the lane's four pieces
    bool fault = false;

    __device__ __forceinline__ Stage(const PagedAttnArgs& p, int seq, int kvh, const SeenTiles<TILE>& s, int a, int b,
                                     int hi, int lo)
        : seen(s), v0(a), v1(b), all_hi(hi), all_lo(lo)
    {
        kp = (const uint8_t*)p.k + (uint64_t)kvh * p.head_stride * ES;
        vp = (const uint8_t*)p.v + (uint64_t)kvh * p.head_stride * ES;
        table = p.b.table + (uint64_t)seq * p.b.table_stride;
        page_bytes = p.page_stride * ES;
        token_bytes = (uint32_t)(p.token_stride * ES);
        n_pages = p.b.n_pages;
        page_shift = p.b.page_shift;
        page_size = p.b.page_size;
        lane = (int)threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        keys = WAVES == 4 || wave >= 4;
        values = WAVES == 4 || wave < 4;
        wave &= 3;
        if constexpr (WAVES == 8) {
            static_assert(C::KW == C::VW && S::VT == 1 && S::KT <= 4, "four pieces of one size");
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // (behind a head's last piece, the first ones again)
                const int k = lane + 64 * (i % S::KT), v = lane % (4 * NCH);
                const int token = keys ? k / (D / 8) : 8 * (v / NCH % 2) + 4 * (v / (2 * NCH)) + i;
                offset[i] = token * token_bytes + (keys ? k % (D / 8) * 8 : v % NCH * CW) * ES;
            }
        }
    }
    __device__ __forceinline__ bool whole(int vt) const  // no column's mask touches the tile
    {
        const int t0 = seen.tile(vt) * TILE;
        return t0 + TILE <= all_hi && t0 >= all_lo;
    }
    __device__ __forceinline__ void look_up(int vt)
    {
        const int t0 = seen.tile(vt + lane) * TILE + 16 * wave;
        uint64_t at = 0;
        if (vt + lane < v1 && seen.any(t0, t0 + 16)) {
            const uint32_t id = (uint32_t)table[t0 >> page_shift];
            if (id >= n_pages) fault = true;
            else at = (uint64_t)id * page_bytes + (uint64_t)((t0 & (page_size - 1)) * token_bytes);
        }
        place_lo = (uint32_t)at;
        place_hi = (uint32_t)(at >> 32);
    }
    // tile vt to registers; tiles come in their order
    __device__ __forceinline__ void fetch(int vt)
    {
        const int turn = (vt - v0) % 64;
        if (turn == 0) look_up(vt);
        const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)place_hi, turn) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane((int)place_lo, turn);
        if constexpr (WAVES == 8) {
            // keys or values by the same four loads: in two branches they would
            // have registers of their own, and be waited for to be put together
            const uint8_t* const from = (keys ? kp : vp) + at;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t o = offset[i];  // (32 bits, and not 64 made before the loop)
                asm volatile("" : "+v"(o));
                load_words<C::KW>(&in.w[i * C::KW], from, o);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < S::KT; i++) {
            const int x = lane + 64 * i;
            load_words<C::KW>(&in.k(i, 0), kp + at, x / (D / 8) * token_bytes + x % (D / 8) * 8 * ES);
        }
#pragma unroll
        for (int i = 0; i < S::VT; i++) {
            const int x = lane + 64 * i;
            if (4 * NCH % 64 == 0 || x < 4 * NCH) {
                const int n = x % NCH, xh = x / NCH % 2, vh = x / (2 * NCH);
#pragma unroll
                for (int y = 0; y < 4; y++)
                    load_words<C::VW>(&in.v(i, y, 0), vp + at, (8 * xh + 4 * vh + y) * token_bytes + n * CW * ES);
            }
        }
    }
    // Values of tokens that no column sees, which hold anything, become zeros;
    // whether some of the others are not finite. For tiles that are not whole.
    __device__ __forceinline__ bool clean(int vt)
    {
        const int t0 = seen.tile(vt) * TILE;
        bool odd = false;
        if (!values) return false;
#pragma unroll
        for (int i = 0; i < S::VT; i++) {
            const int x = lane + 64 * i, xh = x / NCH % 2, vh = x / (2 * NCH);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool some = seen.some(t0 + 16 * wave + 8 * xh + 4 * vh + k);
#pragma unroll
                for (int y = 0; y < C::VW; y++) {
                    in.v(i, k, y) = some ? in.v(i, k, y) : 0u;
                    odd |= word_odd<CT>(in.v(i, k, y));
                }
            }
        }
        return __any(odd && lane < 4 * NCH);
    }
    // registers to LDS: keys [NK][KEYS], values [NK][VALUES]
    __device__ __forceinline__ void put(uint16_t* k_to, uint16_t* v_to)
    {
        if (keys)
#pragma unroll
        for (int i = 0; i < S::KT; i++) {
            const int x = lane + 64 * i;
            uint16_t* to = k_to + key_at<D>(x % (D / 8), 16 * wave + x / (D / 8));
            if constexpr (CT == CT_F32) {
                uint32_t t[4][3];
#pragma unroll
                for (int y = 0; y < 4; y++)
                    split3(__uint_as_float(in.k(i, 2 * y)), __uint_as_float(in.k(i, 2 * y + 1)), t[y]);
#pragma unroll
                for (int n = 0; n < 3; n++) *(pu32x4*)(to + n * S::KEYS) = (pu32x4){t[0][n], t[1][n], t[2][n], t[3][n]};
            } else if constexpr (CT == CT_BF16) {
                *(pu32x4*)to = (pu32x4){in.k(i, 0), in.k(i, 1), in.k(i, 2), in.k(i, 3)};
            } else {
                *(pu32x4*)to = (pu32x4){e4m3_bf16<false>(in.k(i, 0)), e4m3_bf16<true>(in.k(i, 0)),
                                        e4m3_bf16<false>(in.k(i, 1)), e4m3_bf16<true>(in.k(i, 1))};
            }
        }
        if (values)
#pragma unroll
        for (int i = 0; i < S::VT; i++) {
            const int x = lane + 64 * i;
            if (4 * NCH % 64 == 0 || x < 4 * NCH) {
                const int n = x % NCH, xh = x / NCH % 2, vh = x / (2 * NCH);
#pragma unroll
                for (int y = 0; y < CW / 2; y++) {
                    // bf16 pairs of dimensions 2 y, 2 y + 1 of the four tokens
                    uint32_t t[4][NK];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if constexpr (CT == CT_F32)
                            split3(__uint_as_float(in.v(i, k, 2 * y)), __uint_as_float(in.v(i, k, 2 * y + 1)), t[k]);
                        else if constexpr (CT == CT_BF16)
                            t[k][0] = in.v(i, k, y);
                        else
                            t[k][0] = y % 2 ? e4m3_bf16<true>(in.v(i, k, y / 2)) : e4m3_bf16<false>(in.v(i, k, y / 2));
                    }
#pragma unroll
                    for (int e = 0; e < NK; e++) {
                        uint16_t* to = v_to + e * S::VALUES + 4 * xh;
                        *(pu32x2*)(to + value_at<D>(wave, vh, 2 * y * NCH + n)) =
                            (pu32x2){__builtin_amdgcn_perm(t[1][e], t[0][e], 0x05040100u),
                                     __builtin_amdgcn_perm(t[3][e], t[2][e], 0x05040100u)};
                        *(pu32x2*)(to + value_at<D>(wave, vh, (2 * y + 1) * NCH + n)) =
                            (pu32x2){__builtin_amdgcn_perm(t[1][e], t[0][e], 0x07060302u),
                                     __builtin_amdgcn_perm(t[3][e], t[2][e], 0x07060302u)};
                    }
                }
            }
        }
    }
};

// Values of a tile that are not finite, added to the columns that see their
// token (products with ones count the +inf, -inf and NaN a column sees).
template <int D, int NK>
__device__ __forceinline__ void add_odd(const PagedAttnArgs& p, const uint16_t* values, int t0, int pos,
                                        pf32x16 (&acc)[D / 32])
{
    const int lane = (int)threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < D / 32; d++) {
#pragma unroll 1
        for (int j = 0; j < 4; j++) {
            pu32x4 see;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = t0 + 16 * j + 8 * (i / 2) + 4 * h + 2 * i % 4;
                see[i] = (row_sees(pos, t, p.window, p.sinks) ? 0x3f80u : 0u) |
                         (row_sees(pos, t + 1, p.window, p.sinks) ? 0x3f800000u : 0u);
            }
#pragma unroll 1
            for (int kind = 0; kind < 3; kind++) {
                pf32x16 n = {};
#pragma unroll
                for (int e = 0; e < NK; e++) {
                    const pu32x4 w = *(const pu32x4*)(values + e * TILE * D + value_at<D>(j, 0, 32 * d) + lane * 8);
                    const pu32x4 is = {bf16_is(w[0], kind), bf16_is(w[1], kind), bf16_is(w[2], kind), bf16_is(w[3], kind)};
                    n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pbf16x8, is),
                                                                __builtin_bit_cast(pbf16x8, see), n, 0, 0, 0);
                }
                const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (n[i] > 0.0f) acc[d][i] += add;
            }
        }
    }
}
// ... and zeros in their place; words: the values' 32-bit words.
__device__ __forceinline__ void clear_odd(uint16_t* values, int words)
{
    for (int i = (int)threadIdx.x; i < words; i += (int)blockDim.x) {
        uint32_t* w = (uint32_t*)values + i;
        *w = bf16_finite(*w);
    }
}

// A column's maximum followed: only when it has grown by more than 2^8, for
// terms up to 256 are as exact and the rescaling (an operation per output
// register) is seldom needed. The exponent's base.
template <int N>
__device__ __forceinline__ float follow(float top, float& m, float& l, pf32x16 (&acc)[N])
{
    if (__any(top > m + 8.0f)) {
        const float now = fmaxf(m, top), base = now == -INFINITY ? 0.0f : now;
        // (what a first tile's infinities left in acc is kept)
        const float f = m == -INFINITY ? 1.0f : exp2_fast(m - base);
        l *= f;
#pragma unroll
        for (int d = 0; d < N; d++) acc[d] *= f;
        m = now;
    }
    return m == -INFINITY ? 0.0f : m;
}
// Scores of tokens that the column's row does not see: with o the token's
// place behind this lane's first one and `behind` the row's, it sees those of
// 0 <= behind - o < window (one unsigned comparison) and of o < sinks.
// LIMIT: of no token from `limit` on.
template <bool LIMIT>
__device__ __forceinline__ void mask(const PagedAttnArgs& p, int t0, int pos, pf32x16 (&s)[2], int limit = 0)
{
    const int lane0 = t0 + 4 * (((int)threadIdx.x & 63) >> 5);
    const uint32_t window = p.window > 0 ? (uint32_t)p.window : 0x7fffffffu;
    uint32_t behind = (uint32_t)(pos - lane0);
    int sinks = p.window > 0 ? min(p.sinks, pos + 1) - lane0 : 0;
    asm volatile("" : "+v"(behind), "+v"(sinks));
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int o = 32 * u + 8 * (i / 4) + i % 4;
            s[u][i] = (behind - (uint32_t)o < window || o < sinks) && (!LIMIT || lane0 + o < limit) ? s[u][i] : -INFINITY;
        }
}
__device__ __forceinline__ float top_of(const pf32x16 (&s)[2])
{
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[u][i]);
    return max_x32(top);
}
// q of a column as B fragments: lane (column, h) holds dimensions 16 f + 8 h + 0..7
template <int D, int NQ>
__device__ __forceinline__ void load_q(const PagedAttnArgs& p, uint64_t at, bool live, pbf16x8 (&qb)[D / 16][NQ])
{
#pragma unroll
    for (int f = 0; f < D / 16; f++) {
        if constexpr (NQ == 3) {
            pf32x4 a = {}, b = {};
            if (live) {
                a = *(const pf32x4*)((const float*)p.q + at + 16 * f);
                b = *(const pf32x4*)((const float*)p.q + at + 16 * f + 4);
            }
            uint32_t t[4][3];
            split3(a[0], a[1], t[0]);
            split3(a[2], a[3], t[1]);
            split3(b[0], b[1], t[2]);
            split3(b[2], b[3], t[3]);
#pragma unroll
            for (int n = 0; n < 3; n++)
                qb[f][n] = __builtin_bit_cast(pbf16x8, (pu32x4){t[0][n], t[1][n], t[2][n], t[3][n]});
        } else {
            qb[f][0] =
                __builtin_bit_cast(pbf16x8, live ? *(const pu32x4*)((const uint16_t*)p.q + at + 16 * f) : (pu32x4){});
        }
    }
}
// Eight terms of a column (scores from s[i0] on) as a B fragment, added to l. FINITE:
// an infinite term (of an infinite score) may be NaN.
template <int NQ, bool FINITE = false>
__device__ __forceinline__ void terms(const pf32x16& s, int i0, float sc, float base, float& l, pbf16x8 (&b)[NQ])
{
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        e[i] = exp2_fast(fmaf(s[i0 + i], sc, -base));
        l += e[i];
    }
    if constexpr (NQ == 3) {
        uint32_t t[4][3];
#pragma unroll
        for (int i = 0; i < 4; i++) FINITE ? split3_finite(e[2 * i], e[2 * i + 1], t[i]) : split3(e[2 * i], e[2 * i + 1], t[i]);
#pragma unroll
        for (int n = 0; n < 3; n++) b[n] = __builtin_bit_cast(pbf16x8, (pu32x4){t[0][n], t[1][n], t[2][n], t[3][n]});
    } else {
        b[0] = __builtin_bit_cast(pbf16x8, (pu32x4){pk_bf16_rne(e[0], e[1]), pk_bf16_rne(e[2], e[3]),
                                                    pk_bf16_rne(e[4], e[5]), pk_bf16_rne(e[6], e[7])});
    }
}
// A column's output, or its part of it.
template <int D, int CW, bool QF32>
__device__ __forceinline__ void put_out(const PagedAttnArgs& p, const SeqRows& sq, int seq, bool part, int split, int row,
                                        int head, float m, float l, const pf32x16 (&acc)[D / 32], float v_scale)
{
    constexpr int NCH = D / CW;
    const int h = ((int)threadIdx.x & 63) >> 5;
    const int first = p.part_seq ? seq * p.part_seq : sq.a;
    const uint64_t slot = ((uint64_t)split * p.part_rows + first + row) * p.n_heads + head;
#pragma unroll
    for (int a0 = 0; a0 < NCH / 8; a0++)
#pragma unroll
        for (int b0 = 0; b0 < 4; b0++) {
            float o[CW];
#pragma unroll
            for (int j = 0; j < CW; j++) o[j] = acc[j * NCH / 32][4 * (j * NCH % 32 / 8 + a0) + b0];
            const int d = CW * (8 * a0 + 4 * h + b0);
            if (part) {
#pragma unroll
                for (int j = 0; j < CW; j += 4)
                    *(pf32x4*)(p.part_o + slot * D + d + j) = (pf32x4){o[j], o[j + 1], o[j + 2], o[j + 3]};
            } else {
                attn_store<CW, QF32>(p, sq, row, head, d, D, o, l, v_scale);
            }
        }
    if (part && h == 0) {
        p.part_ml[slot * 2] = m;
        p.part_ml[slot * 2 + 1] = l;
    }
}

// Its part, as column `col` of a workgroup's.
template <int D, int CW>
__device__ __forceinline__ void put_part(float* part_o, float* part_ml, int col, float m, float l,
                                         const pf32x16 (&acc)[D / 32])
{
    constexpr int NCH = D / CW;
    const int h = ((int)threadIdx.x & 63) >> 5;
#pragma unroll
    for (int a0 = 0; a0 < NCH / 8; a0++)
#pragma unroll
        for (int b0 = 0; b0 < 4; b0++)
#pragma unroll
            for (int j = 0; j < CW; j += 4) {
                float o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = acc[(j + i) * NCH / 32][4 * ((j + i) * NCH % 32 / 8 + a0) + b0];
                *(pf32x4*)(part_o + col * D + CW * (8 * a0 + 4 * h + b0) + j) = (pf32x4){o[0], o[1], o[2], o[3]};
            }
    if (h == 0) {
        part_ml[col * 2] = m;
        part_ml[col * 2 + 1] = l;
    }
}

// acc += a b over their bf16 terms, small products first; of two three-term
// numbers the products below 2^-24 of the first are left out.
template <int NA, int NB>
__device__ __forceinline__ pf32x16 mul_terms(const pbf16x8 (&a)[NA], const pbf16x8 (&b)[NB], pf32x16 acc)
{
    if constexpr (NA == 3) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], acc, 0, 0, 0);
    }
    if constexpr (NB == 3) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], acc, 0, 0, 0);
    if constexpr (NA == 3) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], acc, 0, 0, 0);
    if constexpr (NB == 3) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], acc, 0, 0, 0);
}

// Column block `at` of all the sequences' ones, laid end to end: first those of
// sequences with several, the last, which sees most, foremost. Every wave looks
// by itself, 64 sequences at a time.
template <int COLS>
__device__ __forceinline__ bool find_block(const PagedAttnArgs& p, int at, int& seq, int& cb)
{
    const int lane = (int)threadIdx.x & 63;
    for (int pass = 0; pass < 2; pass++)
        for (int s0 = 0; s0 < p.b.n_seq; s0 += 64) {
            const int s = s0 + lane;
            int v = s < p.b.n_seq ? (seq_rows(p.b, s).n * p.group + COLS - 1) / COLS : 0;
            if ((v > 1) != (pass == 0)) v = 0;
            int t = v;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int u = __shfl_up(t, d);
                if (lane >= d) t += u;
            }
            const uint64_t behind = __ballot(t > at);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                seq = s0 + l;
                cb = __builtin_amdgcn_readlane(t, l) - 1 - at;
                return true;
            }
            at -= __builtin_amdgcn_readlane(t, 63);
        }
    return false;
}

// What a workgroup of COLS columns has to do.
template <int COLS>
struct Work {
    int seq, kvh, cb, split, pos0, v0, v1, first, last;  // pos0: position of the sequence's row 0; rows first .. last
    SeqRows sq;
    SeenTiles<TILE> seen;
    // false: nothing
    __device__ __forceinline__ bool find(const PagedAttnArgs& p)
    {
        // workgroup -> column block, chunk, sequence and head: the blocks of a
        // head are `pairs` apart, so that with a multiple of 8 pairs they run on
        // one die and share its L2; the last column blocks, which see most, come
        // first
        if (p.blocks == 0) {
            const int pairs = p.b.n_seq * p.n_kv;
            const int pair = (int)(blockIdx.x % (unsigned)pairs), rest = (int)(blockIdx.x / (unsigned)pairs);
            split = rest % p.splits;
            cb = p.col_blocks - 1 - rest / p.splits;
            seq = pair / p.n_kv;
            kvh = pair % p.n_kv;
        } else {
            const int rest = (int)(blockIdx.x / (unsigned)p.n_kv);
            split = rest % p.splits;
            kvh = (int)(blockIdx.x % (unsigned)p.n_kv);
            if (!find_block<COLS>(p, rest / p.splits, seq, cb)) return false;
        }
        sq = seq_rows(p.b, seq);
        const int cols = sq.n * p.group;
        if (cb * COLS >= cols) return false;
        pos0 = (sq.bad ? 0 : sq.len) - sq.n;
        first = cb * COLS / p.group;
        last = (min(cols, (cb + 1) * COLS) - 1) / p.group;
        seen = seen_tiles<TILE>(pos0 + first, pos0 + last, p.window, p.sinks);
        v0 = split * p.chunk;
        v1 = min(v0 + p.chunk, seen.total());
        return v0 < v1 || split == 0;
    }
    __device__ __forceinline__ int all_hi() const { return pos0 + first + 1; }
    __device__ __forceinline__ int all_lo(const PagedAttnArgs& p) const
    {
        return p.window > 0 ? pos0 + last - p.window + 1 : 0;
    }
};
// A wave's 32 columns from w0 on.
struct Columns {
    static constexpr bool LIMIT = false;  // they see what their positions do
    __device__ __forceinline__ int limit() const { return 0; }
    bool active, live;  // it has some; this lane's is one
    int row, head, pos;
    int hi, lo;  // tokens that all of them see
    SeenTiles<TILE> seen;
    template <int COLS>
    __device__ __forceinline__ Columns(const PagedAttnArgs& p, const Work<COLS>& w, int w0)
    {
        const int cols = w.sq.n * p.group, col = w0 + ((int)threadIdx.x & 31);
        active = w0 < cols;
        live = col < cols;
        row = live ? col / p.group : 0;
        head = w.kvh * p.group + (live ? col % p.group : 0);
        pos = w.pos0 + row;
        const int first = active ? w0 / p.group : 0, last = active ? (min(cols, w0 + 32) - 1) / p.group : 0;
        seen = seen_tiles<TILE>(w.pos0 + first, w.pos0 + last, p.window, p.sinks);
        hi = w.pos0 + first + 1;
        lo = p.window > 0 ? w.pos0 + last - p.window + 1 : 0;
    }
};

// What a workgroup of four waves shares.
template <int D, int CT, bool QF32>
struct Shared {
    using S = Shape<D, CT, QF32>;
    uint16_t k[S::NBUF][S::NK][S::KEYS] __attribute__((aligned(16)));
    uint16_t v[S::NBUF][S::NK][S::VALUES] __attribute__((aligned(16)));
    int odd[S::NBUF][4], fault;
};

// Four waves' 128 columns over the tiles of w: outputs, or parts. COLUMNS says
// whose a wave's are and what they see; with LIMIT parts, where w says.
template <int D, int CT, bool QF32, class COLUMNS, class WORK>
__device__ __forceinline__ void attend(const PagedAttnArgs& p, Shared<D, CT, QF32>& sh, const WORK& w)
{
    using S = Shape<D, CT, QF32>;
    const SeqRows& sq = w.sq;
    const SeenTiles<TILE>& seen = w.seen;
    const int kvh = w.kvh, v0 = w.v0, v1 = w.v1;
    Stage<D, CT, 4> stage(p, w.seq, kvh, seen, v0, v1, w.all_hi(), w.all_lo(p));
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int c = lane & 31, h = lane >> 5;
    const COLUMNS my(p, w, w.cb * ATTN_MANY_COLS + 32 * wave);
    const bool active = my.active, live = my.live;
    const int row = my.row, head = my.head, pos = my.pos;
    pbf16x8 qb[D / 16][S::NQ];
    load_q<D, S::NQ>(p, (uint64_t)(sq.a + row) * p.q_row + (uint64_t)head * D + 8 * h, live, qb);
    const float sc = p.scale * (p.k_scale ? p.k_scale[kvh] : 1.0f);

    pf32x16 acc[D / 32] = {};
    float m = -INFINITY, l = 0.0f;
    if (threadIdx.x == 0) sh.fault = 0;  // (read behind the last barrier, written behind the first)
    __syncthreads();
    // q is there: else its first use in the loop would wait, every time
    // around, for all loads in flight
    if (COLUMNS::LIMIT && v0 < v1) stage.fetch(v0);  // (few tiles: together with the first of them)
    __builtin_amdgcn_s_waitcnt(0);
    if (!COLUMNS::LIMIT && v0 < v1) stage.fetch(v0);
    for (int vt = v0; vt < v1; vt++) {
        const int buf = (vt - v0) % S::NBUF;
        const bool all = stage.whole(vt);
        if (S::NBUF == 1 && vt > v0) __syncthreads();  // the tile before is read
        if (!all) {
            const bool odd = stage.clean(vt);
            if (lane == 0 && stage.values) sh.odd[buf][stage.wave] = odd;
        }
        stage.put(&sh.k[buf][0][0], &sh.v[buf][0][0]);
        __syncthreads();
        if (vt + 1 < v1) stage.fetch(vt + 1);
        const int t0 = seen.tile(vt) * TILE;
        if (!all && (sh.odd[buf][0] | sh.odd[buf][1] | sh.odd[buf][2] | sh.odd[buf][3])) {
            if (active) add_odd<D, S::NK>(p, &sh.v[buf][0][0], t0, pos, acc);
            __syncthreads();
            clear_odd(&sh.v[buf][0][0], S::NK * S::VALUES / 2);
            __syncthreads();
        }
        if (!active || !my.seen.any(t0, t0 + TILE)) continue;

        // Operands come from LDS a group ahead of the products that take
        // them: four fragments of keys (half a group's products hide the
        // reads of the next), then a 16-token group's of the values.
        constexpr int KG = 2 * D / 64, VF = D / 32;  // groups of keys, fragments of a group of values
        pbf16x8 frag[2][4][S::NK];
        const auto load_keys = [&](int x) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < S::NK; e++)
                    frag[x & 1][i][e] =
                        *(const pbf16x8*)&sh.k[buf][e][key_at<D>(2 * (4 * x % (D / 16) + i) + h, 32 * (4 * x / (D / 16)) + c)];
        };
        const auto load_values = [&](int j) {
#pragma unroll
            for (int d = 0; d < VF; d++)
#pragma unroll
                for (int e = 0; e < S::NK; e++)
                    frag[j & 1][d][e] = *(const pbf16x8*)&sh.v[buf][e][value_at<D>(j, 0, 32 * d) + lane * 8];
        };
        // scores of two 32-token halves
        pf32x16 s[2] = {};
        load_keys(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < KG; x++) {
            if (x + 1 < KG) load_keys(x + 1);
            else load_values(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[4 * x / (D / 16)] = mul_terms(frag[x & 1][i], qb[4 * x % (D / 16) + i], s[4 * x / (D / 16)]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (t0 + TILE > my.hi || t0 < my.lo) mask<COLUMNS::LIMIT>(p, t0, pos, s, my.limit());
        const float base = follow(top_of(s) * sc, m, l, acc);
        pbf16x8 b[2][S::NQ];
        terms<S::NQ, COLUMNS::LIMIT>(s[0], 0, sc, base, l, b[0]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j < 3) load_values(j + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (j < 3) terms<S::NQ, COLUMNS::LIMIT>(s[(j + 1) / 2], 8 * ((j + 1) % 2), sc, base, l, b[(j + 1) & 1]);
#pragma unroll
            for (int d = 0; d < VF; d++) {
                acc[d] = mul_terms(frag[j & 1][d], b[j & 1], acc[d]);
                // a product, then a share of the next group's exponentials
                __builtin_amdgcn_sched_group_barrier(0x8, S::NK * S::NQ > 3 ? 6 : S::NQ, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, QF32 ? 24 : 7, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (stage.fault) sh.fault = 1;
    __syncthreads();
    if (!live) return;
    l = sum_x32(l);
    if (sh.fault) l = __builtin_nanf("");
    if constexpr (COLUMNS::LIMIT)
        put_part<D, S::CW>(w.part_o, w.part_ml, 32 * wave + c, m, l, acc);
    else
        put_out<D, S::CW, QF32>(p, sq, w.seq, p.splits > 1 && seen.total() > p.chunk, w.split, row, head, m, l, acc,
                                p.v_scale ? p.v_scale[kvh] : 1.0f);
}

}  // namespace many
}  // namespace wpcg
