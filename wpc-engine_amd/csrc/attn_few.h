// A workgroup's work of the attention of few rows (attn_few.hip has the layout and
// the measurements): tiles of keys and values against 16 or 32 columns, for any
// set of rows and tokens that a view describes.
#pragma once
#include "paged.h"
#include "wave.h"

namespace wpcg {
namespace few {

constexpr int WAVES = ATTN_FEW_WAVES;
constexpr int THREADS = 64 * WAVES;
constexpr int TILE = ATTN_FEW_TILE;

// Keys of 16 tokens as A fragments. BF16 and E4M3: D/32 fragments of 32
// dimensions; lane (token, g) holds dimensions key_dim(f, g) + 0..7. F32:
// D/16 of four products of 4 dimensions, product e of fragment f taking
// dimension 16 f + 4 g + e from lane group g.
template <int CT>
__device__ __forceinline__ int key_dim(int f, int g)
{
    return CT == CT_F32 ? 16 * f + 4 * g : CT == CT_BF16 ? 32 * f + 8 * g : 64 * (f / 2) + 16 * g + 8 * (f % 2);
}

template <int D, int CT>
struct Keys {
    static constexpr int LOADS = D * ct_size<CT>() / 64;  // of 16 bytes
    pu32x4 w[LOADS];
    // half: the half tile's place (uniform), at: the lane's token and g
    __device__ __forceinline__ void load(const uint8_t* half, uint32_t at)
    {
#pragma unroll
        for (int i = 0; i < LOADS; i++) w[i] = *(const pu32x4*)(half + at + i * 64);
    }
    __device__ __forceinline__ pbf16x8 frag(int f) const  // not F32
    {
        if (CT == CT_BF16) return __builtin_bit_cast(pbf16x8, w[f]);
        const uint32_t a = w[f / 2][f % 2 * 2], b = w[f / 2][f % 2 * 2 + 1];
        const pu32x4 r = {e4m3_bf16<false>(a), e4m3_bf16<true>(a), e4m3_bf16<false>(b), e4m3_bf16<true>(b)};
        return __builtin_bit_cast(pbf16x8, r);
    }
};

// Values of a tile: lane (n, g) holds dimensions n*DV .. n*DV + DV-1 of its
// eight tokens 4g .. 4g+3 and 16 + 4g .. 16 + 4g+3.
template <int D, int CT>
struct Values {
    static constexpr int DV = D / 16;
    static constexpr int WORDS = DV * ct_size<CT>() / 4;  // of one token
    uint32_t w[8][WORDS];
    // half: the half tile's place (uniform), at: the lane's token and dimensions
    __device__ __forceinline__ void load(int x, const uint8_t* half, uint32_t at)
    {
        const uint8_t* p = half + at;
        if constexpr (WORDS >= 4) {
#pragma unroll
            for (int i = 0; i < WORDS / 4; i++) {
                const pu32x4 v = *(const pu32x4*)(p + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; j++) w[x][4 * i + j] = v[j];
            }
        } else if constexpr (WORDS == 2) {
            const pu32x2 v = *(const pu32x2*)p;
            w[x][0] = v[0];
            w[x][1] = v[1];
        } else {
            w[x][0] = *(const uint32_t*)p;
        }
    }
    // Makes the compiler take the words for new ones: their transposed pairs are
    // made where they are used, not once before a branch or for two blocks of
    // columns, for which there are no registers.
    __device__ __forceinline__ void renew()
    {
#pragma unroll
        for (int x = 0; x < 8; x++)
#pragma unroll
            for (int i = 0; i < WORDS; i++) asm volatile("" : "+v"(w[x][i]));
    }
    __device__ __forceinline__ void keep(int x, bool it)
    {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[x][i] = it ? w[x][i] : 0u;
    }
    // bf16 pair of dimensions 2 i, 2 i + 1 of token x (not F32)
    __device__ __forceinline__ uint32_t pair(int x, int i) const
    {
        if (CT == CT_BF16) return w[x][i];
        return i % 2 ? e4m3_bf16<true>(w[x][i / 2]) : e4m3_bf16<false>(w[x][i / 2]);
    }
    __device__ __forceinline__ bool odd() const  // a value that is not finite
    {
        bool r = false;
#pragma unroll
        for (int x = 0; x < 8; x++) {
            if constexpr (CT == CT_F32) {
#pragma unroll
                for (int i = 0; i < WORDS; i++) r |= (w[x][i] & 0x7f800000u) == 0x7f800000u;
            } else {
#pragma unroll
                for (int i = 0; i < DV / 2; i++) r |= bf16_odd(pair(x, i));
            }
        }
        return r;
    }
};

// acc[j] += A_j B over the tile's 32 tokens, A_j being dimension n*DV + j of
// the values, for NT bf16 terms of B. ODD: what is not finite in A is kept out
// of the products and added to the columns of `see` (1.0 where the column sees
// the token) alone; three more products count the +inf, -inf and NaN a column
// sees.
template <int D, int CT, int NT, bool ODD>
__device__ __forceinline__ void add_values(const Values<D, CT>& v, const pbf16x8 (&b)[NT], pf32x4 (&acc)[D / 16],
                                           pbf16x8 see)
{
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
        uint32_t t[8];
#pragma unroll
        for (int x = 0; x < 8; x++) t[x] = v.pair(x, i);
        const auto side = [&](const uint32_t (&w)[8], bool high) {
            pu32x4 r;
#pragma unroll
            for (int x = 0; x < 4; x++)
                r[x] = __builtin_amdgcn_perm(w[2 * x + 1], w[2 * x], high ? 0x07060302u : 0x05040100u);
            return __builtin_bit_cast(pbf16x8, r);
        };
        if constexpr (ODD) {
#pragma unroll 1
            for (int kind = 0; kind < 3; kind++) {
                uint32_t is[8];
#pragma unroll
                for (int x = 0; x < 8; x++) is[x] = bf16_is(t[x], kind);
                const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const pf32x4 k = __builtin_amdgcn_mfma_f32_16x16x32_bf16(side(is, e), see, (pf32x4){}, 0, 0, 0);
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if (k[y] > 0.0f) acc[2 * i + e][y] += add;
                }
            }
#pragma unroll
            for (int x = 0; x < 8; x++) t[x] = bf16_finite(t[x]);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const pbf16x8 a = side(t, e);
#pragma unroll
            for (int k = NT - 1; k >= 0; k--)  // small terms first
                acc[2 * i + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[k], acc[2 * i + e], 0, 0, 0);
        }
    }
}

// What a workgroup of W waves shares; with W = 1 a wave's own.
template <int D, int CT, bool QF32, int NB, int W = ATTN_FEW_WAVES>
struct Shared {
    static constexpr int WAVES = W, THREADS = 64 * W;
    static constexpr int SLOTS = W > 1 ? W / 2 : 1;  // waves whose outputs lie in LDS at a time
    static constexpr bool F32MM = CT == CT_F32;  // the fp32 matrix cores
    static constexpr int QF = F32MM ? D / 16 : D / 32, QT = F32MM || !QF32 ? 1 : 3;  // q's fragments and their terms
    float o[SLOTS][W > 1 ? 16 * NB : 1][D + 4];
    float ml[WAVES][16 * NB][2];
    pu32x4 q[NB][QF][QT][64];
    uint64_t place[WAVES][64];
};

// Which tokens the columns of attend() take of those that their positions see: all.
struct Whole {
    static constexpr bool PART = false;  // outputs, where no part is asked for
    __device__ __forceinline__ bool takes(int) const { return true; }
    __device__ __forceinline__ void clip(int&, int&) const {}
};

// Columns 16 NB cb .. of a sequence's key-value head over tiles [v0, v1) of
// those that `seen` lists (all that the columns see, and then some). Where
// that is all of them the outputs, else their part: [column][D] unnormalised
// at part_o, [column][2] maximum and sum at part_ml. `of` may narrow the tokens
// that are taken (takes, clip). W = 1: a part, by one wave of several that go their
// own ways.
template <int D, int CT, bool QF32, int NB, int W = ATTN_FEW_WAVES, class OF = Whole,
          class SEEN = SeenTiles<TILE>>
__device__ __forceinline__ void attend(const PagedAttnArgs& p, Shared<D, CT, QF32, NB, W>& sh, const SeqRows& sq, int seq,
                                       int kvh, int cb, const SEEN& seen, int v0, int v1, float* part_o,
                                       float* part_ml, const OF& of = OF())
{
    static_assert(OF::PART == (W == 1), "a wave leaves parts");
    using Sh = Shared<D, CT, QF32, NB, W>;
    constexpr int WAVES = Sh::WAVES, THREADS = Sh::THREADS, SLOTS = Sh::SLOTS;
    constexpr bool F32MM = Sh::F32MM;
    constexpr int NT = QF32 ? 3 : 1;  // bf16 terms of q and of the softmax's terms
    constexpr int DV = D / 16;
    constexpr int ES = ct_size<CT>();
    constexpr int COLS = 16 * NB;
    constexpr int QF = Sh::QF;
    auto& s_o = sh.o;
    auto& s_ml = sh.ml;
    auto& s_q = sh.q;
    const int cols = sq.n * p.group;  // of this sequence and head
    const int lane = (int)threadIdx.x & 63, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int len = sq.bad ? 0 : sq.len;
    const int pos0 = len - sq.n;  // position of the sequence's row 0
    const int first = cb * COLS / p.group, last = (min(cols, (cb + 1) * COLS) - 1) / p.group;
    // tokens that every column of the block sees: no mask there
    int all_hi = pos0 + first + 1;
    int all_lo = p.window > 0 ? pos0 + last - p.window + 1 : 0;
    int pos[NB];  // of this lane's columns
#pragma unroll
    for (int n = 0; n < NB; n++) pos[n] = pos0 + min(cb * COLS + 16 * n + c, cols - 1) / p.group;
    of.clip(all_hi, all_lo);

    const uint8_t* const kp = (const uint8_t*)p.k + (uint64_t)kvh * p.head_stride * ES;
    const uint8_t* const vp = (const uint8_t*)p.v + (uint64_t)kvh * p.head_stride * ES;
    const int32_t* const table = p.b.table + (uint64_t)seq * p.b.table_stride;
    const uint64_t page_bytes = p.page_stride * ES;
    const uint32_t token_bytes = (uint32_t)(p.token_stride * ES);  // a page's tokens span less than 2^31 bytes
    const uint32_t k_at = c * token_bytes + g * 16, v_at = 4 * g * token_bytes + c * DV * ES;

    // q as B fragments for LDS, in the keys' order of dimensions: fragment f of
    // column block n by wave (n QF + f) % WAVES
    constexpr int QX = (NB * QF + WAVES - 1) / WAVES;  // of a wave
    pu32x4 qa[QX], qz[QX];
#pragma unroll
    for (int i = 0; i < QX; i++) {
        const int x = i * WAVES + wave, n = x / QF, f = x % QF, col = cb * COLS + 16 * n + c;
        qa[i] = qz[i] = (pu32x4){};
        if (x < NB * QF && col < cols) {
            const uint64_t q_at = (uint64_t)(sq.a + col / p.group) * p.q_row +
                                  (uint64_t)(kvh * p.group + col % p.group) * D + key_dim<CT>(f, g);
            if constexpr (QF32) {
                qa[i] = *(const pu32x4*)((const float*)p.q + q_at);
                if (!F32MM) qz[i] = *(const pu32x4*)((const float*)p.q + q_at + 4);
            } else {
                qa[i] = *(const pu32x4*)((const uint16_t*)p.q + q_at);
            }
        }
    }

    // The places in the pages of the wave's next 32 tiles, in LDS (registers are
    // short): place i is half i % 2 of tile v + WAVES * (i / 2), lane i's. Halves that no row
    // sees read page 0 unlooked at: they are masked. (Looked up tile by tile,
    // every lookup waited for all the loads before it: 66 us instead of 55 for
    // 131072 tokens of E4M3, 32 / 8 heads.)
    bool fault = false;
    const auto look_up = [&](int v) {
        v += WAVES * (lane / 2);
        const int t0 = seen.tile(v) * TILE + 16 * (lane % 2);
        uint64_t at = 0;
        if (v < v1 && seen.any(t0, t0 + 16)) {
            const uint32_t id = (uint32_t)table[t0 >> p.b.page_shift];
            if (id >= p.b.n_pages) fault = true;
            else at = (uint64_t)id * page_bytes + (uint64_t)((t0 & (p.b.page_size - 1)) * token_bytes);
        }
        sh.place[wave][lane] = at;
    };
    const auto place = [&](int tile, int half) -> uint64_t {
        const uint64_t at = sh.place[wave][2 * tile + half];
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 |
               (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    };

    Keys<D, CT> K[2];
    Values<D, CT> V;
    int vt = v0 + wave, turn = 0;
    uint64_t at[2] = {0, 0};
    if (vt < v1) {
        look_up(vt);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            at[h] = place(0, h);
            K[h].load(kp + at[h], k_at);
        }
#pragma unroll
        for (int x = 0; x < 8; x++) V.load(x, vp + at[x / 4], v_at + (x % 4) * token_bytes);
    }
#pragma unroll
    for (int i = 0; i < QX; i++) {
        const int x = i * WAVES + wave, n = x / QF, f = x % QF;
        if (x >= NB * QF) break;
        if constexpr (QF32 && !F32MM) {
            uint32_t t[4][3];
            split3(__uint_as_float(qa[i][0]), __uint_as_float(qa[i][1]), t[0]);
            split3(__uint_as_float(qa[i][2]), __uint_as_float(qa[i][3]), t[1]);
            split3(__uint_as_float(qz[i][0]), __uint_as_float(qz[i][1]), t[2]);
            split3(__uint_as_float(qz[i][2]), __uint_as_float(qz[i][3]), t[3]);
#pragma unroll
            for (int k = 0; k < 3; k++) s_q[n][f][k][lane] = (pu32x4){t[0][k], t[1][k], t[2][k], t[3][k]};
        } else {
            s_q[n][f][0][lane] = qa[i];
        }
    }

    const float sc = p.scale * (p.k_scale ? p.k_scale[kvh] : 1.0f);
    if constexpr (W > 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (LDS does a wave's operations in their order)

    pf32x4 acc[NB][DV] = {};
    float m[NB], l[NB];
#pragma unroll
    for (int n = 0; n < NB; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    for (; vt < v1; vt += WAVES) {
        const int t0 = seen.tile(vt) * TILE;
        const bool more = vt + WAVES < v1;
        turn = (turn + 1) % 32;
        if (turn == 0 && more) look_up(vt + WAVES);
#pragma unroll
        for (int h = 0; h < 2; h++) at[h] = more ? place(turn, h) : 0;
        int again = lane;  // q's fragments are read anew, not kept in registers
        asm volatile("" : "+v"(again));
        // scores
        pf32x4 s[NB][2] = {};
#pragma unroll
        for (int n = 0; n < NB; n++) {
            if constexpr (F32MM) {
#pragma unroll
                for (int f = 0; f < QF; f++) {
                    const pf32x4 q = __builtin_bit_cast(pf32x4, s_q[n][f][0][again]);
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            s[n][h] =
                                __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(K[h].w[f][e]), q[e], s[n][h], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int k = NT - 1; k >= 0; k--)  // small terms first
#pragma unroll
                    for (int f = 0; f < QF; f++) {
                        const pbf16x8 q = __builtin_bit_cast(pbf16x8, s_q[n][f][k][again]);
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(K[h].frag(f), q, s[n][h], 0, 0, 0);
                    }
            }
        }
        // the next keys; behind the last tile, one address for all lanes, so
        // that the number of loads in flight is known at every wait
#pragma unroll
        for (int h = 0; h < 2; h++) {
            K[h].load(kp + at[h], more ? k_at : 0);
        }
        // mask
        const bool whole = t0 + TILE <= all_hi && t0 >= all_lo;
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const int t = t0 + 16 * (x / 4) + 4 * g + x % 4;
                    if (!(row_sees(pos[n], t, p.window, p.sinks) && of.takes(t))) s[n][x / 4][x % 4] = -INFINITY;
                }
        }
        // what a masked token's value holds stays out: tokens that no column
        // sees are cleared, and values that are not finite and that only some
        // columns see are added to those alone
        bool odd = false;
        if (!whole) {
#pragma unroll
            for (int x = 0; x < 8; x++)
                V.keep(x, seen.some(t0 + 16 * (x / 4) + 4 * g + x % 4));
            odd = __any(V.odd());
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
            // running maximum and terms
            float top = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                              fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            top = max_x16_32(top) * sc;
            const float now = fmaxf(m[n], top);
            const float base = now == -INFINITY ? 0.0f : now;
            if (__any(now > m[n])) {
                const float f = exp2_fast(m[n] - base);
                l[n] *= f;
#pragma unroll
                for (int j = 0; j < DV; j++) acc[n][j] *= f;
                m[n] = now;
            }
            float e[8];
#pragma unroll
            for (int x = 0; x < 8; x++) {
                e[x] = exp2_fast(fmaf(s[n][x / 4][x % 4], sc, -base));
                l[n] += e[x];
            }
            const auto sees = [&](int x) {
                const int t = t0 + 16 * (x / 4) + 4 * g + x % 4;
                return row_sees(pos[n], t, p.window, p.sinks) && of.takes(t);
            };
            if constexpr (F32MM) {
                static_assert(NB == 1, "clears what is not finite for one block of columns");
                if (odd) {
#pragma unroll 1
                    for (int kind = 0; kind < 3; kind++) {
                        const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
                        for (int j = 0; j < DV; j++) {
                            pf32x4 k = {};
#pragma unroll
                            for (int x = 0; x < 8; x++) {
                                const uint32_t w = V.w[x][j];
                                const bool hit = kind == 0   ? w == 0x7f800000u
                                                 : kind == 1 ? w == 0xff800000u
                                                             : (w & 0x7fffffffu) > 0x7f800000u;
                                k = __builtin_amdgcn_mfma_f32_16x16x4f32(hit ? 1.0f : 0.0f, sees(x) ? 1.0f : 0.0f, k, 0, 0, 0);
                            }
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (k[i] > 0.0f) acc[n][j][i] += add;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 8; x++)
#pragma unroll
                        for (int j = 0; j < DV; j++)
                            if ((V.w[x][j] & 0x7f800000u) == 0x7f800000u) V.w[x][j] = 0;
                }
#pragma unroll
                for (int x = 0; x < 8; x++)
#pragma unroll
                    for (int j = 0; j < DV; j++)
                        acc[n][j] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(V.w[x][j]), e[x], acc[n][j], 0, 0, 0);
            } else {
                pbf16x8 b[NT];
                if constexpr (QF32) {
                    uint32_t t[4][3];
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        OF::PART ? split3_finite(e[2 * x], e[2 * x + 1], t[x]) : split3(e[2 * x], e[2 * x + 1], t[x]);
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        b[k] = __builtin_bit_cast(pbf16x8, (pu32x4){t[0][k], t[1][k], t[2][k], t[3][k]});
                } else {
                    pu32x4 t;
#pragma unroll
                    for (int x = 0; x < 4; x++) t[x] = pk_bf16_rne(e[2 * x], e[2 * x + 1]);
                    b[0] = __builtin_bit_cast(pbf16x8, t);
                }
                if (n > 0) V.renew();
                if (odd) {
                    if (NB == 1) V.renew();
                    pu32x4 w;
#pragma unroll
                    for (int x = 0; x < 4; x++) w[x] = (sees(2 * x) ? 0x3f80u : 0u) | (sees(2 * x + 1) ? 0x3f800000u : 0u);
                    add_values<D, CT, NT, true>(V, b, acc[n], __builtin_bit_cast(pbf16x8, w));
                } else {
                    if (NB == 1) V.renew();
                    add_values<D, CT, NT, false>(V, b, acc[n], pbf16x8{});
                }
            }
        }
#pragma unroll
        for (int x = 0; x < 8; x++)
            V.load(x, vp + at[x / 4], more ? v_at + (x % 4) * token_bytes : 0);
    }

    // the waves' parts together; a lane's outputs are dimensions
    // (4g + i) * DV + j of its columns
#pragma unroll
    for (int n = 0; n < NB; n++) {
        l[n] = sum_x16_32(l[n]);
        if (__any(fault)) l[n] = __builtin_nanf("");
        if constexpr (W == 1) {
            float* const to = part_o + (16 * n + c) * D;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < DV; j += 4)
                    *(pf32x4*)(to + (4 * g + i) * DV + j) =
                        (pf32x4){acc[n][j][i], acc[n][j + 1][i], acc[n][j + 2][i], acc[n][j + 3][i]};
            if (g == 0) {
                part_ml[(16 * n + c) * 2] = m[n];
                part_ml[(16 * n + c) * 2 + 1] = l[n];
            }
            continue;
        }
        if (g == 0) {
            s_ml[wave][16 * n + c][0] = m[n];
            s_ml[wave][16 * n + c][1] = l[n];
        }
    }
    if constexpr (W == 1) return;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; n++) {
        float top = s_ml[0][16 * n + c][0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) top = fmaxf(top, s_ml[w][16 * n + c][0]);
        const float f = m[n] == -INFINITY ? 0.0f : exp2_fast(m[n] - top);
#pragma unroll
        for (int j = 0; j < DV; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[n][j][i] = f == 0.0f ? 0.0f : acc[n][j][i] * f;
    }
#pragma unroll
    for (int r = 0; r < WAVES / SLOTS; r++) {
        if (wave / SLOTS == r) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < DV; j += 4) {
                        pf32x4* o = (pf32x4*)&s_o[wave % SLOTS][16 * n + c][(4 * g + i) * DV + j];
                        const pf32x4 v = {acc[n][j][i], acc[n][j + 1][i], acc[n][j + 2][i], acc[n][j + 3][i]};
                        *o = r ? *o + v : v;
                    }
        }
        __syncthreads();
    }

    // thread -> column, four dimensions
    constexpr int PER = D / 4;
    for (int x = (int)threadIdx.x; x < COLS * PER; x += THREADS) {
        const int oc = x / PER, od = x % PER * 4;
        const int ocol = cb * COLS + oc;
        if (ocol >= cols) break;
        float om = s_ml[0][oc][0], ol = 0.0f;
#pragma unroll
        for (int w = 1; w < WAVES; w++) om = fmaxf(om, s_ml[w][oc][0]);
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float wm = s_ml[w][oc][0], wl = s_ml[w][oc][1];
            ol += wm == -INFINITY ? (wl != wl ? wl : 0.0f) : wl * exp2_fast(wm - om);
        }
        pf32x4 o = *(const pf32x4*)&s_o[0][oc][od];
#pragma unroll
        for (int w = 1; w < SLOTS; w++) o += *(const pf32x4*)&s_o[w][oc][od];
        const int orow = ocol / p.group, ohead = kvh * p.group + ocol % p.group;
        if (part_o) {
            *(pf32x4*)(part_o + oc * D + od) = o;
            if (od == 0) {
                part_ml[oc * 2] = om;
                part_ml[oc * 2 + 1] = ol;
            }
        } else {
            const float r[4] = {o[0], o[1], o[2], o[3]};
            attn_store<4, QF32>(p, sq, orow, ohead, od, D, r, ol, p.v_scale ? p.v_scale[kvh] : 1.0f);
        }
    }
}

// What LDS gives a whole wave alike, in a scalar register: the compiler takes
// it for each lane's own, and with it every address and branch that follows.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

}  // namespace few
}  // namespace wpcg
