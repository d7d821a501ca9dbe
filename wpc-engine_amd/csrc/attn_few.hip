// Attention of few rows over paged keys and values: one new token of each
// sequence, or the drafts being verified.
//
// Every key and value is read once for the query heads of its group, and with
// one to a few rows that is all there is to do: the memory is the bound (two
// flops a byte and query head). So the kernel is built to keep loads in
// flight. Keys and values are not staged: a wave loads 32 tokens of them
// straight into the matrix cores' operand layout, 16 bytes a lane, and the
// next tile's keys are on their way while this tile's softmax runs. A wave owns
// every eighth tile of the workgroup's chunk, with a running maximum and sum
// of its own; the eight are put together through LDS at the end.
//
// Layout. Columns are (row, query head) pairs, 16 or 32 a workgroup: lane l
// holds column l % 16 throughout (and column 16 + l % 16), lane group g =
// l / 16. With keys as the A operand (16 tokens) and queries as B, the scores
// S^T leave lane (column, g) the tokens 4g .. 4g+3 of a 16-token half. That is
// what the second product needs as its B operand already: a contraction may
// take its terms in any order, so V^T's A operand just takes tokens 4g .. 4g+3
// of both halves in lane group g too, and the terms never leave their lane.
// The running maximum, the sum and the rescaling factor are one number a lane
// and column. V^T needs one dimension's eight tokens side by side: a lane loads
// D/16 dimensions of eight tokens and transposes them in registers, one byte
// permute per two values. The queries' operands stay in LDS, where all waves
// read them (three bf16 terms of F32 queries would take 96 registers).
//
// Precision. With BF16 queries the products are bf16 x bf16 (keys, values and
// queries exact), the softmax's terms rounded to bf16 for the second: half a
// step of relative error on each term, as the output's own rounding has.
// With F32 queries, q and the terms are carried as three bf16 each, exactly,
// over a BF16 or E4M3 cache, and an F32 cache takes the fp32 matrix cores.
//
// Measured, heads of 128, on one card: 64 sequences of up to 4096 tokens, 32 / 4
// heads, BF16 (310 MB) 67.4 us, 4.6 TB/s; one of 131072 tokens, 32 / 8 heads, F32
// queries over E4M3 (268 MB) 51 us, 5.2 TB/s, and 5.7 to join its chunks; 32 with a
// window of 1024 (136 MB) 28.3 us; 16 of up to 6000 with five rows (227 MB) 57 and 5
// us. A 1 GiB copy reaches 5.1 TB/s. One sequence of 300 tokens 10.4 us.
#include "paged.h"

namespace wpcg {
namespace {

constexpr int WAVES = ATTN_FEW_WAVES;
constexpr int THREADS = 64 * WAVES;
constexpr int TILE = ATTN_FEW_TILE;
constexpr int SLOTS = 4;  // waves whose outputs lie in LDS at a time

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

// Tiles of an item of a sequence, at least one (that writes its rows).
__device__ __forceinline__ int item_tiles(const PagedAttnArgs& p, const SeqRows& r)
{
    return r.bad ? 1 : max(1, seen_tiles<TILE>(r.len - r.n, r.len - 1, p.window, p.sinks).total());
}

// What a workgroup shares.
template <int D, int CT, bool QF32, int NB>
struct Shared {
    static constexpr bool F32MM = CT == CT_F32;  // the fp32 matrix cores
    static constexpr int QF = F32MM ? D / 16 : D / 32, QT = F32MM || !QF32 ? 1 : 3;  // q's fragments and their terms
    float o[SLOTS][16 * NB][D + 4];
    float ml[WAVES][16 * NB][2];
    pu32x4 q[NB][QF][QT][64];
    uint64_t place[WAVES][64];
};

// Columns 16 NB cb .. of a sequence's key-value head over tiles [v0, v1) of
// those that `seen` lists (all that the columns see, and then some). Where
// that is all of them the outputs, else their part: [column][D] unnormalised
// at part_o, [column][2] maximum and sum at part_ml.
template <int D, int CT, bool QF32, int NB>
__device__ __forceinline__ void attend(const PagedAttnArgs& p, Shared<D, CT, QF32, NB>& sh, const SeqRows& sq, int seq,
                                       int kvh, int cb, const SeenTiles<TILE>& seen, int v0, int v1, float* part_o,
                                       float* part_ml)
{
    using Sh = Shared<D, CT, QF32, NB>;
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
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int len = sq.bad ? 0 : sq.len;
    const int pos0 = len - sq.n;  // position of the sequence's row 0
    const int first = cb * COLS / p.group, last = (min(cols, (cb + 1) * COLS) - 1) / p.group;
    // tokens that every column of the block sees: no mask there
    const int all_hi = pos0 + first + 1;
    const int all_lo = p.window > 0 ? pos0 + last - p.window + 1 : 0;
    int pos[NB];  // of this lane's columns
#pragma unroll
    for (int n = 0; n < NB; n++) pos[n] = pos0 + min(cb * COLS + 16 * n + c, cols - 1) / p.group;

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
    __syncthreads();

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
                    if (!row_sees(pos[n], t, p.window, p.sinks)) s[n][x / 4][x % 4] = -INFINITY;
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
                return row_sees(pos[n], t0 + 16 * (x / 4) + 4 * g + x % 4, p.window, p.sinks);
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
                    for (int x = 0; x < 4; x++) split3(e[2 * x], e[2 * x + 1], t[x]);
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
        if (g == 0) {
            s_ml[wave][16 * n + c][0] = m[n];
            s_ml[wave][16 * n + c][1] = l[n];
        }
    }
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

// ---- a workgroup an item (a sequence's key-value head and column block), or a
// chunk of its tiles ---------------------------------------------------------------
template <int D, int CT, bool QF32, int NB>
__global__ __launch_bounds__(THREADS, 2) void k_attn_few(PagedAttnArgs p)
{
    __shared__ Shared<D, CT, QF32, NB> sh;
    constexpr int COLS = 16 * NB;
    // the heads of a sequence are neighbours
    const int pairs = p.b.n_seq * p.n_kv;
    const int pair = (int)(blockIdx.x % (unsigned)pairs), rest = (int)(blockIdx.x / (unsigned)pairs);
    const int cb = rest % p.col_blocks, split = rest / p.col_blocks;
    const int seq = pair / p.n_kv;
    const SeqRows sq = seq_rows(p.b, seq);
    const int cols = sq.n * p.group;
    if (cb * COLS >= cols) return;
    const int pos0 = (sq.bad ? 0 : sq.len) - sq.n;
    const SeenTiles<TILE> seen = seen_tiles<TILE>(
        pos0 + cb * COLS / p.group, pos0 + (min(cols, (cb + 1) * COLS) - 1) / p.group, p.window, p.sinks);
    const int v0 = split * p.chunk, v1 = min(v0 + p.chunk, seen.total());
    if (v0 >= v1 && split > 0) return;
    const uint64_t part = (((uint64_t)split * pairs + pair) * p.col_blocks + cb) * COLS;
    const bool whole = p.splits == 1 || seen.total() <= p.chunk;
    attend<D, CT, QF32, NB>(p, sh, sq, seq, pair % p.n_kv, cb, seen, v0, v1, whole ? nullptr : p.part_o + part * D,
                            whole ? nullptr : p.part_ml + part * 2);
}

// Joins the chunks: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over
// those that the row's workgroups had (where one had all it wrote the outputs),
// in an order that depends on the call's bounds alone. PAR groups of D/4 threads share a (row, query head): one where
// the chunks are few, eight where they are many.
template <int D, bool QF32, int PAR>
__global__ __launch_bounds__(256) void k_attn_few_join(PagedAttnArgs p)
{
    constexpr int TH = D / 4, PER = 256 / (TH * PAR);
    __shared__ float s_o[PAR][PER][D];
    __shared__ float s_ml[PAR][PER][2];
    const int tid = (int)threadIdx.x;
    const int part = tid / TH % PAR, mine = tid / (TH * PAR), d = tid % TH * 4;
    const uint64_t x = (uint64_t)blockIdx.x * PER + mine;
    const int head = (int)(x % (unsigned)p.n_heads);
    const uint64_t rest = x / (unsigned)p.n_heads;
    const int row = (int)(rest / (unsigned)p.b.n_seq), seq = (int)(rest % (unsigned)p.b.n_seq);
    SeqRows sq = {};
    if (row < p.b.max_q) sq = seq_rows(p.b, seq);
    bool live = row < sq.n;
    float m = -INFINITY, l = 0.0f;
    pf32x4 o = {};
    if (live) {
        const int kvh = head / p.group, col = row * p.group + head % p.group, cb = col / p.cols;
        const int cols = sq.n * p.group, pos0 = (sq.bad ? 0 : sq.len) - sq.n;
        const int first = cb * p.cols / p.group, last = (min(cols, (cb + 1) * p.cols) - 1) / p.group;
        const int tiles = seen_tiles<TILE>(pos0 + first, pos0 + last, p.window, p.sinks).total();
        live = tiles > p.chunk;
        const int n = live ? (tiles + p.chunk - 1) / p.chunk : 0;
        const uint64_t step = (uint64_t)p.b.n_seq * p.n_kv * p.col_blocks * p.cols;
        const uint64_t at0 = ((uint64_t)(seq * p.n_kv + kvh) * p.col_blocks + cb) * p.cols + col % p.cols;
        for (int i0 = part; i0 < n; i0 += 8 * PAR) {  // eight in flight
            float mi[8], li[8];
            pf32x4 oi[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = i0 + j * PAR;
                const uint64_t at = at0 + (uint64_t)(i < n ? i : part) * step;
                mi[j] = p.part_ml[at * 2];
                li[j] = p.part_ml[at * 2 + 1];
                oi[j] = *(const pf32x4*)(p.part_o + at * D + d);
                if (i >= n) {
                    mi[j] = -INFINITY;
                    li[j] = 0.0f;
                }
            }
            add_parts<8>(m, l, o, mi, li, oi);
        }
    }
    if constexpr (PAR > 1) {
        *(pf32x4*)&s_o[part][mine][d] = o;
        if (d == 0) {
            s_ml[part][mine][0] = m;
            s_ml[part][mine][1] = l;
        }
        __syncthreads();
        if (part != 0) return;
        float mi[PAR], li[PAR];
        pf32x4 oi[PAR];
#pragma unroll
        for (int i = 0; i < PAR; i++) {
            mi[i] = s_ml[i][mine][0];
            li[i] = s_ml[i][mine][1];
            oi[i] = *(const pf32x4*)&s_o[i][mine][d];
        }
        m = -INFINITY;
        l = 0.0f;
        o = (pf32x4){};
        add_parts<PAR>(m, l, o, mi, li, oi);
    }
    if (!live) return;
    const float r[4] = {o[0], o[1], o[2], o[3]};
    attn_store<4, QF32>(p, sq, row, head, d, D, r, l, p.v_scale ? p.v_scale[head / p.group] : 1.0f);
}
template <int D, bool QF32>
void join(const PagedAttnArgs& p, hipStream_t s)
{
    constexpr int MANY = 8;
    const uint64_t all = (uint64_t)p.b.n_seq * p.b.max_q * p.n_heads;
    const auto blocks = [&](int par) { return dim3((unsigned)((all * (D / 4) * par + 255) / 256)); };
    if (p.splits > 4) k_attn_few_join<D, QF32, MANY><<<blocks(MANY), dim3(256), 0, s>>>(p);
    else k_attn_few_join<D, QF32, 1><<<blocks(1), dim3(256), 0, s>>>(p);
}

// ---- the tiles of all items dealt out evenly -----------------------------------
// Long sequences, whose lengths may differ much: every workgroup (one a CU)
// takes an equal share of all items' tiles, laid end to end. A workgroup's
// first and last items may be parts of one; a second launch joins those.
//
// What LDS gives a whole wave alike, in a scalar register: the compiler takes
// it for each lane's own, and with it every address and branch that follows.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// at[s]: tiles before sequence s's items; returns a workgroup's share. TH: the
// workgroup's threads, wave_sums: TH / 64 ints.
template <int TH, int COLS>
__device__ __forceinline__ int deal(const PagedAttnArgs& p, int* at, int* wave_sums)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    int before = 0;
    for (int s0 = 0; s0 < p.b.n_seq; s0 += TH) {
        const int s = s0 + (int)threadIdx.x;
        int v = 0;
        if (s < p.b.n_seq) {
            const SeqRows r = seq_rows(p.b, s);
            v = p.n_kv * ((r.n * p.group + COLS - 1) / COLS) * item_tiles(p, r);
        }
        int t = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int u = __shfl_up(t, d);
            if (lane >= d) t += u;
        }
        if (lane == 63) wave_sums[wave] = t;
        __syncthreads();
        int all = 0, start = before;
#pragma unroll
        for (int w = 0; w < TH / 64; w++) {
            if (w < wave) start += wave_sums[w];
            all += wave_sums[w];
        }
        if (s < p.b.n_seq) at[s] = start + t - v;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) at[p.b.n_seq] = before;
    __syncthreads();
    before = uniform(before);
    return max((before + p.blocks - 1) / p.blocks, ATTN_SHARE_MIN);
}
// The sequence that tile x of all belongs to.
__device__ __forceinline__ int dealt_seq(const int* at, int n_seq, int x)
{
    int lo = 0, hi = n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (uniform(at[mid]) <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <int D, int CT, bool QF32, int NB>
__global__ __launch_bounds__(THREADS, 2) void k_attn_dealt(PagedAttnArgs p)
{
    __shared__ Shared<D, CT, QF32, NB> sh;
    __shared__ int s_at[ATTN_DEAL_SEQS + 1], s_sums[WAVES];
    const int share = deal<THREADS, 16 * NB>(p, s_at, s_sums);
    const int64_t from = (int64_t)blockIdx.x * share;
    const int end = (int)min(from + share, (int64_t)uniform(s_at[p.b.n_seq]));
    int slot = 0;  // of this workgroup's parts
    if (from >= end && threadIdx.x == 0) p.ends[blockIdx.x].seq = -1;
    for (int64_t x = from; x < end;) {
        const int seq = dealt_seq(s_at, p.b.n_seq, (int)x);
        const SeqRows sq = seq_rows(p.b, seq);
        const int tiles = item_tiles(p, sq), in = (int)x - uniform(s_at[seq]);
        const int item = in / tiles, v0 = in % tiles, v1 = min(tiles, v0 + end - (int)x);
        const int cbs = (sq.n * p.group + 16 * NB - 1) / (16 * NB);
        const int pos0 = (sq.bad ? 0 : sq.len) - sq.n;
        const SeenTiles<TILE> seen = seen_tiles<TILE>(pos0, pos0 + sq.n - 1, p.window, p.sinks);
        const uint64_t part = (uint64_t)(blockIdx.x * 2 + slot) * (16 * NB);
        const bool whole = v0 == 0 && v1 == tiles;
        // for the join: the item that ends here and began before
        if (slot == 0 && threadIdx.x == 0) {
            const int64_t start = x - v0;
            const int b0 = (int)(start / share);
            p.ends[blockIdx.x] = v0 > 0 && v1 == tiles
                                     ? AttnEnd{seq, item / cbs, item % cbs, b0, start != (int64_t)b0 * share}
                                     : AttnEnd{-1, 0, 0, 0, 0};
        }
        attend<D, CT, QF32, NB>(p, sh, sq, seq, item / cbs, item % cbs, seen, v0, min(v1, seen.total()),
                                whole ? nullptr : p.part_o + part * D, whole ? nullptr : p.part_ml + part * 2);
        x += v1 - v0;
        slot = 1;
    }
}

// Joins the item that ends in main workgroup b and began in one before it:
// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over its parts, in their
// order. Four columns a workgroup, two groups of D/4 threads a column (D = 64:
// four).
template <int D, bool QF32, int COLS>
__global__ __launch_bounds__(256) void k_attn_dealt_join(PagedAttnArgs p)
{
    constexpr int TH = D / 4, PAR = 64 / TH;
    __shared__ float s_o[4][PAR][D], s_ml[4][PAR][2];
    const int b = (int)(blockIdx.x / (COLS / 4));
    const AttnEnd e = p.ends[b];
    if (e.seq < 0) return;
    const int b0 = e.first, n = b - b0 + 1, cb = e.cb, kvh = e.kvh;
    const SeqRows sq = seq_rows(p.b, e.seq);
    const int tid = (int)threadIdx.x, mine = tid / 64, part = tid % 64 / TH, d = tid % TH * 4;
    const int oc = (int)(blockIdx.x % (COLS / 4)) * 4 + mine, col = cb * COLS + oc;
    const bool live = col < sq.n * p.group;
    // part i: the first one lies where its workgroup left its last item, unless
    // that was its only one
    const auto place = [&](int i) { return (uint64_t)((b0 + i) * 2 + (i == 0 ? e.second : 0)) * COLS + oc; };
    float m = -INFINITY, l = 0.0f;
    pf32x4 o = {};
    for (int i0 = part; i0 < n; i0 += 8 * PAR) {  // eight in flight
        float mi[8], li[8];
        pf32x4 oi[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j * PAR;
            const uint64_t at = place(i < n ? i : part);
            mi[j] = p.part_ml[at * 2];
            li[j] = p.part_ml[at * 2 + 1];
            oi[j] = *(const pf32x4*)(p.part_o + at * D + d);
            if (i >= n) {
                mi[j] = -INFINITY;
                li[j] = 0.0f;
            }
        }
        add_parts<8>(m, l, o, mi, li, oi);
    }
    *(pf32x4*)&s_o[mine][part][d] = o;
    if (d == 0) {
        s_ml[mine][part][0] = m;
        s_ml[mine][part][1] = l;
    }
    __syncthreads();
    if (part != 0 || !live) return;
    float mi[PAR], li[PAR];
    pf32x4 oi[PAR];
#pragma unroll
    for (int i = 0; i < PAR; i++) {
        mi[i] = s_ml[mine][i][0];
        li[i] = s_ml[mine][i][1];
        oi[i] = *(const pf32x4*)&s_o[mine][i][d];
    }
    m = -INFINITY;
    l = 0.0f;
    o = (pf32x4){};
    add_parts<PAR>(m, l, o, mi, li, oi);
    const float r[4] = {o[0], o[1], o[2], o[3]};
    attn_store<4, QF32>(p, sq, col / p.group, kvh * p.group + col % p.group, d, D, r, l,
                        p.v_scale ? p.v_scale[kvh] : 1.0f);
}

template <int D, int CT, bool QF32, int NB>
void go_cols(const PagedAttnArgs& p, hipStream_t s)
{
    if (p.blocks == 0) {
        k_attn_few<D, CT, QF32, NB>
            <<<dim3((unsigned)(p.b.n_seq * p.n_kv * p.col_blocks * p.splits)), dim3(THREADS), 0, s>>>(p);
        if (p.splits > 1) join<D, QF32>(p, s);
    } else {
        k_attn_dealt<D, CT, QF32, NB><<<dim3((unsigned)p.blocks), dim3(THREADS), 0, s>>>(p);
        k_attn_dealt_join<D, QF32, 16 * NB><<<dim3((unsigned)p.blocks * (4 * NB)), dim3(256), 0, s>>>(p);
    }
}
template <int D, int CT, bool QF32>
void go(const PagedAttnArgs& p, hipStream_t s)
{
    if constexpr (CT != CT_F32) {
        if (p.cols == 2 * ATTN_FEW_COLS) {
            go_cols<D, CT, QF32, 2>(p, s);
            return;
        }
    }
    go_cols<D, CT, QF32, 1>(p, s);
}

template <int D>
void go_types(const PagedAttnArgs& p, int q_dtype, int cache_dtype, hipStream_t s)
{
    if (q_dtype == WPCG_DTYPE_BF16) {
        if (cache_dtype == WPCG_DTYPE_BF16) go<D, CT_BF16, false>(p, s);
        else go<D, CT_E4M3, false>(p, s);
    } else {
        if (cache_dtype == WPCG_DTYPE_F32) go<D, CT_F32, true>(p, s);
        else if (cache_dtype == WPCG_DTYPE_BF16) go<D, CT_BF16, true>(p, s);
        else go<D, CT_E4M3, true>(p, s);
    }
}

}  // namespace

hipError_t launch_attn_few(const PagedAttnArgs& p, int head_dim, int q_dtype, int cache_dtype, hipStream_t s)
{
    if (p.b.n_seq == 0) return hipSuccess;
    if (head_dim == 128) go_types<128>(p, q_dtype, cache_dtype, s);
    else go_types<64>(p, q_dtype, cache_dtype, s);
    return hipGetLastError();
}

}  // namespace wpcg
