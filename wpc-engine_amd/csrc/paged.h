// Device helpers shared by the operators over paged keys and values
// (kv_append.hip, attn_few.hip, attn_many.hip): the batch's rows, the tokens
// a block's rows see, page addresses, bf16 terms and the softmax pieces.
#pragma once
#include <hip/hip_runtime.h>

#include "wpcg_internal.hpp"

namespace wpcg {

typedef __bf16 pbf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pbf16x8 __attribute__((ext_vector_type(8)));
typedef float pf32x2 __attribute__((ext_vector_type(2)));
typedef float pf32x4 __attribute__((ext_vector_type(4)));
typedef float pf32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t pu32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t pu32x4 __attribute__((ext_vector_type(4)));

// Types of a cache's elements as template arguments.
constexpr int CT_F32 = 0, CT_BF16 = 1, CT_E4M3 = 2;
template <int CT>
constexpr int ct_size() { return CT == CT_F32 ? 4 : CT == CT_BF16 ? 2 : 1; }

// ---- the batch ---------------------------------------------------------------
// Sequence s's rows [a, a + n) and tokens; n = 0: nothing to do for it (its row
// range breaks the batch's bounds, or is empty, or is another kernel's). bad: the length is none.
struct SeqRows {
    int a, n, len;
    bool bad;
};
__device__ __forceinline__ SeqRows seq_rows(const PagedBatch& b, int s)
{
    SeqRows r;
    r.a = b.q_start ? b.q_start[s] : s;
    const int e = b.q_start ? b.q_start[s + 1] : s + 1;
    const bool ok = r.a >= 0 && r.a <= e && e <= b.n_rows && e - r.a <= b.max_q && e - r.a >= b.min_q;
    r.n = ok ? e - r.a : 0;
    r.len = b.kv_len[s];
    r.bad = r.len < 0 || r.len > b.max_kv;
    return r;
}

// The sequence that holds row r: how many of start[1 .. n_seq], which rise, are
// at most r. The wave looks at the ends of 64 groups of sequences at a time, of
// one sequence each up to 64.
__device__ __forceinline__ int seq_of_row(const int32_t* start, int n_seq, int r)
{
    int lo = 0;  // so many are
    for (int left = n_seq; left > 0;) {
        const int step = (left + 63) / 64, at = lo + ((int)(threadIdx.x & 63) + 1) * step;
        const uint64_t most = __ballot(at <= lo + left && start[at <= lo + left ? at : 0] <= r);
        const int groups = __popcll(most);
        lo += groups * step;
        // the next group's end is not, or lies behind the last
        left = min(step - 1, left - groups * step);
    }
    return lo;
}

// The tokens that the rows at positions p0 .. p1 (p0 <= p1, p1 >= 0) see
// together, as a list of TILE-token tiles: tiles [0, head) cover the sinks,
// tiles [first, end) the rest. lo, hi: [lo, hi) and [0, sinks) are the tokens
// themselves. Without rows that see anything total() is 0.
template <int TILE>
struct SeenTiles {
    int head, first, end, lo, hi, sinks;
    __device__ __forceinline__ int total() const { return head + end - first; }
    __device__ __forceinline__ int tile(int v) const { return v < head ? v : first + v - head; }
    __device__ __forceinline__ bool any(int t0, int t1) const  // a token of [t0, t1) seen by some row
    {
        return (t0 < hi && t1 > lo) || t0 < sinks;
    }
    __device__ __forceinline__ bool some(int t) const { return (t < hi && t >= lo) || t < sinks; }
};
template <int TILE>
__device__ __forceinline__ SeenTiles<TILE> seen_tiles(int p0, int p1, int window, int sinks)
{
    SeenTiles<TILE> r;
    r.hi = p1 + 1 > 0 ? p1 + 1 : 0;
    r.lo = window > 0 && p0 - window + 1 > 0 ? p0 - window + 1 : 0;
    if (r.lo > r.hi) r.lo = r.hi;
    r.sinks = window > 0 ? (sinks < r.hi ? sinks : r.hi) : 0;
    if (r.sinks >= r.lo) {  // one range
        r.lo = 0;
        r.sinks = 0;
    }
    r.head = (r.sinks + TILE - 1) / TILE;
    r.end = (r.hi + TILE - 1) / TILE;
    r.first = r.lo / TILE;
    if (r.first < r.head) r.first = r.head;
    if (r.end < r.first) r.end = r.first;
    return r;
}
// Whether the row at position p sees token t.
__device__ __forceinline__ bool row_sees(int p, int t, int window, int sinks)
{
    return t <= p && (window <= 0 || p - t < window || t < sinks);
}

// ---- lane exchanges ------------------------------------------------------------
// Maximum and sum over the lanes l, l ^ 32 and l, l ^ 16, l ^ 32, l ^ 48: the
// swaps leave (own half, own half) and (other half, other half) in two
// registers, one VALU operation each.
__device__ __forceinline__ float max_x32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_x32(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_x16_32(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max_x32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_x16_32(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return sum_x32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// ---- numbers -------------------------------------------------------------------
__device__ __forceinline__ uint32_t pk_bf16_rne(float lo, float hi)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((pf32x2){lo, hi}, pbf16x2));
}
// Two fp32 values' upper halves, lo in the low half: bf16 by truncation.
__device__ __forceinline__ uint32_t pk_upper(float lo, float hi)
{
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// x minus its truncation to bf16, exact; 0 where nothing is left (infinities
// among them), NaN stays.
__device__ __forceinline__ float below_bf16(float x)
{
    const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    return x == hi ? 0.0f : x - hi;
}
// An fp32 pair as three bf16 pairs whose sum is the pair exactly: 8 bits of
// the 24-bit significand each, cut off from the top (truncation cannot
// overflow where rounding to bf16 would).
__device__ __forceinline__ void split3(float a, float b, uint32_t (&t)[3])
{
    t[0] = pk_upper(a, b);
    a = below_bf16(a);
    b = below_bf16(b);
    t[1] = pk_upper(a, b);
    t[2] = pk_upper(below_bf16(a), below_bf16(b));
}
// The same without what keeps infinities from becoming NaN.
__device__ __forceinline__ void split3_finite(float a, float b, uint32_t (&t)[3])
{
    const auto upper = [](float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); };
    t[0] = pk_upper(a, b);
    a -= upper(a);
    b -= upper(b);
    t[1] = pk_upper(a, b);
    t[2] = pk_upper(a - upper(a), b - upper(b));
}
// Two E4M3 bytes (the low or the high half of w) as two bf16, exact.
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3_bf16(uint32_t w)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Bit patterns of two bf16: 1.0 in each half where the value is not finite and
// the test holds (kind 0: +inf, 1: -inf, 2: NaN), else 0; and the pair with
// what is not finite replaced by 0.
__device__ __forceinline__ uint32_t bf16_is(uint32_t w, int kind)
{
    const uint32_t l = w & 0xffffu, h = w >> 16;
    const auto hit = [&](uint32_t x) {
        return kind == 0 ? x == 0x7f80u : kind == 1 ? x == 0xff80u : (x & 0x7fffu) > 0x7f80u;
    };
    return (hit(l) ? 0x3f80u : 0u) | (hit(h) ? 0x3f800000u : 0u);
}
__device__ __forceinline__ uint32_t bf16_finite(uint32_t w)
{
    const uint32_t l = (w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu;
    const uint32_t h = (w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u;
    return l | h;
}
__device__ __forceinline__ bool bf16_odd(uint32_t w)  // either half not finite
{
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// A column's state (maximum, sum, four outputs) with N parts' states added in
// their order; a part that saw nothing has maximum -inf, one that met a page
// that is none the sum NaN.
template <int N>
__device__ __forceinline__ void add_parts(float& m, float& l, pf32x4& o, const float (&mi)[N], const float (&li)[N],
                                          const pf32x4 (&oi)[N])
{
    float now = m;
#pragma unroll
    for (int j = 0; j < N; j++) now = fmaxf(now, mi[j]);
    const float base = now == -INFINITY ? 0.0f : now;
    const float old = exp2_fast(m - base);
    l *= old;
    o *= old;
    m = now;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float f = exp2_fast(mi[j] - base);
        l += f == 0.0f && li[j] == li[j] ? 0.0f : li[j] * f;
        if (f != 0.0f) o += oi[j] * f;
    }
}
// N consecutive outputs of a column, from dimension d on: o / l times the
// values' scale; zeros for a row that sees nothing, NaN where its sequence's
// length is none.
template <int N, bool F32>
__device__ __forceinline__ void attn_store(const PagedAttnArgs& p, const SeqRows& sq, int row, int head, int d, int D,
                                           const float* o, float l, float v_scale)
{
    const bool none = !sq.bad && sq.len - sq.n + row < 0;
    const float f = sq.bad ? __builtin_nanf("") : v_scale / l;
    float r[N];
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = none ? 0.0f : o[i] * f;
    const uint64_t at = (uint64_t)(sq.a + row) * p.out_row + (uint64_t)head * D + d;
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *(pf32x4*)((float*)p.out + at + i) = (pf32x4){r[i], r[i + 1], r[i + 2], r[i + 3]};
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8)
            *(pu32x4*)((uint16_t*)p.out + at + i) =
                (pu32x4){pk_bf16_rne(r[i], r[i + 1]), pk_bf16_rne(r[i + 2], r[i + 3]),
                         pk_bf16_rne(r[i + 4], r[i + 5]), pk_bf16_rne(r[i + 6], r[i + 7])};
    } else {
        static_assert(N == 4, "four or a multiple of eight outputs");
        *(pu32x2*)((uint16_t*)p.out + at) = (pu32x2){pk_bf16_rne(r[0], r[1]), pk_bf16_rne(r[2], r[3])};
    }
}

}  // namespace wpcg
