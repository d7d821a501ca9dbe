// Log probabilities of given tokens, their rank, the entropy and the K largest
// entries of rows of logits.
//
// With M the row's largest logit, t_i = (x_i - M) / T and Z = sum e^(t_i):
//   log p_i = t_i - ln Z,   H = ln Z - sum e^(t_i) t_i / Z
// Every term of H's sum has one sign, so nothing cancels. For a confident row
// ln Z is that of a number just above 1: where there is little beside the ids at the
// maximum they are counted, not summed, so that the small terms keep their 24 bits,
// and ln Z is log1p of what is left.
//
// Two launches. The first cuts rows into chunks of 2048 ids, a wave each, held in
// registers: the chunk's maximum, how many reach it, the sums over the others
// relative to it, how many ids come before the given token, and the maximum of
// every 64 ids. Every logit is read once, so memory bounds it: 1500 rows of 151936
// F32 logits (912 MB) 147 us, 6.2 TB/s; 777 rows of 32003 BF16 logits 17.6 us for 50
// MB, where the vector work of an id (some 11 operations) is longer. The second, a
// workgroup a row, joins the chunks' states in fp64 and finds the K best: they
// lie in the K segments of 64 ids whose maxima come first (each of these comes
// before anything in another segment), so 64 K logits are read again, not a row.
// It is a chain of two reads and five barriers: 7.4 us for up to 64 rows, 12 for
// 777 rows and K of 50, which are instructions (1400 a wave) rather than waits.
#include "paged.h"
#include "wave.h"
#define KTH_KEY_FN __device__ __forceinline__
#include "kth_key.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256, CHUNK = LOGPROB_CHUNK, VALUES = CHUNK / 64;
constexpr int LIST = THREADS;  // candidates that are sorted by counting
constexpr int SEG = 64, SEGS = LOGPROB_SEGS;  // ids of a segment, segments of a chunk

// log2(e) / T; 0: T is infinite, all ids with a logit above -inf are alike; -1:
// greedy (T is not above 0).
__device__ __forceinline__ double row_rate_d(const LogprobArgs& p, int row)
{
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    return t > 0.0f ? 1.4426950408889634 / (double)t : -1.0;
}
// (x - from) times any rate in fp32. With low rates a difference may be too large for
// fp32 and its product not: the logits are scaled down before. With high ones it may be a
// denormal, and the rate too large: it is scaled up. The rate stays finite, so that 0
// times it is 0, and not 0, so that -inf times it is -inf (2^-149 makes less than 2^-50 of
// any difference that is left).
__device__ __forceinline__ bool ordinary(double rate) { return rate < 0.0 || (rate >= 0x1p-100 && rate <= 0x1p100); }
struct WideRate {
    float fit, grow, by;
    __device__ __forceinline__ explicit WideRate(double rate)
    {
        const bool low = rate < 1.0;
        fit = low ? 0x1p-32f : 1.0f;
        grow = low ? 1.0f : 0x1p32f;
        by = fmaxf((float)(rate * (low ? 0x1p32 : 0x1p-32)), 0x1p-149f);
    }
    __device__ __forceinline__ float operator()(float x, float from) const { return (x * fit - from * fit) * grow * by; }
};

// Rows need not start on 16 bytes: chunks and segments are of places from the last
// 16-byte border before the row's start on, `skew` places before its first id, and
// what lies outside the row counts as -inf.
__device__ __forceinline__ int row_skew(const LogprobArgs& p, int row)
{
    return p.vec ? (int)((uint64_t)row * p.row % (p.bf16 ? 8u : 4u)) : 0;
}
// A chunk's logits in registers: lane l holds places PER * (l + 64 i) + 0 .. PER-1,
// loads of 16 bytes.
template <bool BF16>
struct Chunk {
    static constexpr int PER = BF16 ? 8 : 4, LOADS = VALUES / PER;
    float v[VALUES];
    __device__ __forceinline__ static int place(int i)  // of v[i]
    {
        return PER * ((int)(threadIdx.x & 63) + 64 * (i / PER)) + i % PER;
    }
    // id0: the id at the chunk's first place
    __device__ __forceinline__ void load(const LogprobArgs& p, int row, int id0)
    {
        // one way for the whole wave, and no load behind a condition
        const uint64_t at = (uint64_t)row * p.row + (uint64_t)(int64_t)id0;
        if (p.vec && at + CHUNK <= p.all) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                if constexpr (BF16) {
                    const pu32x4 w = *(const pu32x4*)((const uint16_t*)p.logits + at + place(i * PER));
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
                        v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    }
                } else {
                    const pf32x4 w = *(const pf32x4*)((const float*)p.logits + at + place(i * PER));
#pragma unroll
                    for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < VALUES; i++) {
                const uint64_t x = (uint64_t)row * p.row + min(max(id0 + place(i), 0), p.vocab - 1);
                v[i] = BF16 ? __uint_as_float((uint32_t)((const uint16_t*)p.logits)[x] << 16) : ((const float*)p.logits)[x];
            }
        }
        if (id0 < 0 || id0 + CHUNK > p.vocab) {
#pragma unroll
            for (int i = 0; i < VALUES; i++)
                if ((uint32_t)(id0 + place(i)) >= (uint32_t)p.vocab) v[i] = -INFINITY;
        }
    }
};

__device__ __forceinline__ float logit(const LogprobArgs& p, int row, int id)
{
    const uint64_t x = (uint64_t)row * p.row + id;
    return p.bf16 ? __uint_as_float((uint32_t)((const uint16_t*)p.logits)[x] << 16) : ((const float*)p.logits)[x];
}

// The lane's share of two maxima: b's with `upper`, a's without, over itself and its
// partner, which is the other kind.
constexpr int DPP_QUAD_MIRROR = 0x1B;
template <int CTRL>
__device__ __forceinline__ float max_over(bool upper, float a, float b)
{
    const float give = upper ? a : b;
    return fmaxf(upper ? b : a, wave_dpp<CTRL>(give, give));
}

template <bool BF16>
__global__ __launch_bounds__(THREADS) void k_logprob_stats(LogprobArgs p)
{
    const int groups = (p.chunks + 3) / 4;
    const int row = (int)(blockIdx.x / (unsigned)groups);
    const int chunk = __builtin_amdgcn_readfirstlane((int)(blockIdx.x % (unsigned)groups) * 4 + ((int)threadIdx.x >> 6));
    if (chunk >= p.chunks) return;
    const int lane = (int)threadIdx.x & 63, id0 = chunk * CHUNK - row_skew(p, row);
    using C = Chunk<BF16>;
    C c;
    c.load(p, row, id0);
    const int token = p.tokens ? p.tokens[row] : -1;
    const bool inside = token >= 0 && token < p.vocab;
    const float xt = inside ? logit(p, row, token) : INFINITY;
    const double rate_d = row_rate_d(p, row);

    // maxima of the 64-id segments, which are SEG / PER lanes of one load, and
    // of the chunk
    constexpr int LANES = SEG / C::PER;
    float m[C::LOADS], best = -INFINITY;
#pragma unroll
    for (int i = 0; i < C::LOADS; i++) {
        m[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < C::PER; j++) m[i] = fmaxf(m[i], c.v[C::PER * i + j]);
        best = fmaxf(best, m[i]);
    }
    if (p.top > 0) {
        // a lane keeps half of its loads and hands its partner the others, so that
        // one is left in the end, the same in lanes 2 n and 2 n + 1
        int load = 0;
        if constexpr (LANES == 16) {
            load = lane >> 3 & 1;
#pragma unroll
            for (int i = 0; i < 4; i++) m[i] = max_over<WDPP_MIRROR>(lane & 8, m[2 * i], m[2 * i + 1]);
        }
        load += (lane >> 2 & 1) * (LANES / 8);
#pragma unroll
        for (int i = 0; i < 2; i++) m[i] = max_over<WDPP_HALF_MIRROR>(lane & 4, m[2 * i], m[2 * i + 1]);
        load += (lane >> 1 & 1) * (LANES / 4);
        m[0] = max_over<DPP_QUAD_MIRROR>(lane & 2, m[0], m[1]);
        m[0] = fmaxf(m[0], wave_dpp<WDPP_XOR1>(m[0], m[0]));
        if (lane % 2 == 0)
            p.seg[((uint64_t)row * p.chunks + chunk) * SEGS + load * (64 / LANES) + lane / LANES] = m[0];
    }
    best = wave_max(best);

    int before = 0;
    // greater logits come before the token's, and equal ones of lower ids
    if (inside && best >= xt) {
        if (id0 > token) {
#pragma unroll
            for (int i = 0; i < VALUES; i++) before += __popcll(__ballot(c.v[i] > xt));
        } else if (id0 >= 0 && id0 + CHUNK <= token) {
#pragma unroll
            for (int i = 0; i < VALUES; i++) before += __popcll(__ballot(c.v[i] >= xt));
        } else {
#pragma unroll
            for (int i = 0; i < VALUES; i++)
                before += __popcll(__ballot(c.v[i] > xt || (c.v[i] == xt && (uint32_t)(id0 + C::place(i)) < (uint32_t)token)));
        }
    }

    // Of the maximum itself e^0 = 1 is added like any other term where the sum is
    // 3 and more: 16 additions' roundings of it are 24 of what is left without it.
    // Else ids at the maximum are counted and the others summed again.
    float base = best == -INFINITY ? 0.0f : best, most = best, rate = (float)rate_d;
    if (!ordinary(rate_d)) {  // t itself in the logits' place
        const WideRate scaled(rate_d);
#pragma unroll
        for (int i = 0; i < VALUES; i++) c.v[i] = scaled(c.v[i], base);
        base = most = 0.0f;
        rate = 1.0f;
    }
    float z[4] = {}, s[2] = {};
    int tops = 1;
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
        const float t = (c.v[i] - base) * rate, e = exp2_fast(t);  // (a NaN reaches z)
        z[i & 3] += e;
        s[i & 1] = fmaf(e, fmaxf(t, -200.0f), s[i & 1]);
    }
    // (s is summed here: behind the branch below all terms would have to be kept)
    asm volatile("" : "+v"(s[0]), "+v"(s[1]));
    float zs = wave_sum((z[0] + z[1]) + (z[2] + z[3])) - 1.0f;
    if (!(zs >= 2.0f)) {
        z[0] = z[1] = z[2] = z[3] = 0.0f;
        tops = 0;
        float from = base;  // (differences anew: kept, they would be 32 registers more)
        asm volatile("" : "+v"(from));
#pragma unroll
        for (int i = 0; i < VALUES; i++) {
            const bool top = c.v[i] == most;
            z[i & 3] += top ? 0.0f : exp2_fast((c.v[i] - from) * rate);
            tops += __popcll(__ballot(top));
        }
        zs = wave_sum((z[0] + z[1]) + (z[2] + z[3]));
        if (best == -INFINITY) tops = 0;
    }
    const float ss = wave_sum(s[0] + s[1]);
    if (lane == 0) p.part[(uint64_t)row * p.chunks + chunk] = LogprobPart{best, zs, ss, tops, before};
}

// ---- the row's state -------------------------------------------------------------
// (x - M) / T for a logit in base 2, the rate in 64 bits
__device__ __forceinline__ double scaled(float x, float m, double rate)
{
    const double d = (double)x - (double)m;
    return rate == 0.0 ? (d == -INFINITY ? d : d * 0.0) : d * rate;
}
// Sums over the workgroup's four waves: from each wave, and with a barrier between
// to all.
struct RowSums {
    double z, s;
    int tops, before;
};
__device__ __forceinline__ void give_sums(const RowSums& v, RowSums* s)
{
    const RowSums w = {wave_sum_d(v.z), wave_sum_d(v.s), wave_sum_i(v.tops), wave_sum_i(v.before)};
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = w;
}
__device__ __forceinline__ RowSums all_sums(const RowSums* s)
{
    return {(s[0].z + s[1].z) + (s[2].z + s[3].z), (s[0].s + s[1].s) + (s[2].s + s[3].s),
            s[0].tops + s[1].tops + s[2].tops + s[3].tops, s[0].before + s[1].before + s[2].before + s[3].before};
}

// ---- the K best ------------------------------------------------------------------
// Keys rise with the value, and fall with the place where values are equal; no
// two are the same, and that of a place without a value (NaN, -inf) is 0. Their
// upper halves are the values' order.
__device__ __forceinline__ uint32_t order_of(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
    const uint32_t order = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return v > -INFINITY ? order : 0;
}
__device__ __forceinline__ float value_of(uint64_t key)
{
    const uint32_t order = (uint32_t)(key >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t at) { return order ? (uint64_t)order << 32 | (uint32_t)~at : 0; }
__device__ __forceinline__ uint32_t place_of(uint64_t key) { return (uint32_t)~key; }

// Candidates, in no order; zeros behind them.
struct List {
    alignas(16) uint64_t key[LIST];
    int n;
};
// The wave's keys (each(f) calls f with the order and the place of each) for which
// take(order, place) holds (not for the order 0), to the list. l.n may come to be more than it holds.
template <class EACH, class TAKE>
__device__ __forceinline__ void collect(List& l, EACH each, TAKE take)
{
    int n = 0;
    each([&](uint32_t order, uint32_t at) { n += __popcll(__ballot(take(order, at))); });
    if (n == 0) return;
    int to = 0;
    if ((threadIdx.x & 63) == 0) to = atomicAdd(&l.n, n);
    to = __builtin_amdgcn_readfirstlane(to);
    each([&](uint32_t order, uint32_t at) {
        const bool it = take(order, at);
        const uint64_t them = __ballot(it);
        const int x = to + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(them >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)them, 0));
        if (it && x < LIST) l.key[x] = key_of(order, at);
        to += __popcll(them);
    });
}
// A key that at least k, and no more of all threads' keys than the list holds, are at or
// above, and the list emptied: where equal values make too many candidates to sort, a
// row of which most is masked by the type's lowest value, say. The k-th key's order is
// `lower` at least, places are below `places`.
template <class EACH>
__device__ uint64_t enough_from(int k, uint32_t lower, int places, List& l, EACH each)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const auto all_waves = [&](int x, uint64_t (&got)[4]) {
        __syncthreads();
        if (lane == 0) l.key[wave] = (uint32_t)x;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++) got[w] = l.key[w];
    };
    const auto sum = [&](int x) {
        uint64_t g[4];
        all_waves(x, g);
        return __builtin_amdgcn_readfirstlane((int)(g[0] + g[1] + g[2] + g[3]));
    };
    if (lower == 0) lower = 1;
    int low = 0x7fffffff;  // (as a signed number)
    each([&](uint32_t order, uint32_t) { low = order >= lower ? min(low, (int)(order ^ 0x80000000u)) : low; });
    uint64_t g[4];
    all_waves(~wave_max_i(~low), g);
    const uint32_t least = (uint32_t)min(min((int)g[0], (int)g[1]), min((int)g[2], (int)g[3])) ^ 0x80000000u;
    const KthKey found = kth_key(
        k, LIST, least, places,
        [&](uint32_t order0) {
            int n = 0;
            each([&](uint32_t order, uint32_t) { n += __popcll(__ballot(order >= order0)); });
            return sum(n);
        },
        [&](uint32_t of, int place) {
            int n = 0;
            each([&](uint32_t order, uint32_t at) { n += __popcll(__ballot(order == of && at <= (uint32_t)place)); });
            return sum(n);
        });
    __syncthreads();
    l.key[threadIdx.x] = 0;
    l.n = 0;
    __syncthreads();
    return key_of(found.order, (uint32_t)found.place);
}
// The thread's entry of the list (0: none), and how many come before it.
__device__ __forceinline__ int rank_in(const List& l, int n, uint64_t& key)
{
    const int tid = (int)threadIdx.x;
    key = 0;
    int before = 0;
    if (__builtin_amdgcn_readfirstlane(tid) >= n) return before;
    key = l.key[tid];
    for (int i = 0; i < n; i += 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) before += l.key[i + j] > key;
    }
    return before;
}
// The k-th largest order of N a lane (0: there are fewer), its lower half cut off:
// two bits a step, from the numbers of lanes at or above.
template <int N>
__device__ __forceinline__ uint32_t kth_about(const uint32_t (&v)[N], int k)
{
    uint32_t at = 0;
#pragma unroll
    for (int bit = 30; bit >= 16; bit -= 2) {
        uint32_t up = 0;
#pragma unroll
        for (uint32_t x = 1; x < 4; x++) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < N; j++) n += __popcll(__ballot(v[j] >= (at | x << bit)));
            up += n >= k;
        }
        at |= up << bit;
    }
    return at;
}

constexpr int HELD = 10;  // segments' maxima that a thread has in registers: vocabularies up to 163840

// One row a workgroup.
__global__ __launch_bounds__(THREADS) void k_logprob_finish(LogprobArgs p)
{
    __shared__ RowSums s_sums[4];
    __shared__ float s_max[4];
    __shared__ uint32_t s_least;
    __shared__ double s_log_z;
    __shared__ List s_list[2];
    __shared__ uint32_t s_best[THREADS];
    __shared__ uint64_t s_key[LOGPROB_TOP];
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LogprobPart* part = p.part + (uint64_t)row * p.chunks;
    s_list[0].key[tid] = 0;
    s_list[1].key[tid] = 0;
    if (tid < 2) s_list[tid].n = 0;
    // everything that is read first, on its way together
    const int n_seg = p.top > 0 ? p.chunks * SEGS : 0;
    const float* seg = p.seg + (uint64_t)row * n_seg;
    float maxima[HELD];
    if (n_seg > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            maxima[i] = -INFINITY;
            if (i * THREADS < n_seg) maxima[i] = seg[min(tid + i * THREADS, n_seg - 1)];
        }
    }
    const LogprobPart mine = part[min(tid, p.chunks - 1)];
    const double rate = row_rate_d(p, row);
    const int token = p.tokens ? p.tokens[row] : -1;
    const bool inside = token >= 0 && token < p.vocab;
    const float x = inside ? logit(p, row, token) : -INFINITY;

    float m = tid < p.chunks ? mine.max : -INFINITY;
    for (int c = tid + THREADS; c < p.chunks; c += THREADS) m = fmaxf(m, part[c].max);
    m = wave_max(m);
    if (lane == 0) s_max[wave] = m;
    // the best of the thread's segments, for below
    uint32_t held[HELD];
    const auto each_seg = [&](auto f) {
        if (n_seg <= HELD * THREADS) {
#pragma unroll
            for (int i = 0; i < HELD; i++) f(held[i], (uint32_t)(tid + i * THREADS));
        } else {
            for (int i0 = 0; i0 < n_seg; i0 += THREADS) {
                const int at = i0 + tid;
                f(at < n_seg ? order_of(seg[at]) : 0, (uint32_t)at);
            }
        }
    };
    if (n_seg > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++) held[i] = tid + i * THREADS < n_seg ? order_of(maxima[i]) : 0;
        uint32_t best = 0;
        each_seg([&](uint32_t order, uint32_t) { best = max(best, order); });
        s_best[tid] = best;
    }
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    // Z without the ids at the maximum, how many those are, and sum e^t t, in base 2
    RowSums v = {0.0, 0.0, 0, 0};
    const auto add = [&](const LogprobPart& q) {
        v.before += q.before;
        if (q.max == m) {
            v.z += (double)q.z;
            v.tops += q.tops;
            v.s += (double)q.s;
        } else {
            const double t = scaled(q.max == -INFINITY ? m : q.max, m, rate), f = exp2(t), all = (double)q.z + (double)q.tops;
            v.z += all * f;
            v.s += ((double)q.s + all * t) * f;
        }
    };
    if (tid < p.chunks) add(mine);
    for (int c = tid + THREADS; c < p.chunks; c += THREADS) add(part[c]);
    give_sums(v, s_sums);

    // The segments: the k-th best of groups of them is no better than the k-th of
    // all. Groups of the threads with one lane number are 64 and the k-th says
    // enough up to k of 24; beyond, half as large ones.
    const int k = p.top;
    if (n_seg > 0) {
        if (wave == THREADS / 64 - 1) {  // (the last wave: it has fewest chunks)
            const uint32_t best[2] = {max(s_best[lane], s_best[64 + lane]), max(s_best[128 + lane], s_best[192 + lane])};
            const uint32_t all[1] = {max(best[0], best[1])};
            s_least = max(k <= 24 ? kth_about(all, k) : kth_about(best, k), 1u);
        }
        __syncthreads();
        const uint32_t least = __builtin_amdgcn_readfirstlane(s_least);
        collect(s_list[0], each_seg, [&](uint32_t order, uint32_t) { return order >= least; });
    }
    __syncthreads();
    // their ids: lane l the l-th of a wave's segments
    constexpr int MOST = LOGPROB_TOP / (THREADS / 64);
    int id[MOST], segs = 0;
    uint32_t own[MOST];  // as they are read
    if (n_seg > 0) {
        if (s_list[0].n > LIST) {
            const uint64_t from = enough_from(k, s_least, n_seg, s_list[0], each_seg);
            collect(s_list[0], each_seg, [&](uint32_t order, uint32_t at) { return order != 0 && key_of(order, at) >= from; });
            __syncthreads();
        }
        const int n = __builtin_amdgcn_readfirstlane(s_list[0].n);
        uint64_t key;
        const int at = rank_in(s_list[0], n, key);
        if (key != 0 && at < k) s_key[at] = key;
        segs = min(n, k);
        __syncthreads();
        const int skew = row_skew(p, row);
#pragma unroll
        for (int i = 0; i < MOST; i++) id[i] = (int)(place_of(s_key[wave + i * (THREADS / 64)]) * SEG) + lane - skew;
        const auto read = [&](auto* x) {
#pragma unroll
            for (int i = 0; i < MOST; i++)
                if (wave + i * (THREADS / 64) < segs) own[i] = x[min(max(id[i], 0), p.vocab - 1)];
        };
        if (p.bf16) read((const uint16_t*)p.logits + (uint64_t)row * p.row);
        else read((const uint32_t*)p.logits + (uint64_t)row * p.row);
    }

    // (while they are on their way)
    const double ln2 = 0.6931471805599453, nan = __builtin_nan("");
    const bool greedy = rate < 0.0;
    const bool none = !(m > -INFINITY) || (!greedy && m == INFINITY);
    if (wave == 0) {
        v = all_sums(s_sums);
        const double z = v.z + (double)(v.tops - 1);  // Z - 1
        const double log_z = none ? nan : greedy ? 0.0 : log1p(z);
        if (tid == 0) {
            s_log_z = log_z;
            if (p.entropy) p.entropy[row] = (float)(none ? nan : greedy ? 0.0 : log_z - ln2 * v.s / (z + 1.0));
            if (p.tokens) {
                const int rank = inside && x == x ? 1 + v.before : 0;
                if (p.rank) p.rank[row] = rank;
                if (p.logprob)
                    p.logprob[row] = (float)(none     ? nan
                                             : greedy ? (rank == 1 && x > -INFINITY ? 0.0 : -INFINITY)
                                                      : ln2 * scaled(x, m, rate) - log_z);
            }
        }
    }
    if (n_seg == 0) return;

    const uint32_t worst = segs < k ? 0u : (uint32_t)(s_key[segs - 1] >> 32);
#pragma unroll
    for (int i = 0; i < MOST; i++)
        if (wave + i * (THREADS / 64) < segs) {
            const uint32_t order = order_of(__uint_as_float(p.bf16 ? own[i] << 16 : own[i]));
            own[i] = (uint32_t)id[i] < (uint32_t)p.vocab && order >= worst ? order : 0;
        }
    const auto each_id = [&](auto f) {
#pragma unroll
        for (int i = 0; i < MOST; i++)
            if (wave + i * (THREADS / 64) < segs) f(own[i], (uint32_t)id[i]);
    };
    collect(s_list[1], each_id, [](uint32_t order, uint32_t) { return order != 0; });
    __syncthreads();
    if (s_list[1].n > LIST) {
        const uint64_t from = enough_from(k, worst, p.vocab, s_list[1], each_id);
        collect(s_list[1], each_id, [&](uint32_t order, uint32_t at) { return order != 0 && key_of(order, at) >= from; });
        __syncthreads();
    }
    const int n = __builtin_amdgcn_readfirstlane(s_list[1].n);
    uint64_t key;
    const int place = rank_in(s_list[1], n, key);
    const double log_z = s_log_z;
    const auto put = [&](int i, int id, double lp) {
        if (p.top_ids) p.top_ids[(uint64_t)row * k + i] = id;
        if (p.top_logprob) p.top_logprob[(uint64_t)row * k + i] = (float)lp;
    };
    if (key != 0 && place < k)
        put(place, (int)place_of(key),
            none ? nan : greedy ? (place == 0 ? 0.0 : -INFINITY) : ln2 * scaled(value_of(key), m, rate) - log_z);
    if (tid >= n && tid < k) put(tid, -1, log_z == log_z ? -INFINITY : nan);
}

}  // namespace

hipError_t launch_logprobs(const LogprobArgs& p, hipStream_t s)
{
    (void)hipGetLastError();  // report only these launches
    if (p.n_rows == 0) return hipSuccess;
    const dim3 grid((unsigned)p.n_rows * ((unsigned)(p.chunks + 3) / 4));
    // F32 rows in many rounds of workgroups come from the memory faster to four of them a
    // CU than to eight, which unused LDS sees to: 1500 rows of 151936 151 us and 158; 64
    // rows, less than a round, 17.3 and 17.0.
    const unsigned room = !p.bf16 && grid.x >= 4 * 8 * 256 ? 40000 : 0;
    if (p.bf16) k_logprob_stats<true><<<grid, dim3(THREADS), 0, s>>>(p);
    else k_logprob_stats<false><<<grid, dim3(THREADS), room, s>>>(p);
    k_logprob_finish<<<dim3((unsigned)p.n_rows), dim3(THREADS), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace wpcg
