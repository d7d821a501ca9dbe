// Log probabilities of given tokens, their rank, the entropy and the K largest
// entries of rows of logits.
//
// With M the row's largest logit, t_i = (x_i - M) / T and Z = sum e^(t_i):
//   log p_i = t_i - ln Z,   H = ln Z - sum e^(t_i) t_i / Z
// Every term of H's sum has one sign, so nothing cancels. For a confident row
// ln Z is that of a number just above 1: the ids at the maximum are counted, not
// summed, so that the small terms beside them keep their 24 bits, and ln Z is
// log1p of what is left.
//
// Two launches. The first cuts rows into chunks of 2048 ids, a wave each, held in
// registers: the chunk's maximum, how many reach it, the sums over the others
// relative to it, how many ids come before the given token, and the maximum of
// every 64 ids. Every logit is read once, so memory bounds it. The second, a
// workgroup a row, joins the chunks' states in fp64 and finds the K best: they
// lie in the K segments of 64 ids whose maxima come first (each of these comes
// before anything in another segment), so 64 K logits are read again, not a row.
#include "paged.h"
#include "wave.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256, CHUNK = LOGPROB_CHUNK, VALUES = CHUNK / 64;
constexpr int SEG = 64, SEGS = LOGPROB_SEGS;  // ids of a segment, segments of a chunk
constexpr int LIST = 256;                    // candidates that are sorted by counting

// log2(e) / T; 0: T is infinite, all ids with a logit above -inf are alike; -1:
// greedy (T is not above 0).
__device__ __forceinline__ double row_rate_d(const LogprobArgs& p, int row)
{
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    return t > 0.0f ? 1.4426950408889634 / (double)t : -1.0;
}
// The same in fp32: finite, so that 0 times it is 0.
__device__ __forceinline__ float row_rate(const LogprobArgs& p, int row)
{
    return (float)fmin(row_rate_d(p, row), 3.0e38);
}

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

template <bool BF16>
__global__ __launch_bounds__(THREADS) void k_logprob_stats(LogprobArgs p)
{
    const int groups = (p.chunks + 3) / 4;
    const int row = (int)(blockIdx.x / (unsigned)groups);
    const int chunk = (int)(blockIdx.x % (unsigned)groups) * 4 + ((int)threadIdx.x >> 6);
    if (chunk >= p.chunks) return;
    const int lane = (int)threadIdx.x & 63, id0 = chunk * CHUNK - row_skew(p, row);
    using C = Chunk<BF16>;
    C c;
    c.load(p, row, id0);
    const int token = p.tokens ? p.tokens[row] : -1;
    const bool inside = token >= 0 && token < p.vocab;
    const float xt = inside ? logit(p, row, token) : INFINITY;
    const float rate = row_rate(p, row);

    // maxima of the 64-id segments, which are SEG / PER lanes of one load, and
    // of the chunk
    constexpr int LANES = SEG / C::PER;
    float best = -INFINITY, seg = -INFINITY;
#pragma unroll
    for (int i = 0; i < C::LOADS; i++) {
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < C::PER; j++) m = fmaxf(m, c.v[C::PER * i + j]);
        if (p.top > 0) {
            m = fmaxf(m, wave_dpp<WDPP_XOR1>(m, m));
            m = fmaxf(m, wave_dpp<WDPP_XOR2>(m, m));
            m = fmaxf(m, wave_dpp<WDPP_HALF_MIRROR>(m, m));
            if (LANES == 16) m = fmaxf(m, wave_dpp<WDPP_MIRROR>(m, m));
            if (lane % LANES == i) seg = m;  // lane i of a segment's keeps load i's
        }
        best = fmaxf(best, m);
    }
    if (p.top > 0 && lane % LANES < C::LOADS)
        p.seg[((uint64_t)row * p.chunks + chunk) * SEGS + lane % LANES * (64 / LANES) + lane / LANES] = seg;
    best = wave_max(best);

    const float base = best == -INFINITY ? 0.0f : best;
    float z[2] = {0.0f, 0.0f}, s[2] = {0.0f, 0.0f};
    int tops = 0, before = 0;
    bool same = false;
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
        const float d = c.v[i] - base;
        float t = d * rate;
        if (rate == 0.0f) t = d == -INFINITY ? d : t;
        const bool top = c.v[i] == best;
        // (a NaN reaches z here, and only here)
        const float e = top ? 0.0f : exp2_fast(t);
        z[i & 1] += e;
        s[i & 1] = fmaf(e, fmaxf(t, -200.0f), s[i & 1]);
        tops += __popcll(__ballot(top));
        before += __popcll(__ballot(c.v[i] > xt));
        same |= c.v[i] == xt;
    }
    if (__any(same)) {  // equal logits of lower ids come before, too
#pragma unroll
        for (int i = 0; i < VALUES; i++) before += __popcll(__ballot(c.v[i] == xt && id0 + C::place(i) < token));
    }
    const float zs = wave_sum(z[0] + z[1]), ss = wave_sum(s[0] + s[1]);
    if (lane == 0)
        p.part[(uint64_t)row * p.chunks + chunk] = LogprobPart{best, zs, ss, best == -INFINITY ? 0 : tops, before};
}

// ---- the row's state -------------------------------------------------------------
// (x - M) / T for a logit in base 2, the rate in 64 bits
__device__ __forceinline__ double scaled(float x, float m, double rate)
{
    const double d = (double)x - (double)m;
    return rate == 0.0 ? (d == -INFINITY ? d : d * 0.0) : d * rate;
}
// Sums over the workgroup's four waves.
struct RowSums {
    double z, s;
    int tops, before;
};
__device__ __forceinline__ RowSums block_sums(RowSums v, RowSums* s)
{
    v = {wave_sum_d(v.z), wave_sum_d(v.s), wave_sum_i(v.tops), wave_sum_i(v.before)};
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return {(s[0].z + s[1].z) + (s[2].z + s[3].z), (s[0].s + s[1].s) + (s[2].s + s[3].s),
            s[0].tops + s[1].tops + s[2].tops + s[3].tops, s[0].before + s[1].before + s[2].before + s[3].before};
}

// ---- the K best ------------------------------------------------------------------
// Keys rise with the value, and fall with the place where values are equal; no
// two are the same, and that of a place without a value (NaN, -inf) is 0.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t at)
{
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
    const uint32_t order = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)order << 32 | (uint32_t)~at;
}
__device__ __forceinline__ float value_of(uint64_t key)
{
    const uint32_t order = (uint32_t)(key >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint32_t place_of(uint64_t key) { return (uint32_t)~key; }

struct Lists {
    uint64_t key[LIST];
    int n[THREADS / 64];
};
// All threads' keys at or above `from` (not 0) to the list; how many there are, which
// may be more than it holds. each(f) calls f for the thread's keys, all threads
// alike.
template <class EACH>
__device__ __forceinline__ int collect(Lists& l, uint64_t from, EACH each)
{
    const int wave = (int)threadIdx.x >> 6;
    int mine = 0;
    each([&](uint64_t key) { mine += __popcll(__ballot(key != 0 && key >= from)); });
    if ((threadIdx.x & 63) == 0) l.n[wave] = mine;
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) {
        if (w == wave) at = all;
        all += l.n[w];
    }
    if (all <= LIST)
        each([&](uint64_t key) {
            const bool it = key != 0 && key >= from;
            const uint64_t them = __ballot(it);
            if (it) l.key[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(them >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)them, 0))] = key;
            at += __popcll(them);
        });
    __syncthreads();
    return all;
}
// The k-th largest of all threads' keys (0 where there are fewer), bit by bit: of
// use where equal values make too many candidates to sort.
template <class EACH>
__device__ uint64_t kth_key(int k, Lists& l, EACH each)
{
    uint64_t at = 0;
    for (int bit = 63; bit >= 0; bit--) {
        const uint64_t next = at | (uint64_t)1 << bit;
        int n = 0;
        each([&](uint64_t key) { n += key >= next; });
        n = wave_sum_i(n);
        if ((threadIdx.x & 63) == 0) l.n[threadIdx.x >> 6] = n;
        __syncthreads();
        if (l.n[0] + l.n[1] + l.n[2] + l.n[3] >= k) at = next;
        __syncthreads();
    }
    return at;
}
// The list's entry of this thread, and how many come before it.
__device__ __forceinline__ int rank_in(const Lists& l, int n, uint64_t& key)
{
    const int tid = (int)threadIdx.x;
    key = tid < n ? l.key[tid] : 0;
    int before = 0;
    if ((tid & ~63) < n)
        for (int i = 0; i < n; i++) before += l.key[i] > key;
    return before;
}

constexpr int HELD = 10;  // segments' maxima that a thread has in registers: vocabularies up to 163840

// One row a workgroup.
__global__ __launch_bounds__(THREADS) void k_logprob_finish(LogprobArgs p)
{
    __shared__ RowSums s_sums[4];
    __shared__ float s_max[4];
    __shared__ Lists s_list;
    __shared__ uint64_t s_key[THREADS];
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const LogprobPart* part = p.part + (uint64_t)row * p.chunks;
    // everything that is read first, on its way together
    const int n_seg = p.top > 0 ? p.chunks * SEGS : 0;
    const float* seg = p.seg + (uint64_t)row * n_seg;
    float held[HELD];
    if (n_seg > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++) held[i] = seg[min(tid + i * THREADS, n_seg - 1)];
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
    const auto each_seg = [&](auto f) {
        if (n_seg <= HELD * THREADS) {
#pragma unroll
            for (int i = 0; i < HELD; i++) {
                const int at = tid + i * THREADS;
                f(at < n_seg ? key_of(held[i], (uint32_t)at) : 0);
            }
        } else {
            for (int i0 = 0; i0 < n_seg; i0 += THREADS) {
                const int at = i0 + tid;
                f(at < n_seg ? key_of(seg[at], (uint32_t)at) : 0);
            }
        }
    };
    if (n_seg > 0) {
        uint64_t best = 0;
        each_seg([&](uint64_t key) { best = key > best ? key : best; });
        s_key[tid] = best;
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
    v = block_sums(v, s_sums);
    const double z = v.z + (double)(v.tops - 1);  // Z - 1
    const double ln2 = 0.6931471805599453, nan = __builtin_nan("");
    const bool greedy = rate < 0.0;
    const bool none = !(m > -INFINITY) || (!greedy && m == INFINITY);
    const double log_z = none ? nan : greedy ? 0.0 : log1p(z);
    if (tid == 0) {
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
    if (n_seg == 0) return;

    // The segments: the k-th best of 64 groups (of the threads of one lane number) is
    // no better than the k-th of all; its value is the least of those that fewer
    // than k groups are above (none: all that there are).
    const int k = p.top;
    uint32_t group = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) group = max(group, (uint32_t)(s_key[64 * w + lane] >> 32));
    int above = 0;
#pragma unroll 16
    for (int i = 0; i < 64; i++) above += (uint32_t)__builtin_amdgcn_readlane((int)group, i) > group;
    const uint32_t least = ~(uint32_t)(0x80000000u ^ (uint32_t)wave_max_i((int)(0x80000000u ^ (above < k ? ~group : 0u))));
    uint64_t from = (uint64_t)least << 32;
    int n = collect(s_list, from, each_seg);
    if (n > LIST) n = collect(s_list, kth_key(k, s_list, each_seg), each_seg);
    uint64_t key;
    const int at = rank_in(s_list, n, key);
    if (tid < n && at < k) s_key[at] = key;
    __syncthreads();
    const int segs = min(n, k);
    // their ids: lane l the l-th of a wave's segments
    constexpr int MOST = LOGPROB_TOP / (THREADS / 64);
    const uint32_t worst = segs < k ? 0u : (uint32_t)(s_key[segs - 1] >> 32);
    const int skew = row_skew(p, row);
    uint64_t own[MOST];
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const int y = wave + i * (THREADS / 64);
        own[i] = 0;
        if (y < segs) {
            const int id = (int)(place_of(s_key[y]) * SEG) + lane - skew;
            own[i] = key_of(logit(p, row, min(max(id, 0), p.vocab - 1)), (uint32_t)id);
            if ((uint32_t)id >= (uint32_t)p.vocab || (uint32_t)(own[i] >> 32) < worst) own[i] = 0;
        }
    }
    const auto each_id = [&](auto f) {
#pragma unroll
        for (int i = 0; i < MOST; i++) f(own[i]);
    };
    n = collect(s_list, 0, each_id);
    if (n > LIST) n = collect(s_list, kth_key(k, s_list, each_id), each_id);
    const int place = rank_in(s_list, n, key);
    const auto put = [&](int i, int id, double lp) {
        if (p.top_ids) p.top_ids[(uint64_t)row * k + i] = id;
        if (p.top_logprob) p.top_logprob[(uint64_t)row * k + i] = (float)lp;
    };
    if (tid < n && place < k)
        put(place, (int)place_of(key),
            none ? nan : greedy ? (place == 0 ? 0.0 : -INFINITY) : ln2 * scaled(value_of(key), m, rate) - log_z);
    if (tid >= n && tid < k) put(tid, -1, log_z == log_z ? -INFINITY : nan);
}

}  // namespace

hipError_t launch_logprobs(const LogprobArgs& p, hipStream_t s)
{
    if (p.n_rows == 0) return hipSuccess;
    const dim3 grid((unsigned)p.n_rows * ((unsigned)(p.chunks + 3) / 4));
    if (p.bf16) k_logprob_stats<true><<<grid, dim3(THREADS), 0, s>>>(p);
    else k_logprob_stats<false><<<grid, dim3(THREADS), 0, s>>>(p);
    k_logprob_finish<<<dim3((unsigned)p.n_rows), dim3(THREADS), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace wpcg
