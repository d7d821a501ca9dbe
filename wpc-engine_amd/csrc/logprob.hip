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

// A chunk's logits in registers: lane l holds ids PER * (l + 64 i) + 0 .. PER-1,
// loads of 16 bytes; -inf behind the row's end.
template <bool BF16>
struct Chunk {
    static constexpr int PER = BF16 ? 8 : 4, LOADS = VALUES / PER;
    float v[VALUES];
    __device__ __forceinline__ static int id(int i)  // of v[i]
    {
        return PER * ((int)(threadIdx.x & 63) + 64 * (i / PER)) + i % PER;
    }
    __device__ __forceinline__ void load(const LogprobArgs& p, int row, int c0)
    {
        const uint64_t at = (uint64_t)row * p.row + c0;
        // one way for the whole wave, and no load behind a condition
        if (p.vec && c0 + CHUNK <= p.vocab) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                if constexpr (BF16) {
                    const pu32x4 w = *(const pu32x4*)((const uint16_t*)p.logits + at + id(i * PER));
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
                        v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    }
                } else {
                    const pf32x4 w = *(const pf32x4*)((const float*)p.logits + at + id(i * PER));
#pragma unroll
                    for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < VALUES; i++) {
                const uint64_t x = (uint64_t)row * p.row + min(c0 + id(i), p.vocab - 1);
                v[i] = BF16 ? __uint_as_float((uint32_t)((const uint16_t*)p.logits)[x] << 16) : ((const float*)p.logits)[x];
            }
#pragma unroll
            for (int i = 0; i < VALUES; i++)
                if (c0 + id(i) >= p.vocab) v[i] = -INFINITY;
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
    const int lane = (int)threadIdx.x & 63, c0 = chunk * CHUNK;
    using C = Chunk<BF16>;
    C c;
    c.load(p, row, c0);
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
        for (int i = 0; i < VALUES; i++) before += __popcll(__ballot(c.v[i] == xt && c0 + C::id(i) < token));
    }
    const float zs = wave_sum(z[0] + z[1]), ss = wave_sum(s[0] + s[1]);
    if (lane == 0)
        p.part[(uint64_t)row * p.chunks + chunk] = LogprobPart{best, zs, ss, best == -INFINITY ? 0 : tops, before};
}

// ---- the row's state -------------------------------------------------------------
__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ double block_sum_f64(double v, double* s)
{
    v = wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ int block_sum_i(int v, int* s)
{
    v = wave_sum_i(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0] + s[1] + s[2] + s[3];
    __syncthreads();
    return v;
}

// (x - M) / T for a logit in base 2, the rate in 64 bits
__device__ __forceinline__ double scaled(float x, float m, double rate)
{
    const double d = (double)x - (double)m;
    return rate == 0.0 ? (d == -INFINITY ? d : d * 0.0) : d * rate;
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
__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// The k-th largest of all threads' keys (0 where there are fewer), bit by bit: of
// use where equal values make too many candidates to sort. each(f) calls f for
// the thread's keys.
template <class EACH>
__device__ uint64_t kth_key(int k, int* s, EACH each)
{
    uint64_t at = 0;
    for (int bit = 63; bit >= 0; bit--) {
        const uint64_t next = at | (uint64_t)1 << bit;
        int n = 0;
        each([&](uint64_t key) { n += key >= next; });
        if (block_sum_i(n, s) >= k) at = next;
    }
    return at;
}

struct Lists {
    uint64_t key[LIST];
    int n;
};
// All threads' keys at or above `from` to the list; how many there are, which may
// be more than it holds.
template <class EACH>
__device__ __forceinline__ int collect(Lists& l, uint64_t from, EACH each)
{
    if (threadIdx.x == 0) l.n = 0;
    __syncthreads();
    each([&](uint64_t key) {
        if (key != 0 && key >= from) {
            const int at = atomicAdd(&l.n, 1);
            if (at < LIST) l.key[at] = key;
        }
    });
    __syncthreads();
    const int n = l.n;
    __syncthreads();
    return n;
}
// The thread's entry of a list of n <= LIST and how many come before it.
__device__ __forceinline__ int rank_of(const Lists& l, int n, uint64_t& key)
{
    const int tid = (int)threadIdx.x;
    key = tid < n ? l.key[tid] : 0;
    int before = 0;
    if ((tid & ~63) < n)
        for (int i = 0; i < n; i++) before += l.key[i] > key;
    return before;
}

// The K best ids of a row with their keys to best[0 .. K), as many as there are.
__device__ int best_ids(const LogprobArgs& p, int row, Lists& list, uint64_t* best, int* s_i)
{
    __shared__ uint64_t s_key[THREADS], s_from;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_seg = p.chunks * SEGS, k = p.top;
    const float* seg = p.seg + (uint64_t)row * n_seg;
    const auto each_seg = [&](auto f) {
        for (int i0 = tid; i0 < n_seg; i0 += 8 * THREADS) {  // eight in flight
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = seg[min(i0 + j * THREADS, n_seg - 1)];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i0 + j * THREADS < n_seg) f(key_of(v[j], (uint32_t)(i0 + j * THREADS)));
        }
    };
    // the k-th of 64 groups' best is at most the k-th of all
    uint64_t mine = 0;
    each_seg([&](uint64_t key) { mine = key > mine ? key : mine; });
    s_key[tid] = mine;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int w = 1; w < THREADS / 64; w++) mine = s_key[64 * w + lane] > mine ? s_key[64 * w + lane] : mine;
        int before = 0;
#pragma unroll 8
        for (int i = 0; i < 64; i++) before += lane_key(mine, i) > mine;
        if (lane == 0) s_from = 0;
        if (mine != 0 && before == k - 1) s_from = mine;  // (0: fewer groups than k hold any)
    }
    __syncthreads();
    uint64_t from = s_from;
    int n = collect(list, from, each_seg);
    if (n > LIST) {
        from = kth_key(k, s_i, each_seg);
        n = collect(list, from, each_seg);
    }
    uint64_t key;
    const int at = rank_of(list, n, key);
    if (tid < n && at < k) s_key[at] = key;
    __syncthreads();
    const int segs = min(n, k);
    // their ids: lane l the l-th of a wave's segments
    constexpr int MOST = LOGPROB_TOP / (THREADS / 64);
    const uint32_t least = segs < k ? 0u : (uint32_t)(s_key[segs - 1] >> 32);
    uint64_t own[MOST];
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const int x = wave + i * (THREADS / 64);
        own[i] = 0;
        if (x < segs) {
            const uint32_t id = (uint32_t)~s_key[x] * SEG + lane;
            own[i] = key_of(logit(p, row, min(id, (uint32_t)p.vocab - 1)), id);
            if (id >= (uint32_t)p.vocab || (uint32_t)(own[i] >> 32) < least) own[i] = 0;
        }
    }
    const auto each_id = [&](auto f) {
#pragma unroll
        for (int i = 0; i < MOST; i++) f(own[i]);
    };
    n = collect(list, 0, each_id);
    if (n > LIST) n = collect(list, kth_key(k, s_i, each_id), each_id);
    const int place = rank_of(list, n, key);
    if (tid < n && place < k) best[place] = key;
    __syncthreads();
    return min(n, k);
}

__global__ __launch_bounds__(THREADS) void k_logprob_finish(LogprobArgs p)
{
    __shared__ double s_d[4];
    __shared__ float s_f[4];
    __shared__ int s_i[4];
    __shared__ Lists s_list;
    __shared__ uint64_t s_best[LOGPROB_TOP];
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x;
    const LogprobPart* part = p.part + (uint64_t)row * p.chunks;
    const double rate = row_rate_d(p, row);

    float m = -INFINITY;
    for (int c = tid; c < p.chunks; c += THREADS) m = fmaxf(m, part[c].max);
    m = wave_max(m);
    if ((tid & 63) == 0) s_f[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
    // Z without the ids at the maximum, how many those are, and sum e^t t, in base 2
    double z = 0.0, s = 0.0;
    int before = 0, tops = 0;
    for (int c = tid; c < p.chunks; c += THREADS) {
        const LogprobPart q = part[c];
        before += q.before;
        if (q.max == m) {
            z += (double)q.z;
            tops += q.tops;
            s += (double)q.s;
        } else {
            const double t = scaled(q.max == -INFINITY ? m : q.max, m, rate), f = exp2(t), all = (double)q.z + (double)q.tops;
            z += all * f;
            s += ((double)q.s + all * t) * f;
        }
    }
    z = block_sum_f64(z, s_d);
    tops = block_sum_i(tops, s_i);
    z += (double)(tops - 1);  // Z - 1
    s = block_sum_f64(s, s_d);
    before = block_sum_i(before, s_i);
    const double ln2 = 0.6931471805599453, nan = __builtin_nan("");
    const bool greedy = rate < 0.0;
    const bool none = !(m > -INFINITY) || (!greedy && m == INFINITY);
    const double log_z = none ? nan : greedy ? 0.0 : log1p(z);
    if (tid == 0) {
        if (p.entropy) p.entropy[row] = (float)(none ? nan : greedy ? 0.0 : log_z - ln2 * s / (z + 1.0));
        if (p.tokens) {
            const int token = p.tokens[row];
            const bool inside = token >= 0 && token < p.vocab;
            const float x = inside ? logit(p, row, token) : -INFINITY;
            const int rank = inside && x == x ? 1 + before : 0;
            if (p.rank) p.rank[row] = rank;
            if (p.logprob)
                p.logprob[row] = (float)(none     ? nan
                                         : greedy ? (rank == 1 && x > -INFINITY ? 0.0 : -INFINITY)
                                                  : ln2 * scaled(x, m, rate) - log_z);
        }
    }
    if (p.top == 0) return;
    const int n = best_ids(p, row, s_list, s_best, s_i);
    if (tid < p.top) {
        const uint64_t at = (uint64_t)row * p.top + tid;
        const int id = tid < n ? (int)(uint32_t)~s_best[tid] : -1;
        if (p.top_ids) p.top_ids[at] = id;
        if (p.top_logprob) {
            double lp = -INFINITY;
            if (none) lp = nan;
            else if (greedy) lp = tid == 0 ? 0.0 : -INFINITY;
            else if (id >= 0) lp = ln2 * scaled(logit(p, row, id), m, rate) - log_z;
            else if (!(log_z == log_z)) lp = nan;
            p.top_logprob[at] = (float)lp;
        }
    }
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
