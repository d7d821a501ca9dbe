// Verification of drafted tokens against the target's probabilities.
//
// Three launches over rows of `vocab` logits, cut into chunks:
//   1 per (row, chunk): the largest logit (and where it is first), and the sum
//     of exp((x - largest) / T);
//   2 per (sequence, chunk): the row's M and Z from the chunks' states, which
//     drafts stand, and the chunk's part of the total weight of the row that
//     the next token comes from, max(0, p - q);
//   3 per sequence: the chunk in which the running sum passes u_next * total,
//     then the place in it; the results.
// Every logit is read once and one row of each sequence a second time (with
// the drafter's row), so memory bounds a batch, and launch latency a single
// sequence. Exponentials, sums and comparisons are fp64: a draft that is as
// good as its target leaves differences p - q far below p, and the running
// sums of 10^5 weights decide which id they pass at. The exponential is the
// Taylor polynomial of degree 10 on +-ln(2)/2 (next term 2.2e-13), times a
// power of two; it costs about as much time as the row's bytes do.
#include "paged.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256;

// 2^y; 0 below the normal numbers, NaN for NaN
__device__ __forceinline__ double exp2_d(double y)
{
    const double n = rint(y);
    const double z = (y - n) * 0.6931471805599453;
    double r = 1.0 / 3628800;
    r = fma(r, z, 1.0 / 362880);
    r = fma(r, z, 1.0 / 40320);
    r = fma(r, z, 1.0 / 5040);
    r = fma(r, z, 1.0 / 720);
    r = fma(r, z, 1.0 / 120);
    r = fma(r, z, 1.0 / 24);
    r = fma(r, z, 1.0 / 6);
    r = fma(r, z, 0.5);
    r = fma(r, z, 1.0);
    r = fma(r, z, 1.0);
    return y < -1000.0 ? 0.0 : ldexp(r, (int)n);
}

struct Rows {
    int a, n;  // n = 0: not within bounds, or empty
};
__device__ __forceinline__ Rows draft_rows(const DraftArgs& p, int s)
{
    const int a = p.q_start ? p.q_start[s] : s * p.max_rows;
    const int e = p.q_start ? p.q_start[s + 1] : a + p.max_rows;
    const bool ok = a >= 0 && a < e && e <= p.n_rows && e - a <= p.max_rows;
    return {a, ok ? e - a : 0};
}
__device__ __forceinline__ int draft_seq(const DraftArgs& p, int r)
{
    if (!p.q_start) return r / p.max_rows;
    int s = 0;
    for (int i = 0; i < p.n_seq; i += 64) {
        const int at = i + (int)(threadIdx.x & 63);
        s += __popcll(__ballot(at < p.n_seq && p.q_start[at < p.n_seq ? at + 1 : 0] <= r));
    }
    return s;
}
// log2(e) / T, or 0: greedy
__device__ __forceinline__ double draft_rate(const DraftArgs& p, int s)
{
    const float t = p.temperature ? p.temperature[s] : 1.0f;
    return t > 0.0f ? 1.4426950408889634 / (double)t : 0.0;
}

__device__ __forceinline__ double wave_sum_d(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}
// The sum of v over the threads before this one, and over all in total; four
// waves, s: four doubles.
__device__ __forceinline__ double block_before(double v, double* s, double& total)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    double t = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double u = __shfl_up(t, d);
        if (lane >= d) t += u;
    }
    double before = __shfl_up(t, 1);
    if (lane == 0) before = 0.0;
    if (lane == 63) s[wave] = t;
    __syncthreads();
    total = 0.0;
    double start = 0.0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w == wave) start = total;
        total += s[w];
    }
    __syncthreads();
    return start + before;
}
// (value, place) of the larger value, of the lower place where they are equal
__device__ __forceinline__ void larger(float& v, int& i, float w, int j)
{
    if (w > v || (w == v && j < i)) {
        v = w;
        i = j;
    }
}

__global__ __launch_bounds__(THREADS) void k_draft_stats(DraftArgs p)
{
    __shared__ float s_v[4];
    __shared__ int s_i[4];
    __shared__ double s_s[4];
    const int row = (int)(blockIdx.x / (unsigned)p.chunks), chunk = (int)(blockIdx.x % (unsigned)p.chunks);
    const int s = draft_seq(p, row);
    if (s >= p.n_seq) return;
    const Rows q = draft_rows(p, s);
    if (row < q.a || row >= q.a + q.n) return;
    const double rate = draft_rate(p, s);
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const float* x = p.logits + (uint64_t)row * p.logits_row;
    const int c0 = chunk * p.chunk, c1 = min(c0 + p.chunk, p.vocab);
    float best = -INFINITY;
    int at = 0x7fffffff;
    for (int i = c0 + (int)threadIdx.x; i < c1; i += THREADS) {
        const float v = x[i];
        if (v > best) {
            best = v;
            at = i;
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const float v = __shfl_xor(best, d);
        const int j = __shfl_xor(at, d);
        larger(best, at, v, j);
    }
    if (lane == 0) {
        s_v[wave] = best;
        s_i[wave] = at;
    }
    __syncthreads();
    best = s_v[0];
    at = s_i[0];
#pragma unroll
    for (int w = 1; w < 4; w++) larger(best, at, s_v[w], s_i[w]);
    double sum = 0.0;
    if (rate > 0.0) {
        const double base = best == -INFINITY ? 0.0 : (double)best;
        for (int i = c0 + (int)threadIdx.x; i < c1; i += THREADS) sum += exp2_d(((double)x[i] - base) * rate);
        sum = wave_sum_d(sum);
        if (lane == 0) s_s[wave] = sum;
        __syncthreads();
        sum = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
    }
    if (threadIdx.x == 0) p.part[(uint64_t)row * p.chunks + chunk] = DraftPart{sum, best, at};
}

// M and Z of a row (Z = sum of 2^((x - M) rate)), by a wave; at: the first
// largest logit
struct RowState {
    double z;
    float m;
    int at;
};
__device__ __forceinline__ RowState row_state(const DraftArgs& p, int row, double rate)
{
    const DraftPart* part = p.part + (uint64_t)row * p.chunks;
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int i = (int)threadIdx.x & 63; i < p.chunks; i += 64) larger(m, at, part[i].max, part[i].at);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const float v = __shfl_xor(m, d);
        const int j = __shfl_xor(at, d);
        larger(m, at, v, j);
    }
    double z = 0.0;
    for (int i = (int)threadIdx.x & 63; i < p.chunks; i += 64) {
        const float v = part[i].max;
        z += part[i].sum * (v == -INFINITY ? 1.0 : exp2_d(((double)v - (double)m) * rate));
    }
    return {wave_sum_d(z), m, at};
}

// The row that a sequence's next token comes from.
struct Choice {
    int accepted;
    RowState st;
    bool rest;  // weights max(0, p - q), else p
};
__device__ __forceinline__ Choice choose(const DraftArgs& p, int s, const Rows& q, double rate, RowState* s_st, int* s_ok)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    for (int i = wave; i < q.n; i += 4) {
        const RowState st = row_state(p, q.a + i, rate);
        int ok = 0;
        if (i + 1 < q.n) {
            const uint32_t d = p.tokens[q.a + i + 1];
            if (rate == 0.0) {
                ok = st.m > -INFINITY && d == (uint32_t)st.at;
            } else if (d < (uint32_t)p.vocab) {
                const uint64_t r = (uint64_t)(q.a + i);
                const double e = exp2_d(((double)p.logits[r * p.logits_row + d] - (double)st.m) * rate);
                const double w = p.probs ? (double)p.probs[r * p.probs_row + d] : 1.0;
                ok = (double)p.u[q.a + i] * w < e / st.z;
            }
        }
        if (lane == 0) {
            s_st[i] = st;
            s_ok[i] = ok;
        }
    }
    __syncthreads();
    Choice c;
    c.accepted = 0;
    while (c.accepted + 1 < q.n && s_ok[c.accepted]) c.accepted++;
    c.st = s_st[c.accepted];
    c.rest = c.accepted + 1 < q.n;
    return c;
}

// Z times the weight of id i in row r
__device__ __forceinline__ double weight(const DraftArgs& p, int r, int i, const Choice& c, double rate, bool rest, int draft)
{
    const double e = exp2_d(((double)p.logits[(uint64_t)r * p.logits_row + i] - (double)c.st.m) * rate);
    if (!rest) return e;
    const double q = p.probs ? (double)p.probs[(uint64_t)r * p.probs_row + i] : i == draft ? 1.0 : 0.0;
    const double w = e - q * c.st.z;
    return w > 0.0 ? w : w != w ? w : 0.0;
}

__global__ __launch_bounds__(THREADS) void k_draft_rest(DraftArgs p)
{
    __shared__ RowState s_st[WPCG_DRAFT_MAX];
    __shared__ int s_ok[WPCG_DRAFT_MAX];
    __shared__ double s_s[4];
    const int s = (int)(blockIdx.x / (unsigned)p.chunks), chunk = (int)(blockIdx.x % (unsigned)p.chunks);
    const Rows q = draft_rows(p, s);
    if (q.n == 0) return;
    const double rate = draft_rate(p, s);
    const Choice c = choose(p, s, q, rate, s_st, s_ok);
    if (chunk == 0 && threadIdx.x == 0) p.choice[s] = DraftChoice{c.st.z, c.st.m, c.st.at, c.accepted, 0};
    if (rate == 0.0 || !c.rest) return;
    const int row = q.a + c.accepted, draft = (int)p.tokens[row + 1];
    const int c0 = chunk * p.chunk, c1 = min(c0 + p.chunk, p.vocab);
    double sum = 0.0;
    for (int i = c0 + (int)threadIdx.x; i < c1; i += THREADS) sum += weight(p, row, i, c, rate, true, draft);
    sum = wave_sum_d(sum);
    if ((threadIdx.x & 63) == 0) s_s[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) p.rest[(uint64_t)s * p.chunks + chunk] = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
}

__global__ __launch_bounds__(THREADS) void k_draft_pick(DraftArgs p)
{
    __shared__ double s_s[4], s_before;
    __shared__ int s_at, s_id, s_last, s_last_id;
    const int s = (int)blockIdx.x, tid = (int)threadIdx.x;
    const Rows q = draft_rows(p, s);
    if (q.n == 0) {
        if (tid == 0) p.accepted[s] = -1;
        return;
    }
    const double rate = draft_rate(p, s);
    const DraftChoice dc = p.choice[s];
    Choice c;
    c.accepted = dc.accepted;
    c.st = {dc.z, dc.m, dc.at};
    const int row = q.a + c.accepted;
    bool rest = c.accepted + 1 < q.n;
    const int draft = rest ? (int)p.tokens[row + 1] : -1;
    int token = -1;
    if (rate == 0.0) {
        token = dc.m > -INFINITY ? dc.at : -1;
    } else if (dc.z > 0.0 && dc.z < INFINITY) {
        // the chunks' weights: those of the rest, or the row's own
        const auto of_chunk = [&](int i) {
            if (rest) return p.rest[(uint64_t)s * p.chunks + i];
            const DraftPart& part = p.part[(uint64_t)row * p.chunks + i];
            return part.max == -INFINITY ? 0.0 : part.sum * exp2_d(((double)part.max - (double)dc.m) * rate);
        };
        // a thread's run of chunks
        const int run = (p.chunks + THREADS - 1) / THREADS;
        const int j0 = min(tid * run, p.chunks), j1 = min(j0 + run, p.chunks);
        double before, total;
        for (int turn = 0; turn < 2; turn++) {
            double sum = 0.0;
            for (int i = j0; i < j1; i++) sum += of_chunk(i);
            before = block_before(sum, s_s, total);
            if (total > 0.0 || !rest) break;
            rest = false;  // nothing is left of p - q: the row's own weights
        }
        const double want = (double)p.u_next[s] * total;
        if (tid == 0) {
            s_at = s_id = 0x7fffffff;
            s_last = s_last_id = -1;
        }
        __syncthreads();
        for (int i = j0; i < j1; i++) {
            const double w = of_chunk(i);
            if (w > 0.0) atomicMax(&s_last, i);  // of use where rounding leaves none
            if (before + w > want) {
                atomicMin(&s_at, i);
                break;
            }
            before += w;
        }
        __syncthreads();
        const int chunk = s_at != 0x7fffffff ? s_at : s_last;
        if (chunk >= 0) {
            if (tid == chunk / run) {
                // this thread stopped at the chunk, or went past its run's end
                if (s_at == 0x7fffffff) before = INFINITY;  // the last id with weight
                s_before = before;
            }
            __syncthreads();
            // the same over the chunk's ids
            const int c0 = chunk * p.chunk, c1 = min(c0 + p.chunk, p.vocab);
            const int ids = (c1 - c0 + THREADS - 1) / THREADS;
            const int i0 = min(c0 + tid * ids, c1), i1 = min(i0 + ids, c1);
            double sum = 0.0, all;
            for (int i = i0; i < i1; i++) sum += weight(p, row, i, c, rate, rest, draft);
            const bool end = s_before == INFINITY;
            double t = s_before + block_before(sum, s_s, all);
            for (int i = i0; i < i1; i++) {
                const double w = weight(p, row, i, c, rate, rest, draft);
                if (w > 0.0) atomicMax(&s_last_id, i);
                t += w;
                if (!end && t > want) {
                    atomicMin(&s_id, i);
                    break;
                }
            }
            __syncthreads();
            token = s_id != 0x7fffffff ? s_id : s_last_id;
        }
    }
    for (int i = tid; i < q.n; i += THREADS)
        p.out[q.a + i] = i < c.accepted ? (int)p.tokens[q.a + i + 1] : i == c.accepted ? token : -1;
    if (tid == 0) p.accepted[s] = c.accepted;
}

}  // namespace

hipError_t launch_draft_verify(const DraftArgs& p, hipStream_t s)
{
    if (p.n_seq == 0) return hipSuccess;
    if (p.n_rows > 0) {
        k_draft_stats<<<dim3((unsigned)((uint64_t)p.n_rows * p.chunks)), dim3(THREADS), 0, s>>>(p);
        k_draft_rest<<<dim3((unsigned)((uint64_t)p.n_seq * p.chunks)), dim3(THREADS), 0, s>>>(p);
    }
    k_draft_pick<<<dim3((unsigned)p.n_seq), dim3(THREADS), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace wpcg
