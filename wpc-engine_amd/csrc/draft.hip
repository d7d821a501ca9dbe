// Verification of drafted tokens against the target's probabilities.
//
// Two launches over rows of `vocab` logits, cut into chunks of 2048 ids, a
// wave each:
//   1 per (row, chunk): the largest logit (greedy rows: and where it is
//     first), and the sum of exp((x - largest) / T), the chunk in registers;
//   2 per (sequence, four chunks): M and Z of the sequence's rows from the
//     chunks' states, which drafts stand, and the chunks' parts of the total
//     weight of the row that the next token comes from, max(0, p - q). The
//     sequence's last workgroup to finish finds the chunk in which the running
//     sum passes u_next * total, then the place in it, and writes the results;
//     the first launch has set the counter that it is known by.
// Every logit is read once and one row of each sequence a second time (with
// the drafter's row), so memory bounds a batch, and launch latency a single
// sequence. Exponentials, sums and comparisons are fp64: a draft that is as
// good as its target leaves differences p - q far below p, and the running
// sums of 10^5 weights decide which id they pass at. The exponential is the
// Taylor polynomial of degree 10 on +-ln(2)/2 (next term 2.2e-13), times a
// power of two.
#include "paged.h"
#include "wave.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256, CHUNK = DRAFT_CHUNK;
static_assert(CHUNK == 8 * THREADS, "pick: eight ids a thread");

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

// A chunk's values of a row in registers: lane l holds ids 4 l + 256 i + 0..3
// of it, -inf behind the row's end. vec: the row starts on 16 bytes.
struct Chunk {
    float v[CHUNK / 64];
    __device__ __forceinline__ void load(const float* x, int c0, int vocab, bool vec, float none)
    {
        const int lane = (int)threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < CHUNK / 256; i++) {
            const int at = c0 + 256 * i + 4 * lane;
            if (vec && at + 4 <= vocab) {
                const pf32x4 w = *(const pf32x4*)(x + at);
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = at + j < vocab ? x[at + j] : none;
            }
        }
    }
};

__global__ __launch_bounds__(THREADS) void k_draft_stats(DraftArgs p)
{
    const int groups = (p.chunks + 3) / 4;
    const int row = (int)(blockIdx.x / (unsigned)groups);
    const int chunk = (int)(blockIdx.x % (unsigned)groups) * 4 + ((int)threadIdx.x >> 6);
    const int lane = (int)threadIdx.x & 63;
    const int s = draft_seq(p, row);
    if (s >= p.n_seq) return;
    const Rows q = draft_rows(p, s);
    if (row < q.a || row >= q.a + q.n) return;
    if (row == q.a && chunk == 0 && lane == 0) p.done[s].done = 0;
    if (chunk >= p.chunks) return;
    const double rate = draft_rate(p, s);
    const float* x = p.logits + (uint64_t)row * p.logits_row;
    Chunk c;
    c.load(x, chunk * CHUNK, p.vocab, p.vec, -INFINITY);
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < CHUNK / 64; i++) best = fmaxf(best, c.v[i]);
    best = wave_max(best);
    int at = 0x7fffffff;
    double sum = 0.0;
    if (rate > 0.0) {
        const double base = best == -INFINITY ? 0.0 : (double)best;
#pragma unroll
        for (int i = 0; i < CHUNK / 64; i++) sum += exp2_d(((double)c.v[i] - base) * rate);
        sum = wave_sum_d(sum);
    } else {
#pragma unroll
        for (int i = CHUNK / 64 - 1; i >= 0; i--)
            if (c.v[i] == best) at = chunk * CHUNK + 256 * (i / 4) + 4 * lane + i % 4;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) at = min(at, __shfl_xor(at, d));
    }
    if (lane == 0) p.part[(uint64_t)row * p.chunks + chunk] = DraftPart{sum, best, best == -INFINITY ? 0x7fffffff : at};
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

// Z times an id's weight in the row, from its logit x and the drafter's q
__device__ __forceinline__ double weight(float x, float q, const RowState& st, double rate, bool rest)
{
    const double e = exp2_d(((double)x - (double)st.m) * rate);
    if (!rest) return e;
    const double w = e - (double)q * st.z;
    return w > 0.0 || w != w ? w : 0.0;
}

// The drafter's q for a lane's ids of a chunk, as Chunk has them.
__device__ __forceinline__ void draft_chunk(Chunk& q, const DraftArgs& p, int row, int chunk, int draft)
{
    if (p.probs) {
        q.load(p.probs + (uint64_t)row * p.probs_row, chunk * CHUNK, p.vocab, p.vec, 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK / 64; i++)
            q.v[i] = chunk * CHUNK + 256 * (i / 4) + 4 * ((int)threadIdx.x & 63) + i % 4 == draft ? 1.0f : 0.0f;
    }
}

// The token of a sampled row: its chunks' weights, then the chunk's ids.
__device__ int pick(const DraftArgs& p, int s, int row, const Choice& c, double rate, int draft)
{
    __shared__ double s_s[4], s_before;
    __shared__ int s_at, s_id, s_last, s_last_id;
    const int tid = (int)threadIdx.x;
    bool rest = c.rest;
    const auto of_chunk = [&](int i) {
        if (rest) return __hip_atomic_load(&p.rest[(uint64_t)s * p.chunks + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const DraftPart& part = p.part[(uint64_t)row * p.chunks + i];
        return part.max == -INFINITY ? 0.0 : part.sum * exp2_d(((double)part.max - (double)c.st.m) * rate);
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
    if (chunk < 0) return -1;
    const bool end = s_at == 0x7fffffff;  // the last id with weight
    if (tid == chunk / run) s_before = before;  // stopped at the chunk
    // ids 8 t .. 8 t + 7 of the chunk
    const int i0 = chunk * CHUNK + 8 * tid;
    double w[8], sum = 0.0, all;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = i0 + j;
        w[j] = 0.0;
        if (i < p.vocab) {
            const float q = p.probs ? (rest ? p.probs[(uint64_t)row * p.probs_row + i] : 0.0f) : i == draft ? 1.0f : 0.0f;
            w[j] = weight(p.logits[(uint64_t)row * p.logits_row + i], q, c.st, rate, rest);
        }
        sum += w[j];
    }
    double t = block_before(sum, s_s, all);
    t += s_before;
    int first = 0x7fffffff, last = -1;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        t += w[j];
        if (w[j] > 0.0) last = i0 + j;
        if (!end && t > want && first == 0x7fffffff) first = i0 + j;
    }
    if (first != 0x7fffffff) atomicMin(&s_id, first);
    if (last >= 0) atomicMax(&s_last_id, last);
    __syncthreads();
    return s_id != 0x7fffffff ? s_id : s_last_id;
}

__global__ __launch_bounds__(THREADS) void k_draft_choose(DraftArgs p)
{
    __shared__ RowState s_st[WPCG_DRAFT_MAX];
    __shared__ int s_ok[WPCG_DRAFT_MAX];
    __shared__ int s_done;
    const int groups = (p.chunks + 3) / 4;
    const int s = (int)(blockIdx.x / (unsigned)groups), group = (int)(blockIdx.x % (unsigned)groups);
    const int tid = (int)threadIdx.x;
    const Rows q = draft_rows(p, s);
    if (q.n == 0) {
        if (group == 0 && tid == 0) p.accepted[s] = -1;
        return;
    }
    const double rate = draft_rate(p, s);
    const Choice c = choose(p, s, q, rate, s_st, s_ok);
    const int row = q.a + c.accepted, draft = c.rest ? (int)p.tokens[row + 1] : -1;
    int token = -1;
    if (rate == 0.0) {
        if (group != 0) return;
        token = c.st.m > -INFINITY ? c.st.at : -1;
    } else if (!(c.st.z > 0.0 && c.st.z < INFINITY)) {
        if (group != 0) return;
    } else {
        if (c.rest) {
            const int chunk = group * 4 + (tid >> 6);
            if (chunk < p.chunks) {
                Chunk x, r;
                x.load(p.logits + (uint64_t)row * p.logits_row, chunk * CHUNK, p.vocab, p.vec, -INFINITY);
                draft_chunk(r, p, row, chunk, draft);
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < CHUNK / 64; i++) sum += weight(x.v[i], r.v[i], c.st, rate, true);
                sum = wave_sum_d(sum);
                if ((tid & 63) == 0)
                    __hip_atomic_store(&p.rest[(uint64_t)s * p.chunks + chunk], sum, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
            }
            // the last of the sequence's workgroups goes on
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                s_done = __hip_atomic_fetch_add(&p.done[s].done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (s_done != groups - 1) return;
        } else if (group != 0) {
            return;
        }
        token = pick(p, s, row, c, rate, draft);
    }
    for (int i = tid; i < q.n; i += THREADS)
        p.out[q.a + i] = i < c.accepted ? (int)p.tokens[q.a + i + 1] : i == c.accepted ? token : -1;
    if (tid == 0) p.accepted[s] = c.accepted;
}

}  // namespace

hipError_t launch_draft_verify(const DraftArgs& p, hipStream_t s)
{
    if (p.n_seq == 0) return hipSuccess;
    const unsigned groups = (unsigned)(p.chunks + 3) / 4;
    if (p.n_rows > 0) k_draft_stats<<<dim3((unsigned)p.n_rows * groups), dim3(THREADS), 0, s>>>(p);
    k_draft_choose<<<dim3((unsigned)p.n_seq * groups), dim3(THREADS), 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace wpcg
