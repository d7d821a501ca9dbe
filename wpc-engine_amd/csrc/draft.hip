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
//     the first launch has set the counter that it is known by, and the parts
//     to a mark that is none: a part is one atomic word, so that whoever reads
//     another value has all of it, and no order between words is needed. (A
//     release of the count writes the L2 back for every workgroup: 64 sequences
//     68 and 102 us.)
// Every logit is read once and one row of each sequence a second time (with
// the drafter's row), so memory bounds a batch, and launch latency a single
// sequence. Exponentials, sums and comparisons are fp64: a draft that is as
// good as its target leaves differences p - q far below p, and the running
// sums of 10^5 weights decide which id they pass at.
//
// Measured at 151936 ids, on four cards: 64 sequences with their drafts (260 MB)
// 63 to 72 us, the first launch 44 (5.2 TB/s) and the second 23; one sequence
// with four drafts 12.3 to 14.7 us, 4.1 and 10.4 of them. (With LDS atomics in
// place of the ballots that find the drawn id 5 us more: 75 threads at one word
// took 2 to 3 us each time.)
#include "paged.h"
#include "wave.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256, CHUNK = DRAFT_CHUNK;
static_assert(CHUNK == 8 * THREADS, "pick: eight ids a thread");
// In `rest` until the chunk's sum is there, which is not negative. Who waits for
// it has seen its workgroup's count, so that the store is on its way.
constexpr double NO_SUM = -1.0;

// 2^(x rate) for x <= 0 (or NaN), a difference of two logits: x rate = n + f, n
// the whole number that adding 1.5 * 2^52 leaves in the low bits, the
// polynomial of degree 8 through 2^f at the nine Chebyshev points of +-1/2
// (within 1.1e-12 of it there), n added to its exponent. 0 below 2^-1000.
__device__ __forceinline__ double exp2_d(double x, double rate)
{
    const double t = fma(x, rate, 6755399441055744.0);
    const double whole = t - 6755399441055744.0;
    const double f = fma(x, rate, -whole);
    double r = 1.3255224878668817e-06;
    r = fma(r, f, 1.5310079402249296e-05);
    r = fma(r, f, 0.00015403455852453838);
    r = fma(r, f, 0.0013333450568000645);
    r = fma(r, f, 0.009618129159402558);
    r = fma(r, f, 0.05550410941205933);
    r = fma(r, f, 0.2402265069581299);
    r = fma(r, f, 0.6931471805459335);
    r = fma(r, f, 1.0);
    const uint64_t n = (uint64_t)(uint32_t)__builtin_bit_cast(uint64_t, t) << 52;
    r = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, r) + n);
    return whole < -1000.0 ? 0.0 : r;
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
// log2(e) / T, or 0: greedy. For an infinite T 2^-1000: a difference of finite
// logits times that is nothing beside 1, and one to -inf stays -inf.
__device__ __forceinline__ double draft_rate(const DraftArgs& p, int s)
{
    const float t = p.temperature ? p.temperature[s] : 1.0f;
    return t > 0.0f ? fmax(1.4426950408889634 / (double)t, 0x1p-1000) : 0.0;
}

// Lane exchanges of doubles: 0 from lanes that there are none.
constexpr int DPP_ROW_SHR = 0x110, DPP_WAVE_SHR1 = 0x138;  // from n lanes before, in a row of 16; of the wave
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ double dpp_d(double v)
{
    const uint64_t w = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)wave_dpp_i<CTRL, ROW_MASK>(0, (int)(uint32_t)w);
    const uint32_t hi = (uint32_t)wave_dpp_i<CTRL, ROW_MASK>(0, (int)(w >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_d(double v, int lane)
{
    const uint64_t w = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Every lane: the sum over its row of 16 lanes.
__device__ __forceinline__ double row_sum_d(double v)
{
    v += dpp_d<WDPP_XOR1>(v);
    v += dpp_d<WDPP_XOR2>(v);
    v += dpp_d<WDPP_HALF_MIRROR>(v);
    return v + dpp_d<WDPP_MIRROR>(v);
}
__device__ __forceinline__ double wave_sum_d(double v)
{
    v = row_sum_d(v);
    v += dpp_d<WDPP_BCAST15, 0xA>(v);
    v += dpp_d<WDPP_BCAST31, 0xC>(v);
    return lane_d(v, 63);
}
// The sums over the lanes up to this one.
__device__ __forceinline__ double wave_scan_d(double v)
{
    v += dpp_d<DPP_ROW_SHR + 1>(v);
    v += dpp_d<DPP_ROW_SHR + 2>(v);
    v += dpp_d<DPP_ROW_SHR + 4>(v);
    v += dpp_d<DPP_ROW_SHR + 8>(v);
    v += dpp_d<WDPP_BCAST15, 0xA>(v);
    return v + dpp_d<WDPP_BCAST31, 0xC>(v);
}
// The sum of v over the threads before this one, and over all in total; four
// waves, s: four doubles.
__device__ __forceinline__ double block_before(double v, double* s, double& total)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const double t = wave_scan_d(v), before = dpp_d<DPP_WAVE_SHR1>(t);
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
        // one way for the whole wave, and no load behind a condition: a lane
        // that skips one would have to wait for those before it
        if (vec && c0 + CHUNK <= vocab) {
#pragma unroll
            for (int i = 0; i < CHUNK / 256; i++) {
                const pf32x4 w = *(const pf32x4*)(x + c0 + 256 * i + 4 * lane);
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < CHUNK / 64; i++) v[i] = x[min(c0 + 256 * (i / 4) + 4 * lane + i % 4, vocab - 1)];
#pragma unroll
            for (int i = 0; i < CHUNK / 64; i++)
                if (c0 + 256 * (i / 4) + 4 * lane + i % 4 >= vocab) v[i] = none;
        }
    }
};

// A chunk's state of a row, by a wave.
__device__ __forceinline__ void chunk_state(const DraftArgs& p, int row, int chunk)
{
    const int lane = (int)threadIdx.x & 63;
    // the values are on their way while the row's sequence is looked for
    Chunk c;
    c.load(p.logits + (uint64_t)row * p.logits_row, chunk * CHUNK, p.vocab, p.vec, -INFINITY);
    const int s = p.q_start ? seq_of_row(p.q_start, p.n_seq, row) : row / p.max_rows;
    if (s >= p.n_seq) return;
    const Rows q = draft_rows(p, s);
    if (row < q.a || row >= q.a + q.n) return;
    const double rate = draft_rate(p, s);
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < CHUNK / 64; i++) best = fmaxf(best, c.v[i]);
    best = wave_max(best);
    int at = 0x7fffffff;
    double sum = 0.0;
    if (rate > 0.0) {
        const double base = best == -INFINITY ? 0.0 : (double)best;
#pragma unroll
        for (int i = 0; i < CHUNK / 64; i++) sum += exp2_d((double)c.v[i] - base, rate);
        sum = wave_sum_d(sum);
    } else {
#pragma unroll
        for (int i = CHUNK / 64 - 1; i >= 0; i--)
            if (c.v[i] == best) at = chunk * CHUNK + 256 * (i / 4) + 4 * lane + i % 4;
        at = ~wave_max_i(~at);
    }
    if (lane == 0) p.part[(uint64_t)row * p.chunks + chunk] = DraftPart{sum, best, best == -INFINITY ? 0x7fffffff : at};
}

__global__ __launch_bounds__(THREADS) void k_draft_stats(DraftArgs p)
{
    const int groups = (p.chunks + 3) / 4;
    const int row = (int)(blockIdx.x / (unsigned)groups);
    const int chunk = (int)(blockIdx.x % (unsigned)groups) * 4 + ((int)threadIdx.x >> 6);
    if (chunk >= p.chunks) return;
    chunk_state(p, row, chunk);
    // The second launch's arrays made ready, of sequences without rows too. (At
    // the end: behind these stores the loads above would not be scalar ones, and
    // wait for the logits: 64 sequences 44 and 52 us.)
    if ((threadIdx.x & 63) == 0) {
        for (int s = row; s < p.n_seq; s += p.n_rows) {
            p.rest[(uint64_t)s * p.chunks + chunk] = NO_SUM;
            if (chunk == 0) p.done[s].done = 0;
        }
    }
}

// M and Z of a row (Z = sum of 2^((x - M) rate)), by 32 lanes; at: the first
// largest logit (greedy)
struct RowState {
    double z;
    float m;
    int at;
};
__device__ __forceinline__ RowState row_state(const DraftArgs& p, int row, double rate)
{
    constexpr int AHEAD = 4;  // states in flight
    const DraftPart* part = p.part + (uint64_t)row * p.chunks;
    const int l = (int)threadIdx.x & 31;
    float m = -INFINITY;
    int at = 0x7fffffff;
    double z = 0.0;
    for (int i0 = l; i0 < p.chunks; i0 += 32 * AHEAD) {
        DraftPart c[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) c[j] = part[min(i0 + 32 * j, p.chunks - 1)];
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
            if (i0 + 32 * j >= p.chunks) c[j] = DraftPart{0.0, -INFINITY, 0x7fffffff};
        const float old = m;
#pragma unroll
        for (int j = 0; j < AHEAD; j++) larger(m, at, c[j].max, c[j].at);
        const auto to_m = [&](float v) { return v == -INFINITY ? 1.0 : exp2_d((double)v - (double)m, rate); };
        z *= to_m(old);
#pragma unroll
        for (int j = 0; j < AHEAD; j++) z += c[j].sum * to_m(c[j].max);
    }
    const float mine = m;
    larger(m, at, wave_dpp<WDPP_XOR1>(m, m), wave_dpp_i<WDPP_XOR1>(at, at));
    larger(m, at, wave_dpp<WDPP_XOR2>(m, m), wave_dpp_i<WDPP_XOR2>(at, at));
    larger(m, at, wave_dpp<WDPP_HALF_MIRROR>(m, m), wave_dpp_i<WDPP_HALF_MIRROR>(at, at));
    larger(m, at, wave_dpp<WDPP_MIRROR>(m, m), wave_dpp_i<WDPP_MIRROR>(at, at));
    // the rows of a half wave
    const auto ms = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    const auto as = __builtin_amdgcn_permlane16_swap((uint32_t)at, (uint32_t)at, false, false);
    m = __uint_as_float(ms[0]);
    at = (int)as[0];
    larger(m, at, __uint_as_float(ms[1]), (int)as[1]);
    z *= mine == -INFINITY ? 1.0 : exp2_d((double)mine - (double)m, rate);
    z = row_sum_d(z);
    const uint64_t w = __builtin_bit_cast(uint64_t, z);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)w, (uint32_t)w, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(w >> 32), (uint32_t)(w >> 32), false, false);
    z = __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
        __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
    return {z, m, at};
}

// The row that a sequence's next token comes from.
struct Choice {
    int accepted;
    RowState st;
    bool rest;  // weights max(0, p - q), else p
};
__device__ __forceinline__ Choice choose(const DraftArgs& p, int s, const Rows& q, double rate, RowState* s_st, int* s_ok)
{
    // half a wave a row, so that the first eight rows' loads go out together
    for (int i = (int)threadIdx.x / 32; i < q.n; i += THREADS / 32) {
        const uint64_t r = (uint64_t)(q.a + i);
        const bool drafted = i + 1 < q.n;
        const uint32_t d = p.tokens[drafted ? r + 1 : r];
        const float u = drafted ? p.u[r] : 0.0f;
        const bool inside = drafted && d < (uint32_t)p.vocab;
        const uint64_t at = inside ? d : 0;
        const float x = p.logits[r * p.logits_row + at];
        const float w = p.probs && drafted ? p.probs[r * p.probs_row + at] : 1.0f;
        const RowState st = row_state(p, (int)r, rate);
        int ok = 0;
        if (rate == 0.0) ok = drafted && st.m > -INFINITY && d == (uint32_t)st.at;
        else if (inside) ok = (double)u * (double)w < exp2_d((double)x - (double)st.m, rate) / st.z;
        if ((threadIdx.x & 31) == 0) {
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
    const double e = exp2_d((double)x - (double)st.m, rate);
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

// The first thread that found something: its number and running sum; and the
// last thread's that has some weight. Numbers rise with the threads; MISSING or
// -1 where there is none. s: of four waves. A thread's running sum starts from
// the scan and ends in its own order, so that the next one's start may be past
// the mark where its end is not: only what has weight itself is found.
constexpr int MISSING = 0x7fffffff;
struct Found {
    int at, last;
    double before;
};
__device__ __forceinline__ Found find_first(bool found, int at, double before, int last, Found* s)
{
    const uint64_t f = __ballot(found), w = __ballot(last >= 0);
    Found r = {MISSING, -1, 0.0};
    if (f) {
        const int l = __builtin_ctzll(f);
        r.at = __builtin_amdgcn_readlane(at, l);
        r.before = lane_d(before, l);
    }
    if (w) r.last = __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(w));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = r;
    __syncthreads();
    r = s[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; i++) {
        if (r.at == MISSING) {
            r.at = s[i].at;
            r.before = s[i].before;
        }
        r.last = max(r.last, s[i].last);
    }
    return r;
}
// Eight consecutive values of a row, i0 a multiple of 8; behind its end the last.
__device__ __forceinline__ void load_eight(float (&v)[8], const float* x, int i0, int vocab, bool vec)
{
    if (vec && i0 + 8 <= vocab) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const pf32x4 w = *(const pf32x4*)(x + i0 + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; j++) v[4 * i + j] = w[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = x[min(i0 + j, vocab - 1)];
    }
}

// The token of a sampled row: its chunks' weights, then the chunk's ids.
__device__ int pick(const DraftArgs& p, int s, int row, const Choice& c, double rate, int draft)
{
    __shared__ double s_s[4];
    __shared__ Found s_chunk[4], s_id[4];
    const int tid = (int)threadIdx.x;
    const double u = (double)p.u_next[s];
    bool rest = c.rest;
    const auto of_chunk = [&](int i) {
        if (rest) {
            double w;
            do w = __hip_atomic_load(&p.rest[(uint64_t)s * p.chunks + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            while (w == NO_SUM);
            return w;
        }
        const DraftPart& part = p.part[(uint64_t)row * p.chunks + i];
        return part.max == -INFINITY ? 0.0 : part.sum * exp2_d((double)part.max - (double)c.st.m, rate);
    };
    // a thread's run of chunks
    const int run = (p.chunks + THREADS - 1) / THREADS;
    const int j0 = min(tid * run, p.chunks), j1 = min(j0 + run, p.chunks);
    double before, total, only = 0.0;
    for (int turn = 0; turn < 2; turn++) {
        double sum = 0.0;
        for (int i = j0; i < j1; i++) sum += only = of_chunk(i);
        before = block_before(sum, s_s, total);
        if (total > 0.0 || !rest) break;
        rest = false;  // nothing is left of p - q: the row's own weights
    }
    const double want = u * total;
    int at = MISSING, last = -1;  // last: of use where rounding leaves none
    for (int i = j0; i < j1; i++) {
        const double w = run == 1 ? only : of_chunk(i);
        if (w > 0.0) {
            last = i;
            if (before + w > want) {
                at = i;
                break;
            }
        }
        before += w;
    }
    const Found f = find_first(at != MISSING, at, before, last, s_chunk);
    const bool end = f.at == MISSING;  // the last id with weight
    const int chunk = end ? f.last : f.at;
    if (chunk < 0) return -1;
    // ids 8 t .. 8 t + 7 of the chunk
    const int i0 = chunk * CHUNK + 8 * tid;
    double w[8], sum = 0.0, all;
    float x[8], q[8] = {};
    load_eight(x, p.logits + (uint64_t)row * p.logits_row, i0, p.vocab, p.vec);
    if (p.probs && rest) load_eight(q, p.probs + (uint64_t)row * p.probs_row, i0, p.vocab, p.vec);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (!p.probs && i0 + j == draft) q[j] = 1.0f;
        w[j] = i0 + j < p.vocab ? weight(x[j], q[j], c.st, rate, rest) : 0.0;
        sum += w[j];
    }
    double t = block_before(sum, s_s, all);
    t += f.before;
    int first = MISSING, final = -1;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        t += w[j];
        if (w[j] > 0.0) {
            final = i0 + j;
            if (!end && t > want && first == MISSING) first = i0 + j;
        }
    }
    const Found id = find_first(first != MISSING, first, 0.0, final, s_id);
    return id.at != MISSING ? id.at : id.last;
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
    const int shown = tid < c.accepted ? (int)p.tokens[q.a + tid + 1] : -1;  // at most 64 rows
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
            if (tid == 0)
                s_done = __hip_atomic_fetch_add(&p.done[s].done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (s_done != groups - 1) return;
        } else if (group != 0) {
            return;
        }
        token = pick(p, s, row, c, rate, draft);
    }
    if (tid < q.n) p.out[q.a + tid] = tid == c.accepted ? token : shown;
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
