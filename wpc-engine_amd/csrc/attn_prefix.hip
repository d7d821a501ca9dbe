// Attention of few rows a sequence in a batch whose sequences come in groups that
// share their first tokens: several answers to one prompt, beams, questions about
// one document.
//
// The softmax over prefix and own tokens is put together from its parts:
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// The prefix of a group is read once for the rows of all its sequences, whose
// (row, query head) pairs are the columns of the many-row kernel's workgroups
// (attn_many.h): what the memory bounds one sequence at a time, the matrix cores
// do for many. Own tokens go through the few-row kernel (attn_few.h). Both leave
// parts, which a last launch joins.
#include "attn_few.h"
#include "attn_many.h"

namespace wpcg {
namespace {

// Group g: sequences s0 .. s0 + n - 1, rows a .. a + rows - 1, and how many tokens
// they share; len = 0: it shares nothing (it has one sequence or none, or its
// numbers are out of bounds).
struct Group {
    int s0, n, a, rows, len;
};
__device__ __forceinline__ Group group_of(const PrefixArgs& p, int g)
{
    const PagedBatch& b = p.a.b;
    Group r;
    r.s0 = p.group_start[g];
    const int s1 = p.group_start[g + 1];
    const bool some = r.s0 >= 0 && r.s0 <= s1 - 2 && s1 <= b.n_seq;
    r.n = some ? s1 - r.s0 : 0;
    const int s = some ? r.s0 : 0, e = some ? s1 : 0;
    r.a = b.q_start ? b.q_start[s] : s;
    const int end = b.q_start ? b.q_start[e] : e;
    const bool rows = some && r.a >= 0 && r.a <= end && end <= b.n_rows;
    // the pages are those of the first sequence, which has no more than its own
    const int len = b.kv_len[s];
    r.len = rows && len <= b.max_kv ? max(0, min(min(p.prefix_len[g], p.max_prefix), len)) : 0;
    r.rows = r.len > 0 ? end - r.a : 0;
    return r;
}
// How many first tokens sequence s shares: a binary search for its group.
__device__ __forceinline__ int shared_by(const PrefixArgs& p, int s, Group* group = nullptr)
{
    int lo = 0, hi = p.n_groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (p.group_start[mid] <= s) lo = mid;
        else hi = mid - 1;
    }
    const Group g = group_of(p, lo);
    if (group) *group = g;
    return s >= g.s0 && s < g.s0 + g.n ? g.len : 0;
}
// The position of a group's row, -1 if it is no sequence's.
__device__ __forceinline__ int row_position(const PagedBatch& b, const Group& g, int row)
{
    int lo = g.s0, hi = g.s0 + g.n - 1;
    if (!b.q_start) lo = row;
    while (b.q_start && lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (b.q_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    const SeqRows r = seq_rows(b, lo);
    return r.bad || row < r.a || row >= r.a + r.n ? -1 : r.len - r.n + (row - r.a);
}

// ---- prefixes ------------------------------------------------------------------
constexpr int PRE_COLS = ATTN_MANY_COLS;

// A workgroup's 128 columns of a group's rows over a chunk of its prefix.
struct PrefixWork {
    const PrefixArgs& args;
    Group g;
    SeqRows sq;  // the group's rows
    int seq, kvh, cb, split, v0, v1;
    int least, most;  // its rows' positions
    SeenTiles<many::TILE> seen;
    __device__ __forceinline__ explicit PrefixWork(const PrefixArgs& p) : args(p) {}
    __device__ __forceinline__ bool find()
    {
        const PagedAttnArgs& p = args.a;
        const int lane = (int)threadIdx.x & 63;
        kvh = (int)(blockIdx.x % (unsigned)p.n_kv);
        const int rest = (int)(blockIdx.x / (unsigned)p.n_kv);
        split = rest % args.splits;
        int at = rest / args.splits, which = -1;
        // column block `at` of all groups' ones, laid end to end
        for (int g0 = 0; g0 < args.n_groups; g0 += 64) {
            int t = g0 + lane < args.n_groups ? (group_of(args, g0 + lane).rows * p.group + PRE_COLS - 1) / PRE_COLS : 0;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int u = __shfl_up(t, d);
                if (lane >= d) t += u;
            }
            const uint64_t behind = __ballot(t > at);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                which = g0 + l;
                cb = at - (l > 0 ? __builtin_amdgcn_readlane(t, max(0, l - 1)) : 0);
                break;
            }
            at -= __builtin_amdgcn_readlane(t, 63);
        }
        if (which < 0) return false;
        g = group_of(args, which);
        seq = g.s0;
        sq = {g.a, g.rows, g.len, false};
        // where its rows stand
        least = 0x7fffffff;
        most = -1;
        for (int i = lane; i < g.n; i += 64) {
            const SeqRows r = seq_rows(p.b, g.s0 + i);
            if (r.n > 0 && !r.bad) {
                least = min(least, r.len - r.n);
                most = max(most, r.len - 1);
            }
        }
        least = ~wave_max_i(~least);
        most = wave_max_i(most);
        seen = seen_tiles<many::TILE>(least, min(most, g.len - 1), p.window, p.sinks);
        v0 = split * args.chunk;
        v1 = min(v0 + args.chunk, seen.total());
        // (chunks that nothing is left for leave empty parts)
        return split == 0 || v0 * many::TILE < g.len;
    }
    __device__ __forceinline__ int all_hi() const { return min(least, g.len - 1) + 1; }
    __device__ __forceinline__ int all_lo(const PagedAttnArgs& p) const { return p.window > 0 ? most - p.window + 1 : 0; }
};
// A wave's 32 columns from w0 on.
struct PrefixColumns {
    static constexpr bool LIMIT = true;
    bool active, live;
    int row, head, pos, hi, lo, len;
    SeenTiles<many::TILE> seen;
    __device__ __forceinline__ int limit() const { return len; }
    __device__ __forceinline__ PrefixColumns(const PagedAttnArgs& p, const PrefixWork& w, int w0)
    {
        const int cols = w.g.rows * p.group, col = w0 + ((int)threadIdx.x & 31);
        active = w0 < cols;
        live = col < cols;
        row = live ? col / p.group : 0;
        head = w.kvh * p.group + (live ? col % p.group : 0);
        len = w.g.len;
        pos = row_position(p.b, w.g, w.g.a + min(col, cols - 1) / p.group);
        const int least = ~wave_max_i(~pos), most = wave_max_i(pos);
        hi = min(least + 1, len);
        lo = p.window > 0 ? most - p.window + 1 : 0;
        seen = seen_tiles<many::TILE>(least, min(most, len - 1), p.window, p.sinks);
    }
};

template <int D, int CT, bool QF32>
__global__ __launch_bounds__(256, QF32 ? 1 : 2) void k_attn_prefix(PrefixArgs p)
{
    __shared__ many::Shared<D, CT, QF32> sh;
    PrefixWork w(p);
    if (!w.find()) return;
    many::attend<D, CT, QF32, PrefixColumns>(p.a, sh, w);
}

// ---- own tokens ----------------------------------------------------------------
// The tiles of tokens that rows at positions p0 .. p1 see, from token `from` on.
struct OwnTiles {
    static constexpr int TILE = few::TILE;
    int head0, head, first, end, lo, hi, from, sinks;
    __device__ __forceinline__ OwnTiles(int p0, int p1, int window, int sinks_, int from_) : from(from_)
    {
        hi = p1 + 1 > from ? p1 + 1 : from;
        lo = window > 0 && p0 - window + 1 > from ? p0 - window + 1 : from;
        if (lo > hi) lo = hi;
        sinks = window > 0 ? min(sinks_, hi) : 0;
        if (sinks >= lo) {  // one range
            lo = from;
            sinks = 0;
        }
        if (sinks <= from) sinks = 0;
        // tiles [head0, head) cover the sinks, [first, end) the rest
        head0 = from / TILE;
        head = sinks > 0 ? (sinks + TILE - 1) / TILE : head0;
        first = max(lo / TILE, head);
        end = hi > lo ? max((hi + TILE - 1) / TILE, first) : first;
    }
    __device__ __forceinline__ int total() const { return head - head0 + end - first; }
    __device__ __forceinline__ int tile(int v) const { return v < head - head0 ? head0 + v : first + v - (head - head0); }
    __device__ __forceinline__ bool any(int t0, int t1) const { return (t0 < hi && t1 > lo) || (t0 < sinks && t1 > from); }
    __device__ __forceinline__ bool some(int t) const { return (t < hi && t >= lo) || (t < sinks && t >= from); }
};
struct OwnTokens {
    static constexpr bool PART = true, POSITIONS = false;
    int from;
    __device__ __forceinline__ bool takes(int t) const { return t >= from; }
    __device__ __forceinline__ void clip(int&, int& lo) const { lo = max(lo, from); }
};
__device__ __forceinline__ OwnTiles own_tiles(const PagedAttnArgs& p, const SeqRows& sq, int from)
{
    const int len = sq.bad ? 0 : sq.len;
    return OwnTiles(len - sq.n, len - 1, p.window, p.sinks, from);
}

template <int D, int CT, bool QF32, int NB>
__global__ __launch_bounds__(few::THREADS, 2) void k_attn_own(PrefixArgs a)
{
    __shared__ few::Shared<D, CT, QF32, NB> sh;
    constexpr int COLS = 16 * NB;
    const PagedAttnArgs& p = a.a;
    const int pairs = p.b.n_seq * p.n_kv;
    const int pair = (int)(blockIdx.x % (unsigned)pairs), rest = (int)(blockIdx.x / (unsigned)pairs);
    const int cb = rest % p.col_blocks, split = rest / p.col_blocks;
    const int seq = pair / p.n_kv;
    const SeqRows sq = seq_rows(p.b, seq);
    if (cb * COLS >= sq.n * p.group) return;
    const int from = shared_by(a, seq);
    const OwnTiles seen = own_tiles(p, sq, from);
    const int v0 = split * p.chunk, v1 = min(v0 + p.chunk, seen.total());
    if (v0 >= v1) return;
    const uint64_t part = (((uint64_t)split * pairs + pair) * p.col_blocks + cb) * COLS;
    few::attend<D, CT, QF32, NB>(p, sh, sq, seq, pair % p.n_kv, cb, seen, v0, v1, p.part_o + part * D, p.part_ml + part * 2,
                                 OwnTokens{from});
}

// ---- the join ------------------------------------------------------------------
// Four groups of D/4 threads a (row, query head).
template <int D, bool QF32>
__global__ __launch_bounds__(256) void k_attn_prefix_join(PrefixArgs a)
{
    constexpr int TH = D / 4, PAR = 4, PER = 256 / (TH * PAR);
    const PagedAttnArgs& p = a.a;
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
    const bool live = row < sq.n;
    float m = -INFINITY, l = 0.0f;
    pf32x4 o = {};
    if (live) {
        const int from = shared_by(a, seq);
        const int n_pre = ((from + many::TILE - 1) / many::TILE + a.chunk - 1) / a.chunk;
        const int n_own = (own_tiles(p, sq, from).total() + p.chunk - 1) / p.chunk;
        const int kvh = head / p.group, col = row * p.group + head % p.group, cb = col / p.cols;
        const uint64_t pre = (uint64_t)(sq.a + row) * p.n_heads + head, pre_step = (uint64_t)p.b.n_rows * p.n_heads;
        const uint64_t own = ((uint64_t)(seq * p.n_kv + kvh) * p.col_blocks + cb) * p.cols + col % p.cols;
        const uint64_t own_step = (uint64_t)p.b.n_seq * p.n_kv * p.col_blocks * p.cols;
        const int n = n_pre + n_own;
        for (int i0 = part; i0 < n; i0 += 4 * PAR) {  // four in flight
            float mi[4], li[4];
            pf32x4 oi[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = min(i0 + j * PAR, n - 1);
                const float* po = i < n_pre ? a.pre_o : p.part_o;
                const float* pm = i < n_pre ? a.pre_ml : p.part_ml;
                const uint64_t at = i < n_pre ? pre + i * pre_step : own + (i - n_pre) * own_step;
                mi[j] = pm[at * 2];
                li[j] = pm[at * 2 + 1];
                oi[j] = *(const pf32x4*)(po + at * D + d);
                if (i0 + j * PAR >= n) {
                    mi[j] = -INFINITY;
                    li[j] = 0.0f;
                }
            }
            add_parts<4>(m, l, o, mi, li, oi);
        }
    }
    *(pf32x4*)&s_o[part][mine][d] = o;
    if (d == 0) {
        s_ml[part][mine][0] = m;
        s_ml[part][mine][1] = l;
    }
    __syncthreads();
    if (part != 0 || !live) return;
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
    const float r[4] = {o[0], o[1], o[2], o[3]};
    attn_store<4, QF32>(p, sq, row, head, d, D, r, l, p.v_scale ? p.v_scale[head / p.group] : 1.0f);
}

template <int D, int CT, bool QF32>
void go(const PrefixArgs& p, hipStream_t s)
{
    PrefixArgs pre = p;  // the many-row pieces write their parts by row
    pre.a.part_o = p.pre_o;
    pre.a.part_ml = p.pre_ml;
    k_attn_prefix<D, CT, QF32><<<dim3((unsigned)(p.a.n_kv * p.blocks * p.splits)), dim3(256), 0, s>>>(pre);
    const dim3 own((unsigned)(p.a.b.n_seq * p.a.n_kv * p.a.col_blocks * p.a.splits));
    if (CT != CT_F32 && p.a.cols == 2 * ATTN_FEW_COLS) {
        if constexpr (CT != CT_F32) k_attn_own<D, CT, QF32, 2><<<own, dim3(few::THREADS), 0, s>>>(p);
    } else {
        k_attn_own<D, CT, QF32, 1><<<own, dim3(few::THREADS), 0, s>>>(p);
    }
    const uint64_t all = (uint64_t)p.a.b.n_seq * p.a.b.max_q * p.a.n_heads;
    k_attn_prefix_join<D, QF32><<<dim3((unsigned)((all * D + 255) / 256)), dim3(256), 0, s>>>(p);
}
template <int D>
void go_types(const PrefixArgs& p, int q_dtype, int cache_dtype, hipStream_t s)
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

hipError_t launch_attn_prefix(const PrefixArgs& p, int head_dim, int q_dtype, int cache_dtype, hipStream_t s)
{
    if (head_dim == 128) go_types<128>(p, q_dtype, cache_dtype, s);
    else go_types<64>(p, q_dtype, cache_dtype, s);
    return hipGetLastError();
}

}  // namespace wpcg
