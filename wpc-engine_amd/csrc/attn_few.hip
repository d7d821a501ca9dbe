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
#include "attn_few.h"

namespace wpcg {
namespace {

using namespace few;

// Tiles of an item of a sequence, at least one (that writes its rows).
__device__ __forceinline__ int item_tiles(const PagedAttnArgs& p, const SeqRows& r)
{
    return r.bad ? 1 : max(1, seen_tiles<TILE>(r.len - r.n, r.len - 1, p.window, p.sinks).total());
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
    (void)hipGetLastError();  // report only these launches
    if (p.b.n_seq == 0) return hipSuccess;
    if (head_dim == 128) go_types<128>(p, q_dtype, cache_dtype, s);
    else go_types<64>(p, q_dtype, cache_dtype, s);
    return hipGetLastError();
}

}  // namespace wpcg
