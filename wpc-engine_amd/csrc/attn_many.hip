// Attention of many rows over paged keys and values: prompts, and chunks of
// prompts behind cached tokens; causal, with a window and sinks.
//
// The work is two matrix products a tile and the exponentials between them:
// the matrix cores are the bound for long prompts, and the vector units come
// close behind. A workgroup takes 128 columns ((row, query head) pairs of one
// key-value head, so that keys and values are shared by the heads of a group),
// or 256, and walks the 64-token tiles they see; each of its four or eight
// waves owns 32 columns and keeps their running maximum, sum and output in
// registers. Tiles no column of a wave sees are skipped, tiles that all see
// whole take no mask.
//
// Layout. 32 x 32 x 16 products with keys as A and queries as B leave the
// scores S^T with column l % 32 in lane l and tokens 8a + 4(l/32) + b, which
// is the second product's B operand as it stands if V^T's A operand takes its
// tokens in the same order. So the softmax's terms stay in their lane, the
// maximum needs one lane exchange, and the rescaling factor is one number a
// lane. Keys go to LDS in rows padded by 16 bytes, so that neither the writes
// (along a row) nor the reads (along tokens) meet in a bank; values are
// transposed in registers by byte permutes on their way to LDS and lie in the
// order the operand is read, 1 KiB a wave without conflicts. The next tile's
// loads are in flight during the products.
//
// Precision is that of attn_few.hip; an F32 cache is carried as three bf16
// terms too, and a product of two fp32 values takes the six of its nine terms
// that reach 2^-24.
//
// Measured, heads of 128, on one card (another one's prompts took 10 % more): a
// prompt of 4096, 32 / 8 heads, BF16 (137 GFLOP) 142 us, 967 TFLOP/s, with the
// matrix cores busy in 41 % of the cycles and the vector units in 42 %; two
// prompts of up to 5000 with a window of 1024, 32 / 4 heads over E4M3 (144 GFLOP)
// 222 us; 777 rows behind 523 tokens, 32 / 4 heads, all F32 (11.6 GFLOP, six
// products each) 124 us with the join's 11. The last 2048 rows of 32768 tokens,
// BF16, 1090 TFLOP/s (a library's 8192^3 product 1300).
#include "attn_many.h"

namespace wpcg {
namespace {

using namespace many;

// Two workgroups of four waves a CU (F32 queries: one).
template <int D, int CT, bool QF32>
__global__ __launch_bounds__(256, QF32 ? 1 : 2) void k_attn_many(PagedAttnArgs p)
{
    __shared__ Shared<D, CT, QF32> sh;
    Work<ATTN_MANY_COLS> w;
    if (!w.find(p)) return;
    attend<D, CT, QF32, Columns>(p, sh, w);
}

// Prompts of BF16 queries with blocks enough: one workgroup of eight waves a CU,
// which brings in each tile once for 256 columns, four waves its values and four
// its keys. With half the registers for tiles on their way, operands are read
// two groups ahead. plan_kernel has its times beside those of two workgroups of
// four waves.
template <int D, int CT>
__global__ __launch_bounds__(512, 2) void k_attn_wide(PagedAttnArgs p)
{
    constexpr int COLS = 2 * ATTN_MANY_COLS;
    using S = Shape<D, CT, false>;
    __shared__ __attribute__((aligned(16))) uint16_t s_k[2][S::KEYS], s_v[2][S::VALUES];
    __shared__ int s_odd[2][4], s_fault;
    Work<COLS> w;
    if (!w.find(p)) return;
    const int kvh = w.kvh, v0 = w.v0, v1 = w.v1;
    Stage<D, CT, 8> stage(p, w.seq, kvh, w.seen, v0, v1, w.all_hi(), w.all_lo(p));
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int c = lane & 31, h = lane >> 5;
    const Columns my(p, w, w.cb * COLS + 32 * wave);
    pbf16x8 qb[D / 16][1];
    load_q<D, 1>(p, (uint64_t)(w.sq.a + my.row) * p.q_row + (uint64_t)my.head * D + 8 * h, my.live, qb);
    const float sc = p.scale * (p.k_scale ? p.k_scale[kvh] : 1.0f);

    pf32x16 acc[D / 32] = {};
    float m = -INFINITY, l = 0.0f;
    if (threadIdx.x == 0) s_fault = 0;  // (read behind the last barrier, written behind the first)
    __syncthreads();
    __builtin_amdgcn_s_waitcnt(0);  // q is there, as in k_attn_many
    if (v0 < v1) stage.fetch(v0);
    for (int vt = v0; vt < v1; vt++) {
        const int b = (vt - v0) & 1;
        const bool all = stage.whole(vt);
        if (!all) {
            const bool odd = stage.clean(vt);
            if (lane == 0 && stage.values) s_odd[b][stage.wave] = odd;
        }
        if (stage.values) stage.put(nullptr, s_v[b]);
        else stage.put(s_k[b], nullptr);
        __syncthreads();
        if (vt + 1 < v1) stage.fetch(vt + 1);
        const int t0 = w.seen.tile(vt) * TILE;
        if (!all && (s_odd[b][0] | s_odd[b][1] | s_odd[b][2] | s_odd[b][3])) {
            if (my.active) add_odd<D, 1>(p, s_v[b], t0, my.pos, acc);
            __syncthreads();
            clear_odd(s_v[b], S::VALUES / 2);
            __syncthreads();
        }
        if (!my.active || !my.seen.any(t0, t0 + TILE)) continue;

        // Operands come from LDS in groups of four fragments, two groups ahead of
        // the products that take them: keys, then values.
        constexpr int KG = 2 * D / 64, VF = D / 32, GROUPS = KG + 4;
        pbf16x8 frag[3][4];
        const auto load = [&](int g) {
            if (g < KG) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    frag[g % 3][i] =
                        *(const pbf16x8*)&s_k[b][key_at<D>(2 * (4 * g % (D / 16) + i) + h, 32 * (4 * g / (D / 16)) + c)];
            } else {
#pragma unroll
                for (int d = 0; d < VF; d++)
                    frag[g % 3][d] = *(const pbf16x8*)&s_v[b][value_at<D>(g - KG, 0, 32 * d) + lane * 8];
            }
        };
        pf32x16 s[2] = {};
        load(0);
        load(1);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int g = 0; g < KG; g++) {
            load(g + 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[4 * g / (D / 16)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    frag[g % 3][i], qb[4 * g % (D / 16) + i][0], s[4 * g / (D / 16)], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (t0 + TILE > my.hi || t0 < my.lo) mask<false>(p, t0, my.pos, s);
        const float base = follow(top_of(s) * sc, m, l, acc);
        pbf16x8 e[2][1];
        terms<1>(s[0], 0, sc, base, l, e[0]);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int g = KG + j;
            if (g + 2 < GROUPS) load(g + 2);
            __builtin_amdgcn_sched_barrier(0);
            if (j < 3) terms<1>(s[(j + 1) / 2], 8 * ((j + 1) % 2), sc, base, l, e[(j + 1) & 1]);
#pragma unroll
            for (int d = 0; d < VF; d++) {
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[g % 3][d], e[j & 1][0], acc[d], 0, 0, 0);
                // a product, then a share of the next group's exponentials
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 7, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    if (stage.fault) s_fault = 1;
    __syncthreads();
    if (!my.live) return;
    l = sum_x32(l);
    if (s_fault) l = __builtin_nanf("");
    put_out<D, S::CW, false>(p, w.sq, w.seq, p.splits > 1 && w.seen.total() > p.chunk, w.split, my.row, my.head, m, l,
                             acc, p.v_scale ? p.v_scale[kvh] : 1.0f);
}

template <int D, int CT, bool QF32>
void go(const PagedAttnArgs& p, unsigned blocks, hipStream_t s)
{
    if constexpr (!QF32) {
        if (p.cols == 2 * ATTN_MANY_COLS) {
            k_attn_wide<D, CT><<<dim3(blocks), dim3(512), 0, s>>>(p);
            return;
        }
    }
    k_attn_many<D, CT, QF32><<<dim3(blocks), dim3(256), 0, s>>>(p);
}

template <int D>
void go_types(const PagedAttnArgs& p, int q_dtype, int cache_dtype, unsigned blocks, hipStream_t s)
{
    if (q_dtype == WPCG_DTYPE_BF16) {
        if (cache_dtype == WPCG_DTYPE_BF16) go<D, CT_BF16, false>(p, blocks, s);
        else go<D, CT_E4M3, false>(p, blocks, s);
    } else {
        if (cache_dtype == WPCG_DTYPE_F32) go<D, CT_F32, true>(p, blocks, s);
        else if (cache_dtype == WPCG_DTYPE_BF16) go<D, CT_BF16, true>(p, blocks, s);
        else go<D, CT_E4M3, true>(p, blocks, s);
    }
}

// ---- the chunks' states joined -------------------------------------------------
// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the chunks that the
// row's workgroups had (where one had all it wrote the outputs), in their order;
// D/4 threads a (row, query head).
template <int D, bool QF32>
__global__ __launch_bounds__(256) void k_attn_many_join(PagedAttnArgs p)
{
    constexpr int TH = D / 4, PER = 256 / TH;
    const int tid = (int)threadIdx.x, d = tid % TH * 4;
    const uint64_t x = (uint64_t)blockIdx.x * PER + tid / TH;
    const int head = (int)(x % (unsigned)p.n_heads);
    const uint64_t at = x / (unsigned)p.n_heads;  // row of the parts
    if (at >= (uint64_t)p.part_rows) return;
    SeqRows sq;
    int row;
    if (p.part_seq) {
        sq = seq_rows(p.b, (int)at / p.part_seq);
        row = (int)at % p.part_seq;
    } else {
        // the row's sequence: the last one that starts at or before it
        int lo = 0, hi = p.b.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if ((p.b.q_start ? p.b.q_start[mid] : mid) <= (int)at) lo = mid;
            else hi = mid - 1;
        }
        sq = seq_rows(p.b, lo);
        row = (int)at - sq.a;
    }
    if (row < 0 || row >= sq.n) return;
    const int cols = sq.n * p.group, cb = (row * p.group + head % p.group) / p.cols;
    const int len = sq.bad ? 0 : sq.len, pos0 = len - sq.n;
    const int first = cb * p.cols / p.group, last = (min(cols, (cb + 1) * p.cols) - 1) / p.group;
    const int tiles = seen_tiles<TILE>(pos0 + first, pos0 + last, p.window, p.sinks).total();
    if (tiles <= p.chunk) return;
    const int n = (tiles + p.chunk - 1) / p.chunk;
    const uint64_t slot0 = at * p.n_heads + head;
    const uint64_t step = (uint64_t)p.part_rows * p.n_heads;
    float m = -INFINITY, l = 0.0f;
    pf32x4 o = {};
    for (int i0 = 0; i0 < n; i0 += 4) {  // four in flight
        float mi[4], li[4];
        pf32x4 oi[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint64_t slot = slot0 + (uint64_t)min(i0 + j, n - 1) * step;
            mi[j] = p.part_ml[slot * 2];
            li[j] = p.part_ml[slot * 2 + 1];
            oi[j] = *(const pf32x4*)(p.part_o + slot * D + d);
            if (i0 + j >= n) {
                mi[j] = -INFINITY;
                li[j] = 0.0f;
            }
        }
        add_parts<4>(m, l, o, mi, li, oi);
    }
    const float r[4] = {o[0], o[1], o[2], o[3]};
    attn_store<4, QF32>(p, sq, row, head, d, D, r, l, p.v_scale ? p.v_scale[head / p.group] : 1.0f);
}
template <int D, bool QF32>
void join(const PagedAttnArgs& p, hipStream_t s)
{
    const uint64_t all = (uint64_t)p.part_rows * p.n_heads;
    k_attn_many_join<D, QF32><<<dim3((unsigned)((all * (D / 4) + 255) / 256)), dim3(256), 0, s>>>(p);
}

}  // namespace

hipError_t launch_attn_many(const PagedAttnArgs& p, int head_dim, int q_dtype, int cache_dtype, hipStream_t s)
{
    (void)hipGetLastError();  // report only these launches
    const uint64_t blocks =
        (p.blocks ? (uint64_t)p.blocks : (uint64_t)p.b.n_seq * p.col_blocks) * p.n_kv * p.splits;
    if (blocks == 0) return hipSuccess;
    const bool f32 = q_dtype == WPCG_DTYPE_F32;
    if (head_dim == 128) {
        go_types<128>(p, q_dtype, cache_dtype, (unsigned)blocks, s);
        if (p.splits > 1) f32 ? join<128, true>(p, s) : join<128, false>(p, s);
    } else {
        go_types<64>(p, q_dtype, cache_dtype, (unsigned)blocks, s);
        if (p.splits > 1) f32 ? join<64, true>(p, s) : join<64, false>(p, s);
    }
    return hipGetLastError();
}

}  // namespace wpcg
