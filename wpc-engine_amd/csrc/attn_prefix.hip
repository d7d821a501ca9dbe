// Attention of few rows a sequence in a batch whose sequences come in groups that
// share their first tokens: several answers to one prompt, beams, questions about
// one document.
//
// The softmax over prefix and own tokens is put together from its parts:
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// The prefix of a group is read once for the rows of all its sequences, whose
// (row, query head) pairs are the columns of the many-row kernel's workgroups
// (attn_many.h), 128 at a time: what the memory bounds one sequence at a time, the
// matrix cores do for many. Own tokens go through the few-row kernel's
// (attn_few.h). Both are dealt out evenly, each over its workgroups of one launch,
// which all fit on the chip at once: with BF16 queries two a CU, of which one as a
// rule waits for the memory with own tokens while the other computes on a prefix.
// Every piece of an item leaves its part, and a second launch joins them.
//
// A CU gets some 20 GB/s from the memory, whatever it has in flight, and a few
// times that from the L2. With prefixes in the few-row kernel's 32 columns, each
// tile loaded for one wave, 8192 tokens shared by 64 rows of 32 / 4 heads took 45
// us for that reason alone.
#include "attn_few.h"
#include "attn_many.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int PCOLS = ATTN_MANY_COLS;

// The batch's row starts and lengths, in LDS, and the lowest and highest position
// of a group's rows.
struct Batch {
    const int *start, *len, *least, *most;
};
__device__ __forceinline__ SeqRows rows_of(const PagedBatch& b, const Batch& x, int s)
{
    const int a = x.start[s], e = b.q_start ? x.start[s + 1] : s + 1, len = x.len[s];
    const bool ok = a >= 0 && a <= e && e <= b.n_rows && e - a <= b.max_q;
    return {a, ok ? e - a : 0, len, len < 0 || len > b.max_kv};
}

// Group g: sequences s0 .. s0 + n - 1, rows a .. a + rows - 1, and how many tokens
// they share; len = 0: it shares nothing (it has one sequence or none, or its
// numbers are out of bounds).
struct Group {
    int s0, n, a, rows, len;
};
__device__ __forceinline__ Group group_of(const PrefixArgs& p, const Batch& x, int g)
{
    const PagedBatch& b = p.a.b;
    Group r;
    r.s0 = p.group_start[g];
    const int s1 = p.group_start[g + 1];
    const bool some = r.s0 >= 0 && r.s0 <= s1 - 2 && s1 <= b.n_seq;
    r.n = some ? s1 - r.s0 : 0;
    r.a = b.q_start ? x.start[some ? r.s0 : 0] : r.s0;
    const int end = b.q_start ? x.start[some ? s1 : 0] : s1;
    const bool rows = some && r.a >= 0 && r.a <= end && end <= b.n_rows && end - r.a <= (int64_t)r.n * b.max_q;
    // the pages are those of the first sequence, which has no more than its own
    const int len = x.len[some ? r.s0 : 0];
    r.len = rows && len <= b.max_kv ? max(0, min(min(p.prefix_len[g], p.max_prefix), len)) : 0;
    r.rows = r.len > 0 ? end - r.a : 0;
    return r;
}
// The group that sequence s is of, if any is: its number, and what is shared.
__device__ __forceinline__ int group_with(const PrefixArgs& p, const Batch& x, int s, Group& g)
{
    int lo = 0, hi = p.n_groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (p.group_start[mid] <= s) lo = mid;
        else hi = mid - 1;
    }
    g = group_of(p, x, lo);
    if (s < g.s0 || s >= g.s0 + g.n) g.len = g.rows = 0;
    return lo;
}
// What came from LDS and is the same in a whole wave, in scalar registers.
using few::uniform;
__device__ __forceinline__ Group uniform(const Group& g)
{
    return {uniform(g.s0), uniform(g.n), uniform(g.a), uniform(g.rows), uniform(g.len)};
}
__device__ __forceinline__ SeqRows uniform(const SeqRows& r)
{
    return {uniform(r.a), uniform(r.n), uniform(r.len), uniform(r.bad) != 0};
}

// ---- prefixes ------------------------------------------------------------------
// A workgroup's 128 columns of a group's rows over some tiles of its prefix.
struct PrefixWork {
    const PrefixArgs& args;
    const Batch& x;
    const Group& g;
    SeqRows sq;  // the group's rows
    int seq, kvh, cb, split, v0, v1;
    int least, most;  // its rows' positions
    SeenTiles<many::TILE> seen;
    float *part_o, *part_ml;
    __device__ __forceinline__ int all_hi() const { return min(least, g.len - 1) + 1; }
    __device__ __forceinline__ int all_lo(const PagedAttnArgs& p) const { return p.window > 0 ? most - p.window + 1 : 0; }
    __device__ __forceinline__ bool part() const { return true; }
};
__device__ __forceinline__ SeenTiles<many::TILE> prefix_tiles(const PagedAttnArgs& p, const Group& g, int least, int most)
{
    return seen_tiles<many::TILE>(least, min(most, g.len - 1), p.window, p.sinks);
}
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
        // where its row stands, -1 if that is no sequence's
        const int at = w.g.a + min(col, cols - 1) / p.group;
        int s = w.g.s0, last = w.g.s0 + w.g.n - 1;
        while (s < last) {
            const int mid = (s + last + 1) / 2;
            if (w.x.start[mid] <= at) s = mid;
            else last = mid - 1;
        }
        const SeqRows r = rows_of(p.b, w.x, s);
        pos = r.bad || at < r.a || at >= r.a + r.n ? -1 : r.len - r.n + (at - r.a);
        const int least = ~wave_max_i(~pos), most = wave_max_i(pos);
        hi = min(least + 1, len);
        lo = p.window > 0 ? most - p.window + 1 : 0;
        seen = seen_tiles<many::TILE>(least, min(most, len - 1), p.window, p.sinks);
    }
};

// ---- own tokens ----------------------------------------------------------------
// The tiles of tokens that rows at positions p0 .. p1 see, from token `from` on.
struct OwnTiles {
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
        head0 = from / few::TILE;
        head = sinks > 0 ? (sinks + few::TILE - 1) / few::TILE : head0;
        first = max(lo / few::TILE, head);
        end = hi > lo ? max((hi + few::TILE - 1) / few::TILE, first) : first;
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

// ---- the deal ------------------------------------------------------------------
// Entries are the groups, then the sequences. A group's items are (key-value head,
// chunk, column block), a sequence's (key-value head, column block): an order in
// which neighbours read the same keys and values. An item costs its tiles and what
// it takes to begin and end; a workgroup whose share of an item is no more than that
// does nothing for it.
//
// What lies before entry e: at[e].x cost (sequences': behind all groups), at[e].y
// items; tiles[g] of the groups.
template <int OCOLS>
__device__ __forceinline__ void deal(const PrefixArgs& p, const Batch& x, int2* at, int* tiles_of, int2* sums)
{
    const PagedAttnArgs& a = p.a;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int entries = p.n_groups + a.b.n_seq;
    int2 before = {0, 0};
    for (int e0 = 0; e0 < entries; e0 += THREADS) {
        const int e = e0 + (int)threadIdx.x;
        int2 v = {0, 0};
        if (e < p.n_groups) {
            const Group g = group_of(p, x, e);
            const int tiles = g.len > 0 ? prefix_tiles(a, g, x.least[e], x.most[e]).total() : 0;
            const int cbs = (g.rows * a.group + PCOLS - 1) / PCOLS;
            tiles_of[e] = tiles;
            v.y = a.n_kv * cbs * ((tiles + p.chunk - 1) / p.chunk);
            v.x = v.y * PREFIX_ITEM + a.n_kv * cbs * tiles;
        } else if (e < entries) {
            const int s = e - p.n_groups;
            Group g;
            group_with(p, x, s, g);
            const SeqRows sq = rows_of(a.b, x, s);
            const int tiles = own_tiles(a, sq, g.len).total();
            v.y = tiles > 0 ? a.n_kv * ((sq.n * a.group + OCOLS - 1) / OCOLS) : 0;
            v.x = v.y * (tiles + OWN_ITEM);
        }
        int2 t = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int ux = __shfl_up(t.x, d), uy = __shfl_up(t.y, d);
            if (lane >= d) {
                t.x += ux;
                t.y += uy;
            }
        }
        if (lane == 63) sums[wave] = t;
        __syncthreads();
        int2 all = {0, 0}, start = before;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            if (w < wave) {
                start.x += sums[w].x;
                start.y += sums[w].y;
            }
            all.x += sums[w].x;
            all.y += sums[w].y;
        }
        if (e < entries) at[e] = {start.x + t.x - v.x, start.y + t.y - v.y};
        before.x += all.x;
        before.y += all.y;
        __syncthreads();
    }
    if (threadIdx.x == 0) at[entries] = before;
    __syncthreads();
}
// How many workgroups of each die's `blocks` take prefixes, and the shares.
__device__ __forceinline__ PrefixDeal shares(const PrefixArgs& p, int pre, int own)
{
    const int blocks = p.a.blocks / 8;
    const double all = (double)pre * p.pre_weight + (double)own * p.own_weight;
    PrefixDeal r;
    r.pre = pre == 0 ? 0 : max(1, min(own == 0 ? blocks : blocks - 1, (int)(blocks * ((double)pre * p.pre_weight / all) + 0.5)));
    const int n = 8 * r.pre, m = 8 * (blocks - r.pre);
    r.pre_share = n == 0 ? 1 : max((pre + n - 1) / n, PREFIX_ITEM + 2);
    r.own_share = m == 0 ? 1 : max((own + m - 1) / m, OWN_ITEM + WAVES);
    return r;
}

template <int D, int CT, bool QF32, int NB>
__global__ __launch_bounds__(THREADS, QF32 ? 1 : 2) void k_attn_shared(PrefixArgs p)
{
    __shared__ union {
        many::Shared<D, CT, QF32> pre;
        few::Shared<D, CT, QF32, NB, WAVES> own;
    } sh;
    __shared__ int2 s_at[PREFIX_SEQS + PREFIX_GROUPS + 1], s_sums[WAVES];
    __shared__ int s_start[PREFIX_SEQS + 1], s_len[PREFIX_SEQS];
    __shared__ int s_least[PREFIX_GROUPS], s_most[PREFIX_GROUPS], s_tiles[PREFIX_GROUPS];
    constexpr int OCOLS = 16 * NB;
    const PagedAttnArgs& a = p.a;
    const int n_seq = a.b.n_seq, entries = p.n_groups + n_seq;
    const Batch x = {s_start, s_len, s_least, s_most};
    for (int s = (int)threadIdx.x; s <= n_seq; s += THREADS) {
        s_start[s] = a.b.q_start ? a.b.q_start[s] : s;
        if (s < n_seq) s_len[s] = a.b.kv_len[s];
    }
    for (int g = (int)threadIdx.x; g < p.n_groups; g += THREADS) {
        s_least[g] = 0x7fffffff;
        s_most[g] = -1;
    }
    __syncthreads();
    for (int s = (int)threadIdx.x; s < n_seq; s += THREADS) {
        Group g;
        const int which = group_with(p, x, s, g);
        const SeqRows r = rows_of(a.b, x, s);
        if (g.len > 0 && r.n > 0 && !r.bad) {
            atomicMin(&s_least[which], r.len - r.n);
            atomicMax(&s_most[which], r.len - 1);
        }
    }
    __syncthreads();
    deal<OCOLS>(p, x, s_at, s_tiles, s_sums);
    const int pre = uniform(s_at[p.n_groups].x), pre_items = uniform(s_at[p.n_groups].y);
    const PrefixDeal sizes = shares(p, pre, uniform(s_at[entries].x) - pre);
    if (blockIdx.x == 0) {  // for the join
        for (int e = (int)threadIdx.x; e <= entries; e += THREADS) p.at[e] = s_at[e];
        for (int g = (int)threadIdx.x; g < p.n_groups; g += THREADS) p.tiles[g] = s_tiles[g];
        if (threadIdx.x == 0) *p.deal = sizes;
    }
    // each die's workgroups take one stretch of the prefixes and one of own tokens;
    // its first ones, one a CU, as a rule the former
    const int die = (int)(blockIdx.x % 8u), j = (int)(blockIdx.x / 8u);
    if (j < sizes.pre) {
        const int b = die * sizes.pre + j;
        const int64_t from = (int64_t)b * sizes.pre_share;
        const int end = (int)min(from + sizes.pre_share, (int64_t)pre);
        for (int64_t at = from; at < end;) {
            int lo = 0, hi = p.n_groups - 1;  // the last group that begins at or before `at`
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (uniform(s_at[mid].x) <= at) lo = mid;
                else hi = mid - 1;
            }
            const int2 base = {uniform(s_at[lo].x), uniform(s_at[lo].y)};
            const int in = (int)at - base.x;
            const Group g = uniform(group_of(p, x, lo));
            const int least = uniform(s_least[lo]), most = uniform(s_most[lo]);
            const int tiles = uniform(s_tiles[lo]), cbs = (g.rows * a.group + PCOLS - 1) / PCOLS;
            const int chunks = (tiles + p.chunk - 1) / p.chunk;
            const int of_kvh = cbs * (tiles + chunks * PREFIX_ITEM), kvh = in / of_kvh;
            const int of_chunk = cbs * (p.chunk + PREFIX_ITEM), ch = in % of_kvh / of_chunk;
            const int n = min(p.chunk, tiles - ch * p.chunk), c = in % of_kvh - ch * of_chunk;
            const int cb = c / (n + PREFIX_ITEM), v = c % (n + PREFIX_ITEM);
            const int take = min(n + PREFIX_ITEM - v, end - (int)at);
            const int v0 = ch * p.chunk + max(0, v - PREFIX_ITEM), v1 = ch * p.chunk + max(0, v + take - PREFIX_ITEM);
            const uint64_t slot = (uint64_t)(base.y + (kvh * chunks + ch) * cbs + cb + b);
            if (v0 < v1 && slot < p.pre_slots) {
                const PrefixWork w = {p, x, g, {g.a, g.rows, g.len, false}, g.s0, kvh, cb, 0, v0, v1, least, most,
                                      prefix_tiles(a, g, least, most), p.pre_o + slot * PCOLS * D, p.pre_ml + slot * PCOLS * 2};
                many::attend<D, CT, QF32, PrefixColumns>(a, sh.pre, w);
            }
            at += take;
            __syncthreads();  // the tiles and states in LDS are read
        }
    } else {
        const int b = die * (a.blocks / 8 - sizes.pre) + j - sizes.pre;
        const int64_t from = pre + (int64_t)b * sizes.own_share;
        const int end = (int)min(from + sizes.own_share, (int64_t)uniform(s_at[entries].x));
        for (int64_t at = from; at < end;) {
            int lo = p.n_groups, hi = entries - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (uniform(s_at[mid].x) <= at) lo = mid;
                else hi = mid - 1;
            }
            const int2 base = {uniform(s_at[lo].x), uniform(s_at[lo].y)};
            const int in = (int)at - base.x, s = lo - p.n_groups;
            Group g;
            group_with(p, x, s, g);
            g.len = uniform(g.len);
            const SeqRows sq = uniform(rows_of(a.b, x, s));
            const OwnTiles seen = own_tiles(a, sq, g.len);
            const int of_item = seen.total() + OWN_ITEM, cbs = (sq.n * a.group + OCOLS - 1) / OCOLS;
            const int item = in / of_item, v = in % of_item, take = min(of_item - v, end - (int)at);
            const int v0 = max(0, v - OWN_ITEM), v1 = max(0, v + take - OWN_ITEM);
            const uint64_t slot = (uint64_t)(base.y - pre_items + item + b);
            if (v0 < v1 && slot < p.own_slots)
                few::attend<D, CT, QF32, NB>(a, sh.own, sq, s, item / cbs, item % cbs, seen, v0, v1,
                                             a.part_o + slot * OCOLS * D, a.part_ml + slot * OCOLS * 2, OwnTokens{g.len});
            at += take;
            __syncthreads();
        }
    }
}

// ---- the join ------------------------------------------------------------------
// Four groups of D/4 threads a (row, query head). The item that a row's column
// is in has a part from each workgroup that takes some of its tiles.
template <int D, bool QF32, int OCOLS>
__global__ __launch_bounds__(256) void k_attn_shared_join(PrefixArgs p)
{
    constexpr int TH = D / 4, PAR = 4, PER = 256 / (TH * PAR);
    const PagedAttnArgs& a = p.a;
    __shared__ float s_o[PAR][PER][D];
    __shared__ float s_ml[PAR][PER][2];
    const int tid = (int)threadIdx.x;
    const int part = tid / TH % PAR, mine = tid / (TH * PAR), d = tid % TH * 4;
    const uint64_t x = (uint64_t)blockIdx.x * PER + mine;
    const int head = (int)(x % (unsigned)a.n_heads);
    const uint64_t rest = x / (unsigned)a.n_heads;
    const int row = (int)(rest / (unsigned)a.b.n_seq), seq = (int)(rest % (unsigned)a.b.n_seq);
    SeqRows sq = {};
    if (row < a.b.max_q) sq = seq_rows(a.b, seq);
    const bool live = row < sq.n;
    float m = -INFINITY, l = 0.0f;
    pf32x4 o = {};
    if (live) {
        const PrefixDeal sizes = *p.deal;
        const int kvh = head / a.group;
        const Batch batch = {a.b.q_start, a.b.kv_len, nullptr, nullptr};
        Group g;
        const int which = group_with(p, batch, seq, g);
        const int2 groups = p.at[p.n_groups];
        // the prefix
        int tiles = 0, cbs = 0, cb = 0, col = 0, chunks = 0;
        int2 base = {0, 0};
        if (g.len > 0) {
            base = p.at[which];
            tiles = p.tiles[which];
            col = (sq.a + row - g.a) * a.group + head % a.group;
            cb = col / PCOLS;
            cbs = (g.rows * a.group + PCOLS - 1) / PCOLS;
            chunks = (tiles + p.chunk - 1) / p.chunk;
        }
        // its own tokens
        const int2 own = p.at[p.n_groups + seq], next = p.at[p.n_groups + seq + 1];
        const int own_col = row * a.group + head % a.group;
        const int of_item = next.y > own.y ? (next.x - own.x) / (next.y - own.y) : 0;
        const int own_item = kvh * ((sq.n * a.group + OCOLS - 1) / OCOLS) + own_col / OCOLS;
        for (int i = part; i <= chunks; i += PAR) {  // the last one: its own
            int from, cost, share;  // where its tiles begin in the deal, and how many they are
            const float *po, *pm;
            uint64_t slot0, slots, at, step;
            if (i < chunks) {
                cost = min(p.chunk, tiles - i * p.chunk);
                from = base.x + kvh * cbs * (tiles + chunks * PREFIX_ITEM) + i * cbs * (p.chunk + PREFIX_ITEM) +
                       cb * (cost + PREFIX_ITEM) + PREFIX_ITEM;
                share = sizes.pre_share;
                slot0 = (uint64_t)(base.y + (kvh * chunks + i) * cbs + cb);
                slots = p.pre_slots;
                po = p.pre_o;
                pm = p.pre_ml;
                at = col % PCOLS;
                step = PCOLS;
            } else {
                cost = of_item - OWN_ITEM;
                from = own.x - groups.x + own_item * of_item + OWN_ITEM;
                share = sizes.own_share;
                slot0 = (uint64_t)(own.y - groups.y + own_item);
                slots = p.own_slots;
                po = a.part_o;
                pm = a.part_ml;
                at = own_col % OCOLS;
                step = OCOLS;
            }
            if (cost <= 0) continue;
            const int b0 = from / share, n = (from + cost - 1) / share - b0 + 1;
            for (int j0 = 0; j0 < n; j0 += 4) {  // four in flight
                float mi[4], li[4];
                pf32x4 oi[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint64_t slot = slot0 + b0 + min(j0 + j, n - 1);
                    const uint64_t to = (slot < slots ? slot : 0) * step + at;
                    mi[j] = pm[to * 2];
                    li[j] = pm[to * 2 + 1];
                    oi[j] = *(const pf32x4*)(po + to * D + d);
                    if (j0 + j >= n) {
                        mi[j] = -INFINITY;
                        li[j] = 0.0f;
                    }
                }
                add_parts<4>(m, l, o, mi, li, oi);
            }
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
    attn_store<4, QF32>(a, sq, row, head, d, D, r, l, a.v_scale ? a.v_scale[head / a.group] : 1.0f);
}

template <int D, int CT, bool QF32, int NB>
void go_cols(const PrefixArgs& p, hipStream_t s)
{
    k_attn_shared<D, CT, QF32, NB><<<dim3((unsigned)p.a.blocks), dim3(THREADS), 0, s>>>(p);
    const uint64_t all = (uint64_t)p.a.b.n_seq * p.a.b.max_q * p.a.n_heads;
    k_attn_shared_join<D, QF32, 16 * NB><<<dim3((unsigned)((all * D + 255) / 256)), dim3(256), 0, s>>>(p);
}
template <int D, int CT, bool QF32>
void go(const PrefixArgs& p, hipStream_t s)
{
    if constexpr (CT != CT_F32) {
        if (p.a.cols == 2 * ATTN_FEW_COLS) {
            go_cols<D, CT, QF32, 2>(p, s);
            return;
        }
    }
    go_cols<D, CT, QF32, 1>(p, s);
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
