// Attention of few rows a sequence in a batch whose sequences come in groups that
// share their first tokens: several answers to one prompt, beams, questions about
// one document.
//
// The softmax over prefix and own tokens is put together from its parts:
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// The prefix of a group is read once for the rows of all its sequences, whose
// (row, query head) pairs are the columns of the many-row kernel's workgroups
// (attn_many.h), 128 at a time: what the memory bounds one sequence at a time, the
// matrix cores do for many. Own tokens are single waves' work, a few tiles of a
// sequence's key-value head each, by the few-row kernel's steps (attn_few.h) without
// its barriers. All of it is one launch whose workgroups are on the chip together,
// with BF16 queries two a CU: the first of them takes prefixes alone, the second
// own tokens, which wait for the memory, and then what is left of its equal share
// of the prefixes. Every piece leaves its part, and a second launch joins them.
//
// A CU gets some 20 GB/s from the memory, whatever it has in flight, and a few
// times that from the L2. With prefixes in the few-row kernel's 32 columns, each
// tile loaded for one wave, 8192 tokens shared by 64 rows of 32 / 4 heads took 45
// us for that reason alone. With own tokens in whole workgroups' items, dealt out
// evenly beside the prefixes, each of them began and ended in 9 us, whatever its
// tiles.
//
// 64 rows of 32 / 4 heads, 8192 shared tokens and up to 1000 own, BF16: 40 us and
// the join's 8, of which the deal 4.5, a workgroup's prefix 5 and 2.2 a tile (64
// tokens, 128 columns: 490 TFLOP/s with the CU's other workgroup waiting for own
// tokens, and twice that with both at prefixes). Six groups of 16 over E4M3, 32 / 8
// heads: 30 and 8. 32 rows over 65536 shared tokens, F32 queries over E4M3, three
// products each: 116 and 9, 0.84 PFLOP/s in all, one wave a SIMD.
//
// Precision is that of the kernels whose pieces these are: BF16 queries round the
// softmax's terms to bf16 for their product with the values (the matrix cores take
// nothing wider at that rate), relative to the maximum of what a part has read; sums,
// maxima and the parts are fp32, as is the join. The first case is off by 2.3e-3 of the
// outputs, root mean square, of which their own rounding to bf16 is 1.7e-3.
#include "attn_few.h"
#include "attn_many.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int PCOLS = ATTN_MANY_COLS;

// The batch in LDS: row starts and lengths, the groups' first sequences, how many tokens
// they share and from whose pages these are read, the lowest and highest position of a
// group's rows.
struct Batch {
    const int *start, *len, *group, *prefix, *least, *most;
    const uint16_t* from;
};
__device__ __forceinline__ SeqRows rows_of(const PagedBatch& b, const Batch& x, int s)
{
    const int a = x.start[s], e = b.q_start ? x.start[s + 1] : s + 1, len = x.len[s];
    const bool ok = a >= 0 && a <= e && e <= b.n_rows && e - a <= b.max_q;
    return {a, ok ? e - a : 0, len, len < 0 || len > b.max_kv};
}

// Group g: sequences s0 .. s0 + n - 1, rows a .. a + rows - 1, and how many tokens
// they share; n = 0: its numbers are out of bounds, or it has one sequence or none.
struct Group {
    int s0, n, a, rows, len;
};
__device__ __forceinline__ Group group_rows(const PrefixArgs& p, const Batch& x, int g)
{
    const PagedBatch& b = p.a.b;
    Group r = {};
    r.s0 = x.group[g];
    const int s1 = x.group[g + 1];
    const bool some = r.s0 >= 0 && r.s0 < s1 && s1 <= b.n_seq && s1 - r.s0 > 1;  // (in this order nothing overflows)
    r.a = x.start[some ? r.s0 : 0];
    const int end = x.start[some ? s1 : 0], n = some ? s1 - r.s0 : 0;
    if (some && r.a >= 0 && r.a <= end && end <= b.n_rows && end - r.a <= (int64_t)n * b.max_q) {
        r.n = n;
        r.rows = end - r.a;
    }
    return r;
}
// How many tokens it shares, at most `prefix` and from the pages of sequence `from`,
// which has no more than its own.
__device__ __forceinline__ int group_length(const PrefixArgs& p, const Batch& x, int g, int from, int prefix)
{
    const Group r = group_rows(p, x, g);
    const int len = x.len[r.n > 0 ? from : 0];
    return r.n > 0 && len <= p.a.b.max_kv ? max(0, min(prefix, len)) : 0;
}
__device__ __forceinline__ Group group_of(const PrefixArgs& p, const Batch& x, int g)
{
    Group r = group_rows(p, x, g);
    r.len = x.prefix[g];
    if (r.len == 0) r.rows = 0;
    return r;
}
// The last group that begins at or before sequence s.
__device__ __forceinline__ int group_at(const PrefixArgs& p, const Batch& x, int s)
{
    int lo = 0, hi = p.n_groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (x.group[mid] <= s) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// The group that sequence s is of, if any is: its number, and what is shared.
__device__ __forceinline__ int group_with(const PrefixArgs& p, const Batch& x, int s, Group& g)
{
    const int which = group_at(p, x, s);
    g = group_of(p, x, which);
    if (s < g.s0 || s >= g.s0 + g.n) g.len = g.rows = 0;
    return which;
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
// The tiles of a prefix of len tokens that rows at positions least .. most see.
__device__ __forceinline__ SeenTiles<many::TILE> prefix_tiles(const PagedAttnArgs& p, int len, int least, int most)
{
    SeenTiles<many::TILE> r = seen_tiles<many::TILE>(least, min(most, len - 1), p.window, p.sinks);
    if (r.lo == r.hi) {  // the windows have left it: none but the sinks'
        r.lo = r.hi = 0;
        r.end = r.first;
    }
    return r;
}
// A workgroup's 128 columns of a group's rows over some tiles of its prefix.
struct PrefixWork {
    const Batch& x;
    const Group& g;
    SeqRows sq;  // the group's rows
    int seq, kvh, cb, v0, v1;
    int least, most;  // its rows' positions
    SeenTiles<many::TILE> seen;
    float *part_o, *part_ml;
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
        seen = prefix_tiles(p, len, least, most);
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
    static constexpr bool PART = true;
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
// Prefixes: a group's items are (key-value head, chunk, column block), an order in
// which neighbours read the same keys and values. An item costs its tiles and what
// it takes to begin and end; a workgroup whose share of an item is no more than that
// does nothing for it. Own tokens: a sequence's items are (key-value head, column
// block, chunk of deal.own_chunk tiles), a wave's work each.
struct Tables {
    int2 at[PREFIX_GROUPS + 1];  // cost and items before a group
    int tiles[PREFIX_GROUPS];    // of its prefix
    int items[PREFIX_SEQS + 1];  // own items before a sequence
};
__device__ __forceinline__ int own_columns(const PagedAttnArgs& a, const SeqRows& sq, int cols)
{
    return (sq.n * a.group + cols - 1) / cols;
}
// The sums over the threads before this one, and over all in total; s: WAVES int3s.
__device__ __forceinline__ int wave_scan_i(int v)
{
    v += wave_dpp_i<0x111>(0, v);  // lanes 1, 2, 4 and 8 before, in rows of 16
    v += wave_dpp_i<0x112>(0, v);
    v += wave_dpp_i<0x114>(0, v);
    v += wave_dpp_i<0x118>(0, v);
    v += wave_dpp_i<WDPP_BCAST15, 0xA>(0, v);
    return v + wave_dpp_i<WDPP_BCAST31, 0xC>(0, v);
}
__device__ __forceinline__ int3 block_before(int3 v, int3* s, int3& total)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int3 t = {wave_scan_i(v.x), wave_scan_i(v.y), wave_scan_i(v.z)};
    if (lane == 63) s[wave] = t;
    __syncthreads();
    int3 start = {0, 0, 0};
    total = start;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w == wave) start = total;
        total = {total.x + s[w].x, total.y + s[w].y, total.z + s[w].z};
    }
    __syncthreads();
    return {start.x + t.x - v.x, start.y + t.y - v.y, start.z + t.z - v.z};
}
template <int OCOLS>
__device__ __forceinline__ PrefixDeal deal(const PrefixArgs& p, const Batch& x, Tables& t, int3* sums)
{
    static_assert(PREFIX_GROUPS <= THREADS && PREFIX_SEQS <= 2 * THREADS, "a group a thread, two sequences");
    const PagedAttnArgs& a = p.a;
    const int tid = (int)threadIdx.x;
    int3 v = {0, 0, 0};  // cost and items of a group, own tiles of two sequences
    if (tid < p.n_groups) {
        const Group g = group_of(p, x, tid);
        const int tiles = g.len > 0 ? prefix_tiles(a, g.len, x.least[tid], x.most[tid]).total() : 0;
        const int cbs = (g.rows * a.group + PCOLS - 1) / PCOLS;
        t.tiles[tid] = tiles;
        v.y = a.n_kv * cbs * ((tiles + p.chunk - 1) / p.chunk);
        v.x = v.y * PREFIX_ITEM + a.n_kv * cbs * tiles;
    }
    int tiles[2] = {0, 0}, cbs[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int s = 2 * tid + i;
        if (s >= a.b.n_seq) continue;
        Group g;
        group_with(p, x, s, g);
        const SeqRows sq = rows_of(a.b, x, s);
        tiles[i] = own_tiles(a, sq, g.len).total();
        cbs[i] = a.n_kv * own_columns(a, sq, OCOLS);
        v.z += tiles[i] * cbs[i];
    }
    int3 total, none;
    const int3 before = block_before(v, sums, total);
    if (tid < p.n_groups) t.at[tid] = {before.x, before.y};
    if (tid == 0) t.at[p.n_groups] = {total.x, total.y};
    const int pre = uniform(total.x), own = uniform(total.z);
    PrefixDeal r;
    // an item a wave, if that makes more than OWN_CHUNK tiles (each sequence's head has
    // half an item more than its tiles make)
    const int n = a.blocks / 8, second = n - p.first;  // workgroups of a die
    const int waves = WAVES * 8 * second, full = waves - min(a.b.n_seq * a.n_kv, waves) / 2;
    r.own_chunk = max(OWN_CHUNK, (own + full - 1) / full);
    int items[2];
#pragma unroll
    for (int i = 0; i < 2; i++) items[i] = cbs[i] * ((tiles[i] + r.own_chunk - 1) / r.own_chunk);
    const int first = block_before({items[0] + items[1], 0, 0}, sums, none).x;
    if (2 * tid <= a.b.n_seq) t.items[2 * tid] = first;
    if (2 * tid + 1 <= a.b.n_seq) t.items[2 * tid + 1] = first + items[0];
    if (tid == THREADS - 1 && a.b.n_seq == 2 * THREADS) t.items[a.b.n_seq] = first + items[0] + items[1];
    // the workgroups' shares of the prefixes: equal with what own tokens cost counted in
    r.first = p.first;
    const int cost = own > 0 ? OWN_ITEM + r.own_chunk : 0;
    const int share = (int)(((int64_t)pre + (int64_t)8 * second * cost + 8 * n - 1) / (8 * n));
    r.share[0] = share;
    r.share[1] = share - cost;
    if (r.first > 0 && r.share[1] < PREFIX_ITEM + 2) {
        r.share[0] = (pre + 8 * r.first - 1) / (8 * r.first);
        r.share[1] = 0;
    }
    r.share[0] = max(r.share[0], PREFIX_ITEM + 2);
    if (r.first == 0 || r.share[1] > 0) r.share[1] = max(r.share[1], PREFIX_ITEM + 2);
    __syncthreads();
    return r;
}

template <int D, int CT, bool QF32, int NB>
__global__ __launch_bounds__(THREADS, QF32 ? 1 : 2) void k_attn_shared(PrefixArgs p)
{
    __shared__ union {
        many::Shared<D, CT, QF32> pre;
        few::Shared<D, CT, QF32, NB, 1> own[WAVES];
    } sh;
    __shared__ Tables t;
    __shared__ int3 s_sums[WAVES];
    __shared__ int s_start[PREFIX_SEQS + 1], s_len[PREFIX_SEQS];
    __shared__ int s_group[PREFIX_GROUPS + 1], s_prefix[PREFIX_GROUPS], s_least[PREFIX_GROUPS], s_most[PREFIX_GROUPS];
    __shared__ uint16_t s_from[PREFIX_GROUPS];  // (two workgroups fill a CU's LDS but for some 300 bytes each)
    constexpr int OCOLS = 16 * NB;
    const PagedAttnArgs& a = p.a;
    const int n_seq = a.b.n_seq, tid = (int)threadIdx.x;
    const Batch x = {s_start, s_len, s_group, s_prefix, s_least, s_most, s_from};
    for (int s = tid; s <= n_seq; s += THREADS) {
        s_start[s] = a.b.q_start ? a.b.q_start[s] : s;
        if (s < n_seq) s_len[s] = a.b.kv_len[s];
    }
    for (int g = tid; g <= p.n_groups; g += THREADS) {
        s_group[g] = p.group_start[g];
        if (g == p.n_groups) break;
        s_prefix[g] = p.prefix_len[g];
        s_least[g] = 0x7fffffff;
        s_most[g] = -1;
        t.tiles[g] = 0x7fffffff;  // (below the sequence whose pages are read)
    }
    __syncthreads();
    const auto sees = [](const SeqRows& r) { return r.n > 0 && !r.bad && r.len > 0; };
    bool falls = false;
    int which[2], least[2];  // of the thread's sequences that see something: group and first position
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int s = tid + i * THREADS;
        which[i] = -1;
        if (s >= n_seq) continue;
        falls |= s_start[s + 1] < s_start[s];
        const int g = group_at(p, x, s);
        const Group of = group_rows(p, x, g);
        const SeqRows r = rows_of(a.b, x, s);
        if (s < of.s0 || s >= of.s0 + of.n || !sees(r)) continue;
        which[i] = g;
        least[i] = r.len - r.n;
        atomicMin(&s_least[g], least[i]);
        atomicMax(&s_most[g], r.len - 1);
        if (a.window <= 0) atomicMin(&t.tiles[g], s);
    }
    const int own_group = THREADS - 1 - tid;  // (of the waves with fewest sequences)
    if (own_group < p.n_groups) falls |= s_group[own_group + 1] < s_group[own_group];
    falls = __any(falls);
    if ((tid & 63) == 0) t.items[tid >> 6] = falls;  // (the deal writes there behind a barrier of its own)
    __syncthreads();
    // Pages are those of the first sequence that has rows: nobody looks at the others'. With a
    // window only the sequence whose rows begin lowest is sure to have all pages that
    // the others' rows see, as far as its own rows go: those that are further on may have
    // given theirs away.
    if (a.window > 0) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (which[i] >= 0 && least[i] == s_least[which[i]]) atomicMin(&t.tiles[which[i]], tid + i * THREADS);
        __syncthreads();
    }
    // Where starts fall, groups or their rows may lie over each other and be more than
    // the parts' places are for: nothing is shared.
    falls = (t.items[0] | t.items[1] | t.items[2] | t.items[3]) != 0;
    if (own_group < p.n_groups) {
        const bool some = t.tiles[own_group] < n_seq && !falls;
        const int from = some ? t.tiles[own_group] : 0;
        s_from[own_group] = (uint16_t)from;
        s_prefix[own_group] = some ? group_length(p, x, own_group, from, min(s_prefix[own_group], p.max_prefix)) : 0;
    }
    __syncthreads();
    const PrefixDeal dealt = deal<OCOLS>(p, x, t, s_sums);
    if (blockIdx.x == 0) {  // for the join
        for (int s = tid; s < n_seq; s += THREADS) {
            Group g;
            const int which = group_with(p, x, s, g);
            const int chunks = (own_tiles(a, rows_of(a.b, x, s), g.len).total() + dealt.own_chunk - 1) / dealt.own_chunk;
            p.seqs[s] = {t.at[which].x, t.at[which].y, g.len > 0 ? t.tiles[which] : 0,
                         g.len > 0 ? (t.tiles[which] + p.chunk - 1) / p.chunk : 0, g.a,
                         (g.rows * a.group + PCOLS - 1) / PCOLS, t.items[s], chunks};
        }
        if (tid == 0) *p.deal = dealt;
    }

    // own tokens: neighbouring items on different CUs
    const int die = (int)(blockIdx.x % 8u), j = (int)(blockIdx.x / 8u);
    if (j >= dealt.first) {
        const int wave = uniform(tid >> 6), groups = a.blocks - 8 * dealt.first;
        const int all = uniform(t.items[n_seq]);
        for (int i = wave * groups + (int)blockIdx.x - 8 * dealt.first; i < all; i += WAVES * groups) {
            int lo = 0, hi = n_seq - 1;  // the last sequence whose items begin at or before i
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (uniform(t.items[mid]) <= i) lo = mid;
                else hi = mid - 1;
            }
            Group g;
            group_with(p, x, lo, g);
            g.len = uniform(g.len);
            const SeqRows sq = uniform(rows_of(a.b, x, lo));
            const OwnTiles seen = own_tiles(a, sq, g.len);
            const int chunks = (seen.total() + dealt.own_chunk - 1) / dealt.own_chunk, cbs = own_columns(a, sq, OCOLS);
            const int in = i - uniform(t.items[lo]), v0 = in % chunks * dealt.own_chunk;
            if ((uint64_t)i < p.own_slots)
                few::attend<D, CT, QF32, NB, 1>(a, sh.own[wave], sq, lo, in / chunks / cbs, in / chunks % cbs, seen, v0,
                                                min(v0 + dealt.own_chunk, seen.total()), a.part_o + (uint64_t)i * OCOLS * D,
                                                a.part_ml + (uint64_t)i * OCOLS * 2, OwnTokens{g.len});
        }
        __syncthreads();  // tiles of prefixes go where their queries lay
    }

    // prefixes: each die's workgroups take one stretch
    const int share = dealt.share[j >= dealt.first];
    const int of_die = dealt.first * dealt.share[0] + (a.blocks / 8 - dealt.first) * dealt.share[1];
    const int64_t from = (int64_t)die * of_die + min(j, dealt.first) * dealt.share[0] + max(j - dealt.first, 0) * dealt.share[1];
    const int end = (int)min(from + share, (int64_t)uniform(t.at[p.n_groups].x));
    const int b = die * (dealt.share[1] > 0 ? a.blocks / 8 : dealt.first) + j;  // of those that take some
    for (int64_t at = from; at < end;) {
        int lo = 0, hi = p.n_groups - 1;  // the last group that begins at or before `at`
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (uniform(t.at[mid].x) <= at) lo = mid;
            else hi = mid - 1;
        }
        const int2 base = {uniform(t.at[lo].x), uniform(t.at[lo].y)};
        const int in = (int)at - base.x;
        const Group g = uniform(group_of(p, x, lo));
        const int least = uniform(s_least[lo]), most = uniform(s_most[lo]);
        const int tiles = uniform(t.tiles[lo]), cbs = (g.rows * a.group + PCOLS - 1) / PCOLS;
        const int chunks = (tiles + p.chunk - 1) / p.chunk;
        const int of_kvh = cbs * (tiles + chunks * PREFIX_ITEM), kvh = in / of_kvh;
        const int of_chunk = cbs * (p.chunk + PREFIX_ITEM), ch = in % of_kvh / of_chunk;
        const int n = min(p.chunk, tiles - ch * p.chunk), c = in % of_kvh - ch * of_chunk;
        const int cb = c / (n + PREFIX_ITEM), v = c % (n + PREFIX_ITEM);
        const int take = min(n + PREFIX_ITEM - v, end - (int)at);
        const int v0 = ch * p.chunk + max(0, v - PREFIX_ITEM), v1 = ch * p.chunk + max(0, v + take - PREFIX_ITEM);
        const uint64_t slot = (uint64_t)(base.y + (kvh * chunks + ch) * cbs + cb + b);
        if (v0 < v1 && slot < p.pre_slots) {
            const PrefixWork w = {x, g, {g.a, g.rows, g.len, false}, uniform((int)s_from[lo]), kvh, cb, v0, v1, least, most,
                                  prefix_tiles(a, g.len, least, most), p.pre_o + slot * PCOLS * D, p.pre_ml + slot * PCOLS * 2};
            many::attend<D, CT, QF32, PrefixColumns>(a, sh.pre, w);
        }
        at += take;
        __syncthreads();  // the tiles and states in LDS are read
    }
}

// ---- the join ------------------------------------------------------------------
// x / d for quotients below 2^20, by = 1 / d.
__device__ __forceinline__ int divided(int x, int d, float by)
{
    const int q = (int)((float)x * by), r = x - q * d;
    return q + (r >= d) - (r < 0);
}
// Four groups of D/4 threads a (row, query head), which take its parts in turn. The
// items that its column is in, of a prefix's chunks, have a part from each workgroup
// that takes some of their tiles; those of its own tokens one each.
template <int D, bool QF32, int OCOLS>
__global__ __launch_bounds__(256) void k_attn_shared_join(PrefixArgs p)
{
    constexpr int TH = D / 4, PAR = 4, PER = 256 / (TH * PAR), AHEAD = 4;
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
    const PrefixSeq q = p.seqs[seq];
    const PrefixDeal dealt = *p.deal;
    const bool live = row < sq.n;
    float m = -INFINITY, l = 0.0f;
    pf32x4 o = {};
    if (live) {
        const int kvh = head / a.group, of_row = head % a.group;
        const int col = (sq.a + row - q.row) * a.group + of_row, cb = col / PCOLS;
        int before = 0;  // parts of the chunks before
        const auto load = [&](bool it, const float* po, const float* pm, uint64_t slot, uint64_t slots, int step, int at,
                              float& mi, float& li, pf32x4& oi) {
            pf32x2 ml = {-INFINITY, 0.0f};
            oi = (pf32x4){};
            if (it && slot < slots) {
                const uint64_t to = slot * step + at;
                ml = *(const pf32x2*)(pm + to * 2);
                oi = *(const pf32x4*)(po + to * D + d);
            }
            mi = ml[0];
            li = ml[1];
        };
        // own parts are on their way while the prefix's are looked for
        const int own_col = row * a.group + of_row;
        const uint64_t own = (uint64_t)(q.own + (kvh * own_columns(a, sq, OCOLS) + own_col / OCOLS) * q.own_chunks);
        float mo[2], lo[2];
        pf32x4 oo[2];
        const auto load_own = [&](int i) {
#pragma unroll
            for (int j = 0; j < 2; j++)
                load(i + j * PAR < q.own_chunks, a.part_o, a.part_ml, own + i + j * PAR, p.own_slots, OCOLS, own_col % OCOLS,
                     mo[j], lo[j], oo[j]);
        };
        load_own(PAR - 1 - part);
        // the workgroup in whose share a place of the prefixes' costs lies
        const int first = dealt.first * dealt.share[0], of_die = first + (a.blocks / 8 - dealt.first) * dealt.share[1];
        const int n = dealt.share[1] > 0 ? a.blocks / 8 : dealt.first;  // of a die
        const float by_die = 1.0f / (float)of_die, by_first = 1.0f / (float)max(1, dealt.share[0]);
        const float by_second = 1.0f / (float)max(1, dealt.share[1]);
        const auto block_at = [&](int at) {
            const int die = divided(at, of_die, by_die), in = at - die * of_die;
            return die * n + (in < first ? divided(in, dealt.share[0], by_first)
                                         : dealt.first + divided(in - first, dealt.share[1], by_second));
        };
        const int from0 = q.cost + kvh * q.cbs * (q.tiles + q.chunks * PREFIX_ITEM) + PREFIX_ITEM;
        for (int i0 = 0; i0 < q.chunks; i0 += AHEAD) {
            float mi[AHEAD], li[AHEAD];
            pf32x4 oi[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                mi[j] = -INFINITY;
                li[j] = 0.0f;
                oi[j] = (pf32x4){};
                const int i = i0 + j, cost = min(p.chunk, q.tiles - i * p.chunk);
                if (i >= q.chunks) continue;
                const int from = from0 + i * q.cbs * (p.chunk + PREFIX_ITEM) + cb * (cost + PREFIX_ITEM);
                const int b0 = block_at(from), parts = block_at(from + cost - 1) - b0 + 1, k = (part - before) & (PAR - 1);
                const uint64_t slot0 = (uint64_t)(q.item + (kvh * q.chunks + i) * q.cbs + cb + b0);
                load(k < parts, p.pre_o, p.pre_ml, slot0 + k, p.pre_slots, PCOLS, col % PCOLS, mi[j], li[j], oi[j]);
                for (int more = k + PAR; more < parts; more += PAR) {
                    float mk[1], lk[1];
                    pf32x4 ok[1];
                    load(true, p.pre_o, p.pre_ml, slot0 + more, p.pre_slots, PCOLS, col % PCOLS, mk[0], lk[0], ok[0]);
                    add_parts<1>(m, l, o, mk, lk, ok);
                }
                before += parts;
            }
            add_parts<AHEAD>(m, l, o, mi, li, oi);
        }
        add_parts<2>(m, l, o, mo, lo, oo);
        for (int i = PAR - 1 - part + 2 * PAR; i < q.own_chunks; i += 2 * PAR) {
            load_own(i);
            add_parts<2>(m, l, o, mo, lo, oo);
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
    (void)hipGetLastError();  // report only these launches
    if (head_dim == 128) go_types<128>(p, q_dtype, cache_dtype, s);
    else go_types<64>(p, q_dtype, cache_dtype, s);
    return hipGetLastError();
}

}  // namespace wpcg
