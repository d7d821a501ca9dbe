// The C boundary of the operators of batched serving (include/wpcg.h): paged
// keys and values, attention over them, verification of drafts. Everything a
// kernel indexes with is bounded here or, where it comes from device arrays,
// in the kernels.
#include <algorithm>
#include <cmath>

#include "wpcg_internal.hpp"

namespace wpcg {
namespace {

constexpr int64_t CUS = 256;  // of an MI355X
constexpr uint64_t INT_BOUND = 1u << 30;  // of rows, tokens, heads: sums of two stay ints
constexpr int64_t GROUPS_256 = 1 << 24, GROUPS_512 = 1 << 23;  // workgroups of a launch: its threads fit 32 bits

uint64_t type_size(int dtype) { return dtype == WPCG_DTYPE_F32 ? 4 : dtype == WPCG_DTYPE_BF16 ? 2 : 1; }
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_rows_dtype(int dtype)
{
    if (dtype != WPCG_DTYPE_F32 && dtype != WPCG_DTYPE_BF16) return fail(WPCG_E_ARG, "rows are F32 or BF16");
    return WPCG_OK;
}

// A row stride in elements (0 = packed): at least the row, 16-byte steps.
int row_stride(uint64_t stride, uint64_t width, int dtype, uint64_t* out)
{
    if (stride == 0) stride = width;
    if (stride < width) return fail(WPCG_E_SHAPE, "row stride shorter than the row");
    if (stride * type_size(dtype) % 16 != 0) return fail(WPCG_E_SHAPE, "row stride not a multiple of 16 bytes");
    if (stride >> 40) return fail(WPCG_E_ARG, "row stride too large");
    *out = stride;
    return WPCG_OK;
}

struct Pages {
    uint64_t page, head, token;  // strides
};

int check_pages(const wpcg_kv_pages* kv, Pages* s)
{
    if (!kv) return fail(WPCG_E_ARG, "null pages");
    if (kv->dtype != WPCG_DTYPE_F32 && kv->dtype != WPCG_DTYPE_BF16 && kv->dtype != WPCG_DTYPE_E4M3)
        return fail(WPCG_E_ARG, "pages are F32, BF16 or E4M3");
    if (kv->head_dim != 64 && kv->head_dim != 128) return fail(WPCG_E_UNSUPPORTED, "head_dim is 64 or 128");
    if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
        return fail(WPCG_E_SHAPE, "page_size is a power of two in 16..256");
    if (kv->n_pages == 0 || kv->n_pages > INT_BOUND) return fail(WPCG_E_ARG, "n_pages out of range");
    if (kv->n_kv_heads == 0 || kv->n_kv_heads > 65536) return fail(WPCG_E_ARG, "n_kv_heads out of range");
    if ((kv->k_scale_dev || kv->v_scale_dev) && kv->dtype != WPCG_DTYPE_E4M3)
        return fail(WPCG_E_ARG, "scales are of an E4M3 cache");
    *s = {kv->page_stride, kv->head_stride, kv->token_stride};
    const uint64_t d = kv->head_dim;
    if (!s->page && !s->head && !s->token) {
        s->token = d;
        s->head = d * kv->page_size;
        s->page = s->head * kv->n_kv_heads;
    }
    const uint64_t es = type_size(kv->dtype);
    for (uint64_t x : {s->page, s->head, s->token}) {
        if (x < d) return fail(WPCG_E_SHAPE, "a page stride is shorter than a head");
        if (x * es % 16 != 0) return fail(WPCG_E_SHAPE, "a page stride is not a multiple of 16 bytes");
        if (x >> 40) return fail(WPCG_E_ARG, "a page stride is too large");
    }
    // (a token's place in its page is a 32-bit offset in the kernels)
    if (s->token * es * kv->page_size >> 31) return fail(WPCG_E_ARG, "a page stride is too large");
    return WPCG_OK;
}

int check_batch(const wpcg_kv_batch* b, const wpcg_kv_pages* kv, PagedBatch* out)
{
    if (!b) return fail(WPCG_E_ARG, "null batch");
    if (b->n_seq > INT_BOUND || b->n_rows > INT_BOUND || b->max_q > INT_BOUND || b->max_kv > INT_BOUND)
        return fail(WPCG_E_ARG, "batch bounds out of range");
    if (b->n_seq > 0) {
        if (b->max_q == 0) return fail(WPCG_E_ARG, "max_q is 0");
        if (!b->q_start_dev && (b->max_q != 1 || b->n_rows < b->n_seq))
            return fail(WPCG_E_ARG, "without q_start every sequence has one row");
        if ((uint64_t)b->table_stride * kv->page_size < b->max_kv)
            return fail(WPCG_E_SHAPE, "the table's rows do not hold max_kv tokens");
    }
    int shift = 0;
    while ((1u << shift) < kv->page_size) shift++;
    *out = {(int)b->n_seq, (int)b->n_rows, 0, (int)std::min(b->max_q, b->n_rows), (int)b->max_kv, kv->n_pages,
            (int)kv->page_size, shift, b->table_stride, b->q_start_dev, b->kv_len_dev, b->table_dev};
    return WPCG_OK;
}

// After the checks that need no pointers: what a call must have.
int check_pointers(const wpcg_kv_pages* kv, const wpcg_kv_batch* b)
{
    if (!kv->k_dev || !kv->v_dev || !b->kv_len_dev || (!b->table_dev && b->max_kv > 0))
        return fail(WPCG_E_ARG, "null argument");
    if (!aligned(kv->k_dev) || !aligned(kv->v_dev)) return fail(WPCG_E_ARG, "pages not aligned to 16 bytes");
    return WPCG_OK;
}

// One kernel's part of a call.
struct Plan {
    PagedBatch b;  // with the rows a sequence that it takes
    bool many;
    int cols, col_blocks, blocks, chunk, splits, part_rows, part_seq;
    double us;       // of a workgroup's tiles, by estimate
    uint64_t parts;  // columns whose states the workspace holds
    uint64_t bytes;
};

// Which kernel, and how many workgroups share a sequence's tokens. The bounds
// stand in for the lengths, which only the device knows; a shorter sequence
// just has fewer chunks.
int plan_kernel(const wpcg_kv_pages* kv, const PagedBatch& b, const wpcg_attention* a, Plan* out)
{
    const int64_t group = a->n_heads / kv->n_kv_heads, cols = (int64_t)b.max_q * group;
    // column blocks of all sequences together: each one's last may be a part of one
    const auto all_blocks = [&](int64_t cw) {
        const int64_t seqs = std::min<int64_t>(b.n_seq, b.n_rows / std::max(1, b.min_q));
        return std::min(b.n_seq * ((cols + cw - 1) / cw), (int64_t)b.n_rows * group / cw + seqs);
    };
    Plan p;
    p.b = b;
    p.many = cols > 2 * ATTN_FEW_COLS;
    const int64_t tw = p.many ? ATTN_MANY_TILE : ATTN_FEW_TILE;
    // tiles that a block of cw columns can see
    const auto tiles_of = [&](int64_t cw) {
        const int64_t all = (b.max_kv + tw - 1) / tw;
        if (a->window == 0) return all;
        const int64_t rows = std::min<int64_t>(b.max_q, cw / group + 2);
        const int64_t seen = (std::min<int64_t>(a->sinks, b.max_kv) + tw - 1) / tw +
                             ((int64_t)std::min<uint64_t>(a->window, INT_BOUND) + rows + tw - 1) / tw + 1;
        return std::min(all, seen);
    };
    if (p.many) {
        // 256 columns a workgroup where that leaves every CU one and a block has
        // tiles enough; over E4M3 more of them, where the narrower form's registers
        // suffice. With 128 and 256 columns, us, one card, one run: two prompts of up
        // to 5000, 32 / 4 heads, by the window:
        //   window        256      512      1024     1500     2048     4000
        //   tiles           7       11        19       26       35       66
        //   BF16        132 125  170 159   249 231  309 294  381 359  553 512
        //   E4M3        115 122  150 155   227 226  287 288  355 351  522 500
        // 32 / 8 heads without one: a prompt of 4096 (64 tiles) BF16 167 and 156, E4M3
        // 161 and 153; eight of up to 1000 (16 tiles) 111 and 105, 99 and 103; the
        // last 2048 rows of 32768 tokens 1121 and 976, 1018 and 948. (BF16 with many
        // blocks gains below its 16 tiles too.)
        const int64_t wide = 2 * ATTN_MANY_COLS, some = kv->dtype == WPCG_DTYPE_E4M3 ? 32 : 16;
        p.cols = a->dtype == WPCG_DTYPE_BF16 && tiles_of(wide) >= some && kv->n_kv_heads * all_blocks(wide) >= CUS
                     ? wide : ATTN_MANY_COLS;
    } else {
        // (over an F32 cache the wider form's registers do not suffice)
        p.cols = cols > ATTN_FEW_COLS && kv->dtype != WPCG_DTYPE_F32 ? 2 * ATTN_FEW_COLS : ATTN_FEW_COLS;
    }
    const int64_t blocks = (cols + p.cols - 1) / p.cols, tiles = tiles_of(p.cols);
    // Workgroups of the many-row kernel look for their work where that saves
    // half of them, for empty ones are not free: 255 sequences of 512 tokens
    // with one new row each and a prompt of 1024, 32 / 8 heads, 223 us without,
    // 154 so; 63 of 2048 and a prompt of 2048 282 and 170
    const bool look = p.many && b.n_seq * blocks > 2 * all_blocks(p.cols);
    const int64_t base = kv->n_kv_heads * (look ? all_blocks(p.cols) : b.n_seq * blocks);
    // The cheapest split by this estimate, in microseconds: workgroups run in
    // rounds of those the chip holds; each has 4 us of start and end and its
    // tiles, and a split one a second launch of 5 us. A tile of the few-row
    // kernel takes what its bytes take at 20 GB/s, a CU's share of the memory's
    // rate, and about what it gets with half of them idle too (64000 tokens of
    // BF16 on 128 workgroups: 100 us, 2.6 TB/s; on 256: 53 us); of the many-row
    // kernel what its products take.
    const bool two = p.many && p.cols == ATTN_MANY_COLS && a->dtype == WPCG_DTYPE_BF16;  // workgroups on a CU
    const int64_t room = two ? 2 * CUS : CUS;
    const double tile = p.many ? (a->dtype == WPCG_DTYPE_BF16 ? 2.4 : kv->dtype == WPCG_DTYPE_F32 ? 6.0 : 3.5) *
                                     (kv->head_dim / 128.0)
                               : 2.0 * tw * kv->head_dim * type_size(kv->dtype) / 20480.0;
    // Without a window a prompt's first blocks see fewest tiles and run last, so
    // that where there are more workgroups than room the sum of their tiles
    // counts (1500 rows in fp32 over BF16, 32 / 4 heads, 376 blocks of 1 to 24
    // tiles: 129 us in equal rounds' split, 81 whole). The many-row kernel's
    // parts are written and read again, at 4 TB/s.
    const int64_t unseen = p.many && a->window == 0 ? std::max<int64_t>(0, b.max_q - p.cols / group) : 0;
    const int64_t lowest = std::max<int64_t>(1, tiles - unseen / tw);
    const double mean = (tiles + lowest) / 2.0;
    const auto cost = [&](int64_t s) {
        const int64_t chunk = (tiles + s - 1) / s;
        // chunks of all blocks of 1 .. t tiles
        const auto chunks = [&](int64_t t) { return (double)chunk * (t / chunk) * (t / chunk + 1) / 2 + (double)(t % chunk) * (t / chunk + 1); };
        const double parts = (chunks(tiles) - chunks(lowest - 1)) / (tiles - lowest + 1);
        double join = s > 1 ? 5.0 : 0.0;
        if (p.many && s > 1) join += base * p.cols * parts * (kv->head_dim + 2) * 8.0 / 4e6;
        if (unseen > 0 && base * parts > room)
            return base * (parts * 4.0 + mean * tile) / room + 0.5 * (s == 1 ? lowest : chunk) * tile + join;
        const int64_t rounds = ((int64_t)(base * parts) + room - 1) / room;
        return rounds * (4.0 + chunk * tile) + join;
    };
    const int64_t least = p.many ? 2 : ATTN_FEW_WAVES;  // tiles of a chunk
    int64_t best = 1;
    for (int64_t s = 2; base > 0 && s <= tiles / least && base * s <= 4 * room; s++)
        if (cost(s) < cost(best)) best = s;
    p.chunk = (int)std::max<int64_t>(1, (tiles + best - 1) / best);
    p.splits = (int)std::max<int64_t>(1, (tiles + p.chunk - 1) / p.chunk);
    p.us = p.chunk * tile;
    p.blocks = look ? (int)all_blocks(p.cols) : 0;
    // Rows that the sequences can have: n_rows may be a looser bound. The blocks'
    // columns are as many at least, so that parts are 4 * room * cols at most.
    const int64_t seq_rows = (int64_t)b.n_seq * b.max_q;
    p.part_seq = seq_rows < b.n_rows ? b.max_q : 0;
    p.part_rows = (int)std::min<int64_t>(seq_rows, b.n_rows);
    p.parts = p.splits == 1 ? 0
              : p.many      ? (uint64_t)p.splits * p.part_rows * a->n_heads
                            : (uint64_t)p.splits * base * p.cols;
    // A chunk that long may be one sequence's alone while the others' are
    // empty, for the bounds do not tell: all tiles are dealt out evenly
    // instead. (63 sequences of 500 tokens and one of 100000, 32 / 4 heads: 1028
    // us with a workgroup a sequence and head, 79 so. It costs a few us more
    // where the lengths are less unlike: 64 sequences of 512 to 4096 tokens 67
    // and 75 us. The border between these was not looked for more closely.)
    if (!p.many && p.us > 130.0 && b.n_seq <= ATTN_DEAL_SEQS && base * tiles < (int64_t)1 << 30) {
        p.blocks = CUS;
        p.parts = 2 * CUS * p.cols;
        p.splits = 1;
    }
    p.col_blocks = (int)std::max<int64_t>(1, blocks);
    // (a batch that is split has few workgroups, and its join few rows)
    if (base * p.splits >= GROUPS_512)
        return fail(WPCG_E_UNSUPPORTED, "the batch needs too many workgroups");
    p.bytes = p.parts * (kv->head_dim + 2) * sizeof(float) + (p.many ? 0 : p.blocks * sizeof(AttnEnd));
    *out = p;
    return WPCG_OK;
}

struct Plans {
    Plan part[2];
    int n;
    uint64_t bytes;  // they share the workspace: one runs behind the other
};

// A batch that may hold prompts and single tokens or drafts is two parts where
// the tokens may be many: the few-row kernel shares a long sequence's tokens out
// over the chip, the many-row one leaves them to a workgroup or few. Sequences
// with one new row each beside one prompt, 32 / 8 heads, by the many-row kernel
// alone and in two parts: 3 of 100000 tokens and a prompt of 2048 656 and 314
// us, 63 of 4096 and 512 224 and 216, 63 of 2048 and 2048 (a workgroup's tiles
// 77 us) 170 and 172.
int plan_attention(const wpcg_kv_pages* kv, const PagedBatch& b, const wpcg_attention* a, Plans* out)
{
    out->n = 1;
    if (int rc = plan_kernel(kv, b, a, &out->part[0])) return rc;
    const int64_t few = 2 * ATTN_FEW_COLS / (a->n_heads / kv->n_kv_heads);  // rows that the few-row kernel takes
    const int64_t all = (int64_t)b.n_seq * b.max_q;
    if (out->part[0].many && few > 0 && b.n_seq > 1 && b.n_rows <= all - b.max_q + few && out->part[0].us > 100.0) {
        PagedBatch part[2] = {b, b};
        part[0].max_q = (int)few;
        part[1].min_q = (int)few + 1;
        out->n = 2;
        for (int i = 0; i < 2; i++)
            if (int rc = plan_kernel(kv, part[i], a, &out->part[i])) return rc;
    }
    out->bytes = 0;
    for (int i = 0; i < out->n; i++) out->bytes = std::max(out->bytes, out->part[i].bytes);
    return WPCG_OK;
}

// A batch whose groups share prefixes: how the tiles are dealt out, and the plans
// of the batch without sharing, where that is what it takes.
struct PrefixPlan {
    bool shared;
    Plans plain;
    PrefixArgs args;  // its weights, chunks, blocks, columns and places for parts
    uint64_t bytes;
};
int plan_prefix(const wpcg_kv_pages* kv, const PagedBatch& b, const wpcg_kv_prefix* x, const wpcg_attention* a,
                PrefixPlan* out)
{
    PrefixPlan& o = *out;
    o = {};
    const int64_t group = a->n_heads / kv->n_kv_heads, cols = (int64_t)b.max_q * group, n_kv = kv->n_kv_heads;
    const int64_t max_prefix = std::min<int64_t>(x->max_prefix, b.max_kv), groups = x->n_groups;
    const int64_t rows = std::min<int64_t>(b.n_rows, (int64_t)b.n_seq * b.max_q);
    const int64_t cw = ATTN_MANY_COLS, tiles = (max_prefix + ATTN_MANY_TILE - 1) / ATTN_MANY_TILE;
    const int64_t blocks = std::min(groups * ((rows * group + cw - 1) / cw), rows * group / cw + groups);
    const int64_t own_cols = cols > ATTN_FEW_COLS && kv->dtype != WPCG_DTYPE_F32 ? 2 * ATTN_FEW_COLS : ATTN_FEW_COLS;
    const int64_t own_blocks = (cols + own_cols - 1) / own_cols, own_tiles = (b.max_kv + ATTN_FEW_TILE - 1) / ATTN_FEW_TILE;
    PrefixArgs& p = o.args;
    // Chunks keep the column blocks' workgroups at keys and values that one die's L2
    // holds; each makes a part more to join: four of a long prefix. (32 / 8 heads, 65536
    // tokens, one column block: 16 chunks 125 us, 4 chunks 120.)
    p.chunk = (int)std::max<int64_t>(64, (tiles + 3) / 4);
    const int64_t chunks = (tiles + p.chunk - 1) / p.chunk;
    const double cost = (double)n_kv * (blocks * (tiles + chunks * PREFIX_ITEM) +
                                        b.n_seq * own_blocks * (own_tiles + OWN_ITEM));
    // Without sharing a prefix comes out of the caches for all sequences but the first,
    // at some 11 TB/s, and the fixed costs are lower: it pays from a number of bytes on
    // that are read again. Shared and not, us, one group's prefix and up to 200 own tokens;
    // read again, MB (sequences x rows; heads of 128 but for 14 / 2):
    //                                     120     250     450     700     1000
    //   BF16 queries
    //     BF16 cache, 32 / 4, 64 x 1    33 16   35 25   35 38   38 68   41  89
    //                 14 / 2, 64 x 1    24 21   26 31   30 48   34 76   43  99
    //                 32 / 8, 16 x 5    36 25   39 34   45 49   56 86   65 104
    //     E4M3        32 / 8, 32 x 1    30 19   31 30   34 45   35 79   39 104
    //   F32 queries
    //     BF16 cache, 32 / 8, 32 x 1    44 18   44 28   46 43   47 74   48  95
    //                 14 / 2, 64 x 1    34 22   36 32   42 47   48 76   56 100
    //                 32 / 8, 16 x 5    51 30   56 42   69 64   84 102 104 131
    //     E4M3        32 / 8, 32 x 1    45 23   46 38   48 58   50 101  58 134
    //     F32         32 / 8, 32 x 1    68 27   70 38   70 54   71 93   72 119
    //                 14 / 2, 64 x 1    43 24   45 34   47 48   52 80   58 104
    // One bound for a pair of types, so that some batches near it take up to 10 us longer
    // than the other way would (BF16, 32 / 4 heads, 250 to 400; F32 cache, 14 / 2, 450 to
    // 700). (36316 tokens, 22 rows of which see the last 106: 44 us and 9.)
    const int64_t seen = a->window > 0 ? std::min<int64_t>(max_prefix, (int64_t)a->window + a->sinks + b.max_q) : max_prefix;
    const double again = (double)(b.n_seq - groups) * seen * 2 * n_kv * kv->head_dim * type_size(kv->dtype) / 1e6;
    const double pays = a->dtype == WPCG_DTYPE_BF16 ? 250 : kv->dtype == WPCG_DTYPE_F32 ? 700 : 450;
    o.shared = rows > 0 && cols <= 2 * ATTN_FEW_COLS && groups > 0 && groups < b.n_seq && groups <= PREFIX_GROUPS &&
               b.n_seq <= PREFIX_SEQS && again >= pays && cost < (double)(1 << 30) &&
               (double)b.n_seq * b.max_q * a->n_heads * kv->head_dim < 256.0 * GROUPS_256;  // the join's workgroups
    if (!o.shared) {
        if (int rc = plan_attention(kv, b, a, &o.plain)) return rc;
        o.bytes = o.plain.bytes;
        return WPCG_OK;
    }
    p.n_groups = (int)groups;
    p.max_prefix = (int)max_prefix;
    const bool bf16 = a->dtype == WPCG_DTYPE_BF16;
    p.a.blocks = bf16 ? 2 * CUS : CUS;
    p.first = bf16 ? CUS / 8 : 0;
    p.a.cols = (int)own_cols;
    p.pre_slots = (uint64_t)(n_kv * blocks * chunks + p.a.blocks);
    p.own_slots = (uint64_t)(n_kv * own_blocks * b.n_seq + 4 * (p.a.blocks - 8 * p.first));
    o.bytes = (p.pre_slots * cw + p.own_slots * own_cols) * (kv->head_dim + 2) * sizeof(float) +
              b.n_seq * sizeof(PrefixSeq) + sizeof(PrefixDeal);
    return WPCG_OK;
}

// The scores' factor in base 2.
float scale_log2(const wpcg_attention* a) { return (float)((double)a->scale * 1.4426950408889634); }

int check_attention(const wpcg_kv_pages* kv, const wpcg_attention* a)
{
    if (!a) return fail(WPCG_E_ARG, "null argument");
    if (int rc = check_rows_dtype(a->dtype)) return rc;
    if (a->dtype == WPCG_DTYPE_BF16 && kv->dtype == WPCG_DTYPE_F32)
        return fail(WPCG_E_UNSUPPORTED, "BF16 queries take a BF16 or E4M3 cache");
    if (a->n_heads == 0 || a->n_heads > 65536 || a->n_heads % kv->n_kv_heads)
        return fail(WPCG_E_SHAPE, "n_heads is a multiple of n_kv_heads");
    if (!(a->scale > 0.0f) || !std::isfinite(scale_log2(a))) return fail(WPCG_E_ARG, "scale is positive, and finite times log2 e");
    return WPCG_OK;
}

int check_prefix(const wpcg_kv_prefix* x)
{
    if (!x) return fail(WPCG_E_ARG, "null argument");
    if (x->n_groups > INT_BOUND || x->max_prefix > INT_BOUND) return fail(WPCG_E_ARG, "prefix bounds out of range");
    return WPCG_OK;
}

// What a call of attention has checked, without its plan and workspace.
int attention_ready(wpcg_ctx* ctx, const wpcg_kv_pages* kv, const wpcg_kv_batch* batch, const wpcg_attention* att,
                    uint64_t bytes, const void* ws, uint64_t ws_bytes)
{
    if (int rc = check_pointers(kv, batch)) return rc;
    if (!att->q_dev || !att->out_dev) return fail(WPCG_E_ARG, "null argument");
    if (!aligned(att->q_dev) || !aligned(att->out_dev)) return fail(WPCG_E_ARG, "rows not aligned to 16 bytes");
    if (bytes) {
        if (!ws || ws_bytes < bytes)
            return fail(WPCG_E_ARG, "the call needs " + std::to_string(bytes) + " bytes of workspace");
        if (!aligned(ws)) return fail(WPCG_E_ARG, "workspace not aligned to 16 bytes");
    }
    return check_ctx(ctx);
}
// A call's arguments for the kernels, without its plan; a.b is there.
int attention_args(const wpcg_kv_pages* kv, const Pages& st, const wpcg_attention* att, PagedAttnArgs& a)
{
    const uint64_t width = (uint64_t)att->n_heads * kv->head_dim;
    if (int rc = row_stride(att->q_stride, width, att->dtype, &a.q_row)) return rc;
    if (int rc = row_stride(att->out_stride, width, att->dtype, &a.out_row)) return rc;
    a.q = att->q_dev;
    a.out = att->out_dev;
    a.k = kv->k_dev;
    a.v = kv->v_dev;
    a.page_stride = st.page;
    a.head_stride = st.head;
    a.token_stride = st.token;
    a.k_scale = kv->k_scale_dev;
    a.v_scale = kv->v_scale_dev;
    a.n_heads = (int)att->n_heads;
    a.n_kv = (int)kv->n_kv_heads;
    a.group = a.n_heads / a.n_kv;
    a.scale = scale_log2(att);
    a.window = (int)std::min<uint64_t>(att->window, INT_BOUND);
    a.sinks = (int)std::min<uint64_t>(att->sinks, INT_BOUND);
    return WPCG_OK;
}
int run_plans(PagedAttnArgs a, const Plans& plan, const wpcg_kv_pages* kv, const wpcg_attention* att, void* ws,
              hipStream_t s)
{
    const int d = (int)kv->head_dim;
    for (int i = 0; i < plan.n; i++) {
        const Plan& p = plan.part[i];
        a.b = p.b;
        a.cols = p.cols;
        a.col_blocks = p.col_blocks;
        a.blocks = p.blocks;
        a.chunk = p.chunk;
        a.splits = p.splits;
        a.part_rows = p.part_rows;
        a.part_seq = p.part_seq;
        a.part_o = (float*)ws;
        a.part_ml = a.part_o + p.parts * kv->head_dim;
        a.ends = (AttnEnd*)(a.part_ml + p.parts * 2);
        WPCG_HIP(p.many ? launch_attn_many(a, d, att->dtype, kv->dtype, s)
                        : launch_attn_few(a, d, att->dtype, kv->dtype, s));
    }
    return WPCG_OK;
}

int check_draft(const wpcg_draft* d, int* chunks, uint64_t* bytes)
{
    if (!d) return fail(WPCG_E_ARG, "null argument");
    if (d->vocab == 0 || d->vocab > INT_BOUND) return fail(WPCG_E_ARG, "vocab out of range");
    if (d->n_seq > INT_BOUND || d->n_rows > INT_BOUND) return fail(WPCG_E_ARG, "batch bounds out of range");
    if (d->n_seq > 0) {
        if (d->max_rows == 0 || d->max_rows > WPCG_DRAFT_MAX)
            return fail(WPCG_E_ARG, "max_rows is in 1.." + std::to_string(WPCG_DRAFT_MAX));
        if (!d->q_start_dev && (uint64_t)d->n_seq * d->max_rows > d->n_rows)
            return fail(WPCG_E_ARG, "without q_start every sequence has max_rows rows");
    }
    if ((d->logits_stride && d->logits_stride < d->vocab) || (d->draft_stride && d->draft_stride < d->vocab))
        return fail(WPCG_E_SHAPE, "row stride shorter than the row");
    if (d->logits_stride >> 40 || d->draft_stride >> 40) return fail(WPCG_E_ARG, "row stride too large");
    *chunks = (int)((d->vocab + DRAFT_CHUNK - 1) / DRAFT_CHUNK);
    if ((uint64_t)std::max(d->n_rows, d->n_seq) * ((*chunks + 3) / 4) >= (uint64_t)GROUPS_256)
        return fail(WPCG_E_UNSUPPORTED, "the batch needs too many workgroups");
    *bytes = (uint64_t)d->n_rows * *chunks * sizeof(DraftPart) + (uint64_t)d->n_seq * *chunks * sizeof(double) +
             (uint64_t)d->n_seq * sizeof(DraftDone);
    return WPCG_OK;
}

// The blocks that pages are counted in, and what a call needs in device memory.
int check_pool(const wpcg_kv_pool* p, PoolArgs* out, int* blocks)
{
    if (!p) return fail(WPCG_E_ARG, "null argument");
    if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
        return fail(WPCG_E_SHAPE, "page_size is a power of two in 16..256");
    if (p->n_pages == 0 || p->n_pages > 1u << 26) return fail(WPCG_E_ARG, "n_pages out of range");
    if (p->n_seq > INT_BOUND || p->table_stride == 0 || (uint64_t)p->n_seq * p->table_stride > INT_BOUND ||
        (uint64_t)p->table_stride * p->page_size > INT_BOUND)
        return fail(WPCG_E_ARG, "table out of range");
    int shift = 0;
    while ((1u << shift) < p->page_size) shift++;
    *out = {(int)p->n_pages, (int)p->page_size, shift, (int)p->n_seq, (int)p->table_stride, p->refs_dev, p->table_dev,
            p->kv_len_dev};
    *blocks = (out->n_pages + POOL_BLOCK - 1) / POOL_BLOCK;
    // workgroups of 1024 threads: a row's 1024 entries, a block of pages
    if ((uint64_t)p->n_seq * ((p->table_stride + 1023) / 1024) + *blocks >= 1u << 22)
        return fail(WPCG_E_UNSUPPORTED, "the pool needs too many workgroups");
    return WPCG_OK;
}
int pool_ready(const wpcg_kv_pool* p, const void* result, const void* ws, uint64_t ws_bytes, uint64_t bytes)
{
    if (!p->refs_dev || (p->n_seq > 0 && (!p->table_dev || !p->kv_len_dev)) || !result)
        return fail(WPCG_E_ARG, "null argument");
    if (!ws || ws_bytes < bytes)
        return fail(WPCG_E_ARG, "the call needs " + std::to_string(bytes) + " bytes of workspace");
    if (!aligned(ws)) return fail(WPCG_E_ARG, "workspace not aligned to 16 bytes");
    return WPCG_OK;
}
// The parts of a workspace, one behind the other.
struct Parts {
    uint8_t* at;
    uint64_t used = 0;
    template <class T>
    T* take(uint64_t n)
    {
        T* r = (T*)(at + used);
        used += (n * sizeof(T) + 15) / 16 * 16;
        return r;
    }
};
uint64_t fork_parts(ForkArgs* a, int blocks, void* ws)
{
    Parts w{(uint8_t*)ws};
    a->blocks = blocks;
    a->writers = w.take<ForkWriters>(a->p.n_pages);
    a->rows = w.take<ForkRow>(a->p.n_seq);
    a->tail = w.take<int>(a->p.n_seq);
    a->kept = w.take<int>((uint64_t)a->p.n_seq * a->p.stride);
    a->count = w.take<int>(blocks);
    a->totals = w.take<int>(2);
    return w.used;
}
uint64_t compact_parts(CompactArgs* a, int blocks, void* ws)
{
    Parts w{(uint8_t*)ws};
    a->blocks = blocks;
    a->count = w.take<int>(blocks);
    a->total = w.take<int>(1);
    a->rank = w.take<int>(a->p.n_pages);
    a->used = w.take<int>(a->p.n_pages);
    a->free = w.take<int>(a->p.n_pages);
    return w.used;
}

int check_logprobs(const wpcg_logprob* d, int* chunks, uint64_t* part_bytes, uint64_t* bytes)
{
    if (!d) return fail(WPCG_E_ARG, "null argument");
    if (int rc = check_rows_dtype(d->dtype)) return rc;
    if (d->vocab == 0 || d->vocab > INT_BOUND) return fail(WPCG_E_ARG, "vocab out of range");
    if (d->n_rows > INT_BOUND) return fail(WPCG_E_ARG, "batch bounds out of range");
    if (d->top > WPCG_LOGPROB_TOP) return fail(WPCG_E_ARG, "top is at most " + std::to_string(WPCG_LOGPROB_TOP));
    if (d->logits_stride && d->logits_stride < d->vocab) return fail(WPCG_E_SHAPE, "row stride shorter than the row");
    if (d->logits_stride >> 40) return fail(WPCG_E_ARG, "row stride too large");
    // (a row that does not start on 16 bytes has up to seven places before it)
    const uint64_t per = 16 / type_size(d->dtype), stride = d->logits_stride ? d->logits_stride : d->vocab;
    *chunks = (int)((d->vocab + (stride % per ? per - 1 : 0) + LOGPROB_CHUNK - 1) / LOGPROB_CHUNK);
    if ((uint64_t)d->n_rows * ((*chunks + 3) / 4) >= (uint64_t)GROUPS_256)
        return fail(WPCG_E_UNSUPPORTED, "the batch needs too many workgroups");
    const uint64_t all = (uint64_t)d->n_rows * *chunks;
    *part_bytes = (all * sizeof(LogprobPart) + 15) / 16 * 16;
    *bytes = *part_bytes + (d->top > 0 ? all * LOGPROB_SEGS * sizeof(float) : 0);
    return WPCG_OK;
}

}  // namespace
}  // namespace wpcg

using namespace wpcg;

extern "C" {

int wpcg_kv_append(wpcg_ctx* ctx, const wpcg_kv_pages* kv, const wpcg_kv_batch* batch, const wpcg_kv_rows* r,
                   wpcg_stream stream)
{
    Pages st;
    if (int rc = check_pages(kv, &st)) return rc;
    KvAppendArgs a{};
    if (int rc = check_batch(batch, kv, &a.b)) return rc;
    if (!r) return fail(WPCG_E_ARG, "null argument");
    if (int rc = check_rows_dtype(r->dtype)) return rc;
    const bool with_q = r->q_dev || r->q_out_dev;
    const uint64_t d = kv->head_dim;
    if (with_q) {
        if (int rc = check_rows_dtype(r->q_out_dtype)) return rc;
        if (r->n_heads == 0 || r->n_heads > 65536 || r->n_heads % kv->n_kv_heads)
            return fail(WPCG_E_SHAPE, "n_heads is a multiple of n_kv_heads");
        if (int rc = row_stride(r->q_stride, r->n_heads * d, r->dtype, &a.q_row)) return rc;
        if (int rc = row_stride(r->q_out_stride, r->n_heads * d, r->q_out_dtype, &a.q_out_row)) return rc;
        if (r->q_dev == r->q_out_dev && (r->dtype != r->q_out_dtype || a.q_row != a.q_out_row))
            return fail(WPCG_E_ARG, "q_out may be q itself only in q's type and stride");
    }
    if (int rc = row_stride(r->k_stride, kv->n_kv_heads * d, r->dtype, &a.k_row)) return rc;
    if (int rc = row_stride(r->v_stride, kv->n_kv_heads * d, r->dtype, &a.v_row)) return rc;
    if ((r->q_norm_dev || r->k_norm_dev) && !(r->eps >= 0.0f)) return fail(WPCG_E_ARG, "eps is not negative");
    a.n_q = with_q ? (int)r->n_heads : 0;
    a.n_kv = (int)kv->n_kv_heads;
    a.n_units = a.n_q + 2 * a.n_kv;
    const uint64_t per = 2048 / d;  // heads of a workgroup
    if ((uint64_t)batch->n_rows * ((a.n_units + per - 1) / per) >= (uint64_t)GROUPS_256)
        return fail(WPCG_E_UNSUPPORTED, "the batch needs too many workgroups");
    if (batch->n_seq == 0 || batch->n_rows == 0) return check_ctx(ctx);
    if (int rc = check_pointers(kv, batch)) return rc;
    if ((with_q && (!r->q_dev || !r->q_out_dev)) || !r->k_dev || !r->v_dev) return fail(WPCG_E_ARG, "null argument");
    for (const void* x : {r->q_dev, (const void*)r->q_out_dev, r->k_dev, r->v_dev, (const void*)r->q_norm_dev,
                          (const void*)r->k_norm_dev})
        if (!aligned(x)) return fail(WPCG_E_ARG, "rows or weights not aligned to 16 bytes");
    if (int rc = check_ctx(ctx)) return rc;
    a.q = r->q_dev;
    a.k = r->k_dev;
    a.v = r->v_dev;
    a.q_out = r->q_out_dev;
    a.q_out_dtype = r->q_out_dtype;
    a.k_pages = kv->k_dev;
    a.v_pages = kv->v_dev;
    a.cache_dtype = kv->dtype;
    a.page_stride = st.page;
    a.head_stride = st.head;
    a.token_stride = st.token;
    a.k_scale = kv->k_scale_dev;
    a.v_scale = kv->v_scale_dev;
    a.q_norm = r->q_norm_dev;
    a.k_norm = r->k_norm_dev;
    a.freq = r->freq_dev;
    a.eps = r->eps;
    WPCG_HIP(launch_kv_append(a, (int)d, r->dtype == WPCG_DTYPE_BF16, pick(ctx, stream)));
    return WPCG_OK;
}

int wpcg_paged_attention_workspace(const wpcg_kv_pages* kv, const wpcg_kv_batch* batch, const wpcg_attention* att,
                                   uint64_t* bytes)
{
    if (!bytes) return fail(WPCG_E_ARG, "null output");
    *bytes = 0;
    Pages st;
    if (int rc = check_pages(kv, &st)) return rc;
    PagedBatch b;
    if (int rc = check_batch(batch, kv, &b)) return rc;
    if (int rc = check_attention(kv, att)) return rc;
    Plans plan;
    if (int rc = plan_attention(kv, b, att, &plan)) return rc;
    *bytes = plan.bytes;
    return WPCG_OK;
}

int wpcg_paged_attention(wpcg_ctx* ctx, const wpcg_kv_pages* kv, const wpcg_kv_batch* batch, const wpcg_attention* att,
                         void* ws_dev, uint64_t ws_bytes, wpcg_stream stream)
{
    Pages st;
    if (int rc = check_pages(kv, &st)) return rc;
    PagedAttnArgs a{};
    if (int rc = check_batch(batch, kv, &a.b)) return rc;
    if (int rc = check_attention(kv, att)) return rc;
    if (int rc = attention_args(kv, st, att, a)) return rc;
    Plans plan;
    if (int rc = plan_attention(kv, a.b, att, &plan)) return rc;
    if (batch->n_seq == 0 || batch->n_rows == 0) return check_ctx(ctx);
    if (int rc = attention_ready(ctx, kv, batch, att, plan.bytes, ws_dev, ws_bytes)) return rc;
    return run_plans(a, plan, kv, att, ws_dev, pick(ctx, stream));
}

int wpcg_prefix_attention_workspace(const wpcg_kv_pages* kv, const wpcg_kv_batch* batch, const wpcg_kv_prefix* prefix,
                                    const wpcg_attention* att, uint64_t* bytes)
{
    if (!bytes) return fail(WPCG_E_ARG, "null output");
    *bytes = 0;
    Pages st;
    if (int rc = check_pages(kv, &st)) return rc;
    PagedBatch b;
    if (int rc = check_batch(batch, kv, &b)) return rc;
    if (int rc = check_prefix(prefix)) return rc;
    if (int rc = check_attention(kv, att)) return rc;
    PrefixPlan plan;
    if (int rc = plan_prefix(kv, b, prefix, att, &plan)) return rc;
    *bytes = plan.bytes;
    return WPCG_OK;
}

int wpcg_prefix_attention(wpcg_ctx* ctx, const wpcg_kv_pages* kv, const wpcg_kv_batch* batch,
                          const wpcg_kv_prefix* prefix, const wpcg_attention* att, void* ws_dev, uint64_t ws_bytes,
                          wpcg_stream stream)
{
    Pages st;
    if (int rc = check_pages(kv, &st)) return rc;
    PagedAttnArgs a{};
    if (int rc = check_batch(batch, kv, &a.b)) return rc;
    if (int rc = check_prefix(prefix)) return rc;
    if (int rc = check_attention(kv, att)) return rc;
    if (int rc = attention_args(kv, st, att, a)) return rc;
    PrefixPlan plan;
    if (int rc = plan_prefix(kv, a.b, prefix, att, &plan)) return rc;
    if (batch->n_seq == 0 || batch->n_rows == 0) return check_ctx(ctx);
    if (prefix->n_groups > 0 && (!prefix->group_start_dev || !prefix->prefix_len_dev))
        return fail(WPCG_E_ARG, "null argument");
    if (int rc = attention_ready(ctx, kv, batch, att, plan.bytes, ws_dev, ws_bytes)) return rc;
    const hipStream_t s = pick(ctx, stream);
    if (!plan.shared) return run_plans(a, plan.plain, kv, att, ws_dev, s);
    PrefixArgs& p = plan.args;
    const uint64_t d = kv->head_dim, own = p.own_slots * p.a.cols, pre = p.pre_slots * ATTN_MANY_COLS;
    a.cols = p.a.cols;
    a.blocks = p.a.blocks;
    a.part_o = (float*)ws_dev;
    p.pre_o = a.part_o + own * d;
    a.part_ml = p.pre_o + pre * d;
    p.pre_ml = a.part_ml + own * 2;
    p.seqs = (PrefixSeq*)(p.pre_ml + pre * 2);
    p.deal = (PrefixDeal*)(p.seqs + a.b.n_seq);
    p.a = a;
    p.group_start = prefix->group_start_dev;
    p.prefix_len = prefix->prefix_len_dev;
    WPCG_HIP(launch_attn_prefix(p, (int)kv->head_dim, att->dtype, kv->dtype, s));
    return WPCG_OK;
}

int wpcg_draft_verify_workspace(const wpcg_draft* d, uint64_t* bytes)
{
    if (!bytes) return fail(WPCG_E_ARG, "null output");
    *bytes = 0;
    int chunks;
    return check_draft(d, &chunks, bytes);
}

int wpcg_draft_verify(wpcg_ctx* ctx, const wpcg_draft* d, void* ws_dev, uint64_t ws_bytes, wpcg_stream stream)
{
    DraftArgs a{};
    uint64_t bytes = 0;
    if (int rc = check_draft(d, &a.chunks, &bytes)) return rc;
    if (d->n_seq == 0) return check_ctx(ctx);
    if (!d->accepted_dev) return fail(WPCG_E_ARG, "null argument");
    if (d->n_rows > 0) {
        if (!d->logits_dev || !d->tokens_dev || !d->u_dev || !d->u_next_dev || !d->out_dev)
            return fail(WPCG_E_ARG, "null argument");
        if (!ws_dev || ws_bytes < bytes)
            return fail(WPCG_E_ARG, "the call needs " + std::to_string(bytes) + " bytes of workspace");
        if (!aligned(ws_dev)) return fail(WPCG_E_ARG, "workspace not aligned to 16 bytes");
    }
    if (int rc = check_ctx(ctx)) return rc;
    a.n_seq = (int)d->n_seq;
    a.n_rows = (int)d->n_rows;
    a.max_rows = (int)d->max_rows;
    a.vocab = (int)d->vocab;
    a.q_start = d->q_start_dev;
    a.logits = d->logits_dev;
    a.logits_row = d->logits_stride ? d->logits_stride : d->vocab;
    a.probs = d->draft_probs_dev;
    a.probs_row = d->draft_stride ? d->draft_stride : d->vocab;
    a.tokens = d->tokens_dev;
    a.u = d->u_dev;
    a.u_next = d->u_next_dev;
    a.temperature = d->temperature_dev;
    a.accepted = d->accepted_dev;
    a.out = d->out_dev;
    a.part = (DraftPart*)ws_dev;
    a.rest = (double*)(a.part + (uint64_t)d->n_rows * a.chunks);
    a.done = (DraftDone*)(a.rest + (uint64_t)d->n_seq * a.chunks);
    a.vec = aligned(a.logits) && a.logits_row % 4 == 0 && aligned(a.probs) && a.probs_row % 4 == 0;
    WPCG_HIP(launch_draft_verify(a, pick(ctx, stream)));
    return WPCG_OK;
}

int wpcg_kv_fork_workspace(const wpcg_kv_pool* pool, uint64_t* bytes)
{
    if (!bytes) return fail(WPCG_E_ARG, "null output");
    *bytes = 0;
    ForkArgs a{};
    int blocks;
    if (int rc = check_pool(pool, &a.p, &blocks)) return rc;
    *bytes = fork_parts(&a, blocks, nullptr);
    return WPCG_OK;
}

int wpcg_kv_fork(wpcg_ctx* ctx, const wpcg_kv_pool* pool, const wpcg_kv_change* c, void* ws_dev, uint64_t ws_bytes,
                 wpcg_stream stream)
{
    ForkArgs a{};
    int blocks;
    if (int rc = check_pool(pool, &a.p, &blocks)) return rc;
    if (!c) return fail(WPCG_E_ARG, "null argument");
    if (int rc = pool_ready(pool, c->result_dev, ws_dev, ws_bytes, fork_parts(&a, blocks, ws_dev))) return rc;
    if (pool->n_seq > 0 && !c->copies_dev) return fail(WPCG_E_ARG, "null argument");
    if (int rc = check_ctx(ctx)) return rc;
    a.parent = c->parent_dev;
    a.keep = c->keep_dev;
    a.grow = c->grow_dev;
    a.grow_all = (int)std::min<uint64_t>(c->grow, INT_BOUND);
    a.window = (int)std::min<uint64_t>(c->window, INT_BOUND);
    a.sinks = (int)std::min<uint64_t>(c->sinks, INT_BOUND);
    a.copies = c->copies_dev;
    a.result = c->result_dev;
    WPCG_HIP(launch_kv_fork(a, pick(ctx, stream)));
    return WPCG_OK;
}

int wpcg_kv_compact_workspace(const wpcg_kv_pool* pool, uint64_t* bytes)
{
    if (!bytes) return fail(WPCG_E_ARG, "null output");
    *bytes = 0;
    CompactArgs a{};
    int blocks;
    if (int rc = check_pool(pool, &a.p, &blocks)) return rc;
    *bytes = compact_parts(&a, blocks, nullptr);
    return WPCG_OK;
}

int wpcg_kv_compact(wpcg_ctx* ctx, const wpcg_kv_pool* pool, uint32_t max_copies, int32_t* copies_dev,
                    int32_t* result_dev, void* ws_dev, uint64_t ws_bytes, wpcg_stream stream)
{
    CompactArgs a{};
    int blocks;
    if (int rc = check_pool(pool, &a.p, &blocks)) return rc;
    if (int rc = pool_ready(pool, result_dev, ws_dev, ws_bytes, compact_parts(&a, blocks, ws_dev))) return rc;
    if (max_copies > 0 && !copies_dev) return fail(WPCG_E_ARG, "null argument");
    if (int rc = check_ctx(ctx)) return rc;
    a.max_copies = (int)std::min<uint64_t>(max_copies, INT_BOUND);
    a.copies = copies_dev;
    a.result = result_dev;
    WPCG_HIP(launch_kv_compact(a, pick(ctx, stream)));
    return WPCG_OK;
}

int wpcg_kv_copy(wpcg_ctx* ctx, const wpcg_kv_pages* layers, uint32_t n_layers, const int32_t* copies_dev,
                 const int32_t* n_copies_dev, uint32_t max_copies, wpcg_stream stream)
{
    if (n_layers > 0 && !layers) return fail(WPCG_E_ARG, "null pages");
    if (n_layers > 65536) return fail(WPCG_E_ARG, "n_layers out of range");
    if (max_copies > 1u << 26) return fail(WPCG_E_ARG, "max_copies out of range");
    Pages st{};
    for (uint32_t i = 0; i < n_layers; i++) {
        const wpcg_kv_pages &l = layers[i], &o = layers[0];
        Pages s;
        if (int rc = check_pages(&l, &s)) return rc;
        if (i == 0) st = s;
        if (l.dtype != o.dtype || l.n_pages != o.n_pages || l.page_size != o.page_size || l.n_kv_heads != o.n_kv_heads ||
            l.head_dim != o.head_dim || s.page != st.page || s.head != st.head || s.token != st.token)
            return fail(WPCG_E_SHAPE, "layers of different pages");
        if (!l.k_dev || !l.v_dev) return fail(WPCG_E_ARG, "null argument");
        if (!aligned(l.k_dev) || !aligned(l.v_dev)) return fail(WPCG_E_ARG, "pages not aligned to 16 bytes");
    }
    if (n_layers == 0 || max_copies == 0) return check_ctx(ctx);
    if (!copies_dev || !n_copies_dev) return fail(WPCG_E_ARG, "null argument");
    if (int rc = check_ctx(ctx)) return rc;
    const wpcg_kv_pages& kv = layers[0];
    const uint64_t es = type_size(kv.dtype);
    CopyArgs a{};
    a.page_bytes = st.page * es;
    a.head_bytes = st.head * es;
    a.token_bytes = (uint32_t)(st.token * es);
    a.heads = kv.n_kv_heads;
    a.n_pages = (int)kv.n_pages;
    a.page = (int)kv.page_size;
    while ((16u << a.piece_shift) < kv.head_dim * es) a.piece_shift++;
    a.max_copies = (int)max_copies;
    a.copies = copies_dev;
    a.n = n_copies_dev;
    for (uint32_t l0 = 0; l0 < n_layers; l0 += COPY_LAYERS) {
        const uint32_t n = std::min<uint32_t>(n_layers - l0, COPY_LAYERS);
        for (uint32_t i = 0; i < n; i++) {
            a.side[2 * i] = (uint8_t*)layers[l0 + i].k_dev;
            a.side[2 * i + 1] = (uint8_t*)layers[l0 + i].v_dev;
        }
        a.units = 2 * n * a.heads;
        WPCG_HIP(launch_kv_copy(a, pick(ctx, stream)));
    }
    return WPCG_OK;
}

int wpcg_logprobs_workspace(const wpcg_logprob* d, uint64_t* bytes)
{
    if (!bytes) return fail(WPCG_E_ARG, "null output");
    *bytes = 0;
    int chunks;
    uint64_t part = 0;
    return check_logprobs(d, &chunks, &part, bytes);
}

int wpcg_logprobs(wpcg_ctx* ctx, const wpcg_logprob* d, void* ws_dev, uint64_t ws_bytes, wpcg_stream stream)
{
    LogprobArgs a{};
    uint64_t part = 0, bytes = 0;
    if (int rc = check_logprobs(d, &a.chunks, &part, &bytes)) return rc;
    if (d->n_rows == 0) return check_ctx(ctx);
    if (!d->logits_dev || (!d->tokens_dev && (d->logprob_dev || d->rank_dev))) return fail(WPCG_E_ARG, "null argument");
    if ((uintptr_t)d->logits_dev % type_size(d->dtype)) return fail(WPCG_E_ARG, "logits not aligned to their type");
    if (!ws_dev || ws_bytes < bytes)
        return fail(WPCG_E_ARG, "the call needs " + std::to_string(bytes) + " bytes of workspace");
    if (!aligned(ws_dev)) return fail(WPCG_E_ARG, "workspace not aligned to 16 bytes");
    if (int rc = check_ctx(ctx)) return rc;
    a.n_rows = (int)d->n_rows;
    a.vocab = (int)d->vocab;
    a.top = d->top_ids_dev || d->top_logprob_dev ? (int)d->top : 0;
    a.bf16 = d->dtype == WPCG_DTYPE_BF16;
    a.logits = d->logits_dev;
    a.row = d->logits_stride ? d->logits_stride : d->vocab;
    a.all = (a.n_rows - 1) * a.row + a.vocab;
    a.vec = aligned(a.logits);
    a.temperature = d->temperature_dev;
    a.tokens = d->tokens_dev;
    a.logprob = d->logprob_dev;
    a.entropy = d->entropy_dev;
    a.rank = d->rank_dev;
    a.top_ids = d->top_ids_dev;
    a.top_logprob = d->top_logprob_dev;
    a.part = (LogprobPart*)ws_dev;
    a.seg = (float*)((uint8_t*)ws_dev + part);
    WPCG_HIP(launch_logprobs(a, pick(ctx, stream)));
    return WPCG_OK;
}

}  // extern "C"
