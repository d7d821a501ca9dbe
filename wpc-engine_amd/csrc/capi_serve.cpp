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
    const uint64_t width = (uint64_t)att->n_heads * kv->head_dim;
    if (int rc = row_stride(att->q_stride, width, att->dtype, &a.q_row)) return rc;
    if (int rc = row_stride(att->out_stride, width, att->dtype, &a.out_row)) return rc;
    Plans plan;
    if (int rc = plan_attention(kv, a.b, att, &plan)) return rc;
    if (batch->n_seq == 0 || batch->n_rows == 0) return check_ctx(ctx);
    if (int rc = check_pointers(kv, batch)) return rc;
    if (!att->q_dev || !att->out_dev) return fail(WPCG_E_ARG, "null argument");
    if (!aligned(att->q_dev) || !aligned(att->out_dev)) return fail(WPCG_E_ARG, "rows not aligned to 16 bytes");
    if (plan.bytes) {
        if (!ws_dev || ws_bytes < plan.bytes)
            return fail(WPCG_E_ARG, "the call needs " + std::to_string(plan.bytes) + " bytes of workspace");
        if (!aligned(ws_dev)) return fail(WPCG_E_ARG, "workspace not aligned to 16 bytes");
    }
    if (int rc = check_ctx(ctx)) return rc;
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
    const hipStream_t s = pick(ctx, stream);
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
        a.part_o = (float*)ws_dev;
        a.part_ml = a.part_o + p.parts * kv->head_dim;
        a.ends = (AttnEnd*)(a.part_ml + p.parts * 2);
        WPCG_HIP(p.many ? launch_attn_many(a, d, att->dtype, kv->dtype, s)
                        : launch_attn_few(a, d, att->dtype, kv->dtype, s));
    }
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

}  // extern "C"
