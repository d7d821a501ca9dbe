// Pages of a cache forked, freed, handed out, moved together and copied.
//
// A pool is the pages' counts of table entries (0: free), the table and the
// sequences' lengths; nothing here looks at the host. The rows of a call change
// all at once, so each step reads the old state and a launch lies between what
// it decides and what it writes:
//   fork     1 counts follow the rows' old and new entries (an atomic an entry
//              that changes); entries of other rows are set aside
//            2 free pages a block of 4096; one workgroup goes through the
//              sequences: who copies the page that it writes next, how many fresh
//              pages each needs, where in the list of fresh pages these begin
//            3 the rows, and the n-th free page to its place in them; or, where
//              pages are missing, the counts back as they were
//   compact  1 pages in use a block, 2 the lists of free pages from below and of
//              used ones from above, 3 the moves, in the counts and the table
// Fresh pages are the lowest free ones in the order of sequences, so results are
// the same whatever order the workgroups run in. The work is a few words a
// sequence and four bytes a page: launches are what it costs, and in each a chain of
// three to five loads that depend on each other. Forks of small pools are one
// workgroup's, which has barriers instead: 8 x 4 beams 8.2 us instead of 12.0. 64
// answers to 2012 tokens 12.6 us; moving 40 sequences' 830 MB together 14 us and the
// copies.
//
// The copies go through all layers in one launch. A wave takes the tokens of one
// page, head and layer, a few KiB side by side, 16 bytes a lane: memory bounds them,
// 830 MB read and written in 170 us, 4.9 TB/s, where a copy of 1 GiB reaches 5.14.
#include <algorithm>

#include "paged.h"
#include "wave.h"

namespace wpcg {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BLOCK = POOL_BLOCK, PER = BLOCK / THREADS;  // pages of a workgroup, of a thread

__device__ __forceinline__ bool is_page(const PoolArgs& p, int id) { return (uint32_t)id < (uint32_t)p.n_pages; }
__device__ __forceinline__ int length_of(const PoolArgs& p, int s) { return min(max(p.kv_len[s], 0), p.stride << p.shift); }
__device__ __forceinline__ int pages_of(const PoolArgs& p, int tokens) { return (tokens + p.page - 1) >> p.shift; }

// What a call makes of sequence s, without what is decided among sequences.
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int s)
{
    const PoolArgs& p = a.p;
    ForkRow r;
    r.parent = a.parent ? a.parent[s] : s;
    if ((uint32_t)r.parent >= (uint32_t)p.n_seq) r.parent = -1;
    const int has = r.parent >= 0 ? length_of(p, r.parent) : 0;
    r.keep = a.keep ? min(max(a.keep[s], 0), has) : has;
    const int grow = a.grow ? a.grow[s] : a.grow_all;
    r.size = r.keep + min(max(grow, 0), (p.stride << p.shift) - r.keep);
    r.old_pages = pages_of(p, length_of(p, s));
    r.kept_pages = pages_of(p, r.keep);
    r.pages = pages_of(p, r.size);
    // pages behind the window of all rows from position `keep` on
    r.dead0 = r.dead1 = 0;
    if (a.window > 0) {
        r.dead0 = pages_of(p, a.sinks);
        r.dead1 = r.keep - a.window + 1 > 0 ? (r.keep - a.window + 1) >> p.shift : 0;
    }
    return r;
}
__device__ __forceinline__ bool writes_tail(const PoolArgs& p, const ForkRow& r)
{
    return (r.keep & (p.page - 1)) != 0 && r.size > r.keep;
}
__device__ __forceinline__ bool keeps(const ForkRow& r, int j)
{
    return j < r.kept_pages && !(j >= r.dead0 && j < r.dead1);
}
// The row's entry j before, and what it keeps there (-1: none).
__device__ __forceinline__ int old_entry(const PoolArgs& p, const ForkRow& r, int s, int j)
{
    const int id = j < r.old_pages ? p.table[(uint64_t)s * p.stride + j] : -1;
    return is_page(p, id) ? id : -1;
}
__device__ __forceinline__ int kept_entry(const PoolArgs& p, const ForkRow& r, int j)
{
    const int id = keeps(r, j) ? p.table[(uint64_t)r.parent * p.stride + j] : -1;
    return is_page(p, id) ? id : -1;
}

// The sum of v over the threads before this one, and over all in total; s: WAVES ints.
__device__ __forceinline__ int block_before(int v, int* s, int& total)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    int t = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int u = __shfl_up(t, d);
        if (lane >= d) t += u;
    }
    if (lane == 63) s[wave] = t;
    __syncthreads();
    int start = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w == wave) start = total;
        total += s[w];
    }
    __syncthreads();
    return start + t - v;
}
// The blocks' counts before block b, and all of them. Every wave adds them up for
// itself: no barrier before what comes next is loaded.
__device__ __forceinline__ void blocks_before(const int* count, int n, int b, int& before, int& total)
{
    int x = 0, y = 0;
    for (int i = (int)threadIdx.x & 63; i < n; i += 64) {
        const int v = count[i];
        x += i < b ? v : 0;
        y += v;
    }
    before = wave_sum_i(x);
    total = wave_sum_i(y);
}

// ---- fork ----------------------------------------------------------------------
// Row chunk `at`: entries [1024 c, 1024 c + 1024) of sequence s.
__device__ __forceinline__ void chunk_of(const PoolArgs& p, int at, int& s, int& j)
{
    const int chunks = (p.stride + THREADS - 1) / THREADS;
    s = at / chunks;
    j = at % chunks * THREADS + (int)threadIdx.x;
}

__global__ __launch_bounds__(THREADS) void k_fork_count(ForkArgs a)
{
    const PoolArgs& p = a.p;
    int s, j;
    chunk_of(p, (int)blockIdx.x, s, j);
    const ForkRow r = fork_row(a, s);
    const bool writer = writes_tail(p, r);
    if (j == 0 && !writer) a.tail[s] = -1;
    if (j >= max(r.old_pages, r.kept_pages)) return;
    const int was = old_entry(p, r, s, j), is = kept_entry(p, r, j);
    if (was != is) {
        if (was >= 0) atomicSub(&p.refs[was], 1);
        if (is >= 0) atomicAdd(&p.refs[is], 1);
    }
    if (r.parent != s && j < r.kept_pages) a.kept[(uint64_t)s * p.stride + j] = is;
    if (writer && j == r.keep >> p.shift) {
        a.tail[s] = is;
        if (is >= 0) a.writers[is] = {0, 0x7fffffff};
    }
}

__global__ __launch_bounds__(THREADS) void k_fork_plan(ForkArgs a)
{
    __shared__ int s_sums[WAVES];
    const PoolArgs& p = a.p;
    const int tid = (int)threadIdx.x;
    if ((int)blockIdx.x < a.blocks) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int page = (int)blockIdx.x * BLOCK + i * THREADS + tid;
            n += page < p.n_pages && p.refs[page] == 0;
        }
        int all;
        block_before(n, s_sums, all);
        if (tid == 0) a.count[blockIdx.x] = all;
        return;
    }
    for (int s = tid; s < p.n_seq; s += THREADS) {
        const int id = a.tail[s];
        if (id >= 0) {
            atomicAdd(&a.writers[id].n, 1);
            atomicMin(&a.writers[id].first, s);
        }
    }
    __syncthreads();
    int fresh = 0, copies = 0;  // of the sequences before
    for (int s0 = 0; s0 < p.n_seq; s0 += THREADS) {
        const int s = s0 + tid;
        ForkRow r = {};
        bool copy = false;
        if (s < p.n_seq) {
            r = fork_row(a, s);
            const int id = a.tail[s];
            r.src = id;
            if (id >= 0) {
                // the first writer keeps it if nobody else has it
                const int n = __hip_atomic_load(&a.writers[id].n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const int first = __hip_atomic_load(&a.writers[id].first, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                copy = first != s || p.refs[id] > n;
            }
            r.from = copy ? r.keep >> p.shift : r.kept_pages;
        }
        int more, some;
        r.base = fresh + block_before(r.pages - r.from, s_sums, more);
        const int at = copies + block_before(copy, s_sums, some);
        r.copy = copy ? at : -1;
        if (s < p.n_seq) a.rows[s] = r;
        fresh += more;
        copies += some;
    }
    if (tid == 0) {
        a.totals[0] = fresh;
        a.totals[1] = copies;
    }
}

constexpr int BASES = 1024;  // sequences whose first fresh page is held in LDS

__global__ __launch_bounds__(THREADS) void k_fork_apply(ForkArgs a)
{
    __shared__ int s_sums[WAVES], s_base[BASES];
    const PoolArgs& p = a.p;
    const int tid = (int)threadIdx.x, b = (int)blockIdx.x, need = a.totals[0];
    int before, free;
    blocks_before(a.count, a.blocks, b, before, free);
    const bool enough = need <= free;
    if (b == 0 && tid == 0) {
        a.result[0] = free - need;
        a.result[1] = enough ? a.totals[1] : 0;
    }
    if (b < a.blocks) {
        // thread t: pages PER t .. of the block, so that ranks rise with threads
        const int page0 = b * BLOCK + PER * tid;
        bool is[PER];
        int n = 0, all;
#pragma unroll
        for (int i = 0; i < PER; i++) is[i] = page0 + i < p.n_pages && p.refs[page0 + i] == 0;
        // every step-th sequence's base, so that few steps of a search read memory
        const int step = max(1, (p.n_seq + BASES - 1) / BASES), bases = (p.n_seq + step - 1) / step;
        if (tid < bases) s_base[tid] = a.rows[tid * step].base;
        if (!enough || before >= need) return;
#pragma unroll
        for (int i = 0; i < PER; i++) n += is[i];
        int rank = before + block_before(n, s_sums, all);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (!is[i] || rank >= need) continue;
            // the last sequence whose fresh pages begin at or before this one
            const auto last = [&](int lo, int hi, auto base) {
                while (lo < hi) {
                    const int mid = (lo + hi + 1) / 2;
                    if (base(mid) <= rank) lo = mid;
                    else hi = mid - 1;
                }
                return lo;
            };
            int to = last(0, bases - 1, [&](int x) { return s_base[x]; }) * step;
            to = last(to, min(to + step, p.n_seq) - 1, [&](int x) { return a.rows[x].base; });
            const ForkRow r = a.rows[to];
            const int j = r.from + rank - r.base;
            p.table[(uint64_t)to * p.stride + j] = page0 + i;
            p.refs[page0 + i] = 1;
            if (r.copy >= 0 && j == r.from) {
                int32_t* c = a.copies + (uint64_t)r.copy * 3;
                c[0] = r.src;
                c[1] = page0 + i;
                c[2] = r.keep & (p.page - 1);
                atomicSub(&p.refs[r.src], 1);
            }
            rank++;
        }
        return;
    }
    int s, j;
    chunk_of(p, b - a.blocks, s, j);
    const ForkRow r = a.rows[s];
    if (!enough) {
        if (j >= max(r.old_pages, r.kept_pages)) return;
        const int was = old_entry(p, r, s, j), is = kept_entry(p, r, j);
        if (was != is) {
            if (was >= 0) atomicAdd(&p.refs[was], 1);
            if (is >= 0) atomicSub(&p.refs[is], 1);
        }
        return;
    }
    if (j == 0) p.kv_len[s] = r.size;
    int32_t* to = p.table + (uint64_t)s * p.stride + j;
    if (j < r.from) {
        if (r.parent != s) *to = a.kept[(uint64_t)s * p.stride + j];
        else if (j >= r.dead0 && j < r.dead1) *to = -1;
    } else if (j >= r.pages && j < r.old_pages) {
        *to = -1;
    }
}

// A whole fork by one workgroup, where every thread has ONE_ENTRIES table entries at
// most and a wave's pages are ONE_PAGES rows of 64: the same three steps with barriers
// between them instead of launches. Thread t: of sequence t / team, the entries
// t % team, + team ..
constexpr int ONE_SEQS = 64, ONE_ENTRIES = 8, ONE_PAGES = 8;
__global__ __launch_bounds__(THREADS) void k_fork_one(ForkArgs a, int team_shift)
{
    __shared__ int s_sums[WAVES];
    __shared__ __attribute__((aligned(16))) int s_tail[ONE_SEQS];
    __shared__ ForkRow s_rows[ONE_SEQS];
    const PoolArgs& p = a.p;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int team = 1 << team_shift, s = tid >> team_shift, t = tid & (team - 1);
    const bool live = s < p.n_seq, leads = live && t == 0;
    const auto count_of = [&](int page) { return __hip_atomic_load(&p.refs[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
    const auto add = [&](int page, int n) {
        (void)__hip_atomic_fetch_add(&p.refs[page], n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    ForkRow r = {};
    r.parent = -1;
    if (live) r = fork_row(a, s);
    const int entries = max(r.old_pages, r.kept_pages);
    const bool writer = writes_tail(p, r);
    if (leads && !writer) s_tail[s] = -1;
    if (tid >= p.n_seq && tid < (p.n_seq + 3) / 4 * 4) s_tail[tid] = -1;
    const int32_t* const old = p.table + (uint64_t)(live ? s : 0) * p.stride;
    const int32_t* const from_row = p.table + (uint64_t)max(r.parent, 0) * p.stride;
    int is[ONE_ENTRIES];
    int was[ONE_ENTRIES];
#pragma unroll
    for (int i = 0; i < ONE_ENTRIES; i++) {
        const int x = min(t + i * team, p.stride - 1);
        was[i] = is[i] = -1;
        if (__any(t + i * team < entries)) {  // (no load behind a condition of its lanes)
            was[i] = old[x];
            is[i] = from_row[x];
        }
    }
#pragma unroll
    for (int i = 0; i < ONE_ENTRIES; i++) {
        const int j = t + i * team;
        if (!__any(j < entries)) continue;
        const int w = j < r.old_pages && is_page(p, was[i]) ? was[i] : -1;
        const int x = keeps(r, j) && is_page(p, is[i]) ? is[i] : -1;
        is[i] = x;
        if (w != x) {
            if (w >= 0) add(w, -1);
            if (x >= 0) add(x, 1);
        }
        if (writer && j == r.keep >> p.shift) s_tail[s] = x;
    }
    __syncthreads();

    // the free pages, ranks rising with the wave's rows
    const int rows = (p.n_pages + THREADS - 1) / THREADS, page0 = wave * rows * 64 + lane;
    int refs[ONE_PAGES];
#pragma unroll
    for (int i = 0; i < ONE_PAGES; i++) {
        refs[i] = 1;
        if (i < rows) refs[i] = count_of(min(page0 + 64 * i, p.n_pages - 1));
    }
    const int tail = leads ? s_tail[s] : -1, held = tail >= 0 ? count_of(tail) : 0;
    uint64_t free_row[ONE_PAGES];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < ONE_PAGES; i++) {
        free_row[i] = 0;
        if (i < rows) free_row[i] = __ballot(refs[i] == 0 && page0 + 64 * i < p.n_pages);
        mine += __popcll(free_row[i]);
    }
    // the first writer of a tail keeps it if nobody else has it
    bool copy = false;
    if (tail >= 0) {
        int n = 0, first = ONE_SEQS;
        for (int i = (p.n_seq + 3) / 4 * 4 - 4; i >= 0; i -= 4) {
            const int4 x = *(const int4*)&s_tail[i];
            const int v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 3; j >= 0; j--) {
                n += v[j] == tail;
                if (v[j] == tail) first = i + j;
            }
        }
        copy = first != s || held > n;
    }
    r.src = tail;
    r.from = copy ? r.keep >> p.shift : r.kept_pages;
    int need, copies, free;
    r.base = block_before(leads ? r.pages - r.from : 0, s_sums, need);
    const int at = block_before(copy, s_sums, copies);
    const int before = block_before(lane == 0 ? mine : 0, s_sums, free);
    r.copy = copy ? at : -1;
    if (leads) s_rows[s] = r;
    __syncthreads();
    const bool enough = need <= free;
    if (tid == 0) {
        a.result[0] = free - need;
        a.result[1] = enough ? copies : 0;
    }
    if (!enough) {
        for (int j = t; j < entries; j += team) {
            const int was = old_entry(p, r, s, j), x = kept_entry(p, r, j);
            if (was != x) {
                if (was >= 0) add(was, 1);
                if (x >= 0) add(x, -1);
            }
        }
        return;
    }
    int rank = __builtin_amdgcn_readfirstlane(before);
#pragma unroll
    for (int i = 0; i < ONE_PAGES; i++) {
        if (i >= rows || rank >= need) continue;
        const int at_page = rank + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(free_row[i] >> 32),
                                                                  __builtin_amdgcn_mbcnt_lo((uint32_t)free_row[i], 0));
        if ((free_row[i] >> lane & 1) != 0 && at_page < need) {
            int lo = 0, hi = p.n_seq - 1;  // the last sequence whose fresh pages begin at or before this one
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (s_rows[mid].base <= at_page) lo = mid;
                else hi = mid - 1;
            }
            const ForkRow to = s_rows[lo];
            const int j = to.from + at_page - to.base, page = page0 + 64 * i;
            p.table[(uint64_t)lo * p.stride + j] = page;
            p.refs[page] = 1;
            if (to.copy >= 0 && j == to.from) {
                int32_t* c = a.copies + (uint64_t)to.copy * 3;
                c[0] = to.src;
                c[1] = page;
                c[2] = to.keep & (p.page - 1);
                add(to.src, -1);
            }
        }
        rank += __popcll(free_row[i]);
    }
    if (!live) return;
    if (leads) p.kv_len[s] = r.size;
    const int from = s_rows[s].from;
#pragma unroll
    for (int i = 0; i < ONE_ENTRIES; i++) {
        const int j = t + i * team;
        if (!__any(j < entries)) continue;
        int32_t* to = p.table + (uint64_t)s * p.stride + j;
        if (j < from) {
            if (r.parent != s) *to = is[i];
            else if (j >= r.dead0 && j < r.dead1) *to = -1;
        } else if (j >= r.pages && j < r.old_pages) {
            *to = -1;
        }
    }
}

// ---- compact -------------------------------------------------------------------
__global__ __launch_bounds__(THREADS) void k_compact_count(CompactArgs a)
{
    __shared__ int s_sums[WAVES];
    int n = 0, all;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int page = (int)blockIdx.x * BLOCK + i * THREADS + (int)threadIdx.x;
        n += page < a.p.n_pages && a.p.refs[page] != 0;
    }
    block_before(n, s_sums, all);
    if (threadIdx.x == 0) a.count[blockIdx.x] = all;
}

// used[i]: the i-th page in use from above, free[i]: the i-th free one from below,
// rank[page]: its i of the used ones, or -1
__global__ __launch_bounds__(THREADS) void k_compact_rank(CompactArgs a)
{
    __shared__ int s_sums[WAVES];
    const int b = (int)blockIdx.x, page0 = b * BLOCK + PER * (int)threadIdx.x;
    int before, used;
    blocks_before(a.count, a.blocks, b, before, used);
    if (b == 0 && threadIdx.x == 0) *a.total = used;
    bool is[PER];
    int n = 0, all;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        is[i] = page0 + i < a.p.n_pages && a.p.refs[page0 + i] != 0;
        n += is[i];
    }
    int up = before + block_before(n, s_sums, all);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int page = page0 + i;
        if (page >= a.p.n_pages) break;
        a.rank[page] = is[i] ? used - 1 - up : -1;
        if (is[i]) a.used[used - 1 - up++] = page;
        else a.free[page - up] = page;
    }
}

__global__ __launch_bounds__(THREADS) void k_compact_apply(CompactArgs a)
{
    const PoolArgs& p = a.p;
    const int used = *a.total, most = min(min(used, p.n_pages - used), a.max_copies);
    const auto moves = [&](int i) { return i < most && a.free[i] < a.used[i]; };
    const int b = (int)blockIdx.x;
    if (b < a.move_blocks) {
        const int i = b * THREADS + (int)threadIdx.x;
        const bool it = moves(i);
        if (i == 0 && !it) {
            a.result[0] = used > 0 ? a.used[0] + 1 : 0;
            a.result[1] = 0;
        }
        if (!it) return;
        const int from = a.used[i], to = a.free[i];
        int32_t* c = a.copies + (uint64_t)i * 3;
        c[0] = from;
        c[1] = to;
        c[2] = p.page;
        p.refs[to] = p.refs[from];
        p.refs[from] = 0;
        if (!moves(i + 1)) {  // the last one: where the pages in use end now
            a.result[0] = 1 + max(to, i + 1 < used ? a.used[i + 1] : -1);
            a.result[1] = i + 1;
        }
        return;
    }
    int s, j;
    chunk_of(p, b - a.move_blocks, s, j);
    if (j >= pages_of(p, length_of(p, s))) return;
    int32_t* at = p.table + (uint64_t)s * p.stride + j;
    const int id = *at;
    if (!is_page(p, id)) return;
    const int i = a.rank[id];
    if (i >= 0 && moves(i)) *at = a.free[i];
}

// ---- copies --------------------------------------------------------------------
constexpr int COPY_THREADS = 256, COPY_WAVES = COPY_THREADS / 64, AHEAD = 4;

// A wave a head of a page, keys or values, of a layer; `step` waves go through
// them all.
__global__ __launch_bounds__(COPY_THREADS) void k_kv_copy(CopyArgs a)
{
    const int n = min(*a.n, a.max_copies);
    const int lane = (int)threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * COPY_WAVES + (threadIdx.x >> 6));
    int copy = (int)(wave / a.units);
    uint32_t unit = wave % a.units;
    while (copy < n) {
        const int src = a.copies[(uint64_t)copy * 3], dst = a.copies[(uint64_t)copy * 3 + 1];
        const int tokens = min(max(a.copies[(uint64_t)copy * 3 + 2], 0), a.page);
        if ((uint32_t)src < (uint32_t)a.n_pages && (uint32_t)dst < (uint32_t)a.n_pages) {
            const uint32_t head = unit % a.heads, side = unit / a.heads;
            uint8_t* const base = a.side[side] + (uint64_t)head * a.head_bytes;
            const uint8_t* const from = base + (uint64_t)src * a.page_bytes;
            uint8_t* const to = base + (uint64_t)dst * a.page_bytes;
            const int pieces = tokens << a.piece_shift, mask = (1 << a.piece_shift) - 1;
            for (int i0 = lane; i0 < pieces; i0 += 64 * AHEAD) {
                pu32x4 w[AHEAD];
                uint32_t at[AHEAD];
#pragma unroll
                for (int x = 0; x < AHEAD; x++) {
                    const int i = min(i0 + 64 * x, pieces - 1);
                    at[x] = (uint32_t)(i >> a.piece_shift) * a.token_bytes + (uint32_t)(i & mask) * 16;
                    w[x] = *(const pu32x4*)(from + at[x]);
                }
#pragma unroll
                for (int x = 0; x < AHEAD; x++)
                    if (i0 + 64 * x < pieces) *(pu32x4*)(to + at[x]) = w[x];
            }
        }
        copy += a.step_copies;
        unit += a.step_units;
        if (unit >= a.units) {
            unit -= a.units;
            copy++;
        }
    }
}

}  // namespace

hipError_t launch_kv_fork(const ForkArgs& a, hipStream_t s)
{
    (void)hipGetLastError();  // report only these launches
    // One workgroup for small pools. It and the three launches, us, sequences x pages
    // each: 8 x 30 6.9 and 11.9, 32 x 38 8.2 and 12.0, 64 x 126 12.6 and 15.5; with room
    // for 256 sequences, 16 entries and 16 rows of pages the first two took 8.6 and 9.7,
    // 100 x 20 13.5 and 14.0, 256 x 62 27 and 16.
    int shift = 10;
    while (shift > 0 && THREADS >> shift < a.p.n_seq) shift--;
    if (a.p.n_seq > 0 && a.p.n_seq <= ONE_SEQS && a.p.stride <= ONE_ENTRIES << shift && a.p.n_pages <= ONE_PAGES * THREADS) {
        k_fork_one<<<dim3(1), dim3(THREADS), 0, s>>>(a, shift);
        return hipGetLastError();
    }
    const unsigned rows = (unsigned)a.p.n_seq * (unsigned)((a.p.stride + THREADS - 1) / THREADS);
    if (rows) k_fork_count<<<dim3(rows), dim3(THREADS), 0, s>>>(a);
    k_fork_plan<<<dim3((unsigned)a.blocks + 1), dim3(THREADS), 0, s>>>(a);
    k_fork_apply<<<dim3((unsigned)a.blocks + rows), dim3(THREADS), 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_compact(CompactArgs a, hipStream_t s)
{
    (void)hipGetLastError();  // report only these launches
    const unsigned rows = (unsigned)a.p.n_seq * (unsigned)((a.p.stride + THREADS - 1) / THREADS);
    a.move_blocks = std::max(1, (std::min(a.p.n_pages / 2, a.max_copies) + THREADS - 1) / THREADS);
    k_compact_count<<<dim3((unsigned)a.blocks), dim3(THREADS), 0, s>>>(a);
    k_compact_rank<<<dim3((unsigned)a.blocks), dim3(THREADS), 0, s>>>(a);
    k_compact_apply<<<dim3((unsigned)a.move_blocks + rows), dim3(THREADS), 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_copy(CopyArgs a, hipStream_t s)
{
    (void)hipGetLastError();  // report only these launches
    // 16 waves a CU at most: enough loads in flight
    const uint64_t all = (uint64_t)a.max_copies * a.units;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((all + COPY_WAVES - 1) / COPY_WAVES, 256 * 4);
    if (blocks == 0) return hipSuccess;
    a.step_copies = (int)(blocks * COPY_WAVES / a.units);
    a.step_units = blocks * COPY_WAVES % a.units;
    k_kv_copy<<<dim3(blocks), dim3(COPY_THREADS), 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace wpcg
