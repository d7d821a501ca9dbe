// Head norm, rotation and the store of new rows into paged keys and values.
//
// Per query or key head of D values, x in fp32:
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_i, y_{i+D/2}) turned by the angle position * freq[i]
// Values are stored as they come. Every value is read once and written once,
// so the memory is the bound. A head is D/8 lanes, each with four values of
// its lower and the four of its upper half that they turn with, so that the
// rotation needs no exchange and the norm's sum is three or four DPP adds. A
// workgroup takes 2048 / D heads of one row; its first D/2 threads make the
// angles while the loads are in flight: the product and the reduction modulo
// 2 pi are fp64 (fp32 would lose the angle's fraction from positions of a few
// thousand on), sine and cosine of what is left, within +-pi, fp32.
//
// Measured, 32 / 8 heads of 128, fp32 rows into E4M3 pages: 3 prompts of up to
// 2000 rows (149 MB) 33.3 us, 4.5 TB/s; 64 sequences of one row, 32 / 4 heads
// into BF16 pages 4.3 us, of which a launch alone is 3.8.
#include "paged.h"
#include "wave.h"

namespace wpcg {
namespace {

constexpr int THREADS = 256;

struct Four {
    float v[4];
};

template <bool BF16>
__device__ __forceinline__ Four load4(const void* base, uint64_t at)
{
    Four r;
    if (BF16) {
        const pu32x2 w = *(const pu32x2*)((const uint16_t*)base + at);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            r.v[2 * i] = __uint_as_float(w[i] << 16);
            r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const pf32x4 w = *(const pf32x4*)((const float*)base + at);
#pragma unroll
        for (int i = 0; i < 4; i++) r.v[i] = w[i];
    }
    return r;
}

// Clamped to the type's range before the conversion, which would make NaN of
// larger values; NaN stays NaN.
__device__ __forceinline__ float e4m3_range(float x) { return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f); }

__device__ __forceinline__ void store4(void* base, uint64_t at, int dtype, const float* v)
{
    if (dtype == WPCG_DTYPE_F32) {
        *(pf32x4*)((float*)base + at) = (pf32x4){v[0], v[1], v[2], v[3]};
    } else if (dtype == WPCG_DTYPE_BF16) {
        *(pu32x2*)((uint16_t*)base + at) = (pu32x2){pk_bf16_rne(v[0], v[1]), pk_bf16_rne(v[2], v[3])};
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(v[0]), e4m3_range(v[1]), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(v[2]), e4m3_range(v[3]), w, true);
        *(int*)((uint8_t*)base + at) = w;
    }
}

template <int D, bool BF16>
__global__ __launch_bounds__(THREADS) void k_kv_append(KvAppendArgs p)
{
    constexpr int LANES = D / 8;           // of a head
    constexpr int HEADS = THREADS / LANES;  // of a workgroup
    __shared__ float2 turn[D / 2];
    const int groups = (p.n_units + HEADS - 1) / HEADS;
    const int r = (int)(blockIdx.x / (unsigned)groups);
    const int s = p.b.q_start ? seq_of_row(p.b.q_start, p.b.n_seq, r) : r;
    if (s >= p.b.n_seq) return;
    const SeqRows q = seq_rows(p.b, s);
    if (r < q.a || r >= q.a + q.n) return;
    const int pos = q.bad ? 0 : q.len - q.n + (r - q.a);
    if (pos < 0) return;

    // the row's place in the pages
    bool bad = q.bad;
    uint64_t place = 0;
    if (!bad) {
        const int id = p.b.table[(uint64_t)s * p.b.table_stride + (pos >> p.b.page_shift)];
        bad = (uint32_t)id >= p.b.n_pages;
        place = (uint64_t)(bad ? 0 : id) * p.page_stride + (uint64_t)(pos & (p.b.page_size - 1)) * p.token_stride;
    }

    const int unit = (int)(blockIdx.x % (unsigned)groups) * HEADS + (int)threadIdx.x / LANES;
    const int lane = (int)threadIdx.x % LANES;
    // units: query heads, key heads, value heads
    const int kind = unit < p.n_q ? 0 : unit < p.n_q + p.n_kv ? 1 : 2;
    const int head = kind == 0 ? unit : kind == 1 ? unit - p.n_q : unit - p.n_q - p.n_kv;
    const bool mine = unit < p.n_units;
    Four lo = {}, hi = {};
    if (mine) {
        const void* src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
        const uint64_t at = (uint64_t)r * (kind == 0 ? p.q_row : kind == 1 ? p.k_row : p.v_row) +
                            (uint64_t)head * D + lane * 4;
        lo = load4<BF16>(src, at);
        hi = load4<BF16>(src, at + D / 2);
    }
    if (p.freq) {
        if (threadIdx.x < D / 2) {
            const double angle = (double)pos * p.freq[threadIdx.x];
            const double n = rint(angle * 0.15915494309189535);
            // 2 pi in two parts
            const double rest = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, angle));
            float sn, cs;
            sincosf((float)rest, &sn, &cs);
            turn[threadIdx.x] = make_float2(cs, sn);
        }
        __syncthreads();
    }
    const float* w = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) sq += lo.v[i] * lo.v[i] + hi.v[i] * hi.v[i];
    sq += wave_dpp<WDPP_XOR1>(0.0f, sq);
    sq += wave_dpp<WDPP_XOR2>(0.0f, sq);
    sq += wave_dpp<WDPP_HALF_MIRROR>(0.0f, sq);
    if (LANES == 16) sq += wave_dpp<WDPP_MIRROR>(0.0f, sq);
    if (!mine) return;
    if (w) {
        const float inv = 1.0f / sqrtf(sq * (1.0f / D) + p.eps);
        const pf32x4 wl = *(const pf32x4*)(w + lane * 4), wh = *(const pf32x4*)(w + D / 2 + lane * 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo.v[i] = lo.v[i] * inv * wl[i];
            hi.v[i] = hi.v[i] * inv * wh[i];
        }
    }
    if (kind < 2 && p.freq) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 t = turn[lane * 4 + i];
            const float a = lo.v[i], b = hi.v[i];
            lo.v[i] = a * t.x - b * t.y;
            hi.v[i] = b * t.x + a * t.y;
        }
    }
    if (kind == 0) {
        if (bad)
#pragma unroll
            for (int i = 0; i < 4; i++) lo.v[i] = hi.v[i] = __builtin_nanf("");
        const uint64_t at = (uint64_t)r * p.q_out_row + (uint64_t)head * D + lane * 4;
        store4(p.q_out, at, p.q_out_dtype, lo.v);
        store4(p.q_out, at + D / 2, p.q_out_dtype, hi.v);
        return;
    }
    if (bad) return;
    const float* scales = kind == 1 ? p.k_scale : p.v_scale;
    if (scales) {
        const float sc = scales[head];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo.v[i] /= sc;
            hi.v[i] /= sc;
        }
    }
    void* pages = kind == 1 ? p.k_pages : p.v_pages;
    const uint64_t at = place + (uint64_t)head * p.head_stride + lane * 4;
    store4(pages, at, p.cache_dtype, lo.v);
    store4(pages, at + D / 2, p.cache_dtype, hi.v);
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& p, int head_dim, bool bf16, hipStream_t s)
{
    const int heads = THREADS * 8 / head_dim;
    const uint64_t blocks = (uint64_t)p.b.n_rows * (uint64_t)((p.n_units + heads - 1) / heads);
    if (blocks == 0) return hipSuccess;
    const dim3 grid((unsigned)blocks), block(THREADS);
    if (head_dim == 128)
        bf16 ? k_kv_append<128, true><<<grid, block, 0, s>>>(p) : k_kv_append<128, false><<<grid, block, 0, s>>>(p);
    else
        bf16 ? k_kv_append<64, true><<<grid, block, 0, s>>>(p) : k_kv_append<64, false><<<grid, block, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace wpcg
