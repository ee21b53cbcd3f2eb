// The paged key / value cache: rows written (rounded to e4m3 with one scale for each row of a head, or kept as bf16) and read
// back.  See include/capdec.h (capdec_kv_write / capdec_kv_read).
//
// Pure streaming: DH / 8 lanes own one (token, head) row of both sides, 8 elements each, so a bf16 row is one 16-byte load a
// lane and the row's largest magnitude is a shuffle tree over 8 or 16 lanes -- the row is read once.  Magnitudes are compared as integers
// with the sign bit cleared: the order is the same and a NaN beats everything, so it reaches the scale.
#include "paged.h"

namespace capdec {

static __device__ unsigned int g_bad_slots;

struct KVParams {
    void* ck; void* cv; float* sk; float* sv;
    const void* rk; const void* rv;  // rows (write)
    void* ok; void* ov;              // rows (read)
    const int* slots;
    int ldk, ldv, rows, heads, page_log2, slots_total;
};

template <typename T>
__device__ __forceinline__ void load_row8(const T* p, float* x);
template <>
__device__ __forceinline__ void load_row8<__bf16>(const __bf16* p, float* x) {
    const bf16x8p v = *reinterpret_cast<const bf16x8p*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}
template <>
__device__ __forceinline__ void load_row8<float>(const float* p, float* x) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void store_row8(__bf16* p, const float* x) {
    bf16x8p v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (__bf16)x[e];
    *reinterpret_cast<bf16x8p*>(p) = v;
}
__device__ __forceinline__ void store_row8(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// place of a slot's row of one head, in rows of the [pages, heads, page] block
__device__ __forceinline__ size_t cache_row(int slot, int head, int heads, int page_log2) {
    const int page = slot >> page_log2, at = slot & ((1 << page_log2) - 1);
    return ((((size_t)page * heads + head) << page_log2) + at);
}

// x / scale rounded as IEEE division rounds it (but for a negative zero, which becomes a positive one), without a division for each
// element: with y the correctly rounded 1 / scale, q = x y is within an ulp of the quotient and q + (x - q scale) y is the rounded
// quotient (Markstein's theorem); eight divisions a lane made the write kernel bound by the vector units (40001 rows of 8 heads:
// 73 us instead of 57)
__device__ __forceinline__ float quotient(float x, float scale, float y) {
    const float q = x * y;
    return __fmaf_rn(__fmaf_rn(-q, scale, x), y, q);
}

template <typename T, bool E4M3, int DH>
__global__ __launch_bounds__(256) void kv_write_kernel(KVParams p) {
    constexpr int LANES = DH / 8, PER = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t item = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    if (item >= (int64_t)p.rows * p.heads) return;
    const int row = (int)(item / p.heads), head = (int)(item % p.heads);
    const int slot = p.slots[row];
    float x[2][8];
    load_row8((const T*)p.rk + (size_t)row * p.ldk + head * DH + lane * 8, x[0]);
    load_row8((const T*)p.rv + (size_t)row * p.ldv + head * DH + lane * 8, x[1]);
    if (slot < 0 || slot >= p.slots_total) {
        if (slot >= 0 && lane == 0 && head == 0) atomicAdd(&g_bad_slots, 1u);
        return;
    }
    const size_t at = cache_row(slot, head, p.heads, p.page_log2);
    if constexpr (E4M3) {
        uint32_t top[2] = {0, 0};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top[s] = max(top[s], __float_as_uint(x[s][e]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) top[s] = max(top[s], (uint32_t)__shfl_xor((int)top[s], o, 64));
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const float scale = __uint_as_float(max(top[s], __float_as_uint(AMAX_FLOOR))) / E4M3_MAX, y = 1.f / scale;
            float c[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = quotient(x[s][e], scale, y);
            int lo = 0, hi = 0;
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], lo, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], hi, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
            *reinterpret_cast<int2*>((unsigned char*)(s ? p.cv : p.ck) + at * DH + lane * 8) = int2{lo, hi};
            if (lane == 0) (s ? p.sv : p.sk)[at] = scale;
        }
    } else {
        store_row8((__bf16*)p.ck + at * DH + lane * 8, x[0]);
        store_row8((__bf16*)p.cv + at * DH + lane * 8, x[1]);
    }
}

template <typename T, bool E4M3, int DH>
__global__ __launch_bounds__(256) void kv_read_kernel(KVParams p) {
    constexpr int LANES = DH / 8, PER = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t item = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    if (item >= (int64_t)p.rows * p.heads) return;
    const int row = (int)(item / p.heads), head = (int)(item % p.heads);
    const int slot = p.slots[row];
    float x[2][8] = {};
    if (slot >= 0 && slot < p.slots_total) {
        const size_t at = cache_row(slot, head, p.heads, p.page_log2);
        if constexpr (E4M3) {
            const int2 c[2] = {*reinterpret_cast<const int2*>((const unsigned char*)p.ck + at * DH + lane * 8),
                               *reinterpret_cast<const int2*>((const unsigned char*)p.cv + at * DH + lane * 8)};
            const float scale[2] = {p.sk[at], p.sv[at]};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8p v = e4m3_to_bf16((uint32_t)c[s].x, (uint32_t)c[s].y);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[s][e] = (float)v[e] * scale[s];
            }
        } else {
            load_row8((const __bf16*)p.ck + at * DH + lane * 8, x[0]);
            load_row8((const __bf16*)p.cv + at * DH + lane * 8, x[1]);
        }
    } else if (slot >= 0 && lane == 0 && head == 0) {
        atomicAdd(&g_bad_slots, 1u);
    }
    store_row8((T*)p.ok + (size_t)row * p.ldk + head * DH + lane * 8, x[0]);
    store_row8((T*)p.ov + (size_t)row * p.ldv + head * DH + lane * 8, x[1]);
}

int kv_cache_check(const char* what, const capdec_kv_cache* c) {
    CAPDEC_REQUIRE(c && c->k && c->v && aligned16(c->k) && aligned16(c->v), "%s: cache matrices must be non-null and 16-byte aligned", what);
    CAPDEC_REQUIRE(c->dtype == CAPDEC_BF16S || c->dtype == CAPDEC_E4M3, "%s: cache dtype %d: CAPDEC_BF16S or CAPDEC_E4M3", what, c->dtype);
    CAPDEC_REQUIRE(c->dtype == CAPDEC_BF16S || (c->k_scale && c->v_scale), "%s: an e4m3 cache needs its scales", what);
    CAPDEC_REQUIRE(c->dh == 64 || c->dh == 128, "%s: head dim %d not in {64,128}", what, c->dh);
    CAPDEC_REQUIRE(c->heads > 0 && c->heads <= 65535 && c->pages > 0, "%s: bad cache: pages=%d heads=%d", what, c->pages, c->heads);
    CAPDEC_REQUIRE(c->page >= 8 && c->page <= 256 && (c->page & (c->page - 1)) == 0, "%s: page=%d must be a power of two from 8 to 256", what, c->page);
    CAPDEC_REQUIRE((int64_t)c->pages * c->page < (1ll << 31), "%s: pages * page passes 2^31", what);
    return 0;
}

static int kv_rows_check(const char* what, const capdec_kv_cache* c, const void* k, int ldk, const void* v, int ldv, int dtype,
                         const int* slots, int rows) {
    if (int rc = kv_cache_check(what, c)) return rc;
    CAPDEC_REQUIRE(rows >= 0, "%s: rows=%d", what, rows);
    CAPDEC_REQUIRE(dtype == CAPDEC_F32 || dtype == CAPDEC_BF16S, "%s: dtype %d: fp32 (CAPDEC_F32) or bf16 (CAPDEC_BF16S) rows", what, dtype);
    if (rows == 0) return 0;
    const int piece = dtype == CAPDEC_F32 ? 4 : 8, width = c->heads * c->dh;
    CAPDEC_REQUIRE(k && v && slots && aligned16(k) && aligned16(v) && ldk % piece == 0 && ldv % piece == 0 && ldk >= width && ldv >= width,
                   "%s: rows must be non-null, 16-byte aligned, with row strides that are multiples of 16 bytes and cover %d elements", what, width);
    CAPDEC_REQUIRE((int64_t)rows * c->heads / (256 * 8 / c->dh) + 1 < (1ll << 31), "%s: too many rows for one launch", what);
    return 0;
}

static KVParams kv_params(const capdec_kv_cache* c, int ldk, int ldv, const int* slots, int rows) {
    KVParams p;
    memset(&p, 0, sizeof(p));
    p.ck = c->k; p.cv = c->v; p.sk = (float*)c->k_scale; p.sv = (float*)c->v_scale;
    p.ldk = ldk; p.ldv = ldv; p.slots = slots; p.rows = rows; p.heads = c->heads;
    p.page_log2 = log2_of(c->page);
    p.slots_total = c->pages * c->page;
    return p;
}

}  // namespace capdec

using namespace capdec;

#define CAPDEC_KV_LAUNCH(kernel)                                                                                     \
    do {                                                                                                             \
        const int per = 256 / (cache->dh / 8);                                                                       \
        const dim3 grid((unsigned)(((int64_t)rows * cache->heads + per - 1) / per));                                 \
        const bool q8 = cache->dtype == CAPDEC_E4M3, f32 = dtype == CAPDEC_F32, wide = cache->dh == 128;             \
        hipStream_t st = (hipStream_t)stream;                                                                        \
        if (wide) {                                                                                                  \
            if (q8 && f32) hipLaunchKernelGGL((kernel<float, true, 128>), grid, dim3(256), 0, st, p);                \
            else if (q8) hipLaunchKernelGGL((kernel<__bf16, true, 128>), grid, dim3(256), 0, st, p);                 \
            else if (f32) hipLaunchKernelGGL((kernel<float, false, 128>), grid, dim3(256), 0, st, p);                \
            else hipLaunchKernelGGL((kernel<__bf16, false, 128>), grid, dim3(256), 0, st, p);                        \
        } else {                                                                                                     \
            if (q8 && f32) hipLaunchKernelGGL((kernel<float, true, 64>), grid, dim3(256), 0, st, p);                 \
            else if (q8) hipLaunchKernelGGL((kernel<__bf16, true, 64>), grid, dim3(256), 0, st, p);                  \
            else if (f32) hipLaunchKernelGGL((kernel<float, false, 64>), grid, dim3(256), 0, st, p);                 \
            else hipLaunchKernelGGL((kernel<__bf16, false, 64>), grid, dim3(256), 0, st, p);                         \
        }                                                                                                            \
    } while (0)

extern "C" int capdec_kv_write(const capdec_kv_cache* cache, const void* k, int ldk, const void* v, int ldv, int dtype, const int* slots,
                               int rows, capdec_stream_t stream) {
    if (int rc = kv_rows_check("capdec_kv_write", cache, k, ldk, v, ldv, dtype, slots, rows)) return rc;
    if (rows == 0) return 0;
    KVParams p = kv_params(cache, ldk, ldv, slots, rows);
    p.rk = k; p.rv = v;
    CAPDEC_KV_LAUNCH(kv_write_kernel);
    return check_launch("capdec_kv_write");
}

extern "C" int capdec_kv_read(const capdec_kv_cache* cache, const int* slots, int rows, void* k, int ldk, void* v, int ldv, int dtype,
                              capdec_stream_t stream) {
    if (int rc = kv_rows_check("capdec_kv_read", cache, k, ldk, v, ldv, dtype, slots, rows)) return rc;
    if (rows == 0) return 0;
    KVParams p = kv_params(cache, ldk, ldv, slots, rows);
    p.ok = k; p.ov = v;
    CAPDEC_KV_LAUNCH(kv_read_kernel);
    return check_launch("capdec_kv_read");
}

extern "C" int capdec_kv_bad_pages(unsigned int* count, int reset) {
    CAPDEC_REQUIRE(count, "capdec_kv_bad_pages: null pointer");
    unsigned int slots = 0, pages = 0;
    // (the copies alone would not wait for kernels on streams that do not block the default one)
    if (hipDeviceSynchronize() != hipSuccess || hipMemcpyFromSymbol(&slots, HIP_SYMBOL(g_bad_slots), sizeof(slots)) != hipSuccess || paged_bad_count(&pages, reset != 0) != 0) {
        set_error("capdec_kv_bad_pages: reading the counters failed");
        return CAPDEC_ERR_LAUNCH;
    }
    if (reset && slots) {
        const unsigned int zero = 0;
        if (hipMemcpyToSymbol(HIP_SYMBOL(g_bad_slots), &zero, sizeof(zero)) != hipSuccess) return CAPDEC_ERR_LAUNCH;
    }
    *count = slots + pages;
    return 0;
}
