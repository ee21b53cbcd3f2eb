// The paged key / value cache as the kernels see it (kv_cache.hip, attention_paged.hip).
#pragma once
#include "common.h"

namespace capdec {

constexpr float E4M3_MAX = 448.f;
constexpr float AMAX_FLOOR = 0x1p-100f;  // a row of zeros gets a scale as well; 448 / amax stays finite

typedef float f32x2p __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2p __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8p __attribute__((ext_vector_type(8)));

// eight e4m3 codes -> eight bf16 values (exact)
__device__ __forceinline__ bf16x8p e4m3_to_bf16(uint32_t lo, uint32_t hi) {
    const bf16x2p a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2p c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return bf16x8p{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// argument checks shared by the entry points; 0 or an error code
int kv_cache_check(const char* what, const capdec_kv_cache* c);
// pages met outside the cache / lengths past the table by capdec_attn_paged on the current device
int paged_bad_count(unsigned int* count, bool reset);

static inline int log2_of(int v) {
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

}  // namespace capdec
