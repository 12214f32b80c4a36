// fm_mix.h — device code that the token mixers (fm_gdn.hip, fm_attn.hip) share: loads and stores of
// either element type, matrix-core operand types.
#pragma once

#include "fm_common.h"
#include "fm_mix_index.h"

#if defined(__HIPCC__)

typedef float fm_v4f __attribute__((ext_vector_type(4)));
typedef short fm_v8s __attribute__((ext_vector_type(8)));
typedef _Float16 fm_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 fm_v2h __attribute__((ext_vector_type(2)));
typedef uint32_t fm_v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float fm_bf16_f(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint16_t fm_f_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// four elements from element offset `at` (a multiple of 4) of a fp32 or bf16 array
template <bool BF16>
__device__ __forceinline__ fm_v4f fm_ld4(const void *p, int64_t at) {
    if constexpr (BF16) {
        const uint2 w = *(const uint2 *)((const uint16_t *)p + at);
        return fm_v4f{fm_bf16_lo(w.x), fm_bf16_hi(w.x), fm_bf16_lo(w.y), fm_bf16_hi(w.y)};
    } else {
        return *(const fm_v4f *)((const float *)p + at);
    }
}
template <bool BF16>
__device__ __forceinline__ float fm_ld1(const void *p, int64_t at) {
    if constexpr (BF16) return fm_bf16_f(((const uint16_t *)p)[at]);
    else return ((const float *)p)[at];
}
template <bool BF16>
__device__ __forceinline__ void fm_st1(void *p, int64_t at, float v) {
    if constexpr (BF16) ((uint16_t *)p)[at] = fm_f_bf16(v);
    else ((float *)p)[at] = v;
}
template <bool BF16>
__device__ __forceinline__ void fm_st4(void *p, int64_t at, fm_v4f v) {
    if constexpr (BF16) {
        uint2 w;
        w.x = (uint32_t)fm_f_bf16(v[0]) | (uint32_t)fm_f_bf16(v[1]) << 16;
        w.y = (uint32_t)fm_f_bf16(v[2]) | (uint32_t)fm_f_bf16(v[3]) << 16;
        *(uint2 *)((uint16_t *)p + at) = w;
    } else {
        *(fm_v4f *)((float *)p + at) = v;
    }
}

// Barrier behind this wave's LDS writes that leaves loads from memory in flight.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

#endif  // __HIPCC__
