// Device helpers shared by the operators that read rows of log scores (lsr_top.hip, lsr_sample.hip, lsr_distill.hip).
//
// Order of a row: value descending, equal values by ascending class.  A score becomes a 32-bit key that sorts like the
// value (sign-magnitude turned into an unsigned number; -0 and +0 are one value), absent scores (-inf and NaN) get key 0;
// key and complemented class together are a 64-bit number that is different for every entry of a row, so that "the first
// m entries" is always "the entries whose number is at least some threshold".
#pragma once

#include "lsr_internal.h"

#define LSR_ROW_THREADS 256

enum { ROW_F32 = LSR_F32, ROW_F16 = LSR_F16, ROW_BF16 = LSR_BF16 };

template <int DT> struct row_type;
template <> struct row_type<ROW_F32> { using type = float; };
template <> struct row_type<ROW_F16> { using type = _Float16; };
template <> struct row_type<ROW_BF16> { using type = __bf16; };

__device__ __forceinline__ uint32_t row_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return x > -INFINITY ? k : 0u;                       // false for NaN as well
}
__device__ __forceinline__ float row_value(uint32_t key) {
    return __uint_as_float(key ^ ((uint32_t)(~((int32_t)key >> 31)) | 0x80000000u));
}
__device__ __forceinline__ uint64_t row_entry(uint32_t key, uint32_t cls) { return (uint64_t)key << 32 | (uint32_t)~cls; }

__device__ __forceinline__ int row_wave_sum(int v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float row_wave_sum(float v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ uint64_t row_wave_sum(uint64_t v) {
    for (int d = 32; d; d >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, d);
    return v;
}
__device__ __forceinline__ uint64_t row_wave_max(uint64_t v) {
    for (int d = 32; d; d >>= 1) {
        const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, d);
        v = o > v ? o : v;
    }
    return v;
}

// Weights of entries as whole numbers: w in [0, 1] in units of 2^-shift, so that sums do not depend on the order of
// addition.  Adding 2^(52 - shift) leaves the rounded number in the low bits of the double.
__device__ __forceinline__ uint64_t row_fixed(double w, double magic) {
    return (uint64_t)__double_as_longlong(w + magic) - (uint64_t)__double_as_longlong(magic);
}

static inline int row_dtype_bytes(int dtype) { return dtype == LSR_F32 ? 4 : 2; }

// argument checks common to the three entry points; 0 or an error code with its message set
int lsr_check_rows(lsr_ctx* ctx, const char* name, const void* scores_d, int dtype, int64_t n_rows, int64_t n_classes,
                   int64_t row_stride);
