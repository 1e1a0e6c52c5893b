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

// 2^y for y <= 0 to 2^-50 of the result: the fraction in [-1/2, 1/2] goes through a polynomial of degree 10 that is 1 at 0
// (interpolation of (2^f - 1) / f at the Chebyshev nodes, largest relative error 5.6e-16).  16 instructions of the same
// rate as 32-bit ones here; the library's exp takes about three times as many.
__device__ __forceinline__ double row_exp2(double y) {
    y = y > -1200.0 ? y : -1200.0;
    const double n = __builtin_rint(y), f = y - n;
    double p = 7.070977866508138e-09;
    p = __builtin_fma(p, f, 1.0205905413765595e-07);
    p = __builtin_fma(p, f, 1.3215451633221434e-06);
    p = __builtin_fma(p, f, 1.5252672924850737e-05);
    p = __builtin_fma(p, f, 0.00015403530424776529);
    p = __builtin_fma(p, f, 0.0013333558200794592);
    p = __builtin_fma(p, f, 0.009618129107618665);
    p = __builtin_fma(p, f, 0.05550410866465167);
    p = __builtin_fma(p, f, 0.24022650695910075);
    p = __builtin_fma(p, f, 0.6931471805599462);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}
#define ROW_LOG2E 1.4426950408889634

// Weights of entries as whole numbers: w in [0, 1] in units of 2^-shift, so that sums do not depend on the order of
// addition.  Adding 2^(52 - shift) leaves the rounded number in the low bits of the double.
__device__ __forceinline__ uint64_t row_fixed(double w, double magic) {
    return (uint64_t)__double_as_longlong(w + magic) - (uint64_t)__double_as_longlong(magic);
}

static inline int row_dtype_bytes(int dtype) { return dtype == LSR_F32 ? 4 : 2; }

// argument checks common to the three entry points; 0 or an error code with its message set
int lsr_check_rows(lsr_ctx* ctx, const char* name, const void* scores_d, int dtype, int64_t n_rows, int64_t n_classes,
                   int64_t row_stride);

// ---- short rows: four adjacent lanes (a quad) hold a row --------------------------------------------------------------
// A row of at most 4 E classes is E registers in each lane of a quad; a wavefront has 16 rows and no LDS or barrier is
// needed to reduce over a row, only lane moves inside quads, which the vector unit makes in the operand read.  Lane q
// holds the runs of four classes q, q + 4, q + 8, ...: sixteen adjacent classes of a row per load instruction.
#define LSR_QUAD_CLASSES 128
#define LSR_QUAD_ROWS (LSR_ROW_THREADS / 4)               // rows of a workgroup

#define QUAD_XOR1 0xB1
#define QUAD_XOR2 0x4E
#define QUAD_XOR3 0x1B
template <int PERM> __device__ __forceinline__ int quad_move(int v) {
    return __builtin_amdgcn_mov_dpp(v, PERM, 0xf, 0xf, true);
}
template <int PERM> __device__ __forceinline__ float quad_move(float v) {
    return __int_as_float(quad_move<PERM>(__float_as_int(v)));
}
template <int PERM> __device__ __forceinline__ double quad_move(double v) {
    const long long b = __double_as_longlong(v);
    const unsigned lo = (unsigned)quad_move<PERM>((int)b), hi = (unsigned)quad_move<PERM>((int)(b >> 32));
    return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
}
__device__ __forceinline__ double row_max(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ double row_min(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float row_max(float a, float b) { return fmaxf(a, b); }
template <typename V> __device__ __forceinline__ V quad_max(V v) {
    v = row_max(v, quad_move<QUAD_XOR1>(v));
    return row_max(v, quad_move<QUAD_XOR2>(v));
}
__device__ __forceinline__ double quad_min(double v) {
    v = row_min(v, quad_move<QUAD_XOR1>(v));
    return row_min(v, quad_move<QUAD_XOR2>(v));
}
__device__ __forceinline__ int quad_max(int v) {
    v = max(v, quad_move<QUAD_XOR1>(v));
    return max(v, quad_move<QUAD_XOR2>(v));
}
__device__ __forceinline__ int quad_min(int v) {
    v = min(v, quad_move<QUAD_XOR1>(v));
    return min(v, quad_move<QUAD_XOR2>(v));
}
template <typename V> __device__ __forceinline__ V quad_sum(V v) {
    v += quad_move<QUAD_XOR1>(v);
    return v + quad_move<QUAD_XOR2>(v);
}
// sum of the lanes of the quad before this one
template <typename V> __device__ __forceinline__ V quad_before(V v, int q) {
    const V a = quad_move<0x00>(v), b = quad_move<0x55>(v), c = quad_move<0xAA>(v);
    return (q > 0 ? a : (V)0) + (q > 1 ? b : (V)0) + (q > 2 ? c : (V)0);
}

// class of register i of lane q
__device__ __forceinline__ int quad_class(int i, int q) { return (i >> 2) * 16 + q * 4 + (i & 3); }

// Four adjacent elements at their own alignment (global memory takes vector loads at any).
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) row_four { T v[4]; };

// One row into the quad's registers; -infinity beyond the row's classes.  `left` is how many elements the matrix holds from
// the start of the row: a run of four that reaches into the next row is loaded whole, at the end of the matrix one by one.
template <int DT, int E>
__device__ __forceinline__ void quad_load(const typename row_type<DT>::type* row, int n_classes, int64_t left, int q, float (&x)[E]) {
    using T = typename row_type<DT>::type;
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        const int c = g * 16 + q * 4;
        row_four<T> f = {};
        if (c < n_classes) {
            if (c + 4 <= left) {
                f = *(const row_four<T>*)(row + c);
            } else {
                for (int j = 0; j < 4 && c + j < n_classes; ++j) f.v[j] = row[c + j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[g * 4 + j] = c + j < n_classes ? (float)f.v[j] : -INFINITY;
    }
}

// The run of four elements that register group g of lane q stands for, into a row of n_classes elements.
template <typename T> __device__ __forceinline__ void quad_store(T* row, int n_classes, int g, int q, const float (&v)[4]) {
    const int c = g * 16 + q * 4;
    row_four<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = (T)v[j];
    if (c + 4 <= n_classes) {
        *(row_four<T>*)(row + c) = f;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < n_classes) row[c + j] = f.v[j];
    }
}

// orders the LDS accesses of one wavefront's lanes (they execute in order; the compiler must not move them)
__device__ __forceinline__ void row_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// An entry of a short row as a double in [2, 4): key and complemented class in the low 39 bits.  Doubles of one sign sort
// like their bits, so one maximum and one minimum instruction order two entries.  An absent score gives QUAD_NONE + class
// bits, below every entry.
#define QUAD_NONE 0x4000000000000000ll
__device__ __forceinline__ double quad_entry(uint32_t key, int cls) {
    return __longlong_as_double(QUAD_NONE | (long long)key << 7 | (127 - cls));
}
__device__ __forceinline__ uint32_t quad_entry_key(double e) { return (uint32_t)(__double_as_longlong(e) >> 7); }
__device__ __forceinline__ int quad_entry_class(double e) { return 127 - (int)(__double_as_longlong(e) & 127); }

// larger one first
__device__ __forceinline__ void quad_order(double& a, double& b) {
    const double hi = row_max(a, b);
    b = row_min(a, b);
    a = hi;
}
// one lane's registers, descending (odd-even merge sort)
template <int E> __device__ __forceinline__ void quad_sort_lane(double (&e)[E]) {
#pragma unroll
    for (int p = 1; p < E; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < E; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < E && (i + j) / (2 * p) == (i + j + k) / (2 * p)) quad_order(e[i + j], e[i + j + k]);
}
// one lane's registers from a bitonic sequence to descending order
template <int E> __device__ __forceinline__ void quad_merge_lane(double (&e)[E]) {
#pragma unroll
    for (int d = E / 2; d >= 1; d /= 2)
#pragma unroll
        for (int i = 0; i < E; ++i)
            if ((i & d) == 0) quad_order(e[i], e[i + d]);
}
// The quad's 4 E entries in descending order, lane q with places q E ... q E + E - 1.
template <int E> __device__ __forceinline__ void quad_sort(double (&e)[E], int q) {
    double o[E];
    quad_sort_lane(e);
    const bool odd = q & 1, upper = q & 2;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR1>(e[E - 1 - i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = odd ? row_min(e[i], o[i]) : row_max(e[i], o[i]);
    quad_merge_lane(e);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR3>(e[E - 1 - i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = upper ? row_min(e[i], o[i]) : row_max(e[i], o[i]);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR1>(e[i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = odd ? row_min(e[i], o[i]) : row_max(e[i], o[i]);
    quad_merge_lane(e);
}
// The first E of the quad's entries in descending order, the same in all four lanes.
template <int E> __device__ __forceinline__ void quad_sort_head(double (&e)[E]) {
    double o[E];
    quad_sort_lane(e);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR1>(e[E - 1 - i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = row_max(e[i], o[i]);
    quad_merge_lane(e);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR2>(e[E - 1 - i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = row_max(e[i], o[i]);
    quad_merge_lane(e);
}

// the instantiation for a row's width: registers per lane
#define LSR_QUAD_SWITCH(classes, ...)                                          \
    do {                                                                       \
        if ((classes) <= 16) { constexpr int E = 4; __VA_ARGS__; }             \
        else if ((classes) <= 32) { constexpr int E = 8; __VA_ARGS__; }        \
        else if ((classes) <= 64) { constexpr int E = 16; __VA_ARGS__; }       \
        else { constexpr int E = 32; __VA_ARGS__; }                            \
    } while (0)
#define LSR_DTYPE_SWITCH(dtype, ...)                                           \
    do {                                                                       \
        if ((dtype) == LSR_F32) { constexpr int DT = ROW_F32; __VA_ARGS__; }   \
        else if ((dtype) == LSR_F16) { constexpr int DT = ROW_F16; __VA_ARGS__; } \
        else { constexpr int DT = ROW_BF16; __VA_ARGS__; }                     \
    } while (0)
