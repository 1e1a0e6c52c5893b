// Device helpers shared by the operators that read rows of log scores (lsr_top.hip, lsr_sample.hip, lsr_distill.hip).
//
// Order of a row: value descending, equal values by ascending class.  A score becomes a 32-bit key that sorts like the
// value (sign-magnitude turned into an unsigned number; -0 and +0 are one value), absent scores (-inf and NaN) get key 0;
// key and complemented class together are a 64-bit number that is different for every entry of a row, so that "the first
// m entries" is always "the entries whose number is at least some threshold".
#pragma once

#include <type_traits>

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

// 2^y for y <= 0 to 2^-50 of the result: the fraction in [-1/2, 1/2] goes through a polynomial of degree 10 that is 1 at 0
// (interpolation of (2^f - 1) / f at the Chebyshev nodes, largest relative error 5.6e-16).  16 instructions, all of them of
// the rate of 32-bit ones on this part; the library's exp takes about three times as many.  The coefficients are held in
// scalar registers from the object's creation on: as literals each would be moved into the accumulator first, two
// instructions more per step.  0 for -infinity and NaN.
struct row_exp2_t {
    double c10 = 7.070977866508138e-09, c9 = 1.0205905413765595e-07, c8 = 1.3215451633221434e-06, c7 = 1.5252672924850737e-05,
           c6 = 0.00015403530424776529, c5 = 0.0013333558200794592, c4 = 0.009618129107618665, c3 = 0.05550410866465167,
           c2 = 0.24022650695910075, c1 = 0.6931471805599462, low = -1200.0;
    __device__ __forceinline__ row_exp2_t() {
        asm("" : "+s"(c10), "+s"(c9), "+s"(c8), "+s"(c7), "+s"(c6), "+s"(c5));
        asm("" : "+s"(c4), "+s"(c3), "+s"(c2), "+s"(c1), "+s"(low));
    }
    __device__ __forceinline__ double operator()(double y) const {
        y = fmax(y, low);
        const double n = __builtin_rint(y), f = y - n;
        double p = __builtin_fma(f, c10, c9);
        p = __builtin_fma(p, f, c8);
        p = __builtin_fma(p, f, c7);
        p = __builtin_fma(p, f, c6);
        p = __builtin_fma(p, f, c5);
        p = __builtin_fma(p, f, c4);
        p = __builtin_fma(p, f, c3);
        p = __builtin_fma(p, f, c2);
        p = __builtin_fma(p, f, c1);
        p = __builtin_fma(p, f, 1.0);
        return __builtin_amdgcn_ldexp(p, (int)n);
    }
};
#define ROW_LOG2E 1.4426950408889634
// Natural logarithm of a positive number to 2^-49 of the result (or 2^-49 for numbers near 1): x = m 2^e with m in
// [sqrt(1/2), sqrt(2)), ln m = 2 artanh(s) with s = (m - 1) / (m + 1), |s| < 0.172, by its series up to s^19 (the next term
// is 2^-58).  The library's log needs several times the registers, which long rows do not have to spare.
__device__ __forceinline__ double row_log(double x) {
    double m = __builtin_amdgcn_frexp_mant(x);            // [1/2, 1)
    int e = __builtin_amdgcn_frexp_exp(x);
    if (m < 0.7071067811865476) {
        m *= 2;
        --e;
    }
    const double s = (m - 1) / (m + 1), q = s * s;
    double p = 1.0 / 19;
    p = __builtin_fma(p, q, 1.0 / 17);
    p = __builtin_fma(p, q, 1.0 / 15);
    p = __builtin_fma(p, q, 1.0 / 13);
    p = __builtin_fma(p, q, 1.0 / 11);
    p = __builtin_fma(p, q, 1.0 / 9);
    p = __builtin_fma(p, q, 1.0 / 7);
    p = __builtin_fma(p, q, 1.0 / 5);
    p = __builtin_fma(p, q, 1.0 / 3);
    p = __builtin_fma(p, q, 1.0);
    return (double)e * 0.6931471805599453 + 2 * s * p;
}

// Weights of entries as whole numbers: w in [0, 1] in units of 2^-shift, so that sums do not depend on the order of
// addition.  Adding 2^(52 - shift) leaves the rounded number in the low bits of the double.
__device__ __forceinline__ uint64_t row_fixed(double w, double magic) {
    return (uint64_t)__double_as_longlong(w + magic) - (uint64_t)__double_as_longlong(magic);
}

static inline int row_dtype_bytes(int dtype) { return dtype == LSR_F32 ? 4 : 2; }

// Rows of one launch: a grid has fewer than 2^32 threads.  The entry points take more rows in several launches.
static inline int64_t lsr_launch_rows(int64_t n_classes) { return n_classes <= 128 ? (int64_t)1 << 29 : (int64_t)1 << 21; }

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
template <int PERM> __device__ __forceinline__ uint32_t quad_move(uint32_t v) { return (uint32_t)quad_move<PERM>((int)v); }
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
        if (g * 16 + 16 <= n_classes) {                   // the same in all rows: no lane reaches the row's end
            const row_four<T> f = *(const row_four<T>*)(row + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[g * 4 + j] = (float)f.v[j];
        } else {
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
}
// -infinity for NaN, +0 for -0: the sum quietens a signalling NaN, a maximum passes over a quiet one
__device__ __forceinline__ float row_clean(float x) { return fmaxf(x + 0.0f, -INFINITY); }

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

// sixteen bytes at any alignment of their elements
typedef uint32_t row_words __attribute__((ext_vector_type(4), aligned(2)));

// orders the LDS accesses of one wavefront's lanes (they execute in order; the compiler must not move them)
__device__ __forceinline__ void row_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// An entry of a short row as a double in [2, 4): the score's key and the complemented class in the low 39 bits.  Doubles of
// one sign sort like their bits, so one maximum and one minimum instruction order two entries.  An absent score, cleaned
// to -infinity, has a key like any other, below those of all scores that are present.
__device__ __forceinline__ double quad_entry(float x, int cls) {
    const uint32_t u = __float_as_uint(x), key = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return __longlong_as_double(0x4000000000000000ll | (long long)key << 7 | (127 - cls));
}
__device__ __forceinline__ float quad_entry_value(double e) { return row_value((uint32_t)(__double_as_longlong(e) >> 7)); }
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
    for (int i = 0; i < E; ++i) e[i] = (e[i] < o[i]) != odd ? o[i] : e[i];
    quad_merge_lane(e);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR3>(e[E - 1 - i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = (e[i] < o[i]) != upper ? o[i] : e[i];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = quad_move<QUAD_XOR1>(e[i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = (e[i] < o[i]) != odd ? o[i] : e[i];
    quad_merge_lane(e);
}
// The first H of the quad's entries in descending order in e[0 ... H - 1], the same in all four lanes (H a power of two, at
// most E): runs of H are sorted, then two at a time only the better half of them is kept and put in order again.
template <int E, int H> __device__ __forceinline__ void quad_sort_head(double (&e)[E]) {
#pragma unroll
    for (int g = 0; g < E; g += H) {
        double s[H];
#pragma unroll
        for (int i = 0; i < H; ++i) s[i] = e[g + i];
        quad_sort_lane<H>(s);
#pragma unroll
        for (int i = 0; i < H; ++i) e[g + i] = s[i];
    }
    double h[H], o[H];
#pragma unroll
    for (int n = E / H; n > 1; n /= 2)
#pragma unroll
        for (int g = 0; g < n / 2; ++g) {
#pragma unroll
            for (int i = 0; i < H; ++i) h[i] = row_max(e[2 * g * H + i], e[(2 * g + 1) * H + H - 1 - i]);
            quad_merge_lane<H>(h);
#pragma unroll
            for (int i = 0; i < H; ++i) e[g * H + i] = h[i];
        }
#pragma unroll
    for (int i = 0; i < H; ++i) h[i] = e[i];
#pragma unroll
    for (int i = 0; i < H; ++i) o[i] = quad_move<QUAD_XOR1>(h[H - 1 - i]);
#pragma unroll
    for (int i = 0; i < H; ++i) h[i] = row_max(h[i], o[i]);
    quad_merge_lane<H>(h);
#pragma unroll
    for (int i = 0; i < H; ++i) o[i] = quad_move<QUAD_XOR2>(h[H - 1 - i]);
#pragma unroll
    for (int i = 0; i < H; ++i) e[i] = row_max(h[i], o[i]);
#pragma unroll
    for (int i = 0; i < H; ++i) h[i] = e[i];
    quad_merge_lane<H>(h);
#pragma unroll
    for (int i = 0; i < H; ++i) e[i] = h[i];
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

// ---- long rows: a team of W wavefronts holds a row ---------------------------------------------------------------------
// Thread t of a team has the runs of 16 bytes t, t + 64 W, t + 128 W, ... of the row: N of them stay in registers from
// the first read on (N = 0: the row is too long for that and every pass reads it again, mostly from L2).
template <int CTRL, int ROWS> __device__ __forceinline__ int wave_shift(int v, int fill) {
    return __builtin_amdgcn_update_dpp(fill, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ float wave_shift(float v, float fill) {
    return __int_as_float(wave_shift<CTRL, ROWS>(__float_as_int(v), __float_as_int(fill)));
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t wave_shift(uint64_t v, uint64_t fill) {
    const uint32_t lo = wave_shift<CTRL, ROWS>((int)v, (int)fill), hi = wave_shift<CTRL, ROWS>((int)(v >> 32), (int)(fill >> 32));
    return (uint64_t)hi << 32 | lo;
}
template <int CTRL, int ROWS> __device__ __forceinline__ double wave_shift(double v, double fill) {
    return __longlong_as_double((long long)wave_shift<CTRL, ROWS>((uint64_t)__double_as_longlong(v), (uint64_t)__double_as_longlong(fill)));
}
// running combination over the lanes of a wavefront, in the same order every time; lane 63 has the whole
#define WAVE_SCAN(v, fill, op)                             \
    do {                                                   \
        v = op(v, wave_shift<0x111, 0xf>(v, fill));        \
        v = op(v, wave_shift<0x112, 0xf>(v, fill));        \
        v = op(v, wave_shift<0x114, 0xf>(v, fill));        \
        v = op(v, wave_shift<0x118, 0xf>(v, fill));        \
        v = op(v, wave_shift<0x142, 0xa>(v, fill));        \
        v = op(v, wave_shift<0x143, 0xc>(v, fill));        \
    } while (0)
template <typename V> __device__ __forceinline__ V row_add(V a, V b) { return a + b; }
__device__ __forceinline__ uint64_t row_max(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t row_max(uint32_t a, uint32_t b) { return max(a, b); }
__device__ __forceinline__ uint32_t row_min(uint32_t a, uint32_t b) { return min(a, b); }

__device__ __forceinline__ float wave_last(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ __forceinline__ int wave_last(int v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ uint64_t wave_last(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)v, 63), hi = __builtin_amdgcn_readlane((int)(v >> 32), 63);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ double wave_last(double v) {
    return __longlong_as_double((long long)wave_last((uint64_t)__double_as_longlong(v)));
}
template <typename V> __device__ __forceinline__ V wave_running(V v) {
    WAVE_SCAN(v, (V)0, row_add);
    return v;
}
template <typename V> __device__ __forceinline__ V wave_sum(V v) { return wave_last(wave_running(v)); }
__device__ __forceinline__ float wave_max(float v) {
    WAVE_SCAN(v, -INFINITY, row_max);
    return wave_last(v);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    WAVE_SCAN(v, (uint64_t)0, row_max);
    return wave_last(v);
}

template <int W> __device__ __forceinline__ void team_sync() {
    if (W == 1)
        row_wave_fence();
    else
        __syncthreads();
}
// Sum / maximum over the team, returned to every thread; `shared` has W places and may be used again at once (two
// barriers; one wavefront needs none).
template <int W, typename V> __device__ __forceinline__ V team_sum(V v, V* shared) {
    v = wave_sum(v);
    if (W == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    V sum = shared[0];
#pragma unroll
    for (int i = 1; i < W; ++i) sum += shared[i];
    return sum;
}
template <int W, typename V> __device__ __forceinline__ V team_max(V v, V* shared) {
    v = wave_max(v);
    if (W == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    V most = shared[0];
#pragma unroll
    for (int i = 1; i < W; ++i) most = row_max(most, shared[i]);
    return most;
}

template <int DT, int W, int N> struct team_row {
    using T = typename row_type<DT>::type;
    // A thread's sum over a row: a kept row has at most 128 terms per thread, one that is read again up to 2^14 (of equal
    // size, as a rule, so that 32-bit sums would be off to one side): those are added up in 64 bits, run by run.
    using sum_t = std::conditional_t<(N > 0), float, double>;
    static constexpr int RUN = 16 / (int)sizeof(T), THREADS = 64 * W, STEP = THREADS * RUN;   // classes of a run, of a step

    const T* row;
    int n_classes, steps, thread;
    uint4 kept[N ? N : 1];

    static __device__ __forceinline__ uint4 nothing() {   // a run of -infinity
        const uint32_t w = DT == ROW_F32 ? 0xff800000u : DT == ROW_F16 ? 0xfc00fc00u : 0xff80ff80u;
        return make_uint4(w, w, w, w);
    }
    __device__ __forceinline__ int first_class(int step) const { return step * STEP + thread * RUN; }

    // the run of the row's last classes, one element at a time
    __device__ __forceinline__ uint4 read_end(int c) const {
        uint32_t w[4] = {nothing().x, nothing().x, nothing().x, nothing().x};
        for (int j = 0; j < RUN && c + j < n_classes; ++j) {
            uint32_t b;
            if constexpr (DT == ROW_F32)
                b = __float_as_uint(row[c + j]);
            else
                b = __builtin_bit_cast(uint16_t, row[c + j]);
#pragma unroll
            for (int i = 0; i < RUN; ++i)
                if (i == j) w[i * 4 / RUN] = RUN == 4 ? b : i & 1 ? (w[i * 4 / RUN] & 0xffffu) | b << 16 : (w[i * 4 / RUN] & 0xffff0000u) | b;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // Loads are not under a condition (the compiler would wait for each before the next): a run that is not whole takes the
    // row's first one, and `settle` blanks it.
    __device__ __forceinline__ uint4 read(int step) const {
        const int c = first_class(step);
        // 32-bit offset from a wave-uniform address: one address register per load
        const uint32_t at = c + RUN <= n_classes ? (uint32_t)c * (uint32_t)sizeof(T) : 0u;
        // rows of a team of 16 do not stay in a first-level cache anyway: not asking for it is 4 to 8 % faster there (4096 x
        // 131072 with gradient 546 -> 524 us), and 4 % slower for the shorter rows of the smaller teams
        if constexpr (W == 16) {
            const row_words v = __builtin_nontemporal_load((const row_words*)((const char*)row + at));
            return make_uint4(v.x, v.y, v.z, v.w);
        } else {
            const row_words v = *(const row_words*)((const char*)row + at);
            return make_uint4(v.x, v.y, v.z, v.w);
        }
    }
    __device__ __forceinline__ uint4 settle(int step, const uint4& u) const {
        const bool whole = first_class(step) + RUN <= n_classes;
        return make_uint4(whole ? u.x : nothing().x, whole ? u.y : nothing().y, whole ? u.z : nothing().z, whole ? u.w : nothing().w);
    }
    __device__ __forceinline__ uint4 read_any(int step) const {
        const int c = first_class(step);
        return c < n_classes && c + RUN > n_classes ? read_end(c) : settle(step, read(step));
    }
    __device__ __forceinline__ void open(const T* r, int classes) {
        row = r;
        n_classes = classes;
        steps = (classes + STEP - 1) / STEP;
        thread = threadIdx.x;
        if (N) {
#pragma unroll
            for (int i = 0; i < (N ? N : 1); ++i) kept[i] = read(i);
        }
    }
    // each_run of a kept row, and right behind each run the request for the same run of the next row
    template <typename F> __device__ __forceinline__ void each_run_then(const T* next, F f) {
        row = next;
#pragma unroll
        for (int i = 0; i < (N ? N : 1); ++i) {
            f(i, kept[i]);
            asm volatile("" ::: "memory");               // the load stays behind the run's last use
            __builtin_amdgcn_sched_barrier(0);
            kept[i] = read(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // waits for the row that `open` has requested
    __device__ __forceinline__ void arrive() {
        // the classes of all runs would otherwise be computed once, before a loop over rows, and kept in registers
        asm volatile("" : "+v"(thread));
        if (N) {
#pragma unroll
            for (int i = 0; i < (N ? N : 1); ++i) kept[i] = settle(i, kept[i]);
            const int end = first_class(steps - 1);
            if (end < n_classes && end + RUN > n_classes) {
                const uint4 u = read_end(end);
#pragma unroll
                for (int i = 0; i < (N ? N : 1); ++i)
                    if (i == steps - 1) kept[i] = u;
            }
        }
    }
    // Between two passes: the compiler is to decode the runs again, not to keep every decoded value of the first pass in
    // registers for the second (which would not fit and spill).
    __device__ __forceinline__ void next_pass() {
        if (N) {
#pragma unroll
            for (int i = 0; i < (N ? N : 1); ++i) asm volatile("" : "+v"(kept[i].x), "+v"(kept[i].y), "+v"(kept[i].z), "+v"(kept[i].w));
        }
    }
    static __device__ __forceinline__ void decode(const uint4& u, float (&v)[RUN]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if (DT == ROW_F32) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] = __uint_as_float(w[i & 3]);
        } else if (DT == ROW_BF16) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] = __uint_as_float(i & 1 ? w[i >> 1 & 3] & 0xffff0000u : w[i >> 1 & 3] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < RUN; ++i)
                v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i >> 1 & 3] >> 16 : w[i >> 1 & 3]));
        }
    }
    // f(step, run) for every step of the row; rows that are not kept are read `AHEAD` steps at a time, so that as many loads
    // are on their way while a pass does little with each
    template <int AHEAD, typename F> __device__ __forceinline__ void each_run(F f) {
        if (N) {
#pragma unroll
            for (int i = 0; i < (N ? N : 1); ++i) f(i, kept[i]);
        } else {
            const int end = n_classes % RUN ? steps - 1 : steps;        // the last step may have the run that is cut short
            int i = 0;
            for (; i + AHEAD <= end; i += AHEAD) {
                uint4 u[AHEAD];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) u[j] = read(i + j);
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) f(i + j, settle(i + j, u[j]));
            }
#pragma unroll 1
            for (; i < steps; ++i) {
                f(i, read_any(i));
            }
        }
    }
    // f(step, values of the thread's run, first class of the run)
    template <int AHEAD, typename F> __device__ __forceinline__ void each(F f) {
        each_run<AHEAD>([&](int i, const uint4& u) {
            float v[RUN];
            decode(u, v);
            f(i, v, first_class(i));
        });
    }
};

// ---- the first entries of a long row ------------------------------------------------------------------------------------
// The classes of a row are dealt out to ROW_GROUPS groups; the kk-th largest of the groups' best scores is a lower bound of
// the row's kk-th largest score, as kk groups have a score that high.  One pass finds the groups' best, a second collects
// what reaches the bound: for scores in no particular order about -G ln(1 - kk / G) entries of G = 256 groups, 73 for
// kk = 64.  Places follow from counting, for each entry, the entries above it.
#define ROW_GROUPS 256
template <int W, int SIZE> struct team_list {
    static constexpr int ROOM = SIZE;
    uint64_t entry[SIZE];
    alignas(16) uint32_t group[ROW_GROUPS];
    int n;
    uint32_t bound;                                       // a key
};

// The groups' best scores of a row, and the row's.
template <int DT, int W, int N, int SIZE>
__device__ __forceinline__ float team_groups(team_row<DT, W, N>& row, team_list<W, SIZE>& list) {
    constexpr int THREADS = 64 * W, RUN = team_row<DT, W, N>::RUN, PER = W == 1 ? 4 : 1;
    const int tid = threadIdx.x;
    float most[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) most[i] = -INFINITY;
    row.template each<4>([&](int step, const float(&v)[RUN], int) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (W == 1 && step % PER != i) continue;
#pragma unroll
            for (int j = 0; j < RUN; ++j) most[i] = row_max(most[i], v[j]);
        }
    });
    if (W == 1) {
#pragma unroll
        for (int i = 0; i < ROW_GROUPS / 64; ++i) list.group[i * 64 + tid] = row_key(most[i < PER ? i : 0]);
    } else {
        float best = most[0];
        if (W >= 8) best = row_max(best, quad_move<QUAD_XOR1>(best));
        if (W >= 16) best = row_max(best, quad_move<QUAD_XOR2>(best));
        constexpr int LANES = W == 1 ? 1 : THREADS / ROW_GROUPS;        // of a group
        if (tid % LANES == 0) list.group[tid / LANES] = row_key(best);
    }
    team_sync<W>();
    const uint4 o = *(const uint4*)&list.group[(tid & 63) * 4];         // every wavefront for itself
    const uint32_t a = o.x > o.y ? o.x : o.y, b = o.z > o.w ? o.z : o.w;
    const uint32_t best = (uint32_t)wave_max((uint64_t)(a > b ? a : b));
    return best ? row_value(best) : -INFINITY;
}
// Collects the entries that reach `bound`; `list.n`, 0 on entry, may exceed the list's size: then only some of them are there.
// SUM: also this thread's sum of e^((x - bound) unit ln 2) over what stays below the bound, in the same pass, added to
// `below`; NaN where the thread has seen one.  NEXT: a kept row is asked for the next row, `next`, on the way.
template <bool SUM, bool NEXT, int DT, int W, int N, int SIZE>
__device__ __forceinline__ void team_take(team_row<DT, W, N>& row, float bound, team_list<W, SIZE>& list, float unit,
                                          typename team_row<DT, W, N>::sum_t& below, const typename row_type<DT>::type* next) {
    constexpr int RUN = team_row<DT, W, N>::RUN;
    row.next_pass();
    auto take = [&](int step, const uint4& packed) {
        float v[RUN];
        team_row<DT, W, N>::decode(packed, v);
        const int c = row.first_class(step);
        bool any = false;
        float sum = N ? below : 0.0f;
#pragma unroll
        for (int j = 0; j < RUN; ++j) any |= v[j] >= bound;
        if (any) {
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                if (v[j] >= bound) {
                    const int at = atomicAdd(&list.n, 1);
                    if (at < SIZE) list.entry[at] = row_entry(row_key(v[j]), c + j);
                }
                if (SUM) sum += v[j] < bound ? __builtin_amdgcn_exp2f((v[j] - bound) * unit) : 0.0f;
            }
        } else if (SUM) {
#pragma unroll
            for (int j = 0; j < RUN; ++j) sum += __builtin_amdgcn_exp2f((v[j] - bound) * unit);
        }
        if (SUM) below = N ? sum : below + sum;
    };
    if constexpr (NEXT)
        row.each_run_then(next, take);
    else
        row.template each_run<4>(take);
    team_sync<W>();
}
// The bound of kk as a score, -FLT_MAX when fewer groups than that have a score; empties the list.
template <int W, int SIZE> __device__ __forceinline__ float team_bound(int kk, team_list<W, SIZE>& list) {
    const int tid = threadIdx.x;
    if (tid < 64) {                                       // the largest number that kk groups reach, bit by bit
        const uint4 o = *(const uint4*)&list.group[tid * 4];
        uint32_t bound = 0;
#pragma unroll 1
        for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
            const uint32_t b = bound | bit;
            const int reach = __popcll(__ballot(o.x >= b)) + __popcll(__ballot(o.y >= b)) + __popcll(__ballot(o.z >= b)) +
                              __popcll(__ballot(o.w >= b));
            if (reach >= kk) bound = b;
        }
        if (tid == 0) {
            list.bound = bound;
            list.n = 0;
        }
    }
    team_sync<W>();
    return list.bound ? row_value(list.bound) : -3.402823466e38f;
}
// how many of the list's first n entries are above e
template <int W, int SIZE> __device__ __forceinline__ int team_above(const team_list<W, SIZE>& list, int n, uint64_t e) {
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) above += list.entry[i] > e;
    return above;
}

// Sorting 64 E numbers of a wavefront, largest first; lane l has the places l E ... l E + E - 1.  A bitonic network whose
// merges begin with a mirrored step, so that every step keeps the larger number in the lower place.
template <int X, typename V> __device__ __forceinline__ V wave_xor(V v) {              // of lane l ^ X
    if constexpr (X == 1) return quad_move<QUAD_XOR1>(v);
    else if constexpr (X == 2) return quad_move<QUAD_XOR2>(v);
    else if constexpr (X == 3) return quad_move<QUAD_XOR3>(v);
    else if constexpr (X == 7) return quad_move<0x141>(v);               // the halves of 16 lanes mirrored
    else if constexpr (X == 8) return quad_move<0x128>(v);               // 16 lanes rotated by 8
    else if constexpr (X == 15) return quad_move<0x140>(v);              // 16 lanes mirrored
    else return __shfl_xor(v, X);
}
template <int E, typename V> __device__ __forceinline__ void wave_sort_own(V (&e)[E]) {
#pragma unroll
    for (int s = E / 2; s; s /= 2)
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (!(i & s)) {
                const V a = e[i], b = e[i + s];
                e[i] = row_max(a, b);
                e[i + s] = row_min(a, b);
            }
}
template <int X, bool MIRROR, int E, typename V> __device__ __forceinline__ void wave_sort_step(V (&e)[E]) {
    const bool upper = threadIdx.x & (MIRROR ? (X + 1) / 2 : X);
    V o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = wave_xor<X>(e[MIRROR ? E - 1 - i : i]);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = upper ? row_min(e[i], o[i]) : row_max(e[i], o[i]);
}
template <int M, int E, typename V> __device__ __forceinline__ void wave_sort_merge(V (&e)[E]) {      // over M lanes
    wave_sort_step<M - 1, true>(e);
    if constexpr (M > 32) wave_sort_step<16, false>(e);
    if constexpr (M > 16) wave_sort_step<8, false>(e);
    if constexpr (M > 8) wave_sort_step<4, false>(e);
    if constexpr (M > 4) wave_sort_step<2, false>(e);
    if constexpr (M > 2) wave_sort_step<1, false>(e);
    wave_sort_own(e);
}
template <int E, typename V> __device__ __forceinline__ void wave_sort(V (&e)[E]) {
#pragma unroll
    for (int k = 2; k <= E; k *= 2) {
        // pairs that are mirrored in their group of k
#pragma unroll
        for (int i = 0; i < E; ++i)
            if ((i & (k - 1)) < k / 2) {
                const int j = (i & ~(k - 1)) + k - 1 - (i & (k - 1));
                const V a = e[i], b = e[j];
                e[i] = row_max(a, b);
                e[j] = row_min(a, b);
            }
#pragma unroll
        for (int s = k / 4; s; s /= 2)
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (!(i & s)) {
                    const V a = e[i], b = e[i + s];
                    e[i] = row_max(a, b);
                    e[i + s] = row_min(a, b);
                }
    }
    wave_sort_merge<2>(e);
    wave_sort_merge<4>(e);
    wave_sort_merge<8>(e);
    wave_sort_merge<16>(e);
    wave_sort_merge<32>(e);
    wave_sort_merge<64>(e);
}
// Puts the first 64 E entries of a list of n in order, by one wavefront.  Key and class take 56 bits and are compared as
// floating-point numbers, for which there is an instruction.
template <int E, int W, int SIZE> __device__ __forceinline__ void team_sort(const team_list<W, SIZE>& list, int n, uint64_t* sorted, int room) {
    double e[E];
    const int lane = threadIdx.x;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint64_t u = i * 64 + lane < n ? list.entry[i * 64 + lane] : 0;
        e[i] = __longlong_as_double((long long)(u >> 32 << 24 | (u & 0xffffffu)));
    }
    wave_sort(e);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint64_t u = (uint64_t)__double_as_longlong(e[i]);
        if (lane * E + i < room) sorted[lane * E + i] = u >> 24 << 32 | 0xff000000u | (u & 0xffffffu);
    }
}
// The list's entries by place, `room` of them at most.  Up to 128 are compared with all others, more are sorted if SORT: the
// comparisons wait for shared memory, one read for every 64 of them (4096 x 1000, k = 200: 76 us, sorted 27).
template <bool SORT, int W, int SIZE> __device__ __forceinline__ void team_order(const team_list<W, SIZE>& list, int n, uint64_t* sorted, int room) {
    if (SORT && n > 128 && n <= 512) {
        if (threadIdx.x < 64) {
            if (n <= 256)
                team_sort<4>(list, n, sorted, room);
            else
                team_sort<8>(list, n, sorted, room);
        }
        return;
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += 64 * W) {
        const uint64_t e = list.entry[i];
        const int place = team_above(list, n, e);
        if (place < room) sorted[place] = e;
    }
}

// Wavefronts per row by the row's width, W, and the runs of it that a thread keeps in registers, N; LSR_WAVES_SWITCH for an
// operator that keeps none.
#define LSR_TEAM_SWITCH(dtype, classes, ...)                                                              \
    do {                                                                                                  \
        if ((dtype) == LSR_F32) {                                                                         \
            constexpr int DT = ROW_F32;                                                                   \
            if ((classes) <= 1024) { constexpr int W = 1, N = 4; __VA_ARGS__; }                           \
            else if ((classes) <= 4096) { constexpr int W = 4, N = 4; __VA_ARGS__; }                      \
            else if ((classes) <= 8192) { constexpr int W = 4, N = 8; __VA_ARGS__; }                      \
            else if ((classes) <= 16384) { constexpr int W = 8, N = 8; __VA_ARGS__; }                     \
            else if ((classes) <= 32768) { constexpr int W = 8, N = 16; __VA_ARGS__; }                    \
            else if ((classes) <= 65536) { constexpr int W = 16, N = 16; __VA_ARGS__; }                   \
            else { constexpr int W = 16, N = 0; __VA_ARGS__; }                                            \
        } else if ((dtype) == LSR_F16) {                                                                  \
            constexpr int DT = ROW_F16;                                                                   \
            LSR_TEAM_SWITCH_16(classes, __VA_ARGS__);                                                     \
        } else {                                                                                          \
            constexpr int DT = ROW_BF16;                                                                  \
            LSR_TEAM_SWITCH_16(classes, __VA_ARGS__);                                                     \
        }                                                                                                 \
    } while (0)
#define LSR_TEAM_SWITCH_16(classes, ...)                                                                  \
    do {                                                                                                  \
        if ((classes) <= 1024) { constexpr int W = 1, N = 2; __VA_ARGS__; }                               \
        else if ((classes) <= 4096) { constexpr int W = 4, N = 2; __VA_ARGS__; }                          \
        else if ((classes) <= 16384) { constexpr int W = 4, N = 8; __VA_ARGS__; }                         \
        else if ((classes) <= 32768) { constexpr int W = 8, N = 8; __VA_ARGS__; }                         \
        else if ((classes) <= 65536) { constexpr int W = 8, N = 16; __VA_ARGS__; }                        \
        else if ((classes) <= 131072) { constexpr int W = 16, N = 16; __VA_ARGS__; }                      \
        else { constexpr int W = 16, N = 0; __VA_ARGS__; }                                                \
    } while (0)
#define LSR_WAVES_SWITCH(classes, ...)                                                                    \
    do {                                                                                                  \
        if ((classes) <= 1024) { constexpr int W = 1; __VA_ARGS__; }                                      \
        else if ((classes) <= 16384) { constexpr int W = 4; __VA_ARGS__; }                                \
        else { constexpr int W = 16; __VA_ARGS__; }                                                       \
    } while (0)
