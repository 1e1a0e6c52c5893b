// The k best classes of every row of log scores, and the log weight of the rest.
//
// Radix selection: the threshold of the first k entries (lsr_rows.h) is found eight bits at a time from a histogram of
// the entries that still match it; the entries at or above it go to a list in LDS, which is sorted and written.
#include <math.h>

#include "lsr_rows.h"

int lsr_check_rows(lsr_ctx* ctx, const char* name, const void* scores_d, int dtype, int64_t n_rows, int64_t n_classes,
                   int64_t row_stride) {
    if (dtype != LSR_F32 && dtype != LSR_F16 && dtype != LSR_BF16)
        return lsr_fail(ctx, LSR_ERR_ARG, "%s: unknown element type %d", name, dtype);
    if (n_rows < 0 || n_classes < 1 || row_stride < 0) return lsr_fail(ctx, LSR_ERR_ARG, "%s: bad sizes", name);
    if (n_classes > LSR_MAX_CLASSES)
        return lsr_fail(ctx, LSR_ERR_LIMIT, "%s: %lld classes > %d", name, (long long)n_classes, LSR_MAX_CLASSES);
    if (n_rows > 0 && !scores_d) return lsr_fail(ctx, LSR_ERR_ARG, "%s: null pointer", name);
    if ((uintptr_t)scores_d % row_dtype_bytes(dtype))
        return lsr_fail(ctx, LSR_ERR_ARG, "%s: scores are not aligned to their element size", name);
    return LSR_OK;
}

template <int DT>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_top_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                                  int64_t n_rows, int n_classes, int64_t row_stride, int k,
                                                                  float inv_t, float* __restrict__ values,
                                                                  int32_t* __restrict__ index, float* __restrict__ rest) {
    __shared__ int hist[256];
    __shared__ uint64_t list[LSR_MAX_TOP];
    __shared__ uint64_t threshold;
    __shared__ int left, n_list;
    __shared__ float part[LSR_ROW_THREADS / 64];
    const int tid = threadIdx.x;
    for (int64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
        const typename row_type<DT>::type* x = scores + r * row_stride;
        if (tid == 0) {
            threshold = 0;
            left = k;
            n_list = 0;
        }
        for (int shift = 56; shift >= 0; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            const uint64_t high = threshold;
            for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
                const uint32_t key = row_key((float)x[c]);
                const uint64_t e = row_entry(key, c);
                if (key && (shift == 56 || (e >> (shift + 8)) == (high >> (shift + 8))))
                    atomicAdd(&hist[(e >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int need = left, d = 255;
                for (; d > 0 && hist[d] < need; --d) need -= hist[d];
                left = need;
                threshold = high | (uint64_t)d << shift;
            }
            __syncthreads();
        }
        const uint64_t least = threshold;
        list[tid] = 0;
        __syncthreads();
        for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
            const uint32_t key = row_key((float)x[c]);
            const uint64_t e = row_entry(key, c);
            if (key && e >= least) {
                const int at = atomicAdd(&n_list, 1);
                if (at < LSR_MAX_TOP) list[at] = e;
            }
        }
        __syncthreads();
        for (int size = 2; size <= LSR_MAX_TOP; size <<= 1)
            for (int step = size >> 1; step; step >>= 1) {
                const int other = tid ^ step;
                if (other > tid) {
                    const uint64_t a = list[tid], b = list[other];
                    if (((tid & size) == 0) == (a < b)) {
                        list[tid] = b;
                        list[other] = a;
                    }
                }
                __syncthreads();
            }
        if (tid < k) {
            const uint64_t e = list[tid];
            values[r * k + tid] = e ? row_value((uint32_t)(e >> 32)) : -INFINITY;
            index[r * k + tid] = e ? (int32_t)~(uint32_t)e : -1;
        }
        if (rest) {
            // relative to the highest score of the rest: relative to the row's best it could underflow to nothing
            const float best = list[0] ? row_value((uint32_t)(list[0] >> 32)) : 0.0f;
            float high = -INFINITY;
            for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
                const float v = (float)x[c];
                const uint32_t key = row_key(v);
                if (key && row_entry(key, c) < least) high = fmaxf(high, v);
            }
            for (int d = 32; d; d >>= 1) high = fmaxf(high, __shfl_xor(high, d));
            if ((tid & 63) == 0) part[tid >> 6] = high;
            __syncthreads();
            high = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
            __syncthreads();
            float sum = 0.0f;
            for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
                const float v = (float)x[c];
                const uint32_t key = row_key(v);
                if (key && row_entry(key, c) < least) sum += v == high ? 1.0f : expf((v - high) * inv_t);
            }
            sum = row_wave_sum(sum);
            if ((tid & 63) == 0) part[tid >> 6] = sum;
            __syncthreads();
            if (tid == 0)
                rest[r] = high > -INFINITY ? (high == best ? 0.0f : (high - best) * inv_t) + logf(part[0] + part[1] + part[2] + part[3])
                                           : -INFINITY;
        }
        __syncthreads();
    }
}

// Short rows (at most LSR_QUAD_CLASSES classes), a quad per row: the entries are sorted by a network over the quad's
// registers; for k <= E only the first E places are merged, which drops half of every exchange between lanes.
template <int DT, int E, bool HEAD, bool REST>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_top_quad_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                                       int64_t n_rows, int n_classes, int64_t row_stride, int k,
                                                                       float inv_t, float* __restrict__ values,
                                                                       int32_t* __restrict__ index, float* __restrict__ rest) {
    const int q = threadIdx.x & 3;
    const int64_t row = (int64_t)blockIdx.x * LSR_QUAD_ROWS + (threadIdx.x >> 2);
    const bool live = row < n_rows;
    const int64_t r = live ? row : n_rows - 1;            // every lane takes part in the exchanges
    float x[E];
    quad_load<DT, E>(scores + r * row_stride, n_classes, (n_rows - 1 - r) * row_stride + n_classes, q, x);
    double e[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] = x[i] > -INFINITY ? x[i] : -INFINITY;      // NaN is absent
        e[i] = quad_entry(row_key(x[i]), quad_class(i, q));
    }
    if (HEAD)
        quad_sort_head<E>(e);
    else
        quad_sort<E>(e, q);
    double least = 3.9;                                   // entry at place k - 1
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int place = HEAD ? i : q * E + i;
        if (REST) least = place == k - 1 ? e[i] : least;
        // with HEAD all lanes hold the same places: lane q writes the places that are q modulo 4
        if (live && place < k && (!HEAD || (place & 3) == q)) {
            const uint32_t key = quad_entry_key(e[i]);
            values[r * k + place] = key ? row_value(key) : -INFINITY;
            index[r * k + place] = key ? quad_entry_class(e[i]) : -1;
        }
    }
    if (!REST) return;
    if (!HEAD) least = quad_min(least);
    // the best entry is at place 0
    const double top = HEAD ? e[0] : quad_move<0x00>(e[0]);
    const uint32_t best_key = quad_entry_key(top);
    const float best = best_key ? row_value(best_key) : 0.0f;
    // relative to the highest score of the rest: relative to the row's best it could underflow to nothing
    const uint32_t last_key = quad_entry_key(least);
    const float last = last_key ? row_value(last_key) : -INFINITY;
    const int last_class = quad_entry_class(least);
    float high = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool beyond = x[i] < last || (x[i] == last && quad_class(i, q) > last_class);
        x[i] = beyond ? x[i] : -INFINITY;
        high = row_max(high, x[i]);
    }
    high = quad_max(high);
    float sum = 0.0f;
    const float unit = inv_t * 1.44269504f;
#pragma unroll
    for (int i = 0; i < E; ++i) sum += x[i] == high ? 1.0f : __builtin_amdgcn_exp2f((x[i] - high) * unit);
    sum = quad_sum(sum);
    if (live && q == 0)
        rest[r] = high > -INFINITY ? (high == best ? 0.0f : (high - best) * inv_t) + logf(sum) : -INFINITY;
}

template <int DT, int E>
static void lsr_top_quad(hipStream_t stream, const void* scores_d, int64_t n_rows, int n_classes, int64_t row_stride, int k,
                         float inv_t, float* values_d, int32_t* index_d, float* rest_d) {
    const auto* scores = (const typename row_type<DT>::type*)scores_d;
    const dim3 grid((unsigned)((n_rows + LSR_QUAD_ROWS - 1) / LSR_QUAD_ROWS));
#define LAUNCH(HEAD, REST)                                                                                                   \
    hipLaunchKernelGGL((lsr_top_quad_kernel<DT, E, HEAD, REST>), grid, dim3(LSR_ROW_THREADS), 0, stream, scores, n_rows,       \
                       n_classes, row_stride, k, inv_t, values_d, index_d, rest_d)
    if (k <= E) {
        if (rest_d) LAUNCH(true, true); else LAUNCH(true, false);
    } else {
        if (rest_d) LAUNCH(false, true); else LAUNCH(false, false);
    }
#undef LAUNCH
}

extern "C" int lsr_top_scores(lsr_ctx* ctx, const void* scores_d, int dtype, int64_t n_rows, int64_t n_classes,
                              int64_t row_stride, int k, double temperature, float* values_d, int32_t* index_d,
                              float* rest_d) {
    if (!ctx) return LSR_ERR_ARG;
    const int rc = lsr_check_rows(ctx, "lsr_top_scores", scores_d, dtype, n_rows, n_classes, row_stride);
    if (rc) return rc;
    if (k < 1 || k > n_classes) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_top_scores: k = %d outside 1..%lld", k, (long long)n_classes);
    if (k > LSR_MAX_TOP) return lsr_fail(ctx, LSR_ERR_LIMIT, "lsr_top_scores: k = %d > %d", k, LSR_MAX_TOP);
    if (!(temperature > 0) || !isfinite(temperature)) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_top_scores: temperature must be positive and finite");
    if (n_rows == 0) return LSR_OK;
    if (!values_d || !index_d) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_top_scores: null pointer");
    LSR_HIP_CHECK(ctx, hipSetDevice(ctx->device));
    const dim3 grid((unsigned)(n_rows < 65536 ? n_rows : 65536));
    const float inv_t = (float)(1.0 / temperature);
    lsr_prof_begin(ctx, LSR_K_TOP);
    if (n_classes <= LSR_QUAD_CLASSES) {
        LSR_DTYPE_SWITCH(dtype, LSR_QUAD_SWITCH(n_classes, lsr_top_quad<DT, E>(ctx->stream, scores_d, n_rows, (int)n_classes,
                                                                               row_stride, k, inv_t, values_d, index_d, rest_d)));
        lsr_prof_end(ctx);
        LSR_LAUNCH_CHECK(ctx, "lsr_top_quad_kernel");
        return LSR_OK;
    }
    if (dtype == LSR_F32)
        hipLaunchKernelGGL(lsr_top_kernel<ROW_F32>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const float*)scores_d,
                           n_rows, (int)n_classes, row_stride, k, inv_t, values_d, index_d, rest_d);
    else if (dtype == LSR_F16)
        hipLaunchKernelGGL(lsr_top_kernel<ROW_F16>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const _Float16*)scores_d,
                           n_rows, (int)n_classes, row_stride, k, inv_t, values_d, index_d, rest_d);
    else
        hipLaunchKernelGGL(lsr_top_kernel<ROW_BF16>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const __bf16*)scores_d,
                           n_rows, (int)n_classes, row_stride, k, inv_t, values_d, index_d, rest_d);
    lsr_prof_end(ctx);
    LSR_LAUNCH_CHECK(ctx, "lsr_top_kernel");
    return LSR_OK;
}
