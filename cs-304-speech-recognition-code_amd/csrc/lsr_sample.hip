// One class per row of log scores, drawn with temperature, top-k, top-p and min-p from a given uniform number.
//
// The three cuts each keep a head of the row's order (lsr_rows.h), so together they are one threshold entry.  Weights
// e^((x - best) / T) are computed in 64 bits and summed as whole numbers: which class a uniform number falls on does not
// depend on the order of the sums.
#include <math.h>

#include "lsr_rows.h"

struct sample_args {
    double temperature, top_p, min_p;
    int top_k;
    const float *temperature_d, *top_p_d, *min_p_d;
    const int32_t* top_k_d;
    double magic, unit;              // 2^(52 - shift), 2^-shift
};

template <int DT>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_sample_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                                     int64_t n_rows, int n_classes, int64_t row_stride,
                                                                     const float* __restrict__ uniform, sample_args a,
                                                                     int32_t* __restrict__ index, float* __restrict__ logprob) {
    __shared__ unsigned long long hist[256];
    __shared__ uint64_t wave_best[LSR_ROW_THREADS / 64];
    __shared__ uint64_t threshold, left;
    const int tid = threadIdx.x;
    for (int64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
        const typename row_type<DT>::type* x = scores + r * row_stride;
        const double t = a.temperature_d ? (double)a.temperature_d[r] : a.temperature;
        const double top_p = a.top_p_d ? (double)a.top_p_d[r] : a.top_p;
        const double min_p = a.min_p_d ? (double)a.min_p_d[r] : a.min_p;
        const int top_k = a.top_k_d ? a.top_k_d[r] : a.top_k;

        uint64_t best_e = 0;
        for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
            const uint32_t key = row_key((float)x[c]);
            const uint64_t e = row_entry(key, c);
            if (key && e > best_e) best_e = e;
        }
        best_e = row_wave_max(best_e);
        __syncthreads();                                  // the previous row is done with the shared variables
        if ((tid & 63) == 0) wave_best[tid >> 6] = best_e;
        __syncthreads();
        for (int w = 0; w < LSR_ROW_THREADS / 64; ++w) best_e = wave_best[w] > best_e ? wave_best[w] : best_e;
        if (best_e == 0 || !(t > 0)) {                    // nothing to draw from, or the best entry itself
            if (tid == 0) {
                index[r] = best_e ? (int32_t)~(uint32_t)best_e : -1;
                logprob[r] = best_e ? 0.0f : -INFINITY;
            }
            continue;
        }
        const float best = row_value((uint32_t)(best_e >> 32));
        const double inv_t = isinf(best) ? 1.0 : 1.0 / t;
        uint64_t least = 1;
        // mass of a class: 1 or its weight, 0 below the threshold
        auto mass = [&](int c, bool count, uint64_t* e) -> uint64_t {
            const float v = (float)x[c];
            const uint32_t key = row_key(v);
            *e = row_entry(key, c);
            if (!key || *e < least) return 0;
            return count ? 1 : row_fixed(v == best ? 1.0 : exp(((double)v - (double)best) * inv_t), a.magic);
        };
        auto total = [&]() -> uint64_t {
            uint64_t sum = 0, e;
            for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) sum += mass(c, false, &e);
            sum = row_wave_sum(sum);
            __syncthreads();
            if ((tid & 63) == 0) wave_best[tid >> 6] = sum;
            __syncthreads();
            return wave_best[0] + wave_best[1] + wave_best[2] + wave_best[3];
        };
        // the lowest entry of the shortest head whose mass is at least `target`
        auto select = [&](uint64_t target, bool count) {
            if (tid == 0) {
                threshold = 0;
                left = target;
            }
            for (int shift = 56; shift >= 0; shift -= 8) {
                hist[tid] = 0;
                __syncthreads();
                const uint64_t high = threshold;
                for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
                    uint64_t e;
                    const uint64_t m = mass(c, count, &e);
                    if (m && (shift == 56 || (e >> (shift + 8)) == (high >> (shift + 8))))
                        atomicAdd(&hist[(e >> shift) & 255], (unsigned long long)m);
                }
                __syncthreads();
                if (tid == 0) {
                    uint64_t need = left;
                    int d = 255;
                    for (; d > 0 && hist[d] < need; --d) need -= hist[d];
                    left = need;
                    threshold = high | (uint64_t)d << shift;
                }
                __syncthreads();
            }
            if (threshold > least) least = threshold;
            __syncthreads();
        };
        if (top_k > 0 && top_k < n_classes) select((uint64_t)top_k, true);
        if (top_p < 1.0) {
            double target = ceil((top_p > 0 ? top_p : 0.0) * (double)total());
            select(target < 1.0 ? 1 : (uint64_t)target, false);
        }
        if (min_p > 0) {
            const double low = (double)best + t * log(min_p < 1.0 ? min_p : 1.0);
            float f = (float)low;
            if ((double)f < low) f = nextafterf(f, INFINITY);
            const uint64_t e = (uint64_t)row_key(f) << 32;
            if (e > least) least = e;
        }
        const uint64_t sum = total();
        double at = (double)uniform[r] * (double)sum;
        if (!(at > 0)) at = 0;
        uint64_t goal = at >= (double)sum ? sum - 1 : (uint64_t)at;
        const bool count = goal == 0;                     // below half a unit: the first entry that is kept
        if (tid == 0) {
            threshold = 0;
            left = goal;
        }
        for (int shift = 16; shift >= 0; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            const int high = (int)threshold;
            for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
                uint64_t e;
                if ((c >> (shift + 8)) != (high >> (shift + 8))) continue;
                const uint64_t m = mass(c, count, &e);
                if (m) atomicAdd(&hist[(c >> shift) & 255], (unsigned long long)m);
            }
            __syncthreads();
            if (tid == 0) {
                uint64_t over = left;
                int d = 0;
                for (; d < 255 && hist[d] <= over; ++d) over -= hist[d];
                left = over;
                threshold = (uint64_t)(high | d << shift);
            }
            __syncthreads();
        }
        if (tid == 0) {
            const int c = (int)threshold;
            const float v = (float)x[c];
            index[r] = c;
            logprob[r] = (float)((v == best ? 0.0 : ((double)v - (double)best) * inv_t) - log((double)sum * a.unit));
        }
    }
}

// Short rows (at most LSR_QUAD_CLASSES classes), a quad per row.  ORDER: some row is cut by its order, so the entries are
// sorted; the sorted weights give the threshold, which the registers in class order are then compared with.  The sums are
// 64-bit floating ones in a fixed order.
template <int DT, int E, bool ORDER>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_sample_quad_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                                          int64_t n_rows, int n_classes, int64_t row_stride,
                                                                          const float* __restrict__ uniform, sample_args a,
                                                                          int32_t* __restrict__ index,
                                                                          float* __restrict__ logprob) {
    const int q = threadIdx.x & 3;
    const int64_t row = (int64_t)blockIdx.x * LSR_QUAD_ROWS + (threadIdx.x >> 2);
    const bool live = row < n_rows;
    const int64_t r = live ? row : n_rows - 1;            // every lane takes part in the exchanges
    float x[E];
    quad_load<DT, E>(scores + r * row_stride, n_classes, (n_rows - 1 - r) * row_stride + n_classes, q, x);
    const double t = a.temperature_d ? (double)a.temperature_d[r] : a.temperature;
    const double min_p = a.min_p_d ? (double)a.min_p_d[r] : a.min_p;
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] = x[i] > -INFINITY ? x[i] : -INFINITY;       // NaN is absent
        best = row_max(best, x[i]);
    }
    best = quad_max(best);
    const bool none = best == -INFINITY;
    if (__any(best == INFINITY)) {                        // only the infinite ones have weight
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (best == INFINITY) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        if (best == INFINITY) best = 0.0f;
    }
    const double unit = ROW_LOG2E / t;
    float last = -INFINITY;                               // the last entry that is kept
    int last_class = n_classes;
    if (ORDER) {
        const double top_p = a.top_p_d ? (double)a.top_p_d[r] : a.top_p;
        const int cut = a.top_k_d ? a.top_k_d[r] : a.top_k;
        const int top_k = cut > 0 ? cut : 4 * E;
        double e[E], w[E];
#pragma unroll
        for (int i = 0; i < E; ++i) e[i] = quad_entry(row_key(x[i]), quad_class(i, q));
        quad_sort<E>(e, q);
        double sum = 0, least = 3.9;
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = 0;
        if (__any(top_p < 1)) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const uint32_t key = quad_entry_key(e[i]);
                w[i] = key && q * E + i < top_k ? row_exp2(((double)row_value(key) - best) * unit) : 0.0;
                sum += w[i];
            }
        }
        const double target = top_p < 1 ? top_p * quad_sum(sum) : INFINITY;
        double run = quad_before(sum, q);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int place = q * E + i;
            // a place is kept while the weight ahead of it is short of the target
            if (place < top_k && (place == 0 || run < target) && quad_entry_key(e[i])) least = row_min(least, e[i]);
            run += w[i];
        }
        least = quad_min(least);
        if (!none) {
            last = row_value(quad_entry_key(least));
            last_class = quad_entry_class(least);
        }
    }
    if (min_p > 0) {
        const double low = (double)best + t * log(min_p < 1.0 ? min_p : 1.0);
        float f = (float)low;
        if ((double)f < low) f = nextafterf(f, INFINITY);
        if (f > last) {
            last = f;
            last_class = n_classes;
        }
    }
    double w[E], total = 0;
    const bool greedy = !(t > 0);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool kept = x[i] > last || (x[i] == last && quad_class(i, q) <= last_class);
        w[i] = kept && x[i] > -INFINITY ? row_exp2(((double)x[i] - best) * unit) : 0.0;
    }
    double lane[E / 4];
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        lane[g] = (w[4 * g] + w[4 * g + 1]) + (w[4 * g + 2] + w[4 * g + 3]);
        total += quad_sum(lane[g]);
    }
    const double goal = (double)uniform[r] * total;
    double base = 0;
    int at = 1 << 30, end = -1;
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        double run = base + quad_before(lane[g], q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            run += w[4 * g + j];
            if (w[4 * g + j] > 0) {
                end = quad_class(4 * g + j, q);
                if (run > goal) at = min(at, end);
            }
        }
        base += quad_sum(lane[g]);
    }
    at = quad_min(at);
    end = quad_max(end);
    if (at >= n_classes) at = end;                        // a uniform number of 1 or more
    if (__any(greedy)) {
        int first = 1 << 30;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (x[i] == best) first = min(first, quad_class(i, q));
        first = quad_min(first);
        if (greedy) at = first;
    }
    if (!live || q) return;
    index[r] = none ? -1 : at;
    float share = -INFINITY;
    if (!none && !greedy) {
        const float v = (float)scores[r * row_stride + at];
        share = (float)((isinf(v) ? 0.0 : ((double)v - best) / t) - log(total));
    }
    logprob[r] = !none && greedy ? 0.0f : share;
}

template <int DT, int E>
static void lsr_sample_quad(hipStream_t stream, const void* scores_d, int64_t n_rows, int n_classes, int64_t row_stride,
                            const float* uniform_d, const sample_args& a, bool order, int32_t* index_d, float* logprob_d) {
    const auto* scores = (const typename row_type<DT>::type*)scores_d;
    const dim3 grid((unsigned)((n_rows + LSR_QUAD_ROWS - 1) / LSR_QUAD_ROWS));
    if (order)
        hipLaunchKernelGGL((lsr_sample_quad_kernel<DT, E, true>), grid, dim3(LSR_ROW_THREADS), 0, stream, scores, n_rows,
                           n_classes, row_stride, uniform_d, a, index_d, logprob_d);
    else
        hipLaunchKernelGGL((lsr_sample_quad_kernel<DT, E, false>), grid, dim3(LSR_ROW_THREADS), 0, stream, scores, n_rows,
                           n_classes, row_stride, uniform_d, a, index_d, logprob_d);
}

extern "C" int lsr_sample_scores(lsr_ctx* ctx, const void* scores_d, int dtype, int64_t n_rows, int64_t n_classes,
                                 int64_t row_stride, const float* uniform_d, double temperature, int top_k, double top_p,
                                 double min_p, const float* temperature_d, const int32_t* top_k_d, const float* top_p_d,
                                 const float* min_p_d, int32_t* index_d, float* logprob_d) {
    if (!ctx) return LSR_ERR_ARG;
    const int rc = lsr_check_rows(ctx, "lsr_sample_scores", scores_d, dtype, n_rows, n_classes, row_stride);
    if (rc) return rc;
    if (isnan(temperature) || isnan(top_p) || isnan(min_p))
        return lsr_fail(ctx, LSR_ERR_ARG, "lsr_sample_scores: a setting is not a number");
    if (n_rows == 0) return LSR_OK;
    if (!uniform_d || !index_d || !logprob_d) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_sample_scores: null pointer");
    LSR_HIP_CHECK(ctx, hipSetDevice(ctx->device));
    // weights of up to n_classes entries have to fit 62 bits together
    int shift = 62;
    for (int64_t n = 1; n < n_classes; n *= 2) --shift;
    if (shift > 52) shift = 52;
    sample_args a = {temperature, top_p,  min_p, top_k, temperature_d, top_p_d, min_p_d, top_k_d, ldexp(1.0, 52 - shift),
                     ldexp(1.0, -shift)};
    const dim3 grid((unsigned)(n_rows < 65536 ? n_rows : 65536));
    const bool order = top_k_d || top_p_d || (top_k > 0 && top_k < n_classes) || top_p < 1;
    lsr_prof_begin(ctx, LSR_K_SAMPLE);
    if (n_classes <= LSR_QUAD_CLASSES) {
        LSR_DTYPE_SWITCH(dtype, LSR_QUAD_SWITCH(n_classes, lsr_sample_quad<DT, E>(ctx->stream, scores_d, n_rows, (int)n_classes,
                                                                                  row_stride, uniform_d, a, order, index_d,
                                                                                  logprob_d)));
        lsr_prof_end(ctx);
        LSR_LAUNCH_CHECK(ctx, "lsr_sample_quad_kernel");
        return LSR_OK;
    }
    if (dtype == LSR_F32)
        hipLaunchKernelGGL(lsr_sample_kernel<ROW_F32>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const float*)scores_d,
                           n_rows, (int)n_classes, row_stride, uniform_d, a, index_d, logprob_d);
    else if (dtype == LSR_F16)
        hipLaunchKernelGGL(lsr_sample_kernel<ROW_F16>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const _Float16*)scores_d,
                           n_rows, (int)n_classes, row_stride, uniform_d, a, index_d, logprob_d);
    else
        hipLaunchKernelGGL(lsr_sample_kernel<ROW_BF16>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const __bf16*)scores_d,
                           n_rows, (int)n_classes, row_stride, uniform_d, a, index_d, logprob_d);
    lsr_prof_end(ctx);
    LSR_LAUNCH_CHECK(ctx, "lsr_sample_kernel");
    return LSR_OK;
}
