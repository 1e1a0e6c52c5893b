// Loss of a student's scores against a teacher's top scores, and its gradient.
//
// Teacher: p over k listed classes and, if given, one bucket for all others.  Student: q = softmax(x / T).  With L the
// listed classes and R the others, the row's loss and gradient are
//   w T^2 [ sum_j p_j (ln p_j - ln q_j) + p_R (ln p_R - ln q_R) ],   w T [ q_i - P_i - (i in R) p_R q_i / q_R ],
// P_i the teacher's weight on class i (an index may be given twice).  Outside L the gradient is a row constant times
// e^((x_i - m_R) / T), m_R the highest score of R.  R has a maximum and a sum of its own, so that a student that is sure
// of L still has the logarithm of q_R (a difference 1 - sum q would be 0, an exponential relative to the row's maximum
// would underflow).
#include <math.h>

#include "lsr_rows.h"

template <int DT>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_distill_kernel(
    const typename row_type<DT>::type* __restrict__ scores, int64_t n_rows, int n_classes, int64_t row_stride,
    const float* __restrict__ values, const int32_t* __restrict__ index, int k, const float* __restrict__ rest,
    double temperature, const float* __restrict__ weight, float* __restrict__ loss,
    typename row_type<DT>::type* __restrict__ grad) {
    using T = typename row_type<DT>::type;
    __shared__ int cls[LSR_MAX_TOP];
    __shared__ float teacher[LSR_MAX_TOP];                // the teacher's values, then probabilities
    __shared__ float student[LSR_MAX_TOP];                // scores of the listed classes
    __shared__ bool first[LSR_MAX_TOP];                   // the class was not listed before
    __shared__ float part[LSR_ROW_THREADS / 64];
    __shared__ double row[8];
    const int tid = threadIdx.x;
    const double inv_t = 1.0 / temperature;
    for (int64_t r = blockIdx.x; r < n_rows; r += gridDim.x) {
        const T* x = scores + r * row_stride;
        T* g = grad ? grad + r * n_classes : nullptr;
        const double w = weight ? (double)weight[r] : 1.0;
        __syncthreads();
        if (tid < k) {
            const int c = index[r * k + tid];
            const float v = values[r * k + tid];
            const bool there = c >= 0 && c < n_classes && v > -INFINITY;
            cls[tid] = there ? c : -1;
            teacher[tid] = there ? v : -INFINITY;
            student[tid] = there ? (float)x[c] : -INFINITY;
        }
        __syncthreads();
        if (tid < k) {
            bool f = cls[tid] >= 0;
            for (int j = 0; j < tid; ++j) f &= cls[j] != cls[tid];
            first[tid] = f;
        }
        // highest score and sum of the classes that are not listed (all of them when there is no bucket for the others)
        auto listed = [&](int c) {
            bool f = false;
            for (int j = 0; j < k; ++j) f |= cls[j] == c;
            return f;
        };
        float high = -INFINITY;
        bool nan = false;
        for (int c = tid; c < n_classes; c += LSR_ROW_THREADS) {
            const float v = (float)x[c];
            nan |= !(v < INFINITY);                        // +infinity makes the softmax undefined as well
            if (v > high && !listed(c)) high = v;
        }
        for (int d = 32; d; d >>= 1) high = fmaxf(high, __shfl_xor(high, d));
        if ((tid & 63) == 0) part[tid >> 6] = high;
        nan = __syncthreads_or(nan);
        high = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        __syncthreads();
        float sum = 0.0f;
        if (high > -INFINITY)
            for (int c = tid; c < n_classes; c += LSR_ROW_THREADS)
                if (!listed(c)) sum += expf(((float)x[c] - high) * (float)inv_t);
        sum = row_wave_sum(sum);
        if ((tid & 63) == 0) part[tid >> 6] = sum;
        __syncthreads();
        if (tid == 0) {                                   // the few numbers of a row, in 64 bits
            const double z_r = (double)part[0] + part[1] + part[2] + part[3], m_r = (double)high * inv_t;
            double best = -INFINITY, m = z_r > 0 ? m_r : -INFINITY, p_sum = 0, p_r = 0;
            for (int j = 0; j < k; ++j) {
                best = fmax(best, (double)teacher[j]);
                m = fmax(m, (double)student[j] * inv_t);
            }
            const bool used = w != 0 && best > -INFINITY && (m > -INFINITY || nan);
            double z = z_r > 0 ? z_r * exp(m_r - m) : 0;
            for (int j = 0; j < k; ++j) {
                const double p = cls[j] < 0 ? 0 : teacher[j] == best ? 1 : exp((teacher[j] - best) * inv_t);
                p_sum += p;
                teacher[j] = (float)p;
                if (first[j]) z += exp(student[j] * inv_t - m);
            }
            if (rest) {
                p_r = exp((double)rest[r]);
                p_sum += p_r;
                p_r /= p_sum;
            }
            double l = 0;
            for (int j = 0; j < k; ++j) {
                const double p = teacher[j] / p_sum;
                teacher[j] = (float)p;
                if (p > 0) l += p * (log(p) - (student[j] * inv_t - m - log(z)));
            }
            if (p_r > 0) l += p_r * (log(p_r) - (z_r > 0 ? log(z_r) + m_r - m - log(z) : -INFINITY));
            row[0] = used;
            row[1] = w * temperature;
            row[2] = m;
            row[3] = 1 / z;
            row[4] = z_r > 0 ? w * temperature * (exp(m_r - m) / z - p_r / z_r) : 0;   // the row constant outside L
            loss[r] = used ? (nan ? NAN : (float)(w * temperature * temperature * l)) : 0.0f;
        }
        __syncthreads();
        if (!g) continue;
        const bool used = row[0] != 0;
        const float scale = (float)row[4];
        for (int c = tid; c < n_classes; c += LSR_ROW_THREADS)
            if (!used)
                g[c] = (T)0.0f;
            else if (nan)
                g[c] = (T)NAN;
            else if (!listed(c))
                g[c] = (T)(high > -INFINITY ? scale * expf(((float)x[c] - high) * (float)inv_t) : 0.0f);
        if (used && !nan && tid < k && first[tid]) {
            double p = 0;
            for (int j = 0; j < k; ++j)
                if (cls[j] == cls[tid]) p += teacher[j];
            g[cls[tid]] = (T)(float)(row[1] * (exp(student[tid] * inv_t - row[2]) * row[3] - p));
        }
    }
}

extern "C" int lsr_distill_scores(lsr_ctx* ctx, const void* scores_d, int dtype, int64_t n_rows, int64_t n_classes,
                                  int64_t row_stride, const float* top_values_d, const int32_t* top_index_d, int k,
                                  const float* rest_d, double temperature, const float* row_weight_d, float* loss_d,
                                  void* grad_d) {
    if (!ctx) return LSR_ERR_ARG;
    const int rc = lsr_check_rows(ctx, "lsr_distill_scores", scores_d, dtype, n_rows, n_classes, row_stride);
    if (rc) return rc;
    if (k < 1) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_distill_scores: k = %d < 1", k);
    if (k > LSR_MAX_TOP) return lsr_fail(ctx, LSR_ERR_LIMIT, "lsr_distill_scores: k = %d > %d", k, LSR_MAX_TOP);
    if (!(temperature > 0) || !isfinite(temperature))
        return lsr_fail(ctx, LSR_ERR_ARG, "lsr_distill_scores: temperature must be positive and finite");
    if (n_rows == 0) return LSR_OK;
    if (!top_values_d || !top_index_d || !loss_d) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_distill_scores: null pointer");
    if ((uintptr_t)grad_d % row_dtype_bytes(dtype))
        return lsr_fail(ctx, LSR_ERR_ARG, "lsr_distill_scores: gradient is not aligned to its element size");
    LSR_HIP_CHECK(ctx, hipSetDevice(ctx->device));
    const dim3 grid((unsigned)(n_rows < 65536 ? n_rows : 65536));
    lsr_prof_begin(ctx, LSR_K_DISTILL);
    if (dtype == LSR_F32)
        hipLaunchKernelGGL(lsr_distill_kernel<ROW_F32>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const float*)scores_d,
                           n_rows, (int)n_classes, row_stride, top_values_d, top_index_d, k, rest_d, temperature, row_weight_d,
                           loss_d, (float*)grad_d);
    else if (dtype == LSR_F16)
        hipLaunchKernelGGL(lsr_distill_kernel<ROW_F16>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const _Float16*)scores_d,
                           n_rows, (int)n_classes, row_stride, top_values_d, top_index_d, k, rest_d, temperature, row_weight_d,
                           loss_d, (_Float16*)grad_d);
    else
        hipLaunchKernelGGL(lsr_distill_kernel<ROW_BF16>, grid, dim3(LSR_ROW_THREADS), 0, ctx->stream, (const __bf16*)scores_d,
                           n_rows, (int)n_classes, row_stride, top_values_d, top_index_d, k, rest_d, temperature, row_weight_d,
                           loss_d, (__bf16*)grad_d);
    lsr_prof_end(ctx);
    LSR_LAUNCH_CHECK(ctx, "lsr_distill_kernel");
    return LSR_OK;
}
