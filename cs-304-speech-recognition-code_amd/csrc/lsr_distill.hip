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

// Short rows (at most LSR_QUAD_CLASSES classes), a quad per row.  The teacher's weights are added up per class in LDS, in
// the place of the quad's own row (no other wavefront touches it), and read back into registers beside the scores.
// With z = (x - m) / T, y = (t - best) / T, S the sum of the teacher's weights e^y and of e^rest:
//   KL = 1/S sum_j e^{y_j} (y_j - z_j) + ln Z - ln S + p_R (rest - ln q_R - ln Z),
// one logarithm instruction sequence for Z, S and the rest together, a lane each.
template <int DT, int E, bool REST, bool GRAD>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_distill_quad_kernel(
    const typename row_type<DT>::type* __restrict__ scores, int64_t n_rows, int n_classes, int64_t row_stride,
    const float* __restrict__ values, const int32_t* __restrict__ index, int k, const float* __restrict__ rest,
    double temperature, const float* __restrict__ weight, float* __restrict__ loss,
    typename row_type<DT>::type* __restrict__ grad) {
    // 16 floats of padding: the runs that 16 lanes read at once, four rows', lie in different banks
    __shared__ float listed[LSR_QUAD_ROWS][4 * E + 16];
    const int q = threadIdx.x & 3, slot = threadIdx.x >> 2;
    const int64_t row = (int64_t)blockIdx.x * LSR_QUAD_ROWS + slot;
    const bool live = row < n_rows;
    const int64_t r = live ? row : n_rows - 1;            // every lane takes part in the exchanges
    const auto* mine = scores + r * row_stride;
    float x[E];
    quad_load<DT, E>(mine, n_classes, (n_rows - 1 - r) * row_stride + n_classes, q, x);
    float4* own = (float4*)&listed[slot][q * 4];
#pragma unroll
    for (int g = 0; g < E / 4; ++g) own[g * 4] = make_float4(0, 0, 0, 0);
    row_wave_fence();
    const double inv_t = 1.0 / temperature, unit = inv_t * ROW_LOG2E;
    float m = -INFINITY;
    int nan = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        nan |= !(x[i] < INFINITY);
        m = row_max(m, x[i]);
    }
    m = quad_max(m);
    nan = quad_max(nan);
    float best = -INFINITY;
    for (int j = q; j < k; j += 4) {
        const int c = index[r * k + j];
        const float v = values[r * k + j];
        if (c >= 0 && c < n_classes && v > best) best = v;
    }
    best = quad_max(best);
    const double w = weight ? (double)weight[r] : 1.0;
    const bool used = w != 0 && best > -INFINITY && (m > -INFINITY || nan);
    double sum = 0, cross = 0;
    for (int j = q; j < k; j += 4) {
        const int c = index[r * k + j];
        const float v = values[r * k + j];
        if (c < 0 || c >= n_classes || !(v > -INFINITY)) continue;
        const double y = v == best ? 0.0 : ((double)v - best) * unit, z = ((double)(float)mine[c] - m) * unit;
        const double p = row_exp2(y);
        sum += p;
        if (p > 0) cross += p * (y - z);
        // at least the smallest normal number: what is in the list is what is not 0
        atomicAdd(&listed[slot][c], fmaxf((float)p, 1.17549435e-38f));
    }
    row_wave_fence();
    sum = quad_sum(sum);
    cross = quad_sum(cross) * (1.0 / ROW_LOG2E);
    float p[E];
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        const float4 f = own[g * 4];
        p[4 * g] = f.x;
        p[4 * g + 1] = f.y;
        p[4 * g + 2] = f.z;
        p[4 * g + 3] = f.w;
    }
    // sums of e^z relative to m for what is listed and relative to m_r for the others (relative to m for all without rest)
    float m_r = m;
    if (REST) {
        m_r = -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (!(p[i] > 0)) m_r = row_max(m_r, x[i]);
        m_r = quad_max(m_r);
    }
    const float unit_f = (float)unit, from = m_r > -INFINITY ? m_r : 0.0f;
    float z_l = 0, z_r = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool in = REST && p[i] > 0;
        x[i] = __builtin_amdgcn_exp2f((x[i] - (in ? m : from)) * unit_f);
        if (in)
            z_l += x[i];
        else
            z_r += x[i];
    }
    z_l = quad_sum(z_l);
    z_r = quad_sum(z_r);
    const double shift = REST && z_r > 0 ? row_exp2(((double)m_r - m) * unit) : 1.0;
    const double z = REST ? z_l + shift * z_r : z_r;
    double p_r = 0, rest_log = 0;
    if (REST) {
        rest_log = (double)rest[r];
        p_r = exp(rest_log);
        sum += p_r;
    }
    const double ln = log(q == 0 ? z : q == 1 ? sum : (double)z_r);
    const double ln_z = quad_move<0x00>(ln), ln_s = quad_move<0x55>(ln), ln_r = quad_move<0xAA>(ln);
    if (live && q == 0) {
        double l = cross / sum + ln_z - ln_s;
        if (REST && p_r > 0) l += p_r / sum * (z_r > 0 ? rest_log - ln_r - ((double)m_r - m) * inv_t : INFINITY);
        loss[r] = used ? (nan ? NAN : (float)(w * temperature * temperature * l)) : 0.0f;
    }
    if (!GRAD || !live) return;
    const double scale = w * temperature;
    const float c_l = (float)(scale / z), c_p = (float)(scale / sum);
    const float c_r = REST ? (z_r > 0 ? (float)(scale * (shift / z - p_r / sum / z_r)) : 0.0f) : c_l;
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        float d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 4 * g + j;
            d[j] = (REST && p[i] > 0 ? c_l : c_r) * x[i] - c_p * p[i];
            d[j] = used ? (nan ? NAN : d[j]) : 0.0f;
        }
        quad_store(grad + r * n_classes, n_classes, g, q, d);
    }
}

template <int DT, int E>
static void lsr_distill_quad(hipStream_t stream, const void* scores_d, int64_t n_rows, int n_classes, int64_t row_stride,
                             const float* values_d, const int32_t* index_d, int k, const float* rest_d, double temperature,
                             const float* weight_d, float* loss_d, void* grad_d) {
    const auto* scores = (const typename row_type<DT>::type*)scores_d;
    auto* grad = (typename row_type<DT>::type*)grad_d;
    const dim3 grid((unsigned)((n_rows + LSR_QUAD_ROWS - 1) / LSR_QUAD_ROWS));
#define LAUNCH(REST, GRAD)                                                                                                   \
    hipLaunchKernelGGL((lsr_distill_quad_kernel<DT, E, REST, GRAD>), grid, dim3(LSR_ROW_THREADS), 0, stream, scores, n_rows,   \
                       n_classes, row_stride, values_d, index_d, k, rest_d, temperature, weight_d, loss_d, grad)
    if (rest_d) {
        if (grad_d) LAUNCH(true, true); else LAUNCH(true, false);
    } else {
        if (grad_d) LAUNCH(false, true); else LAUNCH(false, false);
    }
#undef LAUNCH
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
    if (n_classes <= LSR_QUAD_CLASSES) {
        LSR_DTYPE_SWITCH(dtype, LSR_QUAD_SWITCH(n_classes, lsr_distill_quad<DT, E>(ctx->stream, scores_d, n_rows, (int)n_classes,
                                                                                   row_stride, top_values_d, top_index_d, k,
                                                                                   rest_d, temperature, row_weight_d, loss_d,
                                                                                   grad_d)));
        lsr_prof_end(ctx);
        LSR_LAUNCH_CHECK(ctx, "lsr_distill_quad_kernel");
        return LSR_OK;
    }
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
