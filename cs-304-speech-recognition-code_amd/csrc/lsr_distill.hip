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

// Long rows, a team of W wavefronts per row (lsr_rows.h).  Wavefront 0 handles the list while the row is on its way.  The
// listed classes are marked in a bit map, and where there is an outcome for the rest they are blanked in the registers, so
// that maximum, sum and gradient run over the others alone.  The gradient of the listed classes is written over afterwards.
// One read and one write of the row: 4096 x 131072 takes 517 us, 4.2 TB/s, a copy of that size 4.75.
template <int DT, int W, int N, bool REST, bool GRAD>
__global__ __launch_bounds__(64 * W) void lsr_distill_team_kernel(
    const typename row_type<DT>::type* __restrict__ scores, int n_classes, int64_t row_stride,
    const float* __restrict__ values, const int32_t* __restrict__ index, int k, const float* __restrict__ rest,
    double temperature, const float* __restrict__ weight, float* __restrict__ loss,
    typename row_type<DT>::type* __restrict__ grad) {
    using T = typename row_type<DT>::type;
    using Row = team_row<DT, W, N>;
    const row_exp2_t row_exp2;
    constexpr int THREADS = 64 * W, RUN = Row::RUN, MAP = W == 1 ? 1024 : W == 4 ? 16384 : 131072;   // bits of the map
    __shared__ uint32_t map[MAP / 32];
    __shared__ int cls[LSR_MAX_TOP];                      // listed classes, -1 for absent entries
    __shared__ float teacher[LSR_MAX_TOP];                // values, then weights relative to the best
    __shared__ float student[LSR_MAX_TOP];                // scores of the listed classes
    __shared__ bool first[LSR_MAX_TOP];                   // the class has not been listed before
    __shared__ float part_f[W], list_best, list_high;
    __shared__ double part_d[W], list_sum, list_cross, list_z, list_rest, list_lift;
    __shared__ int again;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const T* mine = scores + r * row_stride;
    Row row;
    // The list is requested before the row: loads are waited for in order, and the list's part below is to run while the
    // row is still on its way.
    constexpr int PER = THREADS < LSR_MAX_TOP ? LSR_MAX_TOP / THREADS : 1;
    int c[PER];
    float tv[PER];
    T sv[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = i * THREADS + tid;
        c[i] = j < k ? index[r * k + j] : -1;
        tv[i] = j < k ? values[r * k + j] : -INFINITY;
        if (!(c[i] >= 0 && c[i] < n_classes && tv[i] > -INFINITY)) c[i] = -1;
        sv[i] = mine[c[i] < 0 ? 0 : c[i]];
    }
    row.open(mine, n_classes);
    for (int i = tid; i < MAP / 32; i += THREADS) map[i] = 0;
    if (tid == 0) again = 0;
    team_sync<W>();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int j = i * THREADS + tid;
        if (j >= k) continue;
        cls[j] = c[i];
        teacher[j] = c[i] < 0 ? -INFINITY : tv[i];
        student[j] = c[i] < 0 ? -INFINITY : (float)sv[i];
        first[j] = c[i] >= 0;
        if (c[i] >= 0 && (atomicOr(&map[(c[i] & (MAP - 1)) >> 5], 1u << (c[i] & 31)) >> (c[i] & 31) & 1)) again = 1;
    }
    team_sync<W>();
    const double inv_t = 1.0 / temperature, unit = inv_t * ROW_LOG2E;
    if (tid < 64) {                                       // the list, in 64 bits, while the row is on its way
        if (again)                                        // a class, or in very long rows two that share a bit, came again
#pragma unroll 1
            for (int j = tid; j < k; j += 64)
#pragma unroll 1
                for (int i = 0; i < j; ++i)
                    if (cls[i] == cls[j]) first[j] = false;
        float best = -INFINITY, high = -INFINITY;
#pragma unroll 1
        for (int j = tid; j < k; j += 64) {
            best = row_max(best, teacher[j]);
            high = row_max(high, student[j]);
        }
        best = wave_max(best);
        high = wave_max(high);
        // a rest so heavy that its weight relative to the list's best leaves 64 bits: everything relative to the rest instead
        const double rest_log = REST ? (double)rest[r] : 0.0, lift = rest_log > 500 ? rest_log : 0.0;
        const double down = lift > 0 ? row_exp2(-lift * ROW_LOG2E) : 1.0;
        // sum of the teacher's weights e^y, of e^y (y - z), of the student's e^z; z relative to the list's highest score
        double sum = 0, cross = 0, z_l = 0;
#pragma unroll 1
        for (int j = tid; j < k; j += 64) {
            if (cls[j] < 0) continue;
            const double y = teacher[j] == best ? 0.0 : ((double)teacher[j] - best) * unit;
            const double z = ((double)student[j] - (high > -INFINITY ? high : 0.0f)) * unit, p = row_exp2(y);
            sum += p;
            if (p > 0) cross += p * (y - z);
            if (REST && first[j]) z_l += student[j] < INFINITY ? row_exp2(z) : NAN;
            teacher[j] = (float)(p * down);
        }
        sum = wave_sum(sum);
        cross = wave_sum(cross);
        if (REST) z_l = wave_sum(z_l);
        if (tid == 0) {
            list_best = best;
            list_high = high;
            list_sum = sum * down;
            list_cross = cross * (1.0 / ROW_LOG2E) * down;
            list_z = z_l;
            list_rest = rest_log - lift;
            list_lift = lift;
        }
    }
    if (W == 1) team_sync<W>();                           // larger teams meet in team_max before they read what is above
    row.arrive();
    // the runs of the row without the listed classes
    auto blank = [&](int step, uint4& u) {
        const int c = row.first_class(step);
        uint32_t b = map[(c & (MAP - 1)) >> 5] >> (c & 31) & ((1u << RUN) - 1);
        if (b == 0) return;
        if (n_classes > MAP) {                            // the bit may be another class's
            uint32_t sure = 0;
#pragma unroll 1
            for (int j = 0; j < k; ++j)
                if (cls[j] >= c && cls[j] < c + RUN) sure |= 1u << (cls[j] - c);
            b &= sure;
        }
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
        const uint32_t none = Row::nothing().x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DT == ROW_F32)
                w[i] = b >> i & 1 ? none : w[i];
            else {
                const uint32_t m = (b >> (2 * i) & 1 ? 0xffffu : 0u) | (b >> (2 * i) & 2 ? 0xffff0000u : 0u);
                w[i] = (w[i] & ~m) | (none & m);
            }
        }
        u = make_uint4(w[0], w[1], w[2], w[3]);
    };
    if (REST && N) {
#pragma unroll
        for (int i = 0; i < (N ? N : 1); ++i) blank(i, row.kept[i]);
    }
    auto each = [&](auto f) {
        row.next_pass();
        row.template each_run<4>([&](int step, uint4 u) {
            if (REST && !N) blank(step, u);
            float v[RUN];
            Row::decode(u, v);
            f(v, row.first_class(step));
        });
    };
    float high = -INFINITY;
    each([&](const float(&v)[RUN], int) {
#pragma unroll
        for (int j = 0; j < RUN; ++j) high = row_max(high, v[j]);
    });
    const float m_r = team_max<W>(high, part_f);
    const float unit_f = (float)unit, from = m_r > -INFINITY ? m_r : 0.0f;
    typename Row::sum_t part = 0;
    each([&](const float(&v)[RUN], int) {
        float sum = N ? part : 0.0f;
#pragma unroll
        for (int j = 0; j < RUN; ++j) sum += __builtin_amdgcn_exp2f((v[j] - from) * unit_f);
        part = N ? sum : part + sum;
    });
    const double z_r = team_sum<W>((double)part, part_d);

    // every thread for itself: no barrier between the sum and the gradient
    const double w = weight ? (double)weight[r] : 1.0, rest_log = REST ? list_rest : 0.0;
    const float high_l = list_high, m = REST ? row_max(m_r, high_l) : m_r;
    // NaN or +infinity among the scores: their exponentials, and with them the sum, are NaN
    const double shift = !REST ? 1.0 : z_r == 0 ? 0.0 : row_exp2(((double)m_r - m) * unit);
    const double shift_l = high_l > -INFINITY ? row_exp2(((double)high_l - m) * unit) : 1.0;
    const double z = (REST ? shift_l * list_z : 0.0) + (z_r == 0 ? 0.0 : shift * z_r);
    const double p_r = REST ? row_exp2(rest_log * ROW_LOG2E) : 0.0, sum = list_sum + p_r;
    const bool nan = z != z, used = w != 0 && list_best > -INFINITY && (m > -INFINITY || nan);
    const double scale = w * temperature;
    if (tid == 0) {
        double l = 0;
        if (used && !nan) {
            // the list's scores were taken relative to its own highest
            const double ln_z = row_log(z), gap = (high_l > -INFINITY ? (double)high_l - m : 0.0) * inv_t;
            l = (list_cross - list_sum * gap) / sum + ln_z - row_log(sum) - list_lift * (list_sum / sum);
            if (REST && p_r > 0) l += p_r / sum * (z_r > 0 ? rest_log - row_log(z_r) - ((double)m_r - m) * inv_t : INFINITY);
        }
        loss[r] = used ? (nan ? NAN : (float)(w * temperature * temperature * l)) : 0.0f;
    }
    if (!GRAD) return;
    T* g = grad + r * n_classes;
    // the row's constant for the others
    const float others = (float)(!REST ? scale / z : z_r > 0 ? scale * (shift / z - p_r / sum / z_r) : 0.0);
    each([&](const float(&v)[RUN], int c) {
        struct __attribute__((packed, aligned(sizeof(T)))) { T e[RUN]; } out;
#pragma unroll
        for (int j = 0; j < RUN; ++j) {
            const float d = others * __builtin_amdgcn_exp2f((v[j] - from) * unit_f);
            out.e[j] = (T)(used ? (nan ? NAN : d) : 0.0f);
        }
        if (c + RUN <= n_classes) {
            const uint4 u = __builtin_bit_cast(uint4, out);
            __builtin_nontemporal_store((row_words){u.x, u.y, u.z, u.w}, (row_words*)(g + c));
        } else {
#pragma unroll
            for (int j = 0; j < RUN; ++j)
                if (c + j < n_classes) g[c + j] = out.e[j];
        }
    });
    if (!used || nan) return;
    team_sync<W>();                                       // the listed classes are written after the pass over the row
#pragma unroll 1
    for (int j = tid; j < k; j += THREADS) {
        if (!first[j]) continue;
        float p = teacher[j];
        if (again) {
            p = 0;
#pragma unroll 1
            for (int i = 0; i < k; ++i) p += cls[i] == cls[j] ? teacher[i] : 0.0f;
        }
        g[cls[j]] = (T)(float)(scale * (row_exp2(((double)student[j] - m) * unit) / z - p / sum));
    }
}

// Short rows (at most LSR_QUAD_CLASSES classes), a quad per row.  The teacher's weights are added up per class in LDS, in
// the place of the quad's own row (no other wavefront touches it), and read back into registers beside the scores.
// With z = (x - m) / T, y = (t - best) / T, S the sum of the teacher's weights e^y and of e^rest:
//   KL = 1/S sum_j e^{y_j} (y_j - z_j) + ln Z - ln S + p_R (rest - ln q_R - ln Z),
// one logarithm instruction sequence for Z, S and the rest together, a lane each.
// HELD: entries of the list that a lane keeps in registers (k <= 4 HELD), 0 to read them again in each of the three loops.
// The sums into that table are atomics of one wavefront, so that their order is fixed.  2.2 M x 58 with k = 8, the rest and the
// gradient takes 308 us, 3.9 TB/s.
template <int DT, int E, int HELD, bool REST, bool GRAD>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_distill_quad_kernel(
    const typename row_type<DT>::type* __restrict__ scores, int64_t n_rows, int n_classes, int64_t row_stride,
    const float* __restrict__ values, const int32_t* __restrict__ index, int k, const float* __restrict__ rest,
    double temperature, const float* __restrict__ weight, float* __restrict__ loss,
    typename row_type<DT>::type* __restrict__ grad) {
    // 16 floats of padding: the runs that 16 lanes read at once, four rows', lie in different banks
    __shared__ float listed[LSR_QUAD_ROWS][4 * E + 16];
    const row_exp2_t row_exp2;
    const int q = threadIdx.x & 3, slot = threadIdx.x >> 2;
    const int64_t row = (int64_t)blockIdx.x * LSR_QUAD_ROWS + slot;
    const bool live = row < n_rows;
    const int64_t r = live ? row : n_rows - 1;            // every lane takes part in the exchanges
    const auto* mine = scores + r * row_stride;
    using T = typename row_type<DT>::type;
    // class (-1: absent), value and student's score of an entry
    int held_c[HELD ? HELD : 1];
    float held_v[HELD ? HELD : 1];
    T held_s[HELD ? HELD : 1];
    auto entry = [&](int j, int& c, float& v) {
        c = j < k ? index[r * k + j] : -1;
        v = j < k ? values[r * k + j] : -INFINITY;
        c = ((c >= 0) & (c < n_classes) & (v > -INFINITY)) ? c : -1;
    };
    if (HELD) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) entry(q + 4 * i, held_c[i], held_v[i]);
    }
    float x[E];
    quad_load<DT, E>(mine, n_classes, (n_rows - 1 - r) * row_stride + n_classes, q, x);
    if (HELD) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) held_s[i] = mine[held_c[i] < 0 ? 0 : held_c[i]];
    }
    auto each_entry = [&](auto f) {                       // f(class, value, student's score) for the entries that are there
        if (HELD) {
#pragma unroll
            for (int i = 0; i < HELD; ++i)
                if (held_c[i] >= 0) f(held_c[i], held_v[i], (float)held_s[i]);
        } else {
            for (int j = q; j < k; j += 4) {
                int c;
                float v;
                entry(j, c, v);
                if (c >= 0) f(c, v, (float)mine[c]);
            }
        }
    };
    float4* own = (float4*)&listed[slot][q * 4];
#pragma unroll
    for (int g = 0; g < E / 4; ++g) own[g * 4] = make_float4(0, 0, 0, 0);
    row_wave_fence();
    const double inv_t = 1.0 / temperature, unit = inv_t * ROW_LOG2E;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) m = row_max(m, x[i]);
    m = quad_max(m);
    float best = -INFINITY;
    each_entry([&](int, float v, float) { best = row_max(best, v); });
    best = quad_max(best);
    const double w = weight ? (double)weight[r] : 1.0;
    // sums over the list: the teacher's weights, those times (y - z), the student's weights of the listed classes
    double sum = 0, cross = 0, z_l = 0;
    each_entry([&](int c, float v, float s) {
        const double y = v == best ? 0.0 : ((double)v - best) * unit, z = ((double)s - m) * unit;
        const double p = row_exp2(y);
        sum += p;
        if (p > 0) cross += p * (y - z);
        // at least the smallest normal number: what is in the list is what is not 0; the first to find 0 counts the class
        const float old = atomicAdd(&listed[slot][c], fmaxf((float)p, 1.17549435e-38f));
        if (REST && old == 0) z_l += s < INFINITY ? row_exp2(z) : NAN;
    });
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
    // the others' maximum and sum of e^z relative to it (without an outcome for the rest: of all classes)
    float m_r = m;
    if (REST) {
        m_r = -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = p[i] > 0 ? -INFINITY : x[i];
            m_r = row_max(m_r, x[i]);
        }
        m_r = quad_max(m_r);
        z_l = quad_sum(z_l);
    }
    const float unit_f = (float)unit, from = m_r > -INFINITY ? m_r : 0.0f;
    float part = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] = __builtin_amdgcn_exp2f((x[i] - from) * unit_f);
        part += x[i];
    }
    const double z_r = quad_sum(part);
    const double shift = !REST ? 1.0 : z_r == 0 ? 0.0 : row_exp2(((double)m_r - m) * unit);
    const double z = z_l + (z_r == 0 ? 0.0 : shift * z_r);
    // NaN or +infinity among the scores: their exponentials, and with them the sum, are NaN
    const bool nan = z != z, used = (w != 0) & (best > -INFINITY) & ((m > -INFINITY) | nan);
    double p_r = 0, rest_log = 0, down = 1, lifted = 0;
    if (REST) {
        rest_log = (double)rest[r];
        if (__any(rest_log > 500)) {                      // the rest's weight relative to the list's best may leave 64 bits:
            const double lift = rest_log > 500 ? rest_log : 0.0;          // everything relative to the rest instead
            down = row_exp2(-lift * ROW_LOG2E);
            lifted = lift * (sum * down);
            rest_log -= lift;
        }
        p_r = row_exp2(rest_log * ROW_LOG2E);
        sum = sum * down + p_r;
    }
    const double ln = row_log(q == 0 ? z : q == 1 ? sum : z_r);
    const double ln_z = quad_move<0x00>(ln), ln_s = quad_move<0x55>(ln), ln_r = quad_move<0xAA>(ln);
    if (live && q == 0) {
        double l = cross * down / sum + ln_z - ln_s - lifted / sum;
        if (REST && p_r > 0) l += p_r / sum * (z_r > 0 ? rest_log - ln_r - ((double)m_r - m) * inv_t : INFINITY);
        loss[r] = used ? (nan ? NAN : (float)(w * temperature * temperature * l)) : 0.0f;
    }
    if (!GRAD) return;
    const double scale = w * temperature;
    const float c_l = (float)(scale / z), c_p = (float)(scale * down / sum);
    const float c_r = REST ? (z_r > 0 ? (float)(scale * (shift / z - p_r / sum / z_r)) : 0.0f) : c_l;
    if (REST) {
        // the student's weights of the listed classes take the place of the teacher's, which are in registers now
        row_wave_fence();
        each_entry([&](int c, float, float s) { listed[slot][c] = __builtin_amdgcn_exp2f((s - m) * unit_f); });
        row_wave_fence();
    }
    const bool plain = __all(used & !nan);
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        const float4 f = REST ? own[g * 4] : make_float4(0, 0, 0, 0);
        const float s[4] = {f.x, f.y, f.z, f.w};
        float d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            d[j] = __builtin_fmaf(c_r, x[4 * g + j], -c_p * p[4 * g + j]);
            if (REST) d[j] = __builtin_fmaf(c_l, s[j], d[j]);
        }
        if (!plain) {
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = used ? (nan ? NAN : d[j]) : 0.0f;
        }
        if (live) quad_store(grad + r * n_classes, n_classes, g, q, d);
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
    if (k <= 8) LAUNCH_HELD(2, REST, GRAD); else LAUNCH_HELD(0, REST, GRAD)
#define LAUNCH_HELD(HELD, REST, GRAD)                                                                                        \
    hipLaunchKernelGGL((lsr_distill_quad_kernel<DT, E, HELD, REST, GRAD>), grid, dim3(LSR_ROW_THREADS), 0, stream, scores, n_rows,   \
                       n_classes, row_stride, values_d, index_d, k, rest_d, temperature, weight_d, loss_d, grad)
    if (rest_d) {
        if (grad_d) { LAUNCH(true, true); } else { LAUNCH(true, false); }
    } else {
        if (grad_d) { LAUNCH(false, true); } else { LAUNCH(false, false); }
    }
#undef LAUNCH
#undef LAUNCH_HELD
}

template <int DT, int W, int N>
static void lsr_distill_team(hipStream_t stream, const void* scores_d, int64_t n_rows, int n_classes, int64_t row_stride,
                             const float* values_d, const int32_t* index_d, int k, const float* rest_d, double temperature,
                             const float* weight_d, float* loss_d, void* grad_d) {
    const auto* scores = (const typename row_type<DT>::type*)scores_d;
    auto* grad = (typename row_type<DT>::type*)grad_d;
#define LAUNCH(REST, GRAD)                                                                                                  \
    hipLaunchKernelGGL((lsr_distill_team_kernel<DT, W, N, REST, GRAD>), dim3((unsigned)n_rows), dim3(64 * W), 0, stream,    \
                       scores, n_classes, row_stride, values_d, index_d, k, rest_d, temperature, weight_d, loss_d, grad)
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
    if (temperature < 1e-30 || temperature > 1e30)        // its reciprocal is used in 32 bits
        return lsr_fail(ctx, LSR_ERR_LIMIT, "lsr_distill_scores: temperature %g outside 1e-30..1e30", temperature);
    if (n_rows == 0) return LSR_OK;
    if (!top_values_d || !top_index_d || !loss_d) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_distill_scores: null pointer");
    if ((uintptr_t)grad_d % row_dtype_bytes(dtype))
        return lsr_fail(ctx, LSR_ERR_ARG, "lsr_distill_scores: gradient is not aligned to its element size");
    LSR_HIP_CHECK(ctx, hipSetDevice(ctx->device));
    const int64_t most = lsr_launch_rows(n_classes);
    if (n_rows > most) {
        const int bytes = row_dtype_bytes(dtype);
        for (int64_t r = 0; r < n_rows; r += most) {
            const int failed = lsr_distill_scores(ctx, (const char*)scores_d + r * row_stride * bytes, dtype,
                                                  n_rows - r < most ? n_rows - r : most, n_classes, row_stride,
                                                  top_values_d + r * k, top_index_d + r * k, k, rest_d ? rest_d + r : nullptr,
                                                  temperature, row_weight_d ? row_weight_d + r : nullptr, loss_d + r,
                                                  grad_d ? (char*)grad_d + r * n_classes * bytes : nullptr);
            if (failed) return failed;
        }
        return LSR_OK;
    }
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
    LSR_TEAM_SWITCH(dtype, n_classes, lsr_distill_team<DT, W, N>(ctx->stream, scores_d, n_rows, (int)n_classes, row_stride,
                                                                 top_values_d, top_index_d, k, rest_d, temperature,
                                                                 row_weight_d, loss_d, grad_d));
    lsr_prof_end(ctx);
    LSR_LAUNCH_CHECK(ctx, "lsr_distill_team_kernel");
    return LSR_OK;
}
