// The k best classes of every row of log scores, and the log weight of the rest.
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

// The lowest of the row's first `want` entries by radix selection, eight bits at a time from a histogram of the entries
// that still match; what the group bound cannot narrow down comes here: more scores above it than the list takes, where
// `want` is near or above the number of groups with a score, or a few groups hold thousands of the best scores.
template <int DT, int W>
__device__ __forceinline__ uint64_t top_radix(const typename row_type<DT>::type* x, int n_classes, int want, int* hist,
                                              uint64_t* shared) {
    constexpr int THREADS = 64 * W;
    const int tid = threadIdx.x;
    int left = want;                                      // of thread 0
    uint64_t threshold = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
        team_sync<W>();
        for (int c = tid; c < n_classes; c += THREADS) {
            const uint32_t key = row_key((float)x[c]);
            const uint64_t e = row_entry(key, c);
            if (key && (shift == 56 || (e >> (shift + 8)) == (threshold >> (shift + 8)))) atomicAdd(&hist[(e >> shift) & 255], 1);
        }
        team_sync<W>();
        if (tid == 0) {
            int d = 255;
            for (; d > 0 && hist[d] < left; --d) left -= hist[d];
            *shared = threshold | (uint64_t)d << shift;
        }
        team_sync<W>();
        threshold = *shared;
    }
    return threshold;
}

// Long rows, a team of W wavefronts per row (lsr_rows.h).  ON: workgroups of 16 wavefronts with kept rows fill their compute
// unit alone; there are as many of them as compute units, and each requests its next row while it collects from this one
// (2048 x 131072, k = 64, with the rest: 152 us, 3.5 TB/s, 12 % less than with a workgroup per row), although 26 registers
// per lane spill in this form.  What it takes is missing for the sorting of longer lists, so that it is for k <= 64, whose
// lists have about 80 entries.
template <int DT, int W, int N, bool ON, bool REST>
__global__ __launch_bounds__(64 * W) void lsr_top_team_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                              int64_t n_rows, int n_classes, int64_t row_stride, int k,
                                                              float inv_t, float* __restrict__ values,
                                                              int32_t* __restrict__ index, float* __restrict__ rest) {
    constexpr int THREADS = 64 * W, RUN = team_row<DT, W, N>::RUN, ROOM = W == 1 ? 512 : 2048;
    __shared__ team_list<W, ROOM> list;
    __shared__ int hist[256];
    __shared__ uint64_t one;
    __shared__ uint64_t sorted[ROOM];                     // by place: the list itself is in the order in which it was filled
    __shared__ float part[W];
    int tid = threadIdx.x;
    const int kk = k + (REST ? 1 : 0);                    // the first entry of the rest as well
    const float unit = inv_t * 1.44269504f;
    team_row<DT, W, N> row;
    row.open(scores + (int64_t)blockIdx.x * row_stride, n_classes);
    int64_t r = blockIdx.x;
    do {
        asm volatile("" : "+v"(tid));                     // nothing that depends on it is kept from row to row in registers
        const auto* mine = scores + r * row_stride;
        row.arrive();
        if (!N) row.open(mine, n_classes);
        team_groups(row, list);
        typename team_row<DT, W, N>::sum_t below = 0;
        float bound = team_bound(kk, list);
        team_take<REST, ON>(row, bound, list, unit, below, mine + (r + gridDim.x < n_rows ? gridDim.x * row_stride : 0));
        team_row<DT, W, 0> again;                         // for the cases that need the row once more
        again.open(mine, n_classes);
        int n = list.n, bound_class = -1;                 // collected: above the bound, or equal up to this class
        bool equal = true;                                // every score that equals the bound is collected
        if (n > ROOM) {                                   // thousands of equal scores, as a rule: first what is above them
            equal = false;
            team_sync<W>();                               // every wavefront has read the count before it is cleared
            if (tid == 0) list.n = 0;
            team_sync<W>();
            again.template each<4>([&](int, const float(&v)[RUN], int c) {
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (v[j] > bound) {
                        const int at = atomicAdd(&list.n, 1);
                        if (at < ROOM) list.entry[at] = row_entry(row_key(v[j]), c + j);
                    }
            });
            team_sync<W>();
            n = list.n;
            // then, in the order of their classes, as many of them as are missing: a masked row is done after one step
#pragma unroll 1
            for (int step = 0; step < again.steps && n < kk; ++step) {
                float v[RUN];
                again.decode(again.read_any(step), v);
                int own = 0, sum = 0;
#pragma unroll
                for (int j = 0; j < RUN; ++j) own += v[j] == bound;
                int run = wave_running(own);
                team_sync<W>();
                if ((tid & 63) == 63) hist[tid >> 6] = run;
                team_sync<W>();
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    if (i < (tid >> 6)) run += hist[i];
                    sum += hist[i];
                }
                int place = n + run - own;
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (v[j] == bound) {
                        if (place < kk) list.entry[place] = row_entry(row_key(v[j]), again.first_class(step) + j);
                        ++place;
                    }
                n = min(n + sum, kk);
                if (n == kk) {
                    team_sync<W>();
                    bound_class = (int)~(uint32_t)list.entry[kk - 1];
                }
            }
        }
        if (n > ROOM) {
            const uint64_t least = top_radix<DT, W>(mine, n_classes, kk, hist, &one);
            bound = row_value((uint32_t)(least >> 32));
            bound_class = (int)~(uint32_t)least;
            if (tid == 0) list.n = 0;
            team_sync<W>();
            again.template each<1>([&](int, const float(&v)[RUN], int c) {
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (v[j] > bound || (v[j] == bound && c + j <= bound_class))
                        list.entry[atomicAdd(&list.n, 1)] = row_entry(row_key(v[j]), c + j);
            });
            team_sync<W>();
            n = list.n;
        }
        team_sync<W>();
        team_order<!ON>(list, n, sorted, ROOM);
        team_sync<W>();
        for (int i = tid; i < k; i += THREADS) {          // places without an entry: -infinity, -1
            const uint64_t e = i < n ? sorted[i] : 0;
            values[r * k + i] = e ? row_value((uint32_t)(e >> 32)) : -INFINITY;
            index[r * k + i] = e ? (int32_t)~(uint32_t)e : -1;
        }
        if (REST) {
            // relative to the highest score of the rest: relative to the row's best it could underflow to nothing
            const float from = n > k ? row_value((uint32_t)(sorted[k] >> 32)) : -INFINITY;
            const float best = n > 0 ? row_value((uint32_t)(sorted[0] >> 32)) : 0.0f;
            float sum = 0.0f;
            for (int i = k + tid; i < n; i += THREADS) {
                const float v = row_value((uint32_t)(sorted[i] >> 32));
                sum += v == from ? 1.0f : __builtin_amdgcn_exp2f((v - from) * unit);
            }
            // a NaN among the scores, absent like -infinity, spoils the sum of the pass that collected: once more, one by one
            const bool spoilt = equal && team_max<W>(below != below ? 1.0f : 0.0f, part) > 0;
            if (from > -INFINITY) {
                if (equal && !spoilt) {                   // relative to the bound, which an entry of the rest reaches
                    if (below > 0) sum += (float)below * __builtin_amdgcn_exp2f((bound - from) * unit);
                } else {
                    double far = 0;
                    again.template each<1>([&](int, const float(&v)[RUN], int c) {
                        float run = 0;
#pragma unroll
                        for (int j = 0; j < RUN; ++j)
                            if (v[j] < bound || (!equal && v[j] == bound && c + j > bound_class))
                                run += v[j] == from ? 1.0f : __builtin_amdgcn_exp2f((v[j] - from) * unit);
                        far += run;
                    });
                    sum += (float)far;
                }
            }
            sum = team_sum<W>(sum, part);
            if (tid == 0) rest[r] = from > -INFINITY ? (from == best ? 0.0f : (from - best) * inv_t) + logf(sum) : -INFINITY;
        }
        if (ON) team_sync<W>();                           // the next row's list takes this one's place
    } while (ON && (r += gridDim.x) < n_rows);
}

template <int DT, int W, int N>
static void lsr_top_team(lsr_ctx* ctx, const void* scores_d, int64_t n_rows, int n_classes, int64_t row_stride, int k,
                         float inv_t, float* values_d, int32_t* index_d, float* rest_d) {
    const auto* scores = (const typename row_type<DT>::type*)scores_d;
    // 64 registers of 32-bit scores and what the passes need do not fit together: 96 x 50001 with the rest takes 37 us kept
    // and spilling, 16.5 us read again
    constexpr int KEEP = DT == ROW_F32 && W == 16 ? 0 : N;
    const dim3 all((unsigned)n_rows), some((unsigned)ctx->n_cus), block(64 * W);
#define LAUNCH(ON, REST)                                                                                                    \
    hipLaunchKernelGGL((lsr_top_team_kernel<DT, W, KEEP, ON, REST>), ON ? some : all, block, 0, ctx->stream, scores, n_rows, \
                       n_classes, row_stride, k, inv_t, values_d, index_d, rest_d)
    if constexpr (W == 16 && KEEP > 0) {
        if (n_rows > ctx->n_cus && k <= 64) {
            if (rest_d) LAUNCH(true, true); else LAUNCH(true, false);
            return;
        }
    }
    if (rest_d) LAUNCH(false, true); else LAUNCH(false, false);
#undef LAUNCH
}

// Short rows (at most LSR_QUAD_CLASSES classes), a quad per row: the entries are sorted by a network over the quad's
// registers.  HEAD: the number of places that are put in order, 0 for all (k > E).  2.2 M x 58 with k = 8 and the rest takes
// 164 us, 4.1 TB/s read and written, and is bound by 686 vector instructions per 16 rows as much as by memory.  Writing the
// eight places one by one, each by one lane of the quad, took 182 us.
template <int DT, int E, int HEAD, bool REST>
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
        x[i] = row_clean(x[i]);
        e[i] = quad_entry(x[i], quad_class(i, q));
    }
    if constexpr (HEAD > 0)
        quad_sort_head<E, HEAD>(e);
    else
        quad_sort<E>(e, q);
    double least = 3.9;                                   // entry at place k - 1
    if (REST) {
#pragma unroll
        for (int i = 0; i < (HEAD ? HEAD : E); ++i) least = (HEAD ? i : q * E + i) == k - 1 ? e[i] : least;
    }
    auto write = [&](int place, double entry) {
        if (live && place < k) {
            const float v = quad_entry_value(entry);
            values[r * k + place] = v;
            index[r * k + place] = v > -INFINITY ? quad_entry_class(entry) : -1;
        }
    };
    if constexpr (HEAD > 0) {                             // all lanes hold the same places: four at a time, a lane each
#pragma unroll
        for (int i = 0; i < HEAD; i += 4) {
            const double one = e[i], two = e[i + 1], three = e[i + 2], four = e[i + 3];
            const double even = q & 2 ? three : one, odd = q & 2 ? four : two;
            write(i + q, q & 1 ? odd : even);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) write(q * E + i, e[i]);
    }
    if (!REST) return;
    if (!HEAD) least = quad_min(least);
    // the best entry is at place 0
    const double top = HEAD ? e[0] : quad_move<0x00>(e[0]);
    const float best = quad_entry_value(top);
    // relative to the highest score of the rest: relative to the row's best it could underflow to nothing
    const float last = quad_entry_value(least);
    const int last_class = quad_entry_class(least);
    float high = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool beyond = (x[i] < last) | ((x[i] == last) & (quad_class(i, q) > last_class));
        x[i] = beyond ? x[i] : -INFINITY;
        high = row_max(high, x[i]);
    }
    high = quad_max(high);
    float sum = 0.0f;
    const float unit = inv_t * 1.44269504f;
#pragma unroll
    for (int i = 0; i < E; ++i) sum += __builtin_amdgcn_exp2f(fminf((x[i] - high) * unit, 0.0f));   // 1 for infinity - infinity
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
    constexpr int HALF = E > 8 ? 8 : E;
    if (k <= HALF) {
        if (rest_d) LAUNCH(HALF, true); else LAUNCH(HALF, false);
    } else if (k <= E) {
        if (rest_d) LAUNCH(E, true); else LAUNCH(E, false);
    } else {
        if (rest_d) LAUNCH(0, true); else LAUNCH(0, false);
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
    if (temperature < 1e-30 || temperature > 1e30)        // its reciprocal is used in 32 bits
        return lsr_fail(ctx, LSR_ERR_LIMIT, "lsr_top_scores: temperature %g outside 1e-30..1e30", temperature);
    if (n_rows == 0) return LSR_OK;
    if (!values_d || !index_d) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_top_scores: null pointer");
    LSR_HIP_CHECK(ctx, hipSetDevice(ctx->device));
    const int64_t most = lsr_launch_rows(n_classes);
    if (n_rows > most) {
        for (int64_t r = 0; r < n_rows; r += most) {
            const int failed = lsr_top_scores(ctx, (const char*)scores_d + r * row_stride * row_dtype_bytes(dtype), dtype,
                                              n_rows - r < most ? n_rows - r : most, n_classes, row_stride, k, temperature,
                                              values_d + r * k, index_d + r * k, rest_d ? rest_d + r : nullptr);
            if (failed) return failed;
        }
        return LSR_OK;
    }
    const float inv_t = (float)(1.0 / temperature);
    lsr_prof_begin(ctx, LSR_K_TOP);
    if (n_classes <= LSR_QUAD_CLASSES) {
        LSR_DTYPE_SWITCH(dtype, LSR_QUAD_SWITCH(n_classes, lsr_top_quad<DT, E>(ctx->stream, scores_d, n_rows, (int)n_classes,
                                                                               row_stride, k, inv_t, values_d, index_d, rest_d)));
        lsr_prof_end(ctx);
        LSR_LAUNCH_CHECK(ctx, "lsr_top_quad_kernel");
        return LSR_OK;
    }
    LSR_TEAM_SWITCH(dtype, n_classes, lsr_top_team<DT, W, N>(ctx, scores_d, n_rows, (int)n_classes, row_stride, k, inv_t,
                                                             values_d, index_d, rest_d));
    lsr_prof_end(ctx);
    LSR_LAUNCH_CHECK(ctx, "lsr_top_team_kernel");
    return LSR_OK;
}
