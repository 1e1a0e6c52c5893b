// One class per row of log scores, drawn with temperature, top-k, top-p and min-p from a given uniform number.
//
// The three cuts each keep a head of the row's order (lsr_rows.h), so together they are one threshold entry.  Weights
// e^((x - best) / T) are computed in 64 bits and summed as whole numbers: which class a uniform number falls on does not
// depend on the order of the sums.
#include <math.h>
#include <type_traits>

#include "lsr_rows.h"

struct sample_args {
    double temperature, top_p, min_p;
    int top_k;
    const float *temperature_d, *top_p_d, *min_p_d;
    const int32_t* top_k_d;
    double magic, unit;              // 2^(52 - shift), 2^-shift
};

// the lowest score that min_p keeps: x >= best + t ln(min_p) in 64 bits, as the next 32-bit number
__device__ __forceinline__ float sample_floor(float best, double t, double min_p) {
    const double low = min_p < 1.0 ? (double)best + t * row_log(min_p) : (double)best;
    const float f = (float)low;
    return (double)f < low ? nextafterf(f, INFINITY) : f;
}
// The lowest score that weighs anything in 64 bits.  What is below (masked with the type's lowest value, say) changes no sum
// and is never drawn; leaving it out keeps thousands of equal scores out of the lists.
__device__ __forceinline__ float sample_least(float best, double unit) {
    return (float)fmax((double)best - 1074.0 / unit, -3.402823466e38);
}
// the mass that top_p asks for: the first whole number that is not below its share of the sum, 1 at least
__device__ __forceinline__ uint64_t sample_target(double top_p, uint64_t sum) {
    if (!(top_p < 1.0)) return ~0ull;
    const double share = ceil(top_p * (double)sum);
    return share < 1.0 ? 1 : (uint64_t)share;
}
// the class sought is the first at which the running weight exceeds this
__device__ __forceinline__ uint64_t sample_goal(float u, uint64_t sum) {
    const double at = (double)u * (double)sum;
    return !(at > 0) ? 0 : at >= (double)sum ? sum - 1 : (uint64_t)at;
}

// The last entry of the shortest head of a list whose mass is at least `left` (1 at least, and not more than the list's).
// Up to 256 entries: each is compared with all others.  More: eight bits at a time, from a histogram of the entries that
// still match; where the whole mass of a digit is needed, the lowest entry of that digit that has mass is the one.  `hist`
// has 257 places.
template <int W>
__device__ __forceinline__ uint64_t list_head(const uint64_t* entry, const uint64_t* mass, int n, uint64_t left, uint64_t* hist) {
    constexpr int THREADS = 64 * W;
    const int tid = threadIdx.x;
    uint64_t found = 0;
    if (n <= (THREADS < 256 ? THREADS : 256)) {
        team_sync<W>();
        if (tid < n) {
            const uint64_t e = entry[tid], m = mass[tid];
            uint64_t before = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) before += entry[j] > e ? mass[j] : 0;
            if (before < left && left <= before + m) hist[0] = e;
        }
        team_sync<W>();
        return hist[0];
    }
#pragma unroll 1
    for (int shift = 56; shift >= 0; shift -= 8) {
        team_sync<W>();
        for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
        team_sync<W>();
#pragma unroll 1
        for (int i = tid; i < n; i += THREADS) {
            const uint64_t e = entry[i];
            if (shift == 56 || (e >> (shift + 8)) == (found >> (shift + 8)))
                atomicAdd((unsigned long long*)&hist[(e >> shift) & 255], (unsigned long long)mass[i]);
        }
        team_sync<W>();
        if (tid < 64) {                                   // lane l has the digits 255 - 4 l ... 252 - 4 l
            uint64_t m[4], own = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) own += m[i] = hist[255 - 4 * tid - i];
            uint64_t run = wave_running(own) - own;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (run < left && left <= run + m[i]) {
                    hist[0] = left - run;
                    hist[1] = left == run + m[i];
                    hist[256] = found | (uint64_t)(255 - 4 * tid - i) << shift;
                }
                run += m[i];
            }
        }
        team_sync<W>();
        found = hist[256];
        left = hist[0];
        if (hist[1]) break;
    }
    team_sync<W>();
    if (tid == 0) hist[0] = ~0ull;
    team_sync<W>();
    for (int i = tid; i < n; i += THREADS)
        if (mass[i] && entry[i] >= found) atomicMin((unsigned long long*)&hist[0], (unsigned long long)entry[i]);
    team_sync<W>();
    return hist[0];
}

// A row in many passes over memory, by radix selection with weights: for rows that the fast form below does not take (an
// infinite score, a cut that falls among thousands of scores that are alike or, by top_p, too near to a score's edge for 32
// bits; a small top_k that is near or above the number of groups with a score).
template <int DT, int W>
__device__ __forceinline__ void sample_by_radix(const typename row_type<DT>::type* x, int n_classes, float best, double t,
                                                int top_k, double top_p, double min_p, float u, const sample_args& a,
                                                uint64_t* hist, uint64_t* shared, int32_t* index, float* logprob) {
    constexpr int THREADS = 64 * W;
    const row_exp2_t row_exp2;
    const int tid = threadIdx.x;
    const double unit = isinf(best) ? 1.0 : ROW_LOG2E / t;
    uint64_t least = (uint64_t)row_key(sample_least(best, unit)) << 32;
    // mass of a class: 1 or its weight, 0 below the threshold
    auto mass = [&](int c, bool count, uint64_t* e) -> uint64_t {
        const float v = (float)x[c];
        const uint32_t key = row_key(v);
        *e = row_entry(key, c);
        if (!key || *e < least) return 0;
        return count ? 1 : row_fixed(v == best ? 1.0 : row_exp2(((double)v - (double)best) * unit), a.magic);
    };
    auto total = [&]() -> uint64_t {
        uint64_t sum = 0, e;
        for (int c = tid; c < n_classes; c += THREADS) sum += mass(c, false, &e);
        return team_sum<W>(sum, hist);
    };
    // the lowest entry of the shortest head whose mass is at least `left` (of thread 0)
    auto select = [&](uint64_t left, bool count) {
        uint64_t threshold = 0;
        for (int shift = 56; shift >= 0; shift -= 8) {
            team_sync<W>();
            for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
            team_sync<W>();
            for (int c = tid; c < n_classes; c += THREADS) {
                uint64_t e;
                const uint64_t m = mass(c, count, &e);
                if (m && (shift == 56 || (e >> (shift + 8)) == (threshold >> (shift + 8))))
                    atomicAdd((unsigned long long*)&hist[(e >> shift) & 255], (unsigned long long)m);
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
        if (threshold > least) least = threshold;
    };
    if (top_k > 0 && top_k < n_classes) select((uint64_t)top_k, true);
    if (top_p < 1.0) {
        const double target = ceil((top_p > 0 ? top_p : 0.0) * (double)total());
        select(target < 1.0 ? 1 : (uint64_t)target, false);
    }
    if (min_p > 0) {
        const uint64_t e = (uint64_t)row_key(sample_floor(best, t, min_p)) << 32;
        if (e > least) least = e;
    }
    const uint64_t sum = total();
    uint64_t left = sample_goal(u, sum);
    const bool count = left == 0;                         // below one unit: the first entry that is kept
    int at = 0;
    for (int shift = 16; shift >= 0; shift -= 8) {
        team_sync<W>();
        for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
        team_sync<W>();
        for (int c = tid; c < n_classes; c += THREADS) {
            uint64_t e;
            if ((c >> (shift + 8)) != (at >> (shift + 8))) continue;
            const uint64_t m = mass(c, count, &e);
            if (m) atomicAdd((unsigned long long*)&hist[(c >> shift) & 255], (unsigned long long)m);
        }
        team_sync<W>();
        if (tid == 0) {
            int d = 0;
            for (; d < 255 && hist[d] <= left; ++d) left -= hist[d];
            *shared = (uint64_t)(at | d << shift);
        }
        team_sync<W>();
        at = (int)*shared;
    }
    if (tid == 0) {
        const float v = (float)x[at];
        *index = at;
        *logprob = (float)((v == best ? 0.0 : ((double)v - (double)best) * unit * (1 / ROW_LOG2E)) - row_log((double)sum * a.unit));
    }
}

// Long rows, a team of W wavefronts per row (lsr_rows.h).
//
// Among the first entries of a row: a top_k of at most LSR_MAX_TOP, a min_p that few entries reach, a top_p that a short
// head seems to hold.  They are collected and put in order as lsr_top_scores does it, weighed, cut, and the uniform number is
// looked up in the order of their classes.  1 x 32768 with top_k 50 takes 9.9 us, 256 x 131072 26 us (reading them alone 18):
// a chain of dependent passes and barriers in one workgroup.  A radix selection in the list instead of comparing its
// entries took 22 us against 15 for one row.
//
// Otherwise every class is weighed, from memory: rows are not kept in registers, which 64-bit weights need.  A cut by order is
// found from a histogram over the distance to the best score, and the entries of the bin in which it falls.  The weights of
// what is kept are summed per step of the row, and the step, the run and the class that the uniform number falls on are
// looked up.  Bound by the 64-bit exponentials of one compute unit per row: 96 x 50001 takes 25 us, with a top_p 47.
template <int DT, int W>
__global__ __launch_bounds__(64 * W) void lsr_sample_team_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                                 int n_classes, int64_t row_stride,
                                                                 const float* __restrict__ uniform, sample_args a,
                                                                 int32_t* __restrict__ index, float* __restrict__ logprob) {
    using Row = team_row<DT, W, 0>;
    constexpr int THREADS = 64 * W, RUN = Row::RUN, ROOM = W == 1 ? 512 : W == 4 ? 2048 : 4096;
    constexpr int BINS = W == 1 ? 512 : W == 4 ? 2048 : 8192, OWN = BINS / THREADS;
    constexpr int STEPS = (W == 1 ? 1024 : W == 4 ? 16384 : LSR_MAX_CLASSES) / Row::STEP;
    __shared__ team_list<W, ROOM> list;
    static_assert(ROOM >= LSR_MAX_TOP, "weights of the few");
    __shared__ uint64_t mass[STEPS > LSR_MAX_TOP ? STEPS : LSR_MAX_TOP];     // of a step, of one of the few
    static_assert(2 * ROOM >= BINS, "the histogram and the weights of the list share their place, one after the other");
    __shared__ uint64_t list_mass[ROOM];
    int* const bin_n = (int*)list_mass;
    __shared__ uint64_t sorted[257], part[W], above, kept_sum;
    __shared__ float part_f[W];
    __shared__ int part_n[W], cut_bin, n_kept;
    constexpr int NUCLEUS = 128;                          // entries that a nucleus is first looked for in
    const row_exp2_t row_exp2;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const auto* mine = scores + r * row_stride;
    Row row;
    row.open(mine, n_classes);
    const double t = a.temperature_d ? (double)a.temperature_d[r] : a.temperature;
    const double top_p = a.top_p_d ? (double)a.top_p_d[r] : a.top_p;
    const double min_p = a.min_p_d ? (double)a.min_p_d[r] : a.min_p;
    const int top_k = a.top_k_d ? a.top_k_d[r] : a.top_k;
    const float u = uniform[r];
    const double unit = ROW_LOG2E / t;

    const float best = team_groups(row, list);
    const float least = sample_least(best, unit);
    if (best == -INFINITY || !(t > 0)) {                  // nothing to draw from, or the best entry itself
        int at = 1 << 30;
        if (best > -INFINITY)
            row.template each<4>([&](int, const float(&v)[RUN], int c) {
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (v[j] == best) at = min(at, c + j);
            });
        at = (int)~(uint32_t)team_max<W>((uint64_t)(uint32_t)~at, part);
        if (tid == 0) {
            index[r] = best == -INFINITY ? -1 : at;
            logprob[r] = best == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    // false: not for here
    auto fast = [&]() -> bool {
        float last = least;                                   // kept: above this score, or equal up to this class
        int last_class = n_classes;
        auto keeps = [&](float v, int c) { return (v > last) | ((v == last) & (c <= last_class)); };
        auto weigh = [&](float v) { return row_fixed(row_exp2(((double)v - best) * unit), a.magic); };
        const float per_bin = (float)fmin(BINS / 24.0 / t, 1e30);
        auto bin_of = [&](float v) { return (int)fminf((best - v) * per_bin, (float)(BINS - 1)); };

        auto cut_at = [&](uint64_t e) {
            last = row_value((uint32_t)(e >> 32));
            last_class = (int)~(uint32_t)e;
        };
        const uint64_t zero = (uint64_t)__double_as_longlong(a.magic);
        bool summed = false;                                  // the weights of the steps are known already
        // adds the weights of the list's entries that are kept to those of their steps
        auto tally = [&](int n) {
            for (int i = tid; i < n; i += THREADS) {
                const uint64_t e = list.entry[i];
                const int c = (int)~(uint32_t)e;
                if (keeps(row_value((uint32_t)(e >> 32)), c))
                    atomicAdd((unsigned long long*)&mass[c / Row::STEP], (unsigned long long)list_mass[i]);
            }
            summed = true;
        };

        // Rows that are answered from a list of their first entries.  few: a small top_k.  level: min_p without top_k, when not
        // many entries reach it.  nucleus: top_p alone, where it looks as if a short head will do: where the best scores of the
        // groups hold that share of the row's weight.
        const bool cut = top_k > 0 && top_k < n_classes, few = cut && top_k <= LSR_MAX_TOP, level = !cut && min_p > 0;
        const float floor = min_p > 0 ? sample_floor(best, t, min_p) : -INFINITY;
        if (!few && top_p < 1 && unit > 3e38) return false;   // a temperature whose reciprocal 32 bits do not hold
        // weights in 32 bits, always a number in [0, 1]: 0 for NaN
        const float unit_f = (float)unit;
        auto weigh_f = [&](float v) { return __builtin_amdgcn_exp2f(row_max((v - best) * unit_f, -INFINITY)); };
        bool nucleus = !cut && !level && top_p < 1;
        // the row's weight in 32 bits: at most 2^14 additions per thread, 22 over the team, and exponentials off by 2^-17, so
        // that it is good to 2^-9
        float guess = 0;
        if (!few && top_p < 1) {
            float head = 0;
            row.template each<4>([&](int, const float(&v)[RUN], int) {
#pragma unroll
                for (int j = 0; j < RUN; ++j) guess += weigh_f(v[j]);
            });
            guess = team_sum<W>(guess, part_f);
            for (int i = tid; i < ROW_GROUPS; i += THREADS)
                if (list.group[i]) head += weigh_f(row_value(list.group[i]));
            nucleus = nucleus && team_sum<W>(head, part_f) >= (float)top_p * guess;
        }
        if (few || level || nucleus) {
            double none = 0;
            float bound = few || nucleus ? team_bound(few ? top_k : NUCLEUS < n_classes ? NUCLEUS : n_classes, list) : floor;
            if (level && tid == 0) list.n = 0;
            if (level) team_sync<W>();
            team_take<false, false>(row, row_max(bound, least), list, 0.0f, none, mine);
            const int n = list.n;
            if (n <= ROOM) {
                // weight of the row, where the list does not hold what top_p is a share of; where the level's entries weigh
                // less than that share by more than the guess can be off, top_p takes nothing away
                uint64_t all = 0;
                bool open = top_p >= 1;
                if (level && !open) {
                    float listed = 0;
                    for (int i = tid; i < n; i += THREADS)
                        listed += weigh_f(row_value((uint32_t)(list.entry[i] >> 32)));
                    open = team_sum<W>(listed, part_f) < (1 - 1.0f / 512) * (float)top_p * guess;
                }
                if (!few && !open) {
                    row.template each<2>([&](int, const float(&v)[RUN], int) {
#pragma unroll
                        for (int j = 0; j < RUN; ++j)
                            all += (uint64_t)__double_as_longlong(row_exp2(((double)v[j] - best) * unit) + a.magic);
                        all -= RUN * (uint64_t)__double_as_longlong(a.magic);
                    });
                    all = team_sum<W>(all, part);
                }
                if (level && n > LSR_MAX_TOP) {               // too many to put in order
                    for (int i = tid; i < n; i += THREADS) list_mass[i] = weigh(row_value((uint32_t)(list.entry[i] >> 32)));
                    for (int i = tid; i < row.steps; i += THREADS) mass[i] = 0;
                    team_sync<W>();
                    uint64_t sum = 0;
                    for (int i = tid; i < n; i += THREADS) sum += list_mass[i];
                    sum = team_sum<W>(sum, part);
                    last = row_max(floor, least);
                    const uint64_t target = open ? ~0ull : sample_target(top_p, all);
                    if (target <= sum) cut_at(list_head<W>(list.entry, list_mass, n, target, sorted));
                    tally(n);
                } else {
                    team_order<true>(list, n, sorted, LSR_MAX_TOP);
                    team_sync<W>();
                    const int most = few ? top_k : LSR_MAX_TOP, m = n < most ? n : most;     // the list is the head of the row, all of it
                    if (tid < 64) {                               // lane l has the places 4 l ... 4 l + 3
                        constexpr int FOUR = LSR_MAX_TOP / 64;
                        uint64_t w[FOUR], own = 0;
                        float v[FOUR];
#pragma unroll
                        for (int i = 0; i < FOUR; ++i) {
                            const int place = tid * FOUR + i;
                            v[i] = place < m ? row_value((uint32_t)(sorted[place] >> 32)) : -INFINITY;
                            w[i] = row_fixed(row_exp2(((double)v[i] - best) * unit), a.magic);
                            own += w[i];
                        }
                        uint64_t run = wave_running(own);
                        const uint64_t listed = wave_last(run), target = open ? ~0ull : sample_target(top_p, few ? listed : all);
                        run -= own;
                        uint64_t sum = 0;
                        int kept = 0;
#pragma unroll
                        for (int i = 0; i < FOUR; ++i) {          // kept: the weight ahead of it is short of the target
                            const int place = tid * FOUR + i;
                            const bool in = (place < m) & ((place == 0) | (run < target)) & (v[i] >= floor);
                            run += w[i];
                            sum += in ? w[i] : 0;
                            kept += in;
                            mass[place] = w[i];
                        }
                        sum = wave_sum(sum);
                        kept = wave_sum(kept);
                        if (tid == 0) {
                            kept_sum = sum;
                            n_kept = few || level || listed >= target ? kept : 0;        // 0: the list is too short for top_p
                        }
                    }
                    team_sync<W>();
                    const int kept = n_kept;
                    const uint64_t goal = sample_goal(u, kept_sum);
                    auto answer = [&](uint64_t e) {
                        index[r] = (int32_t)~(uint32_t)e;
                        logprob[r] = (float)(((double)row_value((uint32_t)(e >> 32)) - best) / t - row_log((double)kept_sum * a.unit));
                    };
                    if (kept > 64) {                              // in the order of their classes, the weights added up
                        if (tid < 64) {
                            constexpr int FOUR = LSR_MAX_TOP / 64;
                            static_assert(LSR_MAX_TOP <= 256 && LSR_MAX_CLASSES <= 1 << 24, "class and place in 32 bits");
                            uint32_t c[FOUR];
#pragma unroll
                            for (int i = 0; i < FOUR; ++i) {
                                const int place = i * 64 + tid;
                                c[i] = place < kept ? (uint32_t)sorted[place] << 8 | place : 0;  // classes are complemented
                            }
                            wave_sort(c);
                            uint64_t own = 0, w[FOUR];
#pragma unroll
                            for (int i = 0; i < FOUR; ++i) {
                                w[i] = tid * FOUR + i < kept ? mass[c[i] & 255] : 0;
                                own += w[i];
                            }
                            uint64_t run = wave_running(own) - own;
#pragma unroll
                            for (int i = 0; i < FOUR; ++i) {
                                if (tid * FOUR + i < kept && (goal == 0 ? tid + i == 0 : run <= goal && goal < run + w[i])) answer(sorted[c[i] & 255]);
                                run += w[i];
                            }
                        }
                        return true;
                    }
#pragma unroll 1
                    for (int i = tid; i < kept; i += THREADS) {
                        // weight of the kept entries of lower classes
                        const uint32_t own = (uint32_t)sorted[i];
                        uint64_t before = 0;
                        int ahead = 0;
#pragma unroll 8
                        for (int j = 0; j < kept; ++j) {
                            const bool lower = (uint32_t)sorted[j] > own;
                            before += lower ? mass[j] : 0;
                            ahead += lower;
                        }
                        if (goal == 0 ? ahead == 0 : before <= goal && goal < before + mass[i]) answer(sorted[i]);
                    }
                    if (kept > 0) return true;
                }
            }
            if (few) return false;                         // thousands of entries are alike
        }

        if (cut) {                                            // the first top_k entries, by a histogram of their numbers
            team_sync<W>();
            for (int i = tid; i < BINS; i += THREADS) bin_n[i] = 0;
            if (tid == 0) list.n = 0;
            team_sync<W>();
            row.template each<4>([&](int, const float(&v)[RUN], int) {
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (v[j] >= least) atomicAdd(&bin_n[bin_of(v[j])], 1);
            });
            team_sync<W>();
            int own = 0, sum = 0;
#pragma unroll
            for (int i = 0; i < OWN; ++i) own += bin_n[tid * OWN + i];
            int run = wave_running(own);
            if ((tid & 63) == 63) part_n[tid >> 6] = run;
            team_sync<W>();
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (i < (tid >> 6)) run += part_n[i];
                sum += part_n[i];
            }
            if (top_k <= sum) {                               // or all are kept
                run -= own;
                if (run < top_k && top_k <= run + own) {
#pragma unroll
                    for (int i = 0; i < OWN; ++i) {
                        const int m = bin_n[tid * OWN + i];
                        if (run < top_k && top_k <= run + m) {
                            cut_bin = tid * OWN + i;
                            n_kept = run;
                        }
                        run += m;
                    }
                }
                team_sync<W>();
                const int b = cut_bin, ahead = n_kept;
                row.template each<4>([&](int, const float(&v)[RUN], int c) {
#pragma unroll
                    for (int j = 0; j < RUN; ++j)
                        if (v[j] >= least && bin_of(v[j]) == b) {
                            const int at = atomicAdd(&list.n, 1);
                            if (at < ROOM) list.entry[at] = row_entry(row_key(v[j]), c + j);
                        }
                });
                team_sync<W>();
                const int n = list.n;
                if (n > ROOM) return false;
                for (int i = tid; i < n; i += THREADS) list_mass[i] = 1;
                team_sync<W>();
                cut_at(list_head<W>(list.entry, list_mass, n, (uint64_t)(top_k - ahead), sorted));
            }
        }
        if (top_p < 1 && !summed) {
            // The entries that hold top_p of what is left.  A histogram of weights in 32 bits (whole numbers: adding floats in
            // shared memory takes eight times as long) says near which bin that cut lies.  One pass in 64 bits then sums
            // everything and, step by step, what is above the neighbours of that bin, and collects what is in the three of
            // them: if the cut is there, everything is known that the draw needs.  It can be elsewhere where it lies as near to
            // an edge as 32 bits are off and empty bins follow.
            team_sync<W>();
            for (int i = tid; i < BINS; i += THREADS) bin_n[i] = 0;
            for (int i = tid; i < row.steps; i += THREADS) mass[i] = 0;
            if (tid == 0) {
                list.n = 0;
                cut_bin = BINS - 1;
            }
            team_sync<W>();
            const float scale = 1073741824.0f / guess;
            row.template each<4>([&](int, const float(&v)[RUN], int c) {
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    const float s = !cut || keeps(v[j], c + j) ? v[j] : -INFINITY;
                    const int m = (int)(weigh_f(s) * scale + 0.5f);
                    if (m) atomicAdd(&bin_n[bin_of(s)], m);
                }
            });
            team_sync<W>();
            uint32_t own = 0, total = 0;
#pragma unroll
            for (int i = 0; i < OWN; ++i) own += (uint32_t)bin_n[tid * OWN + i];
            uint32_t run = (uint32_t)wave_running((int)own);
            if ((tid & 63) == 63) part_n[tid >> 6] = (int)run;
            team_sync<W>();
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (i < (tid >> 6)) run += (uint32_t)part_n[i];
                total += (uint32_t)part_n[i];
            }
            run -= own;
            const uint32_t near = (uint32_t)(top_p * total);
            if (run < near && near <= run + own) {
#pragma unroll
                for (int i = 0; i < OWN; ++i) {
                    if (run < near) cut_bin = tid * OWN + i;
                    run += (uint32_t)bin_n[tid * OWN + i];
                }
            }
            team_sync<W>();
            const float high = best - (cut_bin - 1) / per_bin, low = best - (cut_bin + 2) / per_bin;
            uint64_t all = 0;
            auto weigh_all = [&](auto some) {
                row.template each<2>([&](int step, const float(&v)[RUN], int c) {
                    uint64_t higher = 0;
                    bool any = false;
#pragma unroll
                    for (int j = 0; j < RUN; ++j) {
                        const float s = !some.value || keeps(v[j], c + j) ? v[j] : -INFINITY;
                        const uint64_t m = (uint64_t)__double_as_longlong(row_exp2(((double)s - best) * unit) + a.magic);
                        all += m;
                        higher += s > high ? m : zero;
                        any |= (s >= low) & !(s > high);
                    }
                    if (any) {
#pragma unroll
                        for (int j = 0; j < RUN; ++j) {
                            const float s = !some.value || keeps(v[j], c + j) ? v[j] : -INFINITY;
                            if ((s >= low) & !(s > high) & (s > -INFINITY)) {
                                const int at = atomicAdd(&list.n, 1);
                                if (at < ROOM) {
                                    list.entry[at] = row_entry(row_key(s), c + j);
                                    list_mass[at] = weigh(s);
                                }
                            }
                        }
                    }
                    all -= RUN * zero;
                    higher = wave_sum(higher - RUN * zero);
                    if ((tid & 63) == 0 && higher) atomicAdd((unsigned long long*)&mass[step], (unsigned long long)higher);
                });
            };
            if (cut)
                weigh_all(std::true_type{});
            else
                weigh_all(std::false_type{});
            all = team_sum<W>(all, part);
            team_sync<W>();
            const int n = list.n;
            if (n > ROOM) return false;
            uint64_t ahead = 0, listed = 0;
            for (int i = 0; i < row.steps; ++i) ahead += mass[i];
            for (int i = tid; i < n; i += THREADS) listed += list_mass[i];
            listed = team_sum<W>(listed, part);
            const uint64_t target = sample_target(top_p, all);
            if (ahead >= target || target > ahead + listed) return false;
            cut_at(list_head<W>(list.entry, list_mass, n, target - ahead, sorted));
            if (floor <= last) tally(n);
        }
        if (floor > last) {
            last = floor;
            last_class = n_classes;
        }
        // weight of every step, and the step in which the goal lies
        if (!summed) {
            team_sync<W>();
            for (int i = tid; i < row.steps; i += THREADS) mass[i] = 0;
            team_sync<W>();
            const bool all = last == least && last_class == n_classes;      // not cut
            row.template each<2>([&](int step, const float(&v)[RUN], int c) {
                uint64_t sum = 0;
                if (all) {                                    // what is below `least` weighs nothing
#pragma unroll
                    for (int j = 0; j < RUN; ++j)
                        sum += (uint64_t)__double_as_longlong(row_exp2(((double)v[j] - best) * unit) + a.magic);
                    sum -= RUN * zero;
                } else {
                    float s[RUN], high = -INFINITY;
#pragma unroll
                    for (int j = 0; j < RUN; ++j) {
                        s[j] = keeps(v[j], c + j) ? v[j] : -INFINITY;
                        high = row_max(high, s[j]);
                    }
                    if (high > -INFINITY) {
#pragma unroll
                        for (int j = 0; j < RUN; ++j)
                            sum += (uint64_t)__double_as_longlong(row_exp2(((double)s[j] - best) * unit) + a.magic);
                        sum -= RUN * zero;
                    }
                }
                sum = wave_sum(sum);
                if ((tid & 63) == 0 && sum) atomicAdd((unsigned long long*)&mass[step], (unsigned long long)sum);
            });
        }
        team_sync<W>();
        uint64_t sum = 0;
        for (int i = 0; i < row.steps; ++i) sum += mass[i];
        const uint64_t goal = sample_goal(u, sum);
        const double log_sum = row_log((double)sum * a.unit);
        auto answer = [&](float v, int c) {
            index[r] = c;
            logprob[r] = (float)(((double)v - best) / t - log_sum);
        };
        if (goal == 0) {                                      // below one unit: the first entry that is kept
            int at = 1 << 30;
            row.template each<4>([&](int, const float(&v)[RUN], int c) {
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (keeps(v[j], c + j)) at = min(at, c + j);
            });
            at = (int)~(uint32_t)team_max<W>((uint64_t)(uint32_t)~at, part);
            if (tid == 0) answer((float)mine[at], at);
            return true;
        }
        uint64_t run = 0;
        int step = 0;
        while (run + mass[step] <= goal) run += mass[step++];
        {
            const int c = row.first_class(step);
            float v[RUN];
            Row::decode(row.read_any(step), v);
            uint64_t own = 0;
#pragma unroll
            for (int j = 0; j < RUN; ++j)
                if (keeps(v[j], c + j)) own += weigh(v[j]);
            uint64_t before = wave_running(own);
            if (W > 1) {
                if ((tid & 63) == 63) part[tid >> 6] = before;
                team_sync<W>();
#pragma unroll
                for (int k = 0; k < W; ++k)
                    if (k < (tid >> 6)) before += part[k];
            }
            before += run - own;
            if (before <= goal && goal < before + own) {
                bool found = false;
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    const uint64_t m = keeps(v[j], c + j) ? weigh(v[j]) : 0;
                    if (!found && goal < before + m) {
                        found = true;
                        answer(v[j], c + j);
                    }
                    before += m;
                }
            }
        }
        return true;
    };
    if (best == INFINITY || !fast())
        sample_by_radix<DT, W>(mine, n_classes, best, t, top_k, top_p, min_p, u, a, mass, &above, index + r, logprob + r);
}

template <int DT, int W>
static void lsr_sample_team(hipStream_t stream, const void* scores_d, int64_t n_rows, int n_classes, int64_t row_stride,
                            const float* uniform_d, const sample_args& a, int32_t* index_d, float* logprob_d) {
    hipLaunchKernelGGL((lsr_sample_team_kernel<DT, W>), dim3((unsigned)n_rows), dim3(64 * W), 0, stream,
                       (const typename row_type<DT>::type*)scores_d, n_classes, row_stride, uniform_d, a, index_d, logprob_d);
}

// Short rows (at most LSR_QUAD_CLASSES classes), a quad per row.  ORDER: some row is cut by its order.  The weights fall
// with the scores, so a sorted copy of them, without the classes, says which weight is the last one that is kept and how
// many entries of that weight; where not all of those are, they are taken one by one.  The sums are 64-bit floating ones in
// a fixed order.  Bound by vector instructions: 2.2 M x 58 with a top_p takes 393 us for 1 664 of them per 16 rows,
// five times what reading the rows takes; sorting score and class together instead of the weights was slower.
template <int DT, int E, bool ORDER>
__global__ __launch_bounds__(LSR_ROW_THREADS) void lsr_sample_quad_kernel(const typename row_type<DT>::type* __restrict__ scores,
                                                                          int64_t n_rows, int n_classes, int64_t row_stride,
                                                                          const float* __restrict__ uniform, sample_args a,
                                                                          int32_t* __restrict__ index,
                                                                          float* __restrict__ logprob) {
    const row_exp2_t row_exp2;
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
        x[i] = row_clean(x[i]);
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
    const bool greedy = !(t > 0);
    const double unit = ROW_LOG2E / t;
    const float floor = min_p > 0 ? sample_floor(best, t, min_p) : -INFINITY;
    double w[E];
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = row_exp2(((double)x[i] - best) * unit);      // 0 for -infinity
    if (ORDER) {
        const double top_p = a.top_p_d ? (double)a.top_p_d[r] : a.top_p;
        const int cut = a.top_k_d ? a.top_k_d[r] : a.top_k;
        const int top_k = cut > 0 ? cut : 4 * E;
        double s[E], sum = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) s[i] = w[i];
        quad_sort<E>(s, q);
#pragma unroll
        for (int i = 0; i < E; ++i) sum += q * E + i < top_k ? s[i] : 0.0;
        const double target = top_p < 1 ? top_p * quad_sum(sum) : INFINITY;
        double run = quad_before(sum, q), least = INFINITY;
        int kept = 0;                                     // places: one is kept while the weight ahead of it is short
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int place = q * E + i;
            const bool in = (place < top_k) & ((place == 0) | (run < target));
            least = in ? s[i] : least;
            kept += in;
            run += s[i];
        }
        least = quad_min(least);
        kept = quad_sum(kept);
        // entries above the last weight that is kept, and of that weight
        int above = 0, same = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            above += w[i] > least;
            same += w[i] == least;
        }
        above = quad_sum(above);
        int need = kept - above, taken = 0;               // entries of the last weight still to take; bits of those taken
        const bool some = need < quad_sum(same) && least > 0;
        if (__any(some)) {                                // by score, equal ones by class
            while (__any(some && need > 0)) {
                float high = -INFINITY;
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if ((w[i] == least) & !(taken >> i & 1)) high = row_max(high, x[i]);
                high = quad_max(high);
                int first = 1 << 30;
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if ((w[i] == least) & !(taken >> i & 1) & (x[i] == high)) first = min(first, quad_class(i, q));
                first = quad_min(first);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if ((need > 0) & (quad_class(i, q) == first)) taken |= 1 << i;
                --need;
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i)
            if ((w[i] < least) | (some & (w[i] == least) & !(taken >> i & 1))) w[i] = 0;
    }
    double total = 0;
    double lane[E / 4];
    if (__any(min_p > 0)) {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = x[i] < floor ? 0.0 : w[i];
    }
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        lane[g] = (w[4 * g] + w[4 * g + 1]) + (w[4 * g + 2] + w[4 * g + 3]);
        total += quad_sum(lane[g]);
    }
    const double goal = (double)fmaxf(uniform[r], 0.0f) * total;         // the first class for NaN
    double base = 0;
    int at = 1 << 30, end = -1;
#pragma unroll
    for (int g = 0; g < E / 4; ++g) {
        double run = base + quad_before(lane[g], q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            run += w[4 * g + j];
            const bool there = w[4 * g + j] > 0;
            end = there ? quad_class(4 * g + j, q) : end;
            at = (there & (run > goal)) ? min(at, end) : at;
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
        share = (float)((isinf(v) ? 0.0 : ((double)v - best) / t) - row_log(total));
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
    if (temperature > 0 && (temperature < 1e-45 || temperature > 1e38))           // what float32 settings per row can be
        return lsr_fail(ctx, LSR_ERR_LIMIT, "lsr_sample_scores: temperature %g outside 1e-45..1e38", temperature);
    if (n_rows == 0) return LSR_OK;
    if (!uniform_d || !index_d || !logprob_d) return lsr_fail(ctx, LSR_ERR_ARG, "lsr_sample_scores: null pointer");
    LSR_HIP_CHECK(ctx, hipSetDevice(ctx->device));
    const int64_t most = lsr_launch_rows(n_classes);
    if (n_rows > most) {
        for (int64_t r = 0; r < n_rows; r += most) {
            const int failed = lsr_sample_scores(ctx, (const char*)scores_d + r * row_stride * row_dtype_bytes(dtype), dtype,
                                                 n_rows - r < most ? n_rows - r : most, n_classes, row_stride, uniform_d + r,
                                                 temperature, top_k, top_p, min_p, temperature_d ? temperature_d + r : nullptr,
                                                 top_k_d ? top_k_d + r : nullptr, top_p_d ? top_p_d + r : nullptr,
                                                 min_p_d ? min_p_d + r : nullptr, index_d + r, logprob_d + r);
            if (failed) return failed;
        }
        return LSR_OK;
    }
    // weights of up to n_classes entries have to fit 62 bits together
    int shift = 62;
    for (int64_t n = 1; n < n_classes; n *= 2) --shift;
    if (shift > 52) shift = 52;
    sample_args a = {temperature, top_p,  min_p, top_k, temperature_d, top_p_d, min_p_d, top_k_d, ldexp(1.0, 52 - shift),
                     ldexp(1.0, -shift)};
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
    LSR_DTYPE_SWITCH(dtype, LSR_WAVES_SWITCH(n_classes, lsr_sample_team<DT, W>(ctx->stream, scores_d, n_rows, (int)n_classes,
                                                                               row_stride, uniform_d, a, index_d, logprob_d)));
    lsr_prof_end(ctx);
    LSR_LAUNCH_CHECK(ctx, "lsr_sample_team_kernel");
    return LSR_OK;
}
