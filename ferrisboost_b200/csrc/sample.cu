// Drawing a class from a row of scores (fbgpu_sample).
//
// A class of score x weighs w = floor(2^40 exp((x - max) / T)).  Every limit
// keeps a beginning of the order (score falling, equal scores by class), so
// what is kept is "every class above a threshold score, and the first `ties`
// classes of that score": the threshold is found, and the row is not sorted
// (only the few candidates of a small top_k are).  Sums of weights are 64-bit
// whole numbers: 2^20 classes of at most 2^40 fit, and no order of additions
// changes them, so every kernel below gives the same draw.  2^-40 of the first
// class's weight is the unit because the products by 2^40 are exact in f32 and
// the sums of 2^20 classes fit; what is less is never drawn.
#include <cfloat>

#include <cooperative_groups.h>

#include "ops.h"

namespace fbg {
namespace {

using u64 = unsigned long long;

// A row's limits.
struct Limits {
    float inv_t, min_p;
    double top_p;
    uint32_t top_k;
    bool greedy, use_p;
};

__device__ __forceinline__ Limits limits_of(const fbgpu_sample_params& p, uint64_t r, uint32_t classes) {
    Limits l;
    const float t = p.temperatures ? p.temperatures[r] : p.temperature;
    const int32_t k = p.top_ks ? p.top_ks[r] : p.top_k;
    const float tp = p.top_ps ? p.top_ps[r] : p.top_p;
    const float mp = p.min_ps ? p.min_ps[r] : p.min_p;
    l.greedy = !(t > 0.0f);
    l.inv_t = l.greedy ? 0.0f : __fdiv_rn(1.0f, fminf(fmaxf(t, FLT_MIN), FLT_MAX));  // neither 0 nor infinite
    l.top_k = k < 1 || (uint32_t)k > classes ? classes : (uint32_t)k;
    l.use_p = tp < 1.0f;
    l.top_p = tp > 0.0f ? (double)tp : 0.0;
    l.min_p = mp > 1.0f ? 1.0f : mp;
    return l;
}

// NaN as -infinity; where scores become keys, also -0 as +0 (they are equal scores).
__device__ __forceinline__ float ruled(float x) { return fmaxf(x, -INFINITY); }
__device__ __forceinline__ float score(float x) { return __fadd_rn(ruled(x), 0.0f); }
// Unsigned order of the scores.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// `top` is finite (see the two kernels for a maximum of +infinity).
__device__ __forceinline__ float exp_of(float x, float top, float inv_t) {
    return expf(__fmul_rn(__fsub_rn(x, top), inv_t));
}
// exp * 2^40 is exact; what is below 2^-40 of the maximum weighs nothing.
__device__ __forceinline__ u64 weight_of(float e) { return __float2ull_rz(__fmul_rn(e, 1099511627776.0f)); }

__device__ __forceinline__ u64 goal_of(double top_p, u64 total) {
    const u64 g = (u64)__double2ll_rz(ceil(__dmul_rn(top_p, __ull2double_rn(total))));
    return g < 1 ? 1 : g;
}
__device__ __forceinline__ u64 place_of(float u, u64 total) {
    const u64 p = u > 0.0f ? (u64)__double2ll_rz(__dmul_rn((double)u, __ull2double_rn(total))) : 0;
    return p < total ? p : total - 1;
}
__device__ __forceinline__ float share_of(u64 w, u64 total) {
    return __double2float_rn(__ddiv_rn(__ull2double_rn(w), __ull2double_rn(total)));
}

// Where a > b, u += x, else v += y: predicated additions (choosing the addends instead takes twice the operations).
__device__ __forceinline__ void add_by(float a, float b, u64& u, u64 x, u64& v, u64 y) {
    asm("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %4, %5;\n\t@p add.u64 %0, %0, %2;\n\t@!p add.u64 %1, %1, %3;\n\t}"
        : "+l"(u), "+l"(v)
        : "l"(x), "l"(y), "f"(a), "f"(b));
}
// Where x >= mid, sum += w and over = min(over, x), else under = max(under, x).
__device__ __forceinline__ void part_by(float x, float mid, u64& sum, u64 w, float& over, float& under) {
    asm("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %3, %4;\n\t@p add.u64 %0, %0, %5;\n\t@p min.f32 %1, %1, %3;\n\t"
        "@!p max.f32 %2, %2, %3;\n\t}"
        : "+l"(sum), "+f"(over), "+f"(under)
        : "f"(x), "f"(mid), "l"(w));
}

// ------------------------------------------------------- a thread per row
// Up to KP classes in registers.  A class's place in the order and the weight
// before it come from comparing all pairs.  10^6 rows of 7 f32 with top_p 0.9: 27 us
// (1.5 TB/s; 17 without top_p), bound by the issue of about 560 operations for 32
// rows.
template <class T, int KP>
__global__ void __launch_bounds__(128) k_sample_thread(const T* __restrict__ scores, uint64_t n, uint32_t classes,
                                                       uint64_t stride, const float* __restrict__ u,
                                                       fbgpu_sample_params params, int32_t* __restrict__ out_classes,
                                                       float* __restrict__ out_probs) {
    for (uint64_t r = (uint64_t)blockIdx.x * 128 + threadIdx.x; r < n; r += (uint64_t)gridDim.x * 128) {
        const T* row = scores + r * stride;
        const Limits l = limits_of(params, r, classes);
        float x[KP], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < KP; i++) {
            x[i] = i < classes ? ruled(to_f32(row[i])) : -INFINITY;
            top = fmaxf(top, x[i]);
        }
        int32_t drawn = -1;
        float share = 0.0f;
        if (l.greedy && top > -INFINITY) {
#pragma unroll
            for (int i = KP - 1; i >= 0; i--)
                if (x[i] == top) drawn = i;
            share = 1.0f;
        } else if (top > -INFINITY) {
            if (top == INFINITY) {  // only the infinite ones weigh
#pragma unroll
                for (int i = 0; i < KP; i++) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
                top = 0.0f;
            }
            u64 w[KP];
            uint32_t keep = ~0u;
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const float e = exp_of(x[i], top, l.inv_t);
                w[i] = weight_of(e);
                if (l.min_p > 0.0f && e < l.min_p) keep &= ~(1u << i);
            }
            u64 sum = 0;
            if (l.top_k < classes) {
#pragma unroll
                for (int i = 0; i < KP; i++) {
                    uint32_t rank = 0;
#pragma unroll
                    for (int j = 0; j < KP; j++)
                        if (j != i) rank += j < i ? x[j] >= x[i] : x[j] > x[i];
                    if (rank >= l.top_k) keep &= ~(1u << i);
                    else sum += w[i];
                }
            } else if (l.use_p) {
#pragma unroll
                for (int i = 0; i < KP; i++) sum += w[i];
            }
            if (l.use_p) {
                const u64 goal = goal_of(l.top_p, sum);
                u64 before[KP] = {};  // the weight of the classes in front of each
#pragma unroll
                for (int i = 0; i < KP; i++) {
#pragma unroll
                    for (int j = i + 1; j < KP; j++)  // the later class comes first where its score is above
                        add_by(x[j], x[i], before[i], w[j], before[j], w[i]);
                }
#pragma unroll
                for (int i = 0; i < KP; i++)
                    if (before[i] >= goal) keep &= ~(1u << i);
            }
            u64 total = 0;
#pragma unroll
            for (int i = 0; i < KP; i++) total += w[i] = keep >> i & 1 ? w[i] : 0;
            const u64 place = place_of(u[r], total);
            u64 run = 0, won = 0;
#pragma unroll
            for (int i = 0; i < KP; i++) {
                run += w[i];
                if (run > place && drawn < 0) drawn = i, won = w[i];
            }
            share = share_of(won, total);
        }
        out_classes[r] = drawn;
        if (out_probs) out_probs[r] = share;
    }
}

// -------------------------------------------------- a few lanes of a warp per row
// L lanes (1 to 8) hold a row in registers, lane l the classes [E * l, E * l + E).
// A limit's threshold is found by halving the range of scores it lies in: each
// round sums what is at or above the middle, and the range's new end is the
// nearest score on its side of the middle, so that about log2(classes) rounds
// find it.  Fewer lanes a row mean fewer rounds for the warp's rows together; a
// lane's 32 scores and weights are what its registers take.
template <class T, int L, int E>
__global__ void __launch_bounds__(128) k_sample_lanes(const T* __restrict__ scores, uint64_t n, uint32_t classes,
                                                      uint64_t stride, const float* __restrict__ u,
                                                      fbgpu_sample_params params, int32_t* __restrict__ out_classes,
                                                      float* __restrict__ out_probs) {
    constexpr int kRows = 128 / L;
    constexpr uint32_t kAll = 0xffffffffu;
    __shared__ float staged[128 * (E + 1)];  // a lane's scores one word apart from the next lane's banks
    const int lane = threadIdx.x & (L - 1);
    float* const own = staged + threadIdx.x * (E + 1);
    auto add_lanes = [](u64 v) {
#pragma unroll
        for (int d = L / 2; d; d /= 2) v += __shfl_xor_sync(kAll, v, d);
        return v;
    };
    auto largest = [](float v) {
#pragma unroll
        for (int d = L / 2; d; d /= 2) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
        return v;
    };
    // the rows of a warp stay together: one past the end works on the last row and writes nothing
    for (uint64_t r0 = (uint64_t)blockIdx.x * kRows; r0 < n; r0 += (uint64_t)gridDim.x * kRows) {
        const uint64_t at = r0 + threadIdx.x / L, r = min(at, n - 1);
        __syncwarp();
        if (L == 1) {
            const T* row = scores + r * stride;
            for (int c = 0; c < E; c++) own[c] = c < classes ? ruled(to_f32(row[c])) : -INFINITY;
        } else {
            const T* row = scores + r * stride;
#pragma unroll 4
            for (int c = lane; c < L * E; c += L) {
                float* to = own + (c / E - lane) * (E + 1) + c % E;
                *to = c < classes ? ruled(to_f32(row[c])) : -INFINITY;
            }
        }
        __syncwarp();
        const Limits l = limits_of(params, r, classes);
        float x[E], top = -INFINITY, bottom = INFINITY;
#pragma unroll
        for (int i = 0; i < E; i++) {
            x[i] = own[i];
            top = fmaxf(top, x[i]);
        }
        top = largest(top);
        if (top == INFINITY) {  // only the infinite ones weigh
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
            top = 0.0f;
        }
        const bool empty = top == -INFINITY;
        u64 w[E];
        uint32_t count = 0, kept = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float e = exp_of(x[i], top, l.inv_t);
            w[i] = x[i] > -INFINITY ? weight_of(e) : 0;
            if (!(e < l.min_p)) kept |= 1u << i;
            if (x[i] > -INFINITY) count++, bottom = fminf(bottom, x[i]);
        }
        bottom = -largest(-bottom);
        count = (uint32_t)add_lanes(count);
        // kept: above `cut`, or equal to it and one of the first `ties` of the `same` of that score
        float cut = -INFINITY;
        uint32_t ties = kAll, same = 0;
        if (l.greedy) cut = top, ties = 1, same = kAll;
#pragma unroll 1
        for (int by_weight = 0; by_weight < 2; by_weight++) {
            bool find = !l.greedy && !empty && (by_weight ? l.use_p : l.top_k < count);
            if (!__any_sync(kAll, find)) continue;
            const float w_cut = exp_of(cut, top, l.inv_t);
            u64 goal = l.top_k;
            if (by_weight) {
                u64 total = 0;
#pragma unroll
                for (int i = 0; i < E; i++) total += x[i] > cut ? w[i] : 0;
                total = add_lanes(total);
                if (ties < kAll) total += min(ties, same) * weight_of(w_cut);
                goal = goal_of(l.top_p, total);
                find = find && goal <= total;
            }
            float lo = by_weight ? fmaxf(bottom, cut) : bottom, hi = top;
            u64 above = 0;  // what is above `hi`, below the goal
            while (__any_sync(kAll, find && lo < hi)) {
                float mid = fminf(__fadd_rn(__fmul_rn(lo, 0.5f), __fmul_rn(hi, 0.5f)), hi);
                if (!(mid > lo)) mid = hi;
                // what is at or above the middle, and the nearest scores on either side of it
                constexpr int kSums = 4;  // chains of additions
                float over[2] = {INFINITY, INFINITY}, under[2] = {-INFINITY, -INFINITY};
                u64 part = 0;
                if (by_weight) {
                    u64 sums[kSums] = {};
#pragma unroll
                    for (int i = 0; i < E; i++) part_by(x[i], mid, sums[i % kSums], w[i], over[i & 1], under[i & 1]);
#pragma unroll
                    for (int i = 0; i < kSums; i++) part += sums[i];
                } else {
                    uint32_t sums[kSums] = {};
#pragma unroll
                    for (int i = 0; i < E; i++) {
                        if (x[i] >= mid) sums[i % kSums]++, over[i & 1] = fminf(over[i & 1], x[i]);
                        else under[i & 1] = fmaxf(under[i & 1], x[i]);
                    }
#pragma unroll
                    for (int i = 0; i < kSums; i++) part += sums[i];
                }
                part = add_lanes(part);
                const bool reached = part >= goal;
                const float near = largest(reached ? -fminf(over[0], over[1]) : fmaxf(under[0], under[1]));
                if (find && lo < hi) {
                    if (reached) lo = -near;
                    else above = part, hi = near;
                }
            }
            uint32_t equal = 0;
#pragma unroll
            for (int i = 0; i < E; i++) equal += x[i] == lo;
            equal = (uint32_t)add_lanes(equal);
            if (find) {
                cut = lo;
                same = equal;
                goal -= above;
                if (by_weight) {
                    const u64 one = weight_of(exp_of(cut, top, l.inv_t));
                    ties = same == 1 ? 1 : (uint32_t)((goal + one - 1) / one);
                } else {
                    ties = (uint32_t)goal;
                }
            }
        }
        if (__any_sync(kAll, ties < same)) {  // the lane's first class of the score `cut`, counted over the row
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < E; i++) mine += x[i] == cut;
            uint32_t rank = mine;
#pragma unroll
            for (int d = 1; d < L; d *= 2) {
                const uint32_t y = __shfl_up_sync(kAll, rank, d, L);
                if (lane >= d) rank += y;
            }
            rank -= mine;
#pragma unroll
            for (int i = 0; i < E; i++) {
                if (x[i] == cut) {
                    if (rank >= ties) kept &= ~(1u << i);
                    rank++;
                }
            }
        }
        u64 mine = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            if (!(x[i] >= cut) || !(kept >> i & 1)) w[i] = 0;
            mine += w[i];
        }
        u64 upto = mine;
#pragma unroll
        for (int d = 1; d < L; d *= 2) {
            const u64 y = __shfl_up_sync(kAll, upto, d, L);
            if (lane >= d) upto += y;
        }
        const u64 total = __shfl_sync(kAll, upto, L - 1, L);
        if (at >= n) continue;
        if (empty) {
            if (lane == 0) {
                out_classes[r] = -1;
                if (out_probs) out_probs[r] = 0.0f;
            }
            continue;
        }
        const u64 place = place_of(u[r], total);
        u64 run = upto - mine, won = 0;
        if (place < run || place >= upto) continue;  // another lane's
        int drawn = 0;
#pragma unroll
        for (int i = 0; i < E; i++) {
            if (place >= run && place < run + w[i]) drawn = i, won = w[i];
            run += w[i];
        }
        out_classes[r] = lane * E + drawn;
        if (out_probs) out_probs[r] = share_of(won, total);
    }
}

// ------------------------------------------------- a block or cluster per row
// WARPS warps of CTAS blocks (one cluster) hold a row.  Its scores are brought
// into shared memory once (HELD; other rows are read again for every
// step, from the L2) and every later step is a short loop over them: held in
// registers, the unrolled steps ran out of the instruction cache.  Places are
// counted from the 16-byte boundary at or before the row's first class, so that
// the loads are aligned vectors; the places before that class, and after the
// last, hold -infinity.  Block after block, and in it warp after warp, takes
// a contiguous part of the places; a step is four of a lane.  Up to kSort classes
// are sorted, and short rows take fewer bins.
template <int WARPS, int CTAS> struct alignas(16) RowShared {
    static constexpr int kBins = WARPS <= 4 ? 256 : 1024, kSort = WARPS <= 2 ? 256 : WARPS == 4 ? 512 : 1024;
    static constexpr int kListed = WARPS <= 4 ? 64 : kSort;  // top_k up to here goes by a list: few threads sort slowly
    static constexpr int kCount = 256;                 // lists up to here are ordered by counting
    uint32_t low[kBins], high[kBins];     // a bin's count, or its weight as two words; then the picked keys
    u64 all[CTAS > 1 ? kBins : 1];        // a cluster's bins
    u64 part[2][WARPS];                   // warps' partial sums; two sets, used in turn
    uint32_t found[3];                    // members of the chosen bin; of the list to sort
    u64 scan[WARPS];
    u64 before, pick_above;
    uint32_t bin, pick_key, pick_same, tie_place;
    union {
        uint32_t key[2][kSort];           // members of the chosen bin
        u64 sorted[kSort];
    };
    u64 sorted_weight[kSort];
    u64 chunk[WARPS][8];                  // a warp's kept weight in eighths of its part
};

template <class T, bool HELD, int WARPS, int CTAS> struct RowDraw {
    using Sh = RowShared<WARPS, CTAS>;
    static constexpr int kBins = Sh::kBins, kSort = Sh::kSort, kListed = Sh::kListed, kThreads = WARPS * 32, kStep = 128;

    Sh& s;
    T* x;                 // HELD: the block's places
    const T* row;
    uint32_t classes, shift;
    uint32_t steps;       // of a warp
    uint32_t block_first, warp_first;  // first places
    int lane, warp, tid, cta, parity = 0;
    float most;           // HELD: the largest score that this thread brought

    __device__ __forceinline__ RowDraw(Sh& sh, T* held, uint32_t steps_) : s(sh), x(held), steps(steps_) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        tid = threadIdx.x;
        cta = CTAS == 1 ? 0 : (int)cooperative_groups::this_cluster().block_rank();
        block_first = cta * WARPS * steps * kStep;
        warp_first = block_first + warp * steps * kStep;
    }

    __device__ __forceinline__ void sync_row() {
        if (CTAS == 1) __syncthreads();
        else cooperative_groups::this_cluster().sync();
    }
    // Another block's shared memory.
    template <class V> __device__ __forceinline__ V* at(V* p, int c) {
        if (CTAS == 1) return p;
        return cooperative_groups::this_cluster().map_shared_rank(p, c);
    }
    __device__ __forceinline__ float one(uint32_t place) {
        return place >= shift && place < shift + classes ? to_f32(row[place - shift]) : -INFINITY;
    }
    __device__ __forceinline__ bool inside(uint32_t place, uint32_t count) {
        return place >= shift && place + count <= shift + classes;
    }

    __device__ __forceinline__ void open(const T* row_, uint32_t classes_) {
        constexpr int V = 16 / sizeof(T), kAhead = 4;
        row = row_;
        classes = classes_;
        shift = (uint32_t)(((uintptr_t)row % 16) / sizeof(T));
        if (!HELD) return;
        most = -INFINITY;
        __syncthreads();  // the row before is no longer read
        const uint32_t vectors = WARPS * steps * kStep / V;
        for (uint32_t v0 = tid; v0 < vectors; v0 += kAhead * kThreads) {
            union {
                uint4 u;
                T v[V];
            } p[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const uint32_t place = block_first + (v0 + k * kThreads) * V;
                p[k].u = *(inside(place, V) ? reinterpret_cast<const uint4*>(row + (place - shift)) : &g_zero);
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const uint32_t v = v0 + k * kThreads, place = block_first + v * V;
                if (v >= vectors) break;
                if (!inside(place, V)) {
#pragma unroll
                    for (int i = 0; i < V; i++) p[k].v[i] = from_f32<T>(one(place + i));
                }
#pragma unroll
                for (int i = 0; i < V; i++) most = fmaxf(most, to_f32(p[k].v[i]));
                *reinterpret_cast<uint4*>(x + v * V) = p[k].u;
            }
        }
        __syncthreads();
    }
    // f(four scores, place of the first) for the lane's steps [from, to), in order.  A score may be NaN.
    template <class F> __device__ __forceinline__ void steps_of_warp(uint32_t from, uint32_t to, F&& f) {
        if (HELD) {
            const T* mine = x + (warp_first - block_first) + lane * 4;
#pragma unroll 2
            for (uint32_t i = from; i < to; i++) {
                const Pack<T, 4> q = *reinterpret_cast<const Pack<T, 4>*>(mine + i * kStep);
                Pack<float, 4> p;
#pragma unroll
                for (int j = 0; j < 4; j++) p.v[j] = to_f32(q.v[j]);
                f(p, warp_first + i * kStep + lane * 4);
            }
            return;
        }
        constexpr int kAhead = 4;
#pragma unroll 1
        for (uint32_t i = from; i < to; i += kAhead) {
            const uint32_t place = warp_first + i * kStep + lane * 4;
            if (i + kAhead <= to && inside(warp_first + i * kStep, kAhead * kStep)) {
                Pack<T, 4> q[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; k++)
                    q[k] = *reinterpret_cast<const Pack<T, 4>*>(row + (place - shift) + k * kStep);
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    Pack<float, 4> p;
#pragma unroll
                    for (int j = 0; j < 4; j++) p.v[j] = to_f32(q[k].v[j]);
                    f(p, place + k * kStep);
                }
            } else {
#pragma unroll 1
                for (uint32_t k = 0; k < kAhead && i + k < to; k++) {
                    Pack<float, 4> p;
#pragma unroll
                    for (int j = 0; j < 4; j++) p.v[j] = one(place + k * kStep + j);
                    f(p, place + k * kStep);
                }
            }
        }
    }
    template <class F> __device__ __forceinline__ void each_step(F&& f) { steps_of_warp(0, steps, f); }
    // f(score) for each of the lane's places
    template <class F> __device__ __forceinline__ void each(F&& f) {
        each_step([&](const Pack<float, 4>& p, uint32_t) {
#pragma unroll
            for (int k = 0; k < 4; k++) f(p.v[k]);
        });
    }

    // A reduction over the row's threads; op is commutative.  `before` gets the
    // result over the warps in front of this one.
    template <class Op> __device__ __forceinline__ u64 reduce(u64 v, u64 zero, Op&& op, u64* before = nullptr) {
#pragma unroll
        for (int d = 16; d; d /= 2) v = op(v, (u64)__shfl_xor_sync(0xffffffffu, v, d));
        if (before) *before = zero;
        if (lane == 0) s.part[parity][warp] = v;
        sync_row();
        u64 all = zero, front = zero;
#pragma unroll
        for (int c = 0; c < CTAS; c++) {
            // lane w takes warp w's value
            const u64 y = lane < WARPS ? at(s.part[parity], c)[lane] : zero;
            all = op(all, y);
            if (c < cta || (c == cta && lane < warp)) front = op(front, y);
        }
#pragma unroll
        for (int d = 16; d; d /= 2) {
            all = op(all, (u64)__shfl_xor_sync(0xffffffffu, all, d));
            if (before) front = op(front, (u64)__shfl_xor_sync(0xffffffffu, front, d));
        }
        if (before) *before = front;
        parity ^= 1;
        return all;
    }
    __device__ __forceinline__ u64 sum(u64 v, u64* before = nullptr) {
        return reduce(v, 0, [](u64 a, u64 b) { return a + b; }, before);
    }
    // Over the block's threads: the sum in front of this one, and the total.
    __device__ __forceinline__ u64 block_before(u64 mine, u64& total) {
        u64 upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += y;
        }
        __syncthreads();
        if (lane == 31) s.scan[warp] = upto;
        __syncthreads();
        u64 all = lane < WARPS ? s.scan[lane] : 0, front = lane < warp ? all : 0;
#pragma unroll
        for (int d = 16; d; d /= 2) {
            all += __shfl_xor_sync(0xffffffffu, all, d);
            front += __shfl_xor_sync(0xffffffffu, front, d);
        }
        total = all;
        return upto - mine + front;
    }

    // How far a score lies below the maximum, in bins.
    __device__ __forceinline__ float depth(float v, float top, float per) { return __fmul_rn(__fsub_rn(v, top), -per); }
    // The nearest whole number by the addition of 2^23, whose low bits it becomes; monotone like the depth.
    __device__ __forceinline__ uint32_t bin_of(float d) {
        return __float_as_uint(__fadd_rn(fminf(d, kBins - 1.0f), 8388608.0f)) & (kBins - 1);
    }
    __device__ __forceinline__ void clear_bins(int set) {
        for (int i = tid; i < kBins; i += kThreads) s.low[i] = s.high[i] = 0;
        if (tid == 0) s.found[set] = 0, s.bin = kBins;
        __syncthreads();
    }
    // After the bins are filled: the bin in which the running sum reaches the goal that goal_for(total) names
    // (kBins: none), and the sum before it.  With `whole` over the cluster (each block adds up its share of
    // the bins and tells the others), else over the block.
    template <class G> __device__ __forceinline__ uint32_t find_bin(bool whole, u64& before, u64& goal, G&& goal_for) {
        constexpr int kPer = kBins / kThreads;
        if (CTAS > 1 && whole) {
            sync_row();
            constexpr int kShare = kBins / CTAS;
            for (int i = tid; i < kShare; i += kThreads) {
                const int b = cta * kShare + i;
                u64 v = 0;
#pragma unroll
                for (int c = 0; c < CTAS; c++) v += (u64)at(s.high, c)[b] << 32 | at(s.low, c)[b];
#pragma unroll
                for (int c = 0; c < CTAS; c++) at(s.all, c)[b] = v;
            }
            sync_row();
        } else {
            __syncthreads();
        }
        u64 v[kPer], mine = 0, total;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int b = tid * kPer + i;
            v[i] = CTAS > 1 && whole ? s.all[b] : (u64)s.high[b] << 32 | s.low[b];
            mine += v[i];
        }
        u64 run = block_before(mine, total);
        goal = goal_for(total);
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            if (run < goal && goal <= run + v[i]) {
                s.bin = tid * kPer + i;
                s.before = run;
            }
            run += v[i];
        }
        __syncthreads();
        before = s.before;
        return s.bin;
    }

    // Bitonic, falling, of a power of two of items.
    __device__ __forceinline__ void sort(u64* a, uint32_t count) {
        for (uint32_t k = 2; k <= count; k *= 2) {
            for (uint32_t j = k / 2; j; j /= 2) {
                for (uint32_t i = tid; i < count / 2; i += kThreads) {
                    const uint32_t lo = (i & ~(j - 1)) << 1 | (i & (j - 1)), hi = lo | j;
                    const u64 u = a[lo], v = a[hi];
                    if ((u < v) == ((lo & k) == 0)) a[lo] = v, a[hi] = u;
                }
                __syncthreads();
            }
        }
    }

    // Orders s.sorted[0, members), falling: short lists by counting what is larger than each.
    __device__ __forceinline__ void order(uint32_t members) {
        if (members <= Sh::kCount) {
            for (uint32_t i = tid; i < members; i += kThreads) {
                const u64 mine = s.sorted[i];
                uint32_t rank = 0;
#pragma unroll 8
                for (uint32_t j = 0; j < members; j++) rank += s.sorted[j] > mine;
                s.sorted_weight[rank] = mine;
            }
            __syncthreads();
            for (uint32_t i = tid; i < members; i += kThreads) s.sorted[i] = s.sorted_weight[i];
            __syncthreads();
        } else {
            uint32_t count = Sh::kCount;
            while (count < members) count *= 2;
            for (uint32_t i = members + tid; i < count; i += kThreads) s.sorted[i] = 0;
            __syncthreads();
            sort(s.sorted, count);
        }
    }

    // The draw from a list of the row's first `members` classes, by one block; the limits end inside it.
    __device__ __forceinline__ void draw_sorted(uint32_t members, uint64_t r, const Limits& l, float top, float u,
                                                int32_t* out_classes, float* out_probs) {
        constexpr int kPer = kSort / kThreads;
        __syncthreads();
        order(members);
        u64 item[kPer], w[kPer], mine = 0, total;
        float e[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const uint32_t rank = tid * kPer + i;
            item[i] = rank < members && rank < l.top_k ? s.sorted[rank] : 0;
            e[i] = item[i] ? exp_of(score_of((uint32_t)(item[i] >> 32)), top, l.inv_t) : 0.0f;
            w[i] = weight_of(e[i]);
            mine += w[i];
        }
        u64 before = block_before(mine, total);
        const u64 goal = l.use_p ? goal_of(l.top_p, total) : ~0ull;
        mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const uint32_t rank = tid * kPer + i;
            const bool keep = item[i] && before < goal && !(e[i] < l.min_p);
            before += w[i];
            if (!keep) w[i] = 0;
            mine += w[i];
            s.sorted_weight[rank] = w[i];
            // to be ordered by class: the low word is the class's complement
            s.sorted[rank] = keep ? item[i] << 32 | rank : 0;
        }
        block_before(mine, total);
        const u64 place = place_of(u, total);
        // what is kept is a beginning of the list: at most this many
        const uint32_t kept = min(members, l.top_k);
        auto win = [&](u64 run, u64 weight, uint32_t complement) {
            if (place >= run && place < run + weight) {
                out_classes[r] = (int32_t)~complement;
                if (out_probs) out_probs[r] = share_of(weight, total);
            }
        };
        __syncthreads();
        if (kept <= Sh::kCount) {  // the weight of the lower classes, by comparing each with all
            for (uint32_t i = tid; i < kept; i += kThreads) {
                const u64 key = s.sorted[i];
                u64 run = 0;
#pragma unroll 8
                for (uint32_t j = 0; j < kept; j++) run += s.sorted[j] > key ? s.sorted_weight[j] : 0;
                win(run, s.sorted_weight[i], (uint32_t)(key >> 32));
            }
            return;
        }
        uint32_t count = Sh::kCount;
        while (count < kept) count *= 2;
        sort(s.sorted, count);
        mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const uint32_t q = tid * kPer + i;
            item[i] = q < count ? s.sorted[q] : 0;
            w[i] = item[i] ? s.sorted_weight[(uint32_t)item[i]] : 0;
            mine += w[i];
        }
        u64 all, run = block_before(mine, all);
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            win(run, w[i], (uint32_t)(item[i] >> 32));
            run += w[i];
        }
    }

    __device__ __forceinline__ void draw(uint64_t r, const fbgpu_sample_params& params, const float* u,
                                         int32_t* out_classes, float* out_probs) {
        const Limits l = limits_of(params, r, classes);
        if (!HELD) {
            most = -INFINITY;
            each([&](float v) { most = fmaxf(most, v); });
        }
        const float top = score_of((uint32_t)reduce(key_of(score(most)), 0, [](u64 a, u64 b) { return a > b ? a : b; }));
        if (top == -INFINITY) {
            if (tid == 0 && cta == 0) {
                out_classes[r] = -1;
                if (out_probs) out_probs[r] = 0.0f;
            }
            return;
        }
        // Weights vanish 27.73 T below the maximum: bins over that span, falling, the last for the rest.
        const float per = fminf(__fmul_rn(kBins / 27.75f, l.inv_t), FLT_MAX);
        if (!l.greedy && top < INFINITY && l.top_k < classes && l.top_k <= kListed) {
            // The classes down to a bin that holds the top_k-th of the threads' maxima (or, where there are too few
            // threads, of all classes) are at least top_k: those are sorted.  For a short list a cluster saves
            // the sum of its bins: each block finds the bin of its share, and the lowest of these will do.  (Not for
            // 16-bit scores, whose many equal ones make that list long.)
            const bool whole = CTAS == 1 || l.top_k > 64 || sizeof(T) == 2;
            const uint32_t share = whole ? l.top_k : (l.top_k + CTAS - 1) / CTAS;
            clear_bins(2);
            if (share * 4 <= kThreads * (whole ? CTAS : 1)) {
                if (most > -INFINITY) atomicAdd(&s.low[bin_of(depth(most, top, per))], 1u);
            } else {
                each([&](float v) {
                    if (v > -INFINITY) atomicAdd(&s.low[bin_of(depth(v, top, per))], 1u);
                });
            }
            u64 before, goal;
            uint32_t bin = find_bin(whole, before, goal, [&](u64) { return (u64)share; });
            if (!whole) bin = (uint32_t)reduce(bin, 0, [](u64 a, u64 b) { return a > b ? a : b; });
            const float end = bin >= kBins - 1 ? INFINITY : bin + 0.5f;  // and what is rounded down from just there
            each_step([&](const Pack<float, 4>& p, uint32_t place) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (depth(p.v[i], top, per) <= end && p.v[i] > -INFINITY) {
                        const uint32_t q = atomicAdd(&s.found[2], 1u);
                        if (q < kSort) s.sorted[q] = (u64)key_of(score(p.v[i])) << 32 | ~(place + i - shift);
                    }
                }
            });
            sync_row();
            uint32_t members = 0;
            for (int c = 0; c < CTAS; c++) members += *at(&s.found[2], c);
            if (members <= kSort) {
                if (cta == 0) {
                    uint32_t base = s.found[2];
                    for (int c = 1; c < CTAS; c++) {
                        const uint32_t m = *at(&s.found[2], c);
                        for (uint32_t i = tid; i < m; i += kThreads) s.sorted[base + i] = at(s.sorted, c)[i];
                        base += m;
                    }
                    draw_sorted(members, r, l, top, u[r], out_classes, out_probs);
                }
                return;
            }
        }
        // kept: above `cut`, or equal to it and one of the first `ties` of the `same` classes of that score
        float cut = -INFINITY;
        uint32_t ties = 0xffffffffu, same = 0;
        if (l.greedy) {
            cut = top;
            ties = 1;
            same = 0xffffffffu;
        } else if (top == INFINITY) {  // the infinite ones alone, of one weight
            u64 count = 0;
            each([&](float v) { count += v == INFINITY; });
            cut = top;
            same = (uint32_t)sum(count);
            ties = min(l.top_k, same);
            if (l.use_p) ties = (uint32_t)((goal_of(l.top_p, (u64)ties << 40) + (1ull << 40) - 1) >> 40);
        } else {
            // first by count for top_k, then by weight for top_p
#pragma unroll 1
            for (int by_weight = 0; by_weight < 2; by_weight++) {
                if (by_weight ? !l.use_p : l.top_k >= classes) continue;
                clear_bins(by_weight);
                each([&](float v) {
                    if (!(v >= cut && v > -INFINITY)) return;
                    const uint32_t b = bin_of(depth(v, top, per));
                    if (by_weight) {
                        const u64 w = weight_of(exp_of(v, top, l.inv_t));
                        if (w == 0) return;
                        const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.low[b], lo);
                        const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < lo);
                        if (hi) atomicAdd(&s.high[b], hi);
                    } else {
                        atomicAdd(&s.low[b], 1u);
                    }
                });
                u64 before, goal;
                const uint32_t bin = find_bin(true, before, goal, [&](u64 total) -> u64 {
                    if (!by_weight) return l.top_k;
                    if (ties < same) total -= (same - ties) * weight_of(exp_of(cut, top, l.inv_t));
                    return goal_of(l.top_p, total);
                });
                if (bin == kBins) {  // the whole row stays below the goal
                    if (CTAS > 1) sync_row();  // the other blocks may still read these bins
                    continue;
                }
                goal -= before;
                // the chosen bin's members
                auto member = [&](float v) {
                    return v >= cut && v > -INFINITY && bin_of(depth(v, top, per)) == bin;
                };
                uint32_t* const list = s.key[by_weight];
                each([&](float v) {
                    if (!member(v)) return;
                    const uint32_t q = atomicAdd(&s.found[by_weight], 1u);
                    if (q < kSort) list[q] = key_of(score(v));
                });
                sync_row();
                uint32_t members = 0;
                bool listed = true;
                for (int c = 0; c < CTAS; c++) {
                    const uint32_t m = *at(&s.found[by_weight], c);
                    members += m;
                    listed = listed && m <= kSort;
                }
                auto weight = [&](uint32_t key) -> u64 {
                    return by_weight ? weight_of(exp_of(score_of(key), top, l.inv_t)) : 1;
                };
                u64 above = 0;
                uint32_t key = 0;
                auto least = [](u64 a, u64 b) { return a < b ? a : b; };
                auto largest = [](u64 a, u64 b) { return a > b ? a : b; };
                if (listed) {
                    // While there are many, bins over the range of their keys leave fewer, or one key alone, as
                    // where scores are coarse.
                    const uint32_t* from = list;
                    uint32_t set = by_weight, lo = 0, hi = 0xffffffffu;
                    while (members > Sh::kCount) {
                        const uint32_t mine = s.found[set];
                        lo = 0xffffffffu, hi = 0;
                        for (uint32_t i = tid; i < mine; i += kThreads) lo = min(lo, from[i]), hi = max(hi, from[i]);
                        lo = (uint32_t)reduce(lo, 0xffffffffu, least);
                        hi = (uint32_t)reduce(hi, 0, largest);
                        if (lo == hi) break;
                        int down = 0;
                        while ((hi - lo) >> down >= kBins) down++;
                        // the list of the bin found goes where the other limit's was, and then back
                        const uint32_t other = set == 2 ? by_weight : 2;
                        uint32_t* const to = s.key[other == 2 ? 1 - by_weight : by_weight];
                        clear_bins(other);
                        for (uint32_t i = tid; i < mine; i += kThreads) {
                            const u64 w = weight(from[i]);
                            const uint32_t b2 = (hi - from[i]) >> down, low = (uint32_t)w;
                            const uint32_t old = low ? atomicAdd(&s.low[b2], low) : 0;
                            const uint32_t high = (uint32_t)(w >> 32) + (old + low < low);
                            if (high) atomicAdd(&s.high[b2], high);
                        }
                        u64 front, same_goal;
                        const uint32_t b3 = find_bin(true, front, same_goal, [&](u64) { return goal; });
                        goal -= front;
                        for (uint32_t i = tid; i < mine; i += kThreads) {
                            if ((hi - from[i]) >> down == b3) to[atomicAdd(&s.found[other], 1u)] = from[i];
                        }
                        sync_row();
                        members = 0;
                        for (int c = 0; c < CTAS; c++) members += *at(&s.found[other], c);
                        from = to;
                        set = other;
                    }
                    if (lo == hi) {
                        key = lo;
                        same = members;
                    } else {  // each compared with all
                        uint32_t* const all_key = s.low;  // of no more use
                        u64* const all_weight = s.sorted_weight;
                        uint32_t base = 0;
                        for (int c = 0; c < CTAS; c++) {
                            const uint32_t m = *at(&s.found[set], c);
                            for (uint32_t i = tid; i < m; i += kThreads) {
                                const uint32_t k = at(from, c)[i];
                                all_key[base + i] = k;
                                all_weight[base + i] = weight(k);
                            }
                            base += m;
                        }
                        __syncthreads();
                        for (uint32_t i = tid; i < members; i += kThreads) {
                            const uint32_t k = all_key[i];
                            u64 front = 0;
                            uint32_t equal = 0;
#pragma unroll 4
                            for (uint32_t j = 0; j < members; j++) {
                                const uint32_t other = all_key[j];
                                front += other > k ? all_weight[j] : 0;
                                equal += other == k;
                            }
                            if (front < goal && goal <= front + equal * all_weight[i]) {  // all of that key agree
                                s.pick_key = k;
                                s.pick_same = equal;
                                s.pick_above = front;
                            }
                        }
                        __syncthreads();
                        key = s.pick_key;
                        same = s.pick_same;
                        above = s.pick_above;
                    }
                } else {
                    // More than a list holds, as in flat rows, whose scores lie within few bins: halve the range
                    // of their keys, reading the row (1000 rows of 20000 normal f32 scores with top_p 0.9: 123 us
                    // at deviation 2, 352 at 0.1; 577 at deviation 2 and T = 100).  All above `hi` have the weight
                    // `above`, below the goal; with those from `lo` on it is reached.  The ends are keys that occur.
                    auto each_member = [&](auto&& f) {
                        each([&](float v) {
                            if (member(v)) f(key_of(score(v)));
                        });
                    };
                    uint32_t lo = 0xffffffffu, hi = 0;
                    each_member([&](uint32_t k) { lo = min(lo, k), hi = max(hi, k); });
                    lo = (uint32_t)reduce(lo, 0xffffffffu, least);
                    hi = (uint32_t)reduce(hi, 0, largest);
                    while (lo < hi) {
                        const uint32_t mid = lo + (hi - lo + 1) / 2;
                        u64 part = 0;
                        uint32_t under = 0, over = 0xffffffffu;  // the nearest keys on either side of mid
                        each_member([&](uint32_t k) {
                            if (k < lo || k > hi) return;
                            if (k >= mid) {
                                part += weight(k);
                                over = min(over, k);
                            } else {
                                under = max(under, k);
                            }
                        });
                        part = sum(part);
                        if (above + part >= goal) {
                            lo = (uint32_t)reduce(over, 0xffffffffu, least);
                        } else {
                            above += part;
                            hi = (uint32_t)reduce(under, 0, largest);
                        }
                    }
                    key = lo;
                    u64 equal = 0;
                    each_member([&](uint32_t k) { equal += k == key; });
                    same = (uint32_t)sum(equal);
                }
                cut = score_of(key);
                const u64 each_w = weight(key);
                ties = (uint32_t)((goal - above + each_w - 1) / each_w);
            }
        }
        // Where not all classes of the score `cut` are kept: the last place that is.
        uint32_t tie_place = 0xffffffffu;
        if (ties < same) {
            u64 equal = 0, front;
            each([&](float v) { equal += v == cut; });
            const uint32_t mine = __reduce_add_sync(0xffffffffu, (uint32_t)equal);
            sum(equal, &front);
            if (front < ties && ties <= front + mine) {  // in this warp's part
                uint32_t passed = (uint32_t)front;
                steps_of_warp(0, steps, [&](const Pack<float, 4>& p, uint32_t place) {
                    uint32_t here = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) here += p.v[i] == cut;
                    const uint32_t all = __reduce_add_sync(0xffffffffu, here);
                    if (passed < ties && ties <= passed + all) {
                        uint32_t upto = here;
#pragma unroll
                        for (int d = 1; d < 32; d *= 2) {
                            const uint32_t y = __shfl_up_sync(0xffffffffu, upto, d);
                            if (lane >= d) upto += y;
                        }
                        uint32_t rank = passed + upto - here;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (p.v[i] == cut && ++rank == ties)
                                for (int c = 0; c < CTAS; c++) *at(&s.tie_place, c) = place + i;
                        }
                    }
                    passed += all;
                });
            }
            sync_row();
            tie_place = s.tie_place;
        }
        // The kept weights of a step.
        auto weigh = [&](const Pack<float, 4>& p, uint32_t place, u64* w) -> u64 {
            u64 sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = p.v[i];
                w[i] = 0;
                if (v > cut || (v == cut && place + i <= tie_place)) {
                    const float e = v == top ? 1.0f : exp_of(v, top, l.inv_t);
                    if (!(e < l.min_p)) w[i] = weight_of(e);
                }
                sum += w[i];
            }
            return sum;
        };
        // the warp's weight by eighths of its part, so that only one eighth is walked again
        const uint32_t eighth = (steps + 7) / 8, eighths = (steps + eighth - 1) / eighth;
        u64 mine = 0, before = 0;
#pragma unroll 1
        for (uint32_t e = 0; e < eighths; e++) {
            u64 part = 0;
            steps_of_warp(e * eighth, min(steps, (e + 1) * eighth), [&](const Pack<float, 4>& p, uint32_t place) {
                u64 w[4];
                part += weigh(p, place, w);
            });
            mine += part;
#pragma unroll
            for (int d = 16; d; d /= 2) part += __shfl_xor_sync(0xffffffffu, part, d);
            if (lane == 0) s.chunk[warp][e] = part;
        }
        __syncwarp();
        const u64 total = sum(mine, &before);
        const u64 place = place_of(u[r], total);
        uint32_t e = 0;
        while (e < eighths && place >= before && place >= before + s.chunk[warp][e]) before += s.chunk[warp][e++];
        if (place >= before && e < eighths) {  // this warp holds the class
            u64 run = before;
            steps_of_warp(e * eighth, min(steps, (e + 1) * eighth), [&](const Pack<float, 4>& p, uint32_t at) {
                u64 w[4];
                const u64 sum = weigh(p, at, w);
                u64 upto = sum;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += y;
                }
                const u64 all = __shfl_sync(0xffffffffu, upto, 31);
                u64 low = run + upto - sum;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (place >= low && place < low + w[i]) {
                        out_classes[r] = (int32_t)(at + i - shift);
                        if (out_probs) out_probs[r] = share_of(w[i], total);
                    }
                    low += w[i];
                }
                run += all;
            });
        }
    }
};

template <class T, bool HELD, int WARPS, int CTAS, int BLOCKS>
__global__ void __launch_bounds__(32 * WARPS, BLOCKS)
    k_sample_row(const T* __restrict__ scores, uint64_t n, uint32_t classes, uint32_t steps, uint64_t stride,
                 const float* __restrict__ u, fbgpu_sample_params params, int32_t* __restrict__ out_classes,
                 float* __restrict__ out_probs) {
    using Sh = RowShared<WARPS, CTAS>;
    extern __shared__ __align__(16) unsigned char memory[];
    RowDraw<T, HELD, WARPS, CTAS> d(*reinterpret_cast<Sh*>(memory), reinterpret_cast<T*>(memory + sizeof(Sh)), steps);
    for (uint64_t r = blockIdx.x / CTAS; r < n; r += gridDim.x / CTAS) {
        d.open(scores + r * stride, classes);
        d.draw(r, params, u, out_classes, out_probs);
    }
    if (CTAS > 1) cooperative_groups::this_cluster().sync();  // no block leaves while another reads its memory
}

struct SampleArgs {
    const void* scores;
    uint64_t n, stride;
    uint32_t classes;
    const float* u;
    fbgpu_sample_params params;
    int32_t* out_classes;
    float* out_probs;
    cudaStream_t stream;
};

template <class T, int KP> void launch_thread(const SampleArgs& a) {
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(1u << 20, (a.n + 127) / 128);
    k_sample_thread<T, KP><<<blocks, 128, 0, a.stream>>>(static_cast<const T*>(a.scores), a.n, a.classes, a.stride,
                                                         a.u, a.params, a.out_classes, a.out_probs);
}

template <class T, int L, int E> void launch_lanes(const SampleArgs& a) {
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(1u << 20, (a.n + 128 / L - 1) / (128 / L));
    k_sample_lanes<T, L, E><<<blocks, 128, 0, a.stream>>>(static_cast<const T*>(a.scores), a.n, a.classes, a.stride,
                                                          a.u, a.params, a.out_classes, a.out_probs);
}

// Steps of a warp for rows of `classes` classes, wherever they begin.
template <class T> uint32_t steps_of(uint32_t classes, uint32_t warps) {
    return ceil_div(classes + 16 / sizeof(T) - 1, warps * 128);
}

// `most`: the classes of the longest row that the variant is launched for.  The
// kernel's shared memory limit is one for all threads of the process, so it is
// always set to what those need: a call that set it to its own size could come
// between another thread's setting and launch.
template <class T, bool HELD, int WARPS, int CTAS, int BLOCKS> void launch_row(const SampleArgs& a, uint32_t most = 0) {
    using Sh = RowShared<WARPS, CTAS>;
    const uint32_t steps = steps_of<T>(a.classes, WARPS * CTAS);
    auto bytes_for = [](uint32_t warp_steps) {
        return sizeof(Sh) + (HELD ? (size_t)WARPS * warp_steps * 128 * sizeof(T) : 0);
    };
    const size_t bytes = bytes_for(steps);
    const auto kernel = k_sample_row<T, HELD, WARPS, CTAS, BLOCKS>;
    if (bytes > 48 << 10)
        FB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)bytes_for(steps_of<T>(most, WARPS * CTAS))));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((uint32_t)std::min<uint64_t>(1u << 18, a.n) * CTAS);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = a.stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = CTAS;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = CTAS > 1 ? 1 : 0;
    FB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(a.scores), a.n, a.classes, steps, a.stride,
                                     a.u, a.params, a.out_classes, a.out_probs));
}

// Which kernel takes a row, by its classes and the rows (us measured, both sides of each choice):
//   up to 16     all pairs in a thread's registers: 10^6 rows of 7 f32 with top_p 27 (a warp a row: 1100)
//   up to 256    one to eight lanes and 32 classes each: 800000 rows of 20 bf16 with top_p 100 (a warp a row:
//                1390); fewer lanes a row, fewer rounds
//   up to 8192   a block, the row in shared memory: 2048 rows of 1000 f16 with top_p 20 (32 lanes of 32
//                classes: 44).  Many short rows take blocks of one or two warps, so that all are resident
//                (8000 rows of 300 bf16 with top_p 39 with one warp, 47 with two, 63 with four; 2048 of 1000
//                25, 21, 25), few rows four, for their latency (512 rows of 1000: 23, 17, 13)
//   longer       a batch: a block, up to 64 KB of row in shared memory (1000 rows of 20000 bf16 with top_p 117; read
//                again from the L2 for each step 133), longer ones read again: 256 rows of 131071 bf16 with top_k
//                50 31 (a cluster each, in shared memory: 310).  1024 threads where every SM has at most one
//                row (148 rows with top_p: 103 against 148) or where rows differ in work and the longest one counts
//                (256 rows with limits of their own: 144 against 162), else two rows an SM (256 rows with top_p: 186
//                against 202);
//                up to 8 rows of more than 32768: eight SMs share each, 1 row of 128000 f32 with top_k 50 15; 8 rows
//                of 131071 bf16 with top_p 47 (a block each: 101), 16 rows with top_k 50 29 (23), as not all of 16
//                such clusters run at a time; 18 rows of 20000 with top_p 43 (27).
template <class T> void launch_sample(const SampleArgs& a) {
    count_launch();
    const uint32_t k = a.classes;
    const auto& p = a.params;
    const bool unequal = p.temperatures || p.top_ks || p.top_ps || p.min_ps;
    if (k <= 2) launch_thread<T, 2>(a);
    else if (k <= 3) launch_thread<T, 3>(a);
    else if (k <= 4) launch_thread<T, 4>(a);
    else if (k <= 5) launch_thread<T, 5>(a);
    else if (k <= 6) launch_thread<T, 6>(a);
    else if (k <= 7) launch_thread<T, 7>(a);
    else if (k <= 8) launch_thread<T, 8>(a);
    else if (k <= 10) launch_thread<T, 10>(a);
    else if (k <= 12) launch_thread<T, 12>(a);
    else if (k <= 16) launch_thread<T, 16>(a);
    else if (k <= 24) launch_lanes<T, 1, 24>(a);
    else if (k <= 32) launch_lanes<T, 1, 32>(a);
    else if (k <= 64) launch_lanes<T, 2, 32>(a);
    else if (k <= 128) launch_lanes<T, 4, 32>(a);
    else if (k <= 256) launch_lanes<T, 8, 32>(a);
    else if (k <= 512 && a.n >= 2048) launch_row<T, true, 1, 1, 20>(a, 512);
    else if (k <= 2048 && a.n >= 1024) launch_row<T, true, 2, 1, 16>(a, 2048);
    else if (k <= 2048) launch_row<T, true, 4, 1, 8>(a, 2048);
    else if (k <= 8192) launch_row<T, true, 8, 1, 4>(a, 8192);
    else if (k > 32768 && a.n <= 8 && k <= 262144) launch_row<T, true, 16, 8, 1>(a, 262144);  // up to 136 KB a block
    else if (k > 32768 && a.n <= 8) launch_row<T, false, 16, 8, 1>(a);
    else if (a.n <= 148) launch_row<T, false, 32, 1, 1>(a);
    else if (k * sizeof(T) <= 65536) launch_row<T, true, 16, 1, 2>(a, 65536 / sizeof(T));
    else if (a.n <= 296 && unequal) launch_row<T, false, 32, 1, 1>(a);
    else launch_row<T, false, 16, 1, 2>(a);
}

}  // namespace
}  // namespace fbg

extern "C" fbgpu_status fbgpu_sample(const void* scores, int32_t type, uint64_t n, uint32_t classes, uint64_t stride,
                                     const float* u, const fbgpu_sample_params* params, int32_t* out_classes,
                                     float* out_probs, void* stream) {
    using namespace fbg;
    return ops_guarded([&] {
        const uint32_t size = type_size(type);
        if (classes < 2 || classes > 1u << 20) throw InputError("classes must be in 2..1048576");
        if (!params) throw InputError("params must not be null");
        check_matrix("scores", scores, n, classes, stride, size, false);
        check_matrix("u", u, n, 1, 1, 4, false);
        check_matrix("out_classes", out_classes, n, 1, 1, 4, true);
        if (out_probs) check_matrix("out_probs", out_probs, n, 1, 1, 4, true);
        if (!params->temperatures && !(params->temperature >= 0.0f && params->temperature < INFINITY))
            throw InputError("temperature must be finite and not negative");
        if (!params->top_ks && params->top_k < 0) throw InputError("top_k must not be negative");
        if (!params->top_ps && !(params->top_p >= 0.0f && params->top_p <= 1.0f))
            throw InputError("top_p must be in [0, 1]");
        if (!params->min_ps && !(params->min_p >= 0.0f && params->min_p <= 1.0f))
            throw InputError("min_p must be in [0, 1]");
        const void* per_row[] = {params->temperatures, params->top_ks, params->top_ps, params->min_ps, u};
        const uint64_t column = extent(n, 1, 1, 4);
        for (const void* out : {(const void*)out_classes, (const void*)out_probs}) {
            if (!out) continue;
            bool bad = overlap(out, column, scores, extent(n, classes, stride, size));
            for (const void* p : per_row) bad = bad || (p && overlap(out, column, p, column));
            if (bad) throw InputError("the outputs must not overlap the inputs");
        }
        for (const void* p : per_row)
            if (p && (uintptr_t)p % 4) throw InputError("the limits must be aligned to their elements");
        if (out_probs && overlap(out_classes, column, out_probs, column))
            throw InputError("out_classes and out_probs must not overlap");
        cudaStream_t s = check_stream(stream);
        if (!n) return;
        const SampleArgs a{scores, n, stride, classes, u, *params, out_classes, out_probs, s};
        with_type(type, [&](auto e) { launch_sample<decltype(e)>(a); });
        FB_CUDA_CHECK(cudaGetLastError());
    });
}
