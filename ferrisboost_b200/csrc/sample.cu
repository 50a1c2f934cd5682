// Drawing a class from a row of scores (fbgpu_sample).
//
// A class of score x weighs w = floor(2^40 exp((x - max) / T)).  Every limit
// keeps a beginning of the order (score falling, equal scores by class), so
// what is kept is "every class above a threshold score, and the first `ties`
// classes of that score"; the threshold is found by counting and summing
// weights per digit of an ordered key, not by sorting.  Sums of weights are
// 64-bit whole numbers: 2^20 classes of at most 2^40 fit, and no order of
// additions changes them.
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
    l.inv_t = l.greedy ? 0.0f : __fdiv_rn(1.0f, fminf(t, FLT_MAX));  // never 0: no 0 * infinity in exp_of
    l.top_k = k < 1 || (uint32_t)k > classes ? classes : (uint32_t)k;
    l.use_p = tp < 1.0f;
    l.top_p = tp > 0.0f ? (double)tp : 0.0;
    l.min_p = mp > 1.0f ? 1.0f : mp;
    return l;
}

// -0 as +0 (they are equal scores) and NaN as -infinity.
__device__ __forceinline__ float score(float x) { return x == x ? __fadd_rn(x, 0.0f) : -INFINITY; }
// Unsigned order of the scores.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ float exp_of(float x, float top, float inv_t) {
    if (x == top) return 1.0f;
    return x == -INFINITY || top == INFINITY ? 0.0f : expf(__fmul_rn(__fsub_rn(x, top), inv_t));
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

// ------------------------------------------------------- a thread per row
// Up to KP classes in registers.  A class's place in the order and the weight
// before it come from comparing each pair once.
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
            x[i] = i < classes ? score(to_f32(row[i])) : -INFINITY;
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
            u64 w[KP];
            uint32_t keep = 0;
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const float e = exp_of(x[i], top, l.inv_t);
                w[i] = weight_of(e);
                if (!(e < l.min_p)) keep |= 1u << i;
            }
            if (l.top_k < classes || l.use_p) {
                u64 sum = 0;
                uint32_t first = 0;  // the top_k first
#pragma unroll
                for (int i = 0; i < KP; i++) {
                    uint32_t rank = 0;
#pragma unroll
                    for (int j = 0; j < KP; j++)
                        if (j != i) rank += j < i ? x[j] >= x[i] : x[j] > x[i];
                    if (rank < l.top_k) first |= 1u << i, sum += w[i];
                }
                keep &= first;
                if (l.use_p) {
                    const u64 goal = goal_of(l.top_p, sum);
#pragma unroll
                    for (int i = 0; i < KP; i++) {
                        u64 before = 0;
#pragma unroll
                        for (int j = 0; j < KP; j++)
                            if (j != i && (j < i ? x[j] >= x[i] : x[j] > x[i])) before += w[j];
                        if (before >= goal) keep &= ~(1u << i);
                    }
                }
            }
            u64 total = 0;
#pragma unroll
            for (int i = 0; i < KP; i++) total += w[i] = keep >> i & 1 ? w[i] : 0;
            const u64 place = place_of(u[r], total);
            u64 run = total, won = 0;
#pragma unroll
            for (int i = KP - 1; i >= 0; i--) {
                run -= w[i];
                if (run <= place && place < run + w[i]) drawn = i, won = w[i];
            }
            share = share_of(won, total);
        }
        out_classes[r] = drawn;
        if (out_probs) out_probs[r] = share;
    }
}

// ------------------------------------------- a warp, block or cluster per row
// WARPS warps of CTAS blocks (one cluster) hold a row.  Warp after warp takes a
// contiguous part of it; within the part, lane after lane takes VEC elements a
// step.  NV steps are kept in registers; NV = 0 reads the row again for every
// step.  Vectors are aligned in memory, not in the row: a row that starts off a
// 16-byte boundary has `shift` places before its first class, which are masked.
template <int WARPS, int CTAS> struct RowShared {
    static constexpr int kBins = WARPS == 1 ? 256 : 1024;
    static constexpr int kList = WARPS == 1 ? 64 : 128;
    uint32_t low[kBins], high[kBins];     // a bin's count, or its weight as two words
    u64 part[2][WARPS];                   // warps' partial sums; two sets, used in turn
    uint32_t found[2];                    // members of the chosen bin
    uint32_t key[2][kList], all_key[kList];
    u64 weight[2][kList], all_weight[kList];
    u64 scan[WARPS];
    uint32_t bin;
    u64 before, pick_above;
    uint32_t pick_key, pick_same;
};

template <class T, int VEC, int NV, int WARPS, int CTAS> struct RowDraw {
    using Sh = RowShared<WARPS, CTAS>;
    static constexpr int kSets = NV ? NV : 1;
    static constexpr int kBins = Sh::kBins;
    static constexpr int kThreadsPerRow = WARPS * 32;

    Sh& s;
    const T* row;
    uint32_t classes, shift, first, steps;  // the part's first place (with shift), and its steps
    int lane, warp, tid, cta, parity = 0;
    Pack<T, VEC> held[kSets];

    __device__ __forceinline__ RowDraw(Sh& sh) : s(sh) {
        lane = threadIdx.x & 31;
        warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
        tid = WARPS == 1 ? lane : threadIdx.x;
        cta = CTAS == 1 ? 0 : (int)cooperative_groups::this_cluster().block_rank();
    }

    __device__ __forceinline__ void sync_block() {
        if (WARPS == 1) __syncwarp();
        else __syncthreads();
    }
    __device__ __forceinline__ void sync_row() {
        if (CTAS == 1) sync_block();
        else cooperative_groups::this_cluster().sync();
    }
    // Another block's shared memory.
    template <class V> __device__ __forceinline__ const V* at(const V* p, int c) {
        if (CTAS == 1) return p;
        return cooperative_groups::this_cluster().map_shared_rank(p, c);
    }

    __device__ __forceinline__ Pack<T, VEC> read(uint32_t v) {
        const uint32_t place = first + (v * 32 + lane) * VEC;
        Pack<T, VEC> p;
        if (VEC > 1 && place >= shift && place + VEC <= shift + classes) {
            p = *reinterpret_cast<const Pack<T, VEC>*>(row + (place - shift));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                p.v[i] = place + i >= shift && place + i < shift + classes ? row[place + i - shift]
                                                                           : from_f32<T>(-INFINITY);
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) p.v[i] = from_f32<T>(score(to_f32(p.v[i])));
        return p;
    }
    __device__ __forceinline__ void open(const T* row_, uint32_t classes_) {
        row = row_;
        classes = classes_;
        shift = VEC > 1 ? (uint32_t)(((uintptr_t)row % (VEC * sizeof(T))) / sizeof(T)) : 0;
        const uint32_t vectors = (classes + shift + VEC - 1) / VEC;
        steps = NV ? NV : (vectors + 32 * WARPS * CTAS - 1) / (32 * WARPS * CTAS);
        first = (cta * WARPS + warp) * steps * 32 * VEC;
        if constexpr (NV > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) held[v] = read(v);
        }
    }
    // f(score, step, index within the vector) for each of the lane's places
    template <class F> __device__ __forceinline__ void each(F&& f) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) {
#pragma unroll
                for (int i = 0; i < VEC; i++) f(to_f32(held[v].v[i]));
            }
        } else {
            for (uint32_t v = 0; v < steps; v++) {
                const Pack<T, VEC> p = read(v);
#pragma unroll
                for (int i = 0; i < VEC; i++) f(to_f32(p.v[i]));
            }
        }
    }
    // f(scores of a step, the place of the first) step by step, in order
    template <class F> __device__ __forceinline__ void each_step(F&& f) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) f(held[v], first + (v * 32 + lane) * VEC);
        } else {
            for (uint32_t v = 0; v < steps; v++) f(read(v), first + (v * 32 + lane) * VEC);
        }
    }

    // A reduction over the row's threads; op is commutative.  `before` gets the
    // result over the warps in front of this one (for sums).
    template <class Op> __device__ __forceinline__ u64 reduce(u64 v, u64 zero, Op&& op, u64* before = nullptr) {
#pragma unroll
        for (int d = 16; d; d /= 2) v = op(v, (u64)__shfl_xor_sync(0xffffffffu, v, d));
        if (before) *before = zero;
        if (WARPS == 1) return v;
        if (lane == 0) s.part[parity][warp] = v;
        sync_row();
        u64 all = zero;
        for (int c = 0; c < CTAS; c++) {
            const u64* p = at(s.part[parity], c);
            // lane w takes warp w's value
            u64 x = lane < WARPS ? p[lane] : zero;
            if (before) {
                u64 y = c < cta || (c == cta && lane < warp) ? x : zero;
#pragma unroll
                for (int d = 16; d; d /= 2) y = op(y, (u64)__shfl_xor_sync(0xffffffffu, y, d));
                *before = op(*before, y);
            }
            all = op(all, x);
        }
#pragma unroll
        for (int d = 16; d; d /= 2) all = op(all, (u64)__shfl_xor_sync(0xffffffffu, all, d));
        parity ^= 1;
        return all;
    }
    __device__ __forceinline__ u64 sum(u64 v, u64* before = nullptr) {
        return reduce(v, 0, [](u64 a, u64 b) { return a + b; }, before);
    }

    __device__ __forceinline__ uint32_t bin_of(float x, float top, float per) {
        return min((uint32_t)(kBins - 1), __float2uint_rz(__fmul_rn(__fsub_rn(top, x), per)));
    }

    __device__ void draw(uint64_t r, const fbgpu_sample_params& params, const float* u, int32_t* out_classes,
                         float* out_probs) {
        const Limits l = limits_of(params, r, classes);
        float top = -INFINITY;
        each([&](float x) { top = fmaxf(top, x); });
        {
            const uint32_t k = (uint32_t)reduce(key_of(top), 0, [](u64 a, u64 b) { return a > b ? a : b; });
            top = score_of(k);
        }
        if (top == -INFINITY) {
            if (tid == 0 && cta == 0) {
                out_classes[r] = -1;
                if (out_probs) out_probs[r] = 0.0f;
            }
            return;
        }
        // kept: key > cut, or key == cut and one of the first `ties` of the `same` classes of that key
        uint32_t cut = 0, ties = 0xffffffffu, same = 0;
        if (l.greedy) {
            cut = key_of(top);
            ties = 1;
            same = 0xffffffffu;
        } else {
            // Weights vanish 27.73 T below the maximum: bins over that span, falling, the last for the rest.
            const float per = __fmul_rn(kBins / 27.75f, l.inv_t);
            // first by count for top_k, then by weight for top_p
            for (int by_weight = 0; by_weight < 2; by_weight++) {
                if (by_weight ? !l.use_p : l.top_k >= classes) continue;
                for (int i = tid; i < kBins; i += kThreadsPerRow) s.low[i] = s.high[i] = 0;
                if (tid == 0) s.found[by_weight] = 0;
                sync_block();
                each([&](float x) {
                    if (x == -INFINITY || key_of(x) < cut) return;
                    const uint32_t b = bin_of(x, top, per);
                    if (by_weight) {
                        const u64 w = weight_of(exp_of(x, top, l.inv_t));
                        if (w == 0) return;
                        const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.low[b], lo);
                        const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < lo);
                        if (hi) atomicAdd(&s.high[b], hi);
                    } else {
                        atomicAdd(&s.low[b], 1u);
                    }
                });
                sync_row();
                // each thread: the running sum before its bins (every block of a cluster does the same work)
                constexpr int kPer = kBins / kThreadsPerRow;
                u64 v[kPer], mine = 0;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    v[i] = 0;
                    for (int c = 0; c < CTAS; c++)
                        v[i] += (u64)at(s.high, c)[tid * kPer + i] << 32 | at(s.low, c)[tid * kPer + i];
                    mine += v[i];
                }
                u64 upto = mine;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += y;
                }
                u64 total = __shfl_sync(0xffffffffu, upto, 31);
                if (WARPS > 1) {
                    if (lane == 31) s.scan[warp] = upto;
                    if (tid == 0) s.bin = kBins;
                    sync_block();
                    u64 x = lane < WARPS ? s.scan[lane] : 0, y = lane < warp ? x : 0;
#pragma unroll
                    for (int d = 16; d; d /= 2) {
                        x += __shfl_xor_sync(0xffffffffu, x, d);
                        y += __shfl_xor_sync(0xffffffffu, y, d);
                    }
                    total = x;
                    upto += y;
                } else if (tid == 0) {
                    s.bin = kBins;
                }
                u64 goal = l.top_k;
                if (by_weight) {
                    if (ties < same) total -= (same - ties) * weight_of(exp_of(score_of(cut), top, l.inv_t));
                    goal = goal_of(l.top_p, total);
                }
                sync_block();
                u64 run = upto - mine;
#pragma unroll
                for (int i = 0; i < kPer; i++) {
                    if (run < goal && goal <= run + v[i]) {
                        s.bin = tid * kPer + i;
                        s.before = run;
                    }
                    run += v[i];
                }
                sync_block();
                const uint32_t bin = s.bin;
                if (bin == kBins) {  // the whole row stays below the goal
                    if (CTAS > 1) sync_row();  // the other blocks may still read these bins
                    continue;
                }
                goal -= s.before;
                // the chosen bin's members
                auto member = [&](float x) {
                    return x > -INFINITY && key_of(x) >= cut && bin_of(x, top, per) == bin;
                };
                each([&](float x) {
                    if (!member(x)) return;
                    const uint32_t q = atomicAdd(&s.found[by_weight], 1u);
                    if (q < Sh::kList) {
                        s.key[by_weight][q] = key_of(x);
                        s.weight[by_weight][q] = by_weight ? weight_of(exp_of(x, top, l.inv_t)) : 1;
                    }
                });
                sync_row();
                uint32_t members = 0;
                for (int c = 0; c < CTAS; c++) members += *at(&s.found[by_weight], c);
                u64 above = 0;
                if (members <= Sh::kList) {
                    const uint32_t* keys = s.key[by_weight];
                    const u64* weights = s.weight[by_weight];
                    if (CTAS > 1) {
                        uint32_t base = 0;
                        for (int c = 0; c < CTAS; c++) {
                            const uint32_t m = *at(&s.found[by_weight], c);
                            for (uint32_t i = tid; i < m; i += kThreadsPerRow) {
                                s.all_key[base + i] = at(s.key[by_weight], c)[i];
                                s.all_weight[base + i] = at(s.weight[by_weight], c)[i];
                            }
                            base += m;
                        }
                        keys = s.all_key;
                        weights = s.all_weight;
                        sync_block();
                    }
                    for (uint32_t i = tid; i < members; i += kThreadsPerRow) {
                        const uint32_t key = keys[i];
                        u64 before = 0;
                        uint32_t equal = 0;
                        for (uint32_t j = 0; j < members; j++) {
                            if (keys[j] > key) before += weights[j];
                            if (keys[j] == key) equal++;
                        }
                        if (before < goal && goal <= before + equal * weights[i]) {  // all of that key agree
                            s.pick_key = key;
                            s.pick_same = equal;
                            s.pick_above = before;
                        }
                    }
                    sync_block();
                    cut = s.pick_key;
                    same = s.pick_same;
                    above = s.pick_above;
                } else {
                    // Many members: halve the range of their keys.  All above `hi` have the weight `above`,
                    // below the goal; with those from `lo` on it is reached.
                    uint32_t lo = 0xffffffffu, hi = 0;
                    each([&](float x) {
                        if (member(x)) lo = min(lo, key_of(x)), hi = max(hi, key_of(x));
                    });
                    auto least = [](u64 a, u64 b) { return a < b ? a : b; };
                    auto most = [](u64 a, u64 b) { return a > b ? a : b; };
                    lo = (uint32_t)reduce(lo, 0xffffffffu, least);
                    hi = (uint32_t)reduce(hi, 0, most);
                    while (lo < hi) {
                        const uint32_t mid = lo + (hi - lo + 1) / 2;
                        u64 part = 0;
                        uint32_t under = 0, over = 0xffffffffu;  // the nearest keys on either side of mid
                        each([&](float x) {
                            const uint32_t key = key_of(x);
                            if (key < lo || key > hi || !member(x)) return;
                            if (key >= mid) {
                                part += by_weight ? weight_of(exp_of(x, top, l.inv_t)) : 1;
                                over = min(over, key);
                            } else {
                                under = max(under, key);
                            }
                        });
                        part = sum(part);
                        if (above + part >= goal) {
                            lo = (uint32_t)reduce(over, 0xffffffffu, least);
                        } else {
                            above += part;
                            hi = (uint32_t)reduce(under, 0, most);
                        }
                    }
                    cut = lo;
                    u64 equal = 0;
                    each([&](float x) { equal += key_of(x) == cut; });
                    same = (uint32_t)sum(equal);
                }
                const u64 each_w = by_weight ? weight_of(exp_of(score_of(cut), top, l.inv_t)) : 1;
                ties = (uint32_t)((goal - above + each_w - 1) / each_w);
            }
        }
        // How many of the key `cut` come before this warp's part, where not all of them are kept.
        const bool some = ties < same;
        u64 ties_before = 0;
        if (some) {
            u64 equal = 0;
            each([&](float x) { equal += key_of(x) == cut; });
            sum(equal, &ties_before);
        }
        // The kept weight of each lane's step, in order: f(place, weights, their sum).
        auto walk = [&](auto&& f) {
            uint32_t seen = (uint32_t)ties_before;
            each_step([&](const Pack<T, VEC>& p, uint32_t place) {
                uint32_t rank = 0;
                if (some) {
                    uint32_t mine = 0;
#pragma unroll
                    for (int i = 0; i < VEC; i++) mine += key_of(to_f32(p.v[i])) == cut;
                    rank = mine;
#pragma unroll
                    for (int d = 1; d < 32; d *= 2) {
                        const uint32_t y = __shfl_up_sync(0xffffffffu, rank, d);
                        if (lane >= d) rank += y;
                    }
                    const uint32_t all = __shfl_sync(0xffffffffu, rank, 31);
                    rank += seen - mine;
                    seen += all;
                }
                u64 w[VEC], sum = 0;
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float x = to_f32(p.v[i]);
                    const uint32_t key = key_of(x);
                    w[i] = 0;
                    if (key > cut || (key == cut && (!some || rank < ties))) {
                        const float e = exp_of(x, top, l.inv_t);
                        if (!(e < l.min_p)) w[i] = weight_of(e);
                    }
                    rank += key == cut;
                    sum += w[i];
                }
                f(place, w, sum);
            });
        };
        u64 mine = 0, before = 0;
        walk([&](uint32_t, u64*, u64 w) { mine += w; });
        u64 part = mine;
#pragma unroll
        for (int d = 16; d; d /= 2) part += __shfl_xor_sync(0xffffffffu, part, d);
        const u64 total = sum(mine, &before);
        const u64 place = place_of(u[r], total);
        if (place >= before && place < before + part) {  // this warp holds the class
            u64 run = before;
            walk([&](uint32_t at, u64* w, u64 sum) {
                u64 upto = sum;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += y;
                }
                const u64 all = __shfl_sync(0xffffffffu, upto, 31);
                u64 low = run + upto - sum;
#pragma unroll
                for (int i = 0; i < VEC; i++) {
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

constexpr int kRowsPerBlock = 4;  // of one warp each

template <class T, int VEC, int NV, int WARPS, int CTAS>
__global__ void __launch_bounds__(WARPS == 1 ? 32 * kRowsPerBlock : 32 * WARPS)
    k_sample_row(const T* __restrict__ scores, uint64_t n, uint32_t classes, uint64_t stride,
                 const float* __restrict__ u, fbgpu_sample_params params, int32_t* __restrict__ out_classes,
                 float* __restrict__ out_probs) {
    constexpr int kRows = WARPS == 1 ? kRowsPerBlock : 1;
    __shared__ RowShared<WARPS, CTAS> shared[kRows];
    RowDraw<T, VEC, NV, WARPS, CTAS> d(shared[WARPS == 1 ? threadIdx.x / 32 : 0]);
    const uint64_t start = (uint64_t)(blockIdx.x / CTAS) * kRows + (WARPS == 1 ? threadIdx.x / 32 : 0);
    for (uint64_t r = start; r < n; r += (uint64_t)(gridDim.x / CTAS) * kRows) {
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

template <class T, int VEC, int NV, int WARPS, int CTAS> void launch_row(const SampleArgs& a) {
    constexpr int kRows = WARPS == 1 ? kRowsPerBlock : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((uint32_t)std::min<uint64_t>(1u << 18, (a.n + kRows - 1) / kRows) * CTAS);
    cfg.blockDim = dim3(32 * WARPS * kRows);
    cfg.stream = a.stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = CTAS;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = CTAS > 1 ? 1 : 0;
    FB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k_sample_row<T, VEC, NV, WARPS, CTAS>, static_cast<const T*>(a.scores), a.n,
                                     a.classes, a.stride, a.u, a.params, a.out_classes, a.out_probs));
}

template <class T> void launch_sample(const SampleArgs& a) {
    constexpr int V = 16 / sizeof(T);  // elements of a vector
    count_launch();
    const uint32_t k = a.classes, held = k + V - 1;  // places with the largest shift
    if (k <= 4) launch_thread<T, 4>(a);
    else if (k <= 8) launch_thread<T, 8>(a);
    else if (k <= 16) launch_thread<T, 16>(a);
    else if (k <= 64) launch_row<T, 1, 2, 1, 1>(a);
    else if (k <= 256) launch_row<T, 1, 8, 1, 1>(a);
    else if (k <= 1024) launch_row<T, 1, 32, 1, 1>(a);
    else if (held <= 8192) launch_row<T, V, 32 / V, 8, 1>(a);
    else if (held <= 20480) launch_row<T, V, 40 / V, 16, 1>(a);
    else if (held <= 163840) launch_row<T, V, 40 / V, 16, 8>(a);
    else launch_row<T, V, 0, 16, 8>(a);
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
