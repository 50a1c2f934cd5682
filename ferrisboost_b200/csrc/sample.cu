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

#include "ops.h"

namespace fbg {
namespace {

constexpr int kThreads = 256;
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

struct Shared {
    u64 weight[256];
    uint32_t count[256];
    u64 part[kThreads / 32];
    u64 value;
    uint32_t digit;
    float top;
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int d = 16; d; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Exclusive sum over the block; total to every thread.
__device__ __forceinline__ u64 scan(Shared& s, u64 v, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) s.part[warp] = x;
    __syncthreads();
    u64 before = 0;
    total = 0;
    for (int w = 0; w < kThreads / 32; w++) {
        if (w < warp) before += s.part[w];
        total += s.part[w];
    }
    return before + x - v;
}

// A block per row, reading the row once per step.
template <class T>
__global__ void __launch_bounds__(kThreads) k_sample(const T* __restrict__ scores, uint64_t n, uint32_t classes,
                                                     uint64_t stride, const float* __restrict__ u,
                                                     fbgpu_sample_params params, int32_t* __restrict__ out_classes,
                                                     float* __restrict__ out_probs) {
    __shared__ Shared s;
    for (uint64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T* row = scores + r * stride;
        const Limits l = limits_of(params, r, classes);
        auto get = [&](uint32_t c) { return score(to_f32(row[c])); };
        // the maximum
        float top = -INFINITY;
        for (uint32_t c = threadIdx.x; c < classes; c += kThreads) top = fmaxf(top, get(c));
        for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = __float_as_uint(top);
        __syncthreads();
        for (int w = 0; w < kThreads / 32; w++) top = fmaxf(top, __uint_as_float((uint32_t)s.part[w]));
        if (top == -INFINITY) {
            if (threadIdx.x == 0) {
                out_classes[r] = -1;
                if (out_probs) out_probs[r] = 0.0f;
            }
            continue;
        }
        // kept: key > cut, or key == cut and one of the first `ties` of them
        uint32_t cut = 0, ties = 0xffffffffu;
        // Finds the key at which the running count (or weight) of the falling
        // order reaches `goal`; `above` gets what lies above that key.
        auto select = [&](bool by_weight, u64 goal, u64& above) -> bool {
            uint32_t prefix = 0;
            above = 0;
            const uint32_t floor = cut;
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                for (int i = threadIdx.x; i < 256; i += kThreads) s.weight[i] = 0, s.count[i] = 0;
                __syncthreads();
                for (uint32_t c = threadIdx.x; c < classes; c += kThreads) {
                    const float x = get(c);
                    const uint32_t key = key_of(x);
                    if (key < floor || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
                    if (by_weight)
                        atomicAdd(&s.weight[(key >> shift) & 255], weight_of(exp_of(x, top, l.inv_t)));
                    else
                        atomicAdd(&s.count[(key >> shift) & 255], 1u);
                }
                __syncthreads();
                if (threadIdx.x == 0) {
                    u64 run = above;
                    int d = 255;
                    for (; d >= 0; d--) {
                        const u64 v = by_weight ? s.weight[d] : s.count[d];
                        if (run + v >= goal) break;
                        run += v;
                    }
                    s.digit = d < 0 ? 256 : d;
                    s.value = run;
                }
                __syncthreads();
                if (s.digit == 256) return false;  // the whole row stays below the goal
                above = s.value;
                prefix = prefix << 8 | s.digit;
            }
            cut = prefix;
            return true;
        };
        u64 above;
        if (l.greedy) {
            cut = key_of(top);
            ties = 1;
        } else {
            if (l.top_k < classes) {
                select(false, l.top_k, above);
                ties = l.top_k - (uint32_t)above;
            }
            if (l.use_p) {
                u64 sum = 0, same = 0;
                for (uint32_t c = threadIdx.x; c < classes; c += kThreads) {
                    const float x = get(c);
                    const uint32_t key = key_of(x);
                    if (key > cut) sum += weight_of(exp_of(x, top, l.inv_t));
                    if (key == cut) same++;
                }
                u64 total, found;
                scan(s, sum, total);
                scan(s, same, found);
                total += min(found, (u64)ties) * weight_of(exp_of(score_of(cut), top, l.inv_t));
                u64 goal = (u64)__double2ll_rz(ceil(__dmul_rn(l.top_p, __ull2double_rn(total))));
                if (goal < 1) goal = 1;
                if (select(true, goal, above)) {
                    const u64 w = weight_of(exp_of(score_of(cut), top, l.inv_t));
                    ties = (uint32_t)((goal - above + w - 1) / w);  // w > 0: it carried the sum to the goal
                }
            }
        }
        auto kept = [&](float x, uint32_t tie) -> u64 {
            const uint32_t key = key_of(x);
            if (key < cut || (key == cut && tie >= ties)) return 0;
            const float e = exp_of(x, top, l.inv_t);
            return e < l.min_p ? 0 : weight_of(e);
        };
        // the total, then the first class at which the running sum passes u * total
        u64 total = 0, seen = 0, sum;
        for (uint32_t base = 0; base < classes; base += kThreads) {
            const uint32_t c = base + threadIdx.x;
            const float x = c < classes ? get(c) : -INFINITY;
            const u64 tie = c < classes && key_of(x) == cut;
            const u64 before = scan(s, tie, sum) + seen;
            seen += sum;
            scan(s, c < classes ? kept(x, (uint32_t)before) : 0, sum);
            total += sum;
        }
        const float ur = u[r];
        u64 place = ur > 0.0f ? (u64)__double2ll_rz(__dmul_rn((double)ur, __ull2double_rn(total))) : 0;
        if (place >= total) place = total - 1;
        u64 run = 0;
        seen = 0;
        for (uint32_t base = 0; base < classes; base += kThreads) {
            const uint32_t c = base + threadIdx.x;
            const float x = c < classes ? get(c) : -INFINITY;
            const u64 tie = c < classes && key_of(x) == cut;
            const u64 before = scan(s, tie, sum) + seen;
            seen += sum;
            const u64 w = c < classes ? kept(x, (uint32_t)before) : 0;
            const u64 at = scan(s, w, sum) + run;
            if (place >= at && place < at + w) {
                out_classes[r] = (int32_t)c;
                if (out_probs) out_probs[r] = __double2float_rn(__ddiv_rn(__ull2double_rn(w), __ull2double_rn(total)));
            }
            run += sum;
            if (run > place) break;
        }
    }
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
        const uint32_t blocks = (uint32_t)std::min<uint64_t>(1u << 20, n);
        with_type(type, [&](auto e) {
            using T = decltype(e);
            count_launch();
            k_sample<T><<<blocks, kThreads, 0, s>>>(static_cast<const T*>(scores), n, classes, stride, u, *params,
                                                    out_classes, out_probs);
        });
        FB_CUDA_CHECK(cudaGetLastError());
    });
}
