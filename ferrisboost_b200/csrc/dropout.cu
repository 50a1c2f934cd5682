// Dropout from a counter-based generator (fbgpu_dropout): the mask follows
// from the seed and the element's number, so it is never stored and the same
// call makes the backward pass.
#include <cmath>

#include "ops.h"

namespace fbg {
namespace {

constexpr int kThreads = 256, kAhead = 2, kRounds = 4;  // units in flight, and how often, of a thread
constexpr uint64_t kGamma = 0x9E3779B97F4A7C15ull;

struct DropArgs {
    uint64_t n, x_stride, out_stride, key;
    uint64_t offset, numbers;  // element (r, c) has the number offset + r * numbers + c
    int32_t dim;
    uint32_t threshold;        // kept: 32 bits >= threshold
    float scale;
    uint32_t lanes_log;        // a group of lanes takes up to kAhead * kRounds units a lane of one row
    uint32_t rounds;
    Divisor groups;            // of a row
    uint64_t spans;            // blocks' shares of the groups
    bool aligned;              // x and out are at the same distance from a 16-byte boundary in every row
};

// One element's 32 bits.
__device__ __forceinline__ uint32_t bits_of(const DropArgs& a, uint64_t e) {
    const uint64_t word = mix64(a.key + ((e >> 1) + 1) * kGamma);
    return (uint32_t)(e & 1 ? word >> 32 : word);
}

// Two elements, kept or zero.
__device__ __forceinline__ float kept(uint32_t bits, const DropArgs& a, float v) {
    return bits >= a.threshold ? v * a.scale : 0.0f;
}
__device__ __forceinline__ void drop_pair(float* p, uint32_t b0, uint32_t b1, const DropArgs& a) {
    p[0] = kept(b0, a, p[0]);
    p[1] = kept(b1, a, p[1]);
}
__device__ __forceinline__ void drop_pair(__half* p, uint32_t b0, uint32_t b1, const DropArgs& a) {
    __half2* q = reinterpret_cast<__half2*>(p);
    const float2 v = __half22float2(*q);
    *q = __floats2half2_rn(kept(b0, a, v.x), kept(b1, a, v.y));
}
__device__ __forceinline__ void drop_pair(__nv_bfloat16* p, uint32_t b0, uint32_t b1, const DropArgs& a) {
    __nv_bfloat162* q = reinterpret_cast<__nv_bfloat162*>(p);
    const float2 v = __bfloat1622float2(*q);
    *q = __floats2bfloat162_rn(kept(b0, a, v.x), kept(b1, a, v.y));
}

// A unit is the part of a row that lies in one 16-byte vector of the output: the
// stores are aligned vectors whatever the strides, and the loads are the one or
// two aligned vectors of x that hold the unit.  Only a row's first and last unit
// can be partial; they are moved element by element, as are those where the
// numbers wrap. 65536 x 2048 f32: 178 us, 6.0 TB/s,
// memory bound.  bf16: 113 us, 4.8 TB/s, and 137 us for rows of 1999 off the
// boundaries: bound by integer issue (the 64 bits of two elements are 22
// operations, choosing and rounding them nine).  A thread takes up to eight units
// of a row, as the row's constants cost as much as half a unit.
template <class T> __global__ void __launch_bounds__(kThreads, 4) k_dropout(const T* x, T* out, DropArgs a) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t per_block = kThreads >> a.lanes_log, lanes = 1u << a.lanes_log;
    const int step = lanes * V;
    const uint64_t stride = (step / 2) * kGamma;  // of the generator, from a unit to the next
    for (uint64_t s = blockIdx.x; s < a.spans; s += gridDim.x) {
        const uint64_t r0 = s * per_block / a.groups.d;
        const uint32_t g = (uint32_t)(s * per_block - r0 * a.groups.d) + (threadIdx.x >> a.lanes_log);
        const uint32_t q = a.groups.div(g);
        const uint64_t row = r0 + q;
        if (row >= a.n) continue;
        T* to = out + row * a.out_stride;
        // the column of the first vector's first element: just before the row for its first group
        int c = ((g - q * a.groups.d) * (kAhead * a.rounds << a.lanes_log) + (threadIdx.x & (lanes - 1))) * V -
                (uint32_t)((uintptr_t)to % 16) / sizeof(T);
        to += c;
        const T* from = x + row * a.x_stride + c;
        const uint64_t e = a.offset + row * a.numbers + c;
        const uint32_t shift = (uint32_t)((uintptr_t)from % 16);
        const char* base = reinterpret_cast<const char*>(from) - shift;
        if (e >= ~(uint64_t)(2 * kAhead * kRounds * 32 * V)) {  // the numbers wrap here
            for (uint32_t k = 0; k < kAhead * a.rounds; k++)
                for (int i = 0; i < V; i++) {
                    const int at = k * step + i;
                    if (c + at >= 0 && c + at < a.dim)
                        to[at] = from_f32<T>(kept(bits_of(a, e + at), a, to_f32(from[at])));
                }
            continue;
        }
        uint64_t state = a.key + ((e >> 1) + 1) * kGamma;
        // ODD: the row's units begin with the high half of a word
        auto units = [&](auto odd, auto aligned) {
            constexpr bool ODD = decltype(odd)::value, ALIGNED = decltype(aligned)::value;
            for (uint32_t round = 0; round < a.rounds && c < a.dim; round++) {
                uint4 lo[kAhead], hi[kAhead];
                bool whole[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    whole[k] = c + k * step >= 0 && c + k * step + V <= a.dim;
                    lo[k] = *(whole[k] ? reinterpret_cast<const uint4*>(base + k * 16 * lanes) : &g_zero);
                }
                if (!ALIGNED) {
                    // the vector with the unit's last element: the first one again where the unit is aligned
#pragma unroll
                    for (int k = 0; k < kAhead; k++)
                        hi[k] = *(whole[k] ? reinterpret_cast<const uint4*>(base + k * 16 * lanes + (shift ? 16 : 0))
                                           : &g_zero);
                }
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    if (c + k * step >= a.dim) break;
                    union {
                        uint4 u;
                        T v[V];
                    } p;
                    p.u = ALIGNED ? lo[k] : window(lo[k], hi[k], shift);
                    if (!whole[k]) {
#pragma unroll
                        for (int i = 0; i < V; i++)
                            if ((uint32_t)(c + k * step + i) < (uint32_t)a.dim) p.v[i] = from[k * step + i];
                    }
                    uint64_t at = state + k * stride;
                    uint32_t half[V + 2];  // of the words from that of the first element on
#pragma unroll
                    for (int i = 0; i < V + ODD; i += 2) {
                        const uint64_t w = mix64(at);
                        half[i] = (uint32_t)w;
                        half[i + 1] = (uint32_t)(w >> 32);
                        at += kGamma;
                    }
#pragma unroll
                    for (int i = 0; i < V; i += 2) drop_pair(p.v + i, half[i + ODD], half[i + 1 + ODD], a);
                    if (whole[k]) {
                        *reinterpret_cast<uint4*>(to + k * step) = p.u;
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i++)
                            if ((uint32_t)(c + k * step + i) < (uint32_t)a.dim) to[k * step + i] = p.v[i];
                    }
                }
                c += kAhead * step;
                from += kAhead * step;
                to += kAhead * step;
                base += kAhead * 16 * lanes;
                state += kAhead * stride;
            }
        };
        if (a.aligned) {
            if (e & 1) units(std::true_type{}, std::true_type{});
            else units(std::false_type{}, std::true_type{});
        } else {
            if (e & 1) units(std::true_type{}, std::false_type{});
            else units(std::false_type{}, std::false_type{});
        }
    }
}

}  // namespace
}  // namespace fbg

extern "C" fbgpu_status fbgpu_dropout(const void* x, int32_t type, uint64_t n, uint64_t dim, uint64_t x_stride,
                                      double p, uint64_t seed, uint64_t offset, void* out, uint64_t out_stride,
                                      void* stream) {
    using namespace fbg;
    return ops_guarded([&] {
        const uint32_t size = type_size(type);
        if (!(p >= 0.0 && p <= 1.0)) throw InputError("p must be in [0, 1]");
        check_matrix("x", x, n, dim, x_stride, size, false);
        check_matrix("out", out, n, dim, out_stride, size, true);
        if (n && dim && dim > kMostElements / n) throw InputError("x is too large");
        if (overlap(x, extent(n, dim, x_stride, size), out, extent(n, dim, out_stride, size)) &&
            !(x == out && (n <= 1 || x_stride == out_stride)))
            throw InputError("out must be x itself or not overlap it");
        cudaStream_t s = check_stream(stream);
        if (!n || !dim) return;
        const uint64_t limit = (uint64_t)std::ceil(p * 4294967296.0);
        if (limit >> 32) {  // nothing is kept
            launch_clear(out, n, dim * size, out_stride * size, s);
            FB_CUDA_CHECK(cudaGetLastError());
            return;
        }
        with_type(type, [&](auto e) {
            using T = decltype(e);
            constexpr uint32_t V = 16 / sizeof(T);
            DropArgs a{};
            a.n = n;
            a.x_stride = x_stride;
            a.out_stride = out_stride;
            a.key = mix64(seed);
            a.numbers = dim;
            a.threshold = (uint32_t)limit;
            a.scale = (float)(1.0 / (1.0 - p));
            constexpr uint64_t kMost = 1ull << 30;  // columns of a launch: they are counted in 32 bits
            for (uint64_t c = 0; c < dim; c += kMost) {
                a.dim = (int32_t)std::min(dim - c, kMost);
                a.offset = offset + c;
                const T* from = static_cast<const T*>(x) + c;
                T* to = static_cast<T*>(out) + c;
                a.aligned = ((uintptr_t)from - (uintptr_t)to) % 16 == 0 &&
                            (n == 1 || (x_stride - out_stride) % V == 0);
                const bool starts = (uintptr_t)to % 16 == 0 && (n == 1 || out_stride % V == 0);
                const uint32_t units = (a.dim + V - 1) / V + !starts;
                a.lanes_log = 0;
                while (a.lanes_log < 5 && (1u << a.lanes_log) * kAhead < units) a.lanes_log++;
                // several rounds save the work that a thread does once, as long as every SM has a few blocks
                a.rounds = std::min<uint32_t>(kRounds, ceil_div(units, kAhead << a.lanes_log));
                while (a.rounds > 1 && n * ceil_div(units, kAhead * a.rounds << a.lanes_log) << a.lanes_log < 148ull * 2048)
                    a.rounds /= 2;
                a.groups = Divisor(ceil_div(units, kAhead * a.rounds << a.lanes_log));
                const uint64_t per_block = kThreads >> a.lanes_log;
                a.spans = n / per_block * a.groups.d + (n % per_block * a.groups.d + per_block - 1) / per_block;
                count_launch();
                k_dropout<T><<<(uint32_t)std::min<uint64_t>(1u << 20, a.spans), kThreads, 0, s>>>(from, to, a);
            }
        });
        FB_CUDA_CHECK(cudaGetLastError());
    });
}
