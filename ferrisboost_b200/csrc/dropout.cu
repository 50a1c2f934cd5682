// Dropout from a counter-based generator (fbgpu_dropout): the mask follows
// from the seed and the element's number, so it is never stored and the same
// call makes the backward pass.
#include <cmath>

#include "ops.h"

namespace fbg {
namespace {

struct DropArgs {
    uint64_t n, dim, x_stride, out_stride, key, offset, threshold;  // kept: 32 bits >= threshold (2^32: none)
    float scale;
};

// A thread per element.
template <class T> __global__ void __launch_bounds__(256) k_dropout(const T* x, T* out, DropArgs a) {
    const uint64_t count = a.n * a.dim;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (uint64_t)gridDim.x * 256) {
        const uint64_t r = i / a.dim, c = i - r * a.dim, e = a.offset + i;
        const uint64_t word = mix64(a.key + ((e >> 1) + 1) * 0x9E3779B97F4A7C15ull);
        const uint32_t bits = (uint32_t)(e & 1 ? word >> 32 : word);
        const float v = to_f32(x[r * a.x_stride + c]) * a.scale;
        out[r * a.out_stride + c] = from_f32<T>(bits >= a.threshold ? v : 0.0f);
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
        DropArgs a{};
        a.n = n;
        a.dim = dim;
        a.x_stride = x_stride;
        a.out_stride = out_stride;
        a.key = mix64(seed);
        a.offset = offset;
        a.threshold = (uint64_t)std::ceil(p * 4294967296.0);
        a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
        const uint32_t blocks = (uint32_t)std::min<uint64_t>(1u << 20, (n * dim + 255) / 256);
        with_type(type, [&](auto e) {
            using T = decltype(e);
            count_launch();
            k_dropout<T><<<blocks, 256, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(out), a);
        });
        FB_CUDA_CHECK(cudaGetLastError());
    });
}
