// What the device-pointer operators share (embed.cu, dropout.cu, sample.cu):
// element types, argument checks and the C boundary.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ctx.h"

namespace fbg {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements that move as one load or store.
template <class T, int N> struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// SplitMix64's finalizer (Steele, Lea and Flood 2014), as in row sampling.
__device__ __host__ __forceinline__ uint64_t mix64(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// What is read in place of something that is not there.
static __device__ __align__(16) const uint4 g_zero{0, 0, 0, 0};

// i / d for i < 2^31: with l = ceil(log2 d), floor(i * (floor(2^(31+l) / d) + 1) / 2^(31+l)), as the excess of the
// multiplier over 2^(31+l) / d, at most 1, times i stays below 2^31 and so below a unit of the quotient.
struct Divisor {
    uint32_t d, mul, shift;
    Divisor(uint32_t d_ = 1) : d(d_), mul(0), shift(0) {
        if (d <= 1) return;
        uint32_t l = 0;
        while ((1ull << l) < d) l++;
        mul = (uint32_t)((1ull << (31 + l)) / d + 1);
        shift = l - 1;
    }
    __device__ __forceinline__ uint32_t div(uint32_t i) const { return d <= 1 ? i : __umulhi(i, mul) >> shift; }
};

// The 16 bytes at `shift` bytes into lo:hi, shift a multiple of 2 below 16.  All
// vectors of a row have the same shift, so its words are a branch.
__device__ __forceinline__ uint4 window(const uint4& lo, const uint4& hi, uint32_t shift) {
    const uint32_t bits = (shift & 2) * 8;
    auto part = [&](uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e) {
        return make_uint4(__funnelshift_r(a, b, bits), __funnelshift_r(b, c, bits), __funnelshift_r(c, d, bits),
                          __funnelshift_r(d, e, bits));
    };
    switch (shift >> 2) {
        case 0: return part(lo.x, lo.y, lo.z, lo.w, hi.x);
        case 1: return part(lo.y, lo.z, lo.w, hi.x, hi.y);
        case 2: return part(lo.z, lo.w, hi.x, hi.y, hi.z);
        default: return part(lo.w, hi.x, hi.y, hi.z, hi.w);
    }
}

struct Clear {
    char* p;          // rows of `bytes` bytes, `stride` bytes apart
    uint64_t rows, bytes, stride;
};

// Rows that follow one another are one.
inline Clear clear_of(void* p, uint64_t rows, uint64_t bytes, uint64_t stride) {
    if (stride == bytes) return Clear{static_cast<char*>(p), 1, rows * bytes, 0};
    return Clear{static_cast<char*>(p), rows, bytes, stride};
}
void launch_clear(void* p, uint64_t rows, uint64_t bytes, uint64_t stride, cudaStream_t s);  // embed.cu

// Block `b` of `blocks` clears its share.
__device__ __forceinline__ void clear_rows(const Clear& z, uint64_t b, uint64_t blocks) {
    const uint64_t per = 16ull * blockDim.x;  // bytes of a block's step
    const uint64_t steps = (z.bytes + 15 + per - 1) / per;
    for (uint64_t i = b; i < z.rows * steps; i += blocks) {
        const uint64_t r = z.rows == 1 ? 0 : i / steps;
        char* row = z.p + r * z.stride;
        char* end = row + z.bytes;
        char* at = reinterpret_cast<char*>((uintptr_t)row & ~(uintptr_t)15) + (i - r * steps) * per + 16 * threadIdx.x;
        if (at >= row && at + 16 <= end) {
            *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
        } else {  // elements are two or four bytes
            for (int k = 0; k < 16; k += 2)
                if (at + k >= row && at + k < end) *reinterpret_cast<uint16_t*>(at + k) = 0;
        }
    }
}

// Runs f with a value of the element type `type` names.
template <class F> void with_type(int32_t type, F&& f) {
    switch (type) {
        case FBGPU_F32: f(float{}); break;
        case FBGPU_F16: f(__half{}); break;
        case FBGPU_BF16: f(__nv_bfloat16{}); break;
        default: throw InputError("the element type must be FBGPU_F32, FBGPU_F16 or FBGPU_BF16");
    }
}
template <class F> void with_token(int32_t type, F&& f) {
    switch (type) {
        case FBGPU_I32: f(int32_t{}); break;
        case FBGPU_I64: f(int64_t{}); break;
        default: throw InputError("the token type must be FBGPU_I32 or FBGPU_I64");
    }
}
inline uint32_t type_size(int32_t type) {
    uint32_t size = 0;
    with_type(type, [&](auto v) { size = sizeof(v); });
    return size;
}

// The largest array extent the operators take: byte offsets stay below 2^62.
constexpr uint64_t kMostElements = 1ull << 58;

// A matrix of n rows of dim elements of `size` bytes: not null, aligned, and
// addressable.  Rows may repeat (stride below dim) only in inputs.
inline void check_matrix(const char* what, const void* p, uint64_t n, uint64_t dim, uint64_t stride, uint32_t size,
                         bool written) {
    if (n == 0 || dim == 0) return;
    if (!p) throw InputError(std::string(what) + " must be a device pointer");
    if ((uintptr_t)p % size) throw InputError(std::string(what) + " must be aligned to its elements");
    if (written && n > 1 && stride < dim) throw InputError(std::string(what) + ": the rows overlap");
    if (dim > kMostElements || stride > kMostElements || (n > 1 && stride && n - 1 > kMostElements / stride))
        throw InputError(std::string(what) + " is too large");
}

inline uint64_t extent(uint64_t n, uint64_t dim, uint64_t stride, uint32_t size) {
    return n == 0 || dim == 0 ? 0 : ((n - 1) * stride + dim) * size;
}
inline bool overlap(const void* a, uint64_t an, const void* b, uint64_t bn) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return an && bn && x < y + bn && y < x + an;
}

// The stream, which must be one of the current device.  A capturing stream may
// not be asked (the query ends the capture); its launches are checked when the
// graph is made.
inline cudaStream_t check_stream(void* stream) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (s != nullptr && s != cudaStreamPerThread && s != cudaStreamLegacy) {
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        FB_CUDA_CHECK(cudaStreamIsCapturing(s, &capture));
        if (capture != cudaStreamCaptureStatusNone) return s;
        int device = 0, sdev = -1;
        FB_CUDA_CHECK(cudaGetDevice(&device));
        FB_CUDA_CHECK(cudaStreamGetDevice(s, &sdev));
        if (sdev != device) throw InputError("the stream belongs to another device than the current one");
    }
    return s;
}

// The C boundary: no exception leaves it, and no error of the runtime that it
// reports: the runtime keeps a failed call's error for the thread's next check,
// which would report it for work that ran.
template <class F> fbgpu_status ops_guarded(F&& f) {
    try {
        f();
        return FBGPU_OK;
    } catch (const InputError& ex) {
        noalloc_set_error(ex.what());
        return FBGPU_EINPUT;
    } catch (const CudaError& ex) {
        cudaGetLastError();
        noalloc_set_error(ex.what());
        return FBGPU_ECUDA;
    } catch (const std::exception& ex) {
        noalloc_set_error(ex.what());
        return FBGPU_EINTERNAL;
    } catch (...) {
        noalloc_set_error("unknown error");
        return FBGPU_EINTERNAL;
    }
}

}  // namespace fbg
