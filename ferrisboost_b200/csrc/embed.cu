// Table lookup by token, summed over a row's tokens, and its gradient by
// sorted tokens (fbgpu_embed, fbgpu_embed_grad).
//
//   out[r]   = scale * sum_j table[token(r, j)]
//   d_table[v] = scale * sum of grad[r] over the places (r, j) with token v
//
// The gradient sorts the places by token with a stable radix sort (least
// significant digit first) whose payload is the place's row, so that a token's
// rows are consecutive and in ascending order; each table row is then one
// sum over a run of the sorted list, with no atomics.
#include "ops.h"

namespace fbg {
namespace {

template <class Tok> struct Tokens {
    const Tok* p;
    uint64_t row, col;
    // The token of place (r, j) if it is in [0, vocab), else `vocab`.
    __device__ __forceinline__ uint64_t at(uint64_t r, uint64_t j, uint64_t vocab) const {
        const uint64_t t = (uint64_t)(int64_t)p[r * row + j * col];  // a negative token is above every vocab
        return t < vocab ? t : vocab;
    }
};

// ------------------------------------------------------------------- lookup
// A group of `lanes` threads (a power of two, at most a warp) makes one output
// row; lane l holds the elements [V * l, V * l + V) of each slice of V * lanes.
template <class T, class Tok, int V>
__global__ void __launch_bounds__(256) k_embed(const T* __restrict__ table, uint64_t vocab, uint32_t dim,
                                               uint64_t table_stride, Tokens<Tok> tokens, uint64_t n, uint32_t per_row,
                                               float scale, T* __restrict__ out, uint64_t out_stride, uint32_t lanes) {
    const uint32_t lane = threadIdx.x & (lanes - 1);
    const uint64_t groups = (uint64_t)gridDim.x * (blockDim.x / lanes);
    for (uint64_t r = (uint64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes; r < n; r += groups) {
        for (uint32_t c = lane * V; c < dim; c += lanes * V) {
            float acc[V] = {};
            for (uint32_t j = 0; j < per_row; j++) {
                const uint64_t t = tokens.at(r, j, vocab);
                if (t >= vocab) continue;
                const Pack<T, V> e = *reinterpret_cast<const Pack<T, V>*>(table + t * table_stride + c);
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] += to_f32(e.v[i]);
            }
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; i++) o.v[i] = from_f32<T>(acc[i] * scale);
            *reinterpret_cast<Pack<T, V>*>(out + r * out_stride + c) = o;
        }
    }
}

// -------------------------------------------------------------- radix sort
constexpr int kSortThreads = 256, kSortItems = 16, kTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32, kMaxBits = 9, kMaxBins = 1 << kMaxBits;

struct SortPass {
    const uint32_t *keys, *rows;  // null in the first pass, which reads the tokens
    uint32_t *keys_out, *rows_out;
    uint32_t* hist;   // [bin][tile]: counts, then offsets within the bin
    uint32_t* total;  // [bin]
    uint32_t count, tiles, shift, bins;
};

template <class Tok, bool FIRST>
__device__ __forceinline__ void load_place(const SortPass& a, const Tokens<Tok>& tokens, uint32_t per_row,
                                           uint64_t vocab, uint32_t i, uint32_t& key, uint32_t& row) {
    if (FIRST) {
        row = i / per_row;
        key = (uint32_t)tokens.at(row, i - row * per_row, vocab);
    } else {
        key = a.keys[i];
        row = a.rows[i];
    }
}

// Counts each bin of the pass's digit in a tile of 4096 places.
template <class Tok, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_sort_count(SortPass a, Tokens<Tok> tokens, uint32_t per_row,
                                                             uint64_t vocab) {
    __shared__ uint32_t h[kMaxBins];
    for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) h[b] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile;
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t i = base + k * kSortThreads + threadIdx.x;
        if (i >= a.count) break;
        uint32_t key, row;
        load_place<Tok, FIRST>(a, tokens, per_row, vocab, i, key, row);
        atomicAdd(&h[(key >> a.shift) & (a.bins - 1)], 1u);
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) a.hist[(uint64_t)b * a.tiles + blockIdx.x] = h[b];
}

// Exclusive sum over the block's threads; `sum` gets the total.
template <int THREADS> __device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* part, uint32_t& sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = x;
    __syncthreads();
    uint32_t before = 0;
    sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += part[w];
        sum += part[w];
    }
    return before + x - v;
}

// One block per bin: the bin's counts over the tiles become offsets.
__global__ void __launch_bounds__(kSortThreads) k_sort_scan(SortPass a) {
    __shared__ uint32_t part[kSortWarps];
    uint32_t* h = a.hist + (uint64_t)blockIdx.x * a.tiles;
    uint32_t run = 0;
    for (uint32_t base = 0; base < a.tiles; base += kSortThreads) {
        const uint32_t t = base + threadIdx.x;
        uint32_t sum, v = t < a.tiles ? h[t] : 0;
        const uint32_t off = block_scan<kSortThreads>(v, part, sum);
        if (t < a.tiles) h[t] = run + off;
        run += sum;
    }
    if (threadIdx.x == 0) a.total[blockIdx.x] = run;
}

// Moves a tile's places to their bins, in order.  Each warp ranks its 512
// places 32 at a time by matching digits; the tile is then put in order in
// shared memory, so that a bin's places are written next to one another.
template <class Tok, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) k_sort_scatter(SortPass a, Tokens<Tok> tokens, uint32_t per_row,
                                                               uint64_t vocab) {
    __shared__ uint16_t seen[kSortWarps][kMaxBins];  // at most kTile
    __shared__ uint32_t first[kMaxBins], dest[kMaxBins];
    __shared__ uint32_t part[kSortWarps];
    __shared__ uint32_t skey[kTile], srow[kTile];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads) (&seen[0][0])[b] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile, here = min((uint32_t)kTile, a.count - base);
    uint32_t key[kSortItems], row[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t p = warp * (kTile / kSortWarps) + k * 32 + lane;
        const bool in = p < here;
        key[k] = row[k] = 0;
        if (in) load_place<Tok, FIRST>(a, tokens, per_row, vocab, base + p, key[k], row[k]);
        const uint32_t d = in ? (key[k] >> a.shift) & (a.bins - 1) : kMaxBins;
        const uint32_t peers = __match_any_sync(0xffffffffu, d);
        uint32_t old = 0;
        const int lead = __ffs(peers) - 1;
        if (in && lane == lead) {
            old = seen[warp][d];
            seen[warp][d] = (uint16_t)(old + __popc(peers));
        }
        __syncwarp();
        rank[k] = __shfl_sync(0xffffffffu, old, lead) + __popc(peers & ((1u << lane) - 1));
    }
    __syncthreads();
    // where each bin starts in the tile, and where each bin of the tile starts in the output
    uint32_t run = 0, out_run = 0;
    for (uint32_t b0 = 0; b0 < a.bins; b0 += kSortThreads) {
        const uint32_t b = b0 + threadIdx.x;
        uint32_t mine = 0, all = 0;
        if (b < a.bins) {
            for (int w = 0; w < kSortWarps; w++) {
                const uint32_t c = seen[w][b];
                seen[w][b] = (uint16_t)mine;
                mine += c;
            }
            all = a.total[b];
        }
        uint32_t sum, out_sum;
        const uint32_t f = block_scan<kSortThreads>(mine, part, sum);
        const uint32_t o = block_scan<kSortThreads>(all, part, out_sum);
        if (b < a.bins) {
            first[b] = run + f;
            dest[b] = out_run + o + a.hist[(uint64_t)b * a.tiles + blockIdx.x];
        }
        run += sum;
        out_run += out_sum;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t p = warp * (kTile / kSortWarps) + k * 32 + lane;
        if (p < here) {
            const uint32_t d = (key[k] >> a.shift) & (a.bins - 1);
            const uint32_t q = first[d] + seen[warp][d] + rank[k];
            skey[q] = key[k];
            srow[q] = row[k];
        }
    }
    __syncthreads();
    for (uint32_t q = threadIdx.x; q < here; q += kSortThreads) {
        const uint32_t kq = skey[q], d = (kq >> a.shift) & (a.bins - 1);
        const uint32_t at = dest[d] + (q - first[d]);
        a.keys_out[at] = kq;
        a.rows_out[at] = srow[q];
    }
}

// ------------------------------------------------------------- run sums
// Where each token's run of the sorted places begins and ends (both zero from
// before for a token with none).
__global__ void k_runs(const uint32_t* __restrict__ keys, uint32_t count, uint32_t vocab, uint32_t* __restrict__ begin,
                       uint32_t* __restrict__ end) {
    const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= count) return;
    const uint32_t k = keys[i];
    if (k >= vocab) return;
    if (i == 0 || keys[i - 1] != k) begin[k] = i;
    if (i + 1 == count || keys[i + 1] != k) end[k] = i + 1;
}

// A group of lanes makes one row of the gradient.
template <class T, int V>
__global__ void __launch_bounds__(256) k_run_sums(const T* __restrict__ grad, uint32_t dim, uint64_t grad_stride,
                                                  const uint32_t* __restrict__ rows, const uint32_t* __restrict__ begin,
                                                  const uint32_t* __restrict__ end, uint32_t vocab, float scale,
                                                  T* __restrict__ out, uint64_t out_stride, uint32_t lanes) {
    const uint32_t lane = threadIdx.x & (lanes - 1);
    const uint64_t v = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) / lanes;
    if (v >= vocab) return;
    const uint32_t b = begin[v], e = end[v];
    for (uint32_t c = lane * V; c < dim; c += lanes * V) {
        float acc[V] = {};
        for (uint32_t i = b; i < e; i++) {
            const Pack<T, V> g = *reinterpret_cast<const Pack<T, V>*>(grad + rows[i] * grad_stride + c);
#pragma unroll
            for (int k = 0; k < V; k++) acc[k] += to_f32(g.v[k]);
        }
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < V; k++) o.v[k] = from_f32<T>(acc[k] * scale);
        *reinterpret_cast<Pack<T, V>*>(out + v * out_stride + c) = o;
    }
}

// ------------------------------------------------------------------- host
// Elements per access: the widest power of two up to 16 bytes that divides
// the row length and that every address and stride is a multiple of.
uint32_t vector_width(uint32_t size, uint64_t dim, const void* a, uint64_t a_stride, const void* b, uint64_t b_stride) {
    uint32_t v = 16 / size;
    while (v > 1 && (dim % v || a_stride % v || b_stride % v || (uintptr_t)a % (v * size) || (uintptr_t)b % (v * size)))
        v /= 2;
    return v;
}
template <class T, class F> void with_width(uint32_t v, F&& f) {
    switch (v) {
        case 1: f(std::integral_constant<int, 1>{}); break;
        case 2: f(std::integral_constant<int, 2>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        default: f(std::integral_constant<int, 16 / sizeof(T)>{}); break;
    }
}
uint32_t lanes_for(uint64_t chunks) {
    uint32_t lanes = 1;
    while (lanes < 32 && lanes < chunks) lanes *= 2;
    return lanes;
}

void check_tokens(const void* tokens, uint64_t n, uint64_t per_row, uint64_t row, uint64_t col, uint32_t size) {
    if (!n || !per_row) return;
    if (!tokens) throw InputError("tokens must be a device pointer");
    if ((uintptr_t)tokens % size) throw InputError("tokens must be aligned to their elements");
    if ((n > 1 && row && n - 1 > kMostElements / row) || (per_row > 1 && col && per_row - 1 > kMostElements / col))
        throw InputError("tokens is too large");
}
uint64_t token_extent(uint64_t n, uint64_t per_row, uint64_t row, uint64_t col, uint32_t size) {
    return n && per_row ? ((n - 1) * row + (per_row - 1) * col + 1) * size : 0;
}

// Parts of the gradient's workspace, each 256-byte aligned.
struct GradSpace {
    uint64_t keys[2], rows[2], hist, total, begin, end, bytes;
    uint32_t count, tiles, bits, passes;
    GradSpace(uint64_t n, uint64_t per_row, uint64_t vocab) {
        count = (uint32_t)(n * per_row);
        tiles = ceil_div(count, kTile);
        bits = 1;
        while (bits < 32 && (vocab >> bits)) bits++;  // keys go up to `vocab`, the missing token
        passes = (bits + kMaxBits - 1) / kMaxBits;
        bits = (bits + passes - 1) / passes;
        uint64_t at = 0;
        auto take = [&](uint64_t b) {
            const uint64_t p = at;
            at += (b + 255) / 256 * 256;
            return p;
        };
        for (int i = 0; i < 2; i++) keys[i] = take(4ull * count), rows[i] = take(4ull * count);
        hist = take(4ull * (1ull << bits) * tiles);
        total = take(4ull << bits);
        begin = take(8ull * vocab);
        end = begin + 4 * vocab;
        bytes = at;
    }
};
constexpr uint64_t kMostPlaces = 0x7ffffffeull;

bool grad_sizes_fit(uint64_t n, uint64_t per_row, uint64_t vocab) {
    return vocab <= kMostPlaces && (per_row == 0 || n <= kMostPlaces / per_row);
}

}  // namespace
}  // namespace fbg

extern "C" fbgpu_status fbgpu_embed(const void* table, int32_t type, uint64_t vocab, uint32_t dim,
                                    uint64_t table_stride, const void* tokens, int32_t token_type, uint64_t n,
                                    uint32_t per_row, uint64_t token_row, uint64_t token_col, float scale, void* out,
                                    uint64_t out_stride, void* stream) {
    using namespace fbg;
    return ops_guarded([&] {
        const uint32_t size = type_size(type);
        check_matrix("table", table, vocab, dim, table_stride, size, false);
        check_matrix("out", out, n, dim, out_stride, size, true);
        with_token(token_type, [&](auto tok) {
            using Tok = decltype(tok);
            check_tokens(tokens, n, per_row, token_row, token_col, sizeof(Tok));
            const uint64_t on = extent(n, dim, out_stride, size);
            if (overlap(out, on, table, extent(vocab, dim, table_stride, size)) ||
                overlap(out, on, tokens, token_extent(n, per_row, token_row, token_col, sizeof(Tok))))
                throw InputError("out must not overlap the table or the tokens");
            cudaStream_t s = check_stream(stream);
            if (!n || !dim) return;
            const uint32_t v = vector_width(size, dim, table, table_stride, out, out_stride);
            const uint32_t lanes = lanes_for((dim + v - 1) / v);
            const uint32_t blocks = (uint32_t)std::min<uint64_t>(1u << 20, (n * lanes + 255) / 256);
            with_type(type, [&](auto e) {
                using T = decltype(e);
                with_width<T>(v, [&](auto w) {
                    if constexpr (decltype(w)::value <= 16 / sizeof(T)) {
                        count_launch();
                        k_embed<T, Tok, decltype(w)::value><<<blocks, 256, 0, s>>>(
                            static_cast<const T*>(table), vocab, dim, table_stride,
                            Tokens<Tok>{static_cast<const Tok*>(tokens), token_row, token_col}, n, per_row, scale,
                            static_cast<T*>(out), out_stride, lanes);
                    }
                });
            });
            FB_CUDA_CHECK(cudaGetLastError());
        });
    });
}

extern "C" uint64_t fbgpu_embed_grad_workspace(uint64_t n, uint32_t per_row, uint64_t vocab, uint32_t dim) {
    (void)dim;
    return fbg::grad_sizes_fit(n, per_row, vocab) ? fbg::GradSpace(n, per_row, vocab).bytes : 0;
}

extern "C" fbgpu_status fbgpu_embed_grad(const void* grad, int32_t type, uint64_t n, uint32_t per_row, uint32_t dim,
                                         uint64_t grad_stride, const void* tokens, int32_t token_type,
                                         uint64_t token_row, uint64_t token_col, uint64_t vocab, float scale,
                                         void* out, uint64_t out_stride, void* workspace, uint64_t workspace_bytes,
                                         void* stream) {
    using namespace fbg;
    return ops_guarded([&] {
        const uint32_t size = type_size(type);
        check_matrix("grad", grad, n, dim, grad_stride, size, false);
        check_matrix("out", out, vocab, dim, out_stride, size, true);
        if (!grad_sizes_fit(n, per_row, vocab))
            throw InputError("fbgpu_embed_grad takes at most 2147483646 places and as many tokens");
        with_token(token_type, [&](auto tok) {
            using Tok = decltype(tok);
            check_tokens(tokens, n, per_row, token_row, token_col, sizeof(Tok));
            const GradSpace ws(n, per_row, vocab);
            if (workspace_bytes < ws.bytes || (!workspace && ws.bytes))
                throw InputError("the workspace is smaller than fbgpu_embed_grad_workspace says");
            if ((uintptr_t)workspace % 256) throw InputError("the workspace must be 256-byte aligned");
            const uint64_t on = extent(vocab, dim, out_stride, size);
            const uint64_t gn = extent(n, dim, grad_stride, size);
            const uint64_t tn = token_extent(n, per_row, token_row, token_col, sizeof(Tok));
            if (overlap(out, on, grad, gn) || overlap(out, on, tokens, tn) ||
                overlap(workspace, ws.bytes, out, on) || overlap(workspace, ws.bytes, grad, gn) ||
                overlap(workspace, ws.bytes, tokens, tn))
                throw InputError("out and the workspace must not overlap the gradient, the tokens or each other");
            cudaStream_t s = check_stream(stream);
            if (!vocab || !dim) return;
            char* w = static_cast<char*>(workspace);
            auto at = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(w + off); };
            FB_CUDA_CHECK(cudaMemsetAsync(w + ws.begin, 0, 8 * vocab, s));
            const Tokens<Tok> tk{static_cast<const Tok*>(tokens), token_row, token_col};
            for (uint32_t p = 0; ws.count && p < ws.passes; p++) {
                SortPass a{};
                a.keys = p ? at(ws.keys[(p - 1) & 1]) : nullptr;
                a.rows = p ? at(ws.rows[(p - 1) & 1]) : nullptr;
                a.keys_out = at(ws.keys[p & 1]);
                a.rows_out = at(ws.rows[p & 1]);
                a.hist = at(ws.hist);
                a.total = at(ws.total);
                a.count = ws.count;
                a.tiles = ws.tiles;
                a.shift = p * ws.bits;
                a.bins = 1u << ws.bits;
                for (int k = 0; k < 3; k++) count_launch();
                if (p == 0) {
                    k_sort_count<Tok, true><<<ws.tiles, kSortThreads, 0, s>>>(a, tk, per_row, vocab);
                    k_sort_scan<<<a.bins, kSortThreads, 0, s>>>(a);
                    k_sort_scatter<Tok, true><<<ws.tiles, kSortThreads, 0, s>>>(a, tk, per_row, vocab);
                } else {
                    k_sort_count<Tok, false><<<ws.tiles, kSortThreads, 0, s>>>(a, tk, per_row, vocab);
                    k_sort_scan<<<a.bins, kSortThreads, 0, s>>>(a);
                    k_sort_scatter<Tok, false><<<ws.tiles, kSortThreads, 0, s>>>(a, tk, per_row, vocab);
                }
            }
            const int last = (ws.passes - 1) & 1;
            if (ws.count) {
                count_launch();
                k_runs<<<ceil_div(ws.count, 256), 256, 0, s>>>(at(ws.keys[last]), ws.count, (uint32_t)vocab,
                                                               at(ws.begin), at(ws.end));
            }
            const uint32_t v = vector_width(size, dim, grad, grad_stride, out, out_stride);
            const uint32_t lanes = lanes_for((dim + v - 1) / v);
            with_type(type, [&](auto e) {
                using T = decltype(e);
                with_width<T>(v, [&](auto wd) {
                    if constexpr (decltype(wd)::value <= 16 / sizeof(T)) {
                        count_launch();
                        k_run_sums<T, decltype(wd)::value><<<ceil_div(vocab * lanes, 256), 256, 0, s>>>(
                            static_cast<const T*>(grad), dim, grad_stride, at(ws.rows[last]), at(ws.begin), at(ws.end),
                            (uint32_t)vocab, scale, static_cast<T*>(out), out_stride, lanes);
                    }
                });
            });
            FB_CUDA_CHECK(cudaGetLastError());
        });
    });
}
