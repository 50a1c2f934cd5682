// Table lookup by token, summed over a row's tokens, and its gradient by
// sorted tokens (fbgpu_embed, fbgpu_embed_grad).
//
//   out[r]   = scale * sum_j table[token(r, j)]
//   d_table[v] = scale * sum of grad[r] over the places (r, j) with token v
//
// The gradient sorts the places by token with a stable radix sort (least
// significant digit first) whose payload is the place's row, so that a token's
// rows are consecutive and in ascending order, and then sums the sorted list in
// equal parts, whatever the lengths of the tokens' runs.  A run inside a part is
// written at once; what continues into another part is joined from the parts'
// sums in a second pass.  No atomics: the order of every sum follows from the
// tokens, the sizes and the element type, and is the same in every layout.
#include <type_traits>

#include <cooperative_groups.h>

#include "ops.h"

namespace fbg {
namespace {

__global__ void __launch_bounds__(256) k_clear(Clear z) { clear_rows(z, blockIdx.x, gridDim.x); }

constexpr uint32_t kMostSlices = 65535;  // of columns: a grid's y extent

template <class Tok> struct Tokens {
    // Tokens as unsigned numbers of their own width: a negative one is above every `vocab`, which is at most
    // 2^31 (2^63), as no token of the type is larger.
    using U = std::make_unsigned_t<Tok>;
    const Tok* p;
    uint64_t row, col;
    U vocab;
    Tokens(const void* p_, uint64_t row_, uint64_t col_, uint64_t vocab_)
        : p(static_cast<const Tok*>(p_)), row(row_), col(col_),
          vocab((U)std::min<uint64_t>(vocab_, 1ull << (8 * sizeof(Tok) - 1))) {}
    __device__ __forceinline__ U at(uint64_t r, uint64_t j) const { return (U)p[r * row + j * col]; }
};

// A vector of f32 sums.  Pairs are added by one instruction (add.rn.f32x2), each
// half rounded as an addition of its own.
template <int V> struct Sums {
    float v[V];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = 0.0f;
    }
    __device__ __forceinline__ void add(int i, float a, float b) {
        asm("{.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\t"
            "mov.b64 {%0, %1}, x;}"
            : "+f"(v[i]), "+f"(v[i + 1])
            : "f"(a), "f"(b));
    }
    __device__ __forceinline__ void add(const float* o) {
#pragma unroll
        for (int i = 0; i + 1 < V; i += 2) add(i, o[i], o[i + 1]);
        if (V & 1) v[V - 1] += o[V - 1];
    }
    template <class T> __device__ __forceinline__ void add(const Pack<T, V>& p) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = to_f32(p.v[i]);
        add(o);
    }
    template <class T> __device__ __forceinline__ Pack<T, V> scaled(float scale) const {
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) o.v[i] = from_f32<T>(v[i] * scale);
        return o;
    }
};

// ------------------------------------------------------------------- lookup
// One token a row: a copy with a scale, memory bound.  A group of `lanes`
// threads takes four rows at a time, so that four loads are in flight and a
// token is read once a row.  131072 random rows of 1024 bf16 out of 65534: 90 us,
// 4.5 TB/s of what moves at least once (the table passes the L2 twice).
// Columns are counted in 32 bits, and a lane steps past the last one: wider rows
// are looked up kLookupColumns at a time.
constexpr int kLookupThreads = 256, kLookupRows = 4;
constexpr uint32_t kLookupColumns = 1u << 29;

struct LookupArgs {
    uint64_t table_stride, n, out_stride;
    uint32_t dim, lanes_log;
    float scale;
};

template <class T, class Tok, int V>
__global__ void __launch_bounds__(kLookupThreads) k_lookup(LookupArgs a, const T* __restrict__ table,
                                                           Tokens<Tok> tokens, T* __restrict__ out) {
    using P = Pack<T, V>;
    const uint64_t groups = (uint64_t)gridDim.x * (kLookupThreads >> a.lanes_log);
    const uint32_t lane = threadIdx.x & ((1u << a.lanes_log) - 1);
    for (uint64_t r = ((uint64_t)blockIdx.x * kLookupThreads + threadIdx.x) >> a.lanes_log; r < a.n;
         r += kLookupRows * groups) {
        const T* from[kLookupRows];
        T* to[kLookupRows];
#pragma unroll
        for (int k = 0; k < kLookupRows; k++) {
            from[k] = nullptr;
            to[k] = r + k * groups < a.n ? out + (r + k * groups) * a.out_stride : nullptr;
            if (!to[k]) continue;
            const auto t = tokens.at(r + k * groups, 0);
            if (t < tokens.vocab) from[k] = table + t * a.table_stride;
        }
        for (uint32_t c = lane * V; c < a.dim; c += V << a.lanes_log) {
            P e[kLookupRows];
#pragma unroll
            for (int k = 0; k < kLookupRows; k++)
                e[k] = *(from[k] ? reinterpret_cast<const P*>(from[k] + c) : reinterpret_cast<const P*>(&g_zero));
#pragma unroll
            for (int k = 0; k < kLookupRows; k++) {
                Sums<V> sum;
                sum.clear();
                sum.add(e[k]);
                if (to[k]) *reinterpret_cast<P*>(to[k] + c) = sum.template scaled<T>(a.scale);
            }
        }
    }
}

// The same where the rows do not keep 16-byte boundaries: a lane's vectors are
// those of the output, and each is taken from the one or two vectors of the
// table's row that hold it.  The row's ends, partial vectors, go by element.
// Element by element, four bytes a lane leave too little in flight: 100003 rows
// of 201 f32 took 46 us that way, 36 this way (3.7 TB/s).
template <class T, class Tok>
__global__ void __launch_bounds__(kLookupThreads) k_lookup_odd(LookupArgs a, const T* __restrict__ table,
                                                               Tokens<Tok> tokens, T* __restrict__ out) {
    constexpr int V = 16 / sizeof(T), kRows = 2;
    const uint64_t groups = (uint64_t)gridDim.x * (kLookupThreads >> a.lanes_log);
    const uint32_t lane = threadIdx.x & ((1u << a.lanes_log) - 1);
    const int step = V << a.lanes_log, dim = (int)a.dim;
    for (uint64_t r = ((uint64_t)blockIdx.x * kLookupThreads + threadIdx.x) >> a.lanes_log; r < a.n;
         r += kRows * groups) {
        const T* from[kRows];
        T* to[kRows];
        int col[kRows];  // of the lane's first vector: before the row where that begins inside a vector
        uint32_t shift[kRows];
#pragma unroll
        for (int k = 0; k < kRows; k++) {
            const bool in = r + k * groups < a.n;
            const auto t = in ? tokens.at(r + k * groups, 0) : tokens.vocab;
            to[k] = out + (in ? r + k * groups : r) * a.out_stride;
            col[k] = in ? (int)(lane * V) - (int)((uintptr_t)to[k] % 16 / sizeof(T)) : dim;
            from[k] = t < tokens.vocab ? table + t * a.table_stride : nullptr;
            shift[k] = (uint32_t)((uintptr_t)(from[k] + col[k]) % 16);
        }
        // up to the last vector of the row that begins furthest before its first column
        for (int c = 0; (int)(lane * V) - (V - 1) + c < dim; c += step) {
            uint4 lo[kRows], hi[kRows];
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const bool whole = from[k] && col[k] + c >= 0 && col[k] + c + V <= dim;
                const char* p = reinterpret_cast<const char*>(from[k] + col[k] + c) - shift[k];
                lo[k] = *(whole ? reinterpret_cast<const uint4*>(p) : &g_zero);
                // the vector with the last element: the first one again where it holds all
                hi[k] = *(whole ? reinterpret_cast<const uint4*>(p + (shift[k] ? 16 : 0)) : &g_zero);
            }
#pragma unroll
            for (int k = 0; k < kRows; k++) {
                const int first = col[k] + c;
                if (first >= dim) continue;
                union {
                    uint4 u;
                    Pack<T, V> p;
                } e;
                e.u = window(lo[k], hi[k], shift[k]);
                const bool whole = first >= 0 && first + V <= dim;
                if (!whole && from[k]) {
#pragma unroll
                    for (int i = 0; i < V; i++)
                        if ((uint32_t)(first + i) < (uint32_t)dim) e.p.v[i] = from[k][first + i];
                }
                Sums<V> sum;
                sum.clear();
                sum.add(e.p);
                const Pack<T, V> o = sum.template scaled<T>(a.scale);
                if (whole) {
                    *reinterpret_cast<Pack<T, V>*>(to[k] + first) = o;
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++)
                        if ((uint32_t)(first + i) < (uint32_t)dim) to[k][first + i] = o.v[i];
                }
            }
        }
    }
}

// Several tokens a row: a group of `lanes` threads (a power of two, at most a
// warp) sums a slice of V * lanes columns over the tokens of a row, or of one of
// its `parts` parts, eight loads in flight and the next eight tokens behind
// them; a row's parts are neighbours in their block and are joined in order.
// A missing token reads a zero vector instead of branching: loads inside branches
// leave one at a time, which cost three times as much.  16384 rows of 500 tokens
// of 32 bf16: 49 us; the 524 MB of vectors come from the L2 at 10.7 TB/s and keep
// the L1's data path 81 % busy, which bounds it.  One row of 100 tokens of 64 f32:
// 4 us in 16 parts, 31 in one.
constexpr int kBagThreads = 256, kBagAhead = 8;

struct BagArgs {
    uint64_t table_stride, n, out_stride;
    uint32_t dim, per_row, part_len;
    uint32_t lanes_log, parts_log;
    float scale;
};

template <class T, class Tok, int V, bool FLAT>  // FLAT: a row's tokens are next to one another
__global__ void __launch_bounds__(kBagThreads, 4) k_embed(BagArgs a, const T* __restrict__ table, Tokens<Tok> tokens,
                                                          T* __restrict__ out) {
    using P = Pack<T, V>;
    using U = typename Tokens<Tok>::U;
    __shared__ float joined[kBagThreads * V];
    const uint32_t lane = threadIdx.x & ((1u << a.lanes_log) - 1);
    const uint32_t part = threadIdx.x >> a.lanes_log & ((1u << a.parts_log) - 1);
    const uint32_t rows = kBagThreads >> (a.lanes_log + a.parts_log);  // of a block
    const uint32_t c = (((uint32_t)blockIdx.y << a.lanes_log) + lane) * V;
    // `begin` + part_len may pass 2^32, begin + what is left of the row does not
    const uint32_t begin = min(part * a.part_len, a.per_row), end = begin + min(a.part_len, a.per_row - begin);
    for (uint64_t r0 = (uint64_t)blockIdx.x * rows; r0 < a.n; r0 += (uint64_t)gridDim.x * rows) {
        const uint64_t r = r0 + (threadIdx.x >> (a.lanes_log + a.parts_log));
        Sums<V> sum;
        sum.clear();
        if (r < a.n && c < a.dim) {
            const uint64_t col = FLAT ? 1 : tokens.col;
            const Tok* tok = tokens.p + r * tokens.row + begin * col;
            const char* column = reinterpret_cast<const char*>(table + c);
            const uint64_t stride = a.table_stride * sizeof(T);
            const U vocab = tokens.vocab;
            auto row = [&](U t) {
                return t < vocab ? reinterpret_cast<const P*>(column + t * stride) : reinterpret_cast<const P*>(&g_zero);
            };
            const uint32_t whole = (end - begin) / kBagAhead;
            U t[kBagAhead];
            if (whole) {
#pragma unroll
                for (int k = 0; k < kBagAhead; k++) t[k] = (U)tok[k * col];
            }
            for (uint32_t j = 0; j < whole; j++) {
                P e[kBagAhead];
#pragma unroll
                for (int k = 0; k < kBagAhead; k++) e[k] = *row(t[k]);
                tok += kBagAhead * col;
                if (j + 1 < whole) {
#pragma unroll
                    for (int k = 0; k < kBagAhead; k++) t[k] = (U)tok[k * col];
                }
#pragma unroll
                for (int k = 0; k < kBagAhead; k++) sum.add(e[k]);
            }
            const uint32_t rest = end - begin - whole * kBagAhead;
            if (rest) {
#pragma unroll
                for (int k = 0; k < kBagAhead - 1; k++) t[k] = k < rest ? (U)tok[k * col] : vocab;
                P e[kBagAhead];
#pragma unroll
                for (int k = 0; k < kBagAhead - 1; k++) e[k] = *row(t[k]);
#pragma unroll
                for (int k = 0; k < kBagAhead - 1; k++) sum.add(e[k]);
            }
        }
        if (a.parts_log) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; i++) joined[i * kBagThreads + threadIdx.x] = sum.v[i];
            __syncthreads();
            if (part == 0) {
                for (uint32_t p = 1; p < 1u << a.parts_log; p++) {
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; i++) o[i] = joined[i * kBagThreads + threadIdx.x + (p << a.lanes_log)];
                    sum.add(o);
                }
            }
        }
        if (part == 0 && r < a.n && c < a.dim)
            *reinterpret_cast<P*>(out + r * a.out_stride + c) = sum.template scaled<T>(a.scale);
    }
}

// -------------------------------------------------------------- radix sort
// The sorted items are (token, row) pairs of 32 bits each, nine bits a pass.  For
// 8.2 M places a pass takes 16 us to count, 8 to scan and 63 to scatter: the
// ranks within a warp (about 40 of 150 operations an item) and latency bound it,
// at 2.1 TB/s.  Separate arrays of tokens and rows took 89.
constexpr int kSortThreads = 256, kSortItems = 16, kTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32, kMaxBits = 9, kMaxBins = 1 << kMaxBits;

// Where a pass reads its items: from the pass before, or, the first, from the
// tokens, place i being at tokens + i where they are flat.
enum Source { kItems, kFlat, kStrided };
template <class Tok> struct Places {
    Tokens<Tok> tokens;
    Divisor per_row;
    __device__ __forceinline__ uint32_t row(uint32_t i) const { return per_row.div(i); }
    template <Source S> __device__ __forceinline__ uint32_t key(uint32_t i) const {
        typename Tokens<Tok>::U t;
        if (S == kFlat) {
            t = tokens.p[i];
        } else {
            const uint32_t r = row(i);
            t = tokens.at(r, i - r * per_row.d);
        }
        return (uint32_t)min(t, tokens.vocab);
    }
};

struct SortPass {
    const uint2* in;  // not read by the first pass
    uint2* out;
    uint32_t* hist;   // [bin][tile]: counts, then offsets within the bin
    uint32_t* total;  // [bin]
    uint32_t count, tiles, shift, bits;
    __device__ __forceinline__ uint32_t digit(uint32_t key) const { return (key >> shift) & ((1u << bits) - 1); }
};

// Counts each bin of the pass's digit in a tile of 4096 places.
template <class Tok, Source S>
__global__ void __launch_bounds__(kSortThreads) k_sort_count(SortPass a, Places<Tok> places) {
    __shared__ uint32_t h[kMaxBins];
    const uint32_t bins = 1u << a.bits;
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads) h[b] = 0;
    __syncthreads();
    cudaGridDependencySynchronize();
    const uint32_t base = blockIdx.x * kTile + threadIdx.x;
    uint32_t key[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t i = base + k * kSortThreads;
        const uint32_t q = min(i, a.count - 1);
        if constexpr (S == kItems) key[k] = a.in[q].x;
        else key[k] = places.template key<S>(q);
    }
#pragma unroll
    for (int k = 0; k < kSortItems; k++)
        if (base + k * kSortThreads < a.count) atomicAdd(&h[a.digit(key[k])], 1u);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < bins; b += kSortThreads) a.hist[(uint64_t)b * a.tiles + blockIdx.x] = h[b];
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
    constexpr int kPer = 8;
    uint32_t* h = a.hist + (uint64_t)blockIdx.x * a.tiles;
    uint32_t run = 0;
    cudaGridDependencySynchronize();
    for (uint32_t base = 0; base < a.tiles; base += kSortThreads * kPer) {
        uint32_t v[kPer], mine = 0, sum;
#pragma unroll
        for (int k = 0; k < kPer; k++) {
            const uint32_t t = base + threadIdx.x * kPer + k;
            v[k] = t < a.tiles ? h[t] : 0;
            mine += v[k];
        }
        uint32_t off = run + block_scan<kSortThreads>(mine, part, sum);
#pragma unroll
        for (int k = 0; k < kPer; k++) {
            const uint32_t t = base + threadIdx.x * kPer + k;
            if (t < a.tiles) h[t] = off;
            off += v[k];
        }
        run += sum;
    }
    if (threadIdx.x == 0) a.total[blockIdx.x] = run;
}

// The lanes with this lane's digit, among those with `in`: a vote per bit.
__device__ __forceinline__ uint32_t peers_of(uint32_t digit, uint32_t bits, bool in) {
    uint32_t peers = __ballot_sync(0xffffffffu, in);
#pragma unroll
    for (int b = 0; b < kMaxBits; b++) {
        if (b >= bits) break;
        const bool set = digit >> b & 1;
        const uint32_t vote = __ballot_sync(0xffffffffu, set);
        peers &= set ? vote : ~vote;
    }
    return peers;
}
// This lane's number among the warp's items of its digit so far; `seen` counts them per digit.
__device__ __forceinline__ uint32_t rank_in_warp(uint16_t* seen, uint32_t digit, uint32_t bits, bool in) {
    const int lane = threadIdx.x & 31;
    const uint32_t peers = peers_of(digit, bits, in);
    const uint32_t before = __popc(peers & ((1u << lane) - 1));
    const uint32_t old = in ? seen[digit] : 0;
    __syncwarp();
    if (in && before == 0) seen[digit] = (uint16_t)(old + __popc(peers));
    __syncwarp();
    return old + before;
}

// Moves a tile's places to their bins, in order.  Each warp ranks its 512
// places 32 at a time; the tile is then put in order in shared memory, so that
// a bin's places are written next to one another.
template <class Tok, Source S>
__global__ void __launch_bounds__(kSortThreads, 4) k_sort_scatter(SortPass a, Places<Tok> places) {
    __shared__ uint16_t seen[kSortWarps][kMaxBins];  // at most kTile
    __shared__ uint32_t first[kMaxBins], dest[kMaxBins];
    __shared__ uint32_t part[kSortWarps];
    __shared__ uint2 item[kTile];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t bins = 1u << a.bits;
    for (uint32_t b = threadIdx.x; b < kSortWarps * kMaxBins / 2; b += kSortThreads)
        reinterpret_cast<uint32_t*>(seen)[b] = 0;
    cudaGridDependencySynchronize();
    const uint32_t base = blockIdx.x * kTile, here = min((uint32_t)kTile, a.count - base);
    const uint32_t mine0 = warp * (kTile / kSortWarps) + lane;
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t p = mine0 + k * 32;
        const uint32_t q = base + min(p, here - 1);
        if constexpr (S == kItems) key[k] = a.in[q].x;
        else key[k] = places.template key<S>(q);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; k++)
        rank[k] = rank_in_warp(seen[warp], a.digit(key[k]), a.bits, mine0 + k * 32 < here);
    __syncthreads();
    // where each bin starts in the tile, and where each bin of the tile starts in the output
    uint32_t run = 0, out_run = 0;
    for (uint32_t b0 = 0; b0 < bins; b0 += kSortThreads) {
        const uint32_t b = b0 + threadIdx.x;
        uint32_t mine = 0, all = 0;
        if (b < bins) {
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
        if (b < bins) {
            first[b] = run + f;
            dest[b] = out_run + o + a.hist[(uint64_t)b * a.tiles + blockIdx.x];
        }
        run += sum;
        out_run += out_sum;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t p = mine0 + k * 32;
        if (p < here) {
            const uint32_t d = a.digit(key[k]);
            item[first[d] + seen[warp][d] + rank[k]] =
                make_uint2(key[k], S == kItems ? a.in[base + p].y : places.row(base + p));
        }
    }
    __syncthreads();
    for (uint32_t q = threadIdx.x; q < here; q += kSortThreads) {
        const uint2 it = item[q];
        const uint32_t d = a.digit(it.x);
        a.out[dest[d] + (q - first[d])] = it;
    }
}

// A sort of up to 8 * 512 * ITEMS places in one launch: the blocks of one
// cluster hold the places, read one another's digit counts and exchange places
// through the (L2-resident) buffers.  The remaining blocks of the grid clear the
// output.  Latency bound: 10240 places (two passes) 12 us with eight blocks of
// four items a thread, 43 with two blocks of sixteen; 32768 places 26 us beside
// the clearing of 134 MB, which takes as long.
constexpr int kClusterThreads = 512, kClusterCtas = 8;
constexpr uint32_t kClusterPlaces = kClusterCtas * kClusterThreads * 16;

struct ClusterSort {
    uint2* items[2];  // pass p writes set p & 1
    uint32_t count, bits, passes;
};

template <class Tok, Source S, int ITEMS>
__global__ void __launch_bounds__(kClusterThreads) k_sort_cluster(ClusterSort a, Places<Tok> places, Clear z) {
    if (blockIdx.x >= kClusterCtas) {
        clear_rows(z, blockIdx.x - kClusterCtas, gridDim.x - kClusterCtas);
        return;
    }
    constexpr int kWarps = kClusterThreads / 32;
    __shared__ uint16_t seen[kWarps][kMaxBins];
    __shared__ uint32_t total[kMaxBins], dest[kMaxBins], part[kWarps];
    const auto cluster = cooperative_groups::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = cluster.block_rank();
    const uint32_t base = (cta * kWarps + warp) * (32 * ITEMS) + lane, mask = (1u << a.bits) - 1;
    uint2 *in = nullptr, *out = a.items[0];
    for (uint32_t pass = 0; pass < a.passes; pass++) {
        const uint32_t shift = pass * a.bits;
        uint32_t rank[ITEMS];
        uint2 item[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const uint32_t i = base + k * 32;
            const uint32_t q = min(i, a.count - 1);
            item[k] = pass ? __ldcg(in + q) : make_uint2(places.template key<S>(q), places.row(q));
        }
        for (uint32_t b = threadIdx.x; b < kWarps * kMaxBins / 2; b += kClusterThreads)
            reinterpret_cast<uint32_t*>(seen)[b] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; k++)
            rank[k] = rank_in_warp(seen[warp], (item[k].x >> shift) & mask, a.bits, base + k * 32 < a.count);
        __syncthreads();
        const uint32_t d = threadIdx.x;  // a thread per bin
        uint32_t mine = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const uint32_t c = seen[w][d];
            seen[w][d] = (uint16_t)mine;
            mine += c;
        }
        total[d] = mine;
        cluster.sync();
        uint32_t all = 0, before = 0, sum;
#pragma unroll
        for (int c = 0; c < kClusterCtas; c++) {
            const uint32_t t = cluster.map_shared_rank(total, c)[d];
            all += t;
            if (c < cta) before += t;
        }
        dest[d] = before + block_scan<kClusterThreads>(all, part, sum);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            if (base + k * 32 < a.count) {
                const uint32_t dk = (item[k].x >> shift) & mask;
                out[dest[dk] + seen[warp][dk] + rank[k]] = item[k];
            }
        }
        // the items' order is read by every block, and `total` is no longer read
        cluster.sync();
        in = out;
        out = a.items[~pass & 1];
    }
}
static_assert(kMaxBins == kClusterThreads, "a thread per bin");

// ------------------------------------------------------------- run sums
// A group of `lanes` threads sums `chunk` consecutive places of the sorted list
// (a slice of V * lanes columns of their rows), eight loads in flight.  Its first
// run may continue from the group before (its "head") and its last into the
// next (its "tail"); the others are complete and written.  Then each group
// with a tail that began in it adds the heads of the groups that the run
// goes on through.  What leaves the block is kept in `part`: [block][0] the sum
// of the run that came in, [block][1] of the one that goes out.  Equal parts are
// what a skewed column needs: with a group per token, 32768 tokens of 1024 bf16
// of which a tenth are one token took 3.9 ms, this way 20 us (3.4 TB/s).  8.2 M
// places of 32 bf16: 70 us, 7.5 TB/s from the L2.
constexpr int kRunThreads = 256, kAhead = 8;
constexpr uint32_t kMostChunk = 64, kFewBlocks = 148 * 4;

struct RunSums {
    const uint2* items;
    float* part;
    uint32_t count, vocab, dim, lanes, chunk;
    uint64_t grad_stride, out_stride;
    float scale;
};

__device__ __forceinline__ uint32_t key_at(const RunSums& a, uint64_t i) { return i < a.count ? a.items[i].x : a.vocab; }

template <class T, int V> __device__ __forceinline__ void write_row(const RunSums& a, T* out, uint32_t key, uint32_t c,
                                                                    const Sums<V>& sum) {
    *reinterpret_cast<Pack<T, V>*>(out + key * a.out_stride + c) = sum.template scaled<T>(a.scale);
}

// M vectors of a lane, lanes apart; R times the threads and the lanes, for as many groups
template <class T, int V, int M, int R>
__global__ void __launch_bounds__(kRunThreads * R, R == 1 ? 3 : 2) k_run_sums(RunSums a, const T* __restrict__ grad,
                                                                              T* __restrict__ out) {
    constexpr int kThreads = kRunThreads * R;
    __shared__ float heads[kThreads * V * M];     // [vector][group][V * lanes]
    __shared__ uint8_t goes_on[kRunThreads];      // the group is one run, from before its first place to after its last
    const uint32_t lanes = a.lanes * R, groups = kThreads / lanes, group = threadIdx.x / lanes;
    const uint32_t lane = threadIdx.x & (lanes - 1);
    uint32_t c[M];
    bool column[M];
    const T* from[M];
#pragma unroll
    for (int m = 0; m < M; m++) {
        c[m] = ((blockIdx.y * M + m) * lanes + lane) * V;
        column[m] = c[m] < a.dim;
        from[m] = grad + (column[m] ? c[m] : 0);
    }
    const uint64_t begin = ((uint64_t)blockIdx.x * groups + group) * a.chunk;
    cudaGridDependencySynchronize();  // the sorted list, and the cleared output
    uint32_t cur = key_at(a, begin);
    const bool from_before = begin > 0 && cur < a.vocab && key_at(a, begin - 1) == cur;
    bool head = from_before;  // the current run is the one that came in
    Sums<V> acc[M];
#pragma unroll
    for (int m = 0; m < M; m++) acc[m].clear();
    auto keep_head = [&] {
#pragma unroll
        for (int m = 0; m < M; m++) {
#pragma unroll
            for (int i = 0; i < V; i++) heads[(m * kThreads + threadIdx.x) * V + i] = acc[m].v[i];
        }
    };
    auto write = [&](uint32_t key, const Sums<V>* sum) {
#pragma unroll
        for (int m = 0; m < M; m++)
            if (column[m]) write_row<T, V>(a, out, key, c[m], sum[m]);
    };
    // every place of the chunk holds a token: nothing to check
    const bool whole = begin + a.chunk <= a.count && a.items[begin + a.chunk - 1].x < a.vocab;
    auto batches = [&](auto checked) {
        constexpr bool kChecked = decltype(checked)::value;
        for (uint32_t p = 0; p < a.chunk; p += kAhead) {
            uint32_t key[kAhead], row[kAhead];
            Pack<T, V> g[kAhead][M];
#pragma unroll
            for (int k = 0; k < kAhead; k += 2) {  // the list has room for the last pair
                const uint64_t i = begin + p + k;
                uint4 two = make_uint4(a.vocab, 0, a.vocab, 0);
                if (!kChecked || i < a.count) two = *reinterpret_cast<const uint4*>(a.items + i);
                key[k] = two.x, row[k] = two.y, key[k + 1] = two.z, row[k + 1] = two.w;
                if (kChecked) {  // a place without a token reads row 0, which is not used
                    if (i + 1 >= a.count) key[k + 1] = a.vocab;
                    if (key[k] >= a.vocab) row[k] = 0;
                    if (key[k + 1] >= a.vocab) row[k + 1] = 0;
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
#pragma unroll
                for (int m = 0; m < M; m++)
                    g[k][m] = *reinterpret_cast<const Pack<T, V>*>(from[m] + row[k] * a.grad_stride);
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                if (key[k] != cur) {
                    if (head) keep_head();
                    else write(cur, acc);
                    head = false;
                    cur = key[k];
#pragma unroll
                    for (int m = 0; m < M; m++) acc[m].clear();
                }
#pragma unroll
                for (int m = 0; m < M; m++) acc[m].add(g[k][m]);
            }
        }
    };
    if (whole) batches(std::false_type{});
    else batches(std::true_type{});
    const bool to_after = cur < a.vocab && key_at(a, begin + a.chunk) == cur;
    if (head) keep_head();
    else if (!to_after && cur < a.vocab) write(cur, acc);
    if (lane == 0) goes_on[group] = head && to_after;
    __syncthreads();
    const uint64_t block = (uint64_t)blockIdx.x * 2 * a.dim;
    auto add_head = [&](Sums<V>* sum, uint32_t h) {
#pragma unroll
        for (int m = 0; m < M; m++) sum[m].add(heads + (m * kThreads + h * lanes + lane) * V);
    };
    auto keep_part = [&](uint64_t at, const Sums<V>* sum) {
#pragma unroll
        for (int m = 0; m < M; m++) {
            if (!column[m]) continue;
#pragma unroll
            for (int i = 0; i < V; i++) a.part[at + c[m] + i] = sum[m].v[i];
        }
    };
    if (!head && to_after) {  // a run that began here
        bool open = true;
        for (uint32_t h = group + 1; h < groups && open; h++) {
            add_head(acc, h);
            open = goes_on[h];
        }
        if (open) keep_part(block + a.dim, acc);
        else write(cur, acc);
    }
    if (group == 0 && from_before) {  // the run that came into the block
        Sums<V> sum[M];
#pragma unroll
        for (int m = 0; m < M; m++) sum[m].clear();
        bool open = true;
        for (uint32_t h = 0; h < groups && open; h++) {
            add_head(sum, h);
            open = goes_on[h];
        }
        keep_part(block, sum);
    }
}

// A block joins the run that leaves block x of k_run_sums, if it began there:
// its own part and what the following blocks it goes through (and the one it
// ends in) have of it, each group a share of the blocks, then the groups.
template <class T, int V>
__global__ void __launch_bounds__(kRunThreads) k_run_joins(RunSums a, T* __restrict__ out) {
    __shared__ float sums[kRunThreads * V];
    const uint32_t groups = kRunThreads / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x & (a.lanes - 1);
    const uint64_t span = (uint64_t)groups * a.chunk, begin = blockIdx.x * span, end = begin + span;
    cudaGridDependencySynchronize();  // the blocks' sums
    const uint32_t key = key_at(a, end - 1);
    if (key >= a.vocab || key_at(a, end) != key) return;                            // no run leaves
    if (begin > 0 && key_at(a, begin - 1) == key) return;                           // it only goes through
    uint32_t more = 0;  // the following blocks that start in the run
    for (uint32_t b = 1;; b += kRunThreads) {
        const uint32_t here = __syncthreads_count(key_at(a, begin + (b + threadIdx.x) * span) == key);
        more += here;
        if (here < kRunThreads) break;
    }
    const uint32_t c = (blockIdx.y * a.lanes + lane) * V;
    const bool column = c < a.dim;
    Sums<V> acc;
    acc.clear();
    if (column) {
        const float* part = a.part + (uint64_t)blockIdx.x * 2 * a.dim + c;
        if (group == 0) {
#pragma unroll
            for (int i = 0; i < V; i++) acc.v[i] = part[a.dim + i];
        }
#pragma unroll 4
        for (uint32_t b = 1 + group; b <= more; b += groups) acc.add(part + (uint64_t)b * 2 * a.dim);
    }
#pragma unroll
    for (int i = 0; i < V; i++) sums[threadIdx.x * V + i] = acc.v[i];
    __syncthreads();
    if (group == 0 && column) {
        for (uint32_t h = 1; h < groups && h <= more; h++) acc.add(sums + (h * a.lanes + lane) * V);
        write_row<T, V>(a, out, key, c, acc);
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
    constexpr int kMost = 16 / sizeof(T);
    if (v == 1) f(std::integral_constant<int, 1>{});
    else if (v == 2) f(std::integral_constant<int, 2>{});
    else if (v == 4) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, kMost>{});
}
// The same of rows that keep 16-byte boundaries.  How a sum is split follows from this width, so that its order, and
// with it every bit, depends on the sizes and the type alone; rows off the boundaries take narrower vectors in that
// split.
uint32_t even_width(uint32_t size, uint64_t dim) { return vector_width(size, dim, nullptr, 0, nullptr, 0); }
// Vectors that a lane of k_run_sums takes of an even row: four where each is a single element (a row off the wider
// boundaries), so that a place's key and row serve four loads.  8192 rows of 200 tokens of 127 bf16: 163 us, 220 with
// one; pairs of 16-bit elements gain nothing.
uint32_t vectors_of_lane(uint32_t v, uint32_t vectors) { return v == 1 && vectors > 8 ? 4 : 1; }
// f with constants M and R of k_run_sums, for vectors narrower than even ones: as many a lane as make up for it, up to
// two pairs or four elements, then twice the lanes.  8192 rows of 200 tokens, a bf16 gradient one element off: 112 us for
// rows of 32, 130 without the second; two off: 87 for rows of 32, 142 for 128 (110 and 189); even: 75 and 110.  Where
// the lanes of an even row are a warp already, more of them cost single elements time (1024: 87 us, 81 without).
template <class T, int V, class F> void with_vectors_of_lane(uint32_t each, uint32_t lanes, F&& f) {
    using std::integral_constant;
    constexpr int kEven = 16 / (int)sizeof(T) / V, kMost = V == 1 ? 4 : std::min(2, kEven);
    if constexpr (kEven > kMost) {
        if (each > kMost && (V > 1 || lanes < 32)) return f(integral_constant<int, kMost>{}, integral_constant<int, 2>{});
    }
    if (each > 2) f(integral_constant<int, kMost>{}, integral_constant<int, 1>{});
    else if (each > 1) f(integral_constant<int, std::min(2, kMost)>{}, integral_constant<int, 1>{});
    else f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
}
// Launches a kernel that may be set up while the one before it on the stream
// ends; it waits for that one (cudaGridDependencySynchronize) before it reads
// anything.  Saves about 2 us a kernel where each takes a few.
template <class K, class... A> void launch_behind(K kernel, dim3 grid, int threads, cudaStream_t s, A... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    count_launch();
    FB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
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
    uint64_t items[2], hist, total, part, bytes;
    uint32_t count, tiles, bits, passes;
    GradSpace(uint64_t n, uint64_t per_row, uint64_t vocab, uint32_t dim) {
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
        for (int i = 0; i < 2; i++) items[i] = take(8ull * count + 8);  // a last pair is read whole
        hist = take(4ull * (1ull << bits) * tiles);
        total = take(4ull << bits);
        // two rows for each block of k_run_sums; a chunk below the longest is only taken for few blocks
        const uint32_t groups = kRunThreads / lanes_for(dim);  // the fewest of any vector width
        part = take(8ull * dim * std::min(ceil_div(count, groups * kAhead),
                                          std::max(ceil_div(count, groups * kMostChunk), 2 * kFewBlocks)));
        bytes = at;
    }
};
constexpr uint64_t kMostPlaces = 0x7ffffffeull;

bool grad_sizes_fit(uint64_t n, uint64_t per_row, uint64_t vocab) {
    return vocab <= kMostPlaces && (per_row == 0 || n <= kMostPlaces / per_row);
}

}  // namespace

void launch_clear(void* p, uint64_t rows, uint64_t bytes, uint64_t stride, cudaStream_t s) {
    const Clear z = clear_of(p, rows, bytes, stride);
    const uint64_t units = z.rows * ((z.bytes + 15) / 16);
    count_launch();
    k_clear<<<(uint32_t)std::min<uint64_t>(148 * 8, (units + 255) / 256), 256, 0, s>>>(z);
}

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
            const Tokens<Tok> tk(tokens, token_row, token_col, vocab);
            if (per_row == 1) {
                for (uint64_t c = 0; c < dim; c += kLookupColumns) {
                    const uint32_t columns = (uint32_t)std::min<uint64_t>(dim - c, kLookupColumns);
                    // rows of several 16-byte vectors that do not keep their boundaries
                    const bool odd = v * size < 16 && columns >= 64 / size;
                    LookupArgs a{table_stride, n, out_stride, columns, 0, scale};
                    while (1u << a.lanes_log < lanes_for(odd ? columns / (16 / size) + 2 : columns / v)) a.lanes_log++;
                    // every SM full once, then several rows a group, then more
                    const uint64_t wish = (n + (kLookupThreads >> a.lanes_log) - 1) / (kLookupThreads >> a.lanes_log);
                    const uint64_t full = 148 * 8;
                    const uint32_t blocks = (uint32_t)std::min<uint64_t>(
                        1u << 20, std::max(std::min(wish, full), (wish + kLookupRows - 1) / kLookupRows));
                    count_launch();
                    with_type(type, [&](auto e) {
                        using T = decltype(e);
                        const T* from = static_cast<const T*>(table) + c;
                        T* to = static_cast<T*>(out) + c;
                        if (odd) {
                            k_lookup_odd<T, Tok><<<blocks, kLookupThreads, 0, s>>>(a, from, tk, to);
                            return;
                        }
                        with_width<T>(v, [&](auto w) {
                            k_lookup<T, Tok, decltype(w)::value><<<blocks, kLookupThreads, 0, s>>>(a, from, tk, to);
                        });
                    });
                }
            } else {
                BagArgs a{table_stride, n, out_stride, dim, per_row, per_row, 0, 0, scale};
                // parts of a row, until every SM has about a thousand threads; a part has at least eight tokens.  As for
                // even rows in every layout: 8192 rows of 200 tokens of 32 bf16, one element off, take 47 us in eight
                // parts (37 whole, in another order; even rows 21)
                const uint32_t even = dim / even_width(size, dim), even_lanes = lanes_for(even);
                uint32_t even_log = 0;
                while (1u << even_log < even_lanes) even_log++;
                const uint32_t even_slices = ceil_div(even, even_lanes);
                while (even_log + a.parts_log < 8 && a.part_len > kBagAhead &&
                       n < (148ull * 1024 >> (even_log + a.parts_log)) / even_slices) {
                    a.parts_log++;
                    a.part_len = ceil_div(per_row, 1u << a.parts_log);
                }
                const uint32_t vectors = dim / v;
                while (a.lanes_log + a.parts_log < 8 && 1u << a.lanes_log < lanes_for(vectors)) a.lanes_log++;
                const uint32_t slices = ceil_div(vectors, 1u << a.lanes_log);
                if (slices > kMostSlices) throw InputError("fbgpu_embed takes rows of at most 2097120 elements");
                const uint32_t rows = kBagThreads >> (a.lanes_log + a.parts_log);
                const dim3 grid((uint32_t)std::min<uint64_t>(1u << 20, (n + rows - 1) / rows), slices);
                count_launch();
                with_type(type, [&](auto e) {
                    using T = decltype(e);
                    with_width<T>(v, [&](auto w) {
                        if (token_col == 1)
                            k_embed<T, Tok, decltype(w)::value, true><<<grid, kBagThreads, 0, s>>>(
                                a, static_cast<const T*>(table), tk, static_cast<T*>(out));
                        else
                            k_embed<T, Tok, decltype(w)::value, false><<<grid, kBagThreads, 0, s>>>(
                                a, static_cast<const T*>(table), tk, static_cast<T*>(out));
                    });
                });
            }
            FB_CUDA_CHECK(cudaGetLastError());
        });
    });
}

extern "C" uint64_t fbgpu_embed_grad_workspace(uint64_t n, uint32_t per_row, uint64_t vocab, uint32_t dim) {
    return fbg::grad_sizes_fit(n, per_row, vocab) ? fbg::GradSpace(n, per_row, vocab, dim).bytes : 0;
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
        if (dim > kMostSlices * 32) throw InputError("fbgpu_embed_grad takes rows of at most 2097120 elements");
        with_token(token_type, [&](auto tok) {
            using Tok = decltype(tok);
            check_tokens(tokens, n, per_row, token_row, token_col, sizeof(Tok));
            const GradSpace ws(n, per_row, vocab, dim);
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
            const Tokens<Tok> tk(tokens, token_row, token_col, vocab);
            const Clear z = clear_of(out, vocab, (uint64_t)dim * size, out_stride * size);
            const uint64_t cleared = z.rows * ((z.bytes + 15) / 16);
            if (ws.count == 0 || ws.count > kClusterPlaces)
                launch_clear(out, vocab, (uint64_t)dim * size, out_stride * size, s);
            if (ws.count == 0) {
                FB_CUDA_CHECK(cudaGetLastError());
                return;
            }
            const Places<Tok> places{tk, Divisor(per_row)};
            const bool flat = (per_row == 1 || token_col == 1) && (n == 1 || token_row == per_row);
            uint2* items[2] = {reinterpret_cast<uint2*>(w + ws.items[0]), reinterpret_cast<uint2*>(w + ws.items[1])};
            if (ws.count <= kClusterPlaces) {
                const ClusterSort a{{items[0], items[1]}, ws.count, ws.bits, ws.passes};
                auto launch = [&](auto of) {
                    const uint64_t wish = (cleared + 4 * kClusterThreads - 1) / (4 * kClusterThreads);
                    cudaLaunchConfig_t cfg{};
                    cfg.gridDim = dim3(kClusterCtas * (1 + ceil_div(std::min<uint64_t>(148 * 3, wish), kClusterCtas)));
                    cfg.blockDim = dim3(kClusterThreads);
                    cfg.stream = s;
                    cudaLaunchAttribute attr{};
                    attr.id = cudaLaunchAttributeClusterDimension;
                    attr.val.clusterDim.x = kClusterCtas;
                    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
                    cfg.attrs = &attr;
                    cfg.numAttrs = 1;
                    count_launch();
                    if (flat)
                        FB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k_sort_cluster<Tok, kFlat, decltype(of)::value>, a, places, z));
                    else
                        FB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k_sort_cluster<Tok, kStrided, decltype(of)::value>, a, places, z));
                };
                const uint32_t each = ceil_div(ws.count, kClusterCtas * kClusterThreads);  // places of a thread
                if (each <= 2) launch(std::integral_constant<int, 2>{});
                else if (each <= 4) launch(std::integral_constant<int, 4>{});
                else if (each <= 8) launch(std::integral_constant<int, 8>{});
                else launch(std::integral_constant<int, 16>{});
            } else {
                for (uint32_t p = 0; p < ws.passes; p++) {
                    SortPass a{};
                    a.in = items[~p & 1];
                    a.out = items[p & 1];
                    a.hist = at(ws.hist);
                    a.total = at(ws.total);
                    a.count = ws.count;
                    a.tiles = ws.tiles;
                    a.shift = p * ws.bits;
                    a.bits = ws.bits;
                    auto pass = [&](auto source) {
                        constexpr Source S = decltype(source)::value;
                        launch_behind(k_sort_count<Tok, S>, dim3(ws.tiles), kSortThreads, s, a, places);
                        launch_behind(k_sort_scan, dim3(1u << ws.bits), kSortThreads, s, a);
                        launch_behind(k_sort_scatter<Tok, S>, dim3(ws.tiles), kSortThreads, s, a, places);
                    };
                    if (p) pass(std::integral_constant<Source, kItems>{});
                    else if (flat) pass(std::integral_constant<Source, kFlat>{});
                    else pass(std::integral_constant<Source, kStrided>{});
                }
            }
            const int last = (ws.passes - 1) & 1;
            const uint32_t v = vector_width(size, dim, grad, grad_stride, out, out_stride);
            RunSums a{};
            a.items = items[last];
            a.part = reinterpret_cast<float*>(w + ws.part);
            a.count = ws.count;
            a.vocab = (uint32_t)vocab;
            a.dim = dim;
            const uint32_t even_v = even_width(size, dim), even = dim / even_v, even_each = vectors_of_lane(even_v, even);
            a.lanes = lanes_for(ceil_div(even, even_each));
            a.grad_stride = grad_stride;
            a.out_stride = out_stride;
            a.scale = scale;
            const uint32_t groups = kRunThreads / a.lanes, even_slices = ceil_div(even, a.lanes * even_each);
            // longer chunks mean fewer joins, as long as every SM has a few blocks
            a.chunk = kMostChunk;
            while (a.chunk > kAhead && (uint64_t)ceil_div(ws.count, groups * a.chunk) * even_slices < kFewBlocks) a.chunk /= 2;
            const uint32_t blocks = ceil_div(ws.count, groups * a.chunk), vectors = dim / v;
            with_type(type, [&](auto e) {
                using T = decltype(e);
                with_width<T>(v, [&](auto wd) {
                    constexpr int V = decltype(wd)::value;
                    with_vectors_of_lane<T, V>(even_v * even_each / v, a.lanes, [&](auto m, auto r) {
                        constexpr int M = decltype(m)::value, R = decltype(r)::value;
                        launch_behind(k_run_sums<T, V, M, R>, dim3(blocks, ceil_div(vectors, a.lanes * M * R)),
                                      kRunThreads * R, s, a, static_cast<const T*>(grad), static_cast<T*>(out));
                    });
                    if (blocks > 1)
                        launch_behind(k_run_joins<T, V>, dim3(blocks, ceil_div(vectors, a.lanes)), kRunThreads, s, a,
                                      static_cast<T*>(out));
                });
            });
            FB_CUDA_CHECK(cudaGetLastError());
        });
    });
}
