// Rows by index: lookup in a table, rows to the places of their clusters and back, and the gradients of the weights and scales.
//
// All of them move rows once and compute next to nothing: they are bound by HBM, or for small calls by the launch.  The rows of an
// output (or for to_clusters of the input) are taken as one sequence of 32-byte chunks, 128 x 2 of them to a block whatever the rows'
// width, so that narrow and odd rows fill the lanes as well as wide ones; a row whose address, pitch or width is no multiple of 32
// bytes is taken in chunks of 16, 128 x 4 to a block, and one that these do not fit is left to rows_unaligned.cu, or, if it has less than
// 32 bytes, taken in chunks of 8, 4 or 2.  Products and sums are in fp32 and rounded once.
//
// One B200, each kernel by itself: lookup of 1M x 768 bf16 with scales out of 65 536 rows 309 us, 1.99 GB to and from HBM (0.5 of them rows
// that the second-level cache had lost) at 6.4 TB/s; with chunks of 16 bytes 420, with four of 32 in a thread 347, stores that pass the
// cache by: the same.  131 072 x 2 rows of 1024 bf16 to their clusters 118 us (6.8 TB/s) and back 132 (6.1; blocks of 256 threads 149, one
// choice on its way at a time 221); the gradients of 131 072 x 2 x 768 and their weights 163 (6.2; with chunks of 32 bytes 185).
#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr int kThreads = 128;

// Chunks of a thread, all loaded before the first is stored: 64 bytes, which with the 40 warps of an SM keep 80 KB on their way.
template <int BYTES>
constexpr int kAhead = BYTES == 32 ? 2 : 4;

// The chunks of n rows, `width` to a row.
struct Spread {
    size_t total;
    Divisor width;
};

template <int BYTES>
Spread make_spread(size_t n, size_t row_bytes) {
    const size_t width = row_bytes / BYTES;
    return {n * width, make_divisor(width, width + kThreads * kAhead<BYTES>)};
}
unsigned spread_blocks(const Spread& s, int ahead) { return static_cast<unsigned>((s.total + kThreads * ahead - 1) / (kThreads * ahead)); }

// This thread's chunks: row and place in the row of chunk u, and whether there is one.
template <int BYTES, int AHEAD = kAhead<BYTES>>
struct Mine {
    size_t row0;
    uint32_t off;
    size_t left;   // chunks from this thread's first one to the end
    Divisor width;

    __device__ __forceinline__ explicit Mine(const Spread& s) : width(s.width) {
        const size_t first = static_cast<size_t>(blockIdx.x) * (kThreads * AHEAD);
        row0 = (first >> 32) == 0 ? static_cast<uint32_t>(first) / s.width.d : first / s.width.d;
        off = static_cast<uint32_t>(first - row0 * s.width.d) + threadIdx.x;
        left = first + threadIdx.x < s.total ? s.total - first - threadIdx.x : 0;
    }
    __device__ __forceinline__ bool has(int u) const { return static_cast<size_t>(u) * kThreads < left; }
    __device__ __forceinline__ void at(int u, size_t& row, uint32_t& col) const {
        const uint32_t a = off + u * kThreads, q = divide(a, width);
        row = row0 + q;
        col = a - q * width.d;
    }
};

template <typename C>
__device__ __forceinline__ const C* row_at(const void* p, size_t pitch, size_t row) {
    return reinterpret_cast<const C*>(static_cast<const char*>(p) + row * pitch);
}

template <typename T, int BYTES, bool SCALED>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const void* __restrict__ table, size_t pitch, uint32_t k, const void* __restrict__ ids, bool wide, float scale,
                                                          const float* __restrict__ row_scales, Chunk<BYTES>* __restrict__ out, const Spread spread) {
    constexpr int AHEAD = kAhead<BYTES>;
    const Mine<BYTES> mine(spread);
    size_t row[AHEAD];
    uint32_t col[AHEAD], id[AHEAD];
    Chunk<BYTES> c[AHEAD];
    float f[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        id[u] = k;
        if (mine.has(u)) {
            mine.at(u, row[u], col[u]);
            id[u] = load_id(ids, wide, row[u], k);
            if (SCALED) f[u] = row_scales ? scale * __ldg(row_scales + row[u]) : scale;
        }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) c[u] = id[u] < k ? load_chunk<BYTES>(row_at<Chunk<BYTES>>(table, pitch, id[u]) + col[u]) : zero_chunk<BYTES>();
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        if (!mine.has(u)) continue;
        if (SCALED && id[u] < k) {
            Values<T, BYTES> v;
            v.from(c[u]);
#pragma unroll
            for (int i = 0; i < v.N; ++i) v.v[i] *= f[u];
            c[u] = v.to();
        }
        store_chunk<BYTES>(out + row[u] * spread.width.d + col[u], c[u]);
    }
}

template <int BYTES>
__global__ void __launch_bounds__(kThreads) to_clusters_kernel(const void* __restrict__ x, size_t pitch, const Places at, Chunk<BYTES>* __restrict__ out, const Spread spread) {
    constexpr int AHEAD = kAhead<BYTES>;
    const Mine<BYTES> mine(spread);
    const uint32_t slots = static_cast<uint32_t>(at.n * at.m), held = min(__ldg(at.held), slots);
    Chunk<BYTES> c[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (mine.has(u)) {
            size_t row;
            uint32_t col;
            mine.at(u, row, col);
            c[u] = load_chunk<BYTES>(row_at<Chunk<BYTES>>(x, pitch, row) + col);
        }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (mine.has(u)) {
            size_t row;
            uint32_t col;
            mine.at(u, row, col);
            for (size_t j = 0; j < at.m; ++j) {
                const uint32_t slot = __ldg(at.position + row * at.m + j);
                if (slot < slots) store_chunk<BYTES>(out + static_cast<size_t>(slot) * spread.width.d + col, slot < held ? c[u] : zero_chunk<BYTES>());
            }
        }
}

// Two choices of each chunk are on their way at a time.
template <typename T, int BYTES>
__global__ void __launch_bounds__(kThreads) from_clusters_kernel(const void* __restrict__ y, size_t pitch, const Places at, const float* __restrict__ weights,
                                                                 Chunk<BYTES>* __restrict__ out, const Spread spread) {
    constexpr int AHEAD = kAhead<BYTES> / 2;
    const Mine<BYTES, AHEAD> mine(spread);
    const uint32_t slots = static_cast<uint32_t>(at.n * at.m), held = min(__ldg(at.held), slots);
    size_t row[AHEAD];
    uint32_t col[AHEAD];
    Values<T, BYTES> sum[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        if (mine.has(u)) mine.at(u, row[u], col[u]);
#pragma unroll
        for (int i = 0; i < sum[u].N; ++i) sum[u].v[i] = 0.f;
    }
    for (size_t j = 0; j < at.m; j += 2) {
        Chunk<BYTES> c[AHEAD][2];
        float w[AHEAD][2];
        uint32_t slot[AHEAD][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool there = mine.has(u) && j + e < at.m;
                slot[u][e] = there ? __ldg(at.position + row[u] * at.m + j + e) : 0xffffffffu;
                w[u][e] = there && weights ? __ldg(weights + row[u] * at.m + j + e) : 1.f;
            }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (slot[u][e] < held) c[u][e] = load_chunk<BYTES>(row_at<Chunk<BYTES>>(y, pitch, slot[u][e]) + col[u]);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (slot[u][e] < held) {
                    Values<T, BYTES> v;
                    v.from(c[u][e]);
#pragma unroll
                    for (int i = 0; i < v.N; ++i) sum[u].v[i] = fmaf(w[u][e], v.v[i], sum[u].v[i]);
                }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (mine.has(u)) store_chunk<BYTES>(out + row[u] * spread.width.d + col[u], sum[u].to());
}

// LANES lanes per row of grad: <grad[i], y[slot]> and grad_y[slot] = w * grad[i] for its choices, y read once.
template <typename T, int BYTES, int LANES>
__global__ void __launch_bounds__(kThreads) from_clusters_grad_kernel(const void* __restrict__ grad, size_t grad_pitch, const void* __restrict__ y, size_t y_pitch, const Places at,
                                                                      const float* __restrict__ weights, Chunk<BYTES>* __restrict__ grad_y, float* __restrict__ grad_weights,
                                                                      uint32_t width) {
    const Lanes<LANES> lanes;
    const size_t row = static_cast<size_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
    if (row >= at.n) return;
    const uint32_t lane = lanes.lane;
    const uint32_t slots = static_cast<uint32_t>(at.n * at.m), held = min(__ldg(at.held), slots);
    const Chunk<BYTES>* g = row_at<Chunk<BYTES>>(grad, grad_pitch, row);
    for (size_t j = 0; j < at.m; ++j) {
        const uint32_t slot = __ldg(at.position + row * at.m + j);
        const bool there = slot < held;
        const float w = weights ? __ldg(weights + row * at.m + j) : 1.f;
        const Chunk<BYTES>* from = row_at<Chunk<BYTES>>(y, y_pitch, slot);
        Chunk<BYTES>* to = grad_y + static_cast<size_t>(slot) * width;
        float dot = 0.f;
        if (!there) {
            if (grad_y && slot < slots)
                for (uint32_t c = lane; c < width; c += LANES) store_chunk<BYTES>(to + c, zero_chunk<BYTES>());
        } else {
#pragma unroll 4
            for (uint32_t c = lane; c < width; c += LANES) {
                Values<T, BYTES> a;
                a.from(load_chunk<BYTES>(g + c));
                if (grad_weights) {
                    Values<T, BYTES> b;
                    b.from(load_chunk<BYTES>(from + c));
#pragma unroll
                    for (int i = 0; i < a.N; ++i) dot = fmaf(a.v[i], b.v[i], dot);
                }
                if (grad_y) {
#pragma unroll
                    for (int i = 0; i < a.N; ++i) a.v[i] *= w;
                    store_chunk<BYTES>(to + c, a.to());
                }
            }
        }
        if (grad_weights) {
            dot = lanes.sum(dot);
            if (lane == 0) grad_weights[row * at.m + j] = dot;
        }
    }
}

template <typename T, int BYTES, int LANES>
__global__ void __launch_bounds__(kThreads) lookup_scale_grad_kernel(const void* __restrict__ grad, size_t grad_pitch, const void* __restrict__ table, size_t table_pitch, uint32_t k,
                                                                     const void* __restrict__ ids, bool wide, size_t n, float scale, float* __restrict__ out, uint32_t width) {
    const Lanes<LANES> lanes;
    const size_t row = static_cast<size_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
    if (row >= n) return;
    const uint32_t lane = lanes.lane;
    const uint32_t id = load_id(ids, wide, row, k);
    float dot = 0.f;
    if (id < k) {
        const Chunk<BYTES>* g = row_at<Chunk<BYTES>>(grad, grad_pitch, row);
        const Chunk<BYTES>* t = row_at<Chunk<BYTES>>(table, table_pitch, id);
#pragma unroll 4
        for (uint32_t c = lane; c < width; c += LANES) {
            Values<T, BYTES> a, b;
            a.from(load_chunk<BYTES>(g + c));
            b.from(load_chunk<BYTES>(t + c));
#pragma unroll
            for (int i = 0; i < a.N; ++i) dot = fmaf(a.v[i], b.v[i], dot);
        }
    }
    dot = lanes.sum(dot);
    if (lane == 0) out[row] = id < k ? scale * dot : 0.f;
}

// Lanes to a row: eight where it has no more than 16 chunks (rows of 64 bf16, 300 000 of them: gradient of the scales 61 us with 32 lanes, 19
// with eight; of 150 000 x 2 weights 60 and 24).
bool few_chunks(size_t chunks) { return chunks <= 16; }
unsigned row_blocks(size_t n, int lanes) { return static_cast<unsigned>((n + kThreads / lanes - 1) / (kThreads / lanes)); }

} // namespace

void launch_lookup(const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, const float* row_scales, void* out, cudaStream_t stream) {
    if (n == 0) return;
    const size_t t = type_bytes(type), pitch = table.ld * t;
    const int access = access_bytes({address(table.p), pitch, d * t, address(out)}, 32);
    if (access < 16 && d * t >= 32 && address(out) % 16 == 0) return launch_lookup_unaligned(table, type, k, d, ids, n, scale, row_scales, out, stream);
    with_width<32>(type, access, [&](auto value, auto width) {
        using T = decltype(value);
        constexpr int B = decltype(width)::bytes;
        const Spread s = make_spread<B>(n, d * t);
        // (a product with one changes no value: the plain copy is for that)
        auto* kernel = row_scales || scale != 1.0f ? lookup_kernel<T, B, true> : lookup_kernel<T, B, false>;
        kernel<<<spread_blocks(s, kAhead<B>), kThreads, 0, stream>>>(table.p, pitch, static_cast<uint32_t>(k), ids.p, ids.wide, scale, row_scales, static_cast<Chunk<B>*>(out), s);
    });
    SKM_LAUNCH_CHECK();
}

void launch_lookup_scale_grad(const Rows& grad, const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, float* out, cudaStream_t stream) {
    if (n == 0) return;
    const size_t t = type_bytes(type);
    const int access = access_bytes({address(grad.p), grad.ld * t, address(table.p), table.ld * t, d * t});
    if (use_windows(access, d * t)) return launch_lookup_scale_grad_unaligned(grad, table, type, k, d, ids, n, scale, out, stream);
    with_width(type, access, [&](auto value, auto width) {
        constexpr int B = decltype(width)::bytes;
        const bool narrow = few_chunks(d * t / B);
        auto* kernel = narrow ? lookup_scale_grad_kernel<decltype(value), B, 8> : lookup_scale_grad_kernel<decltype(value), B, 32>;
        kernel<<<row_blocks(n, narrow ? 8 : 32), kThreads, 0, stream>>>(grad.p, grad.ld * t, table.p, table.ld * t, static_cast<uint32_t>(k), ids.p, ids.wide, n, scale, out,
                                                                                            static_cast<uint32_t>(d * t / B));
    });
    SKM_LAUNCH_CHECK();
}

void launch_to_clusters(const Rows& x, Type type, size_t d, const Places& at, void* out, cudaStream_t stream) {
    if (at.n == 0) return;
    const size_t t = type_bytes(type), pitch = x.ld * t;
    const int access = access_bytes({address(x.p), pitch, d * t, address(out)}, 32);
    if (access < 16 && d * t >= 32 && address(out) % 16 == 0) return launch_to_clusters_unaligned(x, type, d, at, nullptr, out, stream);
    with_width<32>(type, access, [&](auto, auto width) {
        constexpr int B = decltype(width)::bytes;
        const Spread s = make_spread<B>(at.n, d * t);
        to_clusters_kernel<B><<<spread_blocks(s, kAhead<B>), kThreads, 0, stream>>>(x.p, pitch, at, static_cast<Chunk<B>*>(out), s);
    });
    SKM_LAUNCH_CHECK();
}

void launch_from_clusters(const Rows& y, Type type, size_t d, const Places& at, const float* weights, void* out, cudaStream_t stream) {
    if (at.n == 0) return;
    const size_t t = type_bytes(type), pitch = y.ld * t;
    const int access = access_bytes({address(y.p), pitch, d * t, address(out)}, 32);
    if (access < 16 && d * t >= 32 && address(out) % 16 == 0) return launch_from_clusters_unaligned(y, type, d, at, weights, out, stream);
    with_width<32>(type, access, [&](auto value, auto width) {
        constexpr int B = decltype(width)::bytes;
        const Spread s = make_spread<B>(at.n, d * t);
        from_clusters_kernel<decltype(value), B><<<spread_blocks(s, kAhead<B> / 2), kThreads, 0, stream>>>(y.p, pitch, at, weights, static_cast<Chunk<B>*>(out), s);
    });
    SKM_LAUNCH_CHECK();
}

void launch_from_clusters_grad(const Rows& grad, const Rows& y, Type type, size_t d, const Places& at, const float* weights, void* grad_y, float* grad_weights, cudaStream_t stream) {
    if (at.n == 0) return;
    const size_t t = type_bytes(type);
    const int access = access_bytes({address(grad.p), grad.ld * t, address(y.p), y.ld * t, d * t, address(grad_y)});
    if (use_windows(access, d * t) && address(grad_y) % 16 == 0) {
        if (grad_y) launch_to_clusters_unaligned(grad, type, d, at, weights, grad_y, stream);
        if (grad_weights) launch_weights_grad_unaligned(grad, y, type, d, at, grad_weights, stream);
        return;
    }
    with_width(type, access, [&](auto value, auto width) {
        constexpr int B = decltype(width)::bytes;
        const bool narrow = few_chunks(d * t / B);
        auto* kernel = narrow ? from_clusters_grad_kernel<decltype(value), B, 8> : from_clusters_grad_kernel<decltype(value), B, 32>;
        kernel<<<row_blocks(at.n, narrow ? 8 : 32), kThreads, 0, stream>>>(grad.p, grad.ld * t, y.p, y.ld * t, at, weights, static_cast<Chunk<B>*>(grad_y), grad_weights,
                                                                                               static_cast<uint32_t>(d * t / B));
    });
    SKM_LAUNCH_CHECK();
}

} // namespace rows
} // namespace skmb
