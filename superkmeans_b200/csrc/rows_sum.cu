// Gradient of a lookup: for every row of the table the sum of the gradients of the pairs that took it, scaled.
//
// The pairs are sorted by id (rows_group.cu) and cut into tiles of equal length, so that a row that half of the pairs took is no
// longer to sum than a thousand rows are.  A warp takes a tile and 32 chunks of its columns, reads the rows that the order names,
// eight ahead, and adds in fp32 registers; a run of equal ids that lies inside the tile goes straight to the output, the tile's first
// and last run, which may go on in the neighbours, into partial sums.  A second launch adds the partial sums of each id in the order of
// their tiles and writes the zeros of ids that nobody took.  Nothing depends on the order of atomics.
#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr int kWarps = 4;
constexpr int kAhead = 8;

struct SumParams {
    const void* grad;
    size_t pitch;
    const uint32_t* order;     // pairs by id
    const uint32_t* keys;      // their ids
    const uint32_t* offsets;   // k + 1
    const float* row_scales;
    float scale;
    uint32_t n, k, d;
    uint32_t width;            // chunks to a row
    uint32_t slabs;            // of 32 chunks
    uint32_t tile;             // pairs to a tile
    float* partials;           // per tile two rows of d: the first run, and the last if it is another
    void* out;
};

template <typename T, typename O, int BYTES>
__device__ __forceinline__ void store_sum(const Values<T, BYTES>& sum, O* to) {
    constexpr int N = Values<T, BYTES>::N, OUT = N * static_cast<int>(sizeof(O));
    if constexpr (OUT <= 16) {
        Values<O, OUT> v;
#pragma unroll
        for (int i = 0; i < N; ++i) v.v[i] = sum.v[i];
        *reinterpret_cast<Chunk<OUT>*>(to) = v.to();
    } else {   // eight sums of halves in fp32
        Values<O, 16> v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v.v[i] = sum.v[4 * h + i];
            reinterpret_cast<Chunk<16>*>(to)[h] = v.to();
        }
    }
}

template <typename T, typename O, int BYTES>
__global__ void __launch_bounds__(32 * kWarps) sum_tiles_kernel(const SumParams p) {
    using V = Values<T, BYTES>;
    const uint32_t lane = threadIdx.x & 31;
    const size_t unit = static_cast<size_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const size_t tile = unit / p.slabs, begin = tile * p.tile;
    const uint32_t held = __ldg(p.offsets + p.k);
    if (begin >= held) return;   // (pairs without an id come last)
    const uint32_t col = static_cast<uint32_t>(unit - tile * p.slabs) * 32 + lane;
    const bool mine = col < p.width;
    const uint32_t s0 = static_cast<uint32_t>(begin), s1 = min(s0 + p.tile, held);
    const size_t at = static_cast<size_t>(col) * V::N;
    float* first_part = p.partials + tile * 2 * p.d + at;
    V sum;
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < V::N; ++i) sum.v[i] = 0.f;
    };
    clear();
    uint32_t now = __ldg(p.keys + s0);
    bool first = true;
    for (uint32_t s = s0; s < s1; s += 32) {
        // a lane's pair of the next 32
        const uint32_t my = s + lane;
        const uint32_t my_pair = my < s1 ? __ldg(p.order + my) : 0u, my_key = my < s1 ? __ldg(p.keys + my) : 0u;
        const float my_factor = p.row_scales ? p.scale * (my < s1 ? __ldg(p.row_scales + my_pair) : 0.f) : p.scale;
        const uint32_t count = min(32u, s1 - s);
        for (uint32_t u0 = 0; u0 < count; u0 += kAhead) {
            Chunk<BYTES> c[kAhead];
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) {
                const uint32_t pair = __shfl_sync(0xffffffffu, my_pair, u0 + u);
                if (u0 + u < count && mine) c[u] = __ldg(reinterpret_cast<const Chunk<BYTES>*>(static_cast<const char*>(p.grad) + pair * p.pitch) + col);
            }
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) {
                const uint32_t key = __shfl_sync(0xffffffffu, my_key, u0 + u);
                const float f = __shfl_sync(0xffffffffu, my_factor, u0 + u);
                if (u0 + u < count) {
                    if (key != now) {
                        if (mine) {
                            if (first) store_sum<T, float, BYTES>(sum, first_part);
                            else store_sum<T, O, BYTES>(sum, static_cast<O*>(p.out) + static_cast<size_t>(now) * p.d + at);
                        }
                        clear();
                        first = false;
                        now = key;
                    }
                    if (mine) {
                        V v;
                        v.from(c[u]);
#pragma unroll
                        for (int i = 0; i < V::N; ++i) sum.v[i] = fmaf(f, v.v[i], sum.v[i]);
                    }
                }
            }
        }
    }
    if (mine) store_sum<T, float, BYTES>(sum, first ? first_part : first_part + p.d);
}

// Eight ids to a block, a warp and 32 chunks each; ids whose pairs fill many tiles are taken by all eight warps together.
constexpr int kJoinWarps = 8;
constexpr uint32_t kLongRun = 32;   // tiles

template <typename T, typename O, int BYTES>
__global__ void __launch_bounds__(32 * kJoinWarps) join_tiles_kernel(const SumParams p) {
    using V = Values<T, BYTES>;
    __shared__ float parts[kJoinWarps][32][V::N + 1];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t id0 = blockIdx.x * kJoinWarps, col = blockIdx.y * 32 + lane;
    const bool mine = col < p.width;
    const size_t at = static_cast<size_t>(col) * V::N;
    // tiles of an id, and whether its sum is in the output already
    auto tiles_of = [&](uint32_t id, uint32_t& t0, uint32_t& t1, uint32_t& begin) {
        begin = __ldg(p.offsets + id);
        const uint32_t end = __ldg(p.offsets + id + 1);
        t0 = begin / p.tile;
        t1 = end > begin ? (end - 1) / p.tile + 1 : t0;
        if (t1 == t0 + 1) {
            // inside its tile, which ends where the pairs with an id end
            const uint32_t tile_end = min(static_cast<size_t>(t0 + 1) * p.tile, static_cast<size_t>(__ldg(p.offsets + p.k)));
            if (begin > t0 * p.tile && end < tile_end) return false;
        }
        return true;
    };
    auto add_tiles = [&](V& sum, uint32_t from, uint32_t to, uint32_t begin) {
        constexpr uint32_t AHEAD = 4;
        for (uint32_t t = from; t < to; t += AHEAD) {
            float v[AHEAD][V::N];
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u) {
                const size_t tile = t + u;
                const float* src = p.partials + (tile * 2 + (begin > tile * p.tile ? 1 : 0)) * p.d + at;
#pragma unroll
                for (int i = 0; i < V::N; ++i) v[u][i] = t + u < to && mine ? __ldg(src + i) : 0.f;
            }
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int i = 0; i < V::N; ++i) sum.v[i] += v[u][i];
        }
    };
    uint32_t t0 = 0, t1 = 0, begin = 0;
    const bool own = id0 + warp < p.k && tiles_of(id0 + warp, t0, t1, begin);
    if (own && t1 - t0 <= kLongRun) {
        V sum;
#pragma unroll
        for (int i = 0; i < V::N; ++i) sum.v[i] = 0.f;
        add_tiles(sum, t0, t1, begin);
        if (mine) store_sum<T, O, BYTES>(sum, static_cast<O*>(p.out) + static_cast<size_t>(id0 + warp) * p.d + at);
    }
    if (!__syncthreads_or(own && t1 - t0 > kLongRun)) return;
    for (uint32_t i = 0; i < kJoinWarps && id0 + i < p.k; ++i) {
        if (!tiles_of(id0 + i, t0, t1, begin) || t1 - t0 <= kLongRun) continue;   // (the same for the whole block)
        const uint32_t share = (t1 - t0 + kJoinWarps - 1) / kJoinWarps, from = min(t0 + warp * share, t1);
        V sum;
#pragma unroll
        for (int e = 0; e < V::N; ++e) sum.v[e] = 0.f;
        add_tiles(sum, from, min(from + share, t1), begin);
#pragma unroll
        for (int e = 0; e < V::N; ++e) parts[warp][lane][e] = sum.v[e];
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
                for (int e = 0; e < V::N; ++e) sum.v[e] += parts[w][lane][e];
            if (mine) store_sum<T, O, BYTES>(sum, static_cast<O*>(p.out) + static_cast<size_t>(id0 + i) * p.d + at);
        }
        __syncthreads();
    }
}

// Pairs to a tile: enough tiles to fill the chip several times over (148 SMs, 16 warps each), and no shorter than it takes to keep the
// partial sums' traffic below the rows'.
uint32_t tile_pairs(size_t n, size_t slabs) {
    uint32_t tile = 256;
    while (tile > 16 && (n + tile - 1) / tile * slabs < 148 * 32) tile /= 2;
    return tile;
}

// (a chunk is at most 16 bytes: with narrower ones there are more slabs, and tiles no shorter)
size_t slabs_of(size_t d, Type type, int bytes) { return (d * type_bytes(type) / bytes + 31) / 32; }

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

} // namespace

size_t lookup_grad_workspace_bytes(size_t n, size_t k, size_t d, Type type) {
    const size_t tile = tile_pairs(n, slabs_of(d, type, 16)), tiles = (n + tile - 1) / tile;
    return rounded(n * 4) * 2 + rounded((k + 1) * 4) + rounded(tiles * 2 * d * 4) + rounded(group_workspace_bytes(n, k));
}

void launch_lookup_grad(const Rows& grad, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, const float* row_scales, void* out, Type out_type, void* workspace,
                        cudaStream_t stream) {
    const size_t t = type_bytes(type);
    if (n == 0) {
        SKM_CUDA(cudaMemsetAsync(out, 0, k * d * type_bytes(out_type), stream));
        return;
    }
    SumParams p{};
    char* at = static_cast<char*>(workspace);
    auto take = [&](size_t bytes) {
        char* here = at;
        at += rounded(bytes);
        return here;
    };
    uint32_t* order = reinterpret_cast<uint32_t*>(take(n * 4));
    uint32_t* keys = reinterpret_cast<uint32_t*>(take(n * 4));
    uint32_t* offsets = reinterpret_cast<uint32_t*>(take((k + 1) * 4));
    p.tile = tile_pairs(n, slabs_of(d, type, 16));
    const size_t tiles = (n + p.tile - 1) / p.tile;
    p.partials = reinterpret_cast<float*>(take(tiles * 2 * d * 4));
    launch_group(ids, n, k, order, nullptr, keys, offsets, at, stream);
    p.grad = grad.p;
    p.pitch = grad.ld * t;
    p.order = order;
    p.keys = keys;
    p.offsets = offsets;
    p.row_scales = row_scales;
    p.scale = scale;
    p.n = static_cast<uint32_t>(n);
    p.k = static_cast<uint32_t>(k);
    p.d = static_cast<uint32_t>(d);
    p.out = out;
    // the output's chunks have as many values as the input's: of the same bytes, or in fp32 up to twice 16
    const size_t ot = type_bytes(out_type);
    const int bytes = access_bytes({address(grad.p), p.pitch, d * t, ot == t ? address(out) : address(out) / 2});
    auto launch = [&](auto value, auto result, auto width) {
        using T = decltype(value);
        using O = decltype(result);
        constexpr int B = decltype(width)::bytes;
        p.width = static_cast<uint32_t>(d * t / B);
        p.slabs = (p.width + 31) / 32;
        const size_t units = tiles * p.slabs;
        sum_tiles_kernel<T, O, B><<<static_cast<unsigned>((units + kWarps - 1) / kWarps), 32 * kWarps, 0, stream>>>(p);
        SKM_LAUNCH_CHECK();
        join_tiles_kernel<T, O, B><<<dim3(static_cast<unsigned>((k + kJoinWarps - 1) / kJoinWarps), p.slabs), 32 * kJoinWarps, 0, stream>>>(p);
        SKM_LAUNCH_CHECK();
    };
    with_width(type, bytes, [&](auto value, auto width) {
        if (out_type == Type::f32) launch(value, float{}, width);
        else launch(value, value, width);   // (the gradient's own type)
    });
}

} // namespace rows
} // namespace skmb
