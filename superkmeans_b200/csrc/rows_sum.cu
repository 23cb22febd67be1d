// Gradient of a lookup: for every row of the table the sum of the gradients of the pairs that took it, scaled.
//
// The pairs are sorted by id (rows_group.cu) and cut into tiles of equal length, so that a row that half of the pairs took is no
// longer to sum than a thousand rows are.  A warp takes a tile and 32 chunks of its columns (eight lanes a tile where rows have no more
// than eight), reads the rows that the order names, eight ahead, and adds in fp32 registers; a run of equal ids that lies inside the
// tile goes straight to the output, the tile's first and last run, which may go on in the neighbours, into partial sums.  A second
// launch adds the partial sums of each id in the order of their tiles and writes the zeros of ids that nobody took.  Nothing depends on
// the order of atomics.
//
// No chain of sums in 32 bits is long, so that fp32 results keep their last places: eight rows are added to one another and then to the
// eights before (32 in a tile), partial sums eight at most, or four at a time and the fours in 64 bits.  A sum of any length is off by less than
// 50 roundings (of few pairs 80) of the sum of the magnitudes; as one chain of a tile's rows and one of the tiles it was off by hundreds.  A
// million positive normal values come out as if rounded once (rms 0.36 of 2^-24; 3.1 before).  Sums of eights in 64 bits too were 10 % slower.
//
// One B200, 500 000 x 1024 bf16 into 16 384 rows: the tiles 162 us, 1.07 GB at 6.6 TB/s (HBM; where runs begin is found for 32 pairs by
// a ballot: with a comparison for each pair the same took 263), the joins 10, the sort 34.
#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr int kWarps = 4;
constexpr uint32_t kAhead = 8;

struct SumParams {
    const void* grad;
    size_t pitch;
    const uint32_t* order;     // pairs by id
    const uint32_t* keys;      // their ids
    const uint32_t* offsets;   // k + 1
    const float* row_scales;
    float scale;
    uint32_t n, k, d;
    uint32_t row_bytes;
    uint32_t width;            // chunks to a row
    uint32_t slabs;            // of 32 chunks
    uint32_t tile;             // pairs to a tile
    uint32_t join_ids;         // ids to a warp of the second launch
    uint32_t apart;            // d, rounded up to whole chunks
    float* partials;           // per tile two rows `apart` from one another: the first run, and the last if it is another
    void* out;
};

// Sums of a chunk's values, and their stores: at `to` as they are or as the output's type.
template <typename T, int BYTES>
struct Sums {
    static constexpr int N = Values<T, BYTES>::N;
    float v[N];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
    }
    __device__ __forceinline__ void add(const Chunk<BYTES>& c) {
        Values<T, BYTES> x;
        x.from(c);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += x.v[i];
    }
    __device__ __forceinline__ void add(const Chunk<BYTES>& c, float f) {
        Values<T, BYTES> x;
        x.from(c);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = fmaf(f, x.v[i], v[i]);
    }
    __device__ __forceinline__ void add(const Sums& other) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += other.v[i];
    }
    // the first `count` of them
    template <typename O>
    __device__ __forceinline__ void store_some(O* to, float scale, uint32_t count) const {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i)
            if (i < count) {
                if constexpr (sizeof(O) == 4) to[i] = v[i] * scale;
                else reinterpret_cast<uint16_t*>(to)[i] = static_cast<uint16_t>(pair_from_float(v[i] * scale, 0.f, static_cast<const O*>(nullptr)));
            }
    }
    template <typename O>
    __device__ __forceinline__ void store(O* to, float scale) const {
        constexpr int ALL = N * static_cast<int>(sizeof(O)), EACH = ALL < 16 ? ALL : 16, PART = EACH / static_cast<int>(sizeof(O));
#pragma unroll
        for (int h = 0; h < ALL / EACH; ++h) {
            Values<O, EACH> x;
#pragma unroll
            for (int i = 0; i < PART; ++i) x.v[i] = v[h * PART + i] * scale;
            reinterpret_cast<Chunk<EACH>*>(to)[h] = x.to();
        }
    }
};

// A chunk of a row of the gradient, and the output's values that belong to it.  WINDOWS: rows that 16-byte accesses do not fit.
template <typename T, int BYTES, bool WINDOWS>
struct Lane {
    uint32_t bytes;   // of the chunk that are the row's

    __device__ __forceinline__ Lane(uint32_t row_bytes, uint32_t col) : bytes(WINDOWS ? min(16u, row_bytes - col * 16) : BYTES) {}
    __device__ __forceinline__ Chunk<BYTES> load(const char* p) const {
        if constexpr (WINDOWS) return load_window<T, true>(p, 0, bytes);
        else return load_now(reinterpret_cast<const Chunk<BYTES>*>(p));
    }
    template <typename O>
    __device__ __forceinline__ void store(const Sums<T, BYTES>& sum, O* to, float scale) const {
        if constexpr (WINDOWS) sum.template store_some<O>(to, scale, bytes / sizeof(T));
        else sum.template store<O>(to, scale);
    }
};

// SCALED: each pair with a factor of its own; otherwise the sums are scaled.  (Blocks to an SM: 500 000 x 1024 bf16 with factors 227 us where the
// compiler is told to fit five, 239 where it is not; without factors 213 and 229.  Windows, 112 749 x 39 bf16: 27.6 where told one, 30.2 where not.)
template <typename T, typename O, int BYTES, bool WINDOWS, bool SCALED, int LANES>
__global__ void __launch_bounds__(32 * kWarps, WINDOWS ? 1 : SCALED && LANES == 32 && BYTES == 16 ? 5 : 0) sum_tiles_kernel(const SumParams p) {
    wait_for_the_one_before();
    constexpr uint32_t AHEAD = kAhead;
    using S = Sums<T, BYTES>;
    const Lanes<LANES> lanes;
    const uint32_t lane = lanes.lane;
    const size_t unit = static_cast<size_t>(blockIdx.x) * (32 * kWarps / LANES) + threadIdx.x / LANES;
    const size_t tile = unit / p.slabs, begin = tile * p.tile;
    const uint32_t held = load_new(p.offsets + p.k);
    if (begin >= held) return;   // (pairs without an id come last)
    const uint32_t col = static_cast<uint32_t>(unit - tile * p.slabs) * LANES + lane;
    const bool mine = col < p.width;
    const uint32_t s0 = static_cast<uint32_t>(begin), s1 = min(s0 + p.tile, held);
    const size_t at = static_cast<size_t>(col) * S::N;
    float* first_part = p.partials + tile * 2 * p.apart + at;
    const Lane<T, BYTES, WINDOWS> chunk(p.row_bytes, mine ? col : 0);
    const char* grad = static_cast<const char*>(p.grad) + static_cast<size_t>(mine ? col : 0) * BYTES;
    const float scale = SCALED ? 1.f : p.scale;
    S sum;
    sum.clear();
    uint32_t now = load_new(p.keys + s0);
    bool first = true;
    for (uint32_t s = s0; s < s1; s += LANES) {
        // a lane's pair of the next ones, and where runs of equal ids begin
        const uint32_t my = s + lane;
        const uint32_t my_pair = my < s1 ? load_new(p.order + my) : 0u, my_key = my < s1 ? load_new(p.keys + my) : 0u;
        float my_factor = 0.f;
        if (SCALED && my < s1) my_factor = p.scale * load_now(p.row_scales + my_pair);
        const uint32_t above = lanes.from(my_key, (lane + LANES - 1) % LANES);
        const uint32_t begins = lanes.ballot(my < s1 && my_key != (lane == 0 ? now : above));
        const uint32_t count = min(static_cast<uint32_t>(LANES), s1 - s);
        for (uint32_t u0 = 0; u0 < count; u0 += AHEAD) {
            Chunk<BYTES> c[AHEAD];
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u) {
                const uint32_t pair = lanes.from(my_pair, u0 + u);   // (behind the last: row 0, which is not added)
                c[u] = chunk.load(grad + pair * p.pitch);
            }
            const uint32_t here = begins >> u0 & ((1u << AHEAD) - 1);
            S eight;
            eight.clear();
            if (here == 0 && u0 + AHEAD <= count) {
#pragma unroll
                for (uint32_t u = 0; u < AHEAD; ++u) {
                    if (SCALED) eight.add(c[u], lanes.from(my_factor, u0 + u));
                    else eight.add(c[u]);
                }
                sum.add(eight);
                continue;
            }
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u) {
                const float f = SCALED ? lanes.from(my_factor, u0 + u) : 1.f;
                if (here >> u & 1) {
                    sum.add(eight);
                    eight.clear();
                    if (mine) {
                        if (first) sum.template store<float>(first_part, scale);
                        else chunk.store(sum, static_cast<O*>(p.out) + static_cast<size_t>(now) * p.d + at, scale);
                    }
                    sum.clear();
                    first = false;
                    now = lanes.from(my_key, u0 + u);
                }
                if (u0 + u < count) {
                    if (SCALED) eight.add(c[u], f);
                    else eight.add(c[u]);
                }
            }
            sum.add(eight);
        }
    }
    if (mine) sum.template store<float>(first ? first_part : first_part + p.apart, scale);
}

// Partial sums are added four at a time, and the fours of ids that have many in 64 bits (there may be thousands, and a chain of so many in 32
// bits is off by many steps of the last place).
template <int N>
struct Total {
    double v[N];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.0;
    }
    template <class S>
    __device__ __forceinline__ S rounded() const {
        S sum;
#pragma unroll
        for (int i = 0; i < N; ++i) sum.v[i] = static_cast<float>(v[i]);
        return sum;
    }
};

// Up to 32 ids and 32 chunks to a warp; ids whose pairs fill many tiles are taken by all eight warps of a block together.
constexpr int kJoinWarps = 8;
constexpr uint32_t kLongRun = 8;   // tiles (300 000 x 16 bf16 by 5000 ids 36 us, with four tiles 50; with 32 1M x 64 bf16 by 1000 ids 65 us instead of 73, but in chains of 32)

template <typename T, typename O, int BYTES, bool WINDOWS>
__global__ void __launch_bounds__(32 * kJoinWarps, 4) join_tiles_kernel(const SumParams p) {
    wait_for_the_one_before();
    using S = Sums<T, BYTES>;
    __shared__ double parts[kJoinWarps][32][S::N + 1];
    __shared__ uint32_t long_ids[kJoinWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t block0 = blockIdx.x * (p.join_ids * kJoinWarps), id0 = block0 + warp * p.join_ids, col = blockIdx.y * 32 + lane;
    const bool mine = col < p.width;
    const size_t at = static_cast<size_t>(col) * S::N;
    O* out = static_cast<O*>(p.out) + at;
    const Lane<T, BYTES, WINDOWS> chunk(p.row_bytes, mine ? col : 0);
    // the tiles t0 .. t1 - 1 of this lane's id, and whether there is something to do: its sum is in the output already if its pairs
    // lie inside their tile, which ends where the pairs with an id end
    uint32_t begin = 0, t0 = 0, t1 = 0;
    bool todo = false;
    if (lane < p.join_ids && id0 + lane < p.k) {
        begin = load_new(p.offsets + id0 + lane);
        const uint32_t end = load_new(p.offsets + id0 + lane + 1), held = load_new(p.offsets + p.k);
        t0 = begin / p.tile;
        t1 = end > begin ? (end - 1) / p.tile + 1 : t0;
        todo = !(t1 == t0 + 1 && begin > t0 * p.tile && end < min(static_cast<size_t>(t1) * p.tile, static_cast<size_t>(held)));
    }
    auto add_tiles = [&](auto& sum, uint32_t from, uint32_t to, uint32_t first) {
        constexpr uint32_t AHEAD = 4;
        for (uint32_t t = from; t < to; t += AHEAD) {
            constexpr int EACH = S::N < 4 ? S::N : 4;   // floats of a load
            Values<float, EACH * 4> v[AHEAD][S::N / EACH];
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; ++u) {
                const size_t tile = t + u;
                const float* src = p.partials + (tile * 2 + (first > tile * p.tile ? 1 : 0)) * p.apart + at;
#pragma unroll
                for (int i = 0; i < S::N / EACH; ++i)
                    v[u][i].from(t + u < to && mine ? load_new(reinterpret_cast<const Chunk<EACH * 4>*>(src) + i) : zero_chunk<EACH * 4>());
            }
            if constexpr (std::is_same_v<std::decay_t<decltype(sum)>, S>) {
#pragma unroll
                for (uint32_t u = 0; u < AHEAD; ++u)
#pragma unroll
                    for (int i = 0; i < S::N; ++i) sum.v[i] += v[u][i / EACH].v[i % EACH];
            } else {
#pragma unroll
                for (int i = 0; i < S::N; ++i) {
                    auto of = [&](uint32_t u) { return v[u][i / EACH].v[i % EACH]; };
                    sum.v[i] += (of(0) + of(1)) + (of(2) + of(3));
                }
            }
        }
    };
    const uint32_t long_here = __ballot_sync(0xffffffffu, todo && t1 - t0 > kLongRun);
    for (uint32_t left = __ballot_sync(0xffffffffu, todo) & ~long_here; left; left &= left - 1) {
        const int l = __ffs(left) - 1;
        S sum;   // (two fours at most)
        sum.clear();
        add_tiles(sum, __shfl_sync(0xffffffffu, t0, l), __shfl_sync(0xffffffffu, t1, l), __shfl_sync(0xffffffffu, begin, l));
        if (mine) chunk.store(sum, out + static_cast<size_t>(id0 + l) * p.d, 1.f);
    }
    if (lane == 0) long_ids[warp] = long_here;
    if (!__syncthreads_or(long_here != 0)) return;
    for (uint32_t w = 0; w < kJoinWarps; ++w)
        for (uint32_t left = long_ids[w]; left; left &= left - 1) {   // (the same for the whole block)
            const uint32_t id = block0 + w * p.join_ids + __ffs(left) - 1;
            const uint32_t first = load_new(p.offsets + id), from0 = first / p.tile, to0 = (load_new(p.offsets + id + 1) - 1) / p.tile + 1;
            const uint32_t share = (to0 - from0 + kJoinWarps - 1) / kJoinWarps, from = min(from0 + warp * share, to0);
            Total<S::N> sum;
            sum.clear();
            add_tiles(sum, from, min(from + share, to0), first);
#pragma unroll
            for (int e = 0; e < S::N; ++e) parts[warp][lane][e] = sum.v[e];
            __syncthreads();
            if (warp == 0) {
#pragma unroll
                for (int q = 1; q < kJoinWarps; ++q)
#pragma unroll
                    for (int e = 0; e < S::N; ++e) sum.v[e] += parts[q][lane][e];
                if (mine) chunk.store(sum.template rounded<S>(), out + static_cast<size_t>(id) * p.d, 1.f);
            }
            __syncthreads();
        }
}

// Few pairs and few ids: one launch, a block for an id and 32 chunks.  Each of its warps looks for the id in its part of the pairs and adds
// the rows that it finds; their sums are added in the order of the warps.  Against sort, tiles and join (three launches, 16 us on the
// GPU and as much on the host) 2001 pairs of 130 halves with 300 ids take 4 us.
constexpr int kFewWarps = 8;
constexpr uint32_t kFewSumPairs = 4096;

template <typename T, typename O, int BYTES, bool WINDOWS>
__global__ void __launch_bounds__(32 * kFewWarps) sum_few_kernel(const SumParams p, const void* __restrict__ ids, bool wide) {
    wait_for_the_one_before();
    using S = Sums<T, BYTES>;
    constexpr uint32_t MOST = kFewSumPairs / kFewWarps;   // pairs of a warp
    __shared__ uint16_t found[kFewWarps][MOST];
    __shared__ float parts[kFewWarps][32][S::N + 1];
    __shared__ uint32_t counts[kFewWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, id = blockIdx.x, col = blockIdx.y * 32 + lane;
    const bool mine = col < p.width;
    const uint32_t share = (p.n + 32 * kFewWarps - 1) / (32 * kFewWarps) * 32, begin = min(warp * share, p.n), end = min(begin + share, p.n);
    uint32_t count = 0;
    constexpr int LOOK = 8;
    for (uint32_t s = begin; s < end; s += 32 * LOOK) {
        uint32_t v[LOOK];
#pragma unroll
        for (int u = 0; u < LOOK; ++u) v[u] = s + u * 32 + lane < end ? load_id(ids, wide, s + u * 32 + lane, p.k) : p.k;
#pragma unroll
        for (int u = 0; u < LOOK; ++u) {
            const uint32_t same = __ballot_sync(0xffffffffu, v[u] == id);
            if (v[u] == id) found[warp][count + __popc(same & ((1u << lane) - 1u))] = static_cast<uint16_t>(s + u * 32 + lane);
            count += __popc(same);
        }
    }
    __syncwarp();
    S sum;
    sum.clear();
    const char* grad = static_cast<const char*>(p.grad) + static_cast<size_t>(mine ? col : 0) * BYTES;
    const Lane<T, BYTES, WINDOWS> chunk(p.row_bytes, mine ? col : 0);
    for (uint32_t s = 0; s < count; s += kAhead) {
        Chunk<BYTES> c[kAhead];
        float f[kAhead];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
            if (s + u < count) {
                const uint32_t pair = found[warp][s + u];
                c[u] = chunk.load(grad + pair * p.pitch);
                f[u] = p.row_scales ? p.scale * load_now(p.row_scales + pair) : p.scale;
            }
        S eight;
        eight.clear();
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
            if (s + u < count) eight.add(c[u], f[u]);
        sum.add(eight);
    }
    if (lane == 0) counts[warp] = count;
    if (count != 0)
#pragma unroll
        for (int e = 0; e < S::N; ++e) parts[warp][lane][e] = sum.v[e];
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < kFewWarps; ++w)
        if (counts[w] != 0)
#pragma unroll
            for (int e = 0; e < S::N; ++e) sum.v[e] += parts[w][lane][e];
    if (mine) chunk.store(sum, static_cast<O*>(p.out) + static_cast<size_t>(id) * p.d + static_cast<size_t>(col) * S::N, 1.f);
}

// (the width of an access is not known where the workspace is sized: it is taken for 16 bytes, and a few more blocks do no harm.  300 pairs of 64 bf16
// with 10 ids 3.1 us, by tiles 7.8; 4096 of 768 with 300 12.3 and 14.4; with 4000 ids and six slabs, which the limit keeps out, 70 and 21.  All 4096 of one
// id, which the rule cannot know, 59 and 17.)
bool few(size_t n, size_t k, size_t d, Type type) { return n <= kFewSumPairs && k * ((d * type_bytes(type) + 511) / 512) <= 4096; }

// Pairs to a tile: enough tiles to fill the chip several times over (148 SMs, 16 warps each), and no shorter than it takes to keep the
// partial sums' traffic below the rows'.  Of narrow rows, which have eight lanes to a tile, twice as many tiles: 2M x 3 fp32 by 1000 ids 83 us (with as many
// as of wide rows 104, with four times as many 78), 1M x 64 bf16 by 300, half of them one's, 166 (124 and 326: more partial sums to join).
uint32_t tile_pairs(size_t n, size_t slabs, bool narrow) {
    uint32_t tile = 256;
    while (tile > 16 && (n + tile - 1) / tile * slabs < 148 * (narrow ? 64 : 32)) tile /= 2;
    return tile;
}

// (a chunk is at most 16 bytes: with narrower ones there are more slabs, and tiles no shorter)
size_t slabs_of(size_t d, Type type, int bytes) { return ((d * type_bytes(type) + bytes - 1) / bytes + 31) / 32; }

uint32_t tile_pairs(size_t n, size_t d, Type type) { return tile_pairs(n, slabs_of(d, type, 16), d * type_bytes(type) <= 8 * 16); }

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t whole_chunks(size_t d) { return (d + 7) / 8 * 8; }

} // namespace

size_t lookup_grad_workspace_bytes(size_t n, size_t k, size_t d, Type type) {
    if (few(n, k, d, type)) return 0;
    const size_t tile = tile_pairs(n, d, type), tiles = (n + tile - 1) / tile;
    return rounded(n * 4) * 2 + rounded((k + 1) * 4) + rounded(tiles * 2 * whole_chunks(d) * 4) + rounded(group_workspace_bytes(n, k));
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
    const bool is_few = few(n, k, d, type);
    size_t tiles = 0;
    if (!is_few) {
        uint32_t* order = reinterpret_cast<uint32_t*>(take(n * 4));
        uint32_t* keys = reinterpret_cast<uint32_t*>(take(n * 4));
        uint32_t* offsets = reinterpret_cast<uint32_t*>(take((k + 1) * 4));
        p.tile = tile_pairs(n, d, type);
        tiles = (n + p.tile - 1) / p.tile;
        p.partials = reinterpret_cast<float*>(take(tiles * 2 * whole_chunks(d) * 4));
        launch_group(ids, n, k, order, nullptr, keys, offsets, at, stream);
        p.order = order;
        p.keys = keys;
        p.offsets = offsets;
    }
    p.grad = grad.p;
    p.pitch = grad.ld * t;
    p.row_scales = row_scales;
    p.scale = scale;
    p.n = static_cast<uint32_t>(n);
    p.k = static_cast<uint32_t>(k);
    p.d = static_cast<uint32_t>(d);
    p.row_bytes = static_cast<uint32_t>(d * t);
    p.apart = static_cast<uint32_t>(whole_chunks(d));
    p.out = out;
    // (the output's chunks have as many values as the input's, and are stored 16 bytes at a time)
    const size_t ot = type_bytes(out_type);
    const int bytes = access_bytes({address(grad.p), p.pitch, d * t, address(out) * t / ot});
    const bool windows = use_windows(bytes, d * t);
    auto launch = [&](auto value, auto result, auto width, auto in_windows) {
        using T = decltype(value);
        using O = decltype(result);
        constexpr int B = decltype(width)::bytes;
        constexpr bool W = decltype(in_windows)::value;
        p.width = static_cast<uint32_t>((d * t + B - 1) / B);
        const uint32_t lanes = p.width <= 8 ? 8 : 32;
        p.slabs = (p.width + 31) / 32;   // (one, where the lanes are eight)
        if (is_few) {
            launch_after(sum_few_kernel<T, O, B, W>, dim3(static_cast<unsigned>(k), p.slabs), 32 * kFewWarps, 0, stream, p, ids.p, ids.wide);
            return;
        }
        const size_t units = tiles * p.slabs;
        auto* kernel = lanes == 8 ? row_scales ? sum_tiles_kernel<T, O, B, W, true, 8> : sum_tiles_kernel<T, O, B, W, false, 8>
                                  : row_scales ? sum_tiles_kernel<T, O, B, W, true, 32> : sum_tiles_kernel<T, O, B, W, false, 32>;
        const size_t of_block = 32 * kWarps / lanes;
        launch_after(kernel, dim3(static_cast<unsigned>((units + of_block - 1) / of_block)), 32 * kWarps, 0, stream, p);
        // a warp takes its ids one after the other: few, as long as there are warps for them (200 000 x 32 bf16 by 65 536 ids: 16 a warp 67 us, one
        // 77, 32 71; 1M x 64 by 300: one 77, four 113)
        p.join_ids = 1;
        while (p.join_ids < 32 && k * p.slabs > static_cast<size_t>(p.join_ids) * 148 * 32) p.join_ids *= 2;
        const size_t ids_of_block = static_cast<size_t>(p.join_ids) * kJoinWarps;
        launch_after(join_tiles_kernel<T, O, B, W>, dim3(static_cast<unsigned>((k + ids_of_block - 1) / ids_of_block), p.slabs), 32 * kJoinWarps, 0, stream, p);
    };
    auto of_type = [&](auto value, auto width, auto in_windows) {
        if (out_type == Type::f32) launch(value, float{}, width, in_windows);
        else launch(value, value, width, in_windows);   // (the gradient's own type)
    };
    with_width(type, windows ? 16 : bytes, [&](auto value, auto width) {
        if constexpr (decltype(width)::bytes == 16) {
            if (windows) return of_type(value, width, std::true_type{});
        }
        of_type(value, width, std::false_type{});
    });
}

} // namespace rows
} // namespace skmb
