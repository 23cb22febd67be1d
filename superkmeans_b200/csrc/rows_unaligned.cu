// Rows whose address, pitch or length is no multiple of 16 bytes: odd widths, slices of wider rows.
//
// An output is contiguous and begins on 16 bytes, whatever the width of its rows: it is written as one sequence of 16-byte chunks, each from
// one row or from the end of one and the beginning of the next, and collected in pieces of the 8, 4 or 2 bytes that the rows' places allow.
// What a block needs to know of its rows (where they are, times what) is looked up once and kept in shared memory: with a look-up
// for every chunk, and one more for the row behind, the kernels were bound by whole-number instructions.
// Against chunks of that size for loads and stores alike (a pass, one B200): lookup of 862 587 rows of 154 fp32 with scales 172 -> 115 us,
// of 185 981 rows of 17 fp32 10.2 -> 7.0; 24 711 x 4 rows of 221 bf16 to their clusters and back 88 -> 67, 112 749 rows of 39 bf16 49 -> 33
// (two-byte pieces: eight loads for a chunk).  Cutting chunks out of aligned blocks, as load_window does, took 170, 8.2, 66 and 31.
// Sums along a row (dots) do take the row's own 16-byte chunks by load_window.
#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr int kThreads = 128;
constexpr int kAhead = 2;                                       // chunks of a thread that are loaded before the first is stored
constexpr int kMoveTurns = 4, kSumTurns = 2;                    // of them, in a block that moves rows or sums them
constexpr uint32_t kLeastRow = 32;                              // bytes
template <int TURNS>
constexpr uint32_t kBlockBytes = kThreads * kAhead * TURNS * 16;
template <int TURNS>
constexpr uint32_t kBlockRows = kBlockBytes<TURNS> / kLeastRow + 2;   // that it can touch

struct Flat {
    size_t rows, bytes;   // of the output
    Divisor row;          // bytes of a row
};
template <int TURNS>
Flat make_flat(size_t rows, size_t row_bytes) {
    return {rows, rows * row_bytes, make_divisor(row_bytes, row_bytes + kBlockBytes<TURNS>)};
}
template <int TURNS>
unsigned flat_blocks(const Flat& f) {
    return static_cast<unsigned>((f.bytes + kBlockBytes<TURNS> - 1) / kBlockBytes<TURNS>);
}

// A block's part of the output: from byte `begin` on, which is byte `off` of row row0; `rows` rows of it.
template <int TURNS>
struct Part {
    size_t begin, row0;
    uint32_t off, rows;

    __device__ __forceinline__ explicit Part(const Flat& f) {
        begin = static_cast<size_t>(blockIdx.x) * kBlockBytes<TURNS>;
        row0 = (begin >> 32) == 0 ? static_cast<uint32_t>(begin) / f.row.d : begin / f.row.d;
        off = static_cast<uint32_t>(begin - row0 * f.row.d);
        rows = static_cast<uint32_t>(min(static_cast<size_t>(divide(off + kBlockBytes<TURNS> - 1, f.row)) + 1, f.rows - row0));
    }
};

// A chunk: byte `at` of the output, in row `row` of the part from byte `col` on; `first` bytes are that row's, the rest the next one's.
struct Piece {
    size_t at;
    uint32_t row, col, first;
    bool has;

    template <int TURNS>
    __device__ __forceinline__ Piece(const Flat& f, const Part<TURNS>& part, uint32_t rel) {
        const uint32_t a = part.off + rel;
        row = divide(a, f.row);
        col = a - row * f.row.d;
        first = min(16u, f.row.d - col);
        at = part.begin + rel;
        has = at < f.bytes;
    }
};

// Where an output's row comes from, and times what; null: nowhere.
struct alignas(16) Source {
    const char* p;
    float factor;
};

template <typename T>
__device__ __forceinline__ void store_piece(char* out, const Flat& f, const Piece& p, const uint4& c) {
    if (p.at + 16 <= f.bytes) {
        *reinterpret_cast<uint4*>(out + p.at) = c;
    } else {   // the end of the output
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        T v[16 / sizeof(T)];
        memcpy(v, w, 16);
#pragma unroll
        for (uint32_t i = 0; i < 16 / sizeof(T); ++i)
            if (p.at + (i + 1) * sizeof(T) <= f.bytes) reinterpret_cast<T*>(out + p.at)[i] = v[i];
    }
}

// Which row an output's row is, if any, and times what.
struct ByIds {
    const void* ids;
    bool wide;
    uint32_t k;
    float scale;
    const float* row_scales;

    __device__ __forceinline__ bool at(size_t row, size_t& from, float& factor) const {
        const uint32_t id = load_id(ids, wide, row, k);
        from = id;
        factor = row_scales ? scale * __ldg(row_scales + row) : scale;
        return id < k;
    }
};
struct BySlot {
    Places places;
    uint32_t slots;
    const float* weights;

    __device__ __forceinline__ bool at(size_t slot, size_t& from, float& factor) const {
        if (slot >= min(__ldg(places.held), slots)) return false;
        const uint32_t pair = __ldg(places.order + slot);
        if (pair >= slots) return false;
        from = pair / static_cast<uint32_t>(places.m);
        factor = weights ? __ldg(weights + pair) : 1.f;
        return true;
    }
};

// The 16 bytes of a chunk out of one or two rows, W bytes at a time.
template <int W>
__device__ __forceinline__ uint4 collect(const Source& row, const Source& next, const Piece& piece) {
    const char *here = row.p + piece.col, *there = next.p - piece.first;
    const bool in_row = row.p != nullptr, in_next = next.p != nullptr;
    Chunk<W> w[16 / W];
#pragma unroll
    for (uint32_t i = 0; i < 16 / W; ++i) {
        const bool mine = i * W < piece.first;
        const char* p = mine ? here : there;
        w[i] = (mine ? in_row : in_next) ? __ldg(reinterpret_cast<const Chunk<W>*>(p + i * W)) : zero_chunk<W>();
    }
    uint4 c;
    memcpy(&c, w, 16);
    return c;
}

template <typename T, int W, bool SCALED, class Index>
__global__ void __launch_bounds__(kThreads) move_rows_kernel(const char* __restrict__ from, size_t pitch, const Index index, char* __restrict__ out, const Flat flat) {
    // looked up once for each row of the block's part (and nowhere for the one behind)
    __shared__ Source sources[kBlockRows<kMoveTurns> + 1];
    const Part<kMoveTurns> part(flat);
    for (uint32_t r = threadIdx.x; r <= part.rows; r += kThreads) {
        size_t row = 0;
        float f = 0.f;
        const bool there = r < part.rows && index.at(part.row0 + r, row, f);
        sources[r] = there ? Source{from + row * pitch, f} : Source{nullptr, 0.f};   // (zeros, whatever the factor of what is not there)
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t turn = 0; turn < kMoveTurns; ++turn) {
        uint4 c[kAhead];
        float f[kAhead], g[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const Piece p(flat, part, ((turn * kAhead + u) * kThreads + threadIdx.x) * 16);
            if (!p.has) continue;
            const Source row = sources[p.row], next = sources[min(p.row + 1, part.rows)];
            c[u] = collect<W>(row, next, p);
            f[u] = row.factor;
            g[u] = next.factor;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const Piece p(flat, part, ((turn * kAhead + u) * kThreads + threadIdx.x) * 16);
            if (!p.has) continue;
            if (SCALED) {
                Values<T, 16> v;
                v.from(c[u]);
#pragma unroll
                for (uint32_t i = 0; i < v.N; ++i) v.v[i] *= i * sizeof(T) < p.first ? f[u] : g[u];
                c[u] = v.to();
            }
            store_piece<T>(out, flat, p, c[u]);
        }
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) sum_rows_kernel(const char* __restrict__ y, size_t pitch, const Places places, const float* __restrict__ weights, char* __restrict__ out,
                                                            const Flat flat) {
    constexpr int ALL = kAhead * kSumTurns;
    __shared__ Source sources[kBlockRows<kSumTurns> + 1];
    const Part<kSumTurns> part(flat);
    const uint32_t m = static_cast<uint32_t>(places.m), slots = static_cast<uint32_t>(places.n) * m, held = min(__ldg(places.held), slots);
    Values<T, 16> sum[ALL];
#pragma unroll
    for (int u = 0; u < ALL; ++u)
#pragma unroll
        for (uint32_t i = 0; i < sum[u].N; ++i) sum[u].v[i] = 0.f;
    for (uint32_t j = 0; j < m; ++j) {
        __syncthreads();   // (the choice before is through)
        for (uint32_t r = threadIdx.x; r <= part.rows; r += kThreads) {
            const size_t pair = (part.row0 + r) * m + j;
            const uint32_t slot = r < part.rows ? __ldg(places.position + pair) : 0xffffffffu;
            const bool there = slot < held;
            // (a choice without a cluster adds nothing, whatever its weight)
            sources[r] = {there ? y + slot * pitch : nullptr, there ? weights ? __ldg(weights + pair) : 1.f : 0.f};
        }
        __syncthreads();
#pragma unroll
        for (int u0 = 0; u0 < ALL; u0 += kAhead) {
            uint4 c[kAhead];
            float f[kAhead], g[kAhead];
            uint32_t first[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const Piece p(flat, part, ((u0 + u) * kThreads + threadIdx.x) * 16);
                const Source row = p.has ? sources[p.row] : Source{nullptr, 0.f}, next = p.has ? sources[min(p.row + 1, part.rows)] : Source{nullptr, 0.f};
                c[u] = collect<W>(row, next, p);
                f[u] = row.factor;
                g[u] = next.factor;
                first[u] = p.first;
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                Values<T, 16> v;
                v.from(c[u]);
#pragma unroll
                for (uint32_t i = 0; i < v.N; ++i) sum[u0 + u].v[i] = fmaf(i * sizeof(T) < first[u] ? f[u] : g[u], v.v[i], sum[u0 + u].v[i]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < ALL; ++u) {
        const Piece p(flat, part, (u * kThreads + threadIdx.x) * 16);
        if (p.has) store_piece<T>(out, flat, p, sum[u].to());
    }
}

// The partner of each of a row's m pairs, if any.
struct TableRow {
    const void* ids;
    bool wide;
    uint32_t k;
    __device__ __forceinline__ bool at(size_t pair, size_t& row) const { return (row = load_id(ids, wide, pair, k)) < k; }
};
struct SlotRow {
    Places places;
    __device__ __forceinline__ bool at(size_t pair, size_t& row) const {
        const uint32_t slots = static_cast<uint32_t>(places.n * places.m);
        return (row = __ldg(places.position + pair)) < min(__ldg(places.held), slots);
    }
};

// out[pair] = scale * <a[row], b[partner of the pair]>, LANES lanes to a row
template <typename T, int LANES, class Partner>
__global__ void __launch_bounds__(kThreads) dots_kernel(const char* __restrict__ a, size_t pitch_a, const char* __restrict__ b, size_t pitch_b, const Partner partner, size_t n, size_t m,
                                                        uint32_t row_bytes, float scale, float* __restrict__ out) {
    const Lanes<LANES> lanes;
    const size_t row = static_cast<size_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
    if (row >= n) return;
    const uint32_t lane = lanes.lane;
    for (size_t j = 0; j < m; ++j) {
        size_t other;
        const bool there = partner.at(row * m + j, other);
        float dot = 0.f;
        if (there) {
#pragma unroll 2
            for (uint32_t col = lane * 16; col < row_bytes; col += LANES * 16) {
                const uint32_t valid = min(16u, row_bytes - col);
                Values<T, 16> x, z;
                x.from(load_window<T>(a + row * pitch_a + col, 0, valid));
                z.from(load_window<T>(b + other * pitch_b + col, 0, valid));
#pragma unroll
                for (uint32_t i = 0; i < x.N; ++i)
                    if ((i + 1) * sizeof(T) <= valid) dot = fmaf(x.v[i], z.v[i], dot);
            }
        }
        dot = lanes.sum(dot);
        if (lane == 0) out[row * m + j] = there ? scale * dot : 0.f;
    }
}

template <class F>
void with_type(Type type, F&& f) {
    if (type == Type::f32) f(float{});
    else if (type == Type::f16) f(__half{});
    else f(__nv_bfloat16{});
}

// f(value of the type, Width<W>) for pieces of W bytes
template <class F>
void with_pieces(Type type, int access, F&& f) {
    with_type(type, [&](auto value) {
        if (access >= 8) f(value, Width<8>{});
        else if (access == 4) f(value, Width<4>{});
        else if constexpr (sizeof(value) == 2) f(value, Width<2>{});
    });
}

template <class Index>
void launch_move(const Rows& from, Type type, size_t d, const Index& index, size_t rows, bool scale, void* out, cudaStream_t stream) {
    const size_t t = type_bytes(type), pitch = from.ld * t;
    const Flat flat = make_flat<kMoveTurns>(rows, d * t);
    with_pieces(type, access_bytes({address(from.p), pitch, d * t}), [&](auto value, auto width) {
        using T = decltype(value);
        constexpr int W = decltype(width)::bytes;
        auto* kernel = scale ? move_rows_kernel<T, W, true, Index> : move_rows_kernel<T, W, false, Index>;
        kernel<<<flat_blocks<kMoveTurns>(flat), kThreads, 0, stream>>>(static_cast<const char*>(from.p), pitch, index, static_cast<char*>(out), flat);
    });
    SKM_LAUNCH_CHECK();
}

template <class Partner>
void launch_dots(const Rows& a, const Rows& b, Type type, size_t d, const Partner& partner, size_t n, size_t m, float scale, float* out, cudaStream_t stream) {
    const size_t t = type_bytes(type);
    with_type(type, [&](auto value) {
        const bool narrow = d * t <= 16 * 16;
        const size_t of_block = kThreads / (narrow ? 8 : 32);
        auto* kernel = narrow ? dots_kernel<decltype(value), 8, Partner> : dots_kernel<decltype(value), 32, Partner>;
        kernel<<<static_cast<unsigned>((n + of_block - 1) / of_block), kThreads, 0, stream>>>(
            static_cast<const char*>(a.p), a.ld * t, static_cast<const char*>(b.p), b.ld * t, partner, n, m, static_cast<uint32_t>(d * t), scale, out);
    });
    SKM_LAUNCH_CHECK();
}

} // namespace

void launch_lookup_unaligned(const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, const float* row_scales, void* out, cudaStream_t stream) {
    launch_move(table, type, d, ByIds{ids.p, ids.wide, static_cast<uint32_t>(k), scale, row_scales}, n, row_scales || scale != 1.0f, out, stream);
}

void launch_lookup_scale_grad_unaligned(const Rows& grad, const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, float* out, cudaStream_t stream) {
    launch_dots(grad, table, type, d, TableRow{ids.p, ids.wide, static_cast<uint32_t>(k)}, n, 1, scale, out, stream);
}

void launch_to_clusters_unaligned(const Rows& x, Type type, size_t d, const Places& at, const float* weights, void* out, cudaStream_t stream) {
    launch_move(x, type, d, BySlot{at, static_cast<uint32_t>(at.n * at.m), weights}, at.n * at.m, weights != nullptr, out, stream);
}

void launch_from_clusters_unaligned(const Rows& y, Type type, size_t d, const Places& at, const float* weights, void* out, cudaStream_t stream) {
    const size_t t = type_bytes(type), pitch = y.ld * t;
    const Flat flat = make_flat<kSumTurns>(at.n, d * t);
    with_pieces(type, access_bytes({address(y.p), pitch, d * t}), [&](auto value, auto width) {
        sum_rows_kernel<decltype(value), decltype(width)::bytes><<<flat_blocks<kSumTurns>(flat), kThreads, 0, stream>>>(static_cast<const char*>(y.p), pitch, at, weights, static_cast<char*>(out), flat);
    });
    SKM_LAUNCH_CHECK();
}

void launch_weights_grad_unaligned(const Rows& grad, const Rows& y, Type type, size_t d, const Places& at, float* grad_weights, cudaStream_t stream) {
    launch_dots(grad, y, type, d, SlotRow{at}, at.n, at.m, 1.f, grad_weights, stream);
}

} // namespace rows
} // namespace skmb
