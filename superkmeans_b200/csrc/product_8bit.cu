// Rows in 8 bits with a scale each, and their product with a matrix in 8 bits with a scale for each of its rows, on the tensor cores:
// out[i][c] = x_scale[i] * w_scale[c] * sum_j x[i][j] w[c][j].  The sums are whole numbers in 32 bits, hence exact however they are
// split; a result is rounded when its sum becomes a float, at each of the two scales, and once more to the output's type.
//
// tcgen05.mma of kind::i8, in two kernels.  Few rows: the matrix's rows ("channels") are the 128 lanes of the accumulator, the rows of x
// ("rows") its columns, so that the accumulator is as narrow as there are rows; one row of 768 by 16 384 channels takes 5.4 us.  Many:
// pairs of CTAs, below.
#include <atomic>
#include <map>
#include <mutex>
#include <string>

#include "rows_access.cuh"
#include "tc_ptx.cuh"
#include "kernels_tc.cuh"

namespace skmb {
namespace rows {

using namespace tc;

namespace {

// ---------------------------------------------------------------------------------------------- rows to 8 bits

// Magnitudes as whole numbers (a NaN is above infinity): the largest of a chunk's values and `most`.  Halves are compared two at a time,
// as what they are stored as.
template <typename T, int BYTES>
struct Largest {
    uint32_t most = 0;   // halves: two of them

    __device__ __forceinline__ void look(const Chunk<BYTES>& c) {
        if constexpr (BYTES == 2) {
            most = max(most, static_cast<uint32_t>(c) & 0x7fffu);
        } else {
            uint32_t w[BYTES / 4];
            memcpy(w, &c, BYTES);
#pragma unroll
            for (int i = 0; i < BYTES / 4; ++i) most = sizeof(T) == 4 ? max(most, w[i] & 0x7fffffffu) : __vmaxu2(most, w[i] & 0x7fff7fffu);
        }
    }
    // as a float's bits
    __device__ __forceinline__ uint32_t bits() const {
        if constexpr (sizeof(T) == 4) return most;
        else return __float_as_uint(pair_to_float(max(most & 0xffffu, most >> 16), static_cast<const T*>(nullptr)).x);
    }
};

// LANES threads to a row, of which each keeps HELD chunks in registers between finding the largest value and dividing by it (the rest of
// longer rows is read twice), while the next row's are on their way: as many blocks as are resident, in turn over the rows.
// Rounding is an addition to 1.5 * 2^23, which leaves the whole number in the low bits (its low byte is q).
template <typename T, int BYTES, bool WINDOWS, int LANES, int HELD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, size_t pitch, size_t n, uint32_t row_bytes, int8_t* __restrict__ q, size_t ldq,
                                                            float* __restrict__ scales) {
    wait_for_the_one_before();
    using V = Values<T, BYTES>;
    const size_t step = static_cast<size_t>(gridDim.x) * (256 / LANES);
    const uint32_t lane = threadIdx.x % LANES;
    const uint32_t width = (row_bytes + BYTES - 1) / BYTES;
    // chunk c of a row: zeros behind the row
    auto load = [&](size_t row, uint32_t c) {
        const char* p = static_cast<const char*>(x) + row * pitch + static_cast<size_t>(c) * BYTES;
        if constexpr (WINDOWS) {
            const uint32_t valid = min(16u, row_bytes - c * 16);
            const uint4 w = load_window<T, true>(p, 0, valid);
            uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) r[i] = valid >= 4 * i + 4 ? r[i] : valid <= 4 * i ? 0u : r[i] & 0xffffu;
            return make_uint4(r[0], r[1], r[2], r[3]);
        } else {
            return load_now(reinterpret_cast<const Chunk<BYTES>*>(p));
        }
    };
    Chunk<BYTES> held[HELD], next[HELD];
    auto fetch = [&](size_t row) {
        const size_t from = row < n ? row : 0;   // (behind the last row: the first, for nothing)
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (h * LANES < width) next[h] = lane + h * LANES < width ? load(from, lane + h * LANES) : zero_chunk<BYTES>();
    };
    size_t row = static_cast<size_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    fetch(row);
    // (whole blocks, and with them the warps of the shuffles, take the same number of turns)
    for (size_t turn = static_cast<size_t>(blockIdx.x) * (256 / LANES); turn < n; turn += step, row += step) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) held[h] = next[h];
        fetch(row + step);
        const bool valid = row < n;
        const size_t from = valid ? row : 0;
        Largest<T, BYTES> largest_of;
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (h * LANES < width) largest_of.look(held[h]);
        for (uint32_t c = lane + HELD * LANES; c < width; c += LANES) largest_of.look(load(from, c));
        uint32_t most = largest_of.bits();
#pragma unroll
        for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        if constexpr (LANES > 32) {
            __shared__ uint32_t of_warp[8];
            __syncthreads();   // (the turn before has read them)
            if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 8; ++w) most = max(most, of_warp[w]);
        }
        if (!valid) continue;
        const bool finite = most < 0x7f800000u, some = finite && most != 0;
        const float largest = __uint_as_float(most);
        // 127 / largest is a float for all but the smallest, which are taken 2^100 times as large
        const float up = largest < 0x1p-100f ? 0x1p100f : 1.0f;
        const float inverse = some ? __fdiv_rn(127.0f, largest * up) : 0.0f;
        const bool plain = some && up == 1.0f;
        if (lane == 0) scales[row] = finite ? __fdiv_rn(largest, 127.0f) : __uint_as_float(0x7fc00000u);
        int8_t* to = q + row * ldq;
        // (the product is rounded before the sum: as operations on pairs, mul2 and add2, it was not, and values at a half went the other way)
        auto whole_of = [&](float w) { return __float_as_uint(__fadd_rn(__fmul_rn(w, inverse), 12582912.0f)); };
        auto put = [&](const Chunk<BYTES>& chunk, uint32_t at) {
            V w;
            w.from(chunk);
            if (!plain) {
#pragma unroll
                for (int i = 0; i < V::N; ++i) w.v[i] = some ? w.v[i] * up : 0.0f;   // (no number times zero is none)
            }
            if constexpr (V::N == 1) {
                to[at] = static_cast<int8_t>(whole_of(w.v[0]));
            } else {
                uint32_t b[V::N];
#pragma unroll
                for (int i = 0; i < V::N; ++i) b[i] = whole_of(w.v[i]);
                Chunk<V::N> packed;
                if constexpr (V::N == 2) packed = static_cast<uint16_t>(__byte_perm(b[0], b[1], 0x0040));
                else {
                    uint32_t words[V::N / 4];
#pragma unroll
                    for (int i = 0; i < V::N / 4; ++i) words[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
                    memcpy(&packed, words, V::N);
                }
                if (WINDOWS && (at + 1) * 16 > row_bytes) {   // (what is behind the row is not written)
#pragma unroll
                    for (uint32_t i = 0; i < V::N; ++i)
                        if (at * 16 + (i + 1) * sizeof(T) <= row_bytes) to[at * V::N + i] = static_cast<int8_t>(b[i]);
                } else {
                    *reinterpret_cast<Chunk<V::N>*>(to + at * V::N) = packed;
                }
            }
        };
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (lane + h * LANES < width) put(held[h], lane + h * LANES);
        for (uint32_t c = lane + HELD * LANES; c < width; c += LANES) put(load(from, c), c);
    }
}

// Rows with a pitch that TMA takes (zeros behind d).
__global__ void __launch_bounds__(256) pad_bytes_kernel(const int8_t* __restrict__ in, size_t ld, size_t n, uint32_t d, uint32_t pitch, int8_t* __restrict__ out) {
    wait_for_the_one_before();
    const size_t row = static_cast<size_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (row >= n) return;
    for (uint32_t j = threadIdx.x & 31; j < pitch / 4; j += 32) {
        uint32_t v = 0;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (4 * j + e < d) v |= load_now(reinterpret_cast<const uint8_t*>(in) + row * ld + 4 * j + e) << (8 * e);
        *reinterpret_cast<uint32_t*>(out + row * pitch + 4 * j) = v;
    }
}

// ---------------------------------------------------------------------------------------------- the product
constexpr int P_THREADS = 128;
constexpr int P_STAGES = 4;
constexpr uint32_t P_CHANNELS = 128;
constexpr uint32_t P_DEPTH = 128;                          // columns of a stage, one 128-byte swizzle
constexpr uint32_t P_W_BYTES = P_CHANNELS * P_DEPTH;

// A tile of rows: row0 .. row1 - 1 of a group; groups and groups + 1 stand for rows that belong to none.
struct RowTile {
    uint32_t row0, row1, group;
};

__device__ __forceinline__ RowTile load_tile(const RowTile* p) { return {load_new(&p->row0), load_new(&p->row1), load_new(&p->group)}; }

struct ProductMaps {
    CUtensorMap w, x;
    CUtensorMap out;   // (where lanes are rows)
};

struct ProductParams {
    const float* x_scales;
    const float* w_scales;
    void* out;
    uint32_t n, m, depth_blocks;
    uint32_t channel_tiles;
    uint32_t groups;             // 0: none
    const RowTile* tiles;        // with groups
    const uint32_t* n_tiles;     // that belong to a group, and all
    uint32_t* given_up;          // the launch whose wait ran out last
    uint32_t launch;             // this one: no two have the same number, but for the replays of a graph
    int* told;                   // in host memory
    long long wait_limit;
    uint32_t producer_stop;
};

// A bounded wait.  One that runs out ends the others of its launch, and those only: what runs beside it on another stream, or after it
// before anybody was told, is a launch of its own.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, const ProductParams& p) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    uint32_t spins = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++spins & 1023u) == 0) {
            volatile uint32_t* given_up = p.given_up;
            if (*given_up == p.launch) return false;
            if (clock64() - t0 > p.wait_limit) {
                *given_up = p.launch;
                return false;
            }
        }
    }
    return true;
}
// A replay of a graph has the number of the one before: what that one may have left is cleared by a thread that has nothing else to do, while the first waits begin
// (a wait looks at it after a thousand polls, some milliseconds).
__device__ __forceinline__ void forget_the_replay_before(const ProductParams& p) {
    volatile uint32_t* given_up = p.given_up;
    if (blockIdx.x == 0 && *given_up == p.launch) *given_up = 0;
}

template <int ROWS>
struct ProductControl {
    uint64_t full[P_STAGES];
    uint64_t empty[P_STAGES];
    uint64_t done;
    uint32_t tmem_base;
    alignas(16) float x_scales[ROWS];
};
template <int ROWS>
constexpr uint32_t kStageBytes = P_W_BYTES + ROWS * P_DEPTH;
template <int ROWS>
constexpr uint32_t kProductSmem = P_STAGES * kStageBytes<ROWS> + sizeof(ProductControl<ROWS>) + 1024;

__device__ __forceinline__ void store_result(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_result(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_result(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float low_of(uint64_t p) { return __uint_as_float(static_cast<uint32_t>(p)); }
__device__ __forceinline__ float high_of(uint64_t p) { return __uint_as_float(static_cast<uint32_t>(p >> 32)); }

// 32 sums times the scales of their columns, and the lane's.
__device__ __forceinline__ void scale_columns(const uint32_t (&r)[32], const float* scales, uint64_t lane_scale2, uint64_t (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(scales + 2 * j);
        v[j] = mul2(mul2(pack2(__int2float_rn(static_cast<int>(r[2 * j])), __int2float_rn(static_cast<int>(r[2 * j + 1]))), s.x), lane_scale2);
        v[j + 1] = mul2(mul2(pack2(__int2float_rn(static_cast<int>(r[2 * j + 2])), __int2float_rn(static_cast<int>(r[2 * j + 3]))), s.y), lane_scale2);
    }
}

// store(c, v) for each 32 of a lane's `count` columns in tensor memory; the next 32 are on their way meanwhile.
template <int MOST, class F>
__device__ __forceinline__ void each_32_columns(uint32_t taddr, uint32_t count, const float* scales, float lane_scale, F&& store) {
    if (count == 0) return;
    const uint64_t lane_scale2 = pack2(lane_scale, lane_scale);
    uint32_t a[32], b[32];
    uint64_t v[16];
    tmem_ld32_issue(taddr, a);
#pragma unroll
    for (uint32_t c = 0; c < MOST; c += 64) {
        if (c >= count) break;
        tmem_ld_wait(a);
        const bool second = c + 32 < MOST && c + 32 < count;
        if (second) tmem_ld32_issue(taddr + c + 32, b);
        scale_columns(a, scales + c, lane_scale2, v);
        store(c, v);
        if (second) {
            tmem_ld_wait(b);
            if (c + 64 < MOST && c + 64 < count) tmem_ld32_issue(taddr + c + 64, a);
            scale_columns(b, scales + c + 32, lane_scale2, v);
            store(c + 32, v);
        }
    }
}

__device__ __forceinline__ void store_32_bytes(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// 32 results of one row, of which `left` are to be stored (a multiple of 32 bytes).
template <typename O>
__device__ __forceinline__ void store_along_row(O* to, const uint64_t (&v)[16], uint32_t left) {
    constexpr uint32_t PAIRS = sizeof(O) == 2 ? 8 : 4;   // in 32 bytes
#pragma unroll
    for (uint32_t j = 0; j < 16; j += PAIRS)
        if (2 * j < left) {
            uint32_t w[8];
#pragma unroll
            for (uint32_t e = 0; e < PAIRS; ++e) {
                if constexpr (sizeof(O) == 2) w[e] = pair_from_float(low_of(v[j + e]), high_of(v[j + e]), static_cast<const O*>(nullptr));
                else {
                    w[2 * e] = static_cast<uint32_t>(v[j + e]);
                    w[2 * e + 1] = static_cast<uint32_t>(v[j + e] >> 32);
                }
            }
            store_32_bytes(to + 2 * j, w);
        }
}

// Results of 32 rows for the channel of each lane, of which `left` rows are to be stored.
template <typename O>
__device__ __forceinline__ void store_across_rows(O* out, uint32_t m, uint32_t channel, bool has_channel, uint32_t lane, const uint64_t (&v)[16], uint32_t left, bool packed) {
    auto all = [&](auto whole) {
        if constexpr (sizeof(O) == 2) {
            if (packed) {
                // two lanes swap halves, so that each stores two channels of one row
                const uint32_t odd = lane & 1, pick = odd ? 0x3276 : 0x5410;
                O* to = out + static_cast<size_t>(odd) * m + (channel - odd);
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    const uint32_t mine = pair_from_float(low_of(v[j]), high_of(v[j]), static_cast<const O*>(nullptr)), other = __shfl_xor_sync(0xffffffffu, mine, 1);
                    if ((whole.value || 2 * j + odd < left) && has_channel) *reinterpret_cast<uint32_t*>(to + static_cast<size_t>(2 * j) * m) = __byte_perm(mine, other, pick);
                }
                return;
            }
        }
        O* to = out + channel;
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) {
            if ((whole.value || 2 * j < left) && has_channel) store_result(to + static_cast<size_t>(2 * j) * m, low_of(v[j]));
            if ((whole.value || 2 * j + 1 < left) && has_channel) store_result(to + static_cast<size_t>(2 * j + 1) * m, high_of(v[j]));
        }
    };
    if (left >= 32) all(std::true_type{});
    else all(std::false_type{});
}

// One tile of 128 channels x ROWS rows per cluster; the CTAs of a cluster share the depth and add their sums at the end, each for its
// part of the rows, out of one another's shared memory.
template <int ROWS, typename O>
__global__ void __launch_bounds__(P_THREADS) product_kernel(const __grid_constant__ ProductMaps maps, const ProductParams p) {
    wait_for_the_one_before();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t* smem = smem_raw + pad;
    const uint32_t smem_base = raw_addr + pad;
    auto* ctrl = reinterpret_cast<ProductControl<ROWS>*>(smem + P_STAGES * kStageBytes<ROWS>);
    constexpr uint32_t COLS = ROWS < 32 ? 32 : ROWS;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = cluster_size(), rank = cluster_rank();

    const uint32_t tile = blockIdx.x / split, channel_tile = tile % p.channel_tiles, row_tile = tile / p.channel_tiles;
    RowTile t;
    if (p.groups) {
        if (row_tile >= load_new(p.n_tiles + 1)) return;   // (the whole cluster)
        t = load_tile(p.tiles + row_tile);
    } else {
        t = {row_tile * ROWS, min(row_tile * ROWS + ROWS, p.n), 0};
    }
    const uint32_t channel = channel_tile * P_CHANNELS + threadIdx.x;
    O* out = static_cast<O*>(p.out);
    if (p.groups && t.group >= p.groups) {   // rows of no group
        if (rank == 0 && channel < p.m)
            for (uint32_t r = t.row0; r < t.row1; ++r) store_result(out + static_cast<size_t>(r) * p.m + channel, 0.f);
        return;
    }

    if (threadIdx.x == 0) {
        tma_prefetch_map(&maps.w);
        tma_prefetch_map(&maps.x);
        for (int s = 0; s < P_STAGES; ++s) {
            mbar_init(&ctrl->full[s], 1);
            mbar_init(&ctrl->empty[s], 1);
        }
        mbar_init(&ctrl->done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 0) tmem_alloc(&ctrl->tmem_base, COLS);
    for (uint32_t r = threadIdx.x; r < ROWS; r += P_THREADS) ctrl->x_scales[r] = t.row0 + r < t.row1 ? load_new(p.x_scales + t.row0 + r) : 0.f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = ctrl->tmem_base;
    const uint32_t k0 = p.depth_blocks * rank / split, k1 = p.depth_blocks * (rank + 1) / split;

    bool ok = true;
    if (threadIdx.x == 0) {
        const int w_row = static_cast<int>(t.group * p.m + channel_tile * P_CHANNELS), x_row = static_cast<int>(t.row0);
        for (uint32_t k = k0, it = 0; k < k1; ++k, ++it) {
            const uint32_t s = it % P_STAGES, ph = (it / P_STAGES) & 1u;
            if ((p.producer_stop != 0 && it >= p.producer_stop) || !wait_for(&ctrl->empty[s], ph ^ 1u, p)) {
                ok = false;
                break;
            }
            const uint32_t st = smem_base + s * kStageBytes<ROWS>;
            mbar_arrive_expect_tx(&ctrl->full[s], kStageBytes<ROWS>);
            tma_load_2d(st, &maps.w, &ctrl->full[s], static_cast<int>(k * P_DEPTH), w_row);
            tma_load_2d(st + P_W_BYTES, &maps.x, &ctrl->full[s], static_cast<int>(k * P_DEPTH), x_row);
        }
    } else if (threadIdx.x == 32) {
        constexpr uint32_t idesc = make_idesc_i8(P_CHANNELS, ROWS);
        for (uint32_t k = k0, it = 0; k < k1; ++k, ++it) {
            const uint32_t s = it % P_STAGES, ph = (it / P_STAGES) & 1u;
            if (!wait_for(&ctrl->full[s], ph, p)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t st = smem_base + s * kStageBytes<ROWS>;
#pragma unroll
            for (uint32_t kk = 0; kk < P_DEPTH / 32; ++kk) umma_i8(tmem_base, make_desc_128(st + kk * 32), make_desc_128(st + P_W_BYTES + kk * 32), it != 0 || kk != 0 ? 1u : 0u, idesc);
            umma_commit(&ctrl->empty[s]);
        }
        if (ok) umma_commit(&ctrl->done);
    } else if (threadIdx.x == P_THREADS - 1) {
        forget_the_replay_before(p);
    }
    __syncwarp();
    const bool summed = __all_sync(0xffffffffu, wait_for(&ctrl->done, 0, p));
    if (!summed && lane == 0) *reinterpret_cast<volatile int*>(p.told) = 43;
    if (!ok) {
        // a millisecond for the copies that are in flight before the block's memory is let go
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
        }
    }
    __syncwarp();
    tc_fence_after();

    const bool has_channel = channel < p.m;
    const float w_scale = has_channel ? load_new(p.w_scales + static_cast<size_t>(t.group) * p.m + channel) : 0.f;
    const uint32_t taddr = tmem_base + (warp * 32 << 16), count = t.row1 - t.row0;
    out += static_cast<size_t>(t.row0) * p.m;
    if (split == 1) {
        if (summed) {
            if constexpr (ROWS >= 32) {
                const bool packed = p.m % 2 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0;
                each_32_columns<ROWS>(taddr, count, ctrl->x_scales, w_scale,
                                      [&](uint32_t c, const uint64_t (&v)[16]) { store_across_rows(out + static_cast<size_t>(c) * p.m, p.m, channel, has_channel, lane, v, count - c, packed); });
            } else {
                uint32_t r[16];
                tmem_ld16(taddr, r);
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j)
                    if (j < count && has_channel) store_result(out + static_cast<size_t>(j) * p.m + channel, __int2float_rn(static_cast<int>(r[j])) * ctrl->x_scales[j] * w_scale);
            }
        }
    } else {
        // the rows' sums into this CTA's shared memory (the stages are through), 128 channels to a row
        int* sums = reinterpret_cast<int*>(smem);
        if (summed)
#pragma unroll 1
            for (uint32_t c = 0; c < count; c += 16) {
                uint32_t r[16];
                tmem_ld16(taddr + c, r);
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) sums[(c + j) * P_CHANNELS + threadIdx.x] = static_cast<int>(r[j]);
            }
        cluster_sync();
        if (summed) {
            constexpr uint32_t AHEAD = 4;
            for (uint32_t r0 = rank; r0 < count; r0 += AHEAD * split) {
                int sum[AHEAD] = {};
                for (uint32_t q = 0; q < split; ++q) {
                    const uint32_t from = cluster_address(sums + threadIdx.x, q);
                    int v[AHEAD];
#pragma unroll
                    for (uint32_t e = 0; e < AHEAD; ++e) v[e] = load_cluster(from + min(r0 + e * split, count - 1) * (P_CHANNELS * 4));
#pragma unroll
                    for (uint32_t e = 0; e < AHEAD; ++e) sum[e] += v[e];
                }
#pragma unroll
                for (uint32_t e = 0; e < AHEAD; ++e) {
                    const uint32_t r = r0 + e * split;
                    if (r < count && has_channel) store_result(out + static_cast<size_t>(r) * p.m + channel, __int2float_rn(sum[e]) * ctrl->x_scales[r] * w_scale);
                }
            }
        }
        cluster_sync();   // nobody reads this CTA's sums any more
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem_base, COLS);
}

// ---- many rows: persistent pairs of CTAs on tiles of 256 lanes x COLS columns, each CTA with its 128 lanes, half of the columns as operand
// and all of them in its accumulator:
//   warp 0       TMA producer
//   warp 1       MMA issuer (the leader's)
//   warps 4-11   epilogue: 32 lanes and half of the columns each, out of one accumulator while the other is filled
// Where rows of the result begin on 32 bytes, the lanes are rows of x: a thread then holds 128 neighbouring results of a row and stores
// 32 bytes at a time, or whole lines by way of shared memory.  Elsewhere, and where the tile is narrow because the groups are small, the
// lanes are channels, and the 32 lanes of a warp store 32 neighbouring results of a row.
//
// One B200: 32 768 x 1024 by 10 000 channels to bf16 262 us in a short run, 2560 T/s, the tensor pipe 70 % busy, and 310 in a long one, 2170 T/s.  In
// short runs: by 10 001 channels 302; to fp32 355; depth 128: 112; depth 4096: 855, 3140 T/s; the single-CTA kernel 1269.  Power is the bound:
// the clock falls to 1.5 GHz, and operands of zeros, which do not draw it, are through depth 4096 in 709 us.  Without results to store it
// would be 208.  Measured and not kept: rows resident in shared memory while the channels pass (266), twice the epilogue warps (314), stores
// with other cache hints (the same).  65 536 x 768 by 256 clusters of 768 channels 55 us where all clusters are of one size, 64 where they are
// as a router makes them, 302 MB of operands and results: HBM.
constexpr int Q_EPI_WARPS = 8;
constexpr int Q_THREADS = 128 + 32 * Q_EPI_WARPS;
constexpr uint32_t Q_TRAY_BYTES = 32 * 128;   // 32 rows of results on their way out, of each epilogue warp
template <bool LANES_ARE_ROWS>
constexpr int kPairStages = LANES_ARE_ROWS ? 5 : 6;

template <int COLS>
struct PairControl {
    uint64_t full[6];            // (the leader's are used)
    uint64_t empty[6];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];       // (the leader's are used)
    uint32_t tmem_base;
    alignas(16) float scales[Q_EPI_WARPS][COLS / 2];   // of a warp's columns
};
template <int COLS>
constexpr uint32_t kPairStageBytes = P_W_BYTES + COLS / 2 * P_DEPTH;
template <int COLS, bool LANES_ARE_ROWS>
constexpr uint32_t kPairSmem = kPairStages<LANES_ARE_ROWS> * kPairStageBytes<COLS> + (LANES_ARE_ROWS ? Q_EPI_WARPS * Q_TRAY_BYTES : 0) + sizeof(PairControl<COLS>) + 1024;

template <int COLS, typename O, bool LANES_ARE_ROWS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Q_THREADS, 1) product_pair_kernel(const __grid_constant__ ProductMaps maps, const ProductParams p) {
    wait_for_the_one_before();
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
    uint8_t* smem = smem_raw + pad;
    const uint32_t smem_base = raw_addr + pad;
    constexpr int STAGES = kPairStages<LANES_ARE_ROWS>;
    constexpr uint32_t TRAYS_AT = STAGES * kPairStageBytes<COLS>;
    auto* ctrl = reinterpret_cast<PairControl<COLS>*>(smem + TRAYS_AT + (LANES_ARE_ROWS ? Q_EPI_WARPS * Q_TRAY_BYTES : 0));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    constexpr uint32_t ROWS = LANES_ARE_ROWS ? 256 : COLS, CHANNELS = LANES_ARE_ROWS ? COLS : 256;   // of a tile

    if (threadIdx.x == 0) {
        tma_prefetch_map(&maps.w);
        tma_prefetch_map(&maps.x);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&ctrl->full[s], 1);
            mbar_init(&ctrl->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctrl->acc_full[b], 1);
            mbar_init(&ctrl->acc_empty[b], 2 * Q_EPI_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 1) tmem_alloc_pair(&ctrl->tmem_base, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // the peer's barriers exist
    tc_fence_after();
    const uint32_t tmem_base = ctrl->tmem_base;

    const uint32_t row_tiles = p.groups ? load_new(p.n_tiles) : (p.n + ROWS - 1) / ROWS;   // that have a group
    const uint32_t n_tiles = row_tiles * p.channel_tiles;
    const uint32_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
    // the rows of tile t and its first channel
    auto tile_at = [&](uint32_t t, uint32_t& channel0) {
        const uint32_t i = t / p.channel_tiles;
        channel0 = (t - i * p.channel_tiles) * CHANNELS;
        if (p.groups) return load_tile(p.tiles + i);
        return RowTile{i * ROWS, min(i * ROWS + ROWS, p.n), 0};
    };

    bool ok = true;
    if (warp == 0 && lane == 0) {
        uint32_t it = 0, next_channel0 = 0;
        RowTile next = first < n_tiles ? tile_at(first, next_channel0) : RowTile{};
        const CUtensorMap* lane_map = LANES_ARE_ROWS ? &maps.x : &maps.w;
        const CUtensorMap* column_map = LANES_ARE_ROWS ? &maps.w : &maps.x;
        for (uint32_t t = first; t < n_tiles && ok; t += step) {
            const uint32_t w_row = next.group * p.m + next_channel0, x_row = next.row0;
            const int at_lanes = static_cast<int>((LANES_ARE_ROWS ? x_row : w_row) + rank * 128), at_columns = static_cast<int>((LANES_ARE_ROWS ? w_row : x_row) + rank * (COLS / 2));
            if (t + step < n_tiles) next = tile_at(t + step, next_channel0);
            for (uint32_t k = 0; k < p.depth_blocks; ++k, ++it) {
                const uint32_t s = it % STAGES, ph = (it / STAGES) & 1u;
                if ((p.producer_stop != 0 && it >= p.producer_stop) || !wait_for(&ctrl->empty[s], ph ^ 1u, p)) {
                    ok = false;
                    break;
                }
                if (rank == 0) mbar_arrive_expect_tx(&ctrl->full[s], 2 * kPairStageBytes<COLS>);
                const uint32_t bar = cluster_address(&ctrl->full[s], 0), st = smem_base + s * kPairStageBytes<COLS>;
                tma_load_2d_pair(st, lane_map, bar, static_cast<int>(k * P_DEPTH), at_lanes);
                tma_load_2d_pair(st + P_W_BYTES, column_map, bar, static_cast<int>(k * P_DEPTH), at_columns);
            }
        }
        if (!ok) {
            // another role gave up: a millisecond for the copies that are in flight before the block's memory is let go
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) {
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        constexpr uint32_t idesc = make_idesc_i8(256, COLS);
        uint32_t it = 0, i = 0;
        for (uint32_t t = first; t < n_tiles && ok; t += step, ++i) {
            const uint32_t b = i & 1u, acc = tmem_base + b * 256;
            if (!wait_for(&ctrl->acc_empty[b], ((i >> 1) & 1u) ^ 1u, p)) {
                ok = false;
                break;
            }
            tc_fence_after();
            for (uint32_t k = 0; k < p.depth_blocks; ++k, ++it) {
                const uint32_t s = it % STAGES, ph = (it / STAGES) & 1u;
                if (!wait_for(&ctrl->full[s], ph, p)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t st = smem_base + s * kPairStageBytes<COLS>;
#pragma unroll
                for (uint32_t kk = 0; kk < P_DEPTH / 32; ++kk) umma_i8_pair(acc, make_desc_128(st + kk * 32), make_desc_128(st + P_W_BYTES + kk * 32), k != 0 || kk != 0 ? 1u : 0u, idesc);
                umma_commit_pair(&ctrl->empty[s]);
            }
            if (ok) umma_commit_pair(&ctrl->acc_full[b]);
        }
    } else if (threadIdx.x == 127) {
        forget_the_replay_before(p);
    } else if (warp >= 4) {
        constexpr uint32_t MINE = COLS / 2, EACH = MINE / 32;   // columns of a warp
        const uint32_t quarter = warp & 3u, half = (warp - 4) >> 2;
        float* scales = ctrl->scales[warp - 4];
        [[maybe_unused]] uint8_t* tray = smem + TRAYS_AT + (warp - 4) * Q_TRAY_BYTES;
        O* out = static_cast<O*>(p.out);
        const bool packed = p.m % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & 3) == 0;
        // a tile's place and scales are looked up while the one before is stored
        uint32_t row = 0, channel = 0, count = 0;   // row and channel of this lane's first column, columns
        bool valid = false;                         // this lane is in the matrix
        float lane_scale = 0.f, scale[EACH];
        auto look_up = [&](uint32_t t) {
            uint32_t channel0;
            const RowTile tile = tile_at(t, channel0);
            const float* w_scales = p.w_scales + static_cast<size_t>(tile.group) * p.m;
            const uint32_t at_lane = rank * 128 + quarter * 32 + lane;
            uint32_t end, column;
            const float* column_scales;
            if constexpr (LANES_ARE_ROWS) {
                row = tile.row0 + at_lane;
                channel = channel0 + half * MINE;
                valid = row < tile.row1;
                column = channel;
                end = p.m;
                column_scales = w_scales;
                lane_scale = valid ? load_new(p.x_scales + row) : 0.f;
            } else {
                row = tile.row0 + half * MINE;
                channel = channel0 + at_lane;
                valid = channel < p.m;
                column = row;
                end = tile.row1;
                column_scales = p.x_scales;
                lane_scale = valid ? load_new(w_scales + channel) : 0.f;
            }
            count = end > column ? min(end - column, MINE) : 0;
#pragma unroll
            for (uint32_t e = 0; e < EACH; ++e) scale[e] = e * 32 + lane < count ? load_new(column_scales + column + e * 32 + lane) : 0.f;
        };
        if (first < n_tiles) look_up(first);
        uint32_t i = 0;
        for (uint32_t t = first; t < n_tiles; t += step, ++i) {
            const uint32_t b = i & 1u, my_row = row, my_channel = channel, my_count = count;
            const bool my_valid = valid;
            const float my_scale = lane_scale;
            __syncwarp();
#pragma unroll
            for (uint32_t e = 0; e < EACH; ++e) scales[e * 32 + lane] = scale[e];
            __syncwarp();
            if (t + step < n_tiles) look_up(t + step);
            if (!__all_sync(0xffffffffu, wait_for(&ctrl->acc_full[b], (i >> 1) & 1u, p))) {
                if (lane == 0) *reinterpret_cast<volatile int*>(p.told) = 47;
                break;
            }
            tc_fence_after();
            const uint32_t taddr = tmem_base + (quarter * 32 << 16) + b * 256 + half * MINE;
            O* to = out + static_cast<size_t>(my_row) * p.m;
            [[maybe_unused]] const bool whole = __all_sync(0xffffffffu, my_valid);   // (what is behind the last column is left out by the copy)
            each_32_columns<MINE>(taddr, my_count, scales, my_scale, [&](uint32_t c, const uint64_t (&v)[16]) {
                if constexpr (LANES_ARE_ROWS) {
                    if (!whole) {
                        if (my_valid) store_along_row(to + my_channel + c, v, my_count - c);
                        return;
                    }
                    // by way of shared memory, so that whole lines go out: 16-byte unit u of row r of the tray lies at unit u ^ (r & 7)
                    constexpr uint32_t TRAY = 128 / sizeof(O), UNITS = 32 * sizeof(O) / 16;   // columns of a tray, units of 32 columns
                    const uint32_t at = c % TRAY / 32 * UNITS;
                    if (at == 0) {
                        if (lane == 0) tma_stores_read();
                        __syncwarp();
                    }
#pragma unroll
                    for (uint32_t u = 0; u < UNITS; ++u) {
                        uint4 w;
                        if constexpr (sizeof(O) == 2) {
                            auto two = [&](uint64_t x) { return pair_from_float(low_of(x), high_of(x), static_cast<const O*>(nullptr)); };
                            w = make_uint4(two(v[4 * u]), two(v[4 * u + 1]), two(v[4 * u + 2]), two(v[4 * u + 3]));
                        } else {
                            w = make_uint4(static_cast<uint32_t>(v[2 * u]), static_cast<uint32_t>(v[2 * u] >> 32), static_cast<uint32_t>(v[2 * u + 1]), static_cast<uint32_t>(v[2 * u + 1] >> 32));
                        }
                        *reinterpret_cast<uint4*>(tray + lane * 128 + (((at + u) ^ (lane & 7)) << 4)) = w;
                    }
                    if (at + UNITS == 8 || c + 32 >= my_count) {
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) tma_store_2d(&maps.out, smem_u32(tray), static_cast<int>(my_channel + c / TRAY * TRAY), static_cast<int>(my_row));
                    }
                } else {
                    store_across_rows(to + static_cast<size_t>(c) * p.m, p.m, my_channel, my_valid, lane, v, my_count - c, packed);
                }
            });
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_read(cluster_address(&ctrl->acc_empty[b], 0));
        }
        if (LANES_ARE_ROWS && lane == 0) tma_stores_done();
        // rows of no group
        if (p.groups) {
            const uint32_t all = load_new(p.n_tiles + 1), threads = threadIdx.x - 128;
            for (uint32_t t = row_tiles * p.channel_tiles + first; t < all * p.channel_tiles; t += step) {
                uint32_t channel0;
                const RowTile tile = tile_at(t, channel0);
                const uint32_t width = min(CHANNELS, p.m - channel0), c = threads % CHANNELS;
                if (c < width)
                    for (uint32_t r = tile.row0 + rank * (256 / CHANNELS) + threads / CHANNELS; r < tile.row1; r += 2 * (256 / CHANNELS))
                        store_result(out + static_cast<size_t>(r) * p.m + channel0 + c, 0.f);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();   // nothing of the pair is in flight towards this CTA any more
    if (warp == 1) tmem_dealloc_pair(tmem_base, TMEM_COLS);
}

// The tiles of `rows` rows that the groups consist of, one block; those of no group come last.  n_tiles: how many belong to a group, and
// all.
__global__ void __launch_bounds__(1024) row_tiles_kernel(const uint32_t* __restrict__ offsets, uint32_t groups, uint32_t n, uint32_t rows, uint32_t room, RowTile* __restrict__ tiles,
                                                         uint32_t* __restrict__ n_tiles) {
    wait_for_the_one_before();
    __shared__ uint32_t sums[32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t base = 0;
    for (uint32_t g0 = 0; g0 < groups + 2; g0 += 1024) {
        const uint32_t g = g0 + threadIdx.x;
        uint32_t a = 0, b = 0;
        if (g < groups) {
            a = min(load_new(offsets + g), n);
            b = min(load_new(offsets + g + 1), n);
        } else if (g == groups) {
            a = min(load_new(offsets + groups), n);
            b = n;
        } else if (g == groups + 1) {
            b = min(load_new(offsets), n);
        }
        const uint32_t count = b > a ? (b - a + rows - 1) / rows : 0;
        uint32_t upto = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= static_cast<uint32_t>(o)) upto += v;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        uint32_t before = base, total = 0;
        for (uint32_t w = 0; w < 32; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        before += upto - count;
        if (g == groups) n_tiles[0] = min(before, room);
        for (uint32_t i = 0; i < count && before + i < room; ++i) tiles[before + i] = {a + i * rows, min(a + (i + 1) * rows, b), g};
        base += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) n_tiles[1] = min(base, room);
}

// Where a kernel records that a wait ran out: for its other waits in device memory, for the host in its own.
struct Status {
    uint32_t* device = nullptr;
    int* host = nullptr;
    int* host_on_device = nullptr;
};
constexpr int kMaxDevices = 64;
__device__ uint32_t g_product_given_up;   // (in host code a handle, no address)
std::atomic<uint32_t> g_product_launches{0};

Status& status_of_current_device() {
    static std::mutex mutex;
    static Status all[kMaxDevices];
    int device = 0;
    SKM_CUDA(cudaGetDevice(&device));
    if (device >= kMaxDevices) throw CudaError("too many CUDA devices");
    std::lock_guard<std::mutex> lock(mutex);
    Status& s = all[device];
    if (!s.host_on_device) {
        // (also when a stream is being captured, which this is no part of)
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        SKM_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
        void* word = nullptr;
        cudaError_t e = cudaGetSymbolAddress(&word, g_product_given_up);
        s.device = static_cast<uint32_t*>(word);
        if (e == cudaSuccess && !s.host) e = cudaHostAlloc(&s.host, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
        if (e == cudaSuccess) {
            *s.host = 0;
            e = cudaHostGetDevicePointer(&s.host_on_device, s.host, 0);
        }
        const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
        SKM_CUDA(e);
        SKM_CUDA(back);
        note_device_alloc();
    }
    return s;
}

void throw_if_told(Status& s, cudaStream_t stream) {
    volatile int* told = s.host;
    if (*told == 0) return;
    const int code = *told;
    // (a capture that fails for this is told, and so is the next call outside)
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    SKM_CUDA(cudaStreamIsCapturing(stream, &capture));
    if (capture == cudaStreamCaptureStatusNone) *told = 0;
    throw CudaError("a product in 8 bits gave up waiting on a barrier (code " + std::to_string(code) + "): its results are not valid");
}

// Blocks of a kernel that are resident at a time, looked up once per kernel and device.
template <typename... A>
size_t resident_blocks(void (*kernel)(A...), int threads) {
    static std::mutex mutex;
    static std::map<std::pair<int, const void*>, size_t> known;
    int device = 0;
    SKM_CUDA(cudaGetDevice(&device));
    std::lock_guard<std::mutex> lock(mutex);
    size_t& blocks = known[{device, reinterpret_cast<const void*>(kernel)}];
    if (blocks == 0) {
        int of_sm = 0, sms = 0;
        SKM_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&of_sm, kernel, threads, 0));
        SKM_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        blocks = static_cast<size_t>(std::max(of_sm, 1)) * sms;
    }
    return blocks;
}

bool tma_takes(const void* p, size_t ld, size_t d) { return (address(p) & 15) == 0 && ld % 16 == 0 && ld >= d; }
size_t pitch_of(size_t d) { return (d + 15) / 16 * 16; }
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct ProductPlan {
    bool pairs, lanes_are_rows;
    uint32_t rows, split, row_tiles;   // row_tiles: with groups at most
};
// Which kernel and tile, by the rows that a matrix has on average (one B200, kernels alone, results in bf16, d = 768):
//   pairs of CTAs from 65 rows and 64 tiles on.  By 16 384 channels (64 tiles and more) 64 rows take 5.7 us with a CTA to a tile and 6.0 with pairs, 65
//   7.6 and 6.2, 256 12.3 and 7.2, 4096 155 and 47; by 4096 channels 256 rows (32 tiles) 5.6 and 6.0, 512 (64) 7.0 and 6.1, 1024 (128) 12.3 and 7.2.
//   By 64 clusters of 768 channels each 64 rows 14.2 and 13.6, 65 20.3 and 14.0; by 256 clusters pairs would be ahead from 8 rows on (34 and 32; of 64
//   55 and 37).
//   256 columns from 192 rows on, 128 below: of 64 clusters 128 rows 14.4 us with 128 and 16.0 with 256, 192 rows 21.1 and 16.0 (between, 129 rows
//   20.5 and 15.8: two tiles to a cluster); of 256 clusters 43.6 and 46.2, 59.5 and 50.0.
//   Without pairs, 16, 32 or 64 rows to a tile, the least that hold them: of 64 clusters 16 rows take 10.5, 12.5 and 12.9 us, 17 14.8, 12.5 and 12.9, 33
//   19.3, 18.1 and 13.9.
ProductPlan make_plan(const Product& p) {
    const size_t channel_tiles = (p.m + P_CHANNELS - 1) / P_CHANNELS, depth_blocks = (p.d + P_DEPTH - 1) / P_DEPTH;
    const size_t typical = p.groups ? (p.n + p.groups - 1) / p.groups : p.n;
    ProductPlan plan{};
    plan.split = 1;
    plan.pairs = typical > 64 && (p.n + 127) / 128 * ((p.m + 255) / 256) >= 64;
    if (plan.pairs) {
        const bool wide = typical >= 192;
        plan.lanes_are_rows = wide && p.m * type_bytes(p.out_type) % 32 == 0 && (address(p.out) & 31) == 0;
        plan.rows = wide ? 256 : 128;
        plan.row_tiles = static_cast<uint32_t>((p.n + plan.rows - 1) / plan.rows + (p.groups ? p.groups + 1 : 0));
        return plan;
    }
    plan.rows = typical <= 16 ? 16 : typical <= 32 ? 32 : 64;
    plan.row_tiles = static_cast<uint32_t>((p.n + plan.rows - 1) / plan.rows + (p.groups ? p.groups + 1 : 0));
    // (adding the sums up costs two barriers of the cluster and 2 us: no block gets fewer than four steps; 64 rows by 1000 channels of depth 4096
    // 6.8 us, 7.8 with eight steps at least, 12.3 undivided; 1 by 16 384 of 768, which has too many tiles to be divided, 4.9)
    if (!p.groups)
        while (plan.split < 8 && plan.row_tiles * channel_tiles * plan.split * 2 <= 148 && depth_blocks >= 8 * plan.split) plan.split *= 2;
    return plan;
}

} // namespace

void launch_quantize_rows(const Rows& x, Type type, size_t n, size_t d, int8_t* q, size_t ldq, float* scales, cudaStream_t stream) {
    if (n == 0) return;
    const size_t t = type_bytes(type), pitch = x.ld * t, each = 16 / t;   // (values, and bytes of q, of a 16-byte chunk)
    const int access = access_bytes({address(x.p), pitch, d * t, address(q) * t, ldq * t});
    const bool windows = use_windows(access, d * t) && address(q) % each == 0 && ldq % each == 0;
    with_width(type, windows ? 16 : access, [&](auto value, auto width) {
        using T = decltype(value);
        constexpr int B = decltype(width)::bytes;
        const size_t chunks = (d * t + B - 1) / B;
        auto launch = [&](auto* kernel, int lanes) {
            // as many blocks as are resident, and the same number of turns for each
            const size_t blocks = (n + 256 / lanes - 1) / (256 / lanes), resident = resident_blocks(kernel, 256), turns = (blocks + resident - 1) / resident;
            launch_after(kernel, dim3(static_cast<unsigned>((blocks + turns - 1) / turns)), 256, 0, stream, x.p, pitch, n, d * t, q, ldq, scales);
        };
        auto of_width = [&](auto in_windows) {
            constexpr bool W = decltype(in_windows)::value;
            // as few lanes to a row as hold it: what a warp does once for its rows (shuffles, divisions, addresses) is half of its instructions
            // (65 536 x 768 bf16: 24 us with 16 lanes, 29 with 32; 500 000 x 64: 20 with 2, 27 with 8)
            if (chunks <= 2 * 6) launch(quantize_rows_kernel<T, B, W, 2, 6>, 2);
            else if (chunks <= 4 * 6) launch(quantize_rows_kernel<T, B, W, 4, 6>, 4);
            else if (chunks <= 8 * 6) launch(quantize_rows_kernel<T, B, W, 8, 6>, 8);
            else if (chunks <= 16 * 6) launch(quantize_rows_kernel<T, B, W, 16, 6>, 16);
            else if (chunks <= 32 * 8) launch(quantize_rows_kernel<T, B, W, 32, 8>, 32);
            else launch(quantize_rows_kernel<T, B, W, 256, 4>, 256);
        };
        if constexpr (B == 16) {
            if (windows) return of_width(std::true_type{});
        }
        of_width(std::false_type{});
    });
}

size_t product_workspace_bytes(const Product& p) {
    const ProductPlan plan = make_plan(p);
    size_t bytes = 0;
    if (!tma_takes(p.x, p.ldx, p.d)) bytes += rounded(p.n * pitch_of(p.d));
    if (!tma_takes(p.w, p.ldw, p.d)) bytes += rounded(std::max<size_t>(1, p.groups) * p.m * pitch_of(p.d));
    if (p.groups) bytes += rounded(plan.row_tiles * sizeof(RowTile)) + 256;
    return bytes;
}

void launch_product(const Product& p, void* workspace, cudaStream_t stream) {
    if (p.n == 0 || p.m == 0) return;
    Status& status = status_of_current_device();
    throw_if_told(status, stream);
    const ProductPlan plan = make_plan(p);
    char* at = static_cast<char*>(workspace);
    auto take = [&](size_t bytes) {
        char* here = at;
        at += rounded(bytes);
        return here;
    };
    auto padded = [&](const int8_t*& rows, size_t& ld, size_t n) {
        if (tma_takes(rows, ld, p.d)) return;
        const size_t pitch = pitch_of(p.d);
        int8_t* copy = reinterpret_cast<int8_t*>(take(n * pitch));
        launch_after(pad_bytes_kernel, dim3(static_cast<unsigned>((n + 7) / 8)), 256, 0, stream, rows, ld, n, static_cast<uint32_t>(p.d), static_cast<uint32_t>(pitch), copy);
        rows = copy;
        ld = pitch;
    };
    const int8_t *x = p.x, *w = p.w;
    size_t ldx = p.ldx, ldw = p.ldw;
    const size_t w_rows = std::max<size_t>(1, p.groups) * p.m;
    padded(x, ldx, p.n);
    padded(w, ldw, w_rows);

    ProductParams k{};
    k.x_scales = p.x_scales;
    k.w_scales = p.w_scales;
    k.out = p.out;
    k.n = static_cast<uint32_t>(p.n);
    k.m = static_cast<uint32_t>(p.m);
    k.depth_blocks = static_cast<uint32_t>((p.d + P_DEPTH - 1) / P_DEPTH);
    const uint32_t channels = plan.pairs ? 256 : P_CHANNELS;
    k.channel_tiles = static_cast<uint32_t>((p.m + channels - 1) / channels);
    k.groups = static_cast<uint32_t>(p.groups);
    k.given_up = status.device;
    do k.launch = ++g_product_launches;
    while (k.launch == 0);   // (no launch)
    k.told = status.host_on_device;
    k.wait_limit = wait_limit();
    k.producer_stop = producer_stop();
    if (p.groups) {
        RowTile* tiles = reinterpret_cast<RowTile*>(take(plan.row_tiles * sizeof(RowTile)));
        uint32_t* n_tiles = reinterpret_cast<uint32_t*>(take(8));
        launch_after(row_tiles_kernel, dim3(1), 1024, 0, stream, p.offsets, k.groups, k.n, plan.rows, plan.row_tiles, tiles, n_tiles);
        k.tiles = tiles;
        k.n_tiles = n_tiles;
    }
    ProductMaps maps{};
    maps.w = make_byte_tmap(w, p.d, w_rows, P_CHANNELS, ldw);
    maps.x = make_byte_tmap(x, p.d, p.n, plan.pairs ? plan.rows / 2 : plan.rows, ldx);
    const size_t all_tiles = static_cast<size_t>(plan.row_tiles) * k.channel_tiles;
    if (all_tiles * plan.split > 0x7fffffff) throw std::invalid_argument("a product of these sizes needs too many tiles");
    auto launch_pairs = [&](auto columns, auto result) {
        constexpr int COLS = decltype(columns)::value;
        using O = decltype(result);
        const unsigned grid = 2 * static_cast<unsigned>(std::min<size_t>(all_tiles, static_cast<size_t>(sm_pairs())));
        auto go = [&](auto* kernel, uint32_t smem) {
            allow_shared(kernel, smem);
            launch_after(kernel, dim3(grid), Q_THREADS, smem, stream, maps, k);
        };
        if constexpr (COLS == 256) {
            if (plan.lanes_are_rows) {
                maps.out = make_result_tmap(p.out, sizeof(O), p.m, p.n, 32);
                go(product_pair_kernel<COLS, O, true>, kPairSmem<COLS, true>);
            } else {
                go(product_pair_kernel<COLS, O, false>, kPairSmem<COLS, false>);
            }
        } else {
            go(product_pair_kernel<COLS, O, false>, kPairSmem<COLS, false>);
        }
    };
    auto launch = [&](auto rows, auto result) {
        constexpr int ROWS = decltype(rows)::value;
        using O = decltype(result);
        auto* kernel = product_kernel<ROWS, O>;
        allow_shared(kernel, kProductSmem<ROWS>);
        launch_clusters_after(kernel, dim3(static_cast<unsigned>(all_tiles * plan.split)), plan.split, P_THREADS, kProductSmem<ROWS>, stream, maps, k);
    };
    auto of_type = [&](auto&& go, auto rows) {
        if (p.out_type == Type::f32) go(rows, float{});
        else if (p.out_type == Type::f16) go(rows, __half{});
        else go(rows, __nv_bfloat16{});
    };
    if (plan.pairs && plan.rows == 256) of_type(launch_pairs, std::integral_constant<int, 256>{});
    else if (plan.pairs) of_type(launch_pairs, std::integral_constant<int, 128>{});
    else if (plan.rows == 16) of_type(launch, std::integral_constant<int, 16>{});
    else if (plan.rows == 32) of_type(launch, std::integral_constant<int, 32>{});
    else of_type(launch, std::integral_constant<int, 64>{});
}

void check_products(cudaStream_t stream) {
    Status& s = status_of_current_device();
    SKM_CUDA(cudaStreamSynchronize(stream));
    throw_if_told(s, stream);
}

} // namespace rows
} // namespace skmb
