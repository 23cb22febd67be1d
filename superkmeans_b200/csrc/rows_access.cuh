// Loads and stores of a few neighbouring values of a row, and their conversion to and from fp32, shared by the operators on rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"
#include "rows.h"

namespace skmb {
namespace rows {

// What one load or store moves.
template <int BYTES>
struct ChunkOf;
struct alignas(32) Words8 {
    uint32_t w[8];
};
template <>
struct ChunkOf<32> {
    using type = Words8;
};
template <>
struct ChunkOf<16> {
    using type = uint4;
};
template <>
struct ChunkOf<8> {
    using type = uint2;
};
template <>
struct ChunkOf<4> {
    using type = uint32_t;
};
template <>
struct ChunkOf<2> {
    using type = uint16_t;
};
template <int BYTES>
using Chunk = typename ChunkOf<BYTES>::type;

template <int BYTES>
__device__ __forceinline__ Chunk<BYTES> zero_chunk() {
    Chunk<BYTES> c;
    memset(&c, 0, BYTES);
    return c;
}

// Loads for kernels that start before the one ahead has ended (launch_after) of what that one may have written: a read-only load (__ldg) is
// for memory that does not change while the kernel lives, and may be moved ahead of the wait.  load_now reads what is visible
// behind the wait; load_new passes the first-level cache by as well, for what is read once.
#define SKM_LOADS(TYPE, SUFFIX, REGISTER)                                                                     \
    __device__ __forceinline__ TYPE load_now(const TYPE* p) {                                                 \
        TYPE v;                                                                                               \
        asm volatile("ld.global." SUFFIX " %0, [%1];" : "=" REGISTER(v) : "l"(p));                            \
        return v;                                                                                             \
    }                                                                                                         \
    __device__ __forceinline__ TYPE load_new(const TYPE* p) {                                                 \
        TYPE v;                                                                                               \
        asm volatile("ld.global.cg." SUFFIX " %0, [%1];" : "=" REGISTER(v) : "l"(p));                         \
        return v;                                                                                             \
    }
SKM_LOADS(uint16_t, "u16", "h")
SKM_LOADS(uint32_t, "u32", "r")
SKM_LOADS(float, "f32", "f")
SKM_LOADS(unsigned long long, "u64", "l")
#undef SKM_LOADS
__device__ __forceinline__ uint32_t load_now(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load_now(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load_new(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.cg.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load_now(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load_new(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Global memory that nobody writes while the kernel lives, and stores.
template <int BYTES>
__device__ __forceinline__ Chunk<BYTES> load_chunk(const Chunk<BYTES>* p) {
    if constexpr (BYTES == 32) {
        Words8 c;
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(c.w[0]), "=r"(c.w[1]), "=r"(c.w[2]), "=r"(c.w[3]), "=r"(c.w[4]), "=r"(c.w[5]), "=r"(c.w[6]), "=r"(c.w[7])
                     : "l"(p));
        return c;
    } else {
        return __ldg(p);
    }
}
template <int BYTES>
__device__ __forceinline__ void store_chunk(Chunk<BYTES>* p, const Chunk<BYTES>& c) {
    if constexpr (BYTES == 32) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(c.w[0]), "r"(c.w[1]), "r"(c.w[2]), "r"(c.w[3]), "r"(c.w[4]), "r"(c.w[5]), "r"(c.w[6]),
                     "r"(c.w[7])
                     : "memory");
    } else {
        *p = c;
    }
}

__device__ __forceinline__ float2 pair_to_float(uint32_t u, const __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ float2 pair_to_float(uint32_t u, const __nv_bfloat16*) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pair_from_float(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_from_float(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The values of a chunk in fp32, and back (rounded to nearest).
template <typename T, int BYTES>
struct Values {
    static constexpr int N = BYTES / static_cast<int>(sizeof(T));
    float v[N];

    __device__ __forceinline__ void from(const Chunk<BYTES>& c) {
        if constexpr (sizeof(T) == 4) {
            memcpy(v, &c, BYTES);
        } else if constexpr (BYTES == 2) {
            v[0] = pair_to_float(c, static_cast<const T*>(nullptr)).x;
        } else {
            uint32_t u[BYTES / 4];
            memcpy(u, &c, BYTES);
#pragma unroll
            for (int i = 0; i < BYTES / 4; ++i) {
                const float2 f = pair_to_float(u[i], static_cast<const T*>(nullptr));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ Chunk<BYTES> to() const {
        Chunk<BYTES> c;
        if constexpr (sizeof(T) == 4) {
            memcpy(&c, v, BYTES);
        } else if constexpr (BYTES == 2) {
            c = static_cast<uint16_t>(pair_from_float(v[0], 0.f, static_cast<const T*>(nullptr)));
        } else {
            uint32_t u[BYTES / 4];
#pragma unroll
            for (int i = 0; i < BYTES / 4; ++i) u[i] = pair_from_float(v[2 * i], v[2 * i + 1], static_cast<const T*>(nullptr));
            memcpy(&c, u, BYTES);
        }
        return c;
    }
};

// The 16 bytes at p, an address of values of T that need not be a multiple of 16, of which bytes from .. to - 1 are wanted: the one or two
// aligned blocks that hold some of them, shifted.  (A block that holds a byte of the rows is memory of theirs or of the same 16 bytes:
// nothing beyond is touched.  The bytes that are not wanted are of no meaning.)
template <typename T, bool NOW = false>
__device__ __forceinline__ uint4 load_window(const char* p, uint32_t from, uint32_t to) {
    const uint32_t s = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uint4* block = reinterpret_cast<const uint4*>(p - s);
    auto load = [](const uint4* b) {
        if constexpr (NOW) return load_now(b);
        else return __ldg(b);
    };
    const uint4 lo = from < 16 - s ? load(block) : make_uint4(0, 0, 0, 0), hi = to > 16 - s ? load(block + 1) : make_uint4(0, 0, 0, 0);
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = s & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = s & 4 ? w[i + 1] : w[i];
    if constexpr (sizeof(T) == 2) {
        const uint32_t bits = (s & 2) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Where a row's own chunks are read one after the other: by windows if neighbouring lanes could take two bytes each otherwise (100 000
// rows of 181 fp16 to 8 bits: 31 us against 42), but not if four or eight (50 000 of 1001 fp32: 169 against 101).
inline bool use_windows(int bytes, size_t row_bytes) { return bytes < 4 && row_bytes >= 32; }

// Kernels that follow one another (launch_after) start before the one ahead has ended and wait for it here, before they touch memory: what
// that one wrote is visible then, to load_now and load_new.  (Sort and sums of 500 000 pairs, by eight launches then: 227 -> 219 us;
// routing of 30 001 x 4 rows: 118 -> 108.)
__device__ __forceinline__ void wait_for_the_one_before() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
// (cluster: blocks to a cluster, 0 where the kernel says itself)
template <typename... P, typename... A>
void launch_clusters_after(void (*kernel)(P...), dim3 grid, unsigned cluster, unsigned threads, size_t shared, cudaStream_t stream, A&&... args) {
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {cluster, 1, 1};
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = cluster == 0 ? 1 : 2;
    SKM_CUDA(cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...));
    SKM_LAUNCH_CHECK();
}
template <typename... P, typename... A>
void launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t shared, cudaStream_t stream, A&&... args) {
    launch_clusters_after(kernel, grid, 0, threads, shared, stream, std::forward<A>(args)...);
}

// Lets a kernel have as much shared memory as it needs, once per kernel and device.
template <typename... A>
void allow_shared(void (*kernel)(A...), uint32_t bytes) {
    static std::mutex mutex;
    static std::set<std::pair<int, const void*>> done;
    int device = 0;
    SKM_CUDA(cudaGetDevice(&device));
    std::lock_guard<std::mutex> lock(mutex);
    const std::pair<int, const void*> key{device, reinterpret_cast<const void*>(kernel)};
    if (done.count(key)) return;
    SKM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    done.insert(key);
}

// Some neighbouring lanes of a warp, which may have a row of their own.
template <int LANES>
struct Lanes {
    uint32_t lane, mask;
    __device__ __forceinline__ Lanes() : lane(threadIdx.x % LANES), mask(LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << ((threadIdx.x & 31) / LANES * LANES)) {}
    template <typename V>
    __device__ __forceinline__ V from(V v, uint32_t lane_) const {
        return __shfl_sync(mask, v, lane_, LANES);
    }
    __device__ __forceinline__ uint32_t ballot(bool b) const { return __ballot_sync(mask, b) >> (LANES == 32 ? 0 : (threadIdx.x & 31) / LANES * LANES); }
    __device__ __forceinline__ float sum(float v) const {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o, LANES);
        return v;
    }
};

// The cluster of pair i, or k.
__device__ __forceinline__ uint32_t load_id(const void* ids, bool wide, size_t i, uint32_t k) {
    if (wide) {
        const unsigned long long v = load_now(static_cast<const unsigned long long*>(ids) + i);   // (a negative one is large)
        return v < k ? static_cast<uint32_t>(v) : k;
    }
    return min(load_now(static_cast<const uint32_t*>(ids) + i), k);
}

// Division of small numbers by one that a launch knows: magic is 0 where multiplication would not give the quotient.
struct Divisor {
    uint32_t d, magic;
};
// for dividends below `most`: floor(a / d) = (a * ceil(2^32 / d)) >> 32 as long as a * (d * ceil(2^32 / d) - 2^32) < 2^32, and the bracket is less than d
inline Divisor make_divisor(size_t d, size_t most) {
    const uint64_t magic = ((uint64_t{1} << 32) + d - 1) / d;
    return {static_cast<uint32_t>(d), d > 1 && most * d < (uint64_t{1} << 32) ? static_cast<uint32_t>(magic) : 0u};
}
__device__ __forceinline__ uint32_t divide(uint32_t a, const Divisor& by) { return by.magic ? __umulhi(a, by.magic) : a / by.d; }

// How many bytes a load of each of these may move at once, up to `most`: all of them are multiples of it.
inline int access_bytes(std::initializer_list<size_t> multiples, size_t most = 16) {
    size_t all = most;
    for (const size_t m : multiples) all |= m;
    return static_cast<int>(all & (~all + 1));
}
inline size_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// f(T{}, Width<BYTES>{}) for a type and a width of access up to MOST
template <int BYTES>
struct Width {
    static constexpr int bytes = BYTES;
};
template <int MOST = 16, class F>
void with_width(Type type, int bytes, F&& f) {
    auto of = [&](auto t) {
        if (MOST >= 32 && bytes >= 32) f(t, Width<MOST>{});
        else if (bytes >= 16) f(t, Width<16>{});
        else if (bytes == 8) f(t, Width<8>{});
        else if (bytes == 4) f(t, Width<4>{});
        else if constexpr (sizeof(t) == 2) f(t, Width<2>{});
    };
    if (type == Type::f32) of(float{});
    else if (type == Type::f16) of(__half{});
    else of(__nv_bfloat16{});
}

} // namespace rows
} // namespace skmb
