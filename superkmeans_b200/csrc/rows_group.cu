// Pairs (row, choice) in the order of their cluster: a stable sort of small numbers by counting.
//
// A few pairs: every pair counts, against all others, how many come before it.  That is n^2 comparisons, but in one launch over the
// whole chip, and a launch is what the time of a small call consists of.
//
// More: a radix sort, up to 11 bits at a time.  A unit of a few hundred pairs belongs to a warp, which counts its digits in shared
// memory; a warp for each digit turns the units' counts into the places where each unit's pairs of that digit begin; and the units,
// read again, rank equal digits among 32 neighbours by __match_any_sync, in order, so that the sort is stable and nothing depends on
// the order of atomics (those add whole numbers).  Up to 2047 clusters need one pass.
#include <algorithm>

#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr size_t kFewPairs = 4096;
constexpr int kMaxBits = 11;
constexpr int kUnitWarps = 4;

// ---------------------------------------------------------------------------------------------- few pairs
// A block ranks 32 pairs (one to a lane) against all: each of its eight warps compares them with an eighth of the keys.
__global__ void __launch_bounds__(256) rank_kernel(const void* __restrict__ ids, bool wide, uint32_t n, uint32_t k, uint32_t* __restrict__ order, uint32_t* __restrict__ position,
                                                   uint32_t* __restrict__ keys_out, uint32_t* __restrict__ offsets) {
    __shared__ uint4 key4[kFewPairs / 4];
    __shared__ uint32_t parts[3][8][32];
    uint32_t* key = reinterpret_cast<uint32_t*>(key4);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t n4 = (n + 3) / 4;
    for (uint32_t i = threadIdx.x; i < 4 * n4; i += 256) key[i] = i < n ? load_id(ids, wide, i, k) : 0xffffffffu;
    __syncthreads();
    const uint32_t mine = blockIdx.x * 32 + lane;
    const uint32_t c = mine < n ? key[mine] : 0u;
    // keys less than c, equal ones of earlier pairs, and 1 + the largest of the lesser ones
    uint32_t less = 0, earlier = 0, below = 0;
    const uint32_t a = warp * n4 / 8, b = (warp + 1) * n4 / 8;
    for (uint32_t i = a; i < b; ++i) {
        const uint4 q = key4[i];
        const uint32_t v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if (v[e] < c) {
                ++less;
                below = max(below, v[e] + 1);
            }
            if (v[e] == c && 4 * i + e < mine) ++earlier;
        }
    }
    parts[0][warp][lane] = less;
    parts[1][warp][lane] = earlier;
    parts[2][warp][lane] = below;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
        less += parts[0][w][lane];
        earlier += parts[1][w][lane];
        below = max(below, parts[2][w][lane]);
    }
    const uint32_t slot = less + earlier;
    // the first pair of a cluster sets where the clusters behind the one before it begin, the last pair of all the rest
    uint32_t from = 1, upto = 0, value = 0;
    if (mine < n) {
        order[slot] = mine;
        if (position) position[mine] = slot;
        if (keys_out) keys_out[slot] = c;
        if (earlier == 0) {
            from = below;
            upto = c;
            value = slot;
        }
    }
    uint32_t rest_from = 1, rest_upto = 0;
    if (mine < n && slot == n - 1) {
        rest_from = c + 1;
        rest_upto = k;
    }
    for (uint32_t l = 0; l < 32; ++l) {
        const uint32_t f = __shfl_sync(0xffffffffu, from, l), t = __shfl_sync(0xffffffffu, upto, l), v = __shfl_sync(0xffffffffu, value, l);
        for (uint32_t i = f + lane; i <= t; i += 32) offsets[i] = v;
        const uint32_t rf = __shfl_sync(0xffffffffu, rest_from, l), rt = __shfl_sync(0xffffffffu, rest_upto, l);
        for (uint32_t i = rf + lane; i <= rt; i += 32) offsets[i] = n;
    }
}

// ---------------------------------------------------------------------------------------------- many pairs
struct Pass {
    size_t n;
    uint32_t k;
    int shift, bits;
    uint32_t n_units, unit;   // a unit has this many pairs, a multiple of 32
};

// What a pass sorts: the caller's ids (the first), or the pass before's keys and pairs.
struct PassInput {
    const void* ids;
    bool wide;
    const uint32_t* keys;
    const uint32_t* pairs;
};

__device__ __forceinline__ uint32_t key_of(const PassInput& in, size_t i, uint32_t k) { return in.keys ? __ldg(in.keys + i) : load_id(in.ids, in.wide, i, k); }

constexpr int kSortAhead = 4;

// table[digit][unit] = the unit's pairs with that digit; totals[digit] += them
__global__ void __launch_bounds__(32 * kUnitWarps) count_kernel(const PassInput in, const Pass p, uint32_t* __restrict__ table, uint32_t* __restrict__ totals) {
    extern __shared__ uint32_t counts[];   // [digit][warp]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digits = 1u << p.bits;
    for (uint32_t i = threadIdx.x; i < digits * kUnitWarps; i += 32 * kUnitWarps) counts[i] = 0;
    __syncthreads();
    const uint32_t unit0 = blockIdx.x * kUnitWarps, unit = unit0 + warp;
    const size_t begin = static_cast<size_t>(unit) * p.unit, end = min(begin + p.unit, p.n);
    for (size_t s = begin; s < end; s += 32 * kSortAhead) {
        uint32_t key[kSortAhead];
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const size_t i = s + u * 32 + lane;
            key[u] = i < end ? key_of(in, i, p.k) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u)
            if (s + u * 32 + lane < end) atomicAdd(&counts[((key[u] >> p.shift) & (digits - 1)) * kUnitWarps + warp], 1u);
    }
    __syncthreads();
    const uint32_t here = min(static_cast<uint32_t>(kUnitWarps), p.n_units - unit0);
    for (uint32_t i = threadIdx.x; i < digits; i += 32 * kUnitWarps) {
        uint32_t sum = 0;
        for (uint32_t w = 0; w < here; ++w) {
            const uint32_t c = counts[i * kUnitWarps + w];
            table[static_cast<size_t>(i) * p.n_units + unit0 + w] = c;
            sum += c;
        }
        if (sum) atomicAdd(totals + i, sum);
    }
}

// table[digit][unit] = the slot of the unit's first pair with that digit; a warp for each digit.  offsets (may be null): of the
// digits up to k.
__global__ void __launch_bounds__(256) place_kernel(const Pass p, uint32_t* __restrict__ table, const uint32_t* __restrict__ totals, uint32_t* __restrict__ offsets) {
    __shared__ uint32_t sums[8];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digits = 1u << p.bits, digit0 = blockIdx.x * 8, digit = digit0 + warp;
    uint32_t before = 0;
    for (uint32_t i = threadIdx.x; i < digit0; i += 256) before += __ldg(totals + i);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) sums[warp] = before;
    __syncthreads();
    uint32_t slot = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) slot += sums[w];
    for (uint32_t i = digit0; i < digit; ++i) slot += __ldg(totals + i);
    if (digit >= digits) return;
    if (offsets && lane == 0 && digit <= p.k) offsets[digit] = slot;
    uint32_t* row = table + static_cast<size_t>(digit) * p.n_units;
    constexpr int AHEAD = 8;
    for (uint32_t s = 0; s < p.n_units; s += 32 * AHEAD) {
        uint32_t v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u] = s + u * 32 + lane < p.n_units ? row[s + u * 32 + lane] : 0u;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            uint32_t upto = v[u];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            if (s + u * 32 + lane < p.n_units) row[s + u * 32 + lane] = slot + upto - v[u];
            slot += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
}

__global__ void __launch_bounds__(32 * kUnitWarps) scatter_kernel(const PassInput in, const Pass p, const uint32_t* __restrict__ table, uint32_t* __restrict__ pairs_out,
                                                                  uint32_t* __restrict__ keys_out, uint32_t* __restrict__ position) {
    extern __shared__ uint32_t next[];   // [digit][warp]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digits = 1u << p.bits;
    const uint32_t unit0 = blockIdx.x * kUnitWarps, unit = unit0 + warp;
    for (uint32_t i = threadIdx.x; i < digits * kUnitWarps; i += 32 * kUnitWarps) {
        const uint32_t w = i % kUnitWarps;
        if (unit0 + w < p.n_units) next[i] = __ldg(table + static_cast<size_t>(i / kUnitWarps) * p.n_units + unit0 + w);
    }
    __syncthreads();
    const size_t begin = static_cast<size_t>(unit) * p.unit, end = min(begin + p.unit, p.n);
    for (size_t s = begin; s < end; s += 32 * kSortAhead) {
        uint32_t key[kSortAhead], pair[kSortAhead];
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const size_t i = s + u * 32 + lane;
            const bool valid = i < end;
            key[u] = valid ? key_of(in, i, p.k) : 0u;
            pair[u] = valid && in.pairs ? __ldg(in.pairs + i) : static_cast<uint32_t>(i);
        }
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const bool valid = s + u * 32 + lane < end;
            const uint32_t digit = valid ? (key[u] >> p.shift) & (digits - 1) : 0xffffffffu;
            const uint32_t same = __match_any_sync(0xffffffffu, digit), rank = __popc(same & ((1u << lane) - 1u));
            if (valid) {
                const uint32_t slot = next[digit * kUnitWarps + warp] + rank;
                pairs_out[slot] = pair[u];
                if (keys_out) keys_out[slot] = key[u];
                if (position) position[pair[u]] = slot;
            }
            __syncwarp();
            if (valid && rank == 0) next[digit * kUnitWarps + warp] += __popc(same);
            __syncwarp();
        }
    }
}

// offsets[c] = first slot whose key is c or more
__global__ void __launch_bounds__(256) offsets_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t k, uint32_t* __restrict__ offsets) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c > k) return;
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (__ldg(keys + mid) < c) lo = mid + 1;
        else hi = mid;
    }
    offsets[c] = lo;
}

struct Plan {
    int passes, bits;
    uint32_t unit, n_units;
};
Plan make_plan(size_t n, size_t k) {
    int all = 1;
    while ((k >> all) != 0) ++all;   // keys are 0 .. k
    const int passes = (all + kMaxBits - 1) / kMaxBits;
    const uint32_t unit = n < (size_t{1} << 17) ? 128 : n < (size_t{1} << 20) ? 512 : n < (size_t{1} << 23) ? 2048 : 16384;
    return {passes, (all + passes - 1) / passes, unit, static_cast<uint32_t>((n + unit - 1) / unit)};
}
size_t rounded(size_t words) { return (words + 63) / 64 * 64; }

} // namespace

size_t group_workspace_bytes(size_t n, size_t k) {
    if (n <= kFewPairs) return 0;
    const Plan plan = make_plan(n, k);
    // digits' totals, the units' table, and between passes two copies of keys and pairs
    const size_t lists = plan.passes == 1 ? 0 : 4;
    return 4 * (rounded(size_t{1} << plan.bits) * plan.passes + rounded(static_cast<size_t>(plan.n_units) << plan.bits) + lists * rounded(n));
}

void launch_group(const Ids& ids, size_t n, size_t k, uint32_t* order, uint32_t* position, uint32_t* keys, uint32_t* offsets, void* workspace, cudaStream_t stream) {
    if (n == 0) {
        SKM_CUDA(cudaMemsetAsync(offsets, 0, (k + 1) * sizeof(uint32_t), stream));
        return;
    }
    if (n <= kFewPairs) {
        rank_kernel<<<static_cast<unsigned>((n + 31) / 32), 256, 0, stream>>>(ids.p, ids.wide, static_cast<uint32_t>(n), static_cast<uint32_t>(k), order, position, keys, offsets);
        SKM_LAUNCH_CHECK();
        return;
    }
    const Plan plan = make_plan(n, k);
    const size_t digits = size_t{1} << plan.bits;
    uint32_t* totals = static_cast<uint32_t*>(workspace);
    uint32_t* table = totals + rounded(digits) * plan.passes;
    uint32_t* lists = table + rounded(static_cast<size_t>(plan.n_units) << plan.bits);
    const unsigned blocks = (plan.n_units + kUnitWarps - 1) / kUnitWarps, shared = static_cast<unsigned>(digits * kUnitWarps * 4);
    SKM_CUDA(cudaMemsetAsync(totals, 0, rounded(digits) * plan.passes * 4, stream));
    PassInput in{ids.p, ids.wide, nullptr, nullptr};
    for (int pass = 0; pass < plan.passes; ++pass) {
        const bool last = pass == plan.passes - 1;
        const Pass p{n, static_cast<uint32_t>(k), pass * plan.bits, plan.bits, plan.n_units, plan.unit};
        uint32_t* keys_here = plan.passes == 1 ? keys : (last && keys) ? keys : lists + rounded(n) * 2 * (pass & 1);
        uint32_t* pairs_here = last ? order : lists + rounded(n) * (2 * (pass & 1) + 1);
        uint32_t* total = totals + rounded(digits) * pass;
        count_kernel<<<blocks, 32 * kUnitWarps, shared, stream>>>(in, p, table, total);
        SKM_LAUNCH_CHECK();
        place_kernel<<<static_cast<unsigned>((digits + 7) / 8), 256, 0, stream>>>(p, table, total, plan.passes == 1 ? offsets : nullptr);
        SKM_LAUNCH_CHECK();
        scatter_kernel<<<blocks, 32 * kUnitWarps, shared, stream>>>(in, p, table, pairs_here, keys_here, last ? position : nullptr);
        SKM_LAUNCH_CHECK();
        in.keys = keys_here;
        in.pairs = pairs_here;
    }
    if (plan.passes > 1) {
        offsets_kernel<<<static_cast<unsigned>(k / 256 + 1), 256, 0, stream>>>(in.keys, static_cast<uint32_t>(n), static_cast<uint32_t>(k), offsets);
        SKM_LAUNCH_CHECK();
    }
}

} // namespace rows
} // namespace skmb
