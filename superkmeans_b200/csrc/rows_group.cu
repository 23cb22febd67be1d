// Pairs (row, choice) in the order of their cluster: a stable sort of small numbers by counting.
//
// A few pairs: every pair's place is looked for among all others, in one launch over the whole chip; a launch is what the time of a small
// call consists of.
//
// More: a radix sort, up to 11 bits at a time.  A unit of a few hundred pairs belongs to a warp, which counts its digits in shared
// memory; a block for each digit turns the units' counts into places; and the units, read again, rank equal digits among 32 neighbours by
// __match_any_sync, in order, so that the sort is stable; no order of atomics matters.  Up to 2047 clusters need one pass.
#include <algorithm>

#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr size_t kFewPairs = 4096;
constexpr int kMaxBits = 11;
// Units of a block, whose tables are in shared memory: 16, where that leaves a block for each SM.
int unit_warps(int bits, size_t n_units) { return bits <= 9 && n_units >= 148 * 16 ? 16 : 4; }

// ---------------------------------------------------------------------------------------------- few pairs
// A key is the cluster and behind it the pair's number, so that no two are equal: a pair's slot is how many keys are less, and the
// largest of those says which cluster comes before.  Every block sorts all keys in groups of 32 (a warp a group, by exchanges between
// lanes) and then looks for the place of one group's keys, one to a lane, in all groups by halving.  (4096 pairs with 1000 clusters:
// 8 us a call; comparing every pair with every key, 13.)
constexpr uint32_t kRankWarps = 16;
constexpr uint32_t kRankAhead = 4;   // groups of a warp at a time
constexpr int kPairBits = 12;
static_assert(kFewPairs <= size_t{1} << kPairBits, "pairs' numbers fit their bits");

__global__ void __launch_bounds__(32 * kRankWarps) rank_kernel(const void* __restrict__ ids, bool wide, uint32_t n, uint32_t k, uint32_t* __restrict__ order, uint32_t* __restrict__ position,
                                                               uint32_t* __restrict__ keys_out, uint32_t* __restrict__ offsets) {
    wait_for_the_one_before();
    __shared__ uint32_t key[kFewPairs];
    __shared__ uint32_t parts[2][kRankWarps][32];
    __shared__ uint32_t fill[3][32];   // of each lane's pair: offsets fill[0] .. fill[1] become fill[2]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, groups = (n + 31) / 32;
    for (uint32_t g0 = warp; g0 < groups; g0 += kRankWarps * kRankAhead) {
        uint32_t v[kRankAhead];
#pragma unroll
        for (uint32_t u = 0; u < kRankAhead; ++u) {
            const uint32_t i = (g0 + u * kRankWarps) * 32 + lane;
            v[u] = i < n ? load_id(ids, wide, i, k) << kPairBits | i : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t size = 2; size <= 32; size *= 2)
#pragma unroll
            for (uint32_t apart = size / 2; apart > 0; apart /= 2) {
                const bool lower = ((lane & apart) == 0) == ((lane & size) == 0);
#pragma unroll
                for (uint32_t u = 0; u < kRankAhead; ++u) {
                    const uint32_t other = __shfl_xor_sync(0xffffffffu, v[u], apart);
                    v[u] = lower ? min(v[u], other) : max(v[u], other);
                }
            }
#pragma unroll
        for (uint32_t u = 0; u < kRankAhead; ++u)
            if (g0 + u * kRankWarps < groups) key[(g0 + u * kRankWarps) * 32 + lane] = v[u];
    }
    __syncthreads();
    const uint32_t own = key[blockIdx.x * 32 + lane];
    const bool mine = own != 0xffffffffu || blockIdx.x * 32 + lane < n;   // (the last group's gaps come last in it)
    uint32_t slot = 0, before = 0;   // keys that are less, and the largest of them
    for (uint32_t g0 = warp; g0 < groups; g0 += kRankWarps * kRankAhead) {
        uint32_t less[kRankAhead];
#pragma unroll
        for (uint32_t u = 0; u < kRankAhead; ++u) less[u] = 0;
#pragma unroll
        for (uint32_t half = 16; half > 0; half /= 2)
#pragma unroll
            for (uint32_t u = 0; u < kRankAhead; ++u) {
                const uint32_t g = g0 + u * kRankWarps;
                if (g < groups && key[g * 32 + less[u] + half - 1] < own) less[u] += half;
            }
#pragma unroll
        for (uint32_t u = 0; u < kRankAhead; ++u) {
            const uint32_t g = g0 + u * kRankWarps;
            if (g < groups) {
                if (key[g * 32 + less[u]] < own) ++less[u];   // (31 at most until here)
                if (less[u] > 0) before = max(before, key[g * 32 + less[u] - 1]);
                slot += less[u];
            }
        }
    }
    parts[0][warp][lane] = slot;
    parts[1][warp][lane] = before;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (uint32_t w = 1; w < kRankWarps; ++w) {
            slot += parts[0][w][lane];
            before = max(before, parts[1][w][lane]);
        }
        const uint32_t cluster = own >> kPairBits, pair = own & (kFewPairs - 1);
        if (mine) {
            order[slot] = pair;
            if (position) position[pair] = slot;
            if (keys_out) keys_out[slot] = cluster;
        }
        // the first pair of a cluster sets where the clusters behind the one before it begin
        fill[0][lane] = !mine ? 1u : slot == 0 ? 0u : (before >> kPairBits) + 1;
        fill[1][lane] = mine ? cluster : 0u;
        fill[2][lane] = slot;
    }
    __syncthreads();
    for (uint32_t l = warp; l < 32; l += kRankWarps) {
        const uint32_t from = fill[0][l], upto = fill[1][l], value = fill[2][l];
        for (uint32_t i = from + lane; i <= upto; i += 32) offsets[i] = value;
        // the last pair of all sets the rest
        if (value == n - 1 && blockIdx.x * 32 + l < n)
            for (uint32_t i = upto + 1 + lane; i <= k; i += 32) offsets[i] = n;
    }
}

bool few(size_t n, size_t k) { return n <= kFewPairs && k < (size_t{1} << (32 - kPairBits)); }

// ---------------------------------------------------------------------------------------------- many pairs
struct Pass {
    size_t n;
    uint32_t k;
    int shift, bits;
    uint32_t n_units, unit;   // a unit has this many pairs, a multiple of 32
    uint32_t pitch;           // of the table: units, rounded up to a multiple of 4
};

// What a pass sorts: the caller's ids (the first), or the pass before's keys and pairs.
struct PassInput {
    const void* ids;
    bool wide;
    const uint32_t* keys;
    const uint32_t* pairs;
};

__device__ __forceinline__ uint32_t key_of(const PassInput& in, size_t i, uint32_t k) { return in.keys ? __ldcg(in.keys + i) : load_id(in.ids, in.wide, i, k); }

constexpr int kSortAhead = 4;

// table[digit][unit] = the unit's pairs with that digit
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) count_kernel(const PassInput in, const Pass p, uint32_t* __restrict__ table) {
    wait_for_the_one_before();
    extern __shared__ uint32_t counts[];   // a row for each warp
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digits = 1u << p.bits, apart = digits + 1;
    for (uint32_t i = threadIdx.x; i < apart * WARPS; i += 32 * WARPS) counts[i] = 0;
    __syncthreads();
    const uint32_t unit0 = blockIdx.x * WARPS, unit = unit0 + warp;
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
            if (s + u * 32 + lane < end) atomicAdd(&counts[warp * apart + ((key[u] >> p.shift) & (digits - 1))], 1u);
    }
    __syncthreads();
    // WARPS neighbouring lanes have a digit (past the last unit, up to the pitch, its counts are zero)
    for (uint32_t i = threadIdx.x; i < digits * WARPS; i += 32 * WARPS) {
        const uint32_t digit = i / WARPS, w = i % WARPS;
        if (unit0 + w < p.pitch) table[static_cast<size_t>(digit) * p.pitch + unit0 + w] = counts[w * apart + digit];
    }
}

// table[digit][unit] = how many pairs of that digit the units before have, totals[digit] all; a block for each digit.
__global__ void __launch_bounds__(256) place_kernel(const Pass p, uint32_t* __restrict__ table, uint32_t* __restrict__ totals) {
    wait_for_the_one_before();
    __shared__ uint32_t sums[2][8];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint4* row = reinterpret_cast<uint4*>(table + static_cast<size_t>(blockIdx.x) * p.pitch);
    const uint32_t n4 = p.pitch / 4;
    uint4 v = threadIdx.x < n4 ? __ldcg(row + threadIdx.x) : make_uint4(0, 0, 0, 0);
    uint32_t before = 0;
    for (uint32_t s = 0; s < n4; s += 256) {
        const uint32_t i = s + threadIdx.x;
        const uint4 c = v;
        v = i + 256 < n4 ? __ldcg(row + i + 256) : make_uint4(0, 0, 0, 0);
        const uint32_t four = c.x + c.y + c.z + c.w;
        uint32_t upto = four;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= static_cast<uint32_t>(o)) upto += t;
        }
        if (lane == 31) sums[s / 256 & 1][warp] = upto;   // (the other half may still be read)
        __syncthreads();
        uint32_t here = before + upto - four;
#pragma unroll
        for (uint32_t w = 0; w < 8; ++w) {
            const uint32_t t = sums[s / 256 & 1][w];
            if (w < warp) here += t;
            before += t;
        }
        if (i < n4) row[i] = make_uint4(here, here + c.x, here + c.x + c.y, here + c.x + c.y + c.z);
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) scatter_kernel(const PassInput in, const Pass p, const uint32_t* __restrict__ table, const uint32_t* __restrict__ totals,
                                                             uint32_t* __restrict__ pairs_out, uint32_t* __restrict__ keys_out, uint32_t* __restrict__ position,
                                                             uint32_t* __restrict__ offsets) {
    wait_for_the_one_before();
    extern __shared__ uint32_t next[];   // a row for each warp
    __shared__ uint32_t sums[WARPS];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digits = 1u << p.bits, apart = digits + 1;
    const uint32_t unit0 = blockIdx.x * WARPS, unit = unit0 + warp;
    // where each digit begins: the totals before it, `each` neighbouring digits to a thread (offsets, if given: of the digits up to k)
    uint32_t* base = next + apart * WARPS;
    const uint32_t each = (digits + 32 * WARPS - 1) / (32 * WARPS), digit0 = threadIdx.x * each;
    uint32_t mine = 0;
    for (uint32_t e = 0; e < each && digit0 + e < digits; ++e) mine += __ldcg(totals + digit0 + e);
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= static_cast<uint32_t>(o)) upto += t;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    uint32_t slot0 = upto - mine;
    for (uint32_t w = 0; w < warp; ++w) slot0 += sums[w];
    for (uint32_t e = 0; e < each && digit0 + e < digits; ++e) {
        base[digit0 + e] = slot0;
        if (offsets && blockIdx.x == 0 && digit0 + e <= p.k) offsets[digit0 + e] = slot0;
        slot0 += __ldcg(totals + digit0 + e);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < digits * WARPS; i += 32 * WARPS) {
        const uint32_t w = i % WARPS, digit = i / WARPS;
        if (unit0 + w < p.n_units) next[w * apart + digit] = base[digit] + __ldcg(table + static_cast<size_t>(digit) * p.pitch + unit0 + w);
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
            pair[u] = valid && in.pairs ? __ldcg(in.pairs + i) : static_cast<uint32_t>(i);
        }
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const bool valid = s + u * 32 + lane < end;
            const uint32_t digit = valid ? (key[u] >> p.shift) & (digits - 1) : 0xffffffffu;
            const uint32_t same = __match_any_sync(0xffffffffu, digit), rank = __popc(same & ((1u << lane) - 1u));
            if (valid) {
                const uint32_t slot = next[warp * apart + digit] + rank;
                pairs_out[slot] = pair[u];
                if (keys_out) keys_out[slot] = key[u];
                if (position) position[pair[u]] = slot;
            }
            __syncwarp();
            if (valid && rank == 0) next[warp * apart + digit] += __popc(same);
            __syncwarp();
        }
    }
}

// offsets[c] = first slot whose key is c or more: where a key begins it sets those of the keys behind the one before, 32 lanes together
__global__ void __launch_bounds__(256) offsets_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t k, uint32_t* __restrict__ offsets) {
    wait_for_the_one_before();
    const uint32_t lane = threadIdx.x & 31, slot = blockIdx.x * 256 + threadIdx.x;
    const uint32_t key = slot < n ? __ldcg(keys + slot) : 0u, from = slot == 0 ? 0u : slot < n ? __ldcg(keys + slot - 1) + 1 : 1u;
    for (uint32_t left = __ballot_sync(0xffffffffu, slot < n && from <= key); left; left &= left - 1) {
        const int l = __ffs(left) - 1;
        const uint32_t f = __shfl_sync(0xffffffffu, from, l), t = __shfl_sync(0xffffffffu, key, l), v = __shfl_sync(0xffffffffu, slot, l);
        for (uint32_t c = f + lane; c <= t; c += 32) offsets[c] = v;
    }
    // behind the last key, by the grid
    for (uint32_t c = __ldcg(keys + n - 1) + 1 + slot; c <= k; c += gridDim.x * 256) offsets[c] = n;
}

struct Plan {
    int passes, bits;
    uint32_t unit, n_units;
};
Plan make_plan(size_t n, size_t k) {
    int all = 1;
    while ((k >> all) != 0) ++all;   // keys are 0 .. k
    const int passes = (all + kMaxBits - 1) / kMaxBits;
    const int bits = (all + passes - 1) / passes;
    // about 4096 units (so many warps hide the latency of what they read), but no table that is larger than the lists by far
    const size_t most = std::min<size_t>(4096, (size_t{1} << 20) >> bits);
    const size_t unit = std::max<size_t>(128, (n + most - 1) / most);
    const uint32_t rounded = static_cast<uint32_t>((unit + 127) / 128 * 128);
    return {passes, bits, rounded, static_cast<uint32_t>((n + rounded - 1) / rounded)};
}
size_t pitch_of(const Plan& plan) { return (plan.n_units + 3) / 4 * 4; }
size_t rounded(size_t words) { return (words + 63) / 64 * 64; }

} // namespace

size_t group_workspace_bytes(size_t n, size_t k) {
    if (n == 0 || few(n, k)) return 0;
    const Plan plan = make_plan(n, k);
    // digits' totals, the units' table, and between passes two copies of keys and pairs
    const size_t lists = plan.passes == 1 ? 0 : 4;
    return 4 * (rounded(size_t{1} << plan.bits) + rounded(pitch_of(plan) << plan.bits) + lists * rounded(n));
}

void launch_group(const Ids& ids, size_t n, size_t k, uint32_t* order, uint32_t* position, uint32_t* keys, uint32_t* offsets, void* workspace, cudaStream_t stream) {
    if (n == 0) {
        SKM_CUDA(cudaMemsetAsync(offsets, 0, (k + 1) * sizeof(uint32_t), stream));
        return;
    }
    if (few(n, k)) {
        launch_after(rank_kernel, dim3(static_cast<unsigned>((n + 31) / 32)), 32 * kRankWarps, 0, stream, ids.p, ids.wide, static_cast<uint32_t>(n), static_cast<uint32_t>(k), order,
                     position, keys, offsets);
        return;
    }
    const Plan plan = make_plan(n, k);
    const size_t digits = size_t{1} << plan.bits;
    uint32_t* totals = static_cast<uint32_t*>(workspace);
    uint32_t* table = totals + rounded(digits);
    uint32_t* lists = table + rounded(pitch_of(plan) << plan.bits);
    const unsigned warps = static_cast<unsigned>(unit_warps(plan.bits, plan.n_units)), blocks = (plan.n_units + warps - 1) / warps, shared = static_cast<unsigned>((digits + 1) * warps * 4);
    PassInput in{ids.p, ids.wide, nullptr, nullptr};
    for (int pass = 0; pass < plan.passes; ++pass) {
        const bool last = pass == plan.passes - 1;
        const Pass p{n, static_cast<uint32_t>(k), pass * plan.bits, plan.bits, plan.n_units, plan.unit, static_cast<uint32_t>(pitch_of(plan))};
        uint32_t* keys_here = plan.passes == 1 ? keys : (last && keys) ? keys : lists + rounded(n) * 2 * (pass & 1);
        uint32_t* pairs_here = last ? order : lists + rounded(n) * (2 * (pass & 1) + 1);
        launch_after(warps == 16 ? count_kernel<16> : count_kernel<4>, dim3(blocks), 32 * warps, shared, stream, in, p, table);
        launch_after(place_kernel, dim3(static_cast<unsigned>(digits)), 256, 0, stream, p, table, totals);
        launch_after(warps == 16 ? scatter_kernel<16> : scatter_kernel<4>, dim3(blocks), 32 * warps, shared + digits * 4, stream, in, p, table, totals, pairs_here, keys_here,
                     last ? position : nullptr, plan.passes == 1 ? offsets : nullptr);
        in.keys = keys_here;
        in.pairs = pairs_here;
    }
    if (plan.passes > 1) {
        launch_after(offsets_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), 256, 0, stream, in.keys, static_cast<uint32_t>(n), static_cast<uint32_t>(k), offsets);
    }
}

} // namespace rows
} // namespace skmb
