// Pairs (row, choice) in the order of their cluster: a stable sort of small numbers by counting.
//
// A few pairs: every pair's place is looked for among all others, in one launch over the whole chip; a launch is what the time of a small
// call consists of.
//
// More, and up to some 18 000 clusters: a counting sort in three launches.  A block has a part of the pairs and counts its clusters in
// shared memory; the counts of all blocks become places; and the block gives each of its pairs a place, in order, so that the sort is
// stable; no order of atomics matters.  Up to 1023 clusters it sorts 4096 pairs at a time in shared memory; with more, its warps have
// a part each, count again for every warp (two bytes a cluster), add up, and rank equal clusters among 32 neighbours by
// __match_any_sync.  One B200, a call: 262 144 pairs with 255 clusters 11.5 us (one pass of the radix sort 26), 300 000 with 5000 18 (two passes
// 36), 4M with 1000 78 (255).  What bounds it is the latency of each launch's few reads, and from a million pairs on the scattered stores.
//
// More clusters, or very many pairs: a radix sort of the same kind, up to 11 bits at a time.  A unit of a few hundred pairs belongs to a warp, which counts its digits in shared
// memory; a block for each digit turns the units' counts into places; and the units, read again, rank equal digits as above.
#include <algorithm>

#include "rows_access.cuh"

namespace skmb {
namespace rows {

namespace {

constexpr size_t kFewPairs = 4096;
constexpr int kMaxBits = 11;
// Units of a block, whose tables are in shared memory: 16, where that leaves a block for each SM (300 000 pairs of 5M clusters 130 us, with four
// 134; 10M of 60 000 945 and 907).
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

// (the gaps between clusters that somebody has are filled by a warp each: not too many clusters.  64 pairs with 16 clusters 2.3 us and by the three
// launches below 7.2, 4096 with 16 6.5 and 8.2, with 60 000 6.8 and 25.)
bool few(size_t n, size_t k) { return n <= kFewPairs && k <= 65536; }
static_assert(65536 < (size_t{1} << (32 - kPairBits)), "clusters fit the bits that are left");

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

__device__ __forceinline__ uint32_t key_of(const PassInput& in, size_t i, uint32_t k) { return in.keys ? load_new(in.keys + i) : load_id(in.ids, in.wide, i, k); }

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
    uint4 v = threadIdx.x < n4 ? load_new(row + threadIdx.x) : make_uint4(0, 0, 0, 0);
    uint32_t before = 0;
    for (uint32_t s = 0; s < n4; s += 256) {
        const uint32_t i = s + threadIdx.x;
        const uint4 c = v;
        v = i + 256 < n4 ? load_new(row + i + 256) : make_uint4(0, 0, 0, 0);
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
    for (uint32_t e = 0; e < each && digit0 + e < digits; ++e) mine += load_new(totals + digit0 + e);
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
        slot0 += load_new(totals + digit0 + e);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < digits * WARPS; i += 32 * WARPS) {
        const uint32_t w = i % WARPS, digit = i / WARPS;
        if (unit0 + w < p.n_units) next[w * apart + digit] = base[digit] + load_new(table + static_cast<size_t>(digit) * p.pitch + unit0 + w);
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
            pair[u] = valid && in.pairs ? load_new(in.pairs + i) : static_cast<uint32_t>(i);
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
    const uint32_t key = slot < n ? load_new(keys + slot) : 0u, from = slot == 0 ? 0u : slot < n ? load_new(keys + slot - 1) + 1 : 1u;
    for (uint32_t left = __ballot_sync(0xffffffffu, slot < n && from <= key); left; left &= left - 1) {
        const int l = __ffs(left) - 1;
        const uint32_t f = __shfl_sync(0xffffffffu, from, l), t = __shfl_sync(0xffffffffu, key, l), v = __shfl_sync(0xffffffffu, slot, l);
        for (uint32_t c = f + lane; c <= t; c += 32) offsets[c] = v;
    }
    // behind the last key, by the grid
    for (uint32_t c = load_new(keys + n - 1) + 1 + slot; c <= k; c += gridDim.x * 256) offsets[c] = n;
}

// ---------------------------------------------------------------------------------------------- many pairs, not too many clusters
struct Direct {
    uint32_t n, k;
    uint32_t digits, pitch;      // clusters and none; of a row of the table, in words
    uint32_t blocks, units;      // units: parts of a block's pairs, a warp's each
    uint32_t share;              // pairs of a unit, a multiple of 32
    uint32_t half_pitch;         // of a unit's counts, in words of two
};
constexpr uint32_t kDirectThreads = 1024;
constexpr size_t kDirectShared = 220 * 1024;

// table[block][cluster] = the block's pairs with it
__global__ void __launch_bounds__(kDirectThreads) direct_count_kernel(const void* __restrict__ ids, bool wide, const Direct p, uint32_t* __restrict__ table) {
    wait_for_the_one_before();
    extern __shared__ uint32_t counts[];
    for (uint32_t i = threadIdx.x; i < p.digits; i += kDirectThreads) counts[i] = 0;
    __syncthreads();
    const size_t begin = static_cast<size_t>(blockIdx.x) * p.units * p.share, end = min(begin + static_cast<size_t>(p.units) * p.share, static_cast<size_t>(p.n));
    for (size_t s = begin; s < end; s += kDirectThreads * kSortAhead) {
        uint32_t key[kSortAhead];
#pragma unroll
        for (uint32_t u = 0; u < kSortAhead; ++u) {
            const size_t i = s + u * kDirectThreads + threadIdx.x;
            key[u] = i < end ? load_id(ids, wide, i, p.k) : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t u = 0; u < kSortAhead; ++u)
            if (key[u] != 0xffffffffu) atomicAdd(&counts[key[u]], 1u);
    }
    __syncthreads();
    uint32_t* row = table + static_cast<size_t>(blockIdx.x) * p.pitch;
    for (uint32_t i = threadIdx.x; i < p.digits; i += kDirectThreads) row[i] = counts[i];
}

// table[block][cluster] = how many pairs of the cluster the blocks before have, totals[cluster] all; 32 clusters to a block, whose
// warps have a part of the table's rows each
__global__ void __launch_bounds__(kDirectThreads) direct_place_kernel(const Direct p, uint32_t* __restrict__ table, uint32_t* __restrict__ totals) {
    wait_for_the_one_before();
    __shared__ uint32_t sums[32][33];
    constexpr uint32_t MOST = 8;   // rows of a warp (256 blocks at most)
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digit = blockIdx.x * 32 + lane;
    const uint32_t each = (p.blocks + 31) / 32, row0 = warp * each;
    uint32_t v[MOST], sum = 0;
#pragma unroll
    for (uint32_t r = 0; r < MOST; ++r) {
        v[r] = r < each && row0 + r < p.blocks && digit < p.digits ? load_new(table + static_cast<size_t>(row0 + r) * p.pitch + digit) : 0u;
        sum += v[r];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t w = 0; w < warp; ++w) before += sums[w][lane];
    if (digit >= p.digits) return;
    if (warp == 31) totals[digit] = before + sum;
#pragma unroll
    for (uint32_t r = 0; r < MOST; ++r)
        if (r < each && row0 + r < p.blocks) {
            table[static_cast<size_t>(row0 + r) * p.pitch + digit] = before;
            before += v[r];
        }
}

__global__ void __launch_bounds__(kDirectThreads) direct_scatter_kernel(const void* __restrict__ ids, bool wide, const Direct p, const uint32_t* __restrict__ table,
                                                                        const uint32_t* __restrict__ totals, uint32_t* __restrict__ order, uint32_t* __restrict__ position,
                                                                        uint32_t* __restrict__ keys_out, uint32_t* __restrict__ offsets) {
    wait_for_the_one_before();
    extern __shared__ uint32_t shared[];
    __shared__ uint32_t sums[32];
    uint32_t* base = shared;                  // of each cluster: the slot of the block's first pair with it
    uint32_t* halves = shared + p.digits;     // of each unit and cluster, two bytes: pairs of the block in the units before, and what was ranked
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t begin = static_cast<size_t>(blockIdx.x) * p.units * p.share;
    constexpr uint32_t AHEAD = 8;
    for (uint32_t i0 = threadIdx.x; i0 < p.digits; i0 += kDirectThreads * AHEAD) {
        uint32_t v[AHEAD];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u) v[u] = i0 + u * kDirectThreads < p.digits ? load_new(totals + i0 + u * kDirectThreads) : 0u;
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; ++u)
            if (i0 + u * kDirectThreads < p.digits) base[i0 + u * kDirectThreads] = v[u];
    }
    for (uint32_t i = threadIdx.x; i < p.units * p.half_pitch; i += kDirectThreads) halves[i] = 0;
    __syncthreads();
    // counts of the units: all warps, `helpers` of them for a unit
    const uint32_t unit = warp % p.units, helpers = 32 / p.units, helper = warp / p.units;
    const size_t u0 = begin + static_cast<size_t>(unit) * p.share, u1 = min(u0 + p.share, static_cast<size_t>(p.n));
    for (size_t s = u0 + helper * 32; s < u1; s += 32 * helpers * kSortAhead) {
        uint32_t key[kSortAhead];
#pragma unroll
        for (uint32_t u = 0; u < kSortAhead; ++u) {
            const size_t i = s + u * 32 * helpers + lane;
            key[u] = i < u1 ? load_id(ids, wide, i, p.k) : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t u = 0; u < kSortAhead; ++u)
            if (key[u] != 0xffffffffu) atomicAdd(&halves[unit * p.half_pitch + key[u] / 2], 1u << (key[u] % 2 * 16));
    }
    // where each cluster begins: the totals before it, some neighbouring ones to a thread
    const uint32_t each = ((p.digits + kDirectThreads - 1) / kDirectThreads) | 1, digit0 = threadIdx.x * each;   // (odd: no two lanes in a bank)
    uint32_t mine = 0;
    for (uint32_t e = 0; e < each && digit0 + e < p.digits; ++e) mine += base[digit0 + e];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= static_cast<uint32_t>(o)) upto += t;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    uint32_t slot = upto - mine;
    for (uint32_t w = 0; w < warp; ++w) slot += sums[w];
    for (uint32_t e = 0; e < each && digit0 + e < p.digits; ++e) {
        const uint32_t here = base[digit0 + e];
        base[digit0 + e] = slot;
        slot += here;
    }
    __syncthreads();
    uint16_t* rank = reinterpret_cast<uint16_t*>(halves);
    for (uint32_t i0 = threadIdx.x; i0 < p.digits; i0 += kDirectThreads * AHEAD) {
        uint32_t v[AHEAD];
#pragma unroll
        for (uint32_t e = 0; e < AHEAD; ++e) {
            const uint32_t i = i0 + e * kDirectThreads;
            v[e] = i < p.digits ? load_new(table + static_cast<size_t>(blockIdx.x) * p.pitch + i) : 0u;
        }
#pragma unroll
        for (uint32_t e = 0; e < AHEAD; ++e) {
            const uint32_t i = i0 + e * kDirectThreads;
            if (i >= p.digits) break;
            if (blockIdx.x == 0) offsets[i] = base[i];
            base[i] += v[e];
            uint32_t before = 0;
            for (uint32_t u = 0; u < p.units; ++u) {
                uint16_t& at = rank[u * p.half_pitch * 2 + i];
                const uint32_t count = at;
                at = static_cast<uint16_t>(before);
                before += count;
            }
        }
    }
    __syncthreads();
    if (warp >= p.units) return;
    rank += warp * p.half_pitch * 2;
    uint32_t* counts = halves + warp * p.half_pitch;
    for (size_t s = u0; s < u1; s += 32 * kSortAhead) {
        uint32_t key[kSortAhead];
#pragma unroll
        for (uint32_t u = 0; u < kSortAhead; ++u) {
            const size_t i = s + u * 32 + lane;
            key[u] = i < u1 ? load_id(ids, wide, i, p.k) : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t u = 0; u < kSortAhead; ++u) {
            const bool valid = key[u] != 0xffffffffu;
            // counted by all 32 at once; only if that finds two of the same do they have to be ranked
            uint32_t before = 0, ahead = 0;
            if (valid) before = rank[key[u]];
            __syncwarp();
            if (valid) atomicAdd(&counts[key[u] / 2], 1u << (key[u] % 2 * 16));
            __syncwarp();
            if (__any_sync(0xffffffffu, valid && rank[key[u]] != before + 1)) ahead = __popc(__match_any_sync(0xffffffffu, key[u]) & ((1u << lane) - 1u));
            if (valid) {
                const uint32_t to = base[key[u]] + before + ahead, pair = static_cast<uint32_t>(s + u * 32 + lane);
                order[to] = pair;
                if (keys_out) keys_out[to] = key[u];
                if (position) position[pair] = to;
            }
            __syncwarp();
        }
    }
}

// Up to 1023 clusters: 4096 of a block's pairs at a time are sorted by cluster in shared memory, after which neighbours have neighbouring
// places and both lists are written in runs.  With few clusters the warps of direct_scatter_kernel rank nearly every 32 pairs by
// __match_any_sync and write each place by itself.  A call with this kernel and with that one: 262 144 pairs with 16 clusters 10.1 and 12.1 us,
// with 255 11.5 and 17.4, with 1000 13.7 and 20.1; 4M with 255 66 and 87; 10 000 with 256 10.6 both; 30 000 with 256 10.9 and 10.1; 12M with 16 182 and 168.
// With more clusters a chunk takes two passes, and 300 000 with 5000 20 and 18, 9M 236 and 150.
constexpr uint32_t kSortedEach = 4, kSortedChunk = kDirectThreads * kSortedEach, kSortedWarps = kDirectThreads / 32;
template <uint32_t DIGITS>
constexpr uint32_t kSortedApart = DIGITS + 2;   // from one warp's counts to the next's
template <uint32_t DIGITS>
constexpr uint32_t kSortedShared = 4 * DIGITS + 2 * (2 * kSortedChunk + kSortedWarps * kSortedApart<DIGITS>);

template <uint32_t DIGITS>
__global__ void __launch_bounds__(kDirectThreads) direct_sorted_kernel(const void* __restrict__ ids, bool wide, const Direct p, const uint32_t* __restrict__ table,
                                                                       const uint32_t* __restrict__ totals, uint32_t* __restrict__ order, uint32_t* __restrict__ position,
                                                                       uint32_t* __restrict__ keys_out, uint32_t* __restrict__ offsets) {
    wait_for_the_one_before();
    constexpr uint32_t APART = kSortedApart<DIGITS>;
    static_assert(2 * kSortedWarps * APART >= 4 * kSortedChunk, "the slots have room where the counts were");
    extern __shared__ uint32_t shared[];
    __shared__ uint32_t sums[kSortedWarps];
    uint32_t* base = shared;                                                  // of each cluster: the slot of the block's next pair with it
    uint16_t* sorted_key = reinterpret_cast<uint16_t*>(shared + DIGITS);
    uint16_t* sorted_pair = sorted_key + kSortedChunk;                        // (its number in the chunk)
    uint16_t* counts = sorted_pair + kSortedChunk;                            // of each warp and cluster
    uint32_t* slots = reinterpret_cast<uint32_t*>(counts);                    // of the chunk's pairs
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t share = static_cast<size_t>(p.units) * p.share, begin = blockIdx.x * share, end = min(begin + share, static_cast<size_t>(p.n));
    auto sum_before = [&](uint32_t mine) {   // of the threads before this one; a barrier lies between a call's end and the next call
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= static_cast<uint32_t>(o)) upto += t;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        uint32_t of_warps = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, of_warps, o);
            if (lane >= static_cast<uint32_t>(o)) of_warps += t;
        }
        const uint32_t before = __shfl_sync(0xffffffffu, of_warps, warp == 0 ? 0 : warp - 1);
        return upto - mine + (warp == 0 ? 0u : before);
    };
    // a warp has 128 neighbouring pairs of a chunk
    const uint32_t item0 = warp * 32 * kSortedEach + lane;
    uint32_t id[kSortedEach];
    auto fetch = [&](size_t chunk0) {
#pragma unroll
        for (uint32_t u = 0; u < kSortedEach; ++u) id[u] = chunk0 + item0 + u * 32 < end ? load_id(ids, wide, chunk0 + item0 + u * 32, p.k) : 0u;
    };
    fetch(begin);
    // where each cluster begins, and the block's part of it
    const bool has = threadIdx.x < p.digits;
    const uint32_t total = has ? load_new(totals + threadIdx.x) : 0u, before_block = has ? load_new(table + static_cast<size_t>(blockIdx.x) * p.pitch + threadIdx.x) : 0u;
    const uint32_t slot0 = sum_before(total);
    if (has) {
        if (blockIdx.x == 0) offsets[threadIdx.x] = slot0;
        base[threadIdx.x] = slot0 + before_block;
    }
    for (size_t chunk0 = begin; chunk0 < end; chunk0 += kSortedChunk) {
        const uint32_t count = static_cast<uint32_t>(min(static_cast<size_t>(kSortedChunk), end - chunk0));
        for (uint32_t i = threadIdx.x; i < kSortedWarps * APART / 2; i += kDirectThreads) slots[i] = 0;
        __syncthreads();
        uint16_t* row = counts + warp * APART;
        uint32_t rank[kSortedEach];
#pragma unroll
        for (uint32_t u = 0; u < kSortedEach; ++u) {
            const bool valid = item0 + u * 32 < count;
            const uint32_t same = __match_any_sync(0xffffffffu, valid ? id[u] : 0xffffffffu), ahead = __popc(same & ((1u << lane) - 1u));
            uint32_t before = 0;
            if (valid) before = row[id[u]];
            __syncwarp();
            if (valid && ahead == 0) row[id[u]] = static_cast<uint16_t>(before + __popc(same));
            __syncwarp();
            rank[u] = before + ahead;
        }
        __syncthreads();
        // the counts become places: a cluster's of WARPS warps to a thread
        constexpr uint32_t PARTS = kDirectThreads / DIGITS, WARPS = kSortedWarps / PARTS;
        uint16_t* column = counts + threadIdx.x % PARTS * WARPS * APART + threadIdx.x / PARTS;
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w) sum += column[w * APART];
        uint32_t place = sum_before(sum);
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w) {
            const uint32_t here = column[w * APART];
            column[w * APART] = static_cast<uint16_t>(place);
            place += here;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < kSortedEach; ++u)
            if (item0 + u * 32 < count) {
                const uint32_t to = row[id[u]] + rank[u];
                sorted_key[to] = static_cast<uint16_t>(id[u]);
                sorted_pair[to] = static_cast<uint16_t>(item0 + u * 32);
            }
        __syncthreads();
        fetch(chunk0 + kSortedChunk);
        // a cluster's place less that of its first pair here, which leaves each pair to add its own; and behind its last one
        uint32_t key[kSortedEach];
        bool last[kSortedEach];
#pragma unroll
        for (uint32_t u = 0; u < kSortedEach; ++u) {
            const uint32_t i = threadIdx.x + u * kDirectThreads;
            if (i >= count) break;
            key[u] = sorted_key[i];
            last[u] = i + 1 == count || sorted_key[i + 1] != key[u];
            if (i == 0 || sorted_key[i - 1] != key[u]) base[key[u]] -= i;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < kSortedEach; ++u) {
            const uint32_t i = threadIdx.x + u * kDirectThreads;
            if (i >= count) break;
            const uint32_t slot = base[key[u]] + i, in_chunk = sorted_pair[i];
            order[slot] = static_cast<uint32_t>(chunk0) + in_chunk;
            if (keys_out) keys_out[slot] = key[u];
            slots[in_chunk] = slot;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < kSortedEach; ++u) {
            const uint32_t i = threadIdx.x + u * kDirectThreads;
            if (i >= count) break;
            if (last[u]) base[key[u]] += i + 1;
            if (position) position[chunk0 + i] = slots[i];
        }
        __syncthreads();   // (the next counts are where the slots are)
    }
}

// Whether the pairs are sorted so, and how.  The sizes alone decide: a workspace is asked for before a device is current.
constexpr size_t kDirectBlocks = 148;   // one to an SM

bool make_direct(size_t n, size_t k, Direct& p) {
    const size_t digits = k + 1;
    if (digits * 12 + 4 * 4 > kDirectShared) return false;
    p.digits = static_cast<uint32_t>(digits);
    p.half_pitch = static_cast<uint32_t>((digits + 1) / 2);
    p.units = 32;
    while (p.units > 4 && 4 * (digits + static_cast<size_t>(p.units) * p.half_pitch) > kDirectShared) p.units /= 2;
    if (4 * (digits + static_cast<size_t>(p.units) * p.half_pitch) > kDirectShared) return false;
    p.blocks = static_cast<uint32_t>(std::min(kDirectBlocks, (n + 1023) / 1024));
    const size_t share = (n + static_cast<size_t>(p.blocks) * p.units - 1) / (static_cast<size_t>(p.blocks) * p.units);
    p.share = static_cast<uint32_t>((share + 31) / 32 * 32);
    p.n = static_cast<uint32_t>(n);
    p.k = static_cast<uint32_t>(k);
    p.pitch = static_cast<uint32_t>((digits + 31) / 32 * 32);
    return digits <= 1024 || static_cast<size_t>(p.units) * p.share < 65536;   // (what two bytes hold)
}

// The same by looking each cluster up, for far more clusters than pairs: where few have pairs, the gaps that a warp fills are long (one pair with 3M
// clusters 56 us, by the kernel above 540; where the pairs are spread evenly that one is the faster: 300 000 with 5M 134 and 69).
__global__ void __launch_bounds__(256) offsets_search_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t k, uint32_t* __restrict__ offsets) {
    wait_for_the_one_before();
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c > k) return;
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (load_new(keys + mid) < c) lo = mid + 1;
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
    Direct direct{};
    if (make_direct(n, k, direct)) return 4 * (rounded(direct.digits) + static_cast<size_t>(direct.blocks) * direct.pitch);
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
    Direct direct{};
    if (make_direct(n, k, direct)) {
        uint32_t* totals = static_cast<uint32_t*>(workspace);
        uint32_t* table = totals + rounded(direct.digits);
        const uint32_t shared = 4 * (direct.digits + direct.units * direct.half_pitch);
        allow_shared(direct_count_kernel, kDirectShared);
        allow_shared(direct_scatter_kernel, kDirectShared);
        launch_after(direct_count_kernel, dim3(direct.blocks), kDirectThreads, 4 * direct.digits, stream, ids.p, ids.wide, direct, table);
        launch_after(direct_place_kernel, dim3((direct.digits + 31) / 32), kDirectThreads, 0, stream, direct, table, totals);
        auto sorted = [&](auto digits) {
            auto* kernel = direct_sorted_kernel<decltype(digits)::value>;
            allow_shared(kernel, kSortedShared<decltype(digits)::value>);
            launch_after(kernel, dim3(direct.blocks), kDirectThreads, kSortedShared<decltype(digits)::value>, stream, ids.p, ids.wide, direct, table, totals, order, position, keys, offsets);
        };
        if (direct.digits <= 256) sorted(std::integral_constant<uint32_t, 256>{});
        else if (direct.digits <= 1024) sorted(std::integral_constant<uint32_t, 1024>{});
        else launch_after(direct_scatter_kernel, dim3(direct.blocks), kDirectThreads, shared, stream, ids.p, ids.wide, direct, table, totals, order, position, keys, offsets);
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
    if (plan.passes > 1 && k / 16 > n) {
        launch_after(offsets_search_kernel, dim3(static_cast<unsigned>(k / 256 + 1)), 256, 0, stream, in.keys, static_cast<uint32_t>(n), static_cast<uint32_t>(k), offsets);
    } else if (plan.passes > 1) {
        launch_after(offsets_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), 256, 0, stream, in.keys, static_cast<uint32_t>(n), static_cast<uint32_t>(k), offsets);
    }
}

} // namespace rows
} // namespace skmb
