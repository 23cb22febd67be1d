// Operators on rows in device memory (rows_group.cu, rows_move.cu, rows_sum.cu, product_8bit.cu): lookup in a table by id and its
// gradient, rows to the places of their clusters and back, products of rows in 8 bits.  All are asynchronous on the caller's
// stream, allocate nothing and read nothing back, so that they can be captured into a graph: what they need beyond inputs and
// outputs is a workspace that the caller passes.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace skmb {
namespace rows {

enum class Type { f32 = 0, f16 = 1, bf16 = 2 };
inline size_t type_bytes(Type t) { return t == Type::f32 ? 4 : 2; }

// Rows of d values, `ld` elements from one to the next.
struct Rows {
    const void* p;
    size_t ld;
};

// Cluster numbers: 32 bits (signed or not) or 64.  One outside [0, k) stands for no cluster.
struct Ids {
    const void* p;
    bool wide;
};

// ---- rows_group.cu
// Stable sort of the pairs 0 .. n-1 by ids[i]; those without a cluster come last.  order[slot] = pair, position[pair] = slot (may be
// null), keys[slot] = cluster or k (may be null), offsets[c] = first slot of cluster c for c in [0, k].  n and k below 2^31.
size_t group_workspace_bytes(size_t n, size_t k);
void launch_group(const Ids& ids, size_t n, size_t k, uint32_t* order, uint32_t* position, uint32_t* keys, uint32_t* offsets, void* workspace, cudaStream_t stream);

// ---- rows_move.cu
// out[i] = scale * row_scales[i] * table[ids[i]] (row_scales may be null), zeros where the id is none
void launch_lookup(const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, const float* row_scales, void* out, cudaStream_t stream);
// out[i] = scale * <grad[i], table[ids[i]]>, zero where the id is none
void launch_lookup_scale_grad(const Rows& grad, const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, float* out, cudaStream_t stream);
// A grouping of n rows with m choices each, as launch_group leaves it: *held slots (= offsets[k]) have a cluster.
struct Places {
    const uint32_t* order;      // n x m: which pair is in a slot
    const uint32_t* position;   // n x m: which slot a pair has
    const uint32_t* held;
    size_t n, m;                // n * m below 2^31; a slot of n * m or more is passed over
};
// out[position[i][j]] = x[i]; zeros in the slots behind *held
void launch_to_clusters(const Rows& x, Type type, size_t d, const Places& at, void* out, cudaStream_t stream);
// out[i] = sum over j of weights[i][j] * y[position[i][j]] (weights null: 1), over the choices that have a cluster
void launch_from_clusters(const Rows& y, Type type, size_t d, const Places& at, const float* weights, void* out, cudaStream_t stream);
// grad_y[position[i][j]] = weights[i][j] * grad[i], zeros behind *held; grad_weights[i][j] = <grad[i], y[position[i][j]]>, zero without a
// cluster.  Either output may be null; y is read for grad_weights only.
void launch_from_clusters_grad(const Rows& grad, const Rows& y, Type type, size_t d, const Places& at, const float* weights, void* grad_y, float* grad_weights, cudaStream_t stream);

// ---- rows_unaligned.cu: the same for rows whose address, pitch or length is no multiple of 16 bytes (of 32 bytes or more; outputs begin
// on 16 bytes)
void launch_lookup_unaligned(const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, const float* row_scales, void* out, cudaStream_t stream);
void launch_lookup_scale_grad_unaligned(const Rows& grad, const Rows& table, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, float* out, cudaStream_t stream);
void launch_to_clusters_unaligned(const Rows& x, Type type, size_t d, const Places& at, const float* weights, void* out, cudaStream_t stream);   // (scaled by the pair's weight, if given)
void launch_from_clusters_unaligned(const Rows& y, Type type, size_t d, const Places& at, const float* weights, void* out, cudaStream_t stream);
void launch_weights_grad_unaligned(const Rows& grad, const Rows& y, Type type, size_t d, const Places& at, float* grad_weights, cudaStream_t stream);

// ---- rows_sum.cu
// out[c] = sum over ids[i] = c of scale * row_scales[i] * grad[i] for c in [0, k), added in a fixed order
size_t lookup_grad_workspace_bytes(size_t n, size_t k, size_t d, Type type);
void launch_lookup_grad(const Rows& grad, Type type, size_t k, size_t d, const Ids& ids, size_t n, float scale, const float* row_scales, void* out, Type out_type, void* workspace,
                        cudaStream_t stream);

// ---- product_8bit.cu
// q[i][j] = rint(x[i][j] * (127 / most)), scales[i] = most / 127 with most = max_j |x[i][j]|; a row of zeros has scale 0, a row with a value
// that is no finite number zeros and the scale NaN.  ldq: bytes from one row of q to the next.
void launch_quantize_rows(const Rows& x, Type type, size_t n, size_t d, int8_t* q, size_t ldq, float* scales, cudaStream_t stream);

struct Product {
    const int8_t* x;             // n rows of d bytes, ldx bytes from one to the next
    size_t ldx;
    const float* x_scales;       // n
    const int8_t* w;             // m rows of d bytes, ldw apart; with groups `groups` times as many
    size_t ldw;
    const float* w_scales;       // m, with groups as many for each
    size_t n, m, d;
    size_t groups;               // 0: none
    const uint32_t* offsets;     // groups + 1: rows offsets[g] .. offsets[g + 1] - 1 are group g's; the others' results are zeros
    void* out;                   // n x m
    Type out_type;
};
constexpr size_t kMaxProductDepth = 131071;   // 128 * 128 * d < 2^31
size_t product_workspace_bytes(const Product& p);
// out[i][c] = x_scales[i] * w_scales[c] * sum_j x[i][j] * w[c][j]; the sum is exact.  Throws if an earlier product's wait ran out.
void launch_product(const Product& p, void* workspace, cudaStream_t stream);
// Throws if a wait of a product on the current device has run out and nobody was told.  Waits for the stream.
void check_products(cudaStream_t stream);

} // namespace rows
} // namespace skmb
