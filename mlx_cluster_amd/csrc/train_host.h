// Host-side internals of the training operators: what their launchers and host
// twins take.  Nothing here is part of the C ABI (include/mlxc_train.h).
#pragma once

#include "train_device.h"
#include "walk_host.h"

namespace mlxc {

// A table of rows.
struct Table {
    const void* p;
    int64_t num_rows;
    int64_t row_stride;
    int32_t dim;
    int32_t dtype;
};

// The walks of a window call.
struct Walks {
    Nodes nodes;
    int64_t num_walks;
    int32_t walk_nodes;
    int32_t ctx;
    __host__ __device__ int64_t windows() const { return walk_nodes - ctx + 1; }
    __host__ __device__ int64_t count() const { return num_walks * walk_nodes; }
};

// Where a gradient goes: rows by node (ids null), or coalesced.
struct GradOut {
    void* p;
    int64_t* ids;
    int32_t dtype;
};

inline size_t elem_bytes(int32_t dtype) { return dtype == MLXC_FLOAT32 ? 4 : 2; }

// The largest number of elements, a power of two of at most `most`, whose
// packs lie aligned in rows of dim elements of esz bytes at p, stride apart.
inline int pack_width(const void* p, int64_t dim, int64_t stride, size_t esz, int most) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(p) | (dim * esz) | (stride * esz) | 16;
    int n = most;
    while (n > 1 && all % (n * esz) != 0) n /= 2;
    return n;
}

// ---- place_sort.hip
// Places of a call sorted by node, in ascending order where nodes are equal;
// places without a node are left out.
struct SortedPlaces {
    const uint32_t* keys;    // [valid] nodes
    const uint32_t* places;  // [valid]
    const uint32_t* valid;   // one word
    const uint32_t* ranks;   // per kSpan places, the distinct nodes that start before (or null)
};
constexpr int kSpan = 32;

// What the launches of a sort fill beside it: bytes of zeros (past the caches if
// streamed), and num_ids ids of -1 (the distinct nodes then replace the first of
// them).
struct ClearOut {
    void* p;
    size_t bytes;
    bool streamed;
    int64_t* ids;
    int64_t num_ids;
};
size_t place_sort_bytes(int64_t num_rows, int64_t count, bool sparse);
// work receives the call's status (MLXC_WORK_WORDS words).  clear.ids not null:
// the distinct nodes go there, and ranks are made.
int launch_place_sort(const Nodes& nodes, int64_t count, const ClearOut& clear, int64_t* work,
                      void* workspace, SortedPlaces& sorted, hipStream_t stream);

// ---- embedding.hip
int launch_embedding(const Table& table, const Nodes& nodes, int64_t count, float scale, void* out,
                     int64_t* status, hipStream_t stream);
// The workspace of a gradient over count places.
size_t grad_workspace_bytes(int64_t num_rows, int32_t dim, int64_t count, bool sparse);
// Gradient rows `rows` ([count, dim] of dtype, by place), added up by node.
int launch_embedding_grad(const void* rows, int32_t dtype, int32_t dim, const Nodes& nodes,
                          int64_t count, float scale, const GradOut& out, void* workspace,
                          hipStream_t stream);

// ---- window_scores.hip
int launch_window_scores(const Table& table, const Walks& walks, float scale, float* scores,
                         int64_t* status, hipStream_t stream);
// The gradient of every place's row: [count, dim] float32.
int launch_window_rows_grad(const float* grad, const Table& table, const Walks& walks, float* rows,
                            hipStream_t stream);

// ---- preference.hip
struct PreferenceCall {
    mlxc_preference_side side[2];  // chosen, rejected
    int64_t pairs;
    int32_t dtype;
    float beta, smoothing;
    bool normalize, sum;
};
int launch_preference_loss(const PreferenceCall& call, float* loss, float* rewards, float* slopes,
                           void* workspace, hipStream_t stream);
int launch_preference_grad(const PreferenceCall& call, const float* slopes, const float* upstream,
                           hipStream_t stream);
size_t preference_workspace_bytes(int64_t pairs);

// ---- host_train.cpp
void host_embedding(const Table& table, const Nodes& nodes, int64_t count, float scale, void* out,
                    int64_t& status);
void host_embedding_grad(const void* rows, int32_t dtype, int32_t dim, const Nodes& nodes,
                         int64_t count, float scale, const GradOut& out, int64_t& status);
void host_window_scores(const Table& table, const Walks& walks, float scale, float* scores,
                        int64_t& status);
void host_window_scores_grad(const float* grad, const Table& table, const Walks& walks, float scale,
                             const GradOut& out, int64_t& status);
void host_preference_loss(const PreferenceCall& call, float* loss, float* rewards, float* slopes);
void host_preference_grad(const PreferenceCall& call, const float* slopes, const float* upstream);

}  // namespace mlxc
