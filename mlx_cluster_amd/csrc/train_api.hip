// The C ABI of the training operators (include/mlxc_train.h): argument checks
// and dispatch to the kernel launchers and the host twins.  Every entry point
// checks its arguments on the host before touching the device.
#include <climits>
#include <cmath>
#include <new>
#include <stdexcept>

#include "train_host.h"

namespace mlxc {

namespace {

// Blocks times threads of a launch stay below 2^32 and row offsets in int64
// whatever the sizes below these.
constexpr int64_t kMaxRows = INT32_MAX;
constexpr int32_t kMaxDim = 65536;

int invalid(const char* msg) { return fail(MLXC_ERR_INVALID_ARGUMENT, msg); }

int check_dtype(int32_t dtype, const char* what) {
    if (dtype == MLXC_FLOAT32 || dtype == MLXC_BFLOAT16 || dtype == MLXC_FLOAT16) return MLXC_OK;
    return fail(MLXC_ERR_INVALID_ARGUMENT,
                std::string(what) + " must be MLXC_FLOAT32, MLXC_BFLOAT16 or MLXC_FLOAT16");
}

int check_sizes(int64_t num_rows, int32_t dim, int64_t count, int32_t node_type) {
    if (num_rows < 0 || num_rows > kMaxRows) return invalid("num_rows must lie in [0, 2^31)");
    if (dim < 1 || dim > kMaxDim) return invalid("dim must lie in [1, 65536]");
    if (count < 0) return invalid("the number of nodes must be >= 0");
    if (node_type != MLXC_OUT_INT64 && node_type != MLXC_OUT_INT32)
        return invalid("node_type must be MLXC_OUT_INT64 or MLXC_OUT_INT32");
    if (count > INT64_MAX / 4 / dim) return invalid("count * dim overflows int64");
    return MLXC_OK;
}

// Sorted places are 32 bits wide.
int check_places(int64_t count) {
    if (count >= INT32_MAX)
        return invalid("at most 2^31 - 2 nodes a call: split it (and add the gradients)");
    return MLXC_OK;
}

int check_table(const void* weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                int32_t dtype) {
    if (int rc = check_dtype(dtype, "dtype")) return rc;
    if (num_rows > 0 && !weight) return invalid("weight must not be NULL");
    if (row_stride < dim) return invalid("row_stride must be at least dim");
    if (num_rows > 0 && row_stride > INT64_MAX / 4 / num_rows)
        return invalid("num_rows * row_stride overflows int64");
    const size_t esz = elem_bytes(dtype);
    if (reinterpret_cast<uintptr_t>(weight) % esz != 0)
        return invalid("weight must be aligned to its elements");
    return MLXC_OK;
}

int check_walks(const void* nodes, int64_t num_walks, int32_t walk_nodes, int32_t ctx) {
    if (num_walks < 0) return invalid("num_walks must be >= 0");
    if (walk_nodes < 1) return invalid("walk_nodes must be >= 1");
    if (ctx < 2 || ctx > 32 || ctx > walk_nodes)
        return invalid("context_size must lie in [2, min(32, nodes per walk)]");
    if (num_walks > 0 && !nodes) return invalid("walks must not be NULL");
    if (num_walks > INT64_MAX / walk_nodes || num_walks * walk_nodes >= INT32_MAX)
        return invalid("num_walks * walk_nodes must be below 2^31 - 1: split the call");
    return MLXC_OK;
}

int check_grad_out(int64_t num_rows, int64_t count, int32_t flags, const int64_t* ids,
                   const void* out, int32_t out_dtype) {
    if (int rc = check_dtype(out_dtype, "out_dtype")) return rc;
    if (flags & ~MLXC_GRAD_SPARSE) return invalid("flags must be 0 or MLXC_GRAD_SPARSE");
    const int64_t rows = flags & MLXC_GRAD_SPARSE ? (count < num_rows ? count : num_rows) : num_rows;
    if (rows > 0 && !out) return invalid("out must not be NULL");
    if (rows > 0 && (flags & MLXC_GRAD_SPARSE) && !ids)
        return invalid("ids must not be NULL with MLXC_GRAD_SPARSE");
    if (reinterpret_cast<uintptr_t>(out) % elem_bytes(out_dtype) != 0)
        return invalid("out must be aligned to its elements");
    return MLXC_OK;
}

int check_train_workspace(const void* ws, size_t bytes, size_t need) {
    if (!ws) return invalid("workspace must not be NULL");
    if (reinterpret_cast<uintptr_t>(ws) % 16 != 0) return invalid("workspace must be 16-byte aligned");
    if (bytes < need)
        return fail(MLXC_ERR_INVALID_ARGUMENT,
                    "workspace holds " + std::to_string(bytes) + " bytes, the call needs " +
                        std::to_string(need));
    return MLXC_OK;
}

Nodes as_nodes(const void* p, int64_t num_rows, int32_t node_type) {
    return Nodes{p, num_rows, node_type == MLXC_OUT_INT64};
}

// A coalesced gradient's ids, which mark it as one, also where it has no rows.
int64_t empty_ids;
GradOut grad_out(void* out, int64_t* ids, int32_t flags, int32_t out_dtype) {
    if (!(flags & MLXC_GRAD_SPARSE)) ids = nullptr;
    else if (!ids) ids = &empty_ids;
    return GradOut{out, ids, out_dtype};
}

// Workspace of a window gradient: the rows' gradients, then the embedding
// gradient's.
size_t rows_grad_bytes(int32_t dim, int64_t count) {
    return (static_cast<size_t>(count) * dim * sizeof(float) + 255) & ~static_cast<size_t>(255);
}

int check_preference(const mlxc_preference_side* chosen, const mlxc_preference_side* rejected,
                     int64_t pairs, int32_t dtype, bool values) {
    if (!chosen || !rejected) return invalid("chosen and rejected must not be NULL");
    if (pairs < 0) return invalid("pairs must be >= 0");
    if (int rc = check_dtype(dtype, "dtype")) return rc;
    for (const mlxc_preference_side* s : {chosen, rejected}) {
        if (s->length < 0 || s->length >= (int64_t{1} << 30))
            return invalid("length must lie in [0, 2^30)");
        if (s->length > 0 && pairs > INT64_MAX / 4 / s->length)
            return invalid("pairs * length overflows int64");
        if (values && pairs > 0 && s->length > 0 && !s->values)
            return invalid("values must not be NULL");
        const uintptr_t all = reinterpret_cast<uintptr_t>(s->values) |
                              reinterpret_cast<uintptr_t>(s->reference) |
                              reinterpret_cast<uintptr_t>(s->grad);
        if (all % elem_bytes(dtype) != 0)
            return invalid("values, reference and grad must be aligned to their elements");
    }
    return MLXC_OK;
}

int check_loss(const mlxc_preference_side* chosen, const mlxc_preference_side* rejected,
               int64_t pairs, int32_t dtype, float beta, float smoothing, int32_t flags,
               const float* loss) {
    if (int rc = check_preference(chosen, rejected, pairs, dtype, true)) return rc;
    if (!std::isfinite(beta)) return invalid("beta must be finite");
    if (!(smoothing >= 0.f && smoothing <= 1.f)) return invalid("label_smoothing must lie in [0, 1]");
    if (flags & ~(MLXC_PREFERENCE_NORMALIZE | MLXC_PREFERENCE_SUM))
        return invalid("flags must be a combination of MLXC_PREFERENCE_NORMALIZE and "
                       "MLXC_PREFERENCE_SUM");
    if (!loss) return invalid("loss must not be NULL");
    return MLXC_OK;
}

PreferenceCall preference_call(const mlxc_preference_side* chosen,
                               const mlxc_preference_side* rejected, int64_t pairs, int32_t dtype,
                               float beta, float smoothing, int32_t flags) {
    return PreferenceCall{{*chosen, *rejected}, pairs, dtype, beta, smoothing,
                          (flags & MLXC_PREFERENCE_NORMALIZE) != 0,
                          (flags & MLXC_PREFERENCE_SUM) != 0};
}

// No exception leaves a C entry: the host twins allocate.
template <typename F>
int no_throw(F&& body) {
    try {
        body();
        return MLXC_OK;
    } catch (const std::bad_alloc&) {
    } catch (const std::length_error&) {  // more than a vector can ever hold
    }
    return fail(MLXC_ERR_HIP, "out of host memory");
}

}  // namespace

}  // namespace mlxc

using namespace mlxc;

extern "C" {

int mlxc_embedding(const void* d_weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                   int32_t dtype, const void* d_nodes, int64_t count, int32_t node_type,
                   float scale, void* d_out, int64_t* d_status, void* stream) {
    if (int rc = check_sizes(num_rows, dim, count, node_type)) return rc;
    if (int rc = check_table(d_weight, num_rows, dim, row_stride, dtype)) return rc;
    if (count > 0 && (!d_nodes || !d_out)) return invalid("nodes and out must not be NULL");
    if (reinterpret_cast<uintptr_t>(d_out) % elem_bytes(dtype) != 0)
        return invalid("out must be aligned to its elements");
    return launch_embedding(Table{d_weight, num_rows, row_stride, dim, dtype},
                            as_nodes(d_nodes, num_rows, node_type), count, scale, d_out, d_status,
                            static_cast<hipStream_t>(stream));
}

size_t mlxc_embedding_grad_workspace_bytes(int64_t num_rows, int32_t dim, int64_t count,
                                           int32_t flags) {
    if (check_sizes(num_rows, dim, count, MLXC_OUT_INT64) || check_places(count)) return 0;
    return grad_workspace_bytes(num_rows, dim, count, (flags & MLXC_GRAD_SPARSE) != 0);
}

int mlxc_embedding_grad(const void* d_grad, int32_t dim, int32_t dtype, const void* d_nodes,
                        int64_t count, int32_t node_type, int64_t num_rows, float scale,
                        int32_t flags, int64_t* d_ids, void* d_out, int32_t out_dtype,
                        void* d_workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes(num_rows, dim, count, node_type)) return rc;
    if (int rc = check_places(count)) return rc;
    if (int rc = check_dtype(dtype, "dtype")) return rc;
    if (int rc = check_grad_out(num_rows, count, flags, d_ids, d_out, out_dtype)) return rc;
    if (count > 0 && (!d_nodes || !d_grad)) return invalid("grad and nodes must not be NULL");
    if (reinterpret_cast<uintptr_t>(d_grad) % elem_bytes(dtype) != 0)
        return invalid("grad must be aligned to its elements");
    const size_t need = mlxc_embedding_grad_workspace_bytes(num_rows, dim, count, flags);
    if (int rc = check_train_workspace(d_workspace, workspace_bytes, need)) return rc;
    return launch_embedding_grad(d_grad, dtype, dim, as_nodes(d_nodes, num_rows, node_type), count,
                                 scale, grad_out(d_out, d_ids, flags, out_dtype), d_workspace,
                                 static_cast<hipStream_t>(stream));
}

int mlxc_window_scores(const void* d_weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                       int32_t dtype, const void* d_walks, int64_t num_walks, int32_t walk_nodes,
                       int32_t context_size, int32_t node_type, float scale, float* d_scores,
                       int64_t* d_status, void* stream) {
    if (int rc = check_walks(d_walks, num_walks, walk_nodes, context_size)) return rc;
    if (int rc = check_sizes(num_rows, dim, num_walks * walk_nodes, node_type)) return rc;
    if (int rc = check_table(d_weight, num_rows, dim, row_stride, dtype)) return rc;
    if (num_walks > 0 && !d_scores) return invalid("scores must not be NULL");
    return launch_window_scores(
        Table{d_weight, num_rows, row_stride, dim, dtype},
        Walks{as_nodes(d_walks, num_rows, node_type), num_walks, walk_nodes, context_size}, scale,
        d_scores, d_status, static_cast<hipStream_t>(stream));
}

size_t mlxc_window_scores_grad_workspace_bytes(int64_t num_rows, int32_t dim, int64_t num_walks,
                                               int32_t walk_nodes, int32_t context_size,
                                               int32_t flags) {
    if (check_walks(&empty_ids, num_walks, walk_nodes, context_size)) return 0;
    const int64_t count = num_walks * walk_nodes;
    const size_t bytes = mlxc_embedding_grad_workspace_bytes(num_rows, dim, count, flags);
    return bytes ? bytes + rows_grad_bytes(dim, count) : 0;
}

int mlxc_window_scores_grad(const float* d_grad, const void* d_weight, int64_t num_rows,
                            int32_t dim, int64_t row_stride, int32_t dtype, const void* d_walks,
                            int64_t num_walks, int32_t walk_nodes, int32_t context_size,
                            int32_t node_type, float scale, int32_t flags, int64_t* d_ids,
                            void* d_out, int32_t out_dtype, void* d_workspace,
                            size_t workspace_bytes, void* stream) {
    if (int rc = check_walks(d_walks, num_walks, walk_nodes, context_size)) return rc;
    const int64_t count = num_walks * walk_nodes;
    if (int rc = check_sizes(num_rows, dim, count, node_type)) return rc;
    if (int rc = check_table(d_weight, num_rows, dim, row_stride, dtype)) return rc;
    if (int rc = check_grad_out(num_rows, count, flags, d_ids, d_out, out_dtype)) return rc;
    if (num_walks > 0 && !d_grad) return invalid("grad must not be NULL");
    const size_t need = mlxc_window_scores_grad_workspace_bytes(num_rows, dim, num_walks,
                                                                walk_nodes, context_size, flags);
    if (int rc = check_train_workspace(d_workspace, workspace_bytes, need)) return rc;
    const Table table{d_weight, num_rows, row_stride, dim, dtype};
    const Walks walks{as_nodes(d_walks, num_rows, node_type), num_walks, walk_nodes, context_size};
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* rows = reinterpret_cast<float*>(static_cast<unsigned char*>(d_workspace) + need -
                                           rows_grad_bytes(dim, count));
    if (int rc = launch_window_rows_grad(d_grad, table, walks, rows, s)) return rc;
    return launch_embedding_grad(rows, MLXC_FLOAT32, dim, walks.nodes, count, scale,
                                 grad_out(d_out, d_ids, flags, out_dtype), d_workspace, s);
}

size_t mlxc_preference_loss_workspace_bytes(int64_t pairs) {
    return pairs < 0 ? 0 : preference_workspace_bytes(pairs);
}

int mlxc_preference_loss(const mlxc_preference_side* chosen, const mlxc_preference_side* rejected,
                         int64_t pairs, int32_t dtype, float beta, float label_smoothing,
                         int32_t flags, float* d_loss, float* d_rewards, float* d_slopes,
                         void* d_workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_loss(chosen, rejected, pairs, dtype, beta, label_smoothing, flags, d_loss))
        return rc;
    if (int rc = check_train_workspace(d_workspace, workspace_bytes,
                                       mlxc_preference_loss_workspace_bytes(pairs)))
        return rc;
    return launch_preference_loss(
        preference_call(chosen, rejected, pairs, dtype, beta, label_smoothing, flags), d_loss,
        d_rewards, d_slopes, d_workspace, static_cast<hipStream_t>(stream));
}

int mlxc_preference_grad(const mlxc_preference_side* chosen, const mlxc_preference_side* rejected,
                         int64_t pairs, int32_t dtype, const float* d_slopes,
                         const float* d_upstream, void* stream) {
    if (int rc = check_preference(chosen, rejected, pairs, dtype, false)) return rc;
    if (pairs > 0 && !d_slopes) return invalid("slopes must not be NULL");
    return launch_preference_grad(preference_call(chosen, rejected, pairs, dtype, 0.f, 0.f, 0),
                                  d_slopes, d_upstream, static_cast<hipStream_t>(stream));
}

// ------------------------------------------------------------- host twins

int mlxc_embedding_cpu(const void* weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                       int32_t dtype, const void* nodes, int64_t count, int32_t node_type,
                       float scale, void* out, int64_t* status) {
    if (int rc = check_sizes(num_rows, dim, count, node_type)) return rc;
    if (int rc = check_table(weight, num_rows, dim, row_stride, dtype)) return rc;
    if (count > 0 && (!nodes || !out)) return invalid("nodes and out must not be NULL");
    int64_t bits = 0;
    host_embedding(Table{weight, num_rows, row_stride, dim, dtype},
                   as_nodes(nodes, num_rows, node_type), count, scale, out, bits);
    if (status) *status = bits;
    return MLXC_OK;
}

int mlxc_embedding_grad_cpu(const void* grad, int32_t dim, int32_t dtype, const void* nodes,
                            int64_t count, int32_t node_type, int64_t num_rows, float scale,
                            int32_t flags, int64_t* ids, void* out, int32_t out_dtype,
                            int64_t* status) {
    if (int rc = check_sizes(num_rows, dim, count, node_type)) return rc;
    if (int rc = check_dtype(dtype, "dtype")) return rc;
    if (int rc = check_grad_out(num_rows, count, flags, ids, out, out_dtype)) return rc;
    if (count > 0 && (!nodes || !grad)) return invalid("grad and nodes must not be NULL");
    int64_t bits = 0;
    const int rc = no_throw([&] {
        host_embedding_grad(grad, dtype, dim, as_nodes(nodes, num_rows, node_type), count, scale,
                            grad_out(out, ids, flags, out_dtype), bits);
    });
    if (status) *status = bits;
    return rc;
}

int mlxc_window_scores_cpu(const void* weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                           int32_t dtype, const void* walks, int64_t num_walks,
                           int32_t walk_nodes, int32_t context_size, int32_t node_type,
                           float scale, float* scores, int64_t* status) {
    if (int rc = check_walks(walks, num_walks, walk_nodes, context_size)) return rc;
    if (int rc = check_sizes(num_rows, dim, num_walks * walk_nodes, node_type)) return rc;
    if (int rc = check_table(weight, num_rows, dim, row_stride, dtype)) return rc;
    if (num_walks > 0 && !scores) return invalid("scores must not be NULL");
    int64_t bits = 0;
    const int rc = no_throw([&] {
        host_window_scores(
            Table{weight, num_rows, row_stride, dim, dtype},
            Walks{as_nodes(walks, num_rows, node_type), num_walks, walk_nodes, context_size}, scale,
            scores, bits);
    });
    if (status) *status = bits;
    return rc;
}

int mlxc_window_scores_grad_cpu(const float* grad, const void* weight, int64_t num_rows,
                                int32_t dim, int64_t row_stride, int32_t dtype, const void* walks,
                                int64_t num_walks, int32_t walk_nodes, int32_t context_size,
                                int32_t node_type, float scale, int32_t flags, int64_t* ids,
                                void* out, int32_t out_dtype, int64_t* status) {
    if (int rc = check_walks(walks, num_walks, walk_nodes, context_size)) return rc;
    const int64_t count = num_walks * walk_nodes;
    if (int rc = check_sizes(num_rows, dim, count, node_type)) return rc;
    if (int rc = check_table(weight, num_rows, dim, row_stride, dtype)) return rc;
    if (int rc = check_grad_out(num_rows, count, flags, ids, out, out_dtype)) return rc;
    if (num_walks > 0 && !grad) return invalid("grad must not be NULL");
    int64_t bits = 0;
    const int rc = no_throw([&] {
        host_window_scores_grad(
            grad, Table{weight, num_rows, row_stride, dim, dtype},
            Walks{as_nodes(walks, num_rows, node_type), num_walks, walk_nodes, context_size}, scale,
            grad_out(out, ids, flags, out_dtype), bits);
    });
    if (status) *status = bits;
    return rc;
}

int mlxc_preference_loss_cpu(const mlxc_preference_side* chosen,
                             const mlxc_preference_side* rejected, int64_t pairs, int32_t dtype,
                             float beta, float label_smoothing, int32_t flags, float* loss,
                             float* rewards, float* slopes) {
    if (int rc = check_loss(chosen, rejected, pairs, dtype, beta, label_smoothing, flags, loss))
        return rc;
    return no_throw([&] {
        host_preference_loss(
            preference_call(chosen, rejected, pairs, dtype, beta, label_smoothing, flags), loss,
            rewards, slopes);
    });
}

int mlxc_preference_grad_cpu(const mlxc_preference_side* chosen,
                             const mlxc_preference_side* rejected, int64_t pairs, int32_t dtype,
                             const float* slopes, const float* upstream) {
    if (int rc = check_preference(chosen, rejected, pairs, dtype, false)) return rc;
    if (pairs > 0 && !slopes) return invalid("slopes must not be NULL");
    host_preference_grad(preference_call(chosen, rejected, pairs, dtype, 0.f, 0.f, 0), slopes,
                         upstream);
    return MLXC_OK;
}

}  // extern "C"
