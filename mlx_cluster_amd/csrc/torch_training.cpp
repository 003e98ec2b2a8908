// Compiled fast path of the training operators (mlx_cluster_amd/training.py)
// for the common call: torch tensors of the right dtypes and shapes,
// contiguous, on the current device, torch's current stream, nothing for
// autograd to record.  It does what training.py does for such calls, without
// the Python layer's per-call cost; any other call returns None and training.py
// takes it, refusals among them.
#include <optional>

#include "mlxc_train.h"
#include "torch_common.h"

namespace mlxc_torch {

namespace {

int float_type(at::ScalarType t) {
    return t == at::kFloat ? MLXC_FLOAT32 : t == at::kBFloat16 ? MLXC_BFLOAT16
         : t == at::kHalf  ? MLXC_FLOAT16 : -1;
}
int node_type(at::ScalarType t) {
    return t == at::kLong ? MLXC_OUT_INT64 : t == at::kInt ? MLXC_OUT_INT32 : -1;
}

// Whether autograd has to see a call of t: to record it, or to refuse a dual tensor.
bool recorded(const at::Tensor& t) {
    return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

// A tensor as it is, on the device that calls run on.
bool here(const at::Tensor& t, const at::Device& device) {
    return t.device() == device && t.is_contiguous();
}
bool current(const at::Tensor& t) {
    return t.is_cuda() && t.device().index() == c10::hip::current_device();
}

void* ptr(const at::Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }

at::Tensor workspace(size_t bytes, const at::Device& device) {
    return at::empty({static_cast<int64_t>((bytes + 7) / 8)},
                     at::TensorOptions().dtype(at::kLong).device(device));
}

hipStream_t current_stream() { return at::hip::getCurrentHIPStream().stream(); }

// Waits for a checked call, whose status is in `word`, and raises for its bits.
// The wait is for all that is queued before the call too: other Python threads (a
// data loader's) run meanwhile.
void check_nodes(const at::Tensor& word, hipStream_t stream, const char* what) {
    int64_t bits = 0;
    {
        const py::gil_scoped_release other_threads_run;
        int64_t* h = status_words();
        if (h) {
            __atomic_store_n(&h[0], int64_t{0}, __ATOMIC_RELAXED);
            if (mlxc_publish_status(word.data_ptr(), h, stream) != MLXC_OK) h = nullptr;
        }
        bits = read_word(word, stream, h, 0);
    }
    if (bits & MLXC_STATUS_BAD_NODE)
        throw py::value_error(std::string(what) + ": a node is outside [0, num_nodes) and not -1");
}

// Sizes that the library takes as 32-bit numbers go to training.py past them.
bool fits(int64_t size) { return size <= INT32_MAX; }

// Whether weight and nodes are a table and its nodes that the library takes.
bool table_call(const at::Tensor& weight, const at::Tensor& nodes) {
    return current(weight) && weight.dim() == 2 && weight.size(1) >= 1 && fits(weight.size(1)) &&
           float_type(weight.scalar_type()) >= 0 && node_type(nodes.scalar_type()) >= 0 &&
           here(weight, weight.device()) && here(nodes, weight.device());
}

py::object embedding(const at::Tensor& weight, const at::Tensor& nodes, double scale, bool check) {
    if (!table_call(weight, nodes) || recorded(weight)) return py::none();
    const int64_t V = weight.size(0), D = weight.size(1);
    std::vector<int64_t> shape = nodes.sizes().vec();
    shape.push_back(D);
    at::Tensor out = at::empty(shape, weight.options().requires_grad(false));
    at::Tensor word;
    if (check) word = workspace(MLXC_WORK_WORDS * 8, weight.device());
    hipStream_t stream = current_stream();
    const int rc = mlxc_embedding(ptr(weight), V, static_cast<int32_t>(D), D,
                                  float_type(weight.scalar_type()), ptr(nodes), nodes.numel(),
                                  node_type(nodes.scalar_type()), static_cast<float>(scale),
                                  ptr(out), check ? word.data_ptr<int64_t>() : nullptr, stream);
    if (rc != MLXC_OK) raise_code(rc, "embedding");
    if (check) check_nodes(word, stream, "embedding");
    return py::cast(out);
}

struct GradBuffers {
    at::Tensor ids, out;
    int32_t flags;
    py::object result() const {
        if (flags & MLXC_GRAD_SPARSE) return py::make_tuple(ids, out);
        return py::cast(out);
    }
};
GradBuffers grad_buffers(int64_t V, int64_t D, int64_t count, bool sparse,
                         const at::TensorOptions& options) {
    GradBuffers b;
    const int64_t rows = sparse && count < V ? count : V;
    b.out = at::empty({rows, D}, options.requires_grad(false));
    if (sparse) b.ids = at::empty({rows}, options.dtype(at::kLong).requires_grad(false));
    b.flags = sparse ? MLXC_GRAD_SPARSE : 0;
    return b;
}
int64_t* ids_ptr(const GradBuffers& b) {
    return b.flags & MLXC_GRAD_SPARSE ? static_cast<int64_t*>(ptr(b.ids)) : nullptr;
}

py::object embedding_grad(const at::Tensor& grad, const at::Tensor& nodes, int64_t num_nodes,
                          double scale, bool sparse, bool check) {
    if (!current(grad) || grad.dim() != nodes.dim() + 1 || grad.size(-1) < 1 || num_nodes < 0 ||
        float_type(grad.scalar_type()) < 0 || node_type(nodes.scalar_type()) < 0 ||
        !here(grad, grad.device()) || !here(nodes, grad.device()) ||
        grad.sizes().slice(0, nodes.dim()) != nodes.sizes())
        return py::none();
    const int64_t D = grad.size(-1), count = nodes.numel();
    if (!fits(D)) return py::none();
    const size_t ws = mlxc_embedding_grad_workspace_bytes(num_nodes, static_cast<int32_t>(D), count,
                                                          sparse ? MLXC_GRAD_SPARSE : 0);
    if (ws == 0) return py::none();
    const GradBuffers b = grad_buffers(num_nodes, D, count, sparse, grad.options());
    const at::Tensor work = workspace(ws, grad.device());
    hipStream_t stream = current_stream();
    const int type = float_type(grad.scalar_type());
    const int rc = mlxc_embedding_grad(
        ptr(grad), static_cast<int32_t>(D), type, ptr(nodes), count, node_type(nodes.scalar_type()),
        num_nodes, static_cast<float>(scale), b.flags, ids_ptr(b), ptr(b.out), type,
        work.data_ptr(), static_cast<size_t>(work.numel()) * 8, stream);
    if (rc != MLXC_OK) raise_code(rc, "embedding_grad");
    if (check) check_nodes(work, stream, "embedding_grad");
    return b.result();
}

// The context of a window call's walks (0: the whole walk), or -1.
int32_t context_of(const at::Tensor& walks, int64_t context_size) {
    if (walks.dim() != 2 || walks.size(1) < 2 || !fits(walks.size(1))) return -1;
    const int64_t c = context_size ? context_size : walks.size(1);
    return c >= 2 && c <= 32 && c <= walks.size(1) ? static_cast<int32_t>(c) : -1;
}

py::object window_scores(const at::Tensor& weight, const at::Tensor& walks, int64_t context_size,
                         double scale, bool check) {
    const int32_t C = context_of(walks, context_size);
    if (C < 0 || !table_call(weight, walks) || recorded(weight)) return py::none();
    const int64_t V = weight.size(0), D = weight.size(1), N = walks.size(0), M = walks.size(1);
    at::Tensor out = at::empty({N, M - C + 1, C - 1},
                               weight.options().dtype(at::kFloat).requires_grad(false));
    at::Tensor word;
    if (check) word = workspace(MLXC_WORK_WORDS * 8, weight.device());
    hipStream_t stream = current_stream();
    const int rc = mlxc_window_scores(
        ptr(weight), V, static_cast<int32_t>(D), D, float_type(weight.scalar_type()), ptr(walks), N,
        static_cast<int32_t>(M), C, node_type(walks.scalar_type()), static_cast<float>(scale),
        static_cast<float*>(ptr(out)), check ? word.data_ptr<int64_t>() : nullptr, stream);
    if (rc != MLXC_OK) raise_code(rc, "window_scores");
    if (check) check_nodes(word, stream, "window_scores");
    return py::cast(out);
}

py::object window_scores_grad(const at::Tensor& grad, const at::Tensor& weight,
                              const at::Tensor& walks, int64_t context_size, double scale,
                              bool sparse, bool check) {
    const int32_t C = context_of(walks, context_size);
    if (C < 0 || !table_call(weight, walks) || !usable(grad, at::kFloat, weight.device()))
        return py::none();
    const int64_t V = weight.size(0), D = weight.size(1), N = walks.size(0), M = walks.size(1);
    if (grad.dim() != 3 || grad.size(0) != N || grad.size(1) != M - C + 1 || grad.size(2) != C - 1)
        return py::none();
    const size_t ws = mlxc_window_scores_grad_workspace_bytes(
        V, static_cast<int32_t>(D), N, static_cast<int32_t>(M), C, sparse ? MLXC_GRAD_SPARSE : 0);
    if (ws == 0) return py::none();
    const GradBuffers b = grad_buffers(V, D, N * M, sparse, weight.options());
    const at::Tensor work = workspace(ws, weight.device());
    hipStream_t stream = current_stream();
    const int type = float_type(weight.scalar_type());
    const int rc = mlxc_window_scores_grad(
        static_cast<const float*>(ptr(grad)), ptr(weight), V, static_cast<int32_t>(D), D, type,
        ptr(walks), N, static_cast<int32_t>(M), C, node_type(walks.scalar_type()),
        static_cast<float>(scale), b.flags, ids_ptr(b), ptr(b.out), type, work.data_ptr(),
        static_cast<size_t>(work.numel()) * 8, stream);
    if (rc != MLXC_OK) raise_code(rc, "window_scores_grad");
    if (check) check_nodes(work, stream, "window_scores_grad");
    return b.result();
}

using Maybe = std::optional<at::Tensor>;

// A side of a preference call, or false.
bool preference_side(const at::Tensor& x, const Maybe& reference, const Maybe& mask,
                     const at::Tensor& grad, mlxc_preference_side& s) {
    const at::Device device = x.device();
    if (reference && (reference->scalar_type() != x.scalar_type() ||
                      reference->sizes() != x.sizes() || !here(*reference, device)))
        return false;
    if (mask && ((mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte) ||
                 mask->sizes() != x.sizes() || !here(*mask, device)))
        return false;
    s.values = ptr(x);
    s.reference = reference ? ptr(*reference) : nullptr;
    s.mask = mask ? static_cast<const uint8_t*>(ptr(*mask)) : nullptr;
    s.length = x.dim() > 1 ? x.size(-1) : 1;
    s.grad = ptr(grad);
    return true;
}

py::object preference_loss_grad(const at::Tensor& chosen, const at::Tensor& rejected,
                                const Maybe& ref_chosen, const Maybe& ref_rejected,
                                const Maybe& chosen_mask, const Maybe& rejected_mask, double beta,
                                double label_smoothing, int32_t flags) {
    const int type = float_type(chosen.scalar_type());
    if (!current(chosen) || type < 0 || rejected.scalar_type() != chosen.scalar_type() ||
        chosen.dim() < 1 || rejected.dim() < 1 || !here(chosen, chosen.device()) ||
        !here(rejected, chosen.device()))
        return py::none();
    const auto pairs_of = [](const at::Tensor& x) {
        return x.dim() > 1 ? x.sizes().slice(0, x.dim() - 1) : x.sizes();
    };
    if (pairs_of(chosen) != pairs_of(rejected)) return py::none();
    int64_t pairs = 1;
    for (const int64_t n : pairs_of(chosen)) pairs *= n;
    const auto options = chosen.options().requires_grad(false);
    at::Tensor d_chosen = at::empty(chosen.sizes(), options);
    at::Tensor d_rejected = at::empty(rejected.sizes(), options);
    mlxc_preference_side c, r;
    if (!preference_side(chosen, ref_chosen, chosen_mask, d_chosen, c) ||
        !preference_side(rejected, ref_rejected, rejected_mask, d_rejected, r))
        return py::none();
    at::Tensor loss = at::empty({}, options.dtype(at::kFloat));
    at::Tensor rewards = at::empty({2, pairs}, options.dtype(at::kFloat));
    const at::Tensor work = workspace(mlxc_preference_loss_workspace_bytes(pairs), chosen.device());
    const int rc = mlxc_preference_loss(
        &c, &r, pairs, type, static_cast<float>(beta), static_cast<float>(label_smoothing), flags,
        loss.data_ptr<float>(), static_cast<float*>(ptr(rewards)), nullptr, work.data_ptr(),
        static_cast<size_t>(work.numel()) * 8, current_stream());
    if (rc != MLXC_OK) raise_code(rc, "preference_loss");
    return py::make_tuple(loss, rewards, d_chosen, d_rejected);
}

}  // namespace

void bind_training(py::module_& m) {
    m.def("embedding", &embedding);
    m.def("embedding_grad", &embedding_grad);
    m.def("window_scores", &window_scores);
    m.def("window_scores_grad", &window_scores_grad);
    m.def("preference_loss_grad", &preference_loss_grad);
}

}  // namespace mlxc_torch
