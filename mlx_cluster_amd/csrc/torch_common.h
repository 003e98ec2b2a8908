// What the files of the compiled binding share: tensor checks, errors, and
// waiting for a call's status word.
#pragma once

#include <ATen/hip/HIPContext.h>
#include <hip/hip_runtime.h>
#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include <chrono>
#include <string>

#include "mlxc.h"

namespace mlxc_torch {

namespace py = pybind11;

// Whether t can be passed as is: a contiguous tensor of dtype on device.
inline bool usable(const at::Tensor& t, at::ScalarType dtype, const at::Device& device) {
    return t.scalar_type() == dtype && t.device() == device && t.is_contiguous();
}

inline const void* data_or_null(const at::Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }

inline void raise_code(int rc, const char* what) {
    const std::string msg = std::string(what) + ": " + mlxc_last_error();
    if (rc == MLXC_ERR_INVALID_ARGUMENT) throw py::value_error(msg);
    throw std::runtime_error(msg);
}

// The calling thread's host words for mlxc_set_status_target: allocated at
// the thread's first validated call (one pinned page) and kept for the rest
// of the process, since freeing them at thread exit could run after the HIP
// runtime has shut down; null if the allocation failed.
inline int64_t* status_words() {
    thread_local int64_t* words = [] {
        void* p = nullptr;
        if (hipHostMalloc(&p, 3 * sizeof(int64_t),
                          hipHostMallocCoherent | hipHostMallocMapped | hipHostMallocPortable) !=
            hipSuccess) {
            (void)hipGetLastError();
            return static_cast<int64_t*>(nullptr);
        }
        return static_cast<int64_t*>(p);
    }();
    return words;
}

// For a validated call: makes the library publish the call's status word into
// the calling thread's host words (mlxc_set_status_target), and puts the
// target that the thread had before back afterwards.
class StatusTarget {
public:
    explicit StatusTarget(bool check) : before(mlxc_status_target()) {
        int64_t* h = check ? status_words() : nullptr;
        if (!h) return;
        __atomic_store_n(&h[0], int64_t{0}, __ATOMIC_RELAXED);
        if (mlxc_set_status_target(h) == MLXC_OK) words = h;
    }
    ~StatusTarget() {
        if (words || before) mlxc_set_status_target(before);
    }
    int64_t* words = nullptr;

private:
    int64_t* const before;
};

// The status word of the call just enqueued on `stream`.  Its last launch
// stores it into `h` and the host waits for the flag: spinning for up to about
// 200 us (the reference tests' calls take tens), then in hipStreamSynchronize.
// Without the host words, torch's scalar read (a copy ordered on the stream,
// about 13 us more per call).
inline bool wait_published(hipStream_t stream, const int64_t* h) {
    if (!h) return false;
    const auto until = std::chrono::steady_clock::now() + std::chrono::microseconds(200);
    for (unsigned i = 1;; ++i) {
        if (__atomic_load_n(&h[0], __ATOMIC_ACQUIRE)) return true;
        __builtin_ia32_pause();
        if (i % 64 == 0 && std::chrono::steady_clock::now() > until) break;
    }
    if (hipStreamSynchronize(stream) != hipSuccess)
        throw std::runtime_error(std::string("hipStreamSynchronize: ") +
                                 hipGetErrorString(hipGetLastError()));
    return __atomic_load_n(&h[0], __ATOMIC_ACQUIRE) != 0;
}
// Word k of the call's workspace (0, or 1 after a CSR build).
inline int64_t read_word(const at::Tensor& work, hipStream_t stream, const int64_t* h, int k) {
    if (wait_published(stream, h)) return __atomic_load_n(&h[1 + k], __ATOMIC_RELAXED);
    return work.select(0, k).item<int64_t>();
}

// The training operators (torch_training.cpp).
void bind_training(py::module_& m);

}  // namespace mlxc_torch
