// Shared helpers for the DI-engine MI355X HIP kernels (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <c10/hip/HIPStream.h>

// current PyTorch stream for this device (hipStream_t)
static inline hipStream_t ding_current_stream() {
    return c10::hip::getCurrentHIPStream().stream();
}

#define CHECK_INPUT(x)                                                                   \
    TORCH_CHECK(x.is_cuda(), #x " must be a HIP tensor");                                \
    TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")

constexpr int kWave = 64;  // CDNA4 wavefront width

static inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

#define HIP_CHECK_LAST()                                                                 \
    do {                                                                                 \
        hipError_t e = hipGetLastError();                                                \
        TORCH_CHECK(e == hipSuccess, "HIP kernel launch failed: ", hipGetErrorString(e)); \
    } while (0)

// What an operator's backward pass returns: where gradients of gradients are asked for they are refused, not taken for
// zero.
static inline torch::autograd::variable_list ding_once_differentiable(
    torch::autograd::variable_list grads, const char* name
) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate twice a function that is differentiable once: ") + name,
        (int64_t)grads.size()
    );
    return (*error)(std::move(grads));
}
