// Gated linear recurrence over time, forward and backward.
//
//   a_t = sigmoid(f_t),  r_t = 0 where an episode starts at t, else 1
//   h_t = r_t a_t h_{t-1} + (1 - a_t) x_t
// Backward, with G_t the whole gradient of h_t:
//   G_t = g_t + r_{t+1} a_{t+1} G_{t+1}   (g_last joins at the last step)
//   dx_t = (1 - a_t) G_t,  df_t = G_t (r_t h_{t-1} - x_t) a_t (1 - a_t),  dh0 = r_0 a_0 G_0
// Bound by memory: two values read and one written a step forward, three read and two written backward. The state is
// 32 bit throughout; the states that the backward pass needs are computed again from starting states kept every
// kChunk steps, not read from the rounded outputs.
//
// One thread walks the time of one column (one batch entry and channel).
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kThreads = 64;
constexpr int kChunk = 16;

__device__ inline float to_f(float v) { return v; }
__device__ inline float to_f(__half v) { return __half2float(v); }
__device__ inline float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }
template <> __device__ inline __half from_f<__half>(float v) { return __float2half(v); }
template <> __device__ inline __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

struct Seq {
    const void* base;
    int64_t t_stride, b_stride;  // elements; channels are dense
};

// a = sigmoid(f) and b = 1 - a, both with a small relative error
__device__ inline void gate(float f, float& a, float& b) {
    float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * f);
    a = __builtin_amdgcn_rcpf(1.f + e);
    b = e > 1e30f ? 1.f : e * a;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) linrec_fwd_kernel(
    Seq x, Seq f, const float* __restrict__ h0, const uint8_t* __restrict__ reset, T* __restrict__ h,
    float* __restrict__ last, float* __restrict__ starts, int64_t steps, int batch, int dim
) {
    int64_t columns = (int64_t)batch * dim;
    int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (c >= columns) return;
    int64_t bi = c / dim, d = c % dim;
    const T* xp = (const T*)x.base + bi * x.b_stride + d;
    const T* fp = (const T*)f.base + bi * f.b_stride + d;
    float state = h0 ? h0[c] : 0.f;
    for (int64_t t = 0; t < steps; ++t) {
        if (t % kChunk == 0) starts[t / kChunk * columns + c] = state;
        float a, b;
        gate(to_f(fp[t * f.t_stride]), a, b);
        if (reset && reset[t * batch + bi]) a = 0.f, state = 0.f;
        state = a * state + b * to_f(xp[t * x.t_stride]);
        h[t * columns + c] = from_f<T>(state);
    }
    last[c] = state;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) linrec_bwd_kernel(
    Seq x, Seq f, const uint8_t* __restrict__ reset, const float* __restrict__ starts, const T* __restrict__ g,
    const float* __restrict__ g_last, T* __restrict__ dx, T* __restrict__ df, float* __restrict__ dh0, int64_t steps,
    int batch, int dim
) {
    int64_t columns = (int64_t)batch * dim;
    int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (c >= columns) return;
    int64_t bi = c / dim, d = c % dim;
    const T* xp = (const T*)x.base + bi * x.b_stride + d;
    const T* fp = (const T*)f.base + bi * f.b_stride + d;
    float carry = g_last ? g_last[c] : 0.f;
    for (int64_t t0 = (steps - 1) / kChunk * kChunk; t0 >= 0; t0 -= kChunk) {
        float before[kChunk], a[kChunk], b[kChunk], xs[kChunk];
        float state = starts[t0 / kChunk * columns + c];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            int64_t t = t0 + i;
            before[i] = a[i] = b[i] = xs[i] = 0.f;
            if (t < steps) {
                gate(to_f(fp[t * f.t_stride]), a[i], b[i]);
                xs[i] = to_f(xp[t * x.t_stride]);
                if (reset && reset[t * batch + bi]) state = 0.f;
                before[i] = state;
                state = a[i] * state + b[i] * xs[i];
            }
        }
#pragma unroll
        for (int i = kChunk - 1; i >= 0; --i) {
            int64_t t = t0 + i;
            if (t < steps) {
                float G = carry + (g ? to_f(g[t * columns + c]) : 0.f);
                dx[t * columns + c] = from_f<T>(b[i] * G);
                df[t * columns + c] = from_f<T>(G * (before[i] - xs[i]) * a[i] * b[i]);
                carry = reset && reset[t * batch + bi] ? 0.f : a[i] * G;
            }
        }
    }
    if (dh0) dh0[c] = carry;
}

Seq seq_of(const torch::Tensor& v) { return {v.data_ptr(), v.stride(0), v.stride(1)}; }

void check_seq(const torch::Tensor& v, const torch::Tensor& x) {
    TORCH_CHECK(v.is_cuda() && v.device() == x.device() && v.dim() == 3 && v.sizes() == x.sizes() &&
                    v.scalar_type() == x.scalar_type() && (v.stride(2) == 1 || v.size(2) == 1),
                "gated_linear_recurrence: x and gate must be [T, B, D] of one type and device with dense channels");
    TORCH_CHECK(v.size(0) >= 1 && v.size(1) * v.size(2) < (int64_t)1 << 31,
                "gated_linear_recurrence: T must be at least 1 and B * D below 2^31");
}

// an empty tensor stands for one that is not there
template <typename T>
const T* given(const torch::Tensor& v, const torch::Tensor& x, int64_t n, c10::ScalarType type) {
    if (v.numel() == 0) return nullptr;
    TORCH_CHECK(v.device() == x.device() && v.is_contiguous() && v.numel() == n && v.scalar_type() == type,
                "gated_linear_recurrence: an argument has another size, type, layout or device");
    return (const T*)v.data_ptr();
}

template <typename F>
void by_type(const torch::Tensor& x, F&& f) {
    switch (x.scalar_type()) {
        case torch::kFloat32: f((float*)nullptr); break;
        case torch::kFloat16: f((__half*)nullptr); break;
        case torch::kBFloat16: f((__hip_bfloat16*)nullptr); break;
        default: TORCH_CHECK(false, "gated_linear_recurrence: expected float32, float16 or bfloat16");
    }
}

}  // namespace

std::vector<torch::Tensor> linrec_fwd(torch::Tensor x, torch::Tensor gate, torch::Tensor h0, torch::Tensor reset) {
    check_seq(x, x);
    check_seq(gate, x);
    c10::OptionalDeviceGuard guard(x.device());
    int64_t steps = x.size(0), columns = x.size(1) * x.size(2);
    auto opt = x.options().dtype(torch::kFloat32);
    auto h = torch::empty(x.sizes(), x.options());
    auto last = torch::empty({x.size(1), x.size(2)}, opt);
    auto starts = torch::empty({(steps + kChunk - 1) / kChunk, columns}, opt);
    if (columns == 0) return {h, last, starts};
    const float* h0p = given<float>(h0, x, columns, torch::kFloat32);
    const uint8_t* rp = given<uint8_t>(reset, x, steps * x.size(1), torch::kBool);
    by_type(x, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        linrec_fwd_kernel<T><<<cdiv(columns, kThreads), kThreads, 0, ding_current_stream()>>>(
            seq_of(x), seq_of(gate), h0p, rp, (T*)h.data_ptr(), last.data_ptr<float>(), starts.data_ptr<float>(),
            steps, (int)x.size(1), (int)x.size(2));
    });
    HIP_CHECK_LAST();
    return {h, last, starts};
}

std::vector<torch::Tensor> linrec_bwd(
    torch::Tensor x, torch::Tensor gate, torch::Tensor reset, torch::Tensor starts, torch::Tensor grad_h,
    torch::Tensor grad_last, int64_t want_h0
) {
    check_seq(x, x);
    check_seq(gate, x);
    c10::OptionalDeviceGuard guard(x.device());
    int64_t steps = x.size(0), columns = x.size(1) * x.size(2);
    auto opt = x.options().dtype(torch::kFloat32);
    auto dx = torch::empty(x.sizes(), x.options());
    auto df = torch::empty(x.sizes(), x.options());
    auto dh0 = want_h0 ? torch::empty({x.size(1), x.size(2)}, opt) : torch::empty({0}, opt);
    if (columns == 0) return {dx, df, dh0};
    const uint8_t* rp = given<uint8_t>(reset, x, steps * x.size(1), torch::kBool);
    const void* gp = given<uint8_t>(grad_h, x, steps * columns, x.scalar_type());
    const float* lp = given<float>(grad_last, x, columns, torch::kFloat32);
    const float* sp = given<float>(starts, x, (steps + kChunk - 1) / kChunk * columns, torch::kFloat32);
    TORCH_CHECK(sp, "gated_linear_recurrence: the kept states are missing");
    by_type(x, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        linrec_bwd_kernel<T><<<cdiv(columns, kThreads), kThreads, 0, ding_current_stream()>>>(
            seq_of(x), seq_of(gate), rp, sp, (const T*)gp, lp, (T*)dx.data_ptr(), (T*)df.data_ptr(),
            want_h0 ? dh0.data_ptr<float>() : nullptr, steps, (int)x.size(1), (int)x.size(2));
    });
    HIP_CHECK_LAST();
    return {dx, df, dh0};
}
