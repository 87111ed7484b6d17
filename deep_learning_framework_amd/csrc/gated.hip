// The gated feed-forward projection: y = act(x . wg^T + bg) * (x . wu^T + bu), and its element-wise gradients.
#include "act_funcs.h"
#include "decoder_ops.h"
#include "gemm_host.h"

namespace kai {
namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads) void gated_activation_kernel(float* y, const float* gate, const float* up, int64_t n,
                                                                    int act, const float* hleaky) {
    const float leaky = hleaky ? *hleaky : 0.0f;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads)
        y[i] = apply_act(gate[i], act, leaky) * up[i];
}

__global__ __launch_bounds__(kThreads) void gated_activation_backward_kernel(float* ggate, float* gup, const float* gy,
                                                                             const float* gate, const float* up, int64_t n,
                                                                             int act, const float* hleaky) {
    const float leaky = hleaky ? *hleaky : 0.0f;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
        const float g = gate[i], d = gy[i];
        const float u = up[i];
        ggate[i] = d * u * act_derivative(g, act, leaky);
        gup[i] = d * apply_act(g, act, leaky);
    }
}

unsigned grid_of(int64_t n) {
    const int64_t groups = (n + kThreads - 1) / kThreads, most = 16 * (int64_t)compute_units();
    return (unsigned)(groups < most ? groups : most);
}

}  // namespace

int launch_gated_activation(float* y, const float* gate, const float* up, int64_t n, int act, const float* hleaky,
                            hipStream_t stream) {
    gated_activation_kernel<<<grid_of(n), kThreads, 0, stream>>>(y, gate, up, n, act, hleaky);
    return check_launch("gated_activation_kernel");
}

int launch_gated_activation_backward(float* ggate, float* gup, const float* gy, const float* gate, const float* up,
                                     int64_t n, int act, const float* hleaky, hipStream_t stream) {
    gated_activation_backward_kernel<<<grid_of(n), kThreads, 0, stream>>>(ggate, gup, gy, gate, up, n, act, hleaky);
    return check_launch("gated_activation_backward_kernel");
}

int launch_gated_forward(const GatedArgs& a, hipStream_t stream) {
    // both products, then the activation and the product; the pre-activations in the caller's buffers or in scratch
    const int64_t n = a.ndat * a.yvec;
    float* gate = a.gate;
    float* up = a.up;
    int64_t held_bytes = 0;
    if (gate == nullptr) {
        held_bytes = 2 * n * (int64_t)sizeof(float);
        KAI_TRY(workspace(held_bytes, &gate));
        up = gate + n;
    }
    ScratchHold held(held_bytes);
    for (int i = 0; i < 2; i++) {
        GemmDesc d;
        d.A = a.x; d.B = i ? a.wu : a.wg; d.C = i ? up : gate; d.bias = i ? a.bu : a.bg;
        d.M = a.ndat; d.N = a.yvec; d.K = a.xvec;
        d.a_rs = a.xvec; d.a_ks = 1; d.b_rs = a.xvec; d.b_ks = 1; d.c_rs = a.yvec; d.c_cs = 1;
        KAI_TRY(launch_gemm(d, stream));
    }
    return launch_gated_activation(a.y, gate, up, n, a.act, a.hleaky, stream);
}

}  // namespace kai
