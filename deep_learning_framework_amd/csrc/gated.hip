// The gated feed-forward projection: y = act(x . wg^T + bg) * (x . wu^T + bu), and its element-wise gradients.
#include "act_funcs.h"
#include "decoder_ops.h"
#include "gated_gemm.h"
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
    GatedGemm p{};
    p.A[0] = a.x; p.B[0] = a.wg; p.B[1] = a.wu;
    p.C[0] = a.y; p.C[1] = a.gate; p.C[2] = a.up;
    p.bias[0] = a.bg; p.bias[1] = a.bu;
    p.hleaky = a.hleaky; p.act = a.act;
    p.M = a.ndat; p.N = a.yvec; p.K = (int)a.xvec;
    p.lda = p.ldb = a.xvec; p.ldc = a.yvec;
    p.nwhich = 1;
    if (a.ndat > 32 && gated_gemm_applies(kGatedForward, p)) return launch_gated_gemm(kGatedForward, p, stream);
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

// Gradients of up to 32 rows, and small ones, take two products of the dense layer's dispatcher each, about 7 us and
// 65 flop a ns: their latency is lower (us with the element-wise kernel in front, two products | this file's: gx of
// 256 x 64 -> 512 10.9 | 13.8, of 1000 x 256 -> 512 17.5 | 20.5, of 128 x 1024 -> 1024 23.3 | 19.0, of 512 x 1024 -> 1024 40.5 | 30.0; gw of
// 512 x 64 -> 512 11.1 | 14.1, of 33 x 1024 -> 1024 14.2 | 9.9).
static bool split_pays(int mode, const GatedGemm& p, int64_t ndat) {
    if (ndat <= 32 || !gated_gemm_applies(mode, p)) return false;
    const double flops = 4.0 * p.M * p.N * p.K * (mode == kGatedGw && p.nwhich == 1 ? 0.5 : 1.0);
    return gated_gemm_us(mode, p) < 7.0 + flops / 65e6;
}

int launch_gated_gradients(const GatedGradArgs& a, hipStream_t stream) {
    GatedGemm p{};
    p.A[0] = a.ggate; p.A[1] = a.gup;
    p.acc = a.acc;
    p.nwhich = 1;
    if (a.gx) {
        p.B[0] = a.wg; p.B[1] = a.wu;
        p.C[0] = a.gx;
        p.M = a.ndat; p.N = a.xvec; p.K = (int)a.yvec;
        p.lda = a.yvec; p.ldb = p.ldc = a.xvec;
        if (split_pays(kGatedGx, p, a.ndat)) {
            KAI_TRY(launch_gated_gemm(kGatedGx, p, stream));
        } else {
            KAI_TRY(kai_matmul_backward_x(0, a.gx, a.ggate, a.wg, a.yvec, a.ndat, a.xvec, a.acc));
            KAI_TRY(kai_matmul_backward_x(0, a.gx, a.gup, a.wu, a.yvec, a.ndat, a.xvec, 1));
        }
    }
    if (a.gwg == nullptr && a.gwu == nullptr) return KAI_OK;
    p.B[0] = a.x; p.B[1] = nullptr;
    p.M = a.yvec; p.N = a.xvec; p.K = (int)a.ndat;
    p.lda = a.yvec; p.ldb = p.ldc = a.xvec;
    p.C[0] = a.gwg; p.C[1] = a.gwu;
    p.nwhich = 2;
    if (a.gwg == nullptr || a.gwu == nullptr) {
        p.nwhich = 1;
        p.C[0] = a.gwg ? a.gwg : a.gwu;
        p.C[1] = nullptr;
        p.A[0] = a.gwg ? a.ggate : a.gup;
    }
    if (split_pays(kGatedGw, p, a.ndat)) return launch_gated_gemm(kGatedGw, p, stream);
    if (a.gwg) KAI_TRY(kai_matmul_backward_w(0, a.gwg, a.ggate, a.x, a.yvec, a.ndat, a.xvec, a.acc));
    if (a.gwu) KAI_TRY(kai_matmul_backward_w(0, a.gwu, a.gup, a.x, a.yvec, a.ndat, a.xvec, a.acc));
    return KAI_OK;
}

}  // namespace kai
