// The gated feed-forward projection: y = act(x . wg^T + bg) * (x . wu^T + bu), and its element-wise gradients.
#include "act_funcs.h"
#include "decoder_ops.h"
#include "elementwise.h"
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

// ggate = gy * up * act'(gate), gup = gy * act(gate) and, on the way, their column sums: a workgroup takes 64 * VEC columns of
// `chunk` rows, a wave every fourth of them, and leaves the sums of its rows in sums[2][chunks][ncol] (null: no sums wanted).
// Bound: HBM, five floats an element; the sums cost nothing beside that, where sums of the stored gradients would read
// two of the five again.  2048 x 4096: 31 .. 37 us = 5.4 .. 4.5 TB/s, and 4.6 for the chunks' sums.
template <int VEC>
__global__ __launch_bounds__(kThreads) void gated_activation_backward_kernel(float* ggate, float* gup, float* sums, const float* gy,
                                                                             const float* gate, const float* up, int64_t nrow,
                                                                             int64_t ncol, int chunk, int act,
                                                                             const float* hleaky) {
    typedef float vec __attribute__((ext_vector_type(VEC)));
    __shared__ float meet[3][2][64 * VEC];
    const float leaky = hleaky ? *hleaky : 0.0f;
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * VEC, r0 = (int64_t)blockIdx.y * chunk;
    const int64_t r1 = r0 + chunk < nrow ? r0 + chunk : nrow;
    float sg[VEC] = {}, su[VEC] = {};
    if (c < ncol) {
        for (int64_t r = r0 + wave; r < r1; r += 4) {
            const int64_t at = r * ncol + c;
            const vec d = *reinterpret_cast<const vec*>(gy + at), g = *reinterpret_cast<const vec*>(gate + at);
            const vec u = *reinterpret_cast<const vec*>(up + at);
            vec a, b;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                a[e] = d[e] * u[e] * act_derivative(g[e], act, leaky);
                b[e] = d[e] * apply_act(g[e], act, leaky);
                sg[e] += a[e];
                su[e] += b[e];
            }
            *reinterpret_cast<vec*>(ggate + at) = a;
            *reinterpret_cast<vec*>(gup + at) = b;
        }
    }
    if (sums == nullptr) return;
    if (wave > 0) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            meet[wave - 1][0][lane * VEC + e] = sg[e];
            meet[wave - 1][1][lane * VEC + e] = su[e];
        }
    }
    __syncthreads();
    if (wave > 0 || c >= ncol) return;
    float* to = sums + (int64_t)blockIdx.y * ncol + c;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        to[e] = sg[e] + meet[0][0][lane * VEC + e] + meet[1][0][lane * VEC + e] + meet[2][0][lane * VEC + e];
        to[(int64_t)gridDim.y * ncol + e] = su[e] + meet[0][1][lane * VEC + e] + meet[1][1][lane * VEC + e] + meet[2][1][lane * VEC + e];
    }
}

// gb (+)= the chunks' sums: 64 columns a workgroup, every fourth chunk a wave; blockIdx.y: gate or up
__global__ __launch_bounds__(kThreads) void gated_bias_kernel(float* gbg, float* gbu, const float* sums, int64_t ncol, int chunks,
                                                              int acc) {
    __shared__ float meet[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float* gb = blockIdx.y ? gbu : gbg;
    if (gb == nullptr) return;
    const float* from = sums + (int64_t)blockIdx.y * chunks * ncol + c;
    float sum = 0.0f;
    if (c < ncol) {
#pragma unroll 8
        for (int i = wave; i < chunks; i += 4) sum += from[i * ncol];
    }
    if (wave > 0) meet[wave - 1][lane] = sum;
    __syncthreads();
    if (wave > 0 || c >= ncol) return;
    sum += meet[0][lane] + meet[1][lane] + meet[2][lane];
    gb[c] = acc ? gb[c] + sum : sum;
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

int launch_gated_activation_backward(float* ggate, float* gup, float* gbg, float* gbu, const float* gy, const float* gate,
                                     const float* up, int64_t nrow, int64_t ncol, int act, const float* hleaky, int acc,
                                     hipStream_t stream) {
    const bool wide = ncol % 4 == 0 && aligned16(ggate) && aligned16(gup) && aligned16(gy) && aligned16(gate) && aligned16(up);
    const int64_t strip = wide ? 256 : 64, strips = (ncol + strip - 1) / strip;
    if (strips >= (1ll << 24)) return fail(KAI_ERR_INVALID_ARGUMENT, "gated_backward: too many columns");
    // eight workgroups for a compute unit, and at least 16 rows for each
    int64_t chunks = (8 * (int64_t)compute_units() + strips - 1) / strips;
    if (chunks > (nrow + 15) / 16) chunks = (nrow + 15) / 16;
    if (chunks > 65535) chunks = 65535;
    const int64_t chunk = (nrow + chunks - 1) / chunks;
    chunks = (nrow + chunk - 1) / chunk;
    float* sums = nullptr;
    // no scratch to be had (the stream is being captured and the buffer would have to grow), or more than a product may ask: the
    // sums read the gradients again
    const bool wanted = gbg || gbu;
    const int64_t sums_bytes = 2 * chunks * ncol * (int64_t)sizeof(float);
    const bool fused = wanted && sums_bytes <= kProductScratchMax && workspace(sums_bytes, &sums) == KAI_OK;
    if (wanted && !fused) {
        sums = nullptr;
        clear_error();
    }
    const dim3 grid((unsigned)strips, (unsigned)chunks);
    if (wide) gated_activation_backward_kernel<4><<<grid, kThreads, 0, stream>>>(ggate, gup, sums, gy, gate, up, nrow, ncol, (int)chunk, act, hleaky);
    else gated_activation_backward_kernel<1><<<grid, kThreads, 0, stream>>>(ggate, gup, sums, gy, gate, up, nrow, ncol, (int)chunk, act, hleaky);
    KAI_TRY(check_launch("gated_activation_backward_kernel"));
    if (!wanted) return KAI_OK;
    if (!fused) {
        if (gbg) KAI_TRY(launch_colsum(gbg, ggate, nrow, ncol, acc, stream));
        return gbu ? launch_colsum(gbu, gup, nrow, ncol, acc, stream) : KAI_OK;
    }
    gated_bias_kernel<<<dim3((unsigned)((ncol + 63) / 64), 2), kThreads, 0, stream>>>(gbg, gbu, sums, ncol, (int)chunks, acc);
    return check_launch("gated_bias_kernel");
}

static GatedGemm forward_product(const GatedArgs& a) {
    GatedGemm p{};
    p.A[0] = a.x; p.B[0] = a.wg; p.B[1] = a.wu;
    p.C[0] = a.y; p.C[1] = a.gate; p.C[2] = a.up;
    p.bias[0] = a.bg; p.bias[1] = a.bu;
    p.hleaky = a.hleaky; p.act = a.act;
    p.M = a.ndat; p.N = a.yvec; p.K = (int)a.xvec;
    p.lda = p.ldb = a.xvec; p.ldc = a.yvec;
    p.nwhich = 1;
    return p;
}
static bool tiled_forward(const GatedArgs& a, const GatedGemm& p) { return a.ndat > 32 && gated_gemm_applies(kGatedForward, p); }

int launch_gated_forward(const GatedArgs& a, hipStream_t stream) {
    const GatedGemm p = forward_product(a);
    if (gated_rows_pays(a)) return launch_gated_rows(a, stream);
    if (tiled_forward(a, p)) return launch_gated_gemm(kGatedForward, p, stream);
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

static GatedGemm x_product(const GatedGradArgs& a) {
    GatedGemm p{};
    p.A[0] = a.ggate; p.A[1] = a.gup;
    p.B[0] = a.wg; p.B[1] = a.wu;
    p.C[0] = a.gx;
    p.M = a.ndat; p.N = a.xvec; p.K = (int)a.yvec;
    p.lda = a.yvec; p.ldb = p.ldc = a.xvec;
    p.acc = a.acc;
    p.nwhich = 1;
    return p;
}
static GatedGemm weight_product(const GatedGradArgs& a) {
    GatedGemm p{};
    p.A[0] = a.ggate; p.A[1] = a.gup;
    p.B[0] = a.x;
    p.C[0] = a.gwg; p.C[1] = a.gwu;
    p.M = a.yvec; p.N = a.xvec; p.K = (int)a.ndat;
    p.lda = a.yvec; p.ldb = p.ldc = a.xvec;
    p.acc = a.acc;
    p.nwhich = 2;
    if (a.gwg == nullptr || a.gwu == nullptr) {
        p.nwhich = 1;
        p.C[0] = a.gwg ? a.gwg : a.gwu;
        p.C[1] = nullptr;
        p.A[0] = a.gwg ? a.ggate : a.gup;
    }
    return p;
}

int launch_gated_gradients(const GatedGradArgs& a, hipStream_t stream) {
    if (a.gx) {
        const GatedGemm p = x_product(a);
        if (split_pays(kGatedGx, p, a.ndat)) {
            KAI_TRY(launch_gated_gemm(kGatedGx, p, stream));
        } else {
            KAI_TRY(kai_matmul_backward_x(0, a.gx, a.ggate, a.wg, a.yvec, a.ndat, a.xvec, a.acc));
            KAI_TRY(kai_matmul_backward_x(0, a.gx, a.gup, a.wu, a.yvec, a.ndat, a.xvec, 1));
        }
    }
    if (a.gwg == nullptr && a.gwu == nullptr) return KAI_OK;
    const GatedGemm p = weight_product(a);
    if (split_pays(kGatedGw, p, a.ndat)) return launch_gated_gemm(kGatedGw, p, stream);
    if (a.gwg) KAI_TRY(kai_matmul_backward_w(0, a.gwg, a.ggate, a.x, a.yvec, a.ndat, a.xvec, a.acc));
    if (a.gwu) KAI_TRY(kai_matmul_backward_w(0, a.gwu, a.gup, a.x, a.yvec, a.ndat, a.xvec, a.acc));
    return KAI_OK;
}

std::string gated_plan_text(int which, int64_t yvec, int64_t ndat, int64_t xvec) {
    static float there;      // of outputs that are wanted; nothing is read
    GatedArgs f{};
    f.yvec = yvec; f.ndat = ndat; f.xvec = xvec;
    GatedGradArgs g{};
    g.gwg = g.gwu = &there;
    g.yvec = yvec; g.ndat = ndat; g.xvec = xvec;
    const int mode = which == 0 ? kGatedForward : which == 1 ? kGatedGx : kGatedGw;
    const GatedGemm p = which == 0 ? forward_product(f) : which == 1 ? x_product(g) : weight_product(g);
    if (which == 0 && gated_rows_pays(f)) return "rows";
    if (which == 0 ? !tiled_forward(f, p) : !split_pays(mode, p, ndat)) return "separate";
    const GatedGemmPlan plan = gated_gemm_plan(mode, p);
    std::string text = "tiles " + std::to_string(plan.rows) + " x " + std::to_string(plan.columns) + ", " + std::to_string(plan.whole) + " whole";
    if (plan.cut > 0) text += ", " + std::to_string(plan.cut) + " in " + std::to_string(plan.parts) + " parts";
    return text + ", scratch " + std::to_string(plan.scratch);
}

}  // namespace kai
