// The gated feed-forward projection of few rows: y[m, j] = act(<x_m, wg_j> + bg_j) * (<x_m, wu_j> + bu_j), m up to 32.
//
// Bound: HBM, the two weights are read once.  A workgroup owns 16 outputs j of all rows and cuts the reduction over its
// eight waves: 16 rows of each weight come straight from memory into the left operands of v_mfma_f32_16x16x32_bf16 (a lane:
// eight steps of a row, so four lanes read 128 contiguous bytes of it), 16 or 32 rows of x from the L2 into the right ones,
// all cut into three bf16 pieces (split_bf16.h).  A lane ends with four outputs of one row of gate and of up each; the waves'
// sums meet in LDS, where a thread takes one output through the epilogue: one launch, no sums in memory.
//
// Measured: 1 x 256 -> 512 3.7 us, 16 x 1024 -> 4096 10.1 (3.3 TB/s), 1 and 16 x 4096 -> 4096 25.4 and 26.7 (5.3 and 5.0).  Four waves
// instead of eight: 35.3 and 35.1 (the chains of steps are twice as long); the weights loaded two steps ahead: 27.0 and 29.0 (the
// registers cost a round of workgroups).
#include <cmath>

#include "act_funcs.h"
#include "decoder_ops.h"
#include "split_bf16.h"

namespace kai {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kWaves = 8;
constexpr int kSteps = 32;             // of the reduction, a matrix instruction's

// eight steps of a row from k on, those below K
__device__ __forceinline__ void load8(float (&to)[8], const float* row, int k, int K) {
    if (k + 8 <= K) {
        const f32x4u a = *reinterpret_cast<const f32x4u*>(row + k), b = *reinterpret_cast<const f32x4u*>(row + k + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            to[i] = a[i];
            to[4 + i] = b[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) to[i] = k + i < K ? row[k + i] : 0.0f;
    }
}

__device__ __forceinline__ float plain_dot(const float* a, const float* b, int64_t K) {
    float sum = 0.0f;
    for (int64_t k = 0; k < K; k++) sum = fmaf(a[k], b[k], sum);
    return sum;
}

template <int XT>
__global__ __launch_bounds__(64 * kWaves, 4) void gated_rows_kernel(GatedArgs a) {
    __shared__ float meet[kWaves][XT * 2 * 4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int n = lane & 15, g = lane >> 4;
    const int K = (int)a.xvec;
    const int64_t j0 = (int64_t)blockIdx.x * 16;
    const int all = (K + kSteps - 1) / kSteps, each = (all + kWaves - 1) / kWaves;
    const int s0 = wave * each, s1 = s0 + each < all ? s0 + each : all;
    // rows behind the last are the last once more, and not stored
    const int64_t j = j0 + n < a.yvec ? j0 + n : a.yvec - 1;
    const float* wrow[2] = {a.wg + j * a.xvec, a.wu + j * a.xvec};
    const float* xrow[XT];
#pragma unroll
    for (int t = 0; t < XT; t++) xrow[t] = a.x + (16 * t + n < a.ndat ? 16 * t + n : a.ndat - 1) * a.xvec;
    f32x4 acc[2][XT];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int t = 0; t < XT; t++) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float w[2][8], x[XT][8];
    const auto load_x = [&](int s) {
#pragma unroll
        for (int t = 0; t < XT; t++) load8(x[t], xrow[t], s * kSteps + 8 * g, K);
    };
    const auto load_w = [&](int s) {
#pragma unroll
        for (int i = 0; i < 2; i++) load8(w[i], wrow[i], s * kSteps + 8 * g, K);
    };
    if (s0 < s1) {
        load_x(s0);
        load_w(s0);
    }
    for (int s = s0; s < s1; s++) {
        const bool more = s + 1 < s1;
        Split8 xs[XT];
#pragma unroll
        for (int t = 0; t < XT; t++) xs[t] = split8([&](int e) { return x[t][e]; });
        if (more) load_x(s + 1);
        Split8 ws[2];
#pragma unroll
        for (int i = 0; i < 2; i++) ws[i] = split8([&](int e) { return w[i][e]; });
        if (more) load_w(s + 1);
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int t = 0; t < XT; t++) {
                f32x4 c = acc[i][t];
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws[i].h, xs[t].l, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws[i].l, xs[t].h, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws[i].m, xs[t].m, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws[i].h, xs[t].m, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws[i].m, xs[t].h, c, 0, 0, 0);
                acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ws[i].h, xs[t].h, c, 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < XT; t++)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) meet[wave][(t * 2 + i) * 4 + e][lane] = acc[i][t][e];
    __syncthreads();
    // a thread's output j0 + c of row m stands in lane 16 (c / 4) + m % 16, element c % 4, of tile m / 16
    const int c = threadIdx.x % 16, m = threadIdx.x / 16;
    if (m >= 16 * XT || m >= a.ndat || j0 + c >= a.yvec) return;
    const int from = 16 * (c / 4) + m % 16, reg = m / 16 * 8 + c % 4;
    float v = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        v += meet[i][reg][from];
        u += meet[i][reg + 4][from];
    }
    const int64_t col = j0 + c, at = (int64_t)m * a.yvec + col;
    // an infinity comes out as a NaN: the plain sums
    if (v != v) v = plain_dot(a.x + m * a.xvec, a.wg + col * a.xvec, a.xvec);
    if (u != u) u = plain_dot(a.x + m * a.xvec, a.wu + col * a.xvec, a.xvec);
    if (a.bg) v += a.bg[col];
    if (a.bu) u += a.bu[col];
    if (a.gate) {
        a.gate[at] = v;
        a.up[at] = u;
    }
    a.y[at] = apply_act(v, a.act, a.hleaky ? *a.hleaky : 0.0f) * u;
}

}  // namespace

// Against two of the dense layer's products and the activation behind them.  Both sides as straight lines through 55
// measurements (1, 4, 16, 24 and 32 rows of 11 shapes, weights from HBM): this kernel takes its waves' chain of steps, one in
// flight at a time, or the weights at 5900 bytes a ns and less with more rows (every workgroup cuts the same x); the products
// take three launches and the weights at 7000 or 6000.  Measured (us, two products | this kernel): 24 x 256 -> 512 8.8 | 5.0,
// 16 x 1024 -> 4096 17.6 | 10.1, 16 and 32 x 4096 -> 4096 29.2 and 37.0 | 26.7 and 33.7, 1 x the same 24.7 | 25.4;
// 16 x 4096 -> 1024, where a quarter of the chip works, 20.7 | 24.5; 1, 16 and 24 x 4096 -> 11008 57.9, 63.5 and
// 72.1 | 64.2, 74.0 and 87.0.
bool gated_rows_pays(const GatedArgs& a) {
    if (a.ndat > 32 || a.xvec <= 0 || a.xvec >= (1ll << 30) || a.yvec >= (1ll << 26)) return false;   // 32-bit step and thread counts
    const double bytes = 8.0 * (double)a.xvec * (double)a.yvec, rows = (double)a.ndat;
    const double rounds = std::ceil((double)((a.yvec + 15) / 16) / (2.0 * compute_units()));
    const double work = 3.2 + rounds * (double)a.xvec / 256.0 * (0.93 + 0.0265 * rows);
    const double read = 3.2 + bytes / (5.9e6 - 0.05e6 * rows);
    const double products = (a.ndat == 1 ? 6.5 : 8.5 + 0.17 * rows) + bytes / (a.ndat <= 16 ? 7.0e6 : 6.0e6);
    return (work > read ? work : read) < products;
}

int launch_gated_rows(const GatedArgs& a, hipStream_t stream) {
    const unsigned grid = (unsigned)((a.yvec + 15) / 16);
    if (a.ndat <= 16) gated_rows_kernel<1><<<grid, 64 * kWaves, 0, stream>>>(a);
    else gated_rows_kernel<2><<<grid, 64 * kWaves, 0, stream>>>(a);
    return check_launch("gated_rows_kernel");
}

}  // namespace kai
