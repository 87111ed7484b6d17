// The matrix products of the gated feed-forward projection (gated_gemm.hip).
#pragma once

#include "kai_common.h"

namespace kai {

enum : int { kGatedForward = 0, kGatedGx = 1, kGatedGw = 2 };

struct GatedGemm {
    const float* A[2];      // forward: x; gx, gw: gradients of gate and up
    const float* B[2];      // forward, gx: the two weights; gw: x
    float* C[3];            // forward: y, gate, up (the last two may be null); gx: gx; gw: gwg, gwu
    const float* bias[2];   // forward: may be null
    const float* hleaky;
    int64_t M, lda, ldb, ldc;
    int64_t N;
    int K;
    int act, acc;
    int nwhich;             // gw: 2 products, or 1; otherwise 1
    // filled by the launcher
    int tiles_m, tiles_n, run, part_steps;
    int whole, cut, nparts; // tiles that one workgroup takes whole; the others, and the parts of the reduction of each
    int wide;               // outputs in rows of whole 16-byte lines
    float* parts;           // [nparts][cut] tiles of sums
};

bool gated_gemm_applies(int mode, const GatedGemm& p);
// what the products would take, as the choice of their tiles estimates it
double gated_gemm_us(int mode, const GatedGemm& p);
// the plan itself: tiles of rows x columns of the products (forward: of gate and up together), those taken whole and those
// whose reduction is cut into parts, and the bytes of scratch that the parts take
struct GatedGemmPlan {
    int rows, columns, whole, cut, parts;
    int64_t scratch;
};
GatedGemmPlan gated_gemm_plan(int mode, const GatedGemm& p);
int launch_gated_gemm(int mode, const GatedGemm& p, hipStream_t stream);

}  // namespace kai
