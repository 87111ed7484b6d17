// The matrix products of the gated feed-forward projection on the bf16 matrix cores at fp32 accuracy
// (split_bf16.h): six v_mfma_f32_32x32x16_bf16 for each 16 steps of the reduction.
//
//   forward   gate | up [M, N] = x[M, K] . wg^T | x . wu^T, both K-contiguous; a wave's blocks alternate between the two
//             weights, so that gate and up of an output meet in one lane: y = act(gate + bg) * (up + bu) in the epilogue
//   gx        [M, N] = gg[M, K] . wg[K, N] + gu . wu: one reduction over both pairs, one after the other
//   gw        gwg | gwu [M, N] = gg^T | gu^T . x, operands [K, M] and [K, N]: the two products side by side in one launch
//
// A workgroup stages 16 steps of its operands' rows at a time: global loads to registers one step ahead, there cut into
// three bf16 planes (which also turns a [K, rows] operand: a thread holds eight steps of one row), LDS double buffered,
// one barrier a step.  LDS holds a plane as [half of the steps][row][8 steps]: fragments are 16-byte chunks of
// consecutive rows, read and (but for K-contiguous operands' half chunks) written without bank conflicts.
//
// What lies outside an operand reads as 0 (buffer loads end with it); the last, partial step of a K-contiguous operand is
// masked.  Where an operand held an infinity, or a value that rounds to one in bf16, sums that came out as NaN are formed
// again in plain fp32, so that an infinity has the effect it has there.
#include "act_funcs.h"
#include "gated_gemm.h"
#include "split_bf16.h"

namespace kai {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kStep = 16;
constexpr int kPadRows = 8;            // between the halves of a plane: the two halves' writes meet different banks
constexpr float kBf16Limit = 3.38e38f; // above 3.3895e38 the first piece rounds to infinity

__device__ __forceinline__ float* uniform_ptr(const float* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
    return reinterpret_cast<float*>(((uint64_t)hi << 32) | lo);
}

// bytes [from, end), as far as 32 bits reach; negative: none
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_from(const float* from, const float* end) {
    const int64_t left = (end - from) * (int64_t)sizeof(float);
    const uint32_t bytes = left <= 0 ? 0u : left > 0xFFFFFFFFll ? 0xFFFFFFFFu : (uint32_t)left;
    return __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(from), 0, (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// One operand's tile of ROWS rows x 16 steps.  Eight floats a thread: KC (steps contiguous): two chunks of four steps,
// otherwise eight steps of one row.
template <bool KC, int ROWS, int NT>
struct Tile {
    static_assert(ROWS * kStep == 8 * NT, "eight floats a thread");
    static constexpr int kHalf = (ROWS + kPadRows) * 16;      // bytes
    static constexpr int kPlane = 2 * kHalf;
    static constexpr int kBytes = 3 * kPlane;

    // row of the tile that chunk i of this thread loads
    static __device__ __forceinline__ int row_of(int i) { return KC ? ((int)threadIdx.x + i * NT) / 4 : (int)threadIdx.x % ROWS; }

    static __device__ __forceinline__ void load_kc(float (&x)[8], int i, __amdgpu_buffer_rsrc_t rsrc, uint32_t off) {
        const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
#pragma unroll
        for (int e = 0; e < 4; e++) x[4 * i + e] = v[e];
    }

    // steps from `left` on do not exist
    static __device__ __forceinline__ void mask_kc(float (&x)[8], int left) {
        const int q = (int)threadIdx.x % 4 * 4;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (q + i % 4 >= left) x[i] = 0.0f;
    }

    static __device__ __forceinline__ void store(char* lds, const float (&x)[8], float& largest) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) largest = fmaxf(fmaxf(fabsf(x[i]), fabsf(x[i + 1])), largest);
        unsigned h[4], m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_pair(x[2 * i], x[2 * i + 1], h[i], m[i], l[i]);
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int q = (int)threadIdx.x % 4;
                char* to = lds + (q / 2) * kHalf + row_of(i) * 16 + (q % 2) * 8;
                *reinterpret_cast<u32x2*>(to) = u32x2{h[2 * i], h[2 * i + 1]};
                *reinterpret_cast<u32x2*>(to + kPlane) = u32x2{m[2 * i], m[2 * i + 1]};
                *reinterpret_cast<u32x2*>(to + 2 * kPlane) = u32x2{l[2 * i], l[2 * i + 1]};
            }
        } else {
            char* to = lds + ((int)threadIdx.x / ROWS) * kHalf + row_of(0) * 16;
            *reinterpret_cast<u32x4v*>(to) = u32x4v{h[0], h[1], h[2], h[3]};
            *reinterpret_cast<u32x4v*>(to + kPlane) = u32x4v{m[0], m[1], m[2], m[3]};
            *reinterpret_cast<u32x4v*>(to + 2 * kPlane) = u32x4v{l[0], l[1], l[2], l[3]};
        }
    }

    // operand of the 32 rows from `row` on
    static __device__ __forceinline__ Split8 fragment(const char* lds, int row) {
        const int lane = threadIdx.x & 63;
        const char* from = lds + (lane >> 5) * kHalf + (row + (lane & 31)) * 16;
        return Split8{*reinterpret_cast<const bf16x8*>(from), *reinterpret_cast<const bf16x8*>(from + kPlane),
                      *reinterpret_cast<const bf16x8*>(from + 2 * kPlane)};
    }
};

// The plain sum of one output, for sums that an infinity entered: the reduction steps [s0, s1) of the launch
template <int MODE>
__device__ float plain_sum(const GatedGemm& p, int which, int64_t m, int64_t n, int s0, int s1) {
    float sum = 0.0f;
    const int steps = (p.K + kStep - 1) / kStep;
    for (int s = s0; s < s1; s++) {
        const int seg = MODE == kGatedGx && s >= steps ? 1 : 0;
        const int k0 = (s - seg * steps) * kStep;
        for (int k = k0; k < k0 + kStep && k < p.K; k++) {
            if (MODE == kGatedForward) sum = fmaf(p.A[0][m * p.lda + k], p.B[which][n * p.ldb + k], sum);
            if (MODE == kGatedGx) sum = fmaf(p.A[seg][m * p.lda + k], p.B[seg][k * p.ldb + n], sum);
            if (MODE == kGatedGw) sum = fmaf(p.A[which][k * p.lda + m], p.B[0][k * p.ldb + n], sum);
        }
    }
    return sum;
}

constexpr int kStageRow = 68;          // floats: a wave's 32 rows of 64 outputs in LDS

// columns n .. n + 3 of a row, those below N
__device__ __forceinline__ void put(float* row, int64_t n, int64_t N, const f32x4& v, int wide) {
    if (wide && n + 4 <= N) {
        *reinterpret_cast<f32x4*>(row + n) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < N) row[n + e] = v[e];
    }
}

template <int MODE, int WM, int WN, int NBM>
struct Shape {
    static constexpr int NBN = 2;
    static constexpr int NT = 64 * WM * WN, BM = 32 * NBM * WM, BN = 32 * NBN * WN;
    static constexpr bool AKC = MODE != kGatedGw, BKC = MODE == kGatedForward;
    using TA = Tile<AKC, BM, NT>;
    using TB = Tile<BKC, BN, NT>;
    static constexpr int kLds = 2 * (TA::kBytes + TB::kBytes);
    static constexpr int kStageFloats = 32 * kStageRow;
    static_assert(kStageFloats * 4 * WM * WN <= kLds, "the epilogue's rows fit where the operands were");
    static constexpr int kColumns = MODE == kGatedForward ? BN / 2 : BN;    // of the output that a tile covers
};

template <int MODE, int WM, int WN, int NBM>
__global__ __launch_bounds__(64 * WM * WN, 2) void gated_gemm_kernel(GatedGemm p) {
    using S = Shape<MODE, WM, WN, NBM>;
    using TA = typename S::TA;
    using TB = typename S::TB;
    constexpr int NBN = S::NBN;
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int wm = wave / WN, wn = wave % WN;

    // Tiles in runs of `run` tile rows by all columns, and consecutive ones on one XCD (workgroup ids go round the eight)
    int tm, tn, which;
    {
        const int tiles_mn = p.tiles_m * p.tiles_n, total = tiles_mn * p.nwhich;
        int id = blockIdx.x;
        const int each = total / 8, rest = total % 8, xcd = id % 8, at = id / 8;
        id = xcd * each + (xcd < rest ? xcd : rest) + at;
        which = id / tiles_mn;
        id -= which * tiles_mn;
        const int run = p.run * p.tiles_n;
        const int first = id / run * p.run;
        const int rows = p.tiles_m - first < p.run ? p.tiles_m - first : p.run;
        const int in = id % run;
        tm = first + in % rows;
        tn = in / rows;
    }
    const int64_t m0 = (int64_t)tm * S::BM, n0 = (int64_t)tn * S::kColumns;
    const int steps = (p.K + kStep - 1) / kStep, all_steps = MODE == kGatedGx ? 2 * steps : steps;
    const int s0 = (int)blockIdx.y * p.part_steps;
    const int s1 = s0 + p.part_steps < all_steps ? s0 + p.part_steps : all_steps;

    // byte offsets of this thread's rows from the tile's first row
    uint32_t aoff[2], boff[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        aoff[i] = S::AKC ? (uint32_t)((TA::row_of(i) * p.lda + (int)threadIdx.x % 4 * 4) * 4) : (uint32_t)TA::row_of(0) * 4;
        boff[i] = S::BKC ? (uint32_t)((TB::row_of(i) % 32 + TB::row_of(i) / 64 * 32) * p.ldb + (int)threadIdx.x % 4 * 4) * 4
                         : (uint32_t)TB::row_of(0) * 4;
    }
    float xa[8], xb[8];
    float largest = 0.0f;
    const auto load = [&](int s) {
        const int seg = MODE == kGatedGx && s >= steps ? 1 : 0;
        const int64_t k0 = (int64_t)(s - seg * steps) * kStep;
        const float* A = MODE == kGatedGx ? p.A[seg] : MODE == kGatedGw ? p.A[which] : p.A[0];
        if constexpr (S::AKC) {
            const auto rsrc = rsrc_from(A + m0 * p.lda + k0, A + (p.M - 1) * p.lda + p.K);
#pragma unroll
            for (int i = 0; i < 2; i++) TA::load_kc(xa, i, rsrc, aoff[i]);
        } else {
            const auto rsrc = rsrc_from(A + k0 * p.lda + m0, A + (p.K - 1) * p.lda + p.M);
            const uint32_t oct = (uint32_t)threadIdx.x / S::BM * 8;
#pragma unroll
            for (int i = 0; i < 8; i++)
                xa[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, aoff[0] + (oct + i) * (uint32_t)(p.lda * 4), 0, 0));
        }
        if constexpr (S::BKC) {
            // rows of the tile alternate between the weights, 32 at a time
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int w = __builtin_amdgcn_readfirstlane(TB::row_of(i) / 32 % 2);
                const float* B = p.B[w];
                TB::load_kc(xb, i, rsrc_from(B + n0 * p.ldb + k0, B + (p.N - 1) * p.ldb + p.K), boff[i]);
            }
        } else {
            const float* B = p.B[seg];
            const auto rsrc = rsrc_from(B + k0 * p.ldb + n0, B + (p.K - 1) * p.ldb + p.N);
            const uint32_t oct = (uint32_t)threadIdx.x / S::BN * 8;
#pragma unroll
            for (int i = 0; i < 8; i++)
                xb[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, boff[0] + (oct + i) * (uint32_t)(p.ldb * 4), 0, 0));
        }
        const int left = p.K - (int)k0;
        if (left < kStep) {
            if constexpr (S::AKC) TA::mask_kc(xa, left);
            if constexpr (S::BKC) TB::mask_kc(xb, left);
        }
    };
    const auto store = [&](int buffer) {
        char* to = lds + buffer * (TA::kBytes + TB::kBytes);
        TA::store(to, xa, largest);
        TB::store(to + TA::kBytes, xb, largest);
    };

    f32x16 acc[NBM][NBN];
#pragma unroll
    for (int i = 0; i < NBM; i++)
#pragma unroll
        for (int j = 0; j < NBN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;

    if (s0 < s1) {
        load(s0);
        store(0);
    }
    __syncthreads();
    for (int s = s0; s < s1; s++) {
        const bool more = s + 1 < s1;
        if (more) load(s + 1);
        const char* from = lds + (s - s0) % 2 * (TA::kBytes + TB::kBytes);
        Split8 b[NBN];
#pragma unroll
        for (int j = 0; j < NBN; j++) b[j] = TB::fragment(from + TA::kBytes, wn * 32 * NBN + 32 * j);
#pragma unroll
        for (int i = 0; i < NBM; i++) {
            const Split8 a = TA::fragment(from, wm * 32 * NBM + 32 * i);
            // the small products first
#pragma unroll
            for (int j = 0; j < NBN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b[j].l, acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NBN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.l, b[j].h, acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NBN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b[j].m, acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NBN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b[j].m, acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NBN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.m, b[j].h, acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < NBN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b[j].h, acc[i][j], 0, 0, 0);
        }
        if (more) store((s + 1 - s0) % 2);
        __syncthreads();
    }

    // Epilogue by way of LDS, a wave's own 32 rows at a time: the accumulators hold one column a lane, the stores want four
    // columns of a row, and the activation's code stands there once instead of once for every register.
    const bool again = __syncthreads_or(!(largest < kBf16Limit));
    const float leaky = MODE == kGatedForward && p.hleaky ? *p.hleaky : 0.0f;
    float* stage = reinterpret_cast<float*>(lds) + wave * S::kStageFloats;
#pragma unroll
    for (int i = 0; i < NBM; i++) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NBN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                stage[(8 * (e / 4) + 4 * (lane >> 5) + e % 4) * kStageRow + 32 * j + (lane & 31)] = acc[i][j][e];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int r = lane / 8; r < 32; r += 8) {
            const int64_t m = m0 + wm * 32 * NBM + 32 * i + r;
            if (m >= p.M) break;
            const float* row = stage + r * kStageRow + lane % 8 * 4;
            f32x4 v = *reinterpret_cast<const f32x4*>(row), u = *reinterpret_cast<const f32x4*>(row + 32);
            const int c = lane % 8 * 4;
            const int64_t n = n0 + wn * (MODE == kGatedForward ? 32 : 64) + c;
            const int64_t n2 = MODE == kGatedForward ? n : n + 32;
            if (again) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (v[e] != v[e] && n + e < p.N) v[e] = plain_sum<MODE>(p, which, m, n + e, s0, s1);
                    if (u[e] != u[e] && n2 + e < p.N) u[e] = plain_sum<MODE>(p, MODE == kGatedForward ? 1 : which, m, n2 + e, s0, s1);
                }
            }
            const int64_t at = m * p.ldc;
            if constexpr (MODE == kGatedForward) {
                if (p.parts) {
                    float* part = p.parts + (int64_t)blockIdx.y * 2 * p.M * p.ldc + at;
                    put(part, n, p.N, v, p.wide);
                    put(part + p.M * p.ldc, n, p.N, u, p.wide);
                } else {
                    f32x4 y;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (n + e < p.N) {
                            v[e] += p.bias[0] ? p.bias[0][n + e] : 0.0f;
                            u[e] += p.bias[1] ? p.bias[1][n + e] : 0.0f;
                        }
                        y[e] = apply_act(v[e], p.act, leaky) * u[e];
                    }
                    if (p.C[1]) {
                        put(p.C[1] + at, n, p.N, v, p.wide);
                        put(p.C[2] + at, n, p.N, u, p.wide);
                    }
                    put(p.C[0] + at, n, p.N, y, p.wide);
                }
            } else if (p.parts) {
                float* part = p.parts + ((int64_t)blockIdx.y * p.nwhich + which) * p.M * p.ldc + at;
                put(part, n, p.N, v, p.wide);
                put(part, n2, p.N, u, p.wide);
            } else {
                float* c0 = p.C[which] + at;
                if (p.acc) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (n + e < p.N) v[e] += c0[n + e];
                        if (n2 + e < p.N) u[e] += c0[n2 + e];
                    }
                }
                put(c0, n, p.N, v, p.wide);
                put(c0, n2, p.N, u, p.wide);
            }
        }
    }
}

// sums the parts, with the forward's epilogue or onto the gradient
template <int MODE>
__global__ __launch_bounds__(256) void gated_parts_kernel(GatedGemm p, int nparts) {
    const int64_t one = p.M * p.ldc, total = one * (MODE == kGatedForward ? 1 : p.nwhich);
    const int64_t all = one * (MODE == kGatedForward ? 2 : p.nwhich);
    const float leaky = MODE == kGatedForward && p.hleaky ? *p.hleaky : 0.0f;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        float v = 0.0f, u = 0.0f;
        for (int s = 0; s < nparts; s++) {
            v += p.parts[s * all + e];
            if (MODE == kGatedForward) u += p.parts[s * all + one + e];
        }
        if constexpr (MODE == kGatedForward) {
            const int64_t n = e % p.ldc;
            v += p.bias[0] ? p.bias[0][n] : 0.0f;
            u += p.bias[1] ? p.bias[1][n] : 0.0f;
            if (p.C[1]) {
                p.C[1][e] = v;
                p.C[2][e] = u;
            }
            p.C[0][e] = apply_act(v, p.act, leaky) * u;
        } else {
            const int which = (int)(e / one);
            float* c = p.C[which] + (e - which * one);
            *c = p.acc ? *c + v : v;
        }
    }
}

template <int MODE, int WM, int WN, int NBM>
int launch_shape(GatedGemm p, int64_t nparts, hipStream_t stream) {
    using S = Shape<MODE, WM, WN, NBM>;
    p.tiles_m = (int)((p.M + S::BM - 1) / S::BM);
    p.tiles_n = (int)((p.N + S::kColumns - 1) / S::kColumns);
    p.run = 8;
    if (S::kLds > 64 * 1024)
        KAI_TRY(check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_gemm_kernel<MODE, WM, WN, NBM>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds),
                          "hipFuncSetAttribute(gated_gemm_kernel)"));
    const int steps = (int)((p.K + kStep - 1) / kStep) * (MODE == kGatedGx ? 2 : 1);
    p.part_steps = (int)((steps + nparts - 1) / nparts);
    nparts = p.part_steps > 0 ? (steps + p.part_steps - 1) / p.part_steps : 1;
    if (nparts > 1) {
        const int64_t outputs = p.M * p.ldc * (MODE == kGatedForward ? 2 : p.nwhich);
        KAI_TRY(workspace(nparts * outputs * (int64_t)sizeof(float), &p.parts));
    }
    p.wide = p.ldc % 4 == 0 && aligned16(p.C[0]) && aligned16(p.C[1]) && aligned16(p.C[2]);
    if (p.parts) p.wide = p.ldc % 4 == 0 && p.M * p.ldc % 4 == 0;
    const dim3 grid((unsigned)((int64_t)p.tiles_m * p.tiles_n * p.nwhich), (unsigned)nparts);
    gated_gemm_kernel<MODE, WM, WN, NBM><<<grid, S::NT, S::kLds, stream>>>(p);
    KAI_TRY(check_launch("gated_gemm_kernel"));
    if (nparts == 1) return KAI_OK;
    const int64_t groups = (p.M * p.ldc * p.nwhich + 255) / 256, most = 16 * (int64_t)compute_units();
    gated_parts_kernel<MODE><<<(unsigned)(groups < most ? groups : most), 256, 0, stream>>>(p, (int)nparts);
    return check_launch("gated_parts_kernel");
}

template <int MODE>
int launch_mode(const GatedGemm& p, hipStream_t stream) {
    const int64_t columns = MODE == kGatedForward ? 2 * p.N : p.N;
    const auto tiles = [&](int64_t b) { return (p.M + b - 1) / b * ((columns + b - 1) / b) * p.nwhich; };
    const int64_t cu = compute_units();
    if (tiles(256) >= cu) return launch_shape<MODE, 2, 4, 4>(p, 1, stream);
    int64_t nparts = (2 * cu) / tiles(128);
    const int64_t steps = (p.K + kStep - 1) / kStep * (MODE == kGatedGx ? 2 : 1);
    if (nparts > steps / 16) nparts = steps / 16;
    if (nparts < 1) nparts = 1;
    if (nparts > 16) nparts = 16;
    return launch_shape<MODE, 2, 2, 2>(p, nparts, stream);
}

}  // namespace

// offsets inside a tile are 32-bit
bool gated_gemm_applies(const GatedGemm& p) {
    return p.M > 0 && p.N > 0 && p.K > 0 && p.lda < (1ll << 21) && p.ldb < (1ll << 21);
}

int launch_gated_gemm(int mode, const GatedGemm& p, hipStream_t stream) {
    if (mode == kGatedForward) return launch_mode<kGatedForward>(p, stream);
    if (mode == kGatedGx) return launch_mode<kGatedGx>(p, stream);
    return launch_mode<kGatedGw>(p, stream);
}

}  // namespace kai
