// The matrix products of the gated feed-forward projection on the bf16 matrix cores at fp32 accuracy
// (split_bf16.h): six v_mfma_f32_32x32x16_bf16 for each 16 steps of the reduction.
//
//   forward   gate | up [M, N] = x[M, K] . wg^T | x . wu^T, both K-contiguous; a wave's blocks alternate between the two
//             weights, so that gate and up of an output meet in one lane: y = act(gate + bg) * (up + bu) in the epilogue
//   gx        [M, N] = gg[M, K] . wg[K, N] + gu . wu: one reduction over both pairs, one after the other
//   gw        gwg | gwu [M, N] = gg^T | gu^T . x, operands [K, M] and [K, N]: the two products side by side in one launch
//
// A workgroup stages 16 steps of its operands' rows at a time: global loads to registers two steps ahead, there cut into
// three bf16 planes (which also turns a [K, rows] operand: a thread holds eight steps of one row), LDS double buffered,
// one barrier a step.  LDS holds a plane as [half of the steps][row][8 steps]: fragments are 16-byte chunks of
// consecutive rows, read and (but for K-contiguous operands' half chunks) written without bank conflicts.
//
// Bound: the matrix cores at a sixth of their bf16 rate (235 TFLOP/s of fp32 products at what large bf16 products reach, 1412),
// with the cutting's vector instructions between them.  4096 x 4096 -> 11008 forward 3.15 ms = 234 TFLOP/s on
// one card, 3.47 on another; gradients of 2048 x 1024 -> 4096 173 .. 184 us each = 199 .. 187 TFLOP/s; small products the chain of
// their steps (1000 x 777 -> 333 17 .. 18 us and 5.4 for the sums of two parts).
//
// What lies outside an operand reads as 0 (buffer loads end with it); the last, partial step of a K-contiguous operand is
// masked.  Where an operand held an infinity, which the pieces turn into a NaN, sums that came out as NaN are formed again in
// plain fp32, so that an infinity has the effect it has there.
#include <type_traits>

#include "act_funcs.h"
#include "gated_gemm.h"
#include "split_bf16.h"

namespace kai {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// f(B), ..., f(E - 1) with compile-time indices
template <int B, int E, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (B < E) {
        f(std::integral_constant<int, B>{});
        static_for<B + 1, E>(f);
    }
}

constexpr int kStep = 16;
constexpr int kPadRows = 8;            // between the halves of a plane: the two halves' writes meet different banks

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

// One operand's tile of ROWS rows x 16 steps, F = 4 or 8 floats a thread: KC (steps contiguous): chunks of four steps,
// otherwise F steps of one row.
template <bool KC, int ROWS, int NT>
struct Tile {
    static constexpr int F = ROWS * kStep / NT, kPieces = F / 4;
    static_assert(F * NT == ROWS * kStep && (F == 4 || F == 8), "four or eight floats a thread");
    static constexpr int kHalf = (ROWS + kPadRows) * 16;      // bytes
    static constexpr int kPlane = 2 * kHalf;
    static constexpr int kBytes = 3 * kPlane;

    // row of the tile that chunk i of this thread loads, and the first step of it
    static __device__ __forceinline__ int row_of(int i) { return KC ? ((int)threadIdx.x + i * NT) / 4 : (int)threadIdx.x % ROWS; }
    static __device__ __forceinline__ int step_of() { return KC ? (int)threadIdx.x % 4 * 4 : (int)threadIdx.x / ROWS * F; }

    static __device__ __forceinline__ void load_kc(float (&x)[F], int i, __amdgpu_buffer_rsrc_t rsrc, uint32_t off) {
        const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
#pragma unroll
        for (int e = 0; e < 4; e++) x[4 * i + e] = v[e];
    }

    // steps from `left` on do not exist
    static __device__ __forceinline__ void mask_kc(float (&x)[F], int left) {
#pragma unroll
        for (int i = 0; i < F; i++)
            if (step_of() + i % 4 >= left) x[i] = 0.0f;
    }

    // Cuts and stores four of the thread's floats.  `cut` keeps what piece 0 leaves for piece 1.
    template <int PIECE>
    static __device__ __forceinline__ void store(char* lds, const float (&x)[F], unsigned (&cut)[6], float& largest) {
        unsigned h[2], m[2], l[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float a = x[4 * PIECE + 2 * i], b = x[4 * PIECE + 2 * i + 1];
            largest = fmaxf(fmaxf(fabsf(a), fabsf(b)), largest);
            split_pair(a, b, h[i], m[i], l[i]);
        }
        char* to = lds + (step_of() / 8) * kHalf + row_of(PIECE) * 16;
        if constexpr (KC || F == 4) {
            to += step_of() % 8 * 2;
            *reinterpret_cast<u32x2*>(to) = u32x2{h[0], h[1]};
            *reinterpret_cast<u32x2*>(to + kPlane) = u32x2{m[0], m[1]};
            *reinterpret_cast<u32x2*>(to + 2 * kPlane) = u32x2{l[0], l[1]};
        } else if constexpr (PIECE == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                cut[i] = h[i];
                cut[2 + i] = m[i];
                cut[4 + i] = l[i];
            }
        } else {
            *reinterpret_cast<u32x4v*>(to) = u32x4v{cut[0], cut[1], h[0], h[1]};
            *reinterpret_cast<u32x4v*>(to + kPlane) = u32x4v{cut[2], cut[3], m[0], m[1]};
            *reinterpret_cast<u32x4v*>(to + 2 * kPlane) = u32x4v{cut[4], cut[5], l[0], l[1]};
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

// The plain sum of one output over what this workgroup reduces (whole steps [s0, s1), and the rests behind the whole steps
// where it has them), for sums that an infinity entered.
template <int MODE>
__device__ float plain_sum(const GatedGemm& p, int which, int64_t m, int64_t n, int s0, int s1, bool rests) {
    float sum = 0.0f;
    const int full = p.K / kStep;
    for (int seg = 0; seg < (MODE == kGatedGx ? 2 : 1); seg++) {
        const int from = s0 - seg * full, to = s1 - seg * full;
        const int k0 = (from < 0 ? 0 : from > full ? full : from) * kStep;
        const int k1 = (to < 0 ? 0 : to > full ? full : to) * kStep;
        for (int k = k0; k < p.K; k++) {
            if (k >= k1 && (!rests || k < full * kStep)) continue;
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

template <int ACT>
__device__ __forceinline__ f32x4 activate_as(const f32x4& x, float leaky) {
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = apply_act(x[e], ACT, leaky);
    return y;
}

// one jump for four values
__device__ __forceinline__ f32x4 activate4(const f32x4& x, int act, float leaky) {
    switch (act) {
    case kActRelu: return activate_as<kActRelu>(x, leaky);
    case kActLeaky: return activate_as<kActLeaky>(x, leaky);
    case kActSigmoid: return activate_as<kActSigmoid>(x, leaky);
    case kActTanh: return activate_as<kActTanh>(x, leaky);
    case kActGelu: return activate_as<kActGelu>(x, leaky);
    case kActSelu: return activate_as<kActSelu>(x, leaky);
    case kActMish: return activate_as<kActMish>(x, leaky);
    case kActSwish: return activate_as<kActSwish>(x, leaky);
    default: return x;
    }
}

// bias[n .. n + 3], 0 where there is none
__device__ __forceinline__ f32x4 bias4(const float* bias, int64_t n, int64_t N) {
    f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
    if (bias) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < N) b[e] = bias[n + e];
    }
    return b;
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

// Neighbouring tiles on one XCD (workgroup ids go round the eight).
__device__ __forceinline__ int on_one_xcd(int id, int total) {
    const int each = total / 8, rest = total % 8, xcd = id % 8, at = id / 8;
    return xcd * each + (xcd < rest ? xcd : rest) + at;
}

struct Place {
    int which, tm, tn;
};
// Tiles in runs of `run` tile rows by all columns
__device__ __forceinline__ Place place_of(const GatedGemm& p, int id) {
    const int tiles_mn = p.tiles_m * p.tiles_n, which = id / tiles_mn;
    id -= which * tiles_mn;
    const int run = p.run * p.tiles_n;
    const int first = id / run * p.run;
    const int rows = p.tiles_m - first < p.run ? p.tiles_m - first : p.run;
    const int in = id % run;
    return Place{which, first + in % rows, in / rows};
}

template <int MODE, int WM, int WN, int NBM>
__global__ __launch_bounds__(64 * WM * WN, WM * WN == 8 ? 2 : NBM == 2 ? 3 : 4) void gated_gemm_kernel(GatedGemm p) {
    using S = Shape<MODE, WM, WN, NBM>;
    using TA = typename S::TA;
    using TB = typename S::TB;
    constexpr int NBN = S::NBN;
    extern __shared__ char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int wm = wave / WN, wn = wave % WN;

    // The first p.whole workgroups take a tile each, those behind them a part of the reduction of one of the p.cut others.
    const bool partial = (int)blockIdx.x >= p.whole;
    const int behind = (int)blockIdx.x - p.whole, part = partial ? behind / p.cut : 0, cut = partial ? behind % p.cut : 0;
    const Place place = partial ? place_of(p, p.whole + on_one_xcd(cut, p.cut)) : place_of(p, on_one_xcd((int)blockIdx.x, p.whole));
    const int which = place.which;
    const int64_t m0 = (int64_t)place.tm * S::BM, n0 = (int64_t)place.tn * S::kColumns;
    // Whole steps [s0, s1) of this part of the reduction; the last part takes the rests (K % 16 steps a segment) as well.
    constexpr int kSegments = MODE == kGatedGx ? 2 : 1;
    const int full = p.K / kStep;
    const int s0 = part * p.part_steps;
    const int s1 = partial && s0 + p.part_steps < kSegments * full ? s0 + p.part_steps : kSegments * full;
    const bool rests = (!partial || part + 1 == p.nparts) && p.K % kStep != 0;

    // Buffers that end with the operands.  K-contiguous operands start at the tile's first row, the others at its first
    // column and, with one segment, at the part's first step: offsets inside stay below 4 GiB.
    const int64_t astart = S::AKC ? m0 * p.lda : m0 + (kSegments == 1 ? (int64_t)s0 * kStep * p.lda : 0);
    const int64_t bstart = S::BKC ? n0 * p.ldb : n0 + (kSegments == 1 ? (int64_t)s0 * kStep * p.ldb : 0);
    const int64_t aend = S::AKC ? (p.M - 1) * p.lda + p.K : (p.K - 1) * p.lda + p.M;
    const int64_t bend = S::BKC ? (p.N - 1) * p.ldb + p.K : (p.K - 1) * p.ldb + p.N;
    __amdgpu_buffer_rsrc_t arsrc[kSegments], brsrc[MODE == kGatedForward ? TB::kPieces : 2];
    // byte offsets of this thread's loads of step 0 from there
    uint32_t aoff[TA::kPieces], boff[TB::kPieces];       // (a transposing thread's other loads are rows further on)
#pragma unroll
    for (int g = 0; g < kSegments; g++) {
        const float* A = MODE == kGatedGw ? p.A[which] : p.A[g];
        arsrc[g] = rsrc_from(A + astart, A + aend);
    }
#pragma unroll
    for (int g = 0; g < (MODE == kGatedForward ? TB::kPieces : 2); g++) {
        // forward: rows of the tile alternate between the weights, 32 at a time, so a load's rows are of one of them
        const float* B = MODE == kGatedForward ? p.B[__builtin_amdgcn_readfirstlane(TB::row_of(g) / 32 % 2)] : p.B[g < kSegments ? g : 0];
        brsrc[g] = rsrc_from(B + bstart, B + bend);
    }
    if constexpr (S::AKC) {
#pragma unroll
        for (int i = 0; i < TA::kPieces; i++) aoff[i] = (uint32_t)(TA::row_of(i) * p.lda + TA::step_of()) * 4;
    } else {
        aoff[0] = (uint32_t)(TA::step_of() * p.lda + TA::row_of(0)) * 4;
    }
    if constexpr (S::BKC) {
#pragma unroll
        for (int i = 0; i < TB::kPieces; i++)
            boff[i] = (uint32_t)((TB::row_of(i) % 32 + TB::row_of(i) / 64 * 32) * p.ldb + TB::step_of()) * 4;
    } else {
        boff[0] = (uint32_t)(TB::step_of() * p.ldb + TB::row_of(0)) * 4;
    }
    float xa[2][TA::F], xb[2][TB::F];     // of the next step and of the one after it
    float largest = 0.0f;
    // 16 steps of a segment from step s on
    const auto load_steps = [&](int segment, int s, auto set) {
        constexpr int q = decltype(set)::value;
        const auto ar = segment == 0 ? arsrc[0] : arsrc[kSegments - 1];
        const uint32_t from = (uint32_t)(kSegments == 1 ? s - s0 : s) * kStep * 4;      // of an operand that starts there
        const uint32_t ka = S::AKC ? (uint32_t)s * kStep * 4 : from * (uint32_t)p.lda;
        const uint32_t kb = S::BKC ? (uint32_t)s * kStep * 4 : from * (uint32_t)p.ldb;
        if constexpr (S::AKC) {
#pragma unroll
            for (int i = 0; i < TA::kPieces; i++) TA::load_kc(xa[q], i, ar, aoff[i] + ka);
        } else {
#pragma unroll
            for (int i = 0; i < TA::F; i++)
                xa[q][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(ar, aoff[0] + (ka + (uint32_t)i * (uint32_t)p.lda * 4), 0, 0));
        }
        if constexpr (S::BKC) {
#pragma unroll
            for (int i = 0; i < TB::kPieces; i++) TB::load_kc(xb[q], i, brsrc[i], boff[i] + kb);
        } else {
            const auto br = segment == 0 ? brsrc[0] : brsrc[kSegments - 1];
#pragma unroll
            for (int i = 0; i < TB::F; i++)
                xb[q][i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(br, boff[0] + (kb + (uint32_t)i * (uint32_t)p.ldb * 4), 0, 0));
        }
    };
    // whole step s of the reduction
    const auto load = [&](int s, auto set) {
        const int segment = kSegments == 2 && s >= full ? 1 : 0;
        load_steps(segment, s - segment * full, set);
    };
    unsigned cut_a[6], cut_b[6];
    // part PIECE of the step's cutting and storing
    constexpr int kPieces = TA::kPieces + TB::kPieces;
    const auto store = [&](auto set, auto piece) {
        constexpr int q = decltype(set)::value, PIECE = decltype(piece)::value;
        char* to = lds + q * (TA::kBytes + TB::kBytes);
        if constexpr (PIECE < TA::kPieces) TA::template store<PIECE>(to, xa[q], cut_a, largest);
        else TB::template store<PIECE - TA::kPieces>(to + TA::kBytes, xb[q], cut_b, largest);
    };

    f32x16 acc[NBM][NBN];
#pragma unroll
    for (int i = 0; i < NBM; i++)
#pragma unroll
        for (int j = 0; j < NBN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;

    const int pairs_end = s1 > s0 ? s0 + (s1 - s0) / 2 * 2 : s0;     // steps go in pairs, the last odd one by itself
    // the products of a buffer's step; between(i) runs behind those of the wave's i-th 32 rows
    const auto products = [&](const char* from, auto between) {
        Split8 b[NBN];
#pragma unroll
        for (int j = 0; j < NBN; j++) b[j] = TB::fragment(from + TA::kBytes, wn * 32 * NBN + 32 * j);
        Split8 next = TA::fragment(from, wm * 32 * NBM);
        static_for<0, NBM>([&](auto block) {
            constexpr int i = decltype(block)::value;
            const Split8 a = next;
            if constexpr (i + 1 < NBM) next = TA::fragment(from, wm * 32 * NBM + 32 * (i + 1));
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
            between(block);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // A step: the loads of two steps further on (in front, or the scheduler sinks them to their use), the products of this
    // one, and between them the cutting of the next.  What is loaded and cut behind the last step is its data once more, and
    // not used.
    const auto step = [&](int s, auto set) {
        constexpr int q = decltype(set)::value;
        load(s + 2 < pairs_end ? s + 2 : pairs_end - 1, set);
        __builtin_amdgcn_sched_barrier(0);
        products(lds + q * (TA::kBytes + TB::kBytes), [&](auto block) {
            constexpr int i = decltype(block)::value;
            static_for<kPieces * i / NBM, kPieces * (i + 1) / NBM>([&](auto piece) { store(std::integral_constant<int, 1 - q>{}, piece); });
        });
        __syncthreads();
    };
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    if (s0 < pairs_end) {
        load(s0, Zero{});
        load(s0 + 1, One{});
        static_for<0, kPieces>([&](auto piece) { store(Zero{}, piece); });
        __syncthreads();
        for (int s = s0; s < pairs_end; s += 2) {
            step(s, Zero{});
            step(s + 1, One{});
        }
    }
    // the odd step, and the rests of the segments
    const int odd = s1 > pairs_end ? 1 : 0, tail = odd + (rests ? kSegments : 0);
#pragma unroll 1
    for (int i = 0; i < tail; i++) {
        const int segment = i < odd ? (kSegments == 2 && pairs_end >= full ? 1 : 0) : i - odd;
        load_steps(segment, i < odd ? pairs_end - segment * full : full, Zero{});
        const int left = i < odd ? kStep : p.K % kStep;
        if constexpr (S::AKC) TA::mask_kc(xa[0], left);
        if constexpr (S::BKC) TB::mask_kc(xb[0], left);
        static_for<0, kPieces>([&](auto piece) { store(Zero{}, piece); });
        __syncthreads();
        products(lds, [](auto) {});
        __syncthreads();
    }

    // Epilogue by way of LDS, a wave's own 32 rows at a time: the accumulators hold one column a lane, the stores want four
    // columns of a row, and the activation's code stands there once instead of once for every register.
    const bool again = __syncthreads_or(!(largest <= kLargestFinite));
    const float leaky = MODE == kGatedForward && p.hleaky ? *p.hleaky : 0.0f;
    float* stage = reinterpret_cast<float*>(lds) + wave * S::kStageFloats;
    const int64_t n = n0 + wn * (MODE == kGatedForward ? 32 : 64) + lane % 8 * 4;      // this lane's columns,
    const int64_t n2 = MODE == kGatedForward ? n : n + 32;                           // and the other block's
    f32x4 bg, bu;
    if (MODE == kGatedForward && !partial) {
        bg = bias4(p.bias[0], n, p.N);
        bu = bias4(p.bias[1], n, p.N);
    }
#pragma unroll
    for (int i = 0; i < NBM; i++) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NBN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                stage[(8 * (e / 4) + 4 * (lane >> 5) + e % 4) * kStageRow + 32 * j + (lane & 31)] = acc[i][j][e];
        __builtin_amdgcn_wave_barrier();
        if (again) {
#pragma unroll 1
            for (int e = lane; e < 32 * 64; e += 64) {
                const int r = e / 64, c = e % 64;
                float* x = stage + r * kStageRow + c;
                const int64_t m = m0 + wm * 32 * NBM + 32 * i + r;
                const int64_t col = MODE == kGatedForward ? n0 + wn * 32 + c % 32 : n0 + wn * 64 + c;
                if (*x != *x && m < p.M && col < p.N) *x = plain_sum<MODE>(p, MODE == kGatedForward ? c / 32 : which, m, col, s0, s1, rests);
            }
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll 1
        for (int r = lane / 8; r < 32; r += 8) {
            const int64_t m = m0 + wm * 32 * NBM + 32 * i + r;
            if (m >= p.M) break;
            const float* row = stage + r * kStageRow + lane % 8 * 4;
            f32x4 v = *reinterpret_cast<const f32x4*>(row), u = *reinterpret_cast<const f32x4*>(row + 32);
            const int64_t at = m * p.ldc;
            if (partial) {
                // the tile as it stands, a wave's two blocks of 32 columns side by side
                f32x4* sums = reinterpret_cast<f32x4*>(p.parts) +
                              (((int64_t)part * p.cut + cut) * S::BM + (m - m0)) * (S::BN / 4) + wn * 16 + lane % 8;
                sums[0] = v;
                sums[8] = u;
            } else if constexpr (MODE == kGatedForward) {
                v += bg;
                u += bu;
                const f32x4 y = activate4(v, p.act, leaky) * u;
                if (p.C[1]) {
                    put(p.C[1] + at, n, p.N, v, p.wide);
                    put(p.C[2] + at, n, p.N, u, p.wide);
                }
                put(p.C[0] + at, n, p.N, y, p.wide);
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

// Sums the parts of the tiles that were cut, with the forward's epilogue or onto the gradient: a thread takes four columns of a
// row and, for the forward, the same four of gate and of up.
template <int MODE, int BM, int BN>
__global__ __launch_bounds__(256) void gated_parts_kernel(GatedGemm p) {
    constexpr int kLines = (MODE == kGatedForward ? BN / 2 : BN) / 4;      // of an output row that a tile covers
    constexpr int kGroups = BM * kLines / 256;                             // workgroups of a tile
    const int64_t all = (int64_t)p.cut * BM * (BN / 4);
    const float leaky = MODE == kGatedForward && p.hleaky ? *p.hleaky : 0.0f;
    const f32x4* parts = reinterpret_cast<const f32x4*>(p.parts);
    const int cut = (int)blockIdx.x / kGroups, e = (int)blockIdx.x % kGroups * 256 + (int)threadIdx.x;
    const int line = e % kLines, row = e / kLines;
    const Place place = place_of(p, p.whole + on_one_xcd(cut, p.cut));
    const int64_t m = (int64_t)place.tm * BM + row, n = ((int64_t)place.tn * kLines + line) * 4;
    if (m >= p.M || n >= p.N) return;
    const f32x4* from = parts + ((int64_t)cut * BM + row) * (BN / 4) + (MODE == kGatedForward ? line / 8 * 16 + line % 8 : line);
    f32x4 v = from[0], u = MODE == kGatedForward ? from[8] : v;
#pragma unroll 4
    for (int s = 1; s < p.nparts; s++) {
        v += from[s * all];
        if (MODE == kGatedForward) u += from[s * all + 8];
    }
    const int64_t at = m * p.ldc;
    if constexpr (MODE == kGatedForward) {
        v += bias4(p.bias[0], n, p.N);
        u += bias4(p.bias[1], n, p.N);
        const f32x4 y = activate4(v, p.act, leaky) * u;
        if (p.C[1]) {
            put(p.C[1] + at, n, p.N, v, p.wide);
            put(p.C[2] + at, n, p.N, u, p.wide);
        }
        put(p.C[0] + at, n, p.N, y, p.wide);
    } else {
        float* c = p.C[place.which] + at;
        if (p.acc) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (n + i < p.N) v[i] += c[n + i];
        }
        put(c, n, p.N, v, p.wide);
    }
}

// Where the reduction is cut, whole rounds of workgroups over the chip still take whole tiles: only the rest is cut, so that few
// sums pass through memory (4096 x 4096 -> 11008, 1376 tiles: all in two parts 3.49 ms, 1280 whole and 96 in eight 3.19; in two,
// what 64 MiB of scratch hold, the same: 3.45, 3.47 | 3.46, 3.47 side by side on a slower card).
int whole_tiles(int64_t tiles) { return (int)(tiles / compute_units() * compute_units()); }

// Tiles of rows x columns of the output, and how their reduction is cut.
template <int MODE>
void place_tiles(GatedGemm& p, int rows, int columns, int64_t nparts) {
    p.tiles_m = (int)((p.M + rows - 1) / rows);
    p.tiles_n = (int)((p.N + columns - 1) / columns);
    p.run = 8;
    const int steps = p.K / kStep * (MODE == kGatedGx ? 2 : 1);
    p.part_steps = (int)((steps + nparts - 1) / nparts + 1) / 2 * 2;
    p.nparts = p.part_steps > 0 ? (steps + p.part_steps - 1) / p.part_steps : 1;
    const int tiles = p.tiles_m * p.tiles_n * p.nwhich;
    p.whole = p.nparts > 1 ? whole_tiles(tiles) : tiles;
    p.cut = tiles - p.whole;
}

int64_t parts_bytes(int64_t nparts, int64_t cut, int64_t rows, int64_t columns) {
    return nparts * cut * rows * columns * (int64_t)sizeof(float);
}

template <int MODE, int WM, int WN, int NBM>
int launch_shape(GatedGemm p, int64_t nparts, hipStream_t stream) {
    using S = Shape<MODE, WM, WN, NBM>;
    place_tiles<MODE>(p, S::BM, S::kColumns, nparts);
    if (S::kLds > 64 * 1024)
        KAI_TRY(check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_gemm_kernel<MODE, WM, WN, NBM>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds),
                          "hipFuncSetAttribute(gated_gemm_kernel)"));
    if (p.cut > 0) KAI_TRY(workspace(parts_bytes(p.nparts, p.cut, S::BM, S::BN), &p.parts));
    p.wide = p.ldc % 4 == 0 && aligned16(p.C[0]) && aligned16(p.C[1]) && aligned16(p.C[2]);
    gated_gemm_kernel<MODE, WM, WN, NBM><<<(unsigned)(p.whole + p.cut * p.nparts), S::NT, S::kLds, stream>>>(p);
    KAI_TRY(check_launch("gated_gemm_kernel"));
    if (p.cut == 0) return KAI_OK;
    gated_parts_kernel<MODE, S::BM, S::BN><<<(unsigned)(p.cut * (S::BM * S::kColumns / 1024)), 256, 0, stream>>>(p);
    return check_launch("gated_parts_kernel");
}

// The tile and the parts of the reduction that this estimate (us) finds cheapest.  A workgroup's step of 16 takes 0.42
// (64 x 128 tiles), 0.70 (128 x 128), 1.25 (256 x 128) or 2.35 (256 x 256), the workgroups of a compute unit one after another (the
// small tiles' run side by side, but share the matrix cores); its start and epilogue `fixed`; parts a launch of 4 and their
// sums written and read at 10 bytes a ns.  Fitted to 35 shapes, 33 to 2048 rows by 64 to 4096 by 333 to 4096, against 1, 2, 3, 4, 6, 8, 12
// and 16 parts of each tile: within a tenth of the fastest for all but a few.  The sides, in us: 1000 x 777 -> 333 20.3 with two parts of
// 64 x 128, 22.0 with four of 128 x 128; 1000 x 1024 -> 4096 90 with 256 x 128, 94 with 128 x 128; 2048 x 1024 -> 4096 161 with 256 x 256, 177 with
// 256 x 128; 256 x 4096 -> 4096 96 with four parts of 256 x 128, 121 with 64 x 128 whole; the weights' gradients of 2048 x 1024 -> 4096
// 200 with 256 x 128, 209 with two parts of 256 x 256, 210 with 128 x 128.
struct Plan {
    int tile = 0;      // 0: 64 x 128, 1: 128 x 128, 2: 256 x 128, 3: 256 x 256
    int parts = 1;
    double us = 1e30;
};

constexpr int kTileRows[4] = {64, 128, 256, 256}, kTileColumns[4] = {128, 128, 128, 256};

template <int MODE>
Plan plan_of(const GatedGemm& p) {
    const int(&rows)[4] = kTileRows, (&columns)[4] = kTileColumns;
    constexpr double step[4] = {0.42, 0.70, 1.25, 2.35};
    constexpr double fixed_forward[4] = {7.7, 12.0, 15.0, 19.0}, fixed_gradient[4] = {5.2, 6.5, 8.0, 14.0};
    const int64_t all_columns = MODE == kGatedForward ? 2 * p.N : p.N, cu = compute_units();
    const int64_t steps = (p.K + kStep - 1) / kStep * (MODE == kGatedGx ? 2 : 1);
    Plan best;
    for (int t = 0; t < 4; t++) {
        const int64_t tiles = (p.M + rows[t] - 1) / rows[t] * ((all_columns + columns[t] - 1) / columns[t]) * p.nwhich;
        for (const int parts : {1, 2, 3, 4, 6, 8, 12, 16}) {
            if (parts > 1 && steps < 4 * parts) break;
            const int64_t each = ((steps + parts - 1) / parts + 1) / 2 * 2;
            const int64_t whole = parts > 1 ? whole_tiles(tiles) : tiles, cut = tiles - whole;
            if (parts > 1 && parts_bytes(parts, cut, rows[t], columns[t]) > kProductScratchMax) break;
            const int64_t rounds = (whole + cu - 1) / cu, cut_rounds = (cut * parts + cu - 1) / cu;
            double us = (MODE == kGatedForward ? fixed_forward : fixed_gradient)[t] + (double)(rounds * steps + cut_rounds * each) * step[t];
            if (cut > 0) us += 4.0 + (double)(parts * cut * rows[t] * columns[t]) * 8.0 / 1e7;
            if (us < best.us) best = Plan{t, parts, us};
        }
    }
    return best;
}

template <int MODE>
GatedGemmPlan full_plan(GatedGemm p) {
    const Plan plan = plan_of<MODE>(p);
    const int rows = kTileRows[plan.tile], columns = kTileColumns[plan.tile];
    place_tiles<MODE>(p, rows, MODE == kGatedForward ? columns / 2 : columns, plan.parts);
    const int parts = p.cut > 0 ? p.nparts : 1;
    return GatedGemmPlan{rows, columns, p.whole, p.cut, parts, p.cut > 0 ? parts_bytes(parts, p.cut, rows, columns) : 0};
}

template <int MODE>
int launch_mode(const GatedGemm& p, hipStream_t stream) {
    const Plan plan = plan_of<MODE>(p);
    if (plan.tile == 0) return launch_shape<MODE, 2, 2, 1>(p, plan.parts, stream);
    if (plan.tile == 1) return launch_shape<MODE, 2, 2, 2>(p, plan.parts, stream);
    if (plan.tile == 2) return launch_shape<MODE, 4, 2, 2>(p, plan.parts, stream);
    return launch_shape<MODE, 2, 4, 4>(p, plan.parts, stream);
}

}  // namespace

// Offsets inside a workgroup's operands are 32-bit (256 rows of a K-contiguous operand, all steps of another), and so are the
// threads of a launch.
bool gated_gemm_applies(int mode, const GatedGemm& p) {
    if (p.M <= 0 || p.N <= 0 || p.K <= 0 || p.lda >= (1ll << 21) || p.ldb >= (1ll << 21)) return false;
    if ((p.M / 64 + 1) * (p.N / 64 + 1) >= (1ll << 22)) return false;
    const int64_t rows = (int64_t)p.K + kStep;
    if (mode != kGatedForward && rows * p.ldb >= (1ll << 30)) return false;
    return mode != kGatedGw || rows * p.lda < (1ll << 30);
}

double gated_gemm_us(int mode, const GatedGemm& p) {
    return mode == kGatedForward ? plan_of<kGatedForward>(p).us : mode == kGatedGx ? plan_of<kGatedGx>(p).us : plan_of<kGatedGw>(p).us;
}

GatedGemmPlan gated_gemm_plan(int mode, const GatedGemm& p) {
    if (mode == kGatedForward) return full_plan<kGatedForward>(p);
    return mode == kGatedGx ? full_plan<kGatedGx>(p) : full_plan<kGatedGw>(p);
}

int launch_gated_gemm(int mode, const GatedGemm& p, hipStream_t stream) {
    if (mode == kGatedForward) return launch_mode<kGatedForward>(p, stream);
    if (mode == kGatedGx) return launch_mode<kGatedGx>(p, stream);
    return launch_mode<kGatedGw>(p, stream);
}

}  // namespace kai
