// fp32 products on the bf16 matrix cores at about fp32's accuracy.
//
// A float is the exact sum of three bf16: h = its upper 16 bits, m = the upper 16 bits of x - h, l = x - h - m: 8 + 8 + 8
// bits of the 24, |m| < 2^-7 |x|, |l| < 2^-15 |x|.  Of the nine products of two such sums six are formed: hh, hm, mh, mm,
// hl, lh.  The three left out, m l, l m and l l, have the product's own sign: a result loses up to 2^-21 of sum |x y|, always
// towards zero.  That is 4e-8 of it on normal or uniform data (0.7 of 2^-24, the most that rounding a product once costs, there
// with either sign), 8e-8 where x and y are spread over [1, 1 + 2^-7), 2.5e-7 .. 4.7e-7 where nearly all of their lower bits
// are set.  The sums' own rounding is above that from some tens of terms on.  The products formed are exact in the 32-bit
// accumulators.
// (Pieces rounded to nearest instead would leave out 2^-26, but v_cvt_pk_bf16_f32 issues in 8 cycles where the 32-bit
// operations here take 4 to 5: 4096 x 4096 -> 11008 3.81 ms with them, 3.67 without.)
// v_mfma_f32_32x32x16_bf16 does 16 times the work of v_mfma_f32_32x32x2_f32 in a cycle, so six of them are 2.67 times
// as fast as fp32 matrix instructions, for 5.5 vector instructions per loaded float (4 masks, 4 subtractions, 3 packings
// for two).  An infinity becomes a NaN (inf - inf): callers look for those.  Pieces below 2^-133 vanish, so values below
// 2^-109 keep fewer than 24 bits.
#pragma once

#include <hip/hip_runtime.h>

namespace kai {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4v __attribute__((ext_vector_type(4)));

constexpr float kLargestFinite = 3.40282347e38f;

struct Split8 {
    bf16x8 h, m, l;
};

__device__ __forceinline__ float upper_half(float x) {
    return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xFFFF0000u);
}
// upper halves of a (low half of the result) and b
__device__ __forceinline__ unsigned upper_halves(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
}

__device__ __forceinline__ void split_pair(float a, float b, unsigned& h, unsigned& m, unsigned& l) {
    h = upper_halves(a, b);
    a -= upper_half(a);
    b -= upper_half(b);
    m = upper_halves(a, b);
    a -= upper_half(a);
    b -= upper_half(b);
    l = upper_halves(a, b);
}

// eight floats x[0], x[stride], ...
template <typename At>
__device__ __forceinline__ Split8 split8(At&& at) {
    u32x4v h, m, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned a, b, c;
        split_pair(at(2 * i), at(2 * i + 1), a, b, c);
        h[i] = a;
        m[i] = b;
        l[i] = c;
    }
    return Split8{__builtin_bit_cast(bf16x8, h), __builtin_bit_cast(bf16x8, m), __builtin_bit_cast(bf16x8, l)};
}

}  // namespace kai
