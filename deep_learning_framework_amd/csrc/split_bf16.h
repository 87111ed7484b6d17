// fp32 products on the bf16 matrix cores without losing fp32's accuracy.
//
// A float is the exact sum of three bf16: x = h + m + l with h = bf16(x), m = bf16(x - h), l = x - h - m, rounded to
// nearest, so that |m| <= 2^-8 |x|, |l| <= 2^-16 |x| and 8 + 8 + 8 bits hold all 24.  Of the nine products of two such
// sums six are formed: hh, hm, mh, mm, hl, lh.  The three left out are below 3 * 2^-24 |x y| at most and 2^-26 |x y| in
// the mean, what one rounding of the product costs; the products themselves are exact in the 32-bit accumulators.
// v_mfma_f32_32x32x16_bf16 does 16 times the work of v_mfma_f32_32x32x2_f32 in a cycle, so six of them are 2.67 times
// as fast as fp32 matrix instructions, for about 5.5 vector instructions per loaded float (3 conversions, 4 widenings,
// 4 subtractions for two).  An infinity (or a value that rounds to one in bf16, above 3.39e38) becomes a NaN: callers
// look for those.  Pieces below 2^-133 vanish, so values below 2^-109 keep fewer than 24 bits.
#pragma once

#include <hip/hip_runtime.h>

namespace kai {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4v __attribute__((ext_vector_type(4)));

struct Split8 {
    bf16x8 h, m, l;
};

__device__ __forceinline__ unsigned to_bf16_pair(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}

__device__ __forceinline__ void split_pair(float a, float b, unsigned& h, unsigned& m, unsigned& l) {
    h = to_bf16_pair(a, b);
    a -= __builtin_bit_cast(float, h << 16);
    b -= __builtin_bit_cast(float, h & 0xFFFF0000u);
    m = to_bf16_pair(a, b);
    a -= __builtin_bit_cast(float, m << 16);
    b -= __builtin_bit_cast(float, m & 0xFFFF0000u);
    l = to_bf16_pair(a, b);
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
