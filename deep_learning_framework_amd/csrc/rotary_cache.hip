// Rotary positions and the writes of the key/value cache.  Bound: HBM (every element read once and written once).
//
// theta(p, i) = p * f_i,  f_i = base^(-2i/nrot), scaled;  (y1, y2) = m * (x1 cos - x2 sin, x2 cos + x1 sin) for the
// two elements of pair i.  The gradient is the same turn by -theta.  The angle's turn p * f_i / 2 pi is formed and
// reduced to [-1/2, 1/2] in 64 bits (at position 10^6 a 32-bit product is off by 0.06 rad), the sine and cosine of
// what is left in 32.  They are the same for every head of a token: a workgroup forms them once for its tokens in
// LDS, so their cost (a 64-bit product and ~40 instructions a pair) is shared by nhead heads.
//
// Measured: 2 x 384 tokens of 12 heads of 64 5.0 us (a launch; 3.7 of them the kernel's), 4 x 4096 of 32 heads of 128 109.7 us = 4.89
// TB/s, the rate of a plain copy; appending 64 tokens of 8 heads of 128 5.2 us, 4 x up to 2000 17.6 us = 5.3 TB/s.
#include "decoder_ops.h"

namespace kai {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;   // tokens of a workgroup at a time

// radians per position / 2 pi of pair i
__device__ double turn_of_pair(const RotaryParams& r, int i) {
    double f = exp2(r.step * i) * 0.15915494309189533577;   // 1 / (2 pi)
    if (r.parts) {
        // turns that the pair makes over the trained length: few turns are stretched, many are kept
        const double turns = r.trained_turns * exp2(r.step * i);
        double keep = (turns - r.low) * r.inv_span;
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        return f * (keep + (1.0 - keep) * r.inv_factor);
    }
    return f * r.inv_factor;
}

// cos and sin of position p's turn of one pair, times the magnitude; `back` turns the other way
__device__ float2 turn(double per_position, int p, float magnitude, bool back) {
    const double t = per_position * (double)p;
    const float r = (float)(t - rint(t));
    float s, c;
    sincospif(2.0f * r, &s, &c);
    s *= magnitude;
    return make_float2(c * magnitude, back ? -s : s);
}

// LDS of a workgroup: frequencies (64 bit) of the half = nrot/2 pairs, then (cos, sin) of `tokens` x half
extern __shared__ double rotary_lds[];

struct TokenTurns {
    double* freq;
    float2* cs;
    int half;
    __device__ TokenTurns(const RotaryParams& r) : freq(rotary_lds), cs(reinterpret_cast<float2*>(rotary_lds + r.nrot / 2)), half(r.nrot / 2) {}
    __device__ void frequencies(const RotaryParams& r) {
        for (int i = threadIdx.x; i < half; i += kThreads) freq[i] = turn_of_pair(r, i);
    }
};

// One head's rotated elements, VEC at a time: units u of a head are halves: elements [VEC*u, +VEC) of both halves,
// pairs: elements [2*VEC*u, +2*VEC).
// Every element is written once and not read here again: the stores do not stay in the L2 (4 x 4096 x 32 heads of 128 117.7 ->
// 113.8 us, appending 4 x 2000 rows 22.1 -> 17.7).  STREAM: nor do the loads, for tensors that the 256 MB behind the L2 does
// not hold anyway (the same 113.8 -> 109.7; appending 4 x 2000 rows, whose 65 MB it holds, 17.7 -> 23.0).
template <int VEC, bool STREAM>
__device__ void turn_unit(float* y, const float* x, const float2* cs, int u, int half, bool pairs) {
    typedef float vec __attribute__((ext_vector_type(VEC)));
    const int i0 = u * VEC;
    float a[VEC], b[VEC];
    const int first = pairs ? 2 * i0 : i0, second = pairs ? 2 * i0 + VEC : half + i0;
    vec v1, v2;
    if constexpr (VEC == 1) {
        v1[0] = x[first];
        v2[0] = x[second];
    } else {
        const vec* from1 = reinterpret_cast<const vec*>(x + first);
        const vec* from2 = reinterpret_cast<const vec*>(x + second);
        v1 = STREAM ? __builtin_nontemporal_load(from1) : *from1;
        v2 = STREAM ? __builtin_nontemporal_load(from2) : *from2;
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        if (pairs) {
            a[e] = 2 * e < VEC ? v1[(2 * e) % VEC] : v2[(2 * e) % VEC];
            b[e] = 2 * e + 1 < VEC ? v1[(2 * e + 1) % VEC] : v2[(2 * e + 1) % VEC];
        } else {
            a[e] = v1[e];
            b[e] = v2[e];
        }
    }
    float ya[VEC], yb[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const float2 t = cs[i0 + e];
        // which product the sum keeps unrounded is written out: the same bits whatever the vectors' width
        ya[e] = fmaf(a[e], t.x, -(b[e] * t.y));
        yb[e] = fmaf(b[e], t.x, a[e] * t.y);
    }
    vec w1, w2;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        if (pairs) {
            if (2 * e < VEC) w1[(2 * e) % VEC] = ya[e]; else w2[(2 * e) % VEC] = ya[e];
            if (2 * e + 1 < VEC) w1[(2 * e + 1) % VEC] = yb[e]; else w2[(2 * e + 1) % VEC] = yb[e];
        } else {
            w1[e] = ya[e];
            w2[e] = yb[e];
        }
    }
    if constexpr (VEC == 1) {
        y[first] = w1[0];
        y[second] = w2[0];
    } else {
        __builtin_nontemporal_store(w1, reinterpret_cast<vec*>(y + first));
        __builtin_nontemporal_store(w2, reinterpret_cast<vec*>(y + second));
    }
}

template <int VEC, bool STREAM>
__device__ void copy_unit(float* y, const float* x, int u) {
    if constexpr (VEC == 1) y[u] = x[u];
    else {
        const f32x4* from = reinterpret_cast<const f32x4*>(x + VEC * u);
        __builtin_nontemporal_store(STREAM ? __builtin_nontemporal_load(from) : *from, reinterpret_cast<f32x4*>(y + VEC * u));
    }
}

template <int VEC, bool STREAM>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int tokens) {
    TokenTurns turns(a.rot);
    const int half = turns.half;
    turns.frequencies(a.rot);
    const int turn_units = half / VEC;                                     // of one head
    const int rest_units = a.y == a.x ? 0 : (a.npiece - a.rot.nrot) / VEC; // copied elements behind the rotated ones
    const int head_units = turn_units + rest_units;
    const int token_units = head_units * a.nhead;
    for (int64_t t0 = (int64_t)blockIdx.x * tokens; t0 < a.ntok; t0 += (int64_t)gridDim.x * tokens) {
        const int nt = (int)(a.ntok - t0 < tokens ? a.ntok - t0 : tokens);
        __syncthreads();
        for (int e = threadIdx.x; e < nt * half; e += kThreads) {
            const int t = e / half, i = e - t * half;
            const int p = a.pos ? a.pos[t0 + t] : (int)((t0 + t) % a.ntimes);
            turns.cs[e] = turn(turns.freq[i], p, a.rot.magnitude, a.back);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < nt * token_units; e += kThreads) {
            const int t = e / token_units, w = e - t * token_units;
            const int h = w / head_units, u = w - h * head_units;
            const int64_t at = (t0 + t) * a.ld + (int64_t)h * a.npiece;
            if (u < turn_units) turn_unit<VEC, STREAM>(a.y + at, a.x + at, turns.cs + t * half, u, half, a.rot.pairs != 0);
            else copy_unit<VEC, STREAM>(a.y + at + a.rot.nrot, a.x + at + a.rot.nrot, u - turn_units);
        }
    }
}

// where new token t of sequence b goes: its row in the cache, or -1
__device__ int64_t cache_row(const CachePages& c, int b, int t) {
    const int count = c.count ? c.count[b] : (int)c.ntimes;
    if (t >= count) return -1;
    const int64_t len = c.len[b];
    const int64_t at = (len < 0 ? 0 : len) + t;
    if (at >= c.page * c.nmaxpage) return -1;
    const int64_t k = at / c.page;
    const int64_t page = c.table ? c.table[b * c.nmaxpage + k] : b;
    if (page < 0 || page >= c.npage) return -1;
    return page * c.page + (at - k * c.page);
}

template <int VEC>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheAppendArgs a, int tokens) {
    __shared__ int64_t row[kMaxTokens];
    TokenTurns turns(a.rot);
    const int half = turns.half;
    turns.frequencies(a.rot);
    const int nkv = a.pages.nkvhead, npiece = a.pages.npiece;
    const int turn_units = half / VEC, rest_units = (npiece - a.rot.nrot) / VEC;
    const int head_units = turn_units + rest_units;
    const int key_units = head_units * nkv, value_units = nkv * npiece / VEC;
    const int token_units = key_units + value_units;
    const int64_t ntok = a.pages.nbat * a.pages.ntimes, width = (int64_t)nkv * npiece;
    for (int64_t t0 = (int64_t)blockIdx.x * tokens; t0 < ntok; t0 += (int64_t)gridDim.x * tokens) {
        const int nt = (int)(ntok - t0 < tokens ? ntok - t0 : tokens);
        __syncthreads();
        if ((int)threadIdx.x < nt) {
            const int64_t tok = t0 + threadIdx.x;
            row[threadIdx.x] = cache_row(a.pages, (int)(tok / a.pages.ntimes), (int)(tok % a.pages.ntimes));
        }
        for (int e = threadIdx.x; e < nt * half; e += kThreads) {
            const int t = e / half, i = e - t * half;
            const int64_t tok = t0 + t;
            const int64_t b = tok / a.pages.ntimes;
            int p;
            if (a.pos) {
                p = a.pos[tok];
            } else {
                const int64_t len = a.pages.len[b];
                p = (int)((len < 0 ? 0 : len) + (tok - b * a.pages.ntimes));
            }
            turns.cs[e] = turn(turns.freq[i], p, a.rot.magnitude, false);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < nt * token_units; e += kThreads) {
            const int t = e / token_units, w = e - t * token_units;
            if (row[t] < 0) continue;
            const int64_t in = (t0 + t) * a.ld, out = row[t] * width;
            if (w >= key_units) {
                copy_unit<VEC, false>(a.cv + out, a.v + in, w - key_units);
                continue;
            }
            const int h = w / head_units, u = w - h * head_units;
            const int64_t x = in + (int64_t)h * npiece, y = out + (int64_t)h * npiece;
            if (u < turn_units) turn_unit<VEC, false>(a.ck + y, a.k + x, turns.cs + t * half, u, half, a.rot.pairs != 0);
            else copy_unit<VEC, false>(a.ck + y + a.rot.nrot, a.k + x + a.rot.nrot, u - turn_units);
        }
    }
}

// 128-bit accesses: rows, heads and both halves start on 16-byte lines
bool whole_lines(const RotaryParams& r, int64_t ld, int npiece) {
    return ld % 4 == 0 && npiece % 4 == 0 && r.nrot % 8 == 0;
}

// Tokens of a workgroup: as many as leave every compute unit four workgroups, at most kMaxTokens.
int tokens_of_workgroup(int64_t ntok) {
    const int64_t t = ntok / (4 * (int64_t)compute_units());
    return (int)(t < 1 ? 1 : t > kMaxTokens ? kMaxTokens : t);
}

size_t lds_bytes(const RotaryParams& r, int tokens) {
    const size_t half = (size_t)r.nrot / 2;
    return half * sizeof(double) + (size_t)tokens * half * sizeof(float2);
}

int64_t grid_of(int64_t ntok, int tokens) {
    const int64_t groups = (ntok + tokens - 1) / tokens, most = 16 * (int64_t)compute_units();
    return groups < most ? groups : most;
}

}  // namespace

int launch_rotary(const RotaryArgs& a, hipStream_t stream) {
    const int tokens = tokens_of_workgroup(a.ntok);
    const bool wide = whole_lines(a.rot, a.ld, a.npiece) && aligned16(a.x) && aligned16(a.y);
    const dim3 grid((unsigned)grid_of(a.ntok, tokens));
    const bool large = a.ntok * a.nhead * a.npiece * (int64_t)sizeof(float) >= 128ll << 20;
    if (wide && large) rotary_kernel<4, true><<<grid, kThreads, lds_bytes(a.rot, tokens), stream>>>(a, tokens);
    else if (wide) rotary_kernel<4, false><<<grid, kThreads, lds_bytes(a.rot, tokens), stream>>>(a, tokens);
    else rotary_kernel<1, false><<<grid, kThreads, lds_bytes(a.rot, tokens), stream>>>(a, tokens);
    return check_launch("rotary_kernel");
}

int launch_cache_append(const CacheAppendArgs& a, hipStream_t stream) {
    const int64_t ntok = a.pages.nbat * a.pages.ntimes;
    const int tokens = tokens_of_workgroup(ntok);
    const bool wide = whole_lines(a.rot, a.ld, a.pages.npiece) && aligned16(a.k) && aligned16(a.v) && aligned16(a.ck) &&
                      aligned16(a.cv);
    const dim3 grid((unsigned)grid_of(ntok, tokens));
    if (wide) cache_append_kernel<4><<<grid, kThreads, lds_bytes(a.rot, tokens), stream>>>(a, tokens);
    else cache_append_kernel<1><<<grid, kThreads, lds_bytes(a.rot, tokens), stream>>>(a, tokens);
    return check_launch("cache_append_kernel");
}

}  // namespace kai
