// Attention of new tokens over a paged cache of keys and values.
//
//   y[b, t, h, :] = sum_j p_j v_j,   p = softmax over the keys j that row (b, t) sees of coef * <q, k_j>
//
// with online statistics: a running maximum m, the sum l of exp(s_j - m) and the sum of exp(s_j - m) v_j, all in
// 32 bits; a row that sees nothing gives zeros.  Few rows meet many keys, so the keys of a sequence are cut into
// parts that run as separate workgroups; cache_attention_join_kernel adds the parts,
//   y = sum_s e^(m_s - M) acc_s / sum_s e^(m_s - M) l_s.
#include "decoder_ops.h"
#include "split_bf16.h"

namespace kai {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr int kMaxPiece = 256;
constexpr int kKeyStep = 32;     // a part of a sequence's keys is a whole number of these

struct Parts {
    float* acc;      // [nsplit][rows][npiece], not yet divided
    float2* ml;      // [nsplit][rows]: maximum, sum
    int nsplit;
};

struct Sequence {
    int len, count, keys;    // old keys, new ones, both
};

__device__ Sequence sequence_of(const CachePages& c, int b) {
    const int64_t reach = c.page * c.nmaxpage;
    int64_t len = c.len[b];
    len = len < 0 ? 0 : len > reach ? reach : len;
    int64_t count = c.count ? c.count[b] : c.ntimes;
    count = count < 0 ? 0 : count > c.ntimes ? c.ntimes : count;
    const int64_t keys = len + count > reach ? reach : len + count;
    return Sequence{(int)len, (int)count, (int)keys};
}

// part s of a sequence's keys
__device__ void part_of(int keys, int nsplit, int s, int* begin, int* end) {
    const int steps = (keys + kKeyStep - 1) / kKeyStep;
    const int each = (steps + nsplit - 1) / nsplit * kKeyStep;
    const int64_t b = (int64_t)s * each;
    *begin = b < keys ? (int)b : keys;
    *end = b + each < keys ? (int)(b + each) : keys;
}

// row of the cache that holds key j of sequence b, or -1
__device__ int64_t row_of_key(const CachePages& c, int b, int j) {
    const int k = j / (int)c.page;
    const int64_t page = c.table ? c.table[b * c.nmaxpage + k] : b;
    if (page < 0 || page >= c.npage) return -1;
    return page * c.page + (j - k * (int)c.page);
}

// whether new token t sees new token s
__device__ bool sees_new(const int* mask, int64_t ntimes, int64_t b, int t, int s) {
    if (mask == nullptr) return s <= t;
    const int64_t nword = (ntimes + 31) / 32;
    return ((unsigned)mask[(b * ntimes + t) * nword + s / 32] >> (s & 31)) & 1u;
}

// Results of a row: straight to y, or the part's sums.
__device__ __forceinline__ int64_t slot_of(const Parts& parts, int64_t rows, int64_t row, int split) {
    return (int64_t)split * rows + row;
}

// One row (b, t, h) over the keys [begin, end), a wave with its lanes along the head: any head size up to kMaxPiece, any
// alignment, plain fp32 sums, and only what the row sees is read into them.
__device__ void attend_row(const CacheAttentionArgs& a, const Parts& parts, const Sequence& seq, int b, int t, int h, int split,
                           int begin, int end) {
    const int lane = threadIdx.x & (kWave - 1);
    const CachePages& c = a.pages;
    const int64_t bt = (int64_t)b * c.ntimes + t, row = bt * a.nhead + h;
    const int np = c.npiece, kvh = h / (a.nhead / c.nkvhead);
    const int64_t width = (int64_t)c.nkvhead * np;
    const float coef = a.hcoef ? *a.hcoef : 0.0f;
    float q[kMaxPiece / kWave], acc[kMaxPiece / kWave];
#pragma unroll
    for (int i = 0; i < kMaxPiece / kWave; i++) {
        const int d = lane + i * kWave;
        q[i] = d < np ? a.q[bt * a.ldq + (int64_t)h * np + d] : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = begin; j < end; j++) {
        if (j >= seq.len && !sees_new(a.mask, c.ntimes, b, t, j - seq.len)) continue;
        const int64_t at = row_of_key(c, b, j);
        if (at < 0) continue;
        const int64_t base = at * width + (int64_t)kvh * np;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxPiece / kWave; i++) {
            const int d = lane + i * kWave;
            if (d < np) s = fmaf(q[i], a.ck[base + d], s);
        }
#pragma unroll
        for (int w = 1; w < kWave; w *= 2) s += __shfl_xor(s, w);
        s *= coef;
        const float top = fmaxf(m, s);
        // the first key, or a maximum of minus infinity so far: nothing to rescale
        const float scale = m == top ? 1.0f : expf(m - top);
        const float p = s == -INFINITY ? 0.0f : expf(s - top);
        l = l * scale + p;
#pragma unroll
        for (int i = 0; i < kMaxPiece / kWave; i++) {
            const int d = lane + i * kWave;
            if (d < np && s != -INFINITY) acc[i] = acc[i] * scale + p * a.cv[base + d];
        }
        m = top;
    }
    float* out = a.y + row * np;
    float inv = 1.0f;
    if (parts.nsplit > 1) {
        const int64_t slot = slot_of(parts, c.nbat * c.ntimes * a.nhead, row, split);
        if (lane == 0) parts.ml[slot] = make_float2(m, l);
        out = parts.acc + slot * np;
    } else {
        inv = l == 0.0f ? 0.0f : 1.0f / l;
    }
#pragma unroll
    for (int i = 0; i < kMaxPiece / kWave; i++) {
        const int d = lane + i * kWave;
        if (d < np) out[d] = acc[i] * inv;
    }
}

__global__ __launch_bounds__(256) void cache_attention_rows_kernel(CacheAttentionArgs a, Parts parts) {
    const CachePages& c = a.pages;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= c.nbat * c.ntimes * a.nhead) return;
    const int h = (int)(row % a.nhead);
    const int64_t bt = row / a.nhead;
    const int b = (int)(bt / c.ntimes), t = (int)(bt % c.ntimes);
    const Sequence seq = sequence_of(c, b);
    if (t >= seq.count) return;
    int begin, end;
    part_of(seq.keys, parts.nsplit, blockIdx.y, &begin, &end);
    attend_row(a, parts, seq, b, t, h, blockIdx.y, begin, end);
}

// The tiled kernel.  The rows that share a key head (new tokens x heads of its group) are taken 16 * NR at a time by a
// workgroup of four waves; each wave takes every fourth tile of 32 keys of the part, and the waves' results are added in
// LDS at the end.  With K as the left and Q as the right operand of v_mfma_f32_16x16x32_bf16 a lane holds scores of ONE
// row (column l & 15), and with key 8 (i / 4) + 4 kb + i % 4 in row i of score block kb it holds the eight keys
// 8 (l >> 4) + 0..7, which is just what the right operand of O^T = V^T P^T wants: the probabilities never leave the lane,
// and maximum, sum and rescaling are the lane's own.  Both operands of both products come straight from memory into
// registers (K: eight elements of a key, V: elements VW n .. VW n + VW - 1 of eight keys, VW = npiece / 16, element
// VW m + j being row m of output block j), as three bf16 each (split_bf16.h); nothing of the cache passes through LDS.
template <int VW, int NR>
struct Tiled {
    static constexpr int np = 16 * VW;
    static constexpr int KC = (np + 31) / 32;
    static constexpr int kRegs = NR * (4 * VW + 2);                                  // of a wave's result, per lane
    static constexpr int kQueryBytes = 3 * KC * NR * kWave * 16;
    static constexpr int kMergeBytes = 2 * kRegs * kWave * 4;
    static constexpr int kLds = (kQueryBytes > kMergeBytes ? kQueryBytes : kMergeBytes) + 16;
};

template <int N>
__device__ __forceinline__ void load_floats(float* to, const float* from) {
    typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef float v2 __attribute__((ext_vector_type(2), aligned(4)));
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
        const v4 v = *reinterpret_cast<const v4*>(from + i);
#pragma unroll
        for (int e = 0; e < 4; e++) to[i + e] = v[e];
    }
    if constexpr (N % 4 >= 2) {
        const v2 v = *reinterpret_cast<const v2*>(from + N / 4 * 4);
        to[N / 4 * 4] = v[0];
        to[N / 4 * 4 + 1] = v[1];
    }
    if constexpr (N % 2 == 1) to[N - 1] = from[N - 1];
}

__device__ __forceinline__ f32x4 mfma6(const Split8& a, const Split8& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.h, b.l, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.l, b.h, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.m, b.m, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.h, b.m, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.m, b.h, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.h, b.h, c, 0, 0, 0);
}

template <int VW, int NR>
__global__ __launch_bounds__(256, VW * NR <= 12 ? 2 : 1) void cache_attention_tiled_kernel(CacheAttentionArgs a, Parts parts, int row_tiles) {
    using T = Tiled<VW, NR>;
    constexpr int np = T::np, KC = T::KC;
    extern __shared__ char lds[];
    const CachePages& c = a.pages;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int n = lane & 15, g = lane >> 4;
    const int split = blockIdx.y;
    const int tile = (int)(blockIdx.x % (unsigned)row_tiles);
    const int bh = (int)(blockIdx.x / (unsigned)row_tiles);
    const int kvh = bh % c.nkvhead, b = bh / c.nkvhead;
    const int group = a.nhead / c.nkvhead;
    const Sequence seq = sequence_of(c, b);
    const int nrow = seq.count * group, row0 = tile * 16 * NR;
    if (row0 >= nrow) return;
    int begin, end;
    part_of(seq.keys, parts.nsplit, split, &begin, &end);
    const int64_t width = (int64_t)c.nkvhead * np;
    const float* ck = a.ck + (int64_t)kvh * np;
    const float* cv = a.cv + (int64_t)kvh * np;

    // the queries, times coef, as three planes of right operands: chunk (plane, kk, r) holds lane's 8 elements
    bf16x8* query = reinterpret_cast<bf16x8*>(lds);
    {
        const float coef = a.hcoef ? *a.hcoef : 0.0f;
        for (int e = threadIdx.x; e < KC * NR * kWave; e += 256) {
            const int el = e & (kWave - 1), r = e / kWave % NR, kk = e / (kWave * NR);
            const int row = row0 + 16 * r + (el & 15), d = 32 * kk + 8 * (el >> 4);
            float x[8] = {};
            if (row < nrow && d < np) {
                const int t = row / group, h = kvh * group + (row - t * group);
                load_floats<8>(x, a.q + ((int64_t)b * c.ntimes + t) * a.ldq + (int64_t)h * np + d);
            }
            const Split8 s = split8([&](int i) { return x[i] * coef; });
            query[e] = s.h;
            query[e + KC * NR * kWave] = s.m;
            query[e + 2 * KC * NR * kWave] = s.l;
        }
    }
    __syncthreads();
    const auto query_at = [&](int kk, int r) {
        const int e = (kk * NR + r) * kWave + lane;
        return Split8{query[e], query[e + KC * NR * kWave], query[e + 2 * KC * NR * kWave]};
    };

    // rows of the cache of a tile's 32 keys, in lanes 0..31 (and once more in 32..63); -1: no such key
    const auto rows_of = [&](int j0) {
        const int j = j0 + (lane & 31);
        return j < end ? (int)row_of_key(c, b, j) : -1;
    };
    float kf[2][KC][8];
    const auto load_keys = [&](int rows) {
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            const int row = __shfl(rows, 8 * (n >> 2) + 4 * kb + (n & 3));
            const float* from = ck + (int64_t)(row < 0 ? 0 : row) * width + 8 * g;
#pragma unroll
            for (int kk = 0; kk < KC; kk++) {
                if (np % 32 == 0 || kk < KC - 1 || g < 2) {
                    load_floats<8>(kf[kb][kk], from + 32 * kk);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) kf[kb][kk][i] = 0.0f;
                }
            }
        }
    };

    f32x4 o[NR][VW];
    float m[NR], l[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < VW; j++) o[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int rows = rows_of(begin + 32 * wave);
    if (begin + 32 * wave < end) load_keys(rows);
    for (int j0 = begin + 32 * wave; j0 < end; j0 += 128) {
        // the queries are read from LDS anew for each tile: kept in registers they would crowd out loads in flight
        __asm__ volatile("" ::: "memory");
        // values of the lane's eight keys
        float vf[8][VW];
        unsigned there = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int row = __shfl(rows, 8 * g + i);
            there |= row < 0 ? 0u : 1u << i;
            load_floats<VW>(vf[i], cv + (int64_t)(row < 0 ? 0 : row) * width + VW * n);
        }
        // in most tiles every row sees every key
        const bool masked = j0 + 32 > seq.len || __any(there != 0xFFu);
        unsigned seen_by_some = 0;
        const int next_rows = rows_of(j0 + 128);
        f32x4 s[NR][2];
#pragma unroll
        for (int r = 0; r < NR; r++) s[r][0] = s[r][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KC; kk++) {
            const Split8 k0 = split8([&](int i) { return kf[0][kk][i]; });
            const Split8 k1 = split8([&](int i) { return kf[1][kk][i]; });
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const Split8 q = query_at(kk, r);
                s[r][0] = mfma6(k0, q, s[r][0]);
                s[r][1] = mfma6(k1, q, s[r][1]);
            }
        }
        if (j0 + 128 < end) load_keys(next_rows);
        Split8 p[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = s[r][i >> 2][i & 3];
            if (masked) {
                const int row = row0 + 16 * r + n;
                const int t = row / group;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int j = j0 + 8 * g + i;
                    const bool seen = row < nrow && (there >> i & 1u) && (j < seq.len || sees_new(a.mask, c.ntimes, b, t, j - seq.len));
                    if (seen) seen_by_some |= 1u << i;
                    else x[i] = -INFINITY;
                }
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
            if (__any(top > m[r])) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                top = fmaxf(top, m[r]);
                const float scale = m[r] == top ? 1.0f : expf(m[r] - top);
                m[r] = top;
                l[r] *= scale;
#pragma unroll
                for (int j = 0; j < VW; j++) o[r][j] *= scale;
            }
            // a row that has seen nothing yet keeps exp(-inf - 0) = 0
            const float base = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = exp2f((x[i] - base) * 1.4426950408889634f);
                l[r] += x[i];
            }
            p[r] = split8([&](int i) { return x[i]; });
        }
        if (masked) {
            // a probability of 0 times a NaN would be one: values that none of the tile's rows sees are not multiplied
#pragma unroll
            for (int w = 1; w < 16; w *= 2) seen_by_some |= __shfl_xor(seen_by_some, w);
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int j = 0; j < VW; j++) vf[i][j] = seen_by_some >> i & 1u ? vf[i][j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < VW; j++) {
            const Split8 v = split8([&](int i) { return vf[i][j]; });
#pragma unroll
            for (int r = 0; r < NR; r++) o[r][j] = mfma6(v, p[r], o[r][j]);
        }
        rows = next_rows;
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        l[r] += __shfl_xor(l[r], 16);
        l[r] += __shfl_xor(l[r], 32);
    }

    // the four waves' results: 2 and 3 into 0 and 1, then 1 into 0
    float* merge = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int step = 2; step >= 1; step /= 2) {
        __syncthreads();
        if (wave >= step && wave < 2 * step) {
            float* to = merge + (wave - step) * T::kRegs * kWave + lane;
#pragma unroll
            for (int r = 0; r < NR; r++) {
                to[(r * (4 * VW + 2)) * kWave] = m[r];
                to[(r * (4 * VW + 2) + 1) * kWave] = l[r];
#pragma unroll
                for (int j = 0; j < VW; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) to[(r * (4 * VW + 2) + 2 + 4 * j + i) * kWave] = o[r][j][i];
            }
        }
        __syncthreads();
        if (wave < step) {
            const float* from = merge + wave * T::kRegs * kWave + lane;
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float om = from[(r * (4 * VW + 2)) * kWave], ol = from[(r * (4 * VW + 2) + 1) * kWave];
                const float top = fmaxf(m[r], om);
                const float mine = m[r] == top ? 1.0f : expf(m[r] - top), theirs = om == top ? 1.0f : expf(om - top);
                m[r] = top;
                l[r] = l[r] * mine + ol * theirs;
#pragma unroll
                for (int j = 0; j < VW; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        o[r][j][i] = o[r][j][i] * mine + from[(r * (4 * VW + 2) + 2 + 4 * j + i) * kWave] * theirs;
            }
        }
    }

    // Infinities and NaN in the cache come out as NaN in any row of the tile, those that do not see them too where others
    // do: the rows are then done again one by one.
    int* again = reinterpret_cast<int*>(lds + T::kLds - 16);
    if (wave == 0) {
        float test = 0.0f;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            test += l[r] * 0.0f;
#pragma unroll
            for (int j = 0; j < VW; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) test += o[r][j][i] * 0.0f;
        }
        const bool bad = __any(test != 0.0f);
        if (lane == 0) *again = bad;
        if (!bad) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const int row = row0 + 16 * r + n;
                if (row < nrow) {
                    const int t = row / group, h = kvh * group + (row - t * group);
                    const int64_t at = ((int64_t)b * c.ntimes + t) * a.nhead + h;
                    float* out = a.y + at * np;
                    float inv = 1.0f;
                    if (parts.nsplit > 1) {
                        const int64_t slot = slot_of(parts, c.nbat * c.ntimes * a.nhead, at, split);
                        if (g == 0) parts.ml[slot] = make_float2(m[r], l[r]);
                        out = parts.acc + slot * np;
                    } else {
                        inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < VW; j++) out[(4 * g + i) * VW + j] = o[r][j][i] * inv;
                }
            }
        }
    }
    __syncthreads();
    if (*again) {
        for (int row = row0 + wave; row < nrow && row < row0 + 16 * NR; row += 4) {
            const int t = row / group;
            attend_row(a, parts, seq, b, t, kvh * group + (row - t * group), split, begin, end);
        }
    }
}

// A wave for a row: y = sum_s e^(m_s - M) acc_s / sum_s e^(m_s - M) l_s over the parts that saw a key.
__global__ __launch_bounds__(256) void cache_attention_join_kernel(CacheAttentionArgs a, Parts parts) {
    const int lane = threadIdx.x & (kWave - 1);
    const CachePages& c = a.pages;
    const int64_t rows = c.nbat * c.ntimes * a.nhead;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= rows) return;
    const int64_t bt = row / a.nhead;
    const Sequence seq = sequence_of(c, (int)(bt / c.ntimes));
    if ((int)(bt % c.ntimes) >= seq.count) return;
    float top = -INFINITY;
    for (int s = 0; s < parts.nsplit; s++) top = fmaxf(top, parts.ml[(int64_t)s * rows + row].x);
    float sum = 0.0f;
    float acc[kMaxPiece / kWave] = {};
    for (int s = 0; s < parts.nsplit; s++) {
        const int64_t slot = (int64_t)s * rows + row;
        const float2 ml = parts.ml[slot];
        if (ml.y == 0.0f) continue;
        const float w = ml.x == top ? 1.0f : expf(ml.x - top);
        sum += w * ml.y;
#pragma unroll
        for (int i = 0; i < kMaxPiece / kWave; i++) {
            const int d = lane + i * kWave;
            if (d < c.npiece) acc[i] += w * parts.acc[slot * c.npiece + d];
        }
    }
#pragma unroll
    for (int i = 0; i < kMaxPiece / kWave; i++) {
        const int d = lane + i * kWave;
        if (d < c.npiece) a.y[row * c.npiece + d] = sum == 0.0f ? 0.0f : acc[i] / sum;
    }
}

int parts_buffer(Parts* parts, int64_t rows, int npiece) {
    float* buf = nullptr;
    const int64_t slots = (int64_t)parts->nsplit * rows;
    KAI_TRY(workspace(slots * (npiece + 2) * (int64_t)sizeof(float), &buf));
    parts->ml = reinterpret_cast<float2*>(buf);
    parts->acc = buf + 2 * slots;
    return KAI_OK;
}

template <int VW, int NR>
int launch_tiled(const CacheAttentionArgs& a, const Parts& parts, int64_t row_tiles, hipStream_t stream) {
    const CachePages& c = a.pages;
    constexpr int lds = Tiled<VW, NR>::kLds;
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    if (lds > 64 * 1024)
        KAI_TRY(check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&cache_attention_tiled_kernel<VW, NR>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                          "hipFuncSetAttribute(cache_attention_tiled_kernel)"));
    const dim3 grid((unsigned)(c.nbat * c.nkvhead * row_tiles), (unsigned)parts.nsplit);
    cache_attention_tiled_kernel<VW, NR><<<grid, 256, lds, stream>>>(a, parts, (int)row_tiles);
    return check_launch("cache_attention_tiled_kernel");
}

template <int VW>
int launch_tiled_rows(const CacheAttentionArgs& a, const Parts& parts, int nr, int64_t row_tiles, hipStream_t stream) {
    if (nr == 1) return launch_tiled<VW, 1>(a, parts, row_tiles, stream);
    if (nr == 2) return launch_tiled<VW, 2>(a, parts, row_tiles, stream);
    return launch_tiled<VW, 4>(a, parts, row_tiles, stream);
}

bool tiled_applies(const CacheAttentionArgs& a) {
    const int np = a.pages.npiece;
    return np == 32 || np == 64 || np == 80 || np == 96 || np == 128;
}

int launch_tiled_any(const CacheAttentionArgs& a, const Parts& parts, int nr, int64_t row_tiles, hipStream_t stream) {
    switch (a.pages.npiece) {
    case 32: return launch_tiled_rows<2>(a, parts, nr, row_tiles, stream);
    case 64: return launch_tiled_rows<4>(a, parts, nr, row_tiles, stream);
    case 80: return launch_tiled_rows<5>(a, parts, nr, row_tiles, stream);
    case 96: return launch_tiled_rows<6>(a, parts, nr, row_tiles, stream);
    default: return launch_tiled_rows<8>(a, parts, nr, row_tiles, stream);
    }
}

}  // namespace

int launch_cache_attention(const CacheAttentionArgs& a, hipStream_t stream) {
    const CachePages& c = a.pages;
    const int64_t rows = c.nbat * c.ntimes * a.nhead;
    const int64_t reach = c.page * c.nmaxpage;
    const bool tiled = tiled_applies(a);
    const int64_t shared_rows = c.ntimes * (a.nhead / c.nkvhead);      // of a key head
    const int nr = shared_rows <= 16 ? 1 : shared_rows <= 32 ? 2 : 4;
    const int64_t row_tiles = (shared_rows + 16 * nr - 1) / (16 * nr);
    const int64_t groups = tiled ? c.nbat * c.nkvhead * row_tiles : (rows + 3) / 4;
    // four workgroups for a compute unit, a part of at least 256 keys
    int64_t nsplit = (4 * (int64_t)compute_units() + groups - 1) / groups;
    if (nsplit > reach / 256) nsplit = reach / 256;
    if (nsplit < 1) nsplit = 1;
    if (nsplit > 256) nsplit = 256;
    Parts parts{nullptr, nullptr, (int)nsplit};
    if (nsplit > 1) KAI_TRY(parts_buffer(&parts, rows, c.npiece));
    if (tiled) {
        KAI_TRY(launch_tiled_any(a, parts, nr, row_tiles, stream));
    } else {
        cache_attention_rows_kernel<<<dim3((unsigned)groups, (unsigned)nsplit), 256, 0, stream>>>(a, parts);
        KAI_TRY(check_launch("cache_attention_rows_kernel"));
    }
    if (nsplit == 1) return KAI_OK;
    cache_attention_join_kernel<<<(unsigned)((rows + 3) / 4), 256, 0, stream>>>(a, parts);
    return check_launch("cache_attention_join_kernel");
}

}  // namespace kai
