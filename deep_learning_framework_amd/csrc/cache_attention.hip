// Attention of new tokens over a paged cache of keys and values.
//
//   y[b, t, h, :] = sum_j p_j v_j,   p = softmax over the keys j that row (b, t) sees of coef * <q, k_j>
//
// with online statistics: a running maximum m, the sum l of exp(s_j - m) and the sum of exp(s_j - m) v_j, all in
// 32 bits; a row that sees nothing gives zeros.  Few rows meet many keys, so the keys of a sequence are cut into
// parts that run as separate workgroups; cache_attention_join_kernel adds the parts' own results y_s = acc_s / l_s,
//   y = sum_s w_s y_s,   w_s = e^(m_s - M) l_s / sum_s e^(m_s - M) l_s,
// a weighted mean, which stays finite where the sums of large values would not.
//
// Bound: HBM (the keys and values once, 8 bytes an element pair) while a key head has few rows: 32 sequences x 1 token of 32 heads
// of 128 on 8 key heads over up to 4096 keys 135 us = 5.4 TB/s.  From some 50 rows of a key head on the matrix cores and the
// cutting of keys and values take as long as the bytes: 1 x 16 tokens over 131072 keys 276 .. 297 us = 3.9 .. 3.6 TB/s and 124 .. 115 TFLOP/s.
// Short caches are a chain of latencies (lengths, page, keys, the joining launch): 3 x up to 61 tokens of 12 heads of 64 over up to
// 1500 keys 22.0 us, 17.6 of them the tiled kernel's (three tiles of keys a wave) and 4.6 the join's.
//
// Not done here: tiles of keys that a causal run's rows cannot see are loaded and multiplied all the same (a prompt on an empty
// cache takes about twice its work), and the parts are cut by the pages' capacity, which one recorded launch serves at every
// length, not by the length: a short sequence behind a long table has parts with too few keys for four waves, or none.
#include <type_traits>

#include "decoder_ops.h"
#include "split_bf16.h"

namespace kai {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr int kMaxPiece = 256;
constexpr int kMaxParts = 256;   // a thread of the joining workgroup each
constexpr int kKeyStep = 32;     // a part of a sequence's keys is a whole number of these

struct Parts {
    float* acc;      // [nsplit][rows][npiece]: the parts' results
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

// Which of the keys j .. j + 7 new token t sees, as bits; none for rows behind the count.  Keys behind the new ones are the
// caller's to leave out.
__device__ __forceinline__ unsigned eight_seen(const int* mask, int64_t ntimes, const Sequence& seq, int64_t b, int t, int j) {
    if (t >= seq.count) return 0u;
    const int s = j - seq.len;
    if (s <= -8) return 0xFFu;
    const int from = s < 0 ? 0 : s;
    unsigned bits;
    if (mask == nullptr) {
        const int seen = t + 1 - from;       // new tokens from `from` on
        bits = seen >= 8 ? 0xFFu : seen <= 0 ? 0u : (1u << seen) - 1;
    } else {
        const int nword = (int)((ntimes + 31) / 32), w = from / 32 < nword ? from / 32 : nword - 1;
        const unsigned* words = reinterpret_cast<const unsigned*>(mask) + (b * ntimes + t) * nword;
        const unsigned lo = words[w], hi = words[w + 1 < nword ? w + 1 : w];
        bits = (unsigned)((((uint64_t)hi << 32) | lo) >> (from & 31)) & 0xFFu;
    }
    return s < 0 ? (bits << -s | ((1u << -s) - 1)) & 0xFFu : bits;
}

// Results of a row: straight to y, or the part's.
__device__ __forceinline__ int64_t slot_of(const Parts& parts, int64_t rows, int64_t row, int split) {
    return (int64_t)split * rows + row;
}

// One row (b, t, h) over the keys [begin, end), a wave with its lanes along the head: any head size up to kMaxPiece, any
// alignment, plain fp32 sums, and only what the row sees is read into them.  Where sums pass the largest float (up to 2^30 values
// below 2^128), a second pass with the weights times 2^-32 forms them anew, and only them: smaller ones beside them would lose bits.
__device__ void attend_row(const CacheAttentionArgs& a, const Parts& parts, const Sequence& seq, int b, int t, int h, int split,
                           int begin, int end) {
    const int lane = threadIdx.x & (kWave - 1);
    const CachePages& c = a.pages;
    const int64_t bt = (int64_t)b * c.ntimes + t, row = bt * a.nhead + h;
    const int np = c.npiece, kvh = h / (a.nhead / c.nkvhead);
    const int64_t width = (int64_t)c.nkvhead * np;
    const float coef = a.hcoef ? *a.hcoef : 0.0f;
    float* out = a.y + row * np;
    float2* ml = nullptr;
    if (parts.nsplit > 1) {
        const int64_t slot = slot_of(parts, c.nbat * c.ntimes * a.nhead, row, split);
        ml = parts.ml + slot;
        out = parts.acc + slot * np;
    }
    float q[kMaxPiece / kWave];
#pragma unroll
    for (int i = 0; i < kMaxPiece / kWave; i++) {
        const int d = lane + i * kWave;
        q[i] = d < np ? a.q[bt * a.ldq + (int64_t)h * np + d] : 0.0f;
    }
    float down = 1.0f;
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
        float acc[kMaxPiece / kWave] = {};
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
            const float weight = p * down;
#pragma unroll
            for (int i = 0; i < kMaxPiece / kWave; i++) {
                const int d = lane + i * kWave;
                if (d < np && s != -INFINITY) acc[i] = acc[i] * scale + weight * a.cv[base + d];
            }
            m = top;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / (l * down);
        bool passed = false;
#pragma unroll
        for (int i = 0; i < kMaxPiece / kWave; i++) {
            const int d = lane + i * kWave;
            const bool over = !(fabsf(acc[i]) <= kLargestFinite);
            if (d < np && (pass == 0 || !(fabsf(out[d]) <= kLargestFinite))) out[d] = acc[i] * inv;
            passed |= over;
        }
        if (ml && lane == 0) *ml = make_float2(m, l);
        if (!(l <= kLargestFinite) || !__any(passed)) break;     // a NaN among the scores: every element is one
        down = 0x1p-32f;
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
    static constexpr int kQueryChunks = KC * NR * kWave;                 // of 8 elements, and three planes of them
    static constexpr int kQueryBytes = 3 * kQueryChunks * 16;
    static constexpr int kWaveChunks = NR * VW * kWave;                  // of a wave's result, 4 elements each
    static constexpr int kMergeBytes = 4 * kWaveChunks * 16;
    static constexpr int kRows = 16 * NR;
    static constexpr int kLds = (kQueryBytes > kMergeBytes ? kQueryBytes : kMergeBytes);
};

// f(0), ..., f(N - 1) with compile-time indices
template <int B, int E, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (B < E) {
        f(std::integral_constant<int, B>{});
        static_for<B + 1, E>(f);
    }
}

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

// c[i] += a(i) . b(i), the small products first, a product's turn going round the N independent sums
template <int N, typename A, typename B>
__device__ __forceinline__ void mfma6(f32x4* const* c, A&& a, B&& b) {
#pragma unroll
    for (int i = 0; i < N; i++) *c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(i).h, b(i).l, *c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < N; i++) *c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(i).l, b(i).h, *c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < N; i++) *c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(i).m, b(i).m, *c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < N; i++) *c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(i).h, b(i).m, *c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < N; i++) *c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(i).m, b(i).h, *c[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < N; i++) *c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a(i).h, b(i).h, *c[i], 0, 0, 0);
}

// Asks the scheduler to spread the N matrix instructions of a block of code over its vector instructions.
template <int N>
__device__ __forceinline__ void interleave() {
    static_for<0, N>([](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
    });
}

template <int VW, int NR>
__global__ __launch_bounds__(256, VW * NR > 16 ? 1 : 2) void cache_attention_tiled_kernel(CacheAttentionArgs a, Parts parts, int row_tiles) {
    using T = Tiled<VW, NR>;
    constexpr int np = T::np, KC = T::KC;
    extern __shared__ char lds[];
    __shared__ float2 part_ml[4][T::kRows];
    const CachePages& c = a.pages;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int n = lane & 15, g = lane >> 4;
    const int split = blockIdx.y;
    const int tile = (int)(blockIdx.x % (unsigned)row_tiles);
    const int bh = (int)(blockIdx.x / (unsigned)row_tiles);
    const int kvh = bh % c.nkvhead, b = bh / c.nkvhead;
    const int group = a.nhead / c.nkvhead;
    const int row0 = tile * T::kRows;
    // The start is one chain of loads: lengths, page, keys.  The queries come meanwhile.
    constexpr int kQueryLoads = (T::kQueryChunks + 256 - 1) / 256;
    float qx[kQueryLoads][8];
#pragma unroll
    for (int i = 0; i < kQueryLoads; i++) {
        const int e = (int)threadIdx.x + 256 * i;
        const int row = row0 + 16 * (e / kWave % NR) + (e & 15), d = 32 * (e / (kWave * NR)) + (e >> 4 & 3) * 8;
        const int t = row / group, h = kvh * group + (row - t * group);
#pragma unroll
        for (int k = 0; k < 8; k++) qx[i][k] = 0.0f;
        if (e < T::kQueryChunks && t < c.ntimes && d < np)
            load_floats<8>(qx[i], a.q + ((int64_t)b * c.ntimes + t) * a.ldq + (int64_t)h * np + d);
    }
    const Sequence seq = sequence_of(c, b);
    const int nrow = seq.count * group;
    if (row0 >= nrow) return;
    int begin, end;
    part_of(seq.keys, parts.nsplit, split, &begin, &end);
    const int64_t width = (int64_t)c.nkvhead * np;
    const float* ck = a.ck + (int64_t)kvh * np;
    const float* cv = a.cv + (int64_t)kvh * np;

    // rows of the cache of a tile's 32 keys, in lanes 0..31 (and once more in 32..63); -1: no such key
    const auto rows_of = [&](int j0) {
        const int j = j0 + (lane & 31);
        return j < end ? (int)row_of_key(c, b, j) : -1;
    };
    // Where a key does not exist row 0 is loaded and not used.
    const auto existing = [](int row) { return (int64_t)(row < 0 ? 0 : row); };
    float kf[2][KC][8], vf[8][VW];
    unsigned there = 0;
    const auto load_key = [&](const float* key, int kb, int kk) {
        if (np % 32 == 0 || kk < KC - 1 || g < 2) {
            load_floats<8>(kf[kb][kk], key + 32 * kk);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) kf[kb][kk][i] = 0.0f;
        }
    };
    const auto key_of = [&](int rows, int kb) {
        return ck + existing(__shfl(rows, 8 * (n >> 2) + 4 * kb + (n & 3))) * width + 8 * g;
    };
    int vrow[8];
    const auto value_rows = [&](int rows) {
        there = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            vrow[i] = __shfl(rows, 8 * g + i);
            there |= vrow[i] < 0 ? 0u : 1u << i;
        }
    };
    constexpr int kGroups = (VW + 3) / 4;
    // With one tile of rows a wave, each register is loaded for the wave's next tile as soon as this tile's use of it is
    // over.  With more rows there is no room for a whole tile in flight (two waves of a SIMD share its 512 registers): the
    // values' second half and the next keys' two halves follow one another through the same registers.
    constexpr bool kLate = NR == 2 && VW > 4;
    const auto load_values = [&](auto group) {
        constexpr int j0 = 4 * decltype(group)::value, count = VW - j0 < 4 ? VW - j0 : 4;
#pragma unroll
        for (int i = 0; i < 8; i++) load_floats<count>(vf[i] + j0, cv + existing(vrow[i]) * width + VW * n + j0);
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
    const int first = begin + 32 * wave;
    if (first < end) {
        const int rows = rows_of(first);
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int kk = 0; kk < KC; kk++) load_key(key_of(rows, kb), kb, kk);
        value_rows(rows);
        if constexpr (!kLate) static_for<0, kGroups>(load_values);
    }
    // the queries, times coef, as three planes of right operands: chunk (plane, kk, r) holds a lane's 8 elements
    bf16x8* query = reinterpret_cast<bf16x8*>(lds);
    {
        const float coef = a.hcoef ? *a.hcoef : 0.0f;
#pragma unroll
        for (int i = 0; i < kQueryLoads; i++) {
            const int e = (int)threadIdx.x + 256 * i;
            if (e >= T::kQueryChunks) break;
            const Split8 s = split8([&](int k) { return qx[i][k] * coef; });
            query[e] = s.h;
            query[e + T::kQueryChunks] = s.m;
            query[e + 2 * T::kQueryChunks] = s.l;
        }
    }
    __syncthreads();
    const auto query_at = [&](int kk, int r) {
        const int e = (kk * NR + r) * kWave + lane;
        return Split8{query[e], query[e + T::kQueryChunks], query[e + 2 * T::kQueryChunks]};
    };
    int next_rows = rows_of(first + 128);
    for (int j0 = first; j0 < end; j0 += 128) {
        // the queries are read from LDS anew for each tile: kept in registers they would crowd out loads in flight
        __asm__ volatile("" ::: "memory");
        const bool masked = j0 + 32 > seq.len || __any(there != 0xFFu);     // in most tiles every row sees every key
        unsigned sees[NR], seen_by_some = 0;
        if (masked) {
#pragma unroll
            for (int r = 0; r < NR; r++) sees[r] = there & eight_seen(a.mask, c.ntimes, seq, b, (row0 + 16 * r + n) / group, j0 + 8 * g);
        }
        const float* next_key[2] = {key_of(next_rows, 0), key_of(next_rows, 1)};
        if constexpr (kLate) load_values(std::integral_constant<int, 0>{});
        f32x4 s[NR][2];
#pragma unroll
        for (int r = 0; r < NR; r++) s[r][0] = s[r][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KC; kk++) {
            const Split8 k[2] = {split8([&](int i) { return kf[0][kk][i]; }), split8([&](int i) { return kf[1][kk][i]; })};
            if constexpr (!kLate) {
                load_key(next_key[0], 0, kk);
                load_key(next_key[1], 1, kk);
            } else if (kk == (KC - 1) / 2) {
                static_for<1, kGroups>(load_values);
            }
            if constexpr (NR == 1) {
                const Split8 q = query_at(kk, 0);
                f32x4* const sums[2] = {&s[0][0], &s[0][1]};
                mfma6<2>(sums, [&](int i) { return k[i]; }, [&](int) { return q; });
            } else {
#pragma unroll
                for (int r = 0; r < NR; r += 2) {
                    const Split8 q[2] = {query_at(kk, r), query_at(kk, r + 1)};
                    f32x4* const sums[4] = {&s[r][0], &s[r][1], &s[r + 1][0], &s[r + 1][1]};
                    mfma6<4>(sums, [&](int i) { return k[i & 1]; }, [&](int i) { return q[i >> 1]; });
                }
            }
        }
        if constexpr (NR > 1) interleave<12 * KC * NR>();
        Split8 p[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = s[r][i >> 2][i & 3];
            if (masked) {
                seen_by_some |= sees[r];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = sees[r] >> i & 1u ? x[i] : -INFINITY;
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
            // e^-d as 2^(-d log2 e): the constant and the product, rounded, move it by 2 d 2^-24 of itself at most, which is below
            // 0.74 * 2^-24 of the largest probability (d e^-d <= 1 / e); what is below 2^-126 of that becomes 0
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __builtin_amdgcn_exp2f((x[i] - base) * 1.4426950408889634f);
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
        value_rows(next_rows);
        if constexpr (!kLate) next_rows = rows_of(j0 + 256);
        static_for<0, kGroups>([&](auto group) {
            constexpr int first_j = 4 * decltype(group)::value, last_j = VW < first_j + 4 ? VW : first_j + 4;
#pragma unroll
            for (int j = first_j; j < last_j; j++) {
                const Split8 v = split8([&](int i) { return vf[i][j]; });
                f32x4* sums[NR];
#pragma unroll
                for (int r = 0; r < NR; r++) sums[r] = &o[r][j];
                mfma6<NR>(sums, [&](int) { return v; }, [&](int i) { return p[i]; });
            }
            if constexpr (!kLate) {
                load_values(group);
            } else {
#pragma unroll
                for (int kk = decltype(group)::value * KC / kGroups; kk < (decltype(group)::value + 1) * KC / kGroups; kk++) {
                    load_key(next_key[0], 0, kk);
                    load_key(next_key[1], 1, kk);
                }
            }
        });
        if constexpr (NR > 1) interleave<6 * VW * NR>();
        if constexpr (kLate) next_rows = rows_of(j0 + 256);
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
        l[r] += __shfl_xor(l[r], 16);
        l[r] += __shfl_xor(l[r], 32);
    }

    // The four waves' results meet in LDS.  A thread then takes element i of group g of each sixteenth row's VW blocks: VW
    // consecutive elements of the row.
    __syncthreads();
    f32x4* merge = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int r = 0; r < NR; r++) {
        if (g == 0) part_ml[wave][16 * r + n] = make_float2(m[r], l[r]);
#pragma unroll
        for (int j = 0; j < VW; j++) merge[((wave * NR + r) * VW + j) * kWave + lane] = o[r][j];
    }
    __syncthreads();
    // Infinities and NaN in the cache come out as NaN in any row of the tile, those that do not see them too where others
    // do, and sums of large values as infinities: the rows are then done again one by one.
    float test = 0.0f;
    const int i = threadIdx.x & 3, rn = threadIdx.x >> 2 & 15, rg = wave;
#pragma unroll 1
    for (int r = 0; r < NR; r++) {
        const int row = row0 + 16 * r + rn;
        if (row >= nrow) break;
        float2 ml[4];
#pragma unroll
        for (int w = 0; w < 4; w++) ml[w] = part_ml[w][16 * r + rn];
        const float top = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
        float sum = 0.0f, v[VW] = {};
        const float* from = reinterpret_cast<const float*>(merge + r * VW * kWave + rg * 16 + rn) + i;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float scale = ml[w].x == top ? 1.0f : expf(ml[w].x - top);
            sum += ml[w].y * scale;
#pragma unroll
            for (int j = 0; j < VW; j++) v[j] += from[(w * T::kWaveChunks + j * kWave) * 4] * scale;
        }
        const int t = row / group, h = kvh * group + (row - t * group);
        const int64_t at = ((int64_t)b * c.ntimes + t) * a.nhead + h;
        float* out = a.y + at * np;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (parts.nsplit > 1) {
            const int64_t slot = slot_of(parts, c.nbat * c.ntimes * a.nhead, at, split);
            if (threadIdx.x % 4 == 0 && rg == 0) parts.ml[slot] = make_float2(top, sum);
            out = parts.acc + slot * np;
        }
        test += sum * 0.0f;
#pragma unroll
        for (int j = 0; j < VW; j++) {
            test += v[j] * 0.0f;
            out[(4 * rg + i) * VW + j] = v[j] * inv;
        }
    }
    if (__syncthreads_or(test != 0.0f)) {
#pragma unroll 1
        for (int row = row0 + wave; row < nrow && row < row0 + T::kRows; row += 4) {
            const int t = row / group;
            attend_row(a, parts, seq, b, t, kvh * group + (row - t * group), split, begin, end);
        }
    }
}

// A workgroup for a row: y = sum_s w_s y_s over the parts that saw a key.  Each thread finds a part's weight; then the four waves
// take every fourth part, the lanes along the head, and meet in LDS.
__global__ __launch_bounds__(256) void cache_attention_join_kernel(CacheAttentionArgs a, Parts parts) {
    __shared__ float weight[kMaxParts], scratch[8], sums[4][kMaxPiece];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const CachePages& c = a.pages;
    const int64_t rows = c.nbat * c.ntimes * a.nhead, row = blockIdx.x;
    const int64_t bt = row / a.nhead;
    const Sequence seq = sequence_of(c, (int)(bt / c.ntimes));
    if ((int)(bt % c.ntimes) >= seq.count) return;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if ((int)threadIdx.x < parts.nsplit) ml = parts.ml[slot_of(parts, rows, row, threadIdx.x)];
    float top = ml.x;
#pragma unroll
    for (int w = 1; w < kWave; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
    if (lane == 0) scratch[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
    // a part that saw no key has a sum of 0; one whose scores are all NaN has a NaN, and no maximum that weighs it
    const float mine = ml.y == 0.0f ? 0.0f : ml.y != ml.y ? ml.y : ml.x == top ? ml.y : ml.y * expf(ml.x - top);
    float sum = mine;
#pragma unroll
    for (int w = 1; w < kWave; w *= 2) sum += __shfl_xor(sum, w);
    if (lane == 0) scratch[4 + wave] = sum;
    __syncthreads();
    sum = scratch[4] + scratch[5] + scratch[6] + scratch[7];
    weight[threadIdx.x] = sum == 0.0f ? 0.0f : mine / sum;
    __syncthreads();
    float acc[kMaxPiece / kWave] = {};
#pragma unroll 4
    for (int s = wave; s < parts.nsplit; s += 4) {
        const float w = weight[s];
        const float* from = parts.acc + slot_of(parts, rows, row, s) * c.npiece;
#pragma unroll
        for (int i = 0; i < kMaxPiece / kWave; i++) {
            const int d = lane + i * kWave;
            acc[i] += w * (d < c.npiece ? from[d] : 0.0f);
        }
    }
#pragma unroll
    for (int i = 0; i < kMaxPiece / kWave; i++) sums[wave][lane + i * kWave] = acc[i];
    __syncthreads();
    for (int d = threadIdx.x; d < c.npiece; d += 256) a.y[row * c.npiece + d] = sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d];
}

template <int VW, int NR>
int launch_tiled(const CacheAttentionArgs& a, const Parts& parts, int64_t row_tiles, hipStream_t stream) {
    const CachePages& c = a.pages;
    using T = Tiled<VW, NR>;
    static_assert(T::kLds + 4 * T::kRows * 8 <= 160 * 1024, "LDS of a compute unit");
    if (T::kLds + 4 * T::kRows * 8 > 64 * 1024)
        KAI_TRY(check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(&cache_attention_tiled_kernel<VW, NR>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds),
                          "hipFuncSetAttribute(cache_attention_tiled_kernel)"));
    const dim3 grid((unsigned)(c.nbat * c.nkvhead * row_tiles), (unsigned)parts.nsplit);
    cache_attention_tiled_kernel<VW, NR><<<grid, 256, T::kLds, stream>>>(a, parts, (int)row_tiles);
    return check_launch("cache_attention_tiled_kernel");
}

template <int VW>
int launch_tiled_rows(const CacheAttentionArgs& a, const Parts& parts, int nr, int64_t row_tiles, hipStream_t stream) {
    if (nr == 1) return launch_tiled<VW, 1>(a, parts, row_tiles, stream);
    if (nr == 2) return launch_tiled<VW, 2>(a, parts, row_tiles, stream);
    return launch_tiled<VW, 4>(a, parts, row_tiles, stream);
}

bool tiled_applies(int npiece) {
    return npiece == 32 || npiece == 64 || npiece == 80 || npiece == 96 || npiece == 128;
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

int cache_attention_plan(const CachePages& c, int nhead, CacheAttentionPlan* plan) {
    const int64_t rows = c.nbat * c.ntimes * nhead;
    const int64_t reach = c.page * c.nmaxpage;
    const bool tiled = tiled_applies(c.npiece);
    const int64_t shared_rows = c.ntimes * (nhead / c.nkvhead);      // of a key head
    const int64_t cu = compute_units();
    // parts down to a tile of 32 keys for each wave
    const int64_t tiles = (reach + 127) / 128, most = tiles < 1 ? 1 : tiles > kMaxParts ? kMaxParts : tiles;
    // The largest tile of rows that the rows fill: each tile cuts the same keys and values into pieces.  64 rows where that leaves
    // two workgroups for a compute unit, 32 where it leaves half a one (32 heads of 128 on 8 key heads, 16 tokens over 4000 keys:
    // 64 rows, 256 workgroups 27.3 us, 32 rows 23.8; over 2000 32 rows, 256 workgroups 18.0, 16 rows 21.5; 8 over 1000 32 rows, 64
    // workgroups 15.7, 16 rows 14.3).
    int nr = shared_rows <= 16 ? 1 : shared_rows <= 32 ? 2 : 4;
    const auto tiles_of_rows = [&](int n) { return (shared_rows + 16 * n - 1) / (16 * n); };
    while (nr > 1 && c.nbat * c.nkvhead * tiles_of_rows(nr) * most < (nr == 4 ? 2 * cu : cu / 2)) nr /= 2;
    const int64_t row_tiles = tiles_of_rows(nr);
    const int64_t groups = tiled ? c.nbat * c.nkvhead * row_tiles : (rows + 3) / 4;
    // threads of a launch are counted in 32 bits
    if (groups >= 1ll << 24) return fail(KAI_ERR_INVALID_ARGUMENT, "cache_attention: nbat * nkvhead above 2^23");
    const int64_t resident = nr == 4 ? 1 : 2;      // workgroups of a compute unit
    // One round of workgroups over the chip; two where sequences of different lengths may stand side by side and the parts
    // stay long (their workgroups then even out).  32 x 1 over 4096 to 1366 keys: one round 155 us, two 138; 1 x 16 over
    // 131072: 294 and 314; 3 x 61 over 1500 to 834, where two rounds' parts are of 195 keys: 22.7 and 26.6.
    int64_t nsplit = resident * cu / groups;
    if (c.nbat > 1 && reach >= 2 * nsplit * 512) nsplit *= 2;
    if (nsplit > most) nsplit = most;
    if (nsplit < 1) nsplit = 1;
    plan->row_tile = tiled ? 16 * nr : 0;
    plan->row_tiles = row_tiles;
    plan->groups = groups;
    plan->nsplit = (int)nsplit;
    plan->scratch = nsplit > 1 ? nsplit * rows * (c.npiece + 2) * (int64_t)sizeof(float) : 0;
    return KAI_OK;
}

int launch_cache_attention(const CacheAttentionArgs& a, hipStream_t stream) {
    const CachePages& c = a.pages;
    const int64_t rows = c.nbat * c.ntimes * a.nhead;
    CacheAttentionPlan plan;
    KAI_TRY(cache_attention_plan(c, a.nhead, &plan));
    Parts parts{nullptr, nullptr, plan.nsplit};
    if (plan.nsplit > 1) {
        float* buf = nullptr;
        KAI_TRY(workspace(plan.scratch, &buf));
        parts.ml = reinterpret_cast<float2*>(buf);
        parts.acc = buf + 2 * plan.nsplit * rows;
    }
    if (plan.row_tile > 0) {
        KAI_TRY(launch_tiled_any(a, parts, plan.row_tile / 16, plan.row_tiles, stream));
    } else {
        cache_attention_rows_kernel<<<dim3((unsigned)plan.groups, (unsigned)plan.nsplit), 256, 0, stream>>>(a, parts);
        KAI_TRY(check_launch("cache_attention_rows_kernel"));
    }
    if (plan.nsplit == 1) return KAI_OK;
    cache_attention_join_kernel<<<(unsigned)rows, 256, 0, stream>>>(a, parts);
    return check_launch("cache_attention_join_kernel");
}

}  // namespace kai
