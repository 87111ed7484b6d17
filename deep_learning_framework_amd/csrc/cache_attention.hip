// Attention of new tokens over a paged cache of keys and values.
//
//   y[b, t, h, :] = sum_j p_j v_j,   p = softmax over the keys j that row (b, t) sees of coef * <q, k_j>
//
// with online statistics: a running maximum m, the sum l of exp(s_j - m) and the sum of exp(s_j - m) v_j, all in
// 32 bits; a row that sees nothing gives zeros.  Few rows meet many keys, so the keys of a sequence are cut into
// parts that run as separate workgroups; cache_attention_join_kernel adds the parts,
//   y = sum_s e^(m_s - M) acc_s / sum_s e^(m_s - M) l_s.
#include "decoder_ops.h"

namespace kai {
namespace {

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

// A wave for a row and a part of the keys, the lanes along the head: any head size up to kMaxPiece, any alignment.
__global__ __launch_bounds__(256) void cache_attention_rows_kernel(CacheAttentionArgs a, Parts parts) {
    const int lane = threadIdx.x & (kWave - 1);
    const CachePages& c = a.pages;
    const int64_t rows = c.nbat * c.ntimes * a.nhead;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= rows) return;
    const int split = blockIdx.y;
    const int h = (int)(row % a.nhead);
    const int64_t bt = row / a.nhead;
    const int b = (int)(bt / c.ntimes), t = (int)(bt % c.ntimes);
    const Sequence seq = sequence_of(c, b);
    if (t >= seq.count) return;
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
    int begin, end;
    part_of(seq.keys, parts.nsplit, split, &begin, &end);
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
            if (d < np) acc[i] = acc[i] * scale + p * a.cv[base + d];
        }
        m = top;
    }
    if (parts.nsplit == 1) {
#pragma unroll
        for (int i = 0; i < kMaxPiece / kWave; i++) {
            const int d = lane + i * kWave;
            if (d < np) a.y[row * np + d] = l == 0.0f ? 0.0f : acc[i] / l;
        }
        return;
    }
    const int64_t slot = (int64_t)split * rows + row;
    if (lane == 0) parts.ml[slot] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < kMaxPiece / kWave; i++) {
        const int d = lane + i * kWave;
        if (d < np) parts.acc[slot * np + d] = acc[i];
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

}  // namespace

int launch_cache_attention(const CacheAttentionArgs& a, hipStream_t stream) {
    const CachePages& c = a.pages;
    const int64_t rows = c.nbat * c.ntimes * a.nhead;
    const int64_t groups = (rows + 3) / 4;
    // four workgroups for a compute unit, a part of at least 256 keys
    const int64_t reach = c.page * c.nmaxpage;
    int64_t nsplit = (4 * (int64_t)compute_units() + groups - 1) / groups;
    if (nsplit > reach / 256) nsplit = reach / 256;
    if (nsplit < 1) nsplit = 1;
    if (nsplit > 256) nsplit = 256;
    Parts parts{nullptr, nullptr, (int)nsplit};
    if (nsplit > 1) KAI_TRY(parts_buffer(&parts, rows, c.npiece));
    cache_attention_rows_kernel<<<dim3((unsigned)groups, (unsigned)nsplit), 256, 0, stream>>>(a, parts);
    KAI_TRY(check_launch("cache_attention_rows_kernel"));
    if (nsplit == 1) return KAI_OK;
    cache_attention_join_kernel<<<(unsigned)groups, 256, 0, stream>>>(a, parts);
    return check_launch("cache_attention_join_kernel");
}

}  // namespace kai
