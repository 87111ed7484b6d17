// Launchers of the operators of a decoder block: rotary positions and the cache of keys and values
// (rotary_cache.hip), attention over that cache (cache_attention.hip), the gated feed-forward projection
// (gated.hip).  Their C-ABI and its argument checks are in kai_abi_decoder.hip.
#pragma once

#include "kai_common.h"

namespace kai {

// What the kernels need of a kai_rotary_desc, in 64 bits: the turn (angle / 2 pi) of pair i at position p is
// p * exp2(step * i) / (2 pi), scaled as `scaling` says.
struct RotaryParams {
    double step;            // log2 of the ratio of two neighbouring frequencies
    double inv_factor;      // 1 / factor (linear, parts), else 1
    double trained_turns;   // parts: trained length / (2 pi)
    double low, inv_span;   // parts: low_turns, 1 / (high_turns - low_turns)
    float magnitude;
    int nrot;               // rotated elements at the front of a head, even; 0: none
    int pairs;              // 1: elements (2i, 2i+1) turn together; 0: (i, i + nrot/2)
    int parts;              // 1: scaled by parts
};

struct RotaryArgs {
    float* y;
    const float* x;
    const int* pos;         // null: the row's place in its sequence
    int64_t ntok, ntimes, ld;
    int nhead, npiece;
    RotaryParams rot;
    bool back;
};
int launch_rotary(const RotaryArgs& a, hipStream_t stream);

// The pages of a cache: key j of sequence b is row (table[b * nmaxpage + j / page]) * page + j % page of width
// floats; a null table is the identity with one page a sequence.  Page numbers outside [0, npage) and keys behind
// nmaxpage pages do not exist.
struct CachePages {
    const int* table;
    const int* len;         // keys of each sequence in front of the new ones
    const int* count;       // new tokens of each sequence; null: ntimes
    int64_t nbat, ntimes, npage, page, nmaxpage;
    int nkvhead, npiece;
};

struct CacheAppendArgs {
    CachePages pages;
    float* ck;
    float* cv;
    const float* k;
    const float* v;
    const int* pos;         // null: len[b] + t
    int64_t ld;
    RotaryParams rot;
};
int launch_cache_append(const CacheAppendArgs& a, hipStream_t stream);

struct CacheAttentionArgs {
    CachePages pages;
    float* y;
    const float* q;
    const float* ck;
    const float* cv;
    const int* mask;        // visibility words of the new tokens, null: each sees itself and those before it
    int64_t ldq;
    int nhead;
    const float* hcoef;
};
int launch_cache_attention(const CacheAttentionArgs& a, hipStream_t stream);
// How it runs this geometry (host arithmetic; the pages' pointers are not read).
struct CacheAttentionPlan {
    int row_tile;           // rows of a key head that a workgroup takes, 0: a wave takes a row
    int nsplit;             // parts of the keys
    int64_t row_tiles, groups, scratch;   // tiles of a key head's rows; workgroups of a part; bytes
};
int cache_attention_plan(const CachePages& c, int nhead, CacheAttentionPlan* plan);

struct GatedArgs {
    float* y;               // forward
    float* gate;            // forward: may be null; backward: the stored pre-activations
    float* up;
    const float* wg;
    const float* wu;
    const float* bg;
    const float* bu;
    const float* x;
    int64_t yvec, ndat, xvec;
    int act;
    const float* hleaky;
};
int launch_gated_forward(const GatedArgs& a, hipStream_t stream);
// up to 32 rows in one launch (gated_rows.hip), where that is the faster way
bool gated_rows_pays(const GatedArgs& a);
int launch_gated_rows(const GatedArgs& a, hipStream_t stream);

struct GatedGradArgs {
    float* gx;              // any of the three may be null
    float* gwg;
    float* gwu;
    const float* ggate;     // gradients of the two sums
    const float* gup;
    const float* wg;
    const float* wu;
    const float* x;
    int64_t yvec, ndat, xvec;
    int acc;
};
// gx (+)= ggate . wg + gup . wu, gwg (+)= ggate^T . x, gwu (+)= gup^T . x
int launch_gated_gradients(const GatedGradArgs& a, hipStream_t stream);
// how the forward (0), the gradient of x (1) or those of both weights (2) run with 16-byte aligned operands, as text
std::string gated_plan_text(int which, int64_t yvec, int64_t ndat, int64_t xvec);

// ggate = gy * up * act'(gate), gup = gy * act(gate), [nrow, ncol] each, and their column sums gbg, gbu (+= with acc; null:
// not wanted)
int launch_gated_activation_backward(float* ggate, float* gup, float* gbg, float* gbu, const float* gy, const float* gate,
                                     const float* up, int64_t nrow, int64_t ncol, int act, const float* hleaky, int acc,
                                     hipStream_t stream);
// y = act(gate) * up
int launch_gated_activation(float* y, const float* gate, const float* up, int64_t n, int act, const float* hleaky,
                            hipStream_t stream);

}  // namespace kai
