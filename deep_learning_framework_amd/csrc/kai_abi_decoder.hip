// extern "C" surface of the operators of a decoder block (declared in include/kai_hip.h): argument checks and the
// host arithmetic in front of the launchers of decoder_ops.h.
#include <cmath>
#include <cstdio>

#include "decoder_ops.h"
#include "elementwise.h"
#include "gemm_host.h"

using namespace kai;

#define KAI_REQUIRE_PTR(p) KAI_REQUIRE((p) != nullptr, KAI_ERR_INVALID_POINTER, "null pointer: " #p)
#define KAI_REQUIRE_DIM(v) \
    KAI_REQUIRE((v) >= 0 && (v) <= kMaxDim, KAI_ERR_INVALID_ARGUMENT, "dimension out of range: " #v)

namespace {

constexpr int64_t kMaxWidth = 1ll << 24;     // floats of a token's heads
constexpr int64_t kMaxRotary = 512;          // rotated elements of a head
constexpr int64_t kMaxAttentionPiece = 256;
constexpr int64_t kMaxReach = 1ll << 30;           // keys of a sequence: indices a few tiles further on still fit 32 bits
constexpr int64_t kMaxAttentionRows = 1ll << 25;   // a wave each: the threads of a launch stay below 2^32

int rotary_params(const char* who, const kai_rotary_desc* desc, int64_t npiece, RotaryParams* out) {
    RotaryParams r{};
    r.inv_factor = 1.0;
    r.magnitude = 1.0f;
    *out = r;
    if (desc == nullptr) return KAI_OK;
    const std::string name = who;
    const auto bad = [&](const char* text) { return fail(KAI_ERR_INVALID_ARGUMENT, name + ": rotary: " + text); };
    if (desc->nrot < 0 || desc->nrot % 2 != 0 || desc->nrot > npiece) return bad("nrot must be even, 0 .. npiece");
    if (desc->nrot > kMaxRotary) return bad("nrot above 512");
    if (desc->layout != KAI_ROTARY_HALVES && desc->layout != KAI_ROTARY_PAIRS) return bad("unknown layout");
    if (desc->nrot == 0) return KAI_OK;
    // comparisons that a NaN fails as well
    if (!(desc->base > 0.0 && std::isfinite(desc->base))) return bad("base must be positive and finite");
    if (!std::isfinite((float)desc->magnitude)) return bad("magnitude must be finite, in 32 bits too");
    const bool scaled = desc->scaling != KAI_ROTARY_SCALE_NONE;
    if (scaled && !(desc->factor > 0.0 && std::isfinite(desc->factor) && std::isfinite(1.0 / desc->factor)))
        return bad("factor must be positive and finite, and so must its inverse");
    double log2_base = std::log2(desc->base);
    switch (desc->scaling) {
    case KAI_ROTARY_SCALE_NONE:
        break;
    case KAI_ROTARY_SCALE_LINEAR:
        r.inv_factor = 1.0 / desc->factor;
        break;
    case KAI_ROTARY_SCALE_BASE:
        // the last pair turns `factor` times slower, the first as before; a single pair stays as it is
        if (desc->nrot > 2) log2_base += std::log2(desc->factor) * (double)desc->nrot / (double)(desc->nrot - 2);
        break;
    case KAI_ROTARY_SCALE_PARTS:
        if (!(desc->trained > 0.0 && std::isfinite(desc->trained))) return bad("trained length must be positive and finite");
        if (!(desc->low_turns < desc->high_turns && std::isfinite(desc->low_turns) && std::isfinite(desc->high_turns)))
            return bad("low_turns must be below high_turns");
        r.inv_factor = 1.0 / desc->factor;
        r.parts = 1;
        r.low = desc->low_turns;
        r.inv_span = 1.0 / (desc->high_turns - desc->low_turns);
        r.trained_turns = desc->trained * 0.15915494309189533577;
        if (!(r.inv_span > 0.0 && std::isfinite(r.inv_span))) return bad("low_turns and high_turns too near or too far apart");
        break;
    default:
        return bad("unknown scaling");
    }
    r.step = -2.0 * log2_base / (double)desc->nrot;
    // the fastest pair's angle at position 2^31 has to be a number (a base below 1 turns the last pair fastest)
    const double fastest = std::fmax(0.0, r.step * (double)(desc->nrot / 2 - 1)) + std::fmax(0.0, std::log2(r.inv_factor));
    if (!(fastest + 31.0 < 1000.0)) return bad("angles out of range");
    r.magnitude = (float)desc->magnitude;
    r.nrot = (int)desc->nrot;
    r.pairs = desc->layout == KAI_ROTARY_PAIRS;
    *out = r;
    return KAI_OK;
}

int check_head_rows(const char* who, int64_t nbat, int64_t ntimes, int64_t nvec, int64_t nhead, int64_t npiece) {
    const std::string name = who;
    if (nbat < 0 || ntimes < 0 || nvec < 0 || nhead < 0 || npiece < 0)
        return fail(KAI_ERR_INVALID_ARGUMENT, name + ": negative dimension");
    if (nbat > kMaxDim || ntimes > kMaxDim || nvec > kMaxDim || nhead > kMaxWidth || npiece > kMaxWidth ||
        nhead * npiece > kMaxWidth)
        return fail(KAI_ERR_INVALID_ARGUMENT, name + ": dimension out of range");
    if (nhead * npiece > nvec) return fail(KAI_ERR_INVALID_ARGUMENT, name + ": nhead * npiece exceeds nvec");
    if (nbat * ntimes > kMaxDim) return fail(KAI_ERR_INVALID_ARGUMENT, name + ": nbat * ntimes out of range");
    return KAI_OK;
}

int rotate(const char* who, float* py, const float* px, const int* ppos, int64_t nbat, int64_t ntimes, int64_t nvec,
           int64_t nhead, int64_t npiece, const kai_rotary_desc* desc, bool back) {
    KAI_TRY(check_head_rows(who, nbat, ntimes, nvec, nhead, npiece));
    RotaryArgs a{};
    KAI_TRY(rotary_params(who, desc, npiece, &a.rot));
    if (desc == nullptr) return fail(KAI_ERR_INVALID_POINTER, std::string(who) + ": null pointer: desc");
    if (nbat == 0 || ntimes == 0 || nhead == 0 || npiece == 0) return KAI_OK;
    if (py == nullptr || px == nullptr) return fail(KAI_ERR_INVALID_POINTER, std::string(who) + ": null pointer: data");
    if (py == px && a.rot.nrot == 0) return KAI_OK;
    a.y = py; a.x = px; a.pos = ppos;
    a.ntok = nbat * ntimes; a.ntimes = ntimes; a.ld = nvec;
    a.nhead = (int)nhead; a.npiece = (int)npiece;
    a.back = back;
    return launch_rotary(a, current_stream());
}

int cache_pages(const char* who, CachePages* c, const int* ppage, const int* plen, const int* pcount, int64_t nbat,
                int64_t ntimes, int64_t nkvhead, int64_t npiece, int64_t npage, int64_t npagelen, int64_t nmaxpage) {
    const std::string name = who;
    if (nkvhead < 0 || npage < 0 || npagelen < 0 || nmaxpage < 0)
        return fail(KAI_ERR_INVALID_ARGUMENT, name + ": negative dimension");
    if (nkvhead > kMaxWidth || nkvhead * npiece > kMaxWidth || npage > kMaxDim || npagelen > kMaxDim || nmaxpage > kMaxDim ||
        npagelen * nmaxpage > kMaxReach || npage * npagelen > kMaxDim)
        return fail(KAI_ERR_INVALID_ARGUMENT, name + ": dimension out of range");
    if (ppage == nullptr && (nmaxpage > 1 || npage < nbat))
        return fail(KAI_ERR_INVALID_ARGUMENT, name + ": without a page table each sequence has one page, its own");
    c->table = ppage; c->len = plen; c->count = pcount;
    // no page, no key: a kernel reads row 0 in place of a key that does not exist, so one must be there where keys are
    c->nbat = nbat; c->ntimes = ntimes; c->npage = npage; c->page = npagelen; c->nmaxpage = npage > 0 ? nmaxpage : 0;
    c->nkvhead = (int)nkvhead; c->npiece = (int)npiece;
    return KAI_OK;
}

bool overlap(const void* p, int64_t np, const void* q, int64_t nq) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return a < b + (uintptr_t)nq && b < a + (uintptr_t)np;
}

}  // namespace

extern "C" {

int kai_rotary(int device, float* py, const float* px, const int* ppos, int64_t nbat, int64_t ntimes, int64_t nvec,
               int64_t nhead, int64_t npiece, const kai_rotary_desc* desc) {
    KAI_REQUIRE_DEVICE(device);
    return rotate(__func__, py, px, ppos, nbat, ntimes, nvec, nhead, npiece, desc, false);
}

int kai_rotary_backward(int device, float* pgx, const float* pgy, const int* ppos, int64_t nbat, int64_t ntimes,
                        int64_t nvec, int64_t nhead, int64_t npiece, const kai_rotary_desc* desc) {
    KAI_REQUIRE_DEVICE(device);
    return rotate(__func__, pgx, pgy, ppos, nbat, ntimes, nvec, nhead, npiece, desc, true);
}

int kai_cache_append(int device, float* pcK, float* pcV, const float* pK, const float* pV, const int* ppage,
                     const int* plen, const int* pcount, const int* ppos, int64_t nbat, int64_t ntimes, int64_t nvec,
                     int64_t nkvhead, int64_t npiece, int64_t npage, int64_t npagelen, int64_t nmaxpage,
                     const kai_rotary_desc* desc) {
    KAI_REQUIRE_DEVICE(device);
    KAI_TRY(check_head_rows(__func__, nbat, ntimes, nvec, nkvhead, npiece));
    CacheAppendArgs a{};
    KAI_TRY(cache_pages(__func__, &a.pages, ppage, plen, pcount, nbat, ntimes, nkvhead, npiece, npage, npagelen, nmaxpage));
    KAI_TRY(rotary_params(__func__, desc, npiece, &a.rot));
    if (nbat == 0 || ntimes == 0 || nkvhead == 0 || npiece == 0) return KAI_OK;
    if (npage == 0 || npagelen == 0 || nmaxpage == 0) return KAI_OK;   // a cache of no rows takes nothing
    KAI_REQUIRE_PTR(pcK); KAI_REQUIRE_PTR(pcV); KAI_REQUIRE_PTR(pK); KAI_REQUIRE_PTR(pV); KAI_REQUIRE_PTR(plen);
    a.ck = pcK; a.cv = pcV; a.k = pK; a.v = pV; a.pos = ppos; a.ld = nvec;
    return launch_cache_append(a, current_stream());
}

int kai_cache_attention(int device, float* py, const float* pQ, const float* pcK, const float* pcV, const int* ppage,
                        const int* plen, const int* pcount, const int* pmask, int64_t nbat, int64_t ntimes, int64_t nvec,
                        int64_t nhead, int64_t nkvhead, int64_t npiece, int64_t npage, int64_t npagelen, int64_t nmaxpage,
                        const float* hCoef) {
    KAI_REQUIRE_DEVICE(device);
    KAI_TRY(check_head_rows(__func__, nbat, ntimes, nvec, nhead, npiece));
    CacheAttentionArgs a{};
    KAI_TRY(cache_pages(__func__, &a.pages, ppage, plen, pcount, nbat, ntimes, nkvhead, npiece, npage, npagelen, nmaxpage));
    KAI_REQUIRE(npiece <= kMaxAttentionPiece, KAI_ERR_INVALID_ARGUMENT, "npiece above 256");
    if (nbat == 0 || ntimes == 0 || nhead == 0 || npiece == 0) return KAI_OK;
    KAI_REQUIRE(nkvhead > 0 && nhead % nkvhead == 0, KAI_ERR_INVALID_ARGUMENT, "nhead must be a multiple of nkvhead");
    KAI_REQUIRE(nbat * ntimes <= kMaxAttentionRows / nhead, KAI_ERR_INVALID_ARGUMENT, "nbat * ntimes * nhead above 2^25");
    KAI_REQUIRE_PTR(py); KAI_REQUIRE_PTR(pQ); KAI_REQUIRE_PTR(plen);
    if (npage > 0 && npagelen > 0 && nmaxpage > 0) { KAI_REQUIRE_PTR(pcK); KAI_REQUIRE_PTR(pcV); }
    KAI_REQUIRE(!overlap(py, nbat * ntimes * nhead * npiece * 4, pQ, ((nbat * ntimes - 1) * nvec + nhead * npiece) * 4),
                KAI_ERR_INVALID_ARGUMENT, "the result overlaps the queries");
    a.y = py; a.q = pQ; a.ck = pcK; a.cv = pcV; a.mask = pmask; a.ldq = nvec; a.nhead = (int)nhead; a.hcoef = hCoef;
    return launch_cache_attention(a, current_stream());
}

int kai_gated_forward(int device, float* py, float* pgate, float* pup, const float* pwg, const float* pwu,
                      const float* pbg, const float* pbu, const float* px, int64_t yvec, int64_t ndat, int64_t xvec,
                      int actFunc, const float* hLeakyAlpha) {
    KAI_REQUIRE_DEVICE(device);
    KAI_REQUIRE_DIM(yvec); KAI_REQUIRE_DIM(ndat); KAI_REQUIRE_DIM(xvec);
    KAI_REQUIRE(actFunc >= KAI_ACT_NONE && actFunc <= KAI_ACT_SWISH, KAI_ERR_CONDITIONAL_STATEMENT, "activation code must be 0..8");
    KAI_REQUIRE((pgate == nullptr) == (pup == nullptr), KAI_ERR_INVALID_POINTER, "pgate and pup come together");
    if (ndat == 0 || yvec == 0) return KAI_OK;
    KAI_REQUIRE_PTR(py);
    if (xvec > 0) { KAI_REQUIRE_PTR(pwg); KAI_REQUIRE_PTR(pwu); KAI_REQUIRE_PTR(px); }
    GatedArgs a{};
    a.y = py; a.gate = pgate; a.up = pup; a.wg = pwg; a.wu = pwu; a.bg = pbg; a.bu = pbu; a.x = px;
    a.yvec = yvec; a.ndat = ndat; a.xvec = xvec; a.act = actFunc; a.hleaky = hLeakyAlpha;
    return launch_gated_forward(a, current_stream());
}

int kai_gated_backward(int device, float* pgx, float* pgwg, float* pgwu, float* pgbg, float* pgbu, float* pga_work,
                       const float* pgy, const float* pwg, const float* pwu, const float* px, const float* pgate,
                       const float* pup, int64_t yvec, int64_t ndat, int64_t xvec, int actFunc, const float* hLeakyAlpha,
                       int acc) {
    KAI_REQUIRE_DEVICE(device);
    KAI_REQUIRE_DIM(yvec); KAI_REQUIRE_DIM(ndat); KAI_REQUIRE_DIM(xvec);
    KAI_REQUIRE(actFunc >= KAI_ACT_NONE && actFunc <= KAI_ACT_SWISH, KAI_ERR_CONDITIONAL_STATEMENT, "activation code must be 0..8");
    const int64_t n = ndat * yvec;
    if (n > 0) { KAI_REQUIRE_PTR(pgy); KAI_REQUIRE_PTR(pgate); KAI_REQUIRE_PTR(pup); }
    if (pgx && n > 0 && xvec > 0) { KAI_REQUIRE_PTR(pwg); KAI_REQUIRE_PTR(pwu); }
    if ((pgwg || pgwu) && n > 0 && xvec > 0) KAI_REQUIRE_PTR(px);
    float* work = pga_work;
    int64_t held_bytes = 0;
    if (n > 0) {
        if (work == nullptr) {
            held_bytes = 2 * n * (int64_t)sizeof(float);
            KAI_TRY(workspace(held_bytes, &work));
        }
    }
    ScratchHold held(held_bytes);
    if (n > 0) {
        KAI_TRY(launch_gated_activation_backward(work, work + n, pgbg, pgbu, pgy, pgate, pup, ndat, yvec, actFunc, hLeakyAlpha,
                                                 acc != 0, current_stream()));
    } else {
        if (pgbg) KAI_TRY(kai_add_bias_backward_b(device, pgbg, nullptr, ndat, yvec, acc));
        if (pgbu) KAI_TRY(kai_add_bias_backward_b(device, pgbu, nullptr, ndat, yvec, acc));
    }
    GatedGradArgs a{};
    a.gx = pgx; a.gwg = pgwg; a.gwu = pgwu;
    a.ggate = work; a.gup = n > 0 ? work + n : nullptr;
    a.wg = pwg; a.wu = pwu; a.x = px;
    a.yvec = yvec; a.ndat = ndat; a.xvec = xvec; a.acc = acc != 0;
    return launch_gated_gradients(a, current_stream());
}

int kai_cache_attention_plan(int64_t nbat, int64_t ntimes, int64_t nhead, int64_t nkvhead, int64_t npiece, int64_t npagelen,
                             int64_t nmaxpage, char* out, int buflen) {
    KAI_REQUIRE_PTR(out);
    KAI_REQUIRE(buflen > 0, KAI_ERR_INVALID_ARGUMENT, "buflen <= 0");
    KAI_TRY(check_head_rows(__func__, nbat, ntimes, kMaxWidth, nhead, npiece));
    const int some = 0;      // the table is not read
    CachePages c{};
    KAI_TRY(cache_pages(__func__, &c, &some, nullptr, nullptr, nbat, ntimes, nkvhead, npiece, 1, npagelen, nmaxpage));
    KAI_REQUIRE(npiece <= kMaxAttentionPiece, KAI_ERR_INVALID_ARGUMENT, "npiece above 256");
    std::string text = "nothing";
    if (nbat > 0 && ntimes > 0 && nhead > 0 && npiece > 0) {
        KAI_REQUIRE(nkvhead > 0 && nhead % nkvhead == 0, KAI_ERR_INVALID_ARGUMENT, "nhead must be a multiple of nkvhead");
        KAI_REQUIRE(nbat * ntimes <= kMaxAttentionRows / nhead, KAI_ERR_INVALID_ARGUMENT, "nbat * ntimes * nhead above 2^25");
        CacheAttentionPlan plan;
        KAI_TRY(cache_attention_plan(c, (int)nhead, &plan));
        text = plan.row_tile > 0 ? "tiles of " + std::to_string(plan.row_tile) + " rows" : std::string("a wave a row");
        text += ", " + std::to_string(plan.nsplit) + (plan.nsplit == 1 ? " part" : " parts") + ", scratch " + std::to_string(plan.scratch);
    }
    snprintf(out, (size_t)buflen, "%s", text.c_str());
    return KAI_OK;
}

int kai_gated_plan(int which, int64_t yvec, int64_t ndat, int64_t xvec, char* out, int buflen) {
    KAI_REQUIRE_PTR(out);
    KAI_REQUIRE(buflen > 0, KAI_ERR_INVALID_ARGUMENT, "buflen <= 0");
    KAI_REQUIRE(which >= 0 && which <= 2, KAI_ERR_INVALID_ARGUMENT, "which must be 0..2");
    KAI_REQUIRE_DIM(yvec); KAI_REQUIRE_DIM(ndat); KAI_REQUIRE_DIM(xvec);
    const std::string text = yvec == 0 || ndat == 0 ? "nothing" : gated_plan_text(which, yvec, ndat, xvec);
    snprintf(out, (size_t)buflen, "%s", text.c_str());
    return KAI_OK;
}

}  // extern "C"
