// Test driver for the decoder block's methods of the C++ operator mirror (include/vmath_hip.h), called as engine code calls
// VMath.  Built with the host compiler against libkai_hip.so (tests/Makefile), started by tests/test_decoder_mirror.py.
//
//   decoder_mirror_driver cpu    refused calls and their codes, no GPU
//   decoder_mirror_driver gpu    one token through rotary, cache, attention and the gated projection, values that are exact
//
// Exit status 0 = every check passed; each check prints one line.
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "kai_hip.h"
#include "vmath_hip.h"

static int g_failed = 0;

static void report(bool ok, const std::string& what) {
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", what.c_str());
    std::fflush(stdout);
    if (!ok) g_failed++;
}

template <class F>
static void expect_error(int code, const std::string& what, F call) {
    try {
        call();
        report(false, what + ": no exception");
    } catch (const KaiMathError& e) {
        report(e.code() == code && std::strlen(e.what()) > 0, what + ": KaiMathError " + std::to_string(e.code()));
    }
}

static float* on_device(const std::vector<float>& v) {
    float* p = (float*)VMath::mem_alloc(0, (int64)(v.size() * sizeof(float)));
    VMath::memcpy_from_host(0, p, (void*)v.data(), (int64)(v.size() * sizeof(float)));
    return p;
}

static bool holds(float* p, const std::vector<float>& want) {
    std::vector<float> got(want.size());
    VMath::memcpy_to_host(0, got.data(), p, (int64)(want.size() * sizeof(float)));
    return got == want;
}

static kai_rotary_desc plain_rotary(int64_t nrot) {
    kai_rotary_desc d{};
    d.nrot = nrot;
    d.base = 10000.0;
    d.magnitude = 1.0;
    return d;
}

static void cpu_checks() {
    float* p = (float*)4096;     // never read by a refused call
    int* n = (int*)4096;
    const kai_rotary_desc d = plain_rotary(4), odd = plain_rotary(3);
    expect_error(510, "rotary on device -1", [&] { VMath::rotary(-1, p, p, nullptr, 1, 1, 8, 2, 4, &d); });
    expect_error(510, "rotary of an odd count", [&] { VMath::rotary(0, p, p, nullptr, 1, 1, 8, 2, 4, &odd); });
    expect_error(523, "rotary_backward with a null gradient", [&] { VMath::rotary_backward(0, p, nullptr, nullptr, 1, 1, 8, 2, 4, &d); });
    expect_error(523, "cache_append without lengths", [&] { VMath::cache_append(0, p, p, p, p, n, nullptr, nullptr, nullptr, 1, 1, 8, 2, 4, 1, 16, 1, &d); });
    expect_error(510, "cache_attention of heads that do not divide", [&] { VMath::cache_attention(0, p, p + 64, p, p, n, n, nullptr, nullptr, 1, 1, 12, 3, 2, 4, 1, 16, 1, nullptr); });
    expect_error(523, "gated_forward with one kept sum", [&] { VMath::gated_forward(0, p, p, nullptr, p, p, nullptr, nullptr, p, 4, 2, 3, 0, nullptr); });
    expect_error(8, "gated_backward with code 9", [&] { VMath::gated_backward(0, p, p, p, p, p, p, p, p, p, p, p, p, 4, 2, 3, 9, nullptr, false); });
}

static void gpu_checks() {
    const kai_rotary_desc d = plain_rotary(4);
    const std::vector<float> k = {1, 2, 3, 4, 5, 6, 7, 8}, v = {8, -7, 6, -5, 4, -3, 2, -1}, zero(8, 0.0f);
    float *dk = on_device(k), *dv = on_device(v), *turned = on_device(zero), *y = on_device(zero);
    float *ck = on_device(std::vector<float>(16 * 8, -1.0f)), *cv = on_device(std::vector<float>(16 * 8, -1.0f)), *coef = on_device({0.5f});
    int* len = (int*)on_device({0.0f});      // the bits of 0
    VMath::rotary(0, turned, dk, nullptr, 1, 1, 8, 2, 4, &d);
    report(holds(turned, k), "position 0 turns nothing");
    VMath::rotary_backward(0, turned, turned, nullptr, 1, 1, 8, 2, 4, &d);
    report(holds(turned, k), "nor does its gradient");
    VMath::cache_append(0, ck, cv, dk, dv, nullptr, len, nullptr, nullptr, 1, 1, 8, 2, 4, 1, 16, 1, &d);
    std::vector<float> row(16 * 8, -1.0f);
    std::copy(k.begin(), k.end(), row.begin());
    report(holds(ck, row), "the key stands in row 0, the rest as it was");
    VMath::cache_attention(0, y, dk, ck, cv, nullptr, len, nullptr, nullptr, 1, 1, 8, 2, 2, 4, 1, 16, 1, coef);
    report(holds(y, v), "a token alone sees its own value");
    // x [1, 2] = (1, 2), wg [2, 2] = (1 0; 0 3), wu = (2 1; 1 1): gate (1, 6), up (4, 3)
    float *x = on_device({1, 2}), *wg = on_device({1, 0, 0, 3}), *wu = on_device({2, 1, 1, 1}), *gy = on_device({1, 1});
    float *out = on_device({0, 0}), *gate = on_device({0, 0}), *up = on_device({0, 0}), *gx = on_device({0, 0}), *gwg = on_device({1, 1, 1, 1}), *gbu = on_device({0, 0});
    VMath::gated_forward(0, out, gate, up, wg, wu, nullptr, nullptr, x, 2, 1, 2, 0, nullptr);
    report(holds(out, {4, 18}) && holds(gate, {1, 6}) && holds(up, {4, 3}), "gated_forward");
    // gg = up = (4, 3), gu = gate = (1, 6): gx = gg . wg + gu . wu
    VMath::gated_backward(0, gx, gwg, nullptr, nullptr, gbu, nullptr, gy, wg, wu, x, gate, up, 2, 1, 2, 0, nullptr, true);
    report(holds(gx, {12, 16}) && holds(gwg, {5, 9, 4, 7}) && holds(gbu, {1, 6}), "gated_backward, added to what is there");
    for (void* p : {(void*)dk, (void*)dv, (void*)turned, (void*)y, (void*)ck, (void*)cv, (void*)coef, (void*)len, (void*)x, (void*)wg, (void*)wu, (void*)gy,
                    (void*)out, (void*)gate, (void*)up, (void*)gx, (void*)gwg, (void*)gbu})
        VMath::mem_free(0, p);
}

int main(int argc, char** argv) {
    if (argc != 2) return 2;
    try {
        if (std::strcmp(argv[1], "cpu") == 0) cpu_checks();
        else gpu_checks();
    } catch (const KaiMathError& e) {
        report(false, std::string("exception: ") + e.what());
    }
    if (g_failed == 0) std::printf("all checks passed\n");
    return g_failed;
}
