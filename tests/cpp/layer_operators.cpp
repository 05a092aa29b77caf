// The layer operators through the C++ host interface
// (hephaestus_amd/host/hephaestus.hpp): small cases of exact values, immediate
// and prepared, and their refusals.
//
// Exit status: 0 when every check passes, 1 otherwise, 77 when no GPU is
// present (the usual "skipped" code).
#include "../../hephaestus_amd/host/hephaestus.hpp"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <vector>

using namespace hephaestus;

namespace {

int g_failures = 0;
int g_checks = 0;

#define CHECK(cond)                                                                                        \
    do {                                                                                                   \
        ++g_checks;                                                                                        \
        if (!(cond)) {                                                                                     \
            ++g_failures;                                                                                  \
            std::printf("  FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);                                  \
        }                                                                                                  \
    } while (0)

template <typename F> void expect_refusal(const char *text, F &&f) {
    ++g_checks;
    try {
        f();
    } catch (const Error &e) {
        if (std::strstr(e.what(), text)) return;
        std::printf("  FAIL: got \"%s\", expected \"%s\"\n", e.what(), text);
        ++g_failures;
        return;
    }
    std::printf("  FAIL: expected a refusal with \"%s\"\n", text);
    ++g_failures;
}

std::vector<Bfloat16> bf16(std::initializer_list<float> values) {
    std::vector<Bfloat16> v;
    for (float f : values) v.emplace_back(f);
    return v;
}

void bfloat16_values(RocmDevice &) {
    CHECK(Bfloat16(1.0f).bits == 0x3F80);
    CHECK(Bfloat16(1.0f + 0x1p-8f).bits == 0x3F80); // a tie, to even
    CHECK(Bfloat16(1.0f + 0x1.8p-7f).bits == 0x3F82);
    CHECK(Bfloat16(-INFINITY).bits == 0xFF80);
    CHECK(std::isnan((float)Bfloat16(NAN)));
    CHECK((float)Bfloat16(-3.5f) == -3.5f);
}

// h = x + r = {3, -4, 0, 5}, largest |h w| 5 at the last element.
void norm(RocmDevice &dev) {
    const RocmNormOps ops;
    const Layout row = Layout::c_contiguous({1, 4});
    auto x = dev.upload(bf16({1, -6, 0, 2})), r = dev.upload(bf16({2, 2, 0, 3})), w = dev.upload(bf16({1, 1, 1, 1}));
    auto h = dev.alloc_zeroed<Bfloat16>(4);
    auto q = dev.alloc_zeroed<int8_t>(4);
    auto s = dev.alloc_zeroed<float>(1);
    const std::vector<int8_t> want{76, -102, 0, 127}; // 3/5 and -4/5 of 127
    const double scale = 5.0 / std::sqrt(12.5) / 127;
    const auto right = [&] {
        const auto hv = dev.download_owned(h);
        CHECK((float)hv[0] == 3 && (float)hv[1] == -4 && (float)hv[2] == 0 && (float)hv[3] == 5);
        CHECK(dev.download_owned(q) == want);
        CHECK(std::fabs(dev.download_owned(s)[0] - scale) < 4e-7 * scale);
    };
    ops.rms_norm_quantize_into(dev, StridedView<Bfloat16>{x, row}, w, 0.0f, StridedView<int8_t>{q, row}, s,
                               StridedView<Bfloat16>{r, row}, StridedView<Bfloat16>{h, row});
    right();
    const PreparedPlan plan =
        ops.prepare_rms_norm_quantize(dev, StridedView<Bfloat16>{x, row}, w, 0.0f, StridedView<int8_t>{q, row}, s,
                                      StridedView<Bfloat16>{r, row}, StridedView<Bfloat16>{h, row});
    for (int i = 0; i < 2; ++i) {
        dev.write_buffer(q, std::vector<int8_t>(4));
        plan.dispatch();
        right();
    }
    // Without a residual, in f32.
    auto xf = dev.upload(std::vector<float>{3, -4, 0, 5}), wf = dev.upload(std::vector<float>{1, 1, 1, 1});
    ops.rms_norm_quantize_into(dev, StridedView<float>{xf, row}, wf, 0.0f, StridedView<int8_t>{q, row}, s);
    right();
    auto narrow = dev.alloc_zeroed<float>(3);
    expect_refusal("host length 4 does not match device buffer length 3", [&] {
        ops.rms_norm_quantize_into(dev, StridedView<float>{xf, row}, narrow, 0.0f, StridedView<int8_t>{q, row}, s);
    });
}

void product(RocmDevice &dev) {
    const RocmMatrixOps ops;
    const Layout a_rows = Layout::c_contiguous({2, 3}), b_rows = Layout::c_contiguous({4, 3}),
                 out_rows = Layout::c_contiguous({2, 4});
    auto a = dev.upload(std::vector<int8_t>{1, 2, 3, -128, 0, 127});
    auto b = dev.upload(std::vector<int8_t>{1, 0, 0, 0, 1, 0, 1, 1, 1, -128, 5, 127});
    auto sa = dev.upload(std::vector<float>{0.5f, 2}), sb = dev.upload(std::vector<float>{1, 2, 4, 8});
    auto out = dev.alloc_zeroed<float>(8);
    const std::vector<float> want{0.5f, 2, 12, 4 * (-128 + 10 + 381), -256, 0, -8, 16 * (16384 + 16129)};
    ops.matmul_i8_into(dev, StridedView<int8_t>{a, a_rows}, sa, StridedView<int8_t>{b, b_rows}, sb,
                       StridedView<float>{out, out_rows});
    CHECK(dev.download_owned(out) == want);
    const PreparedPlan plan = ops.prepare_matmul_i8(dev, StridedView<int8_t>{a, a_rows}, sa,
                                                    StridedView<int8_t>{b, b_rows}, sb, StridedView<float>{out, out_rows});
    dev.write_buffer(out, std::vector<float>(8));
    plan.dispatch();
    CHECK(dev.download_owned(out) == want);
    expect_refusal("host length 2 does not match device buffer length 4", [&] {
        ops.matmul_i8_into(dev, StridedView<int8_t>{a, a_rows}, sb, StridedView<int8_t>{b, b_rows}, sb,
                           StridedView<float>{out, out_rows});
    });
}

// One head, no decay, q = k = the unit vectors in turn: o_t = sum of the v_s at
// equal unit vectors, and the state's rows are those sums.
void attention(RocmDevice &dev) {
    const RocmLinearAttentionOps ops;
    const uint64_t tokens = 70; // a chunk and more
    const Layout rows = Layout::c_contiguous({1, tokens, 1, 2}), state = Layout::c_contiguous({1, 1, 2, 2});
    std::vector<float> unit, value, want;
    double sums[2][2] = {{1, 2}, {3, 4}};
    for (uint64_t t = 0; t < tokens; ++t) {
        const int e = t % 2;
        for (int c = 0; c < 2; ++c) {
            unit.push_back(c == e ? 1.0f : 0.0f);
            value.push_back((float)(t + c));
            sums[e][c] += (double)(t + c);
        }
        for (int c = 0; c < 2; ++c) want.push_back((float)(2 * sums[e][c]));
    }
    auto qk = dev.upload(unit), v = dev.upload(value), g = dev.upload(std::vector<float>{0});
    auto s = dev.upload(std::vector<float>{1, 2, 3, 4}), out = dev.alloc_zeroed<float>(tokens * 2);
    const std::vector<float> last{(float)sums[0][0], (float)sums[0][1], (float)sums[1][0], (float)sums[1][1]};
    const StridedView<float> vqk{qk, rows}, vv{v, rows}, vo{out, rows}, vs{s, state};
    ops.linear_attention_into(dev, vqk, vqk, vv, g, vo, 2.0f, vs, vs);
    CHECK(dev.download_owned(out) == want);
    CHECK(dev.download_owned(s) == last);
    // No tokens: the state stays, the outputs are zeros.
    auto none = dev.upload(std::vector<uint32_t>{0});
    const PreparedPlan plan = ops.prepare_linear_attention(dev, vqk, vqk, vv, g, vo, 2.0f, vs, vs, &none);
    plan.dispatch();
    CHECK(dev.download_owned(out) == std::vector<float>(tokens * 2));
    CHECK(dev.download_owned(s) == last);
    expect_refusal("scale", [&] { ops.linear_attention_into(dev, vqk, vqk, vv, g, vo, INFINITY); });
}

} // namespace

int main() {
    int32_t count = 0;
    if (hx_device_count(&count) != HX_OK || count == 0) {
        std::printf("no ROCm device: skipped\n");
        return 77;
    }
    RocmDevice dev = RocmDevice::try_default();
    const std::pair<const char *, std::function<void(RocmDevice &)>> clauses[] = {
        {"bfloat16", bfloat16_values},
        {"norm", norm},
        {"product", product},
        {"attention", attention},
    };
    for (const auto &c : clauses) {
        const int before = g_failures;
        try {
            c.second(dev);
        } catch (const Error &e) {
            ++g_failures;
            std::printf("  FAIL: unexpected error kind %d: %s\n", (int)e.kind(), e.what());
        }
        std::printf("%-20s %s\n", c.first, g_failures == before ? "ok" : "FAILED");
        std::fflush(stdout);
    }
    std::printf("%d checks, %d failures\n", g_checks, g_failures);
    return g_failures == 0 ? 0 : 1;
}
