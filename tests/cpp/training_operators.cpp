// The training operators through the C++ host interface
// (hephaestus_amd/host/hephaestus.hpp): small cases with results that can be
// written down, immediate and prepared, and their refusals.
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

// Each value within a few roundings of f32 of what is wanted.
bool near(const std::vector<float> &got, const std::vector<double> &want) {
    if (got.size() != want.size()) return false;
    for (size_t i = 0; i < got.size(); ++i)
        if (!(std::fabs(got[i] - want[i]) <= 1e-6 * (1 + std::fabs(want[i])))) return false;
    return true;
}

// h = x + r = {1, -1, 3, -3}: mean 0, mean square 5.
void norm(RocmDevice &dev) {
    const RocmLayerNormOps ops;
    const Layout row = Layout::c_contiguous({1, 4});
    auto x = dev.upload(std::vector<float>{1, 0, 2, -3}), r = dev.upload(std::vector<float>{0, -1, 1, 0});
    auto w = dev.upload(std::vector<float>{1, 2, 1, 1}), b = dev.upload(std::vector<float>{0, 0, 10, 0});
    auto y = dev.alloc_zeroed<float>(4), h = dev.alloc_zeroed<float>(4);
    auto mean = dev.upload(std::vector<float>{7}), rstd = dev.upload(std::vector<float>{7});
    const double s = 1 / std::sqrt(5.0);
    const RocmLayerNormOps::Forward<float> forward{
        {x, row}, w, &b, 0.0f, {y, row}, StridedView<float>{r, row}, StridedView<float>{h, row}, &mean, &rstd};
    const auto right = [&] {
        CHECK((dev.download_owned(h) == std::vector<float>{1, -1, 3, -3}));
        CHECK(near(dev.download_owned(y), {s, -2 * s, 3 * s + 10, -3 * s}));
        CHECK(near(dev.download_owned(mean), {0}) && near(dev.download_owned(rstd), {s}));
    };
    ops.layer_norm_into(dev, forward);
    right();
    dev.write_buffer(y, std::vector<float>(4));
    ops.prepare_layer_norm(dev, forward).dispatch();
    right();
    // dy = {1, 0, 0, 0}: t = dy·w, u = h·s.
    auto dy = dev.upload(std::vector<float>{1, 0, 0, 0}), dx = dev.alloc_zeroed<float>(4);
    auto dw = dev.alloc_zeroed<float>(4), db = dev.alloc_zeroed<float>(4);
    const RocmLayerNormOps::Backward<float> backward{{dy, row}, {h, row}, w, mean, rstd, {dx, row}, {}, &dw, &db};
    ops.layer_norm_backward_into(dev, backward);
    const double mt = 0.25, mtu = s / 4;
    CHECK(near(dev.download_owned(dx), {s * (1 - mt - s * mtu), s * (-mt + s * mtu), s * (-mt - 3 * s * mtu),
                                        s * (-mt + 3 * s * mtu)}));
    CHECK(near(dev.download_owned(dw), {s, 0, 0, 0}));
    CHECK(near(dev.download_owned(db), {1, 0, 0, 0}));
    dev.write_buffer(dw, std::vector<float>(4, 3.0f));
    ops.prepare_layer_norm_backward(dev, backward).dispatch();
    CHECK(near(dev.download_owned(dw), {s, 0, 0, 0}));
    auto narrow = dev.alloc_zeroed<float>(3);
    expect_refusal("host length 4 does not match device buffer length 3",
                   [&] { ops.layer_norm_into(dev, RocmLayerNormOps::Forward<float>{{x, row}, narrow, nullptr, 0.0f, {y, row}}); });
}

// Gates of 0: f = 1/2, so that h halves the way to x each token.
void recurrence(RocmDevice &dev) {
    const RocmRecurrenceOps ops;
    const uint64_t tokens = 40;
    const Layout rows = Layout::c_contiguous({1, tokens, 1}), state = Layout::c_contiguous({1, 1});
    std::vector<float> ones(tokens, 1.0f);
    std::vector<double> want, grad;
    for (uint64_t t = 0; t < tokens; ++t) want.push_back(1 + 3 * std::pow(0.5, (double)t + 1)); // from 4 towards 1
    auto gate = dev.alloc_zeroed<float>(tokens), x = dev.upload(ones), h = dev.alloc_zeroed<float>(tokens);
    auto first = dev.upload(std::vector<float>{4}), last = dev.alloc_zeroed<float>(1);
    const RocmRecurrenceOps::Forward<float> forward{
        {gate, rows}, {x, rows}, {h, rows}, StridedView<float>{first, state}, StridedView<float>{last, state}};
    ops.gated_recurrence_into(dev, forward);
    CHECK(near(dev.download_owned(h), want) && near(dev.download_owned(last), {want.back()}));
    dev.write_buffer(h, std::vector<float>(tokens));
    ops.prepare_gated_recurrence(dev, forward).dispatch();
    CHECK(near(dev.download_owned(h), want));
    // The last state's gradient alone, 1: halved at each token.
    auto dy = dev.alloc_zeroed<float>(tokens), dz = dev.alloc_zeroed<float>(tokens), dx = dev.alloc_zeroed<float>(tokens);
    auto after = dev.upload(std::vector<float>{1}), before = dev.alloc_zeroed<float>(1);
    const RocmRecurrenceOps::Backward<float> backward{{gate, rows},
                                                      {x, rows},
                                                      {h, rows},
                                                      {dy, rows},
                                                      {dz, rows},
                                                      {dx, rows},
                                                      StridedView<float>{first, state},
                                                      StridedView<float>{after, state},
                                                      StridedView<float>{before, state}};
    ops.gated_recurrence_backward_into(dev, backward);
    std::vector<double> want_x, want_z;
    for (uint64_t t = 0; t < tokens; ++t) {
        const double g = std::pow(0.5, (double)(tokens - 1 - t)), prev = t ? want[t - 1] : 4;
        want_x.push_back(g / 2);
        want_z.push_back(g / 4 * (prev - 1));
    }
    CHECK(near(dev.download_owned(dx), want_x) && near(dev.download_owned(dz), want_z));
    CHECK(near(dev.download_owned(before), {std::pow(0.5, (double)tokens)}));
    ops.prepare_gated_recurrence_backward(dev, backward).dispatch();
    CHECK(near(dev.download_owned(dx), want_x));
    // No tokens: the state passes, the outputs are zeros.
    auto none = dev.upload(std::vector<uint32_t>{0});
    RocmRecurrenceOps::Forward<float> empty = forward;
    empty.lengths = &none;
    ops.gated_recurrence_into(dev, empty);
    CHECK(dev.download_owned(h) == std::vector<float>(tokens) && dev.download_owned(last)[0] == 4);
    expect_refusal("must not overlap", [&] {
        ops.gated_recurrence_into(dev, RocmRecurrenceOps::Forward<float>{{gate, rows}, {x, rows}, {x, rows}, {}, {}, nullptr});
    });
}

// Two words with logits 0 and log 3: their shares are 1/4 and 3/4.
void loss(RocmDevice &dev) {
    const RocmLossOps ops;
    const Layout x_rows = Layout::c_contiguous({2, 1}), w_rows = Layout::c_contiguous({2, 1});
    const float log3 = std::log(3.0f);
    auto x = dev.upload(std::vector<float>{1, 1}), w = dev.upload(std::vector<float>{0, log3});
    auto targets = dev.upload(std::vector<uint32_t>{0, RocmLossOps::no_target});
    auto out = dev.alloc_zeroed<float>(2), lse = dev.alloc_zeroed<float>(2);
    const RocmLossOps::Forward<float> forward{{x, x_rows}, {w, w_rows}, targets, out, &lse};
    ops.linear_cross_entropy_into(dev, forward);
    CHECK(near(dev.download_owned(out), {std::log(4.0), 0}));
    CHECK(near(dev.download_owned(lse), {std::log(4.0), std::log(4.0)}));
    ops.prepare_linear_cross_entropy(dev, forward).dispatch();
    CHECK(near(dev.download_owned(out), {std::log(4.0), 0}));
    auto grad = dev.upload(std::vector<float>{2, 2}), dx = dev.upload(std::vector<float>{5, 5}),
         dw = dev.upload(std::vector<float>{5, 5});
    const RocmLossOps::Backward<float> backward{
        {x, x_rows}, {w, w_rows}, targets, lse, grad, StridedView<float>{dx, x_rows}, StridedView<float>{dw, w_rows}};
    ops.linear_cross_entropy_backward_into(dev, backward);
    CHECK(near(dev.download_owned(dx), {2 * 0.75 * log3, 0}) && near(dev.download_owned(dw), {-1.5, 1.5}));
    dev.write_buffer(dw, std::vector<float>{5, 5});
    ops.prepare_linear_cross_entropy_backward(dev, backward).dispatch();
    CHECK(near(dev.download_owned(dw), {-1.5, 1.5}));
    auto bx = dev.upload(std::vector<Bfloat16>{Bfloat16(1.0f), Bfloat16(1.0f)}),
         bw = dev.upload(std::vector<Bfloat16>{Bfloat16(0.0f), Bfloat16(0.0f)});
    ops.linear_cross_entropy_into(dev, RocmLossOps::Forward<Bfloat16>{{bx, x_rows}, {bw, w_rows}, targets, out});
    CHECK(near(dev.download_owned(out), {std::log(2.0), 0}));
    auto few = dev.alloc_zeroed<uint32_t>(1);
    expect_refusal("host length 2 does not match device buffer length 1",
                   [&] { ops.linear_cross_entropy_into(dev, RocmLossOps::Forward<float>{{x, x_rows}, {w, w_rows}, few, out}); });
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
        {"norm", norm},
        {"recurrence", recurrence},
        {"loss", loss},
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
