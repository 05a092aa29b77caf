// Entry points of the training operators (layer norm, gated recurrence,
// softmax cross entropy over a vocabulary, each with its backward pass).  Every
// check runs before the first launch, so a refused call writes nothing.
#include "operand_checks.hpp"

#include <cmath>

using namespace hx;

namespace {

constexpr uint64_t kMost32 = 0x7FFFFFFFull;
// Columns of the sums over rows: 65535 blocks of 1024 f32 in a grid's second dimension.
constexpr uint64_t kMostNormGradCols = 65535ull * 1024;

// An operand as the C ABI takes it.
struct View {
    const void *buf;
    uint64_t len;
    const hx_layout *layout;
};
struct Vector {
    const void *buf;
    uint64_t len;
    bool given() const { return buf || len; }
};

// The operands of a call as they are checked: where each lies, and that no output
// meets another operand but in the ways that were allowed.
class Operands {
  public:
    hx_status in(const View &v, uint32_t rank, const uint64_t *shape, uint32_t size, const char *what) {
        return view(v, rank, shape, size, false, what);
    }
    hx_status out(const View &v, uint32_t rank, const uint64_t *shape, uint32_t size, const char *what) {
        return view(v, rank, shape, size, true, what);
    }
    hx_status in(const Vector &v, uint64_t want, uint32_t size, const char *what) {
        return vector(v, want, size, false, what);
    }
    hx_status out(const Vector &v, uint64_t want, uint32_t size, const char *what) {
        return vector(v, want, size, true, what);
    }
    // The operand that was checked last.
    uint32_t last() const { return n_ - 1; }
    // An output that may be the very view of an input, by their places: views of one
    // call may share a layout.
    void may_be(uint32_t out, uint32_t in) {
        same_[n_same_].out = out;
        same_[n_same_++].in = in;
    }
    hx_status apart() const {
        for (uint32_t i = 0; i < n_; ++i) {
            if (!all_[i].written) continue;
            for (uint32_t j = 0; j < n_; ++j) {
                if (j == i || (all_[j].written && j < i) || !overlap(all_[i].span, all_[j].span)) continue;
                bool allowed = false;
                for (uint32_t s = 0; s < n_same_; ++s)
                    allowed |= same_[s].out == i && same_[s].in == j;
                if (!allowed)
                    return fail(HX_ERR_DISPATCH_FAILED, "%s must not overlap %s", all_[i].what, all_[j].what);
                if (!same_view(all_[i].span, all_[j].span))
                    return fail(HX_ERR_DISPATCH_FAILED, "%s must be the view of %s or not overlap it", all_[i].what,
                                all_[j].what);
            }
        }
        return HX_OK;
    }

  private:
    struct One {
        Span span;
        bool written;
        const char *what;
    };
    static constexpr uint32_t kMost = 12; // operands of a call
    One all_[kMost];
    uint32_t n_ = 0;
    struct {
        uint32_t out, in;
    } same_[4];
    uint32_t n_same_ = 0;

    hx_status view(const View &v, uint32_t rank, const uint64_t *shape, uint32_t size, bool written,
                   const char *what) {
        One o{Span{}, written, what};
        HX_TRY(check_view(v.buf, v.len, v.layout, rank, shape, size, written, what, &o.span));
        all_[n_++] = o;
        return HX_OK;
    }
    hx_status vector(const Vector &v, uint64_t want, uint32_t size, bool written, const char *what) {
        One o{Span{}, written, what};
        HX_TRY(check_vector(v.buf, v.len, want, size, what, &o.span));
        all_[n_++] = o;
        return HX_OK;
    }
};

hx_status check_left_out(const View &v, const char *what) {
    return hx::check_left_out(v.buf, v.len, v.layout, what);
}
// A rank-2 view, f32 whatever the operands' type: [batch, channels].
hx_status check_state(Operands &ops, const View &v, const uint64_t *shape, bool written, const char *what) {
    HX_TRY(check_left_out(v, what));
    if (!v.layout) return HX_OK;
    return written ? ops.out(v, 2, shape, 4, what) : ops.in(v, 2, shape, 4, what);
}

template <typename T = void> T *first_of(const View &v, uint32_t size) {
    return v.layout ? (T *)at(const_cast<void *>(v.buf), v.layout, size) : nullptr;
}
template <typename T = void> T *first_of(const Vector &v) { return v.len ? (T *)const_cast<void *>(v.buf) : nullptr; }
int64_t row_stride(const View &v) { return v.layout ? stride_of(v.layout, 0) : 0; }
SequenceView sequence(const View &v) { return {stride_of(v.layout, 0), stride_of(v.layout, 1)}; }

// ---------------------------------------------------------------- norm

hx_status plan_norm(hx_dtype dtype, const View &x, const View &residual, const Vector &weight, const Vector &bias,
                    float epsilon, const View &residual_out, const View &out, const Vector &mean, const Vector &rstd,
                    LayerNormArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    if (!(epsilon >= 0.0f) || !std::isfinite(epsilon))
        return fail(HX_ERR_INVALID_CONFIGURATION, "norm epsilon must be finite and not negative, got %g",
                    (double)epsilon);
    HX_TRY(layout_basic_check(x.layout, "norm input"));
    const uint64_t shape[2] = {x.layout->shape[0], x.layout->shape[1]};
    Operands ops;
    HX_TRY(ops.in(x, 2, shape, size, "norm input"));
    const uint32_t at_x = ops.last();
    HX_TRY(check_left_out(residual, "residual"));
    HX_TRY(check_left_out(residual_out, "residual output"));
    if (residual.layout) HX_TRY(ops.in(residual, 2, shape, size, "residual"));
    const uint32_t at_residual = ops.last();
    HX_TRY(ops.in(weight, shape[1], size, "norm weight"));
    if (bias.given()) HX_TRY(ops.in(bias, shape[1], size, "norm bias"));
    if (residual_out.layout) {
        HX_TRY(ops.out(residual_out, 2, shape, size, "residual output"));
        // In place: each element of h is written by the thread that read it.
        ops.may_be(ops.last(), at_x);
        if (residual.layout) ops.may_be(ops.last(), at_residual);
    }
    HX_TRY(ops.out(out, 2, shape, size, "norm output"));
    if (mean.given()) HX_TRY(ops.out(mean, shape[0], 4, "norm mean"));
    if (rstd.given()) HX_TRY(ops.out(rstd, shape[0], 4, "norm rstd"));
    HX_TRY(ops.apart());
    if (shape[0] > kMost32 || shape[1] > kMost32)
        return fail(HX_ERR_DISPATCH_FAILED, "norm of shape %s exceeds the grid range", shape_string(*x.layout).c_str());
    LayerNormArgs &a = *args;
    a = LayerNormArgs{};
    a.dtype = dtype;
    a.rows = shape[0];
    a.cols = shape[1];
    a.x = first_of(x, size);
    a.residual = first_of(residual, size);
    a.weight = weight.buf;
    a.bias = first_of(bias);
    a.residual_out = first_of(residual_out, size);
    a.out = first_of(out, size);
    a.mean = first_of<float>(mean);
    a.rstd = first_of<float>(rstd);
    a.x_stride = row_stride(x);
    a.residual_stride = row_stride(residual);
    a.residual_out_stride = row_stride(residual_out);
    a.out_stride = row_stride(out);
    a.epsilon = epsilon;
    return HX_OK;
}

hx_status plan_norm_grad(hx_dtype dtype, const View &grad_out, const View &x, const Vector &weight, const Vector &mean,
                         const Vector &rstd, const View &residual_grad, const View &grad_in, const Vector &grad_weight,
                         const Vector &grad_bias, LayerNormGradArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    HX_TRY(layout_basic_check(x.layout, "norm input"));
    const uint64_t shape[2] = {x.layout->shape[0], x.layout->shape[1]};
    Operands ops;
    HX_TRY(ops.in(x, 2, shape, size, "norm input"));
    HX_TRY(ops.in(grad_out, 2, shape, size, "gradient of the norm output"));
    const uint32_t at_grad_out = ops.last();
    HX_TRY(ops.in(weight, shape[1], size, "norm weight"));
    HX_TRY(ops.in(mean, shape[0], 4, "norm mean"));
    HX_TRY(ops.in(rstd, shape[0], 4, "norm rstd"));
    HX_TRY(check_left_out(residual_grad, "gradient past the norm"));
    if (residual_grad.layout) HX_TRY(ops.in(residual_grad, 2, shape, size, "gradient past the norm"));
    const uint32_t at_past = ops.last();
    HX_TRY(ops.out(grad_in, 2, shape, size, "gradient of the norm input"));
    const uint32_t at_grad_in = ops.last();
    ops.may_be(at_grad_in, at_grad_out); // in place: written by the thread that read it
    if (residual_grad.layout) ops.may_be(at_grad_in, at_past);
    if (grad_weight.given()) HX_TRY(ops.out(grad_weight, shape[1], 4, "gradient of the norm weight"));
    if (grad_bias.given()) HX_TRY(ops.out(grad_bias, shape[1], 4, "gradient of the norm bias"));
    HX_TRY(ops.apart());
    if (shape[0] > kMost32 || shape[1] > kMostNormGradCols)
        return fail(HX_ERR_DISPATCH_FAILED, "norm of shape %s exceeds the grid range", shape_string(*x.layout).c_str());
    LayerNormGradArgs &a = *args;
    a = LayerNormGradArgs{};
    a.dtype = dtype;
    a.rows = shape[0];
    a.cols = shape[1];
    a.grad_out = first_of(grad_out, size);
    a.x = first_of(x, size);
    a.residual_grad = first_of(residual_grad, size);
    a.weight = weight.buf;
    a.mean = (const float *)mean.buf;
    a.rstd = (const float *)rstd.buf;
    a.grad_in = first_of(grad_in, size);
    a.grad_weight = first_of<float>(grad_weight);
    a.grad_bias = first_of<float>(grad_bias);
    a.grad_out_stride = row_stride(grad_out);
    a.x_stride = row_stride(x);
    a.residual_grad_stride = row_stride(residual_grad);
    a.grad_in_stride = row_stride(grad_in);
    return HX_OK;
}

// ---------------------------------------------------------- recurrence

// Blocks count sequences in the grid's second dimension.
hx_status check_sequences(const uint64_t *shape, const hx_layout &l) {
    if (shape[0] > 65535)
        return fail(HX_ERR_DISPATCH_FAILED, "recurrence takes at most 65535 sequences, got %llu",
                    (unsigned long long)shape[0]);
    if (shape[1] > kMost32 || shape[2] > kMost32)
        return fail(HX_ERR_DISPATCH_FAILED, "recurrence of shape %s exceeds the grid range", shape_string(l).c_str());
    return HX_OK;
}

hx_status plan_recurrence(hx_dtype dtype, const View &gate, const View &x, const View &state_in,
                          const Vector &lengths, const View &out, const View &state_out, RecurrenceArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    HX_TRY(layout_basic_check(x.layout, "recurrence input"));
    const uint64_t shape[3] = {x.layout->shape[0], x.layout->shape[1], x.layout->shape[2]};
    const uint64_t states[2] = {shape[0], shape[2]};
    Operands ops;
    HX_TRY(ops.in(x, 3, shape, size, "recurrence input"));
    HX_TRY(ops.in(gate, 3, shape, size, "recurrence gate"));
    if (lengths.given()) HX_TRY(ops.in(lengths, shape[0], 4, "sequence lengths"));
    HX_TRY(check_state(ops, state_in, states, false, "recurrence state"));
    const uint32_t at_state_in = ops.last();
    HX_TRY(ops.out(out, 3, shape, size, "recurrence output"));
    HX_TRY(check_state(ops, state_out, states, true, "recurrence state output"));
    if (state_in.layout && state_out.layout) ops.may_be(ops.last(), at_state_in);
    HX_TRY(ops.apart());
    HX_TRY(check_sequences(shape, *x.layout));
    RecurrenceArgs &a = *args;
    a = RecurrenceArgs{};
    a.dtype = dtype;
    a.batch = shape[0];
    a.tokens = shape[1];
    a.channels = shape[2];
    a.gate = first_of(gate, size);
    a.x = first_of(x, size);
    a.out = first_of(out, size);
    a.state_in = first_of<float>(state_in, 4);
    a.state_out = first_of<float>(state_out, 4);
    a.lengths = first_of<uint32_t>(lengths);
    a.s_gate = sequence(gate);
    a.s_x = sequence(x);
    a.s_out = sequence(out);
    a.s_state_in = row_stride(state_in);
    a.s_state_out = row_stride(state_out);
    return HX_OK;
}

hx_status plan_recurrence_grad(hx_dtype dtype, const View &gate, const View &x, const View &h, const View &state_in,
                               const Vector &lengths, const View &grad_out, const View &grad_state_out,
                               const View &grad_gate, const View &grad_x, const View &grad_state_in,
                               RecurrenceGradArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    HX_TRY(layout_basic_check(x.layout, "recurrence input"));
    const uint64_t shape[3] = {x.layout->shape[0], x.layout->shape[1], x.layout->shape[2]};
    const uint64_t states[2] = {shape[0], shape[2]};
    Operands ops;
    HX_TRY(ops.in(x, 3, shape, size, "recurrence input"));
    HX_TRY(ops.in(gate, 3, shape, size, "recurrence gate"));
    HX_TRY(ops.in(h, 3, shape, size, "recurrence output"));
    if (lengths.given()) HX_TRY(ops.in(lengths, shape[0], 4, "sequence lengths"));
    HX_TRY(check_state(ops, state_in, states, false, "recurrence state"));
    HX_TRY(ops.in(grad_out, 3, shape, size, "gradient of the recurrence output"));
    HX_TRY(check_state(ops, grad_state_out, states, false, "gradient of the state output"));
    HX_TRY(ops.out(grad_gate, 3, shape, size, "gradient of the gate"));
    HX_TRY(ops.out(grad_x, 3, shape, size, "gradient of the recurrence input"));
    HX_TRY(check_state(ops, grad_state_in, states, true, "gradient of the state"));
    HX_TRY(ops.apart());
    HX_TRY(check_sequences(shape, *x.layout));
    RecurrenceGradArgs &a = *args;
    a = RecurrenceGradArgs{};
    a.dtype = dtype;
    a.batch = shape[0];
    a.tokens = shape[1];
    a.channels = shape[2];
    a.gate = first_of(gate, size);
    a.x = first_of(x, size);
    a.h = first_of(h, size);
    a.grad_out = first_of(grad_out, size);
    a.grad_gate = first_of(grad_gate, size);
    a.grad_x = first_of(grad_x, size);
    a.state_in = first_of<float>(state_in, 4);
    a.grad_state_out = first_of<float>(grad_state_out, 4);
    a.grad_state_in = first_of<float>(grad_state_in, 4);
    a.lengths = first_of<uint32_t>(lengths);
    a.s_gate = sequence(gate);
    a.s_x = sequence(x);
    a.s_h = sequence(h);
    a.s_grad_out = sequence(grad_out);
    a.s_grad_gate = sequence(grad_gate);
    a.s_grad_x = sequence(grad_x);
    a.s_state_in = row_stride(state_in);
    a.s_grad_state_out = row_stride(grad_state_out);
    a.s_grad_state_in = row_stride(grad_state_in);
    return HX_OK;
}

// ------------------------------------------------------- cross entropy

// x [rows, width] and weight [vocab, width].
hx_status check_logits(Operands &ops, const View &x, const View &weight, const Vector &targets, uint32_t size,
                       uint64_t *rows, uint64_t *vocab, uint64_t *width) {
    HX_TRY(layout_basic_check(x.layout, "loss input"));
    HX_TRY(layout_basic_check(weight.layout, "vocabulary weight"));
    *rows = x.layout->shape[0];
    *width = x.layout->shape[1];
    *vocab = weight.layout->shape[0];
    const uint64_t x_shape[2] = {*rows, *width}, w_shape[2] = {*vocab, *width};
    HX_TRY(ops.in(x, 2, x_shape, size, "loss input"));
    HX_TRY(ops.in(weight, 2, w_shape, size, "vocabulary weight"));
    HX_TRY(ops.in(targets, *rows, 4, "targets"));
    if (*rows >= 1ull << 28 || *vocab >= 1ull << 28)
        return fail(HX_ERR_DISPATCH_FAILED, "loss of %llu rows over a vocabulary of %llu: each is below 2^28",
                    (unsigned long long)*rows, (unsigned long long)*vocab);
    if (*width > kCrossEntropyWidth)
        return fail(HX_ERR_DISPATCH_FAILED, "loss of width %llu: at most %llu", (unsigned long long)*width,
                    (unsigned long long)kCrossEntropyWidth);
    return HX_OK;
}

hx_status plan_loss(hx_dtype dtype, const View &x, const View &weight, const Vector &targets, const Vector &loss,
                    const Vector &lse, CrossEntropyArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    Operands ops;
    CrossEntropyArgs a{};
    HX_TRY(check_logits(ops, x, weight, targets, size, &a.rows, &a.vocab, &a.width));
    HX_TRY(ops.out(loss, a.rows, 4, "loss"));
    if (lse.given()) HX_TRY(ops.out(lse, a.rows, 4, "logarithms of the denominators"));
    HX_TRY(ops.apart());
    a.dtype = dtype;
    a.x = first_of(x, size);
    a.weight = first_of(weight, size);
    a.targets = first_of<uint32_t>(targets);
    a.loss = first_of<float>(loss);
    a.lse = first_of<float>(lse);
    a.x_stride = row_stride(x);
    a.weight_stride = row_stride(weight);
    *args = a;
    return HX_OK;
}

hx_status plan_loss_grad(hx_dtype dtype, const View &x, const View &weight, const Vector &targets, const Vector &lse,
                         const Vector &grad, const View &grad_x, const View &grad_weight, CrossEntropyGradArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    Operands ops;
    CrossEntropyGradArgs a{};
    HX_TRY(check_logits(ops, x, weight, targets, size, &a.rows, &a.vocab, &a.width));
    const uint64_t x_shape[2] = {a.rows, a.width}, w_shape[2] = {a.vocab, a.width};
    HX_TRY(ops.in(lse, a.rows, 4, "logarithms of the denominators"));
    HX_TRY(ops.in(grad, a.rows, 4, "gradient of the loss"));
    HX_TRY(check_left_out(grad_x, "gradient of the loss input"));
    HX_TRY(check_left_out(grad_weight, "gradient of the vocabulary weight"));
    if (grad_x.layout) HX_TRY(ops.out(grad_x, 2, x_shape, size, "gradient of the loss input"));
    if (grad_weight.layout) HX_TRY(ops.out(grad_weight, 2, w_shape, size, "gradient of the vocabulary weight"));
    HX_TRY(ops.apart());
    a.dtype = dtype;
    a.x = first_of(x, size);
    a.weight = first_of(weight, size);
    a.targets = first_of<uint32_t>(targets);
    a.lse = first_of<float>(lse);
    a.grad = first_of<float>(grad);
    a.grad_x = first_of(grad_x, size);
    a.grad_weight = first_of(grad_weight, size);
    a.x_stride = row_stride(x);
    a.weight_stride = row_stride(weight);
    a.grad_x_stride = row_stride(grad_x);
    a.grad_weight_stride = row_stride(grad_weight);
    *args = a;
    return HX_OK;
}

// ------------------------------------------------------------ dispatch

// What each operator's arguments need and run.
uint64_t workspace_bytes(const LayerNormArgs &) { return 0; }
uint64_t workspace_bytes(const LayerNormGradArgs &a) { return layer_norm_grad_workspace_bytes(a); }
uint64_t workspace_bytes(const RecurrenceArgs &a) { return gated_recurrence_workspace_bytes(a); }
uint64_t workspace_bytes(const RecurrenceGradArgs &a) { return gated_recurrence_grad_workspace_bytes(a); }
uint64_t workspace_bytes(const CrossEntropyArgs &a) { return cross_entropy_workspace_bytes(a); }
uint64_t workspace_bytes(const CrossEntropyGradArgs &a) { return cross_entropy_grad_workspace_bytes(a); }
hx_status launch(const LayerNormArgs &a, void *, hipStream_t s) { return launch_layer_norm(a, s); }
hx_status launch(const LayerNormGradArgs &a, void *ws, hipStream_t s) { return launch_layer_norm_grad(a, ws, s); }
hx_status launch(const RecurrenceArgs &a, void *ws, hipStream_t s) { return launch_gated_recurrence(a, ws, s); }
hx_status launch(const RecurrenceGradArgs &a, void *ws, hipStream_t s) {
    return launch_gated_recurrence_grad(a, ws, s);
}
hx_status launch(const CrossEntropyArgs &a, void *ws, hipStream_t s) { return launch_cross_entropy(a, ws, s); }
hx_status launch(const CrossEntropyGradArgs &a, void *ws, hipStream_t s) {
    return launch_cross_entropy_grad(a, ws, s);
}

template <typename Args> struct TrainingPlan final : hx_plan {
    Args args;
    hx_status dispatch(hipStream_t stream) override { return launch(args, ws, stream); }
};

template <typename Args> hx_status run_now(hx_device *dev, const Args &args, hx_stream stream) {
    HX_TRY(bind_device(dev));
    const hipStream_t s = pick_stream(dev, stream);
    const uint64_t bytes = workspace_bytes(args);
    if (bytes == 0) {
        HX_TRY(launch(args, nullptr, s));
        return ok();
    }
    Immediate im;
    HX_TRY(im.open(dev, s));
    void *scratch = nullptr;
    HX_TRY(im.scratch(bytes, &scratch));
    HX_TRY(launch(args, scratch, s));
    return ok();
}

template <typename Args> hx_status keep(hx_device *dev, const Args &args, hx_plan **plan) {
    return make_plan<TrainingPlan<Args>>(dev, args, workspace_bytes(args), plan);
}

hx_status check_plan(hx_plan **plan) {
    if (!plan) return fail(HX_ERR_INVALID_CONFIGURATION, "null plan out-pointer");
    *plan = nullptr;
    return HX_OK;
}

} // namespace

extern "C" {

#define HX_NORM_ARGS                                                                                                   \
    dtype, {x, x_buf_len, x_layout}, {residual, residual_buf_len, residual_layout}, {weight, weight_len},              \
        {bias, bias_len}, epsilon, {residual_out, residual_out_buf_len, residual_out_layout},                          \
        {out, out_buf_len, out_layout}, {mean, mean_len}, {rstd, rstd_len}

hx_status hx_layer_norm(hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len, const hx_layout *x_layout,
                        const void *residual, uint64_t residual_buf_len, const hx_layout *residual_layout,
                        const void *weight, uint64_t weight_len, const void *bias, uint64_t bias_len, float epsilon,
                        void *residual_out, uint64_t residual_out_buf_len, const hx_layout *residual_out_layout,
                        void *out, uint64_t out_buf_len, const hx_layout *out_layout, float *mean, uint64_t mean_len,
                        float *rstd, uint64_t rstd_len, hx_stream stream) {
    LayerNormArgs a;
    HX_TRY(plan_norm(HX_NORM_ARGS, &a));
    return run_now(dev, a, stream);
}

hx_status hx_prepare_layer_norm(hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len,
                                const hx_layout *x_layout, const void *residual, uint64_t residual_buf_len,
                                const hx_layout *residual_layout, const void *weight, uint64_t weight_len,
                                const void *bias, uint64_t bias_len, float epsilon, void *residual_out,
                                uint64_t residual_out_buf_len, const hx_layout *residual_out_layout, void *out,
                                uint64_t out_buf_len, const hx_layout *out_layout, float *mean, uint64_t mean_len,
                                float *rstd, uint64_t rstd_len, hx_plan **plan) {
    HX_TRY(check_plan(plan));
    LayerNormArgs a;
    HX_TRY(plan_norm(HX_NORM_ARGS, &a));
    return keep(dev, a, plan);
}

#define HX_NORM_GRAD_ARGS                                                                                              \
    dtype, {grad_out, grad_out_buf_len, grad_out_layout}, {x, x_buf_len, x_layout}, {weight, weight_len},              \
        {mean, mean_len}, {rstd, rstd_len}, {residual_grad, residual_grad_buf_len, residual_grad_layout},              \
        {grad_in, grad_in_buf_len, grad_in_layout}, {grad_weight, grad_weight_len}, {grad_bias, grad_bias_len}

hx_status hx_layer_norm_backward(hx_device *dev, hx_dtype dtype, const void *grad_out, uint64_t grad_out_buf_len,
                                 const hx_layout *grad_out_layout, const void *x, uint64_t x_buf_len,
                                 const hx_layout *x_layout, const void *weight, uint64_t weight_len, const float *mean,
                                 uint64_t mean_len, const float *rstd, uint64_t rstd_len, const void *residual_grad,
                                 uint64_t residual_grad_buf_len, const hx_layout *residual_grad_layout, void *grad_in,
                                 uint64_t grad_in_buf_len, const hx_layout *grad_in_layout, float *grad_weight,
                                 uint64_t grad_weight_len, float *grad_bias, uint64_t grad_bias_len,
                                 hx_stream stream) {
    LayerNormGradArgs a;
    HX_TRY(plan_norm_grad(HX_NORM_GRAD_ARGS, &a));
    return run_now(dev, a, stream);
}

hx_status hx_prepare_layer_norm_backward(
    hx_device *dev, hx_dtype dtype, const void *grad_out, uint64_t grad_out_buf_len, const hx_layout *grad_out_layout,
    const void *x, uint64_t x_buf_len, const hx_layout *x_layout, const void *weight, uint64_t weight_len,
    const float *mean, uint64_t mean_len, const float *rstd, uint64_t rstd_len, const void *residual_grad,
    uint64_t residual_grad_buf_len, const hx_layout *residual_grad_layout, void *grad_in, uint64_t grad_in_buf_len,
    const hx_layout *grad_in_layout, float *grad_weight, uint64_t grad_weight_len, float *grad_bias,
    uint64_t grad_bias_len, hx_plan **plan) {
    HX_TRY(check_plan(plan));
    LayerNormGradArgs a;
    HX_TRY(plan_norm_grad(HX_NORM_GRAD_ARGS, &a));
    return keep(dev, a, plan);
}

#define HX_RECURRENCE_ARGS                                                                                             \
    dtype, {gate, gate_buf_len, gate_layout}, {x, x_buf_len, x_layout}, {state_in, state_in_buf_len, state_in_layout}, \
        {lengths, lengths_len}, {out, out_buf_len, out_layout}, {state_out, state_out_buf_len, state_out_layout}

hx_status hx_gated_recurrence(hx_device *dev, hx_dtype dtype, const void *gate, uint64_t gate_buf_len,
                              const hx_layout *gate_layout, const void *x, uint64_t x_buf_len,
                              const hx_layout *x_layout, const float *state_in, uint64_t state_in_buf_len,
                              const hx_layout *state_in_layout, const uint32_t *lengths, uint64_t lengths_len,
                              void *out, uint64_t out_buf_len, const hx_layout *out_layout, float *state_out,
                              uint64_t state_out_buf_len, const hx_layout *state_out_layout, hx_stream stream) {
    RecurrenceArgs a;
    HX_TRY(plan_recurrence(HX_RECURRENCE_ARGS, &a));
    return run_now(dev, a, stream);
}

hx_status hx_prepare_gated_recurrence(hx_device *dev, hx_dtype dtype, const void *gate, uint64_t gate_buf_len,
                                      const hx_layout *gate_layout, const void *x, uint64_t x_buf_len,
                                      const hx_layout *x_layout, const float *state_in, uint64_t state_in_buf_len,
                                      const hx_layout *state_in_layout, const uint32_t *lengths, uint64_t lengths_len,
                                      void *out, uint64_t out_buf_len, const hx_layout *out_layout, float *state_out,
                                      uint64_t state_out_buf_len, const hx_layout *state_out_layout, hx_plan **plan) {
    HX_TRY(check_plan(plan));
    RecurrenceArgs a;
    HX_TRY(plan_recurrence(HX_RECURRENCE_ARGS, &a));
    return keep(dev, a, plan);
}

#define HX_RECURRENCE_GRAD_ARGS                                                                                        \
    dtype, {gate, gate_buf_len, gate_layout}, {x, x_buf_len, x_layout}, {h, h_buf_len, h_layout},                      \
        {state_in, state_in_buf_len, state_in_layout}, {lengths, lengths_len},                                         \
        {grad_out, grad_out_buf_len, grad_out_layout},                                                                 \
        {grad_state_out, grad_state_out_buf_len, grad_state_out_layout},                                               \
        {grad_gate, grad_gate_buf_len, grad_gate_layout}, {grad_x, grad_x_buf_len, grad_x_layout},                     \
        {grad_state_in, grad_state_in_buf_len, grad_state_in_layout}

hx_status hx_gated_recurrence_backward(
    hx_device *dev, hx_dtype dtype, const void *gate, uint64_t gate_buf_len, const hx_layout *gate_layout,
    const void *x, uint64_t x_buf_len, const hx_layout *x_layout, const void *h, uint64_t h_buf_len,
    const hx_layout *h_layout, const float *state_in, uint64_t state_in_buf_len, const hx_layout *state_in_layout,
    const uint32_t *lengths, uint64_t lengths_len, const void *grad_out, uint64_t grad_out_buf_len,
    const hx_layout *grad_out_layout, const float *grad_state_out, uint64_t grad_state_out_buf_len,
    const hx_layout *grad_state_out_layout, void *grad_gate, uint64_t grad_gate_buf_len,
    const hx_layout *grad_gate_layout, void *grad_x, uint64_t grad_x_buf_len, const hx_layout *grad_x_layout,
    float *grad_state_in, uint64_t grad_state_in_buf_len, const hx_layout *grad_state_in_layout, hx_stream stream) {
    RecurrenceGradArgs a;
    HX_TRY(plan_recurrence_grad(HX_RECURRENCE_GRAD_ARGS, &a));
    return run_now(dev, a, stream);
}

hx_status hx_prepare_gated_recurrence_backward(
    hx_device *dev, hx_dtype dtype, const void *gate, uint64_t gate_buf_len, const hx_layout *gate_layout,
    const void *x, uint64_t x_buf_len, const hx_layout *x_layout, const void *h, uint64_t h_buf_len,
    const hx_layout *h_layout, const float *state_in, uint64_t state_in_buf_len, const hx_layout *state_in_layout,
    const uint32_t *lengths, uint64_t lengths_len, const void *grad_out, uint64_t grad_out_buf_len,
    const hx_layout *grad_out_layout, const float *grad_state_out, uint64_t grad_state_out_buf_len,
    const hx_layout *grad_state_out_layout, void *grad_gate, uint64_t grad_gate_buf_len,
    const hx_layout *grad_gate_layout, void *grad_x, uint64_t grad_x_buf_len, const hx_layout *grad_x_layout,
    float *grad_state_in, uint64_t grad_state_in_buf_len, const hx_layout *grad_state_in_layout, hx_plan **plan) {
    HX_TRY(check_plan(plan));
    RecurrenceGradArgs a;
    HX_TRY(plan_recurrence_grad(HX_RECURRENCE_GRAD_ARGS, &a));
    return keep(dev, a, plan);
}

#define HX_LOSS_ARGS                                                                                                   \
    dtype, {x, x_buf_len, x_layout}, {weight, weight_buf_len, weight_layout}, {targets, targets_len}, {loss, loss_len}, \
        {lse, lse_len}

hx_status hx_linear_cross_entropy(hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len,
                                  const hx_layout *x_layout, const void *weight, uint64_t weight_buf_len,
                                  const hx_layout *weight_layout, const uint32_t *targets, uint64_t targets_len,
                                  float *loss, uint64_t loss_len, float *lse, uint64_t lse_len, hx_stream stream) {
    CrossEntropyArgs a;
    HX_TRY(plan_loss(HX_LOSS_ARGS, &a));
    return run_now(dev, a, stream);
}

hx_status hx_prepare_linear_cross_entropy(hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len,
                                          const hx_layout *x_layout, const void *weight, uint64_t weight_buf_len,
                                          const hx_layout *weight_layout, const uint32_t *targets,
                                          uint64_t targets_len, float *loss, uint64_t loss_len, float *lse,
                                          uint64_t lse_len, hx_plan **plan) {
    HX_TRY(check_plan(plan));
    CrossEntropyArgs a;
    HX_TRY(plan_loss(HX_LOSS_ARGS, &a));
    return keep(dev, a, plan);
}

#define HX_LOSS_GRAD_ARGS                                                                                              \
    dtype, {x, x_buf_len, x_layout}, {weight, weight_buf_len, weight_layout}, {targets, targets_len}, {lse, lse_len},  \
        {grad, grad_len}, {grad_x, grad_x_buf_len, grad_x_layout},                                                     \
        {grad_weight, grad_weight_buf_len, grad_weight_layout}

hx_status hx_linear_cross_entropy_backward(
    hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len, const hx_layout *x_layout, const void *weight,
    uint64_t weight_buf_len, const hx_layout *weight_layout, const uint32_t *targets, uint64_t targets_len,
    const float *lse, uint64_t lse_len, const float *grad, uint64_t grad_len, void *grad_x, uint64_t grad_x_buf_len,
    const hx_layout *grad_x_layout, void *grad_weight, uint64_t grad_weight_buf_len,
    const hx_layout *grad_weight_layout, hx_stream stream) {
    CrossEntropyGradArgs a;
    HX_TRY(plan_loss_grad(HX_LOSS_GRAD_ARGS, &a));
    return run_now(dev, a, stream);
}

hx_status hx_prepare_linear_cross_entropy_backward(
    hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len, const hx_layout *x_layout, const void *weight,
    uint64_t weight_buf_len, const hx_layout *weight_layout, const uint32_t *targets, uint64_t targets_len,
    const float *lse, uint64_t lse_len, const float *grad, uint64_t grad_len, void *grad_x, uint64_t grad_x_buf_len,
    const hx_layout *grad_x_layout, void *grad_weight, uint64_t grad_weight_buf_len,
    const hx_layout *grad_weight_layout, hx_plan **plan) {
    HX_TRY(check_plan(plan));
    CrossEntropyGradArgs a;
    HX_TRY(plan_loss_grad(HX_LOSS_GRAD_ARGS, &a));
    return keep(dev, a, plan);
}

} // extern "C"
