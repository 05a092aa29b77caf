// Entry points of the layer operators (RMS norm with an 8-bit output, product
// of 8-bit integers, linear attention).  Every check runs before the first
// launch, so a refused call writes nothing.
#include "operand_checks.hpp"

#include <cmath>

using namespace hx;

namespace {

// Products of two int8 are at most 2^14, so this many sum within int32.
constexpr uint64_t kMaxMatmulK = 131071;
constexpr uint64_t kMaxAttentionDk = 256;
constexpr uint64_t kMaxGridY = 65535;

// ---------------------------------------------------------------- norm

hx_status plan_norm(hx_dtype dtype, const void *x, uint64_t x_buf_len, const hx_layout *x_layout, const void *residual,
                    uint64_t residual_buf_len, const hx_layout *residual_layout, const void *weight,
                    uint64_t weight_len, float epsilon, void *residual_out, uint64_t residual_out_buf_len,
                    const hx_layout *residual_out_layout, void *quantized, uint64_t quantized_buf_len,
                    const hx_layout *quantized_layout, float *scales, uint64_t scales_len, NormArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    if (!(epsilon >= 0.0f) || !std::isfinite(epsilon))
        return fail(HX_ERR_INVALID_CONFIGURATION, "norm epsilon must be finite and not negative, got %g",
                    (double)epsilon);
    HX_TRY(layout_basic_check(x_layout, "norm input"));
    const uint64_t shape[2] = {x_layout->shape[0], x_layout->shape[1]};
    Span sx, sr, sw, so, sq, ss;
    HX_TRY(check_view(x, x_buf_len, x_layout, 2, shape, size, false, "norm input", &sx));
    HX_TRY(check_left_out(residual, residual_buf_len, residual_layout, "residual"));
    HX_TRY(check_left_out(residual_out, residual_out_buf_len, residual_out_layout, "residual output"));
    if (residual_layout)
        HX_TRY(check_view(residual, residual_buf_len, residual_layout, 2, shape, size, false, "residual", &sr));
    HX_TRY(check_vector(weight, weight_len, shape[1], size, "norm weight", &sw));
    if (residual_out_layout)
        HX_TRY(check_view(residual_out, residual_out_buf_len, residual_out_layout, 2, shape, size, true,
                          "residual output", &so));
    HX_TRY(check_view(quantized, quantized_buf_len, quantized_layout, 2, shape, 1, true, "quantized output", &sq));
    HX_TRY(check_vector(scales, scales_len, shape[0], 4, "quantized scales", &ss));
    if (residual_out_layout) {
        // In place: each element of h is written by the thread that read it.
        if (overlap(so, sx) && !same_view(so, sx))
            return fail(HX_ERR_DISPATCH_FAILED, "residual output must be the view of the norm input or not overlap it");
        if (residual_layout && overlap(so, sr) && !same_view(so, sr))
            return fail(HX_ERR_DISPATCH_FAILED, "residual output must be the view of the residual or not overlap it");
        HX_TRY(check_apart(so, "residual output", sw, "the norm weight"));
        HX_TRY(check_apart(so, "residual output", sq, "the quantized output"));
        HX_TRY(check_apart(so, "residual output", ss, "the quantized scales"));
    }
    const Span inputs[3] = {sx, sr, sw};
    const char *names[3] = {"the norm input", "the residual", "the norm weight"};
    for (int i = 0; i < 3; ++i) {
        HX_TRY(check_apart(sq, "quantized output", inputs[i], names[i]));
        HX_TRY(check_apart(ss, "quantized scales", inputs[i], names[i]));
    }
    HX_TRY(check_apart(sq, "quantized output", ss, "the quantized scales"));
    if (shape[0] > 0x7FFFFFFFull || shape[1] > 0x7FFFFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "norm of shape %s exceeds the grid range",
                    shape_string(*x_layout).c_str());
    NormArgs &a = *args;
    a = NormArgs{};
    a.dtype = dtype;
    a.rows = shape[0];
    a.cols = shape[1];
    a.x = at(x, x_layout, size);
    a.x_stride = stride_of(x_layout, 0);
    if (residual_layout) {
        a.residual = at(residual, residual_layout, size);
        a.residual_stride = stride_of(residual_layout, 0);
    }
    if (residual_out_layout) {
        a.residual_out = at(residual_out, residual_out_layout, size);
        a.residual_out_stride = stride_of(residual_out_layout, 0);
    }
    a.weight = weight;
    a.quantized = (int8_t *)at(quantized, quantized_layout, 1);
    a.quantized_stride = stride_of(quantized_layout, 0);
    a.scales = scales;
    a.epsilon = epsilon;
    return HX_OK;
}

struct NormPlan final : hx_plan {
    NormArgs args;
    hx_status dispatch(hipStream_t stream) override { return launch_norm_quantize(args, stream); }
};

// -------------------------------------------------------------- matmul

hx_status plan_matmul(const void *a, uint64_t a_buf_len, const hx_layout *a_layout, const float *a_scales,
                      uint64_t a_scales_len, const void *b, uint64_t b_buf_len, const hx_layout *b_layout,
                      const float *b_scales, uint64_t b_scales_len, hx_dtype dtype, void *out, uint64_t out_buf_len,
                      const hx_layout *out_layout, MatmulArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    HX_TRY(layout_basic_check(a_layout, "matmul a"));
    HX_TRY(layout_basic_check(b_layout, "matmul b"));
    const uint64_t m = a_layout->shape[0], k = a_layout->shape[1], n = b_layout->shape[0];
    const uint64_t a_shape[2] = {m, k}, b_shape[2] = {n, k}, o_shape[2] = {m, n};
    Span sa, sb, so, va, vb;
    HX_TRY(check_view(a, a_buf_len, a_layout, 2, a_shape, 1, false, "matmul a", &sa));
    HX_TRY(check_view(b, b_buf_len, b_layout, 2, b_shape, 1, false, "matmul b", &sb));
    HX_TRY(check_vector(a_scales, a_scales_len, m, 4, "matmul a scales", &va));
    HX_TRY(check_vector(b_scales, b_scales_len, n, 4, "matmul b scales", &vb));
    HX_TRY(check_view(out, out_buf_len, out_layout, 2, o_shape, size, true, "matmul output", &so));
    if (k > kMaxMatmulK)
        return fail(HX_ERR_DISPATCH_FAILED, "matmul of %llu terms exceeds the 32-bit sums: at most %llu",
                    (unsigned long long)k, (unsigned long long)kMaxMatmulK);
    if (m > 0x7FFFFFFFull || n > 0x7FFFFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "matmul output of shape %s exceeds the grid range",
                    shape_string(*out_layout).c_str());
    HX_TRY(check_apart(so, "matmul output", sa, "matmul a"));
    HX_TRY(check_apart(so, "matmul output", sb, "matmul b"));
    HX_TRY(check_apart(so, "matmul output", va, "the scales of a"));
    HX_TRY(check_apart(so, "matmul output", vb, "the scales of b"));
    MatmulArgs &r = *args;
    r = MatmulArgs{};
    r.dtype = dtype;
    r.a = (const int8_t *)at(a, a_layout, 1);
    r.b = (const int8_t *)at(b, b_layout, 1);
    r.a_scales = a_scales;
    r.b_scales = b_scales;
    r.out = at(out, out_layout, size);
    r.m = m;
    r.n = n;
    r.k = k;
    r.a_stride = stride_of(a_layout, 0);
    r.b_stride = stride_of(b_layout, 0);
    r.out_stride = stride_of(out_layout, 0);
    return HX_OK;
}

struct MatmulPlan final : hx_plan {
    MatmulArgs args;
    hx_status dispatch(hipStream_t stream) override { return launch_matmul_i8(args, ws, stream); }
};

// ----------------------------------------------------------- attention

AttentionView view_of(const hx_layout *l, bool state) {
    // A state is [batch, heads, dk, dv], the rest [batch, tokens, heads, width].
    return AttentionView{stride_of(l, 0), stride_of(l, state ? 2 : 1), stride_of(l, state ? 1 : 2)};
}

hx_status plan_attention(hx_dtype dtype, const void *q, uint64_t q_buf_len, const hx_layout *q_layout, const void *k,
                         uint64_t k_buf_len, const hx_layout *k_layout, const void *v, uint64_t v_buf_len,
                         const hx_layout *v_layout, const float *log_decay, uint64_t log_decay_len, float scale,
                         const float *state_in, uint64_t state_in_buf_len, const hx_layout *state_in_layout,
                         float *state_out, uint64_t state_out_buf_len, const hx_layout *state_out_layout,
                         const uint32_t *lengths, uint64_t lengths_len, void *out, uint64_t out_buf_len,
                         const hx_layout *out_layout, AttentionArgs *args) {
    uint32_t size = 0;
    HX_TRY(check_layer_dtype(dtype, &size));
    if (!std::isfinite(scale))
        return fail(HX_ERR_INVALID_CONFIGURATION, "attention scale must be finite, got %g", (double)scale);
    HX_TRY(layout_basic_check(q_layout, "attention query"));
    HX_TRY(layout_basic_check(k_layout, "attention key"));
    HX_TRY(layout_basic_check(v_layout, "attention value"));
    const uint64_t batch = q_layout->shape[0], tokens = q_layout->shape[1], heads = q_layout->shape[2];
    const uint64_t dk = q_layout->shape[3], kv_heads = k_layout->shape[2], dv = v_layout->shape[3];
    const uint64_t q_shape[4] = {batch, tokens, heads, dk}, k_shape[4] = {batch, tokens, kv_heads, dk};
    const uint64_t v_shape[4] = {batch, tokens, kv_heads, dv}, o_shape[4] = {batch, tokens, heads, dv};
    const uint64_t s_shape[4] = {batch, heads, dk, dv};
    Span sq, sk, sv, so, si, st, sd, sl;
    HX_TRY(check_view(q, q_buf_len, q_layout, 4, q_shape, size, false, "attention query", &sq));
    HX_TRY(check_view(k, k_buf_len, k_layout, 4, k_shape, size, false, "attention key", &sk));
    HX_TRY(check_view(v, v_buf_len, v_layout, 4, v_shape, size, false, "attention value", &sv));
    HX_TRY(check_view(out, out_buf_len, out_layout, 4, o_shape, size, true, "attention output", &so));
    if (kv_heads == 0 ? heads != 0 : heads % kv_heads != 0)
        return fail(HX_ERR_DISPATCH_FAILED, "attention heads (%llu) must be a multiple of the key/value heads (%llu)",
                    (unsigned long long)heads, (unsigned long long)kv_heads);
    if (dk > kMaxAttentionDk)
        return fail(HX_ERR_DISPATCH_FAILED, "attention keys are at most %llu wide, got %llu",
                    (unsigned long long)kMaxAttentionDk, (unsigned long long)dk);
    HX_TRY(check_vector(log_decay, log_decay_len, heads, 4, "log decay", &sd));
    if (lengths || lengths_len) HX_TRY(check_vector(lengths, lengths_len, batch, 4, "sequence lengths", &sl));
    HX_TRY(check_left_out(state_in, state_in_buf_len, state_in_layout, "attention state"));
    HX_TRY(check_left_out(state_out, state_out_buf_len, state_out_layout, "attention state output"));
    if (state_in_layout)
        HX_TRY(check_view(state_in, state_in_buf_len, state_in_layout, 4, s_shape, 4, false, "attention state", &si));
    if (state_out_layout)
        HX_TRY(check_view(state_out, state_out_buf_len, state_out_layout, 4, s_shape, 4, true,
                          "attention state output", &st));
    if (batch > kMaxGridY || heads > kMaxGridY)
        return fail(HX_ERR_DISPATCH_FAILED, "attention takes at most %llu sequences and heads, got %llu and %llu",
                    (unsigned long long)kMaxGridY, (unsigned long long)batch, (unsigned long long)heads);
    if (tokens > 0x7FFFFFFFull || dv > 0x7FFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "attention of shape %s exceeds the grid range",
                    shape_string(*out_layout).c_str());
    const Span inputs[5] = {sq, sk, sv, sd, sl};
    const char *names[5] = {"the query", "the key", "the value", "the log decay", "the sequence lengths"};
    for (int i = 0; i < 5; ++i) {
        HX_TRY(check_apart(so, "attention output", inputs[i], names[i]));
        HX_TRY(check_apart(st, "attention state output", inputs[i], names[i]));
    }
    HX_TRY(check_apart(so, "attention output", si, "the state"));
    HX_TRY(check_apart(so, "attention output", st, "the state output"));
    // In place: each element of the state is written by the thread that read it.
    if (state_in_layout && state_out_layout && overlap(st, si) && !same_view(st, si))
        return fail(HX_ERR_DISPATCH_FAILED, "attention state output must be the view of the state or not overlap it");
    AttentionArgs &a = *args;
    a = AttentionArgs{};
    a.dtype = dtype;
    a.q = at(q, q_layout, size);
    a.k = at(k, k_layout, size);
    a.v = at(v, v_layout, size);
    a.out = at(out, out_layout, size);
    a.log_decay = log_decay;
    a.lengths = lengths;
    a.batch = batch;
    a.tokens = tokens;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.dk = dk;
    a.dv = dv;
    a.sq = view_of(q_layout, false);
    a.sk = view_of(k_layout, false);
    a.sv = view_of(v_layout, false);
    a.so = view_of(out_layout, false);
    if (state_in_layout) {
        a.state_in = at(state_in, state_in_layout, 4);
        a.si = view_of(state_in_layout, true);
    }
    if (state_out_layout) {
        a.state_out = at(state_out, state_out_layout, 4);
        a.st = view_of(state_out_layout, true);
    }
    a.scale = scale;
    return HX_OK;
}

struct AttentionPlan final : hx_plan {
    AttentionArgs args;
    hx_status dispatch(hipStream_t stream) override { return launch_linear_attention(args, ws, stream); }
};

} // namespace

namespace hx {

hx_status allow_lds(const void *kernel, uint32_t bytes, std::atomic<uint64_t> &allowed) {
    if (bytes <= 65536) return HX_OK;
    int device = 0;
    HX_HIP(hipGetDevice(&device), HX_ERR_DISPATCH_FAILED, "hipGetDevice");
    const uint64_t bit = device < 64 ? 1ull << device : 0; // asked for anew where there is no bit
    if (allowed.load(std::memory_order_relaxed) & bit) return HX_OK;
    HX_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), HX_ERR_DISPATCH_FAILED,
           "LDS size");
    allowed.fetch_or(bit, std::memory_order_relaxed);
    return HX_OK;
}

} // namespace hx

extern "C" {

hx_status hx_rms_norm_quantize(hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len,
                               const hx_layout *x_layout, const void *residual, uint64_t residual_buf_len,
                               const hx_layout *residual_layout, const void *weight, uint64_t weight_len,
                               float epsilon, void *residual_out, uint64_t residual_out_buf_len,
                               const hx_layout *residual_out_layout, void *quantized, uint64_t quantized_buf_len,
                               const hx_layout *quantized_layout, float *scales, uint64_t scales_len,
                               hx_stream stream) {
    NormArgs a;
    HX_TRY(plan_norm(dtype, x, x_buf_len, x_layout, residual, residual_buf_len, residual_layout, weight, weight_len,
                     epsilon, residual_out, residual_out_buf_len, residual_out_layout, quantized, quantized_buf_len,
                     quantized_layout, scales, scales_len, &a));
    HX_TRY(bind_device(dev));
    HX_TRY(launch_norm_quantize(a, pick_stream(dev, stream)));
    return ok();
}

hx_status hx_prepare_rms_norm_quantize(hx_device *dev, hx_dtype dtype, const void *x, uint64_t x_buf_len,
                                       const hx_layout *x_layout, const void *residual, uint64_t residual_buf_len,
                                       const hx_layout *residual_layout, const void *weight, uint64_t weight_len,
                                       float epsilon, void *residual_out, uint64_t residual_out_buf_len,
                                       const hx_layout *residual_out_layout, void *quantized,
                                       uint64_t quantized_buf_len, const hx_layout *quantized_layout, float *scales,
                                       uint64_t scales_len, hx_plan **plan) {
    if (!plan) return fail(HX_ERR_INVALID_CONFIGURATION, "null plan out-pointer");
    *plan = nullptr;
    NormArgs a;
    HX_TRY(plan_norm(dtype, x, x_buf_len, x_layout, residual, residual_buf_len, residual_layout, weight, weight_len,
                     epsilon, residual_out, residual_out_buf_len, residual_out_layout, quantized, quantized_buf_len,
                     quantized_layout, scales, scales_len, &a));
    return make_plan<NormPlan>(dev, a, 0, plan);
}

hx_status hx_matmul_i8(hx_device *dev, const void *a, uint64_t a_buf_len, const hx_layout *a_layout,
                       const float *a_scales, uint64_t a_scales_len, const void *b, uint64_t b_buf_len,
                       const hx_layout *b_layout, const float *b_scales, uint64_t b_scales_len, hx_dtype dtype,
                       void *out, uint64_t out_buf_len, const hx_layout *out_layout, hx_stream stream) {
    MatmulArgs args;
    HX_TRY(plan_matmul(a, a_buf_len, a_layout, a_scales, a_scales_len, b, b_buf_len, b_layout, b_scales, b_scales_len,
                       dtype, out, out_buf_len, out_layout, &args));
    HX_TRY(bind_device(dev));
    const hipStream_t s = pick_stream(dev, stream);
    Immediate im;
    HX_TRY(im.open(dev, s));
    void *scratch = nullptr;
    HX_TRY(im.scratch(matmul_i8_workspace_bytes(args), &scratch));
    HX_TRY(launch_matmul_i8(args, scratch, s));
    return ok();
}

hx_status hx_prepare_matmul_i8(hx_device *dev, const void *a, uint64_t a_buf_len, const hx_layout *a_layout,
                               const float *a_scales, uint64_t a_scales_len, const void *b, uint64_t b_buf_len,
                               const hx_layout *b_layout, const float *b_scales, uint64_t b_scales_len, hx_dtype dtype,
                               void *out, uint64_t out_buf_len, const hx_layout *out_layout, hx_plan **plan) {
    if (!plan) return fail(HX_ERR_INVALID_CONFIGURATION, "null plan out-pointer");
    *plan = nullptr;
    MatmulArgs args;
    HX_TRY(plan_matmul(a, a_buf_len, a_layout, a_scales, a_scales_len, b, b_buf_len, b_layout, b_scales, b_scales_len,
                       dtype, out, out_buf_len, out_layout, &args));
    return make_plan<MatmulPlan>(dev, args, matmul_i8_workspace_bytes(args), plan);
}

hx_status hx_linear_attention(hx_device *dev, hx_dtype dtype, const void *q, uint64_t q_buf_len,
                              const hx_layout *q_layout, const void *k, uint64_t k_buf_len, const hx_layout *k_layout,
                              const void *v, uint64_t v_buf_len, const hx_layout *v_layout, const float *log_decay,
                              uint64_t log_decay_len, float scale, const float *state_in, uint64_t state_in_buf_len,
                              const hx_layout *state_in_layout, float *state_out, uint64_t state_out_buf_len,
                              const hx_layout *state_out_layout, const uint32_t *lengths, uint64_t lengths_len,
                              void *out, uint64_t out_buf_len, const hx_layout *out_layout, hx_stream stream) {
    AttentionArgs a;
    HX_TRY(plan_attention(dtype, q, q_buf_len, q_layout, k, k_buf_len, k_layout, v, v_buf_len, v_layout, log_decay,
                          log_decay_len, scale, state_in, state_in_buf_len, state_in_layout, state_out,
                          state_out_buf_len, state_out_layout, lengths, lengths_len, out, out_buf_len, out_layout, &a));
    HX_TRY(bind_device(dev));
    const hipStream_t s = pick_stream(dev, stream);
    Immediate im;
    HX_TRY(im.open(dev, s));
    void *scratch = nullptr;
    HX_TRY(im.scratch(linear_attention_workspace_bytes(a), &scratch));
    HX_TRY(launch_linear_attention(a, scratch, s));
    return ok();
}

hx_status hx_prepare_linear_attention(hx_device *dev, hx_dtype dtype, const void *q, uint64_t q_buf_len,
                                      const hx_layout *q_layout, const void *k, uint64_t k_buf_len,
                                      const hx_layout *k_layout, const void *v, uint64_t v_buf_len,
                                      const hx_layout *v_layout, const float *log_decay, uint64_t log_decay_len,
                                      float scale, const float *state_in, uint64_t state_in_buf_len,
                                      const hx_layout *state_in_layout, float *state_out, uint64_t state_out_buf_len,
                                      const hx_layout *state_out_layout, const uint32_t *lengths,
                                      uint64_t lengths_len, void *out, uint64_t out_buf_len,
                                      const hx_layout *out_layout, hx_plan **plan) {
    if (!plan) return fail(HX_ERR_INVALID_CONFIGURATION, "null plan out-pointer");
    *plan = nullptr;
    AttentionArgs a;
    HX_TRY(plan_attention(dtype, q, q_buf_len, q_layout, k, k_buf_len, k_layout, v, v_buf_len, v_layout, log_decay,
                          log_decay_len, scale, state_in, state_in_buf_len, state_in_layout, state_out,
                          state_out_buf_len, state_out_layout, lengths, lengths_len, out, out_buf_len, out_layout, &a));
    return make_plan<AttentionPlan>(dev, a, linear_attention_workspace_bytes(a), plan);
}

} // extern "C"
