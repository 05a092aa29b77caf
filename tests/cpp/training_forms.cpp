// The rules by which calls of the training operators go to kernels, for
// tests/test_training_forms.py: host code only.
#include "../../hephaestus_amd/csrc/training_forms.hpp"

using namespace hx;

extern "C" {

int norm_row(uint64_t cols, uint64_t size) { return (int)layer_norm_row(cols, size); }

// [tile, parts, on dwords] of dense operands whose first elements lie `at` bytes into
// their buffers.
void recurrence_form(int32_t f32, int32_t is_backward, uint64_t batch, uint64_t tokens, uint64_t channels, uint64_t at,
                     uint32_t *form) {
    RecurrenceArgs a{};
    RecurrenceGradArgs g{};
    a.dtype = g.dtype = f32 ? HX_DTYPE_F32 : HX_DTYPE_BF16;
    a.batch = g.batch = batch;
    a.tokens = g.tokens = tokens;
    a.channels = g.channels = channels;
    a.gate = a.x = g.gate = g.x = g.h = g.grad_out = (const void *)(0x1000 + at);
    a.out = g.grad_gate = g.grad_x = (void *)(0x1000 + at);
    const SequenceView dense{(int64_t)(tokens * channels), (int64_t)channels};
    a.s_gate = a.s_x = a.s_out = dense;
    g.s_gate = g.s_x = g.s_h = g.s_grad_out = g.s_grad_gate = g.s_grad_x = dense;
    const bool on_dwords = is_backward ? recurrence_on_dwords(g) : recurrence_on_dwords(a);
    const uint64_t vector = !f32 && on_dwords ? 2 : 1;
    const RecurrenceParts cut = is_backward ? recurrence_parts(g, vector, true) : recurrence_parts(a, vector, false);
    form[0] = (uint32_t)cut.tile;
    form[1] = cut.parts;
    form[2] = on_dwords;
    form[3] = cut.span;
}

// [tile, parts] of a product.
void product_form(uint64_t m, uint64_t n, uint64_t k, uint64_t size, uint64_t *form) {
    const ProductCut cut = product_cut(m, n, k, size);
    form[0] = (uint64_t)cut.tile;
    form[1] = cut.parts;
    form[2] = cut.span;
}

// Whether rows `stride` elements apart from `at` on are copied first: the forward pass's, and the
// backward pass's of a weight `width` wide.
int copies(uint64_t size, uint64_t at, int64_t stride, uint64_t width) {
    CrossEntropyArgs a{};
    CrossEntropyGradArgs g{};
    a.dtype = g.dtype = size == 4 ? HX_DTYPE_F32 : HX_DTYPE_BF16;
    a.x = a.weight = g.weight = (const void *)(0x1000 + at);
    a.x_stride = a.weight_stride = g.weight_stride = stride;
    a.width = g.width = width;
    return cross_entropy_copies(a) + 2 * cross_entropy_copies(g);
}

// [pieces, workspace bytes] of the loss's gradients.
void gradient_pieces(uint64_t size, uint64_t rows, uint64_t vocab, uint64_t width, uint64_t *form) {
    CrossEntropyGradArgs g{};
    g.dtype = size == 4 ? HX_DTYPE_F32 : HX_DTYPE_BF16;
    g.weight = (const void *)0x1000;
    g.grad_x = g.grad_weight = (void *)0x1000;
    g.weight_stride = width;
    g.rows = rows;
    g.vocab = vocab;
    g.width = width;
    const CrossEntropyGradPlan p = cross_entropy_grad_plan(g);
    form[0] = ceil_div(vocab, p.piece);
    form[1] = p.bytes;
}

} // extern "C"
