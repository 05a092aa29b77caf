// How products of more tiles than a launch has blocks are cut, for
// tests/test_training_launches.py: host code only.
#include "../../hephaestus_amd/csrc/training_forms.hpp"

extern "C" uint64_t tiles_of_a_launch(uint64_t threads) { return hx::tiles_a_launch(threads); }

// The words of a piece of the vocabulary, and the bytes of G of it and of the whole
// workspace, of the loss's gradients.
extern "C" void gradient_piece(uint64_t size, uint64_t rows, uint64_t vocab, uint64_t width, uint64_t *form) {
    hx::CrossEntropyGradArgs g{};
    g.dtype = size == 4 ? HX_DTYPE_F32 : HX_DTYPE_BF16;
    g.weight = (const void *)0x1000;
    g.grad_x = g.grad_weight = (void *)0x1000;
    g.weight_stride = (int64_t)width;
    g.rows = rows;
    g.vocab = vocab;
    g.width = width;
    const hx::CrossEntropyGradPlan p = hx::cross_entropy_grad_plan(g);
    form[0] = p.piece;
    form[1] = rows * p.piece_pitch * size;
    form[2] = p.bytes;
}

// Runs of rows of the norm's backward pass.
extern "C" uint64_t norm_runs(uint64_t size, uint64_t rows, uint64_t cols) {
    hx::LayerNormGradArgs a{};
    a.dtype = size == 4 ? HX_DTYPE_F32 : HX_DTYPE_BF16;
    a.rows = rows;
    a.cols = cols;
    return hx::layer_norm_grad_split(a).blocks;
}

// Bytes of the maps of a recurrence's parts, of dense operands.
extern "C" uint64_t map_bytes(uint64_t vector, int is_backward, uint64_t batch, uint64_t tokens, uint64_t channels) {
    hx::RecurrenceArgs a{};
    a.batch = batch;
    a.tokens = tokens;
    a.channels = channels;
    const uint32_t parts = hx::recurrence_parts(a, vector, is_backward != 0).parts;
    return parts > 1 ? batch * parts * channels * 8 : 0;
}
