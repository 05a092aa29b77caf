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
