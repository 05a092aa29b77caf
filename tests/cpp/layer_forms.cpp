// The rules by which calls of the layer operators go to kernels, for
// tests/test_layer_forms.py: host code only.
#include "../../hephaestus_amd/csrc/layer_forms.hpp"

using namespace hx;

extern "C" {

// Tokens, wide and on dwords of the form for few tokens: 100 + 4·(32 tokens) +
// 2·wide + dwords.  A tile: its place in MatmulTile.  1000 more where rows are copied first.
int matmul_form(uint64_t m, uint64_t n, uint64_t k, uint64_t a, uint64_t b, int64_t a_stride, int64_t b_stride) {
    MatmulArgs p{};
    p.a = (const int8_t *)a;
    p.b = (const int8_t *)b;
    p.m = m;
    p.n = n;
    p.k = k;
    p.a_stride = a_stride;
    p.b_stride = b_stride;
    if (matmul_is_skinny(p)) return 100 + 4 * (m > 16) + 2 * skinny_is_wide(n) + !matmul_off_dwords(p);
    if (!matmul_needs_copy(p)) return (int)matmul_tile(m, n, k);
    return 1000 + (int)matmul_tile(m, n, matmul_copy_pitch(p));
}

// [by chunks, state streamed, waves a block, direct, parts, chunks of a part] of dense operands
// whose first elements lie `at` bytes into their buffers.
void attention_form(int32_t f32, uint64_t batch, uint64_t tokens, uint64_t heads, uint64_t dk, uint64_t dv, uint64_t at,
                    uint32_t *form) {
    AttentionArgs a{};
    a.dtype = f32 ? HX_DTYPE_F32 : HX_DTYPE_BF16;
    a.q = a.k = a.v = (const void *)(0x1000 + at);
    a.batch = batch;
    a.tokens = tokens;
    a.heads = a.kv_heads = heads;
    a.dk = dk;
    a.dv = dv;
    const auto dense = [&](uint64_t width) {
        return AttentionView{(int64_t)(tokens * heads * width), (int64_t)(heads * width), (int64_t)width};
    };
    a.sq = a.sk = dense(dk);
    a.sv = dense(dv);
    const AttentionParts parts = attention_parts(a);
    form[0] = attention_by_chunks(a);
    form[1] = attention_streams_state(a);
    form[2] = attention_waves(a);
    form[3] = attention_is_direct(a);
    form[4] = parts.parts;
    form[5] = parts.span / (f32 ? 32 : 64);
}

} // extern "C"
