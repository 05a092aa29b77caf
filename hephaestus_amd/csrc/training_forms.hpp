// The training operators' arguments (training_ops.cpp checks, then launches) and
// the rules by which a call goes to a kernel, as plain host code, so that they can
// be asked without a device.
#pragma once

#include "layer_forms.hpp"

namespace hx {

// Pointers are to the first element of each view, strides count elements; the last
// dimension of every view has stride 1.
struct LayerNormArgs {
    hx_dtype dtype;
    const void *x, *residual, *weight, *bias; // residual and bias may be null
    void *residual_out, *out;                 // residual_out may be null
    float *mean, *rstd;                       // may be null
    uint64_t rows, cols;
    int64_t x_stride, residual_stride, residual_out_stride, out_stride;
    float epsilon;
};

struct LayerNormGradArgs {
    hx_dtype dtype;
    const void *grad_out, *x, *residual_grad, *weight; // residual_grad may be null
    const float *mean, *rstd;
    void *grad_in;
    float *grad_weight, *grad_bias; // may be null
    uint64_t rows, cols;
    int64_t grad_out_stride, x_stride, residual_grad_stride, grad_in_stride;
};

struct SequenceView {
    int64_t batch, token; // strides
};
struct RecurrenceArgs {
    hx_dtype dtype;
    const void *gate, *x;
    void *out;
    const float *state_in;   // may be null
    float *state_out;        // may be null
    const uint32_t *lengths; // may be null
    uint64_t batch, tokens, channels;
    SequenceView s_gate, s_x, s_out;
    int64_t s_state_in, s_state_out; // of a sequence
};

struct RecurrenceGradArgs {
    hx_dtype dtype;
    const void *gate, *x, *h, *grad_out;
    void *grad_gate, *grad_x;
    const float *state_in, *grad_state_out; // may be null
    float *grad_state_in;                   // may be null
    const uint32_t *lengths;                // may be null
    uint64_t batch, tokens, channels;
    SequenceView s_gate, s_x, s_h, s_grad_out, s_grad_gate, s_grad_x;
    int64_t s_state_in, s_grad_state_out, s_grad_state_in;
};

struct CrossEntropyArgs {
    hx_dtype dtype;
    const void *x, *weight;
    const uint32_t *targets;
    float *loss, *lse; // lse may be null
    uint64_t rows, vocab, width;
    int64_t x_stride, weight_stride;
};

struct CrossEntropyGradArgs {
    hx_dtype dtype;
    const void *x, *weight;
    const uint32_t *targets;
    const float *lse, *grad;
    void *grad_x, *grad_weight; // may be null
    uint64_t rows, vocab, width;
    int64_t x_stride, weight_stride, grad_x_stride, grad_weight_stride;
};

inline uint64_t element_size(hx_dtype d) { return d == HX_DTYPE_F32 ? 4 : 2; }
inline uint64_t round_up(uint64_t n, uint64_t to) { return ceil_div(n, to) * to; }

// ------------------------------------------------------------------- norm

// The most 16-byte vectors of a row that a kernel is made for.
enum class NormRow : uint32_t { k16, k64, k128, k256, k512, k1024, k2048, k4096, kLong };
inline NormRow layer_norm_row(uint64_t cols, uint64_t size) {
    const uint64_t vectors = ceil_div(cols, 16 / size);
    if (vectors <= 16) return NormRow::k16;
    if (vectors <= 64) return NormRow::k64;
    if (vectors <= 128) return NormRow::k128;
    if (vectors <= 256) return NormRow::k256;
    if (vectors <= 512) return NormRow::k512;
    if (vectors <= 1024) return NormRow::k1024;
    if (vectors <= 2048) return NormRow::k2048;
    if (vectors <= 4096) return NormRow::k4096;
    return NormRow::kLong;
}

// The backward pass: runs of rows, a block each.
struct NormGradSplit {
    uint32_t blocks, rows_a_block;
};
inline NormGradSplit layer_norm_grad_split(const LayerNormGradArgs &a) {
    const uint64_t vectors = ceil_div(a.cols, 16 / element_size(a.dtype));
    const uint64_t at_once = vectors <= 16 ? 16 : vectors <= 128 ? 4 : 1; // rows of a block
    const uint64_t most = 1024;
    const uint64_t rows = std::max<uint64_t>(at_once, round_up(ceil_div(a.rows, most), at_once));
    return {(uint32_t)std::max<uint64_t>(1, ceil_div(a.rows, rows)), (uint32_t)rows};
}

// ------------------------------------------------------------- recurrence

// Whether two channels of bf16 can be read as a dword.
inline bool recurrence_on_dwords(const RecurrenceArgs &a) {
    const uint64_t bits = (uintptr_t)a.gate / 2 | (uintptr_t)a.x / 2 | (uintptr_t)a.out / 2 | a.channels;
    const int64_t strides = a.s_gate.batch | a.s_gate.token | a.s_x.batch | a.s_x.token | a.s_out.batch | a.s_out.token;
    return bits % 2 == 0 && (strides & 1) == 0;
}
inline bool recurrence_on_dwords(const RecurrenceGradArgs &a) {
    const uint64_t bits = (uintptr_t)a.gate / 2 | (uintptr_t)a.x / 2 | (uintptr_t)a.h / 2 | (uintptr_t)a.grad_out / 2 |
                          (uintptr_t)a.grad_gate / 2 | (uintptr_t)a.grad_x / 2 | a.channels;
    const int64_t strides = a.s_gate.batch | a.s_gate.token | a.s_x.batch | a.s_x.token | a.s_h.batch | a.s_h.token |
                            a.s_grad_out.batch | a.s_grad_out.token | a.s_grad_gate.batch | a.s_grad_gate.token |
                            a.s_grad_x.batch | a.s_grad_x.token;
    return bits % 2 == 0 && (strides & 1) == 0;
}

// Tokens that a block takes together: one wave's, or eight waves'.
enum class RecurrenceTile : uint32_t { kOne, kFew, kMany };
inline uint64_t recurrence_tile_tokens(const RecurrenceArgs &) { return 8 * 16; }
inline uint64_t recurrence_tile_tokens(const RecurrenceGradArgs &) { return 8 * 8; }

struct RecurrenceParts {
    RecurrenceTile tile;
    uint32_t parts, span;
};
// `vector` channels a lane.
template <typename Args> RecurrenceParts recurrence_parts(const Args &a, uint64_t vector) {
    const uint64_t all = std::max<uint64_t>(1, a.tokens);
    if (a.tokens <= 1) return {RecurrenceTile::kOne, 1, (uint32_t)all};
    if (a.tokens <= 32) return {RecurrenceTile::kFew, 1, (uint32_t)all};
    const uint64_t tile = recurrence_tile_tokens(a), blocks = a.batch * ceil_div(a.channels, 64 * vector);
    const uint64_t tiles = ceil_div(all, tile);
    uint64_t parts = 1;
    if (blocks < 192) parts = std::min(ceil_div(512, blocks), ceil_div(tiles, 2));
    const uint64_t span = ceil_div(tiles, std::max<uint64_t>(1, parts)) * tile;
    return {RecurrenceTile::kMany, (uint32_t)ceil_div(all, span), (uint32_t)span};
}

// ---------------------------------------------------------- cross entropy

enum class ProductTile : uint32_t { k256x256, k128x128, k64x64, k32x64 };
struct ProductTileSize {
    uint64_t m, n;
};
inline ProductTileSize product_tile_size(ProductTile t) {
    switch (t) {
    case ProductTile::k256x256: return {256, 256};
    case ProductTile::k128x128: return {128, 128};
    case ProductTile::k64x64: return {64, 64};
    default: return {32, 64};
    }
}
inline ProductTile product_tile(uint64_t m, uint64_t n) {
    const auto tiles = [&](uint64_t bm, uint64_t bn) { return ceil_div(m, bm) * ceil_div(n, bn); };
    if (m <= 32) return ProductTile::k32x64;
    if (tiles(256, 256) >= 160) return ProductTile::k256x256;
    if (tiles(128, 128) >= 192) return ProductTile::k128x128;
    return ProductTile::k64x64;
}

// The widest rows: places in 256 of them are counted in 32 bits.
constexpr uint64_t kCrossEntropyWidth = 1 << 20;

// Rows that a product reads where they lie begin on dwords and follow each other by at
// most 4 MiB; others are copied first.
inline bool product_reads_rows(const void *rows, int64_t stride, uint64_t size) {
    return ((uintptr_t)rows | (uint64_t)stride * size) % 4 == 0 && stride >= 0 && (uint64_t)stride * size <= 4 << 20;
}
inline bool cross_entropy_copies(const CrossEntropyArgs &a) {
    const uint64_t size = element_size(a.dtype);
    return !product_reads_rows(a.x, a.x_stride, size) || !product_reads_rows(a.weight, a.weight_stride, size);
}
// x is copied in any case; the weight is read across too, 16 bytes at a time.
inline bool cross_entropy_copies(const CrossEntropyGradArgs &a) {
    const uint64_t size = element_size(a.dtype);
    return !product_reads_rows(a.weight, a.weight_stride, size) || a.width * size % 16 != 0;
}

// Places of the workspace, in bytes.
struct CrossEntropyPlan {
    bool copies;
    uint64_t tiles_n, stats, picked, x, weight, bytes;
};
inline CrossEntropyPlan cross_entropy_plan(const CrossEntropyArgs &a) {
    CrossEntropyPlan p{};
    const uint64_t row = round_up(a.width * element_size(a.dtype), 128);
    p.copies = cross_entropy_copies(a);
    p.tiles_n = ceil_div(a.vocab, product_tile_size(product_tile(a.rows, a.vocab)).n);
    p.stats = 0;
    p.picked = round_up(p.tiles_n * a.rows * 8, 256);
    p.x = round_up(p.picked + a.rows * 4, 256);
    p.weight = p.x + (p.copies ? a.rows * row : 0);
    p.bytes = p.weight + (p.copies ? a.vocab * row : 0);
    return p;
}

// The backward pass takes the vocabulary in pieces of `piece` words, such that G of
// one has at most 256 MiB.
struct CrossEntropyGradPlan {
    bool copies;
    uint64_t piece, piece_pitch, sums_pitch; // elements
    uint64_t x, weight, g, sums, bytes;
};
inline CrossEntropyGradPlan cross_entropy_grad_plan(const CrossEntropyGradArgs &a) {
    CrossEntropyGradPlan p{};
    const uint64_t size = element_size(a.dtype), whole = 128 / size, row = round_up(a.width * size, 128);
    p.copies = cross_entropy_copies(a);
    const uint64_t most = std::max<uint64_t>(256, (256ull << 20) / (std::max<uint64_t>(1, a.rows) * size) / 256 * 256);
    const uint64_t pieces = std::max<uint64_t>(1, ceil_div(a.vocab, most));
    p.piece = std::max<uint64_t>(256, round_up(ceil_div(a.vocab, pieces), 256));
    p.piece_pitch = round_up(std::min(p.piece, std::max<uint64_t>(1, a.vocab)), whole);
    p.sums_pitch = round_up(a.width, 4);
    uint64_t at = 256; // the largest gradient lies first
    const auto take = [&](bool is_used, uint64_t bytes) {
        const uint64_t here = at;
        if (is_used) at += round_up(bytes, 256);
        return here;
    };
    p.x = take(true, a.rows * row);
    p.weight = take(p.copies, p.piece * row);
    p.g = take(true, a.rows * p.piece_pitch * size);
    p.sums = take(a.grad_x && p.piece < a.vocab, a.rows * p.sums_pitch * 4);
    p.bytes = at;
    return p;
}

} // namespace hx
