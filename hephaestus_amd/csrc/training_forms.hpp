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

// The backward pass: runs of rows, a block each, in whole rounds of the 256 CUs where
// the rows allow.  Blocks of few waves need more of them side by side, and so do those
// of eight waves whose f32 rows leave registers for three on a CU.  Measured (us, with
// the launch that adds up the blocks' sums):
//   16384 x 8192 bf16  256 blocks 167   382 blocks 216   512 blocks 180   1024 blocks 200
//   16384 x 2048 bf16  256 blocks 76    512 blocks 51    1024 blocks 52   2048 blocks 71
//   16384 x 1024 bf16  256 blocks 33    512 blocks 32    1024 blocks 43
//   2282 x 14976 bf16  256 blocks 56    512 blocks 71
//   16384 x 4096 bf16  256 blocks 110   384 blocks 126   512 blocks 119   1024 blocks 137
//   9971 x 1268 f32    256 blocks 68    384 blocks 56    512 blocks 49    1024 blocks 59
//   8192 x 2048 f32    256 blocks 70    384 blocks 68    512 blocks 57    1024 blocks 70
//   1000 x 5001 f32    250 blocks 24    500 blocks 33    1000 blocks 44
struct NormGradSplit {
    uint32_t blocks, rows_a_block;
};
inline NormGradSplit layer_norm_grad_split(const LayerNormGradArgs &a) {
    const uint64_t vectors = ceil_div(a.cols, 16 / element_size(a.dtype));
    const uint64_t at_once = vectors <= 16 ? 16 : vectors <= 128 ? 4 : 1; // rows of a block
    const uint64_t most = vectors <= (a.dtype == HX_DTYPE_F32 ? 512 : 256) ? 512 : 256;
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

// Tokens that a block takes together: one wave's 1 or 8, or eight waves' 8 or 16 each.
enum class RecurrenceTile : uint32_t { kOne, kFew, kMany, kLong };

// Where sequences and channels give fewer blocks than half the card takes, the tokens
// are cut into parts, at the price of reading two of the operands twice.  Tiles of 128 tokens
// keep more loads under way in a block, tiles of 64 take fewer registers where two
// blocks share a CU; the backward pass has no registers for 128.  Measured (us, both launches):
//   8 x 4096 x 4096 bf16, 256 blocks   128 tokens 179   64 tokens 234   two parts 286
//   4 x 2000 x 1600 bf16, 52 blocks    8 parts of 64-token tiles 39, of 128 46   4 parts 56
//   1 x 65536 x 2048, backward, 16     32 parts 477   64 parts 500   16 parts 497
//   8 x 4096 x 4096, backward, 256     one part 320   two parts 463
// A part may be a single tile: a block's own loads and join take longer than to follow
// the maps of the parts in front of it.
//   1 x 4406 x 96 bf16, backward       a tile each 23   two 30   four 41   one part 281
//   6 x 1961 x 112 f32                 a tile each 16   two 18   four 25   one part 60
//   1 x 300 x 64 bf16                  a tile each 10   two 19   one part 16
//   2 x 130 x 512 bf16                 a tile each 9.8  one part 10.6
//   1 x 65536 x 256 f32, 4 blocks      512 blocks 66    256 72   1024 80
struct RecurrenceParts {
    RecurrenceTile tile;
    uint32_t parts, span;
};
// `vector` channels a lane.
template <typename Args> RecurrenceParts recurrence_parts(const Args &a, uint64_t vector, bool is_backward) {
    const uint64_t all = std::max<uint64_t>(1, a.tokens);
    if (a.tokens <= 1) return {RecurrenceTile::kOne, 1, (uint32_t)all};
    if (a.tokens <= 32) return {RecurrenceTile::kFew, 1, (uint32_t)all};
    const uint64_t blocks = a.batch * ceil_div(a.channels, 64 * vector), tiles = ceil_div(all, 64);
    if (blocks >= 160 || tiles < 3) {
        const bool is_long = !is_backward && all > 64;
        return {is_long ? RecurrenceTile::kLong : RecurrenceTile::kMany, 1, (uint32_t)round_up(all, 64)};
    }
    const uint64_t parts = std::min<uint64_t>(512 / std::max<uint64_t>(1, blocks), tiles);
    const uint64_t span = ceil_div(tiles, parts) * 64;
    return {RecurrenceTile::kMany, (uint32_t)ceil_div(all, span), (uint32_t)span};
}

// ---------------------------------------------------------- cross entropy

// Tiles of a product: rows x columns.
enum class ProductTile : uint32_t { k256x256, k128x128, k64x128, k64x64, k32x64 };
struct ProductTileRule {
    uint64_t m, n;
    uint64_t at_once; // blocks that share a CU
    // us that a round of blocks takes besides its steps: to its first step, and for what
    // becomes of the sums, which at 256 x 256 no other block's steps hide.
    double ends;
    // us for a step of 128 bytes of k with one block on each CU, and with all that share
    // it: of bf16, as measured on products of 256 x 4096 x 4096 to 2048 x 8192 x 2048, by rows
    // and across; of f32, where the matrix instructions bound all of them.
    double one, all, one_f32, all_f32;
};
constexpr ProductTileRule kProductTiles[] = {
    {256, 256, 1, 7.5, 1.70, 1.70, 7.60, 7.60}, {128, 128, 1, 3.4, 0.56, 0.56, 2.00, 2.00},
    {64, 128, 2, 2.9, 0.34, 0.60, 1.08, 2.10},  {64, 64, 2, 2.1, 0.30, 0.44, 0.60, 1.06},
    {32, 64, 2, 1.9, 0.23, 0.31, 0.33, 0.58}};

// How a product is cut: into tiles, and along k into parts whose sums are added up by a
// launch of their own.
struct ProductCut {
    ProductTile tile;
    uint32_t parts;
    uint64_t span; // k of a part, a whole number of steps
};
// The shortest by an estimate: rounds of blocks on the card's 256 CUs times a block's
// steps, a launch and the parts' sums, written and read at 5 TB/s.  Measured (us):
//   1000 x 5008 x 1040 bf16   64 x 128 25.6   128 x 128 28.8   256 x 256 37.7   64 x 64 29.4
//   2048 x 8192 x 2048 bf16  256 x 256 59.9   128 x 128 77.0   64 x 128 83.6
//   256 x 4096 x 4096 bf16    64 x 64 20.4     64 x 128 25.9   128 x 128 34.7
//   1000 x 5008 x 1040 f32    64 x 64 100.6   128 x 128 145
//   32 x 51200 x 64 bf16      64 x 128 5.4    128 x 128 8.8    256 x 256 9.3     64 x 64 6.7
//   4096 x 16384 x 64 bf16   256 x 256 33.4   64 x 128 53.9    128 x 128 62.2    64 x 64 79.3
inline ProductCut product_cut(uint64_t m, uint64_t n, uint64_t k, uint64_t size) {
    constexpr uint64_t kCus = 256;
    const uint64_t step = 128 / size, steps = std::max<uint64_t>(1, ceil_div(k, step));
    ProductCut best{ProductTile::k32x64, 1, steps * step};
    double best_us = 0.0;
    for (uint32_t t = 0; t < sizeof(kProductTiles) / sizeof(*kProductTiles); ++t) {
        const ProductTileRule &r = kProductTiles[t];
        const double one = size == 4 ? r.one_f32 : r.one, all = size == 4 ? r.all_f32 : r.all;
        const uint64_t tiles = ceil_div(m, r.m) * ceil_div(n, r.n);
        for (uint64_t parts = 1; parts <= 32 && (parts == 1 || steps / parts >= 4); parts *= 2) {
            const uint64_t blocks = tiles * parts, full = blocks / (kCus * r.at_once), rest = blocks % (kCus * r.at_once);
            const double rounds = full * all + (rest == 0 ? 0.0 : rest <= kCus ? one : all);
            double us = rounds * ceil_div(steps, parts) + r.ends * (full + (rest > 0)) + 2.0;
            if (parts > 1) us += 4.0 + (double)(m * n * parts) * 8 / 5e6;
            if (best_us == 0.0 || us < best_us) {
                best_us = us;
                const uint64_t span = ceil_div(steps, parts) * step;
                best = {(ProductTile)t, (uint32_t)std::max<uint64_t>(1, ceil_div(k, span)), span};
            }
        }
    }
    return best;
}

// Blocks of a launch, whole turns of the eight XCDs: it has fewer than 2^32 threads.
constexpr uint64_t tiles_a_launch(uint64_t threads) { return (1ull << 32) / threads - 8; }

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
    ProductCut cut;
    uint64_t tiles_n, stats, picked, parts, x, weight, bytes;
};
inline CrossEntropyPlan cross_entropy_plan(const CrossEntropyArgs &a) {
    CrossEntropyPlan p{};
    const uint64_t row = round_up(a.width * element_size(a.dtype), 128);
    p.copies = cross_entropy_copies(a);
    p.cut = product_cut(a.rows, a.vocab, a.width, element_size(a.dtype));
    p.tiles_n = ceil_div(a.vocab, p.cut.parts > 1 ? 1024 : kProductTiles[(uint32_t)p.cut.tile].n);
    p.stats = 0;
    p.picked = round_up(p.tiles_n * a.rows * 8, 256);
    p.parts = round_up(p.picked + a.rows * 4, 256);
    p.x = round_up(p.parts + (p.cut.parts > 1 ? p.cut.parts * a.rows * round_up(a.vocab, 4) * 4 : 0), 256);
    p.weight = p.x + (p.copies ? a.rows * row : 0);
    p.bytes = p.weight + (p.copies ? a.vocab * row : 0);
    return p;
}

// The backward pass takes the vocabulary in pieces of `piece` words, such that G of one
// has at most 256 MiB, but of no fewer than 256 words: past 524288 rows of bf16, 262144 of
// f32, G has 256 words of every row.
struct CrossEntropyGradPlan {
    bool copies;
    uint64_t piece, piece_pitch, sums_pitch; // elements
    uint64_t x, weight, g, sums, parts, bytes;
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
    // Sums of parts of k: of a piece's logits, of grad_x, or of a piece of grad_weight.
    uint64_t parts = 0;
    const auto fold = [&](uint64_t m, uint64_t n, uint64_t k, uint64_t pitch) {
        const uint32_t count = product_cut(m, n, k, size).parts;
        if (count > 1) parts = std::max(parts, count * m * pitch * 4);
    };
    const uint64_t piece = std::min(p.piece, a.vocab);
    for (uint64_t words : {piece, a.vocab % p.piece ? a.vocab % p.piece : piece}) { // the last piece's cut may differ
        fold(a.rows, words, a.width, round_up(words, 4));
        if (a.grad_x) fold(a.rows, a.width, words, p.sums_pitch);
        if (a.grad_weight) fold(words, a.width, a.rows, p.sums_pitch);
    }
    p.parts = take(parts > 0, parts);
    p.bytes = at;
    return p;
}

} // namespace hx
