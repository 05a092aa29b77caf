// The layer operators' arguments (layer_ops.cpp checks, then launches) and the
// rules by which a call goes to a kernel, as plain host code, so that they can be
// asked without a device.
#pragma once

#include "../../include/hx.h"

#include <algorithm>
#include <cstdint>

namespace hx {

inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Pointers are to the first element of each view, strides count elements; the last
// dimension of every view has stride 1.
struct NormArgs {
    hx_dtype dtype;
    const void *x, *residual, *weight; // residual may be null
    void *residual_out;                // may be null
    int8_t *quantized;
    float *scales;
    uint64_t rows, cols;
    int64_t x_stride, residual_stride, residual_out_stride, quantized_stride;
    float epsilon;
};

struct MatmulArgs {
    hx_dtype dtype; // of out
    const int8_t *a, *b;
    const float *a_scales, *b_scales;
    void *out;
    uint64_t m, n, k;
    int64_t a_stride, b_stride, out_stride;
};

struct AttentionView {
    int64_t batch, token, head; // strides; of a state `token` is the stride of dk
};
struct AttentionArgs {
    hx_dtype dtype;
    const void *q, *k, *v;
    void *out;
    const float *log_decay;
    const float *state_in; // may be null
    float *state_out;      // may be null
    const uint32_t *lengths; // may be null
    uint64_t batch, tokens, heads, kv_heads, dk, dv;
    AttentionView sq, sk, sv, so, si, st; // q, k, v, out, state_in, state_out
    float scale;
};

// ---------------------------------------------------------------- product

constexpr int kMatmulDepth = 128; // bytes of k a step

// Up to 16 tokens take the form that reads rows as they lie.  Up to 32 do where
// rows lie off dwords, so that tiles would need a copy first, unless a few blocks
// would have long rows to read (us, so and by copy and tiles):
//   20 x 8192 x 16384   46.2, 87.2     32 x 8192 x 16384   52.3, 89.0
//   20 x 4096 x 4097     9.7, 13.3     32 x 4096 x 4097    11.1, 13.2
//   20 x 1000 x 1001     4.0,  7.7     32 x 16384 x 600     6.3, 11.1
//   20 x 100 x 16384    24.4, 12.3     64 x 4096 x 4097    16.8, 14.4
inline bool matmul_off_dwords(const MatmulArgs &p) {
    return ((uintptr_t)p.a | (uintptr_t)p.b | (uint64_t)p.a_stride | (uint64_t)p.b_stride) % 4 != 0;
}
inline bool matmul_is_skinny(const MatmulArgs &p) {
    return p.m <= 16 || (p.m <= 32 && matmul_off_dwords(p) && (p.k <= 4096 || p.n >= 4096));
}
inline bool matmul_needs_copy(const MatmulArgs &p) { return !matmul_is_skinny(p) && p.k > 0 && matmul_off_dwords(p); }
inline uint64_t matmul_copy_pitch(const MatmulArgs &p) { return ceil_div(p.k, kMatmulDepth) * kMatmulDepth; }

// Two fragments of channels a block halve its reads of a, from the size on where
// there is a block for each CU all the same.
inline bool skinny_is_wide(uint64_t n) { return n >= 2 * 16 * 256; }

// Pairs: two blocks share a CU.  Groups: of waves, which take the steps of k in
// turn; the smaller tiles have them always.
enum class MatmulTile : uint32_t {
    k256x256,
    k128x128Pairs,
    k128x128,
    k96x96,
    k64x64Groups,
    k64x64,
    k64x32Pairs,
    k64x32,
    k32x32Pairs,
    k32x32,
    k32x16
};

// The largest tile of which there are enough for the 256 CUs: a smaller tile
// moves more bytes to the same CUs.  Where there are more tiles than CUs two
// blocks share one, with LDS for half the steps in flight.  A last round of the
// largest tiles that leaves most CUs idle costs more than they gain: two blocks
// of 128 x 128 on each CU take 0.54 of the time of one of 256 x 256.  Groups that share a
// block's k keep more loads under way in a block, for about 2 us to add their
// sums: worth it for long rows, or where tiles are too few to fill the card.
// Measured (us):
//   8192 x 8192 x 1024   256 x 256 123     128 x 128 143
//   831 x 14912 x 1792   256 x 256 39.5    128 x 128 41.4
//   6144 x 6144 x 6144   256 x 256 280     128 x 128 253     (2.25 rounds, 4.5)
//   1308 x 11648 x 2624  256 x 256 83.9    128 x 128 48.4    (1.08 rounds, 1.96)
//   1000 x 8192 x 8192   128 x 128 71.1    64 x 64 109     256 x 256 115
//   2048 x 2048 x 2048   128 x 128 16.6    64 x 64 19.0    256 x 256 37.8
//   1500 x 1500 x 8192    96 x  96 28.6    64 x 64 39.2
//   128 x 8192 x 4096     64 x  64 10.9 in three groups, 11.8 in one
//   700 x 1500 x 1500     64 x  64 22.5 in three groups, 12.6 in one
//   256 x 1024 x 8192     32 x  32 10.2    64 x 32 13.5    64 x 64 17.4
//   20 x 4096 x 4096      32 x  16 6.0     32 x 32 7.0     64 x 32 8.3
inline MatmulTile matmul_tile(uint64_t m, uint64_t n, uint64_t k) {
    const auto tiles = [&](uint64_t bm, uint64_t bn) { return ceil_div(m, bm) * ceil_div(n, bn); };
    constexpr uint64_t kCus = 256, kEnough = 160, kFull = 192;
    const bool long_rows = k >= 4096;
    const uint64_t rounds = ceil_div(tiles(256, 256), kCus), pairs = ceil_div(tiles(128, 128), 2 * kCus);
    if (tiles(256, 256) >= kEnough && rounds <= 0.54 * pairs) return MatmulTile::k256x256;
    if (tiles(128, 128) > kCus) return MatmulTile::k128x128Pairs;
    if (tiles(128, 128) >= kFull) return MatmulTile::k128x128;
    if (long_rows && tiles(96, 96) >= kFull && tiles(96, 96) <= kCus) return MatmulTile::k96x96;
    if (long_rows && tiles(64, 64) >= kEnough && tiles(64, 64) <= kCus) return MatmulTile::k64x64Groups;
    if (tiles(64, 64) >= kEnough) return MatmulTile::k64x64;
    if (tiles(64, 32) > kCus) return MatmulTile::k64x32Pairs;
    if (tiles(64, 32) >= kEnough) return MatmulTile::k64x32;
    if (tiles(32, 32) > kCus) return MatmulTile::k32x32Pairs;
    if (tiles(32, 32) >= kEnough) return MatmulTile::k32x32;
    return MatmulTile::k32x16;
}

// -------------------------------------------------------------- attention

// States that the caches cannot hold until the next token are streamed.
inline bool attention_streams_state(const AttentionArgs &a) {
    return a.batch * a.heads * a.dk * a.dv * sizeof(float) > 64ull << 20;
}

// A few tokens go through the recurrence.  Its time grows with each, that of a
// chunk does not (us, recurrence and chunk):
//   1 x 32 heads of 128 x 128    4 tokens 6.4, 11.0    8 tokens 9.5, 11.5     10 tokens 11.4, 11.0
//   32 x 32, the same            34.4, 51.2            48.5, 51.6             55.9, 50.6
//   32 x 32, the same in f32     37.6, 72.3            12 tokens 64.1, 70.8   16 tokens 77.3, 71.3
//   8 x 32 heads of 64 x 64      6.5, 8.0              6 tokens 8.2, 8.2      8 tokens 9.9, 8.0
inline bool attention_by_chunks(const AttentionArgs &a) {
    return a.tokens > (a.dk <= 64 ? 6 : a.dtype == HX_DTYPE_F32 ? 12 : 8) && a.dk > 0;
}

// Whether the rows of a chunk can be loaded without registers (Stager in
// linear_attention.hip).
inline bool attention_rows_direct(const void *base, const AttentionView &s, uint64_t width, uint64_t size) {
    const uint64_t bits = (uintptr_t)base | (uint64_t)(s.token | s.head | s.batch) * size;
    return bits % 4 == 0 && width % (16 / size) == 0 && s.token >= 0 && s.token < 1 << 24;
}
inline bool attention_is_direct(const AttentionArgs &a) {
    const uint64_t size = a.dtype == HX_DTYPE_F32 ? 4 : 2;
    return attention_rows_direct(a.q, a.sq, a.dk, size) && attention_rows_direct(a.k, a.sk, a.dk, size) &&
           attention_rows_direct(a.v, a.sv, a.dv, size);
}

// Waves a block, each with 16 columns of v: with wider keys than 128, two chunks
// of q, k and 128 columns of v would not fit LDS.
inline uint32_t attention_waves(const AttentionArgs &a) { return a.dv <= 64 || a.dk > 128 ? 4 : 8; }

// The keys' width that a kernel is made for.
inline uint32_t attention_key_width(uint64_t dk) { return dk <= 64 ? 64 : dk <= 96 ? 96 : dk <= 128 ? 128 : 256; }

// A prompt cut into `parts` of `span` tokens each, a multiple of the chunk.
struct AttentionParts {
    uint32_t parts, span;
    float *states; // [batch, heads, parts, dk, dv]: each part's own sum, then the state before it
};

// How many parts a prompt is cut into where there are fewer heads than the card
// takes blocks.  The parts run side by side, but their own sums have to be taken
// first, in half the time of the outputs, and their states written, joined and
// read.  Times in us as measured: a chunk of bf16 3.0, 4.2 and 6.6 for keys of 64,
// 128 and 256, whatever the columns (LDS reads of q and k); of f32 3.0 to 6.9 for
// 64 x 64 to 128 x 128 a block (matrix instructions); two more launches 7.5; the
// states 7 TB/s.  Heads x tokens of keys x columns, us:
//   16 x 16384 of 128 x 128, 16 parts 124, 8 parts 195, uncut 1003
//   64 x 512, the same, 4 parts 36.5, 2 parts 40.0, uncut 38.4
//   8 x 256 of 128 x 2048, 2 parts 34.6, uncut 25.1
//   16 x 256 and 16 x 192 of 128 x 128, one chunk a part 20.7 and 20.1, uncut 21.6 and 17.9
//   8 x 256 of 64 x 64, 4 parts 16.5, uncut 14.7;  8 x 384, 6 parts 16.1, uncut 19.7
//   128 x 4096, the same, 4 parts 113, 2 parts 145, uncut 201
//   8 x 128 of 128 x 1024 in f32, 4 parts 32.0, 2 parts 37.7, uncut 34.7
inline AttentionParts attention_parts(const AttentionArgs &a) {
    const bool f32 = a.dtype == HX_DTYPE_F32;
    const uint64_t chunk = f32 ? 32 : 64, chunks = ceil_div(a.tokens, chunk), columns = 16 * attention_waves(a);
    const uint64_t blocks = a.batch * a.heads * ceil_div(a.dv, columns);
    // Blocks of the narrowest heads take half a CU's LDS.
    const uint64_t card = a.dk <= 64 && a.dv <= 64 ? 512 : 256;
    const double width = attention_key_width(a.dk);
    const double chunk_us = f32 ? 1.7 + 5.2 * (width * columns) / (128 * 128) : 1.8 + 2.4 * width / 128;
    uint64_t best = 1;
    double best_us = chunks * chunk_us;
    for (uint64_t parts = 2; parts <= std::min(chunks, card / blocks); ++parts) {
        const double states_us = (double)(a.batch * a.heads * parts) * (a.dk * a.dv * 16) / 7e6;
        const double us = ceil_div(chunks, parts) * 1.5 * chunk_us + 7.5 + states_us;
        if (us < best_us) {
            best_us = us;
            best = parts;
        }
    }
    const uint64_t span = ceil_div(chunks, best) * chunk;
    return AttentionParts{(uint32_t)ceil_div(a.tokens, span), (uint32_t)span, nullptr};
}

} // namespace hx
