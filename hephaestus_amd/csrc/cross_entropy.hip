// Softmax cross entropy of the logits x·wᵀ over a vocabulary, without keeping the
// logits (hx_linear_cross_entropy), and its backward pass, for gfx950.
//
// Forward: the product goes tile by tile; a tile leaves, for each of its rows, the
// largest logit and the sum of the exponentials of the others' distances from it, and
// the target's logit where it lies in the tile.  A second launch joins the tiles.  Of few
// tiles the logits are summed in parts of the width, in scratch, and then taken row by row.
//
// Backward, a piece of the vocabulary after another: the logits again, as
//   G = (grad / most)·(e^(logit - lse) - [target]),   most = max |grad|,
// in the operands' type, then dx += G·w and dw = Gᵀ·x on matrix instructions, with
// sums in f32 that are multiplied by `most` at the end.  With the mean's gradients,
// which are all alike, the factor is 1 and G keeps the places of e^(logit - lse):
// a factor's rounding would be the same in every term of a sum and stay in it.
//
// The products bound large calls: 8192 x 32768 x 4096 bf16 takes 1.63 ms forward (1.35
// PFLOP/s) and 5.4 ms backward (1.22), where the library's products of such sizes reach 1.24
// to 1.40; the matrix units are busy 69% and 57 to 64% of the cycles, at the clock that
// the power leaves, with no bank conflicts in LDS.  16 x 32000 x 2048 reads the weight at
// 4.1 TB/s (32 us).  f32 is bound by rounds of 512 tiles whose last one is short: 1000 x 5003 x
// 1025 takes 329 us backward, 94 TFLOP/s, where a full round reaches 126 and the library's
// product 154.
#include "hx_internal.hpp"
#include "layer_device.hpp"

#include <atomic>
#include <type_traits>

namespace hx {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kDepth = 128; // bytes of k a step

__device__ const u32x4 kZeros[1] = {{0, 0, 0, 0}}; // read in place of what lies past an end

// 16 bytes of k of 16 rows of either operand.  Of f32 these are four instructions,
// each with an element of every lane: k in another order, the same for both.  The
// fragments' instructions of one element go first: no two in a row add to the same sums.
template <typename T, int FM, int FN>
__device__ __forceinline__ void mma(const u32x4 (&b)[FN], const u32x4 (&a)[FM], f32x4 (&sum)[FM][FN]) {
    constexpr int kEach = sizeof(T) == 2 ? 1 : 4;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if constexpr (sizeof(T) == 2)
                    sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, b[j]), __builtin_bit_cast(bf16x8, a[i]), sum[i][j], 0, 0, 0);
                else
                    sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                        __builtin_bit_cast(f32x4, b[j])[e], __builtin_bit_cast(f32x4, a[i])[e], sum[i][j], 0, 0, 0);
            }
}

// 16 bytes of a row from `k` on, zeros from `end` on: of rows of 16 bytes and more in one
// load, the last 16 bytes' where it would pass the end.
__device__ __forceinline__ u32x4 load_bytes(const int8_t *row, uint32_t k, uint32_t end) {
    if (end >= 16) {
        const uint32_t from = min(k, end - 16), past = min(k - from, 16u);
        const auto v = __builtin_bit_cast(unsigned __int128, (u32x4)*(const u32x4_any *)(row + from));
        return past < 16 ? __builtin_bit_cast(u32x4, v >> (8 * past)) : u32x4{0, 0, 0, 0};
    }
    u32x4 v = {0, 0, 0, 0};
    for (uint32_t i = 0; k + i < end; ++i) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
    return v;
}

// e^x for x of at most about 0.  The product's rounding leaves a relative error of up to
// |x|·2^-24: nothing in a sum of such terms, where e^x outweighs it, nor before a
// rounding to 16 bits.
__device__ __forceinline__ float exp_near(float x) { return __builtin_amdgcn_exp2f(x * 1.44269502f); }

// The same to a rounding or two, with the rest that the product with log2(e) leaves.
__device__ __forceinline__ float exp_of(float x) {
    constexpr float kLog2e = 1.44269502f, kLow = 1.92596299e-8f;
    if (x < -120.0f) return 0.0f;
    const float t = x * kLog2e, low = __builtin_fmaf(x, kLog2e, -t) + x * kLow;
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, low * 0.693147181f, e);
}

// ---------------------------------------------------------------- product
// out[m, n] = Σ_k a(m, k)·b(n, k), handed to an epilogue in tiles of BM x BN.  An
// operand lies in memory by rows of k, a row for each m or n, or across: a row for each
// k.  The tile's WM x WN waves each take a part of it.
struct Operand {
    const int8_t *rows;
    int64_t stride; // bytes, of its rows in memory
};
struct Product {
    Operand a, b;
    uint64_t m, n, k; // elements
    uint64_t span;    // of k, of a part of the grid's second dimension
};

// The barrier between steps is written out: all of the wave's LDS reads and
// writes and all but its last N loads have ended when it is passed.
template <int N> __device__ __forceinline__ void step_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

// Turned reads of LDS, two for each address: x[i] is a column's elements from 4 rows at
// p[i] and from 4 rows NEXT bytes on.  The builtin would wait for all loads to LDS that
// are under way, whichever place they go to; the block has the reads' own wait.
template <int NEXT> __device__ __forceinline__ void read_turned(const uint32_t (&p)[1], u32x4 (&x)[1]) {
    uint64_t v[2];
    asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1])
                 : "v"(p[0]), "n"(NEXT)
                 : "memory");
    __builtin_memcpy(x, v, sizeof(v));
}
template <int NEXT> __device__ __forceinline__ void read_turned(const uint32_t (&p)[2], u32x4 (&x)[2]) {
    uint64_t v[4];
    asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                 "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                 : "v"(p[0]), "v"(p[1]), "n"(NEXT)
                 : "memory");
    __builtin_memcpy(x, v, sizeof(v));
}
template <int NEXT> __device__ __forceinline__ void read_turned(const uint32_t (&p)[4], u32x4 (&x)[4]) {
    uint64_t v[8];
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),
                   "=&v"(v[7])
                 : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "n"(NEXT)
                 : "memory");
    __builtin_memcpy(x, v, sizeof(v));
}
template <int NEXT> __device__ __forceinline__ void read_turned(const uint32_t (&p)[8], u32x4 (&x)[8]) {
    uint64_t v[16];
    asm volatile("ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %2, %17\n\tds_read_b64_tr_b16 %3, %17 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %18 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %6, %19\n\tds_read_b64_tr_b16 %7, %19 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %8, %20\n\tds_read_b64_tr_b16 %9, %20 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %10, %21\n\tds_read_b64_tr_b16 %11, %21 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %12, %22\n\tds_read_b64_tr_b16 %13, %22 offset:%24\n\t"
                 "ds_read_b64_tr_b16 %14, %23\n\tds_read_b64_tr_b16 %15, %23 offset:%24\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),
                   "=&v"(v[7]), "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]),
                   "=&v"(v[14]), "=&v"(v[15])
                 : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "n"(NEXT)
                 : "memory");
    __builtin_memcpy(x, v, sizeof(v));
}

// One operand's part of a step in LDS, WIDTH rows of m or n; loads go from memory
// to LDS without registers, each wave's 64 chunks of 16 bytes side by side, so that the
// exchange of places is made on the memory's side.  Rows begin on dwords.
//
// By rows: 128 bytes of each row, chunk c of row r at place c ^ (r % 8), so that
// the rows that a matrix instruction reads at one c fall on all banks.
// Across: WIDTH elements of each k, in segments of what 16 lanes take at once (32
// bytes of bf16, 64 of f32); segment s of row k at place s ^ turn(k), for the same reason.
// bf16 is turned by the read: 16 lanes that address 4 rows of 16 elements receive
// a column's 4 elements each.
template <typename T, int WIDTH, int THREADS, bool ACROSS> struct Staged {
    static constexpr int kBytes = WIDTH * kDepth, kLoads = WIDTH * 8 / THREADS;
    static constexpr int kN = 16 / sizeof(T);              // elements of a chunk
    static constexpr int kRow = ACROSS ? WIDTH * (int)sizeof(T) : kDepth;
    static constexpr int kChunks = kRow / 16;              // of a row
    static constexpr int kSegment = sizeof(T) == 2 ? 2 : 4; // chunks
    static constexpr int kTurns = kChunks / kSegment < 8 ? kChunks / kSegment : 8;
    static_assert(kLoads * THREADS == WIDTH * 8);

    static __device__ __forceinline__ uint32_t turn(uint32_t k) {
        if constexpr (sizeof(T) == 2) return (k % 4 + k / 8 % 2 * 4) % kTurns;
        else return k / 4 % 4 % kTurns;
    }

    // What this thread loads: its chunks' places from `base` on, the tile's first row or
    // column at k = 0.  Strides are such that 32 bits hold them.
    const int8_t *base;
    uint32_t from[kLoads];
    uint32_t stride, last;
    __device__ __forceinline__ void open(const Operand &o, uint64_t first, uint64_t end, int wave, int lane) {
        stride = (uint32_t)o.stride;
        base = o.rows + (ACROSS ? first * sizeof(T) : first * (uint64_t)stride);
        // Rows past the end repeat the last one, columns past it the last chunk; they
        // are dropped at the end.
        last = (uint32_t)min((uint64_t)WIDTH, end - first) - 1;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint32_t q = (wave * kLoads + j) * kWave + lane, row = q / kChunks, place = q % kChunks;
            if constexpr (ACROSS) {
                const uint32_t chunk = (place / kSegment ^ turn(row)) * kSegment + place % kSegment;
                from[j] = row * stride + min(chunk, last / kN) * 16;
            } else {
                from[j] = min(row, last) * stride + (place ^ (row % 8)) * 16;
            }
        }
    }
    __device__ __forceinline__ const int8_t *at_step(uint32_t step) const {
        return base + (uint64_t)step * (ACROSS ? kDepth / sizeof(T) * stride : kDepth);
    }
    __device__ __forceinline__ void fetch(int8_t *stage, uint32_t step, int wave) const {
        int8_t *to = stage + wave * (kLoads * 1024);
        const int8_t *p = at_step(step);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            __builtin_amdgcn_global_load_lds((const void *)(p + from[j]), (lds_void *)(to + j * 1024), 16, 0, 0);
    }
    // The last, partial step: zeros past the end of k, from a line of them.  Only rows that
    // end inside a chunk go through registers, few at a time: more would take them from
    // the sums.
    __device__ __forceinline__ void fetch_rest(int8_t *stage, uint32_t step, uint64_t k, int wave, int lane) const {
        int8_t *to = stage + wave * (kLoads * 1024);
        const int8_t *p = at_step(step);
        const uint32_t left = (uint32_t)(k - (uint64_t)step * (kDepth / sizeof(T))); // elements
        if (ACROSS || left * sizeof(T) % 16 == 0) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const uint32_t row = ((wave * kLoads + j) * kWave + lane) / kChunks, place = lane % kChunks;
                const bool is_in = ACROSS ? row < left : (place ^ (row % 8)) * 16 < left * sizeof(T);
                __builtin_amdgcn_global_load_lds((const void *)(is_in ? p + from[j] : (const int8_t *)kZeros),
                                                 (lds_void *)(to + j * 1024), 16, 0, 0);
            }
            return;
        }
        constexpr int kTogether = kLoads % 2 ? 1 : 2;
#pragma unroll 1
        for (int first = 0; first < kLoads; first += kTogether) {
            u32x4 v[kTogether];
#pragma unroll
            for (int j = 0; j < kTogether; ++j) {
                const uint32_t row = ((wave * kLoads + first + j) * kWave + lane) / kChunks;
                v[j] = load_bytes(base + min(row, last) * stride, step * kDepth + (lane % kChunks ^ (row % 8)) * 16,
                                  (uint32_t)(k * sizeof(T)));
            }
#pragma unroll
            for (int j = 0; j < kTogether; ++j) *(u32x4 *)(to + (first + j) * 1024 + lane * 16) = v[j];
        }
    }

    // Where this lane reads: 16 bytes of k, half `s` of the step, of row `part` + 16·i + lane % 16.
    uint32_t at;
    __device__ __forceinline__ void place(uint32_t part, int lane) {
        if constexpr (!ACROSS) at = (part + lane % 16) * kDepth + ((lane / 16 ^ lane % 8) * 16);
        else if constexpr (sizeof(T) == 2)
            at = (lane / 16 * 8 + lane % 16 / 4) * kRow + ((part / 16 ^ turn(lane / 16 * 8 + lane % 16 / 4)) * 32) + lane % 4 * 8;
        else at = (lane / 16 * 4) * kRow + ((part / 16 ^ turn(lane / 16 * 4)) * 64) + lane % 16 * 4;
    }
    // N fragments of half `s`.
    template <int N> __device__ __forceinline__ void read(const int8_t *stage, int s, u32x4 (&x)[N]) const {
        if constexpr (!ACROSS) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *(const u32x4 *)(stage + (at ^ (64 * s)) + i * (16 * kDepth));
        } else if constexpr (sizeof(T) == 2) {
            uint32_t p[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
                p[i] = (uint32_t)(uintptr_t)(lds_void *)(stage + s * (32 * kRow)) + (at ^ (32 * i));
            read_turned<4 * kRow>(p, x);
        } else {
            const int8_t *p = stage + s * (16 * kRow);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = *(const uint32_t *)(p + (at ^ (64 * i)) + e * kRow);
        }
    }
};

template <int BM_, int BN_, int WM_, int WN_, int S_> struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
    static constexpr int kThreads = WM * WN * kWave;
    static constexpr int kStage = (BM + BN) * kDepth, kLds = kStage * S;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    static_assert(kLds <= 160 * 1024);
    // Two waves on each SIMD, which take turns.
    static constexpr bool kTurns = WM == 2 && WN == 4 && S == 2;
    // Rows of tiles in a strip: 4 x 8 tiles of 256 x 256 at a time on an XCD's 32 CUs (a
    // product of 8192 x 16384 x 4096 takes 1087 us, 1148 with 8 rows), 8 x 8 smaller ones.
    static constexpr int kStrip = BM == 256 ? 4 : 8;
};

// What an epilogue knows of its place: lane l has, of fragment (i, j), the sums of
// row m + 16·i and columns n + 16·j + 0..3.
struct Place {
    uint64_t m, n;       // this lane's first row and column
    uint64_t m0, tile_n; // the tile's first row; its place among the columns' tiles
    int wave_n;
};

template <typename T, typename C, bool ACROSS_A, bool ACROSS_B, typename E>
__global__ __launch_bounds__(C::kThreads) void product_kernel(Product p, E epilogue, uint32_t tiles_m,
                                                             uint32_t tiles_n, uint32_t first_tile) {
    constexpr int BM = C::BM, BN = C::BN, FM = C::FM, FN = C::FN, S = C::S;
    extern __shared__ __align__(16) int8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

    // Blocks go to the eight XCDs in turn.  Each XCD takes a run of tiles in strips of a
    // few rows of tiles, so that its L2 serves both operands of those that are under way.
    const uint32_t share = gridDim.x / 8, rest = gridDim.x % 8;
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t tile = first_tile + xcd * share + min(xcd, rest) + turn;
    const uint32_t strip = tile / (C::kStrip * tiles_n), in_strip = tile % (C::kStrip * tiles_n);
    const uint32_t height = min((uint32_t)C::kStrip, tiles_m - C::kStrip * strip);
    const uint64_t m0 = (uint64_t)(C::kStrip * strip + in_strip % height) * BM, n0 = (uint64_t)(in_strip / height) * BN;

    constexpr uint32_t kStep = kDepth / sizeof(T);
    const uint64_t k0 = blockIdx.y * p.span; // parts are whole steps
    p.k = min(p.span, p.k - k0);
    p.a.rows += k0 * (ACROSS_A ? (uint64_t)p.a.stride : sizeof(T));
    p.b.rows += k0 * (ACROSS_B ? (uint64_t)p.b.stride : sizeof(T));
    const uint32_t steps = (uint32_t)((p.k + kStep - 1) / kStep), whole = (uint32_t)(p.k / kStep);
    Staged<T, BM, C::kThreads, ACROSS_A> a;
    Staged<T, BN, C::kThreads, ACROSS_B> b;
    constexpr int kLoads = a.kLoads + b.kLoads;
    static_assert((S - 1) * kLoads < 64);
    a.open(p.a, m0, p.m, wave, lane);
    b.open(p.b, n0, p.n, wave, lane);
    const int wm = wave / C::WN * (BM / C::WM), wn = wave % C::WN * (BN / C::WN);
    a.place(wm, lane);
    b.place(wn, lane);

    f32x4 acc[FM][FN] = {};
    struct Half {
        u32x4 a[FM], b[FN];
    };
    const auto read = [&](Half &h, uint32_t t, int s) {
        const int8_t *stage = lds + t % S * C::kStage;
        b.read(stage + a.kBytes, s, h.b);
        a.read(stage, s, h.a);
    };
    const auto compute = [&](const Half &h) { mma<T>(h.b, h.a, acc); };
    const auto fetch = [&](uint32_t t) {
        int8_t *stage = lds + t % S * C::kStage;
        a.fetch(stage, t, wave);
        b.fetch(stage + a.kBytes, t, wave);
    };
    const auto fetch_any = [&](uint32_t t) {
        if (t < whole) {
            fetch(t);
        } else if (t < steps) {
            int8_t *stage = lds + t % S * C::kStage;
            a.fetch_rest(stage, t, p.k, wave, lane);
            b.fetch_rest(stage + a.kBytes, t, p.k, wave, lane);
        }
    };
    if constexpr (C::kTurns) {
        // Of the two waves on a SIMD one reads and loads while the other one sums, and the
        // waves meet between the turns: the second four are a turn behind the first four.
        // A step has four turns of a wave: its first half is read, and summed, then its
        // second half.  The step after next is loaded to the place of the step before,
        // which all have read, and has landed two turns later.
        const auto turn_end = [](auto reads) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (reads) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        const auto sum = [&](const Half &h) {
            __builtin_amdgcn_s_setprio(1);
            compute(h);
            __builtin_amdgcn_s_setprio(0);
            turn_end(std::false_type{});
        };
        fetch_any(0);
        fetch_any(1);
        step_barrier<0>();
        if (wave >= 4) turn_end(std::false_type{});
        Half h;
        for (uint32_t t = 0; t < steps; ++t) {
            read(h, t, 0);
            if (t > 0) fetch_any(t + 1);
            turn_end(std::true_type{});
            sum(h);
            read(h, t, 1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            turn_end(std::true_type{});
            sum(h);
        }
        if (wave < 4) turn_end(std::false_type{});
    } else {
        // A step's second half is read while the first is summed, the next step's
        // first half while the second is.  Between the two the waves meet: all have read the
        // step, so that its place is free, and the next step has landed once no more
        // loads are under way than those of the S - 2 steps behind it.
        Half first, second;
        for (int t = 0; t < S; ++t) fetch_any(t);
        if (steps > 0) {
            if (S <= whole) step_barrier<(S - 1) * kLoads>();
            else step_barrier<0>();
            read(first, 0, 0);
        }
        uint32_t t = 0;
        for (; t + S < whole; ++t) {
            read(second, t, 1);
            compute(first);
            step_barrier<(S - 2) * kLoads>();
            fetch(t + S);
            read(first, t + 1, 0);
            compute(second);
        }
        for (; t < steps; ++t) { // the last ones, not all of them direct loads
            read(second, t, 1);
            compute(first);
            step_barrier<0>();
            if (t + S < steps) fetch_any(t + S);
            if (t + 1 < steps) read(first, t + 1, 0);
            compute(second);
        }
    }
    __syncthreads(); // LDS is the epilogue's
    epilogue.template finish<C>(acc, Place{m0 + wm + lane % 16, n0 + wn + lane / 16 * 4, m0, n0 / BN, wave % C::WN}, p,
                                (float *)lds);
}

// The place of a target among a lane's columns from `first` on, 4 of every 16; ~0 where it
// is none of them.
template <int FN> __device__ __forceinline__ uint32_t place_among(uint64_t target, uint64_t first) {
    const uint64_t d = target - first;
    return d < 16 * FN && d % 16 < 4 ? (uint32_t)d : ~0u;
}

// The largest logit of each row of the tile, the sum of e^(logit - largest), and the
// target's logit: [tiles of columns][rows].  A tile of 256 x 256 has 128 logits a lane:
// what few rows or the last columns alone need stands behind a wave's branch.  1427 x 47616
// x 169 bf16 took 121 us where each logit was compared with the target and the end, and 93
// so; it takes 57 with the last step's loads under way together.
struct TileStats {
    float2 *stats;
    float *picked;
    const uint32_t *targets;
    template <typename C>
    __device__ __forceinline__ void finish(f32x4 (&acc)[C::FM][C::FN], const Place &at, const Product &p, float *lds) {
        float2 *joined = (float2 *)lds; // [WN][BM]
        if (__any(at.n + 16 * (C::FN - 1) + 4 > p.n)) {
#pragma unroll
            for (int i = 0; i < C::FM; ++i)
#pragma unroll
                for (int j = 0; j < C::FN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at.n + 16 * j + e >= p.n) acc[i][j][e] = -__builtin_inff();
        }
        uint32_t row_targets[C::FM];
#pragma unroll
        for (int i = 0; i < C::FM; ++i) row_targets[i] = targets[min(at.m + 16 * i, p.m - 1)];
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = at.m + 16 * i, target = row_targets[i];
            const uint32_t hit = target < p.n && row < p.m ? place_among<C::FN>(target, at.n) : ~0u;
            if (__any(hit != ~0u)) {
                float logit = 0.0f;
#pragma unroll
                for (int j = 0; j < C::FN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) logit = hit == 16u * j + e ? acc[i][j][e] : logit;
                if (hit != ~0u) picked[row] = logit;
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top > -__builtin_inff() ? top : 0.0f; // of no logits, or of none above -inf
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += exp_near(acc[i][j][e] - from);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane_id() < 16) joined[at.wave_n * C::BM + (int)(row - at.m0)] = float2{top, sum};
        }
        __syncthreads();
        for (uint32_t r = threadIdx.x; r < C::BM; r += C::kThreads) {
            if (at.m0 + r >= p.m) break;
            float2 s = joined[r];
#pragma unroll
            for (int w = 1; w < C::WN; ++w) s = join(s, joined[w * C::BM + r]);
            stats[at.tile_n * p.m + at.m0 + r] = s;
        }
    }
    static __device__ __forceinline__ float2 join(float2 a, float2 b) {
        const float top = fmaxf(a.x, b.x), from = top > -__builtin_inff() ? top : 0.0f;
        return {top, a.y * exp_of(a.x - from) + b.y * exp_of(b.x - from)};
    }
};

// COUNT columns of a row at the alignment of the elements, those before `end`.
template <typename T, int COUNT>
__device__ __forceinline__ void store_columns(T *p, uint64_t n, uint64_t end, const T (&v)[COUNT]) {
    typedef T any __attribute__((ext_vector_type(COUNT), aligned(sizeof(T))));
    if (n + COUNT <= end) {
        any all;
#pragma unroll
        for (int e = 0; e < COUNT; ++e) all[e] = v[e];
        *(any *)p = all;
    } else {
#pragma unroll
        for (int e = 0; e < COUNT; ++e)
            if (n + e < end) p[e] = v[e];
    }
}

// A wave's fragments of 16 rows to memory: `row` is this lane's row, from the tile's
// columns of the wave on, which begin at column `n`.  Of bf16 a lane holds 8 bytes of each 32.
// Two fragments are exchanged among the four lanes of a row, such that these store 64
// bytes side by side: the fragments' and the lanes' places are bits that change places.
// G of 4096 x 16384 x 64 takes 52.5 us with 8 bytes a lane and 42.5 with 16.
template <typename T, int FN>
__device__ __forceinline__ void store_fragments(T *row, bool is_in, uint64_t n, uint64_t end, const f32x4 (&v)[FN]) {
    const int q = lane_id() / 16;
    if constexpr (sizeof(T) == 4 || FN % 2 != 0) {
        if (!is_in) return;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int c = 16 * j + 4 * q;
            const T each[4] = {(T)v[j][0], (T)v[j][1], (T)v[j][2], (T)v[j][3]};
            store_columns(row + c, n + c, end, each);
        }
    } else {
        const auto pack = [](float a, float b) {
            typedef bf16 pair __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, pair{(bf16)a, (bf16)b});
        };
#pragma unroll
        for (int h = 0; h < FN / 2; ++h) {
            u32x4 all;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const uint32_t first = pack(v[2 * h][2 * d], v[2 * h][2 * d + 1]);
                const uint32_t second = pack(v[2 * h + 1][2 * d], v[2 * h + 1][2 * d + 1]);
                const auto by_half = __builtin_amdgcn_permlane32_swap(first, second, false, false);
                const auto by_row = __builtin_amdgcn_permlane16_swap(by_half[0], by_half[1], false, false);
                all[d] = by_row[0];
                all[2 + d] = by_row[1];
            }
            const int c = 32 * h + 8 * q;
            struct Each {
                T v[8];
            };
            if (is_in) store_columns(row + c, n + c, end, __builtin_bit_cast(Each, all).v);
        }
    }
}

// G of a piece of the vocabulary that begins at `first`.
template <typename T> struct TileGradient {
    T *g;
    uint64_t pitch; // elements
    uint64_t first, vocab;
    const uint32_t *targets;
    const float *lse, *grad, *most;
    template <typename C>
    __device__ __forceinline__ void finish(f32x4 (&acc)[C::FM][C::FN], const Place &at, const Product &p, float *) {
        // What all the rows need is asked for together.
        uint32_t row_targets[C::FM];
        float row_lse[C::FM], row_grad[C::FM];
        const float largest = *most;
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = min(at.m + 16 * i, p.m - 1);
            row_targets[i] = targets[row], row_lse[i] = lse[row], row_grad[i] = grad[row];
        }
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = at.m + 16 * i, target = row_targets[i];
            const bool counts = target < vocab;
            const float from = row_lse[i], weight = counts ? row_grad[i] / largest : 0.0f;
            const uint32_t hit = place_among<C::FN>(target, first + at.n);
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[i][j][e] = sizeof(T) == 2 ? exp_near(acc[i][j][e] - from) : exp_of(acc[i][j][e] - from);
            if (__any(hit != ~0u)) {
#pragma unroll
                for (int j = 0; j < C::FN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] -= hit == 16u * j + e ? 1.0f : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < C::FN; ++j) acc[i][j] *= weight;
            if (__any(!counts)) { // whatever the logits were
#pragma unroll
                for (int j = 0; j < C::FN; ++j)
                    if (!counts) acc[i][j] = f32x4{0, 0, 0, 0};
            }
            const uint64_t n = at.n - lane_id() / 16 * 4;
            store_fragments(g + row * pitch + n, row < p.m, n, p.n, acc[i]);
        }
    }
};

// scale·(sum + what earlier pieces summed up): to `out`, or, the sum alone, to `after`, where
// it goes on to the next piece or is a part's.  Rows without a target get zeros where
// `targets` is given.
template <typename T> struct TileOut {
    const float *scale;
    const float *before; // may be null
    float *after;        // may be null
    T *out;
    uint64_t sum_pitch;
    int64_t out_stride;
    const uint32_t *targets; // may be null
    uint64_t vocab;
    template <typename C>
    __device__ __forceinline__ void finish(f32x4 (&acc)[C::FM][C::FN], const Place &at, const Product &p, float *) {
        const float by = scale ? *scale : 1.0f; // parts have none
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = at.m + 16 * i;
            const bool is_in = row < p.m;
            if (before || after) {
#pragma unroll
                for (int j = 0; j < C::FN; ++j) {
                    const uint64_t n = at.n + 16 * j;
                    if (!is_in || n >= p.n) continue;
                    if (before) acc[i][j] += *(const f32x4 *)(before + row * sum_pitch + n); // the pitch is whole vectors
                    if (after) *(f32x4 *)(after + (blockIdx.y * p.m + row) * sum_pitch + n) = acc[i][j];
                }
                if (after) continue;
            }
            const bool is_left_out = is_in && targets && targets[row] >= vocab;
#pragma unroll
            for (int j = 0; j < C::FN; ++j) acc[i][j] = is_left_out ? f32x4{0, 0, 0, 0} : acc[i][j] * by;
            const uint64_t n = at.n - lane_id() / 16 * 4;
            store_fragments(out + (int64_t)row * out_stride + (int64_t)n, is_in, n, p.n, acc[i]);
        }
    }
};

// The parts' sums of four columns, added up in order, eight asked for at a time.
__device__ __forceinline__ f32x4 sum_of_parts(const float *at, uint32_t count, uint64_t apart) {
    f32x4 v = *(const f32x4 *)at;
    uint32_t p = 1;
    for (; p + 8 <= count; p += 8) {
        f32x4 more[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) more[i] = *(const f32x4 *)(at + (p + i) * apart);
#pragma unroll
        for (int i = 0; i < 8; ++i) v += more[i];
    }
    for (; p < count; ++p) v += *(const f32x4 *)(at + p * apart);
    return v;
}

// A wave's 64 vectors of the result, such that few of them are spread over many CUs.
template <typename T>
__global__ __launch_bounds__(64) void fold_parts_kernel(const float *parts, uint32_t count, uint64_t m, uint64_t n,
                                                       TileOut<T> out) {
    const uint64_t vectors = out.sum_pitch / 4;
    for (uint64_t i = (uint64_t)blockIdx.x * 64 + threadIdx.x; i < m * vectors; i += (uint64_t)gridDim.x * 64) {
        const uint64_t row = i / vectors, c = i % vectors * 4, at = row * out.sum_pitch + c;
        f32x4 v = sum_of_parts(parts + at, count, m * out.sum_pitch);
        if (out.before) v += *(const f32x4 *)(out.before + at);
        if (out.after) {
            *(f32x4 *)(out.after + at) = v;
        } else {
            v *= *out.scale;
            if (out.targets && out.targets[row] >= out.vocab) v = f32x4{0, 0, 0, 0};
            const T each[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            store_columns(out.out + (int64_t)row * out.out_stride + (int64_t)c, c, n, each);
        }
    }
}

// Logits of parts to what TileStats leaves of a tile: 1024 columns of a row, a block.  The
// rows from `first` on.
__global__ __launch_bounds__(256) void fold_stats_kernel(const float *parts, uint32_t count, uint64_t m, uint64_t n,
                                                        uint64_t pitch, TileStats out, uint64_t first) {
    __shared__ float2 joined[256 / kWave];
    const uint64_t row = first + blockIdx.x, c = ((uint64_t)blockIdx.y * 256 + threadIdx.x) * 4, target = out.targets[row];
    f32x4 v = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
    if (c < n) {
        const f32x4 all = sum_of_parts(parts + row * pitch + c, count, m * pitch);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (c + e < n) v[e] = all[e];
            if (c + e == target && target < n) out.picked[row] = all[e];
        }
    }
    float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const float from = top > -__builtin_inff() ? top : 0.0f;
    float sum = exp_near(v[0] - from) + exp_near(v[1] - from) + exp_near(v[2] - from) + exp_near(v[3] - from);
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d);
    if (lane_id() == 0) joined[threadIdx.x / kWave] = float2{top, sum};
    __syncthreads();
    if (threadIdx.x) return;
    float2 s = joined[0];
#pragma unroll
    for (int w = 1; w < 256 / kWave; ++w) s = TileStats::join(s, joined[w]);
    out.stats[blockIdx.y * m + row] = s;
}

// Logits of parts to G, as TileGradient makes it.
template <typename T>
__global__ __launch_bounds__(64) void fold_gradient_kernel(const float *parts, uint32_t count, uint64_t m, uint64_t n,
                                                          uint64_t pitch, TileGradient<T> out) {
    const uint64_t vectors = pitch / 4;
    for (uint64_t i = (uint64_t)blockIdx.x * 64 + threadIdx.x; i < m * vectors; i += (uint64_t)gridDim.x * 64) {
        const uint64_t row = i / vectors, c = i % vectors * 4, target = out.targets[row];
        const f32x4 v = sum_of_parts(parts + row * pitch + c, count, m * pitch);
        const bool counts = target < out.vocab;
        const float from = out.lse[row], weight = counts ? out.grad[row] / *out.most : 0.0f;
        T each[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float s = exp_of(v[e] - from) - (out.first + c + e == target ? 1.0f : 0.0f);
            each[e] = (T)(counts ? s * weight : 0.0f);
        }
        store_columns(out.g + row * out.pitch + c, c, n, each);
    }
}

template <typename T, typename C, bool ACROSS_A, bool ACROSS_B, typename E>
hx_status launch_tiles(const Product &p, uint32_t parts, const E &epilogue, hipStream_t stream) {
    const auto kernel = product_kernel<T, C, ACROSS_A, ACROSS_B, E>;
    static std::atomic<uint64_t> allowed{0};
    HX_TRY(allow_lds((const void *)kernel, C::kLds, allowed));
    const uint64_t tm = ceil_div(p.m, C::BM), tn = ceil_div(p.n, C::BN);
    // Tiles are counted in 32 bits; no operands or workspace that fit a device have more.
    if (tm * tn > 0xFFFFFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "product of %llu tiles exceeds the grid range", (unsigned long long)(tm * tn));
    constexpr uint64_t kMost = tiles_a_launch(C::kThreads);
    for (uint64_t first = 0; first < tm * tn; first += kMost)
        hipLaunchKernelGGL(kernel, dim3((uint32_t)std::min(kMost, tm * tn - first), parts), dim3(C::kThreads), C::kLds,
                           stream, p, epilogue, (uint32_t)tm, (uint32_t)tn, (uint32_t)first);
    return check_launch("product_kernel");
}
template <typename T, bool ACROSS_A, bool ACROSS_B, typename E>
hx_status launch_product(Product p, const ProductCut &cut, const E &epilogue, hipStream_t stream) {
    if (p.m == 0 || p.n == 0) return HX_OK;
    // A tile's places from its first row on are counted in 32 bits.
    const auto fits = [&](const Operand &o, uint64_t rows, bool is_across) {
        const uint64_t most = is_across ? std::min<uint64_t>(p.k, kDepth / sizeof(T)) : std::min<uint64_t>(rows, 256);
        return o.stride >= 0 && (uint64_t)o.stride * most < 0xFFFF0000ull;
    };
    if (!fits(p.a, p.m, ACROSS_A) || !fits(p.b, p.n, ACROSS_B))
        return fail(HX_ERR_DISPATCH_FAILED, "product of rows %lld and %lld bytes apart exceeds the range of a tile",
                    (long long)p.a.stride, (long long)p.b.stride);
    p.span = cut.span;
    switch (cut.tile) {
    case ProductTile::k256x256:
        return launch_tiles<T, Tile<256, 256, 2, 4, 2>, ACROSS_A, ACROSS_B>(p, cut.parts, epilogue, stream);
    case ProductTile::k128x128:
        return launch_tiles<T, Tile<128, 128, 2, 4, 4>, ACROSS_A, ACROSS_B>(p, cut.parts, epilogue, stream);
    case ProductTile::k64x128:
        return launch_tiles<T, Tile<64, 128, 2, 4, 3>, ACROSS_A, ACROSS_B>(p, cut.parts, epilogue, stream);
    case ProductTile::k64x64:
        return launch_tiles<T, Tile<64, 64, 2, 2, 4>, ACROSS_A, ACROSS_B>(p, cut.parts, epilogue, stream);
    case ProductTile::k32x64:
        return launch_tiles<T, Tile<32, 64, 1, 4, 6>, ACROSS_A, ACROSS_B>(p, cut.parts, epilogue, stream);
    }
    return HX_OK;
}
// A product's parts of k, [parts][m][pitch].
template <typename T, bool ACROSS_A, bool ACROSS_B>
hx_status launch_parts(const Product &p, const ProductCut &cut, float *parts, uint64_t pitch, hipStream_t stream) {
    const TileOut<T> part{nullptr, nullptr, parts, nullptr, pitch, 0, nullptr, 0};
    return launch_product<T, ACROSS_A, ACROSS_B>(p, cut, part, stream);
}
constexpr uint64_t kBlocksOf256 = tiles_a_launch(256); // of a launch
inline dim3 fold_blocks(uint64_t m, uint64_t pitch) {
    return dim3((uint32_t)std::min<uint64_t>(ceil_div(m * (pitch / 4), 64), 1 << 18));
}
// A product to `out`, in parts where that is shorter.
template <typename T, bool ACROSS_A, bool ACROSS_B>
hx_status launch_sums(const Product &p, const TileOut<T> &out, float *parts, hipStream_t stream) {
    const ProductCut cut = product_cut(p.m, p.n, p.k, sizeof(T));
    if (cut.parts <= 1 || p.m == 0 || p.n == 0) return launch_product<T, ACROSS_A, ACROSS_B>(p, cut, out, stream);
    HX_TRY((launch_parts<T, ACROSS_A, ACROSS_B>)(p, cut, parts, out.sum_pitch, stream));
    hipLaunchKernelGGL(fold_parts_kernel<T>, fold_blocks(p.m, out.sum_pitch), dim3(64), 0, stream, parts, cut.parts, p.m,
                       p.n, out);
    return check_launch("fold_parts_kernel");
}

// ------------------------------------------------------------------ rows

// The largest finite |grad| of a row that has a target; 1 where there is none.
struct Largest {
    const float *grad;
    const uint32_t *targets;
    uint64_t rows, vocab;
    float *most; // null: not asked for
    __device__ void find() const {
        constexpr int kEach = 8;
        float top = 0.0f;
        for (uint64_t first = threadIdx.x; first < rows; first += 256 * kEach) {
            float g[kEach];
            uint32_t target[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint64_t r = min(first + i * 256, rows - 1);
                g[i] = fabsf(grad[r]), target[i] = targets[r];
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (target[i] < vocab && g[i] < __builtin_inff()) top = fmaxf(top, g[i]);
        }
        __shared__ float tops[256 / kWave];
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        if (lane_id() == 0) tops[threadIdx.x / kWave] = top;
        __syncthreads();
        if (threadIdx.x) return;
        for (int i = 1; i < 256 / kWave; ++i) top = fmaxf(top, tops[i]);
        *most = top > 0.0f ? top : 1.0f;
    }
};

// Rows at any byte, copied to rows of whole steps with zeros after their ends, and
// zeros in the place of rows that have no target where `targets` is given: whatever such a
// row holds, it adds nothing.  A last block looks for the largest gradient meanwhile.
__global__ __launch_bounds__(256) void copy_rows_kernel(const int8_t *from, int64_t stride, uint64_t rows, uint32_t bytes,
                                                       int8_t *to, uint32_t pitch, const uint32_t *targets,
                                                       uint64_t vocab, Largest largest) {
    const uint32_t chunks = pitch / 16, blocks = gridDim.x - (largest.most ? 1 : 0);
    if (blockIdx.x == blocks) return largest.find();
    for (uint64_t first = (uint64_t)blockIdx.x * 256; first < rows * chunks; first += (uint64_t)blocks * 256) {
        const uint32_t i = (uint32_t)(first % chunks) + threadIdx.x, at = i % chunks * 16;
        const uint64_t r = first / chunks + i / chunks;
        if (r >= rows) return;
        u32x4 v = {0, 0, 0, 0};
        if (!targets || targets[r] < vocab) v = load_bytes(from + (int64_t)r * stride, at, bytes);
        *(u32x4 *)(to + r * pitch + at) = v;
    }
}

// The tiles' sums of a row, joined in one order: ROWS rows a block, 256 / ROWS threads a
// row.  Many rows are read side by side, few rows by more threads.  The rows from `first` on.
template <int ROWS>
__global__ __launch_bounds__(256) void join_stats_kernel(const float2 *stats, const float *picked,
                                                         const uint32_t *targets, uint64_t tiles, uint64_t rows,
                                                         uint64_t vocab, float *loss, float *lse, uint64_t first) {
    constexpr int kThreads = 256 / ROWS;
    __shared__ float2 part[kThreads][ROWS];
    const uint64_t row = first + (uint64_t)blockIdx.x * ROWS + threadIdx.x % ROWS;
    float2 s = {-__builtin_inff(), 0.0f};
    if (row < rows)
        for (uint64_t t = threadIdx.x / ROWS; t < tiles; t += kThreads) s = TileStats::join(s, stats[t * rows + row]);
    part[threadIdx.x / ROWS][threadIdx.x % ROWS] = s;
#pragma unroll
    for (int half = kThreads / 2; half > 0; half /= 2) {
        __syncthreads();
        if ((int)threadIdx.x / ROWS < half) {
            s = TileStats::join(s, part[threadIdx.x / ROWS + half][threadIdx.x % ROWS]);
            part[threadIdx.x / ROWS][threadIdx.x % ROWS] = s;
        }
    }
    if (threadIdx.x >= ROWS || row >= rows) return;
    const float sum = logf(s.y);
    if (lse) lse[row] = s.x + sum;
    // Not lse - picked: where the target has the largest logit, the digits of `sum` would
    // end at the logits' rounding.
    loss[row] = targets[row] < vocab ? s.x - picked[row] + sum : 0.0f;
}

template <typename T>
hx_status copy_rows(const void *from, int64_t stride, uint64_t rows, uint64_t width, void *to, const uint32_t *targets,
                    uint64_t vocab, const Largest &largest, hipStream_t stream) {
    const uint32_t bytes = (uint32_t)(width * sizeof(T)), pitch = (uint32_t)round_up(bytes, kDepth);
    const uint64_t blocks = std::min<uint64_t>(ceil_div(rows * (pitch / 16), 256), 1 << 22) + (largest.most ? 1 : 0);
    if (blocks == 0) return HX_OK;
    hipLaunchKernelGGL(copy_rows_kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, (const int8_t *)from,
                       stride * (int64_t)sizeof(T), rows, bytes, (int8_t *)to, pitch, targets, vocab, largest);
    return check_launch("copy_rows_kernel");
}

template <typename T> hx_status launch(const CrossEntropyArgs &a, void *ws, hipStream_t stream) {
    const CrossEntropyPlan plan = cross_entropy_plan(a);
    char *base = (char *)ws;
    float2 *stats = (float2 *)(base + plan.stats);
    float *picked = (float *)(base + plan.picked);
    const int64_t size = sizeof(T), row = (int64_t)round_up(a.width * size, kDepth);
    Product p{{(const int8_t *)a.x, a.x_stride * size}, {(const int8_t *)a.weight, a.weight_stride * size}, a.rows,
              a.vocab, a.width, 0};
    if (plan.copies) {
        HX_TRY(copy_rows<T>(a.x, a.x_stride, a.rows, a.width, base + plan.x, nullptr, 0, {}, stream));
        HX_TRY(copy_rows<T>(a.weight, a.weight_stride, a.vocab, a.width, base + plan.weight, nullptr, 0, {}, stream));
        p.k = row / size; // zeros after the rows' ends
        p.a = {(const int8_t *)base + plan.x, row};
        p.b = {(const int8_t *)base + plan.weight, row};
    }
    const TileStats out{stats, picked, a.targets};
    if (plan.cut.parts > 1) {
        float *parts = (float *)(base + plan.parts);
        const uint64_t pitch = round_up(a.vocab, 4);
        HX_TRY((launch_parts<T, false, false>)(p, plan.cut, parts, pitch, stream));
        for (uint64_t first = 0; first < a.rows; first += kBlocksOf256)
            hipLaunchKernelGGL(fold_stats_kernel, dim3((uint32_t)std::min(kBlocksOf256, a.rows - first), (uint32_t)plan.tiles_n),
                               dim3(256), 0, stream, parts, plan.cut.parts, a.rows, a.vocab, pitch, out, first);
        HX_TRY(check_launch("fold_stats_kernel"));
    } else {
        HX_TRY((launch_product<T, false, false>)(p, plan.cut, out, stream));
    }
    const uint64_t tiles = a.vocab ? plan.tiles_n : 0;
    const auto join = [&](auto kernel, uint64_t rows) { // of a block
        for (uint64_t first = 0; first < a.rows; first += kBlocksOf256 * rows) {
            const uint64_t blocks = std::min(kBlocksOf256, ceil_div(a.rows - first, rows));
            hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, stats, picked, a.targets, tiles, a.rows,
                               a.vocab, a.loss, a.lse, first);
        }
        return check_launch("join_stats_kernel");
    };
    return a.rows >= 2048 ? join(join_stats_kernel<16>, 16) : join(join_stats_kernel<1>, 1);
}

template <typename T> hx_status launch(const CrossEntropyGradArgs &a, void *ws, hipStream_t stream) {
    const CrossEntropyGradPlan plan = cross_entropy_grad_plan(a);
    char *base = (char *)ws;
    float *most = (float *)base;
    const int64_t size = sizeof(T), row = (int64_t)round_up(a.width * size, kDepth);
    const Operand x{(const int8_t *)base + plan.x, row};
    HX_TRY(copy_rows<T>(a.x, a.x_stride, a.rows, a.width, base + plan.x, a.targets, a.vocab,
                        Largest{a.grad, a.targets, a.rows, a.vocab, most}, stream));
    float *sums = (float *)(base + plan.sums), *parts = (float *)(base + plan.parts);
    T *g = (T *)(base + plan.g);
    const Operand go{(const int8_t *)g, (int64_t)plan.piece_pitch * size};
    for (uint64_t first = 0; first < a.vocab || first == 0; first += plan.piece) {
        const uint64_t n = std::min<uint64_t>(plan.piece, a.vocab - first);
        const T *from = (const T *)a.weight + (int64_t)first * a.weight_stride;
        Operand w{(const int8_t *)from, a.weight_stride * size};
        if (plan.copies) {
            HX_TRY(copy_rows<T>(from, a.weight_stride, n, a.width, base + plan.weight, nullptr, 0, {}, stream));
            w = {(const int8_t *)base + plan.weight, row};
        }
        const Product logits{x, w, a.rows, n, plan.copies ? row / size : a.width, 0};
        const TileGradient<T> to{g, plan.piece_pitch, first, a.vocab, a.targets, a.lse, a.grad, most};
        const ProductCut cut = product_cut(a.rows, n, a.width, size);
        if (cut.parts > 1 && n > 0) {
            const uint64_t pitch = round_up(n, 4);
            HX_TRY((launch_parts<T, false, false>)(logits, cut, parts, pitch, stream));
            hipLaunchKernelGGL(fold_gradient_kernel<T>, fold_blocks(a.rows, pitch), dim3(64), 0, stream, parts, cut.parts,
                               a.rows, n, pitch, to);
            HX_TRY(check_launch("fold_gradient_kernel"));
        } else {
            HX_TRY((launch_product<T, false, false>)(logits, cut, to, stream));
        }
        if (a.grad_x) {
            const bool is_last = first + n >= a.vocab;
            const TileOut<T> out{most, first ? sums : nullptr, is_last ? nullptr : sums, (T *)a.grad_x, plan.sums_pitch,
                                 a.grad_x_stride, a.targets, a.vocab};
            HX_TRY((launch_sums<T, false, true>)(Product{go, w, a.rows, a.width, n, 0}, out, parts, stream));
        }
        if (a.grad_weight) {
            const TileOut<T> out{most, nullptr, nullptr, (T *)a.grad_weight + (int64_t)first * a.grad_weight_stride, plan.sums_pitch,
                                 a.grad_weight_stride, nullptr, 0};
            HX_TRY((launch_sums<T, true, true>)(Product{go, x, n, a.width, a.rows, 0}, out, parts, stream));
        }
    }
    return HX_OK;
}

} // namespace

uint64_t cross_entropy_workspace_bytes(const CrossEntropyArgs &args) {
    return args.rows ? cross_entropy_plan(args).bytes : 0;
}
hx_status launch_cross_entropy(const CrossEntropyArgs &args, void *ws, hipStream_t stream) {
    if (args.rows == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, ws, stream) : launch<bf16>(args, ws, stream);
}

uint64_t cross_entropy_grad_workspace_bytes(const CrossEntropyGradArgs &args) {
    return args.grad_x || args.grad_weight ? cross_entropy_grad_plan(args).bytes : 0;
}
hx_status launch_cross_entropy_grad(const CrossEntropyGradArgs &args, void *ws, hipStream_t stream) {
    if (!args.grad_x && !args.grad_weight) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, ws, stream) : launch<bf16>(args, ws, stream);
}

} // namespace hx
