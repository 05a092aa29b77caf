// Softmax cross entropy of the logits x·wᵀ over a vocabulary, without keeping the
// logits (hx_linear_cross_entropy), and its backward pass, for gfx950.
//
// Forward: the product goes tile by tile; a tile leaves, for each of its rows, the
// largest logit and the sum of the exponentials of the others' distances from it, and
// the target's logit where it lies in the tile.  A second launch joins the tiles.
//
// Backward, a piece of the vocabulary after another: the logits again, as
//   G = (grad / most)·(e^(logit - lse) - [target]),   most = max |grad|,
// in the operands' type, then dx += G·w and dw = Gᵀ·x on matrix instructions, with
// sums in f32 that are multiplied by `most` at the end.  With the mean's gradients,
// which are all alike, the factor is 1 and G keeps the places of e^(logit - lse):
// a factor's rounding would be the same in every term of a sum and stay in it.
#include "hx_internal.hpp"
#include "layer_device.hpp"

#include <atomic>
#include <type_traits>

namespace hx {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kDepth = 128; // bytes of a row a step

// 16 bytes of k of 16 rows of either operand.  Of f32 these are four instructions,
// each with an element of every lane: k in another order, the same for both.
template <typename T> __device__ __forceinline__ f32x4 mma(u32x4 b, u32x4 a, f32x4 sum) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a),
                                                       sum, 0, 0, 0);
    } else {
        const f32x4 fb = __builtin_bit_cast(f32x4, b), fa = __builtin_bit_cast(f32x4, a);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[i], fa[i], sum, 0, 0, 0);
        return sum;
    }
}

// 16 bytes of a row from `k` on, zeros from `end` on.
__device__ __forceinline__ u32x4 load_bytes(const int8_t *row, uint32_t k, uint32_t end) {
    if (k + 16 <= end) return *(const u32x4_any *)(row + k);
    u32x4 v = {0, 0, 0, 0};
    if (k >= end) return v;
    if (end >= 16) {
        const u32x4 last = *(const u32x4_any *)(row + end - 16);
        return __builtin_bit_cast(u32x4, __builtin_bit_cast(unsigned __int128, last) >> (8 * (k + 16 - end)));
    }
    for (uint32_t i = 0; k + i < end; ++i) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
    return v;
}

// e^x for x of at most about 0, to a rounding or two: with the rest that the product
// with log2(e) leaves.
__device__ __forceinline__ float exp_of(float x) {
    constexpr float kLog2e = 1.44269502f, kLow = 1.92596299e-8f;
    if (x < -120.0f) return 0.0f;
    const float t = x * kLog2e, low = __builtin_fmaf(x, kLog2e, -t) + x * kLow;
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, low * 0.693147181f, e);
}

// ---------------------------------------------------------------- product
// out[m, n] = Σ_k a[m, k]·b[n, k], handed to an epilogue in tiles of BM x BN.  The
// tile's WM x WN waves each take a part.  A step's 128 bytes of k of each row
// lie in LDS as eight chunks of 16, chunk c of row r at place c ^ (r % 8), so that the
// 16 rows that a matrix instruction reads at one c fall on all banks.  Loads go from
// memory to LDS without registers, S - 1 steps ahead; they need rows that begin
// on dwords.
struct Product {
    const int8_t *a, *b;
    uint64_t m, n;
    uint32_t k;                // bytes
    int64_t a_stride, b_stride; // bytes
};

// The barrier between steps is written out: all of the wave's LDS reads and
// writes and all but its last N loads have ended when it is passed.
template <int N> __device__ __forceinline__ void step_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <int BM_, int BN_, int WM_, int WN_, int S_> struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
    static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
    static constexpr int kRows = BM + BN, kStage = kRows * kDepth, kLds = kStage * S;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    static constexpr int kLoads = kRows * 8 / kThreads; // chunks a thread and step
    static_assert(kLds <= 160 * 1024 && kLoads * kThreads == kRows * 8 && (S - 2) * kLoads < 64);
};

// What an epilogue knows of its place: lane l has, of fragment (i, j), the sums of
// row m + 16·i and columns n + 16·j + 0..3.
struct Place {
    uint64_t m, n;      // this lane's first row and column
    uint64_t m0, tile_n; // the tile's first row; its place among the columns' tiles
    int wave_m, wave_n;
};

template <typename T, typename C, typename E>
__global__ __launch_bounds__(C::kThreads, 2) void product_kernel(Product p, E epilogue, uint32_t tiles_m,
                                                                uint32_t tiles_n) {
    constexpr int BM = C::BM, BN = C::BN, FM = C::FM, FN = C::FN, kLoads = C::kLoads, S = C::S;
    extern __shared__ __align__(16) int8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

    // Blocks go to the eight XCDs in turn: each XCD takes a run of tiles, in
    // strips of eight tiles of m so that its L2 serves both operands.
    const uint32_t total = tiles_m * tiles_n, share = total / 8, rest = total % 8;
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t tile = xcd * share + min(xcd, rest) + turn;
    const uint32_t strip = tile / (8 * tiles_n), in_strip = tile % (8 * tiles_n);
    const uint32_t height = min(8u, tiles_m - 8 * strip);
    const uint64_t m0 = (uint64_t)(8 * strip + in_strip % height) * BM, n0 = (uint64_t)(in_strip / height) * BN;

    const uint32_t k_end = p.k, steps = (k_end + kDepth - 1) / kDepth, whole = k_end / kDepth;
    // A thread's chunk of each row that it loads: rows past the operands
    // repeat the last one and are dropped at the end.
    const uint32_t row0 = wave * (kLoads * 8) + lane / 8, chunk = (lane % 8 ^ (row0 % 8)) * 16;
    const int8_t *src[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const uint32_t r = row0 + j * 8;
        src[j] = r < BM ? p.a + (int64_t)min(m0 + r, p.m - 1) * p.a_stride
                        : p.b + (int64_t)min(n0 + (r - BM), p.n - 1) * p.b_stride;
    }
    const uint32_t to = wave * (kLoads * 1024); // this wave's first row in a stage

    const int wm = wave / C::WN * (BM / C::WM), wn = wave % C::WN * (BN / C::WN);
    const uint32_t swizzled = (lane / 16 ^ (lane % 8)) * 16; // of k bytes 0..63; 64..127: ^ 64
    const uint32_t at_a = (wm + lane % 16) * kDepth + swizzled, at_b = (BM + wn + lane % 16) * kDepth + swizzled;
    f32x4 acc[FM][FN] = {};
    const auto compute = [&](const int8_t *stage) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = *(const u32x4 *)(stage + (at_b ^ (64 * s)) + j * (16 * kDepth));
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = *(const u32x4 *)(stage + (at_a ^ (64 * s)) + i * (16 * kDepth));
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
        }
    };
    // Whole steps: no branch in the loads.
    const auto fetch = [&](uint32_t t) {
        int8_t *stage = lds + t % S * C::kStage + to;
        const uint32_t k = t * kDepth + chunk;
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            __builtin_amdgcn_global_load_lds((const void *)(src[j] + k), (lds_void *)(stage + j * 1024), 16, 0, 0);
    };
    // The step of the last, partial 128 bytes: zeros past the end of k.
    const auto fetch_any = [&](uint32_t t) {
        if (t < whole) {
            fetch(t);
        } else if (t < steps) {
            int8_t *stage = lds + t % S * C::kStage + to;
            for (int j = 0; j < kLoads; ++j)
                *(u32x4 *)(stage + j * 1024 + lane * 16) = load_bytes(src[j], t * kDepth + chunk, k_end);
        }
    };
    for (int t = 0; t < S - 1; ++t) fetch_any(t);
    // Step t has landed once no more loads are under way than those of the
    // S - 2 steps behind it.
    uint32_t t = 0;
    for (; t + (S - 1) < whole; ++t) {
        step_barrier<(S - 2) * kLoads>();
        fetch(t + S - 1);
        compute(lds + t % S * C::kStage);
    }
    for (; t < steps; ++t) { // the last ones, not all of them direct loads
        step_barrier<0>();
        if (t + S - 1 < steps) fetch_any(t + S - 1);
        compute(lds + t % S * C::kStage);
    }
    __syncthreads(); // LDS is the epilogue's
    epilogue.template finish<C>(acc, Place{m0 + wm + lane % 16, n0 + wn + lane / 16 * 4, m0, n0 / BN, wm, wave % C::WN},
                                p, (float *)lds);
}

// The largest logit of each row of the tile, the sum of e^(logit - largest), and the
// target's logit: [tiles of columns][rows].
struct TileStats {
    float2 *stats;
    float *picked;
    const uint32_t *targets;
    template <typename C>
    __device__ __forceinline__ void finish(f32x4 (&acc)[C::FM][C::FN], const Place &at, const Product &p, float *lds) {
        float2 *joined = (float2 *)lds; // [WN][BM]
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = at.m + 16 * i;
            const uint64_t target = targets[min(row, p.m - 1)];
            float top = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t n = at.n + 16 * j + e;
                    if (n == target && row < p.m && n < p.n) picked[row] = acc[i][j][e];
                    if (n >= p.n) acc[i][j][e] = -__builtin_inff();
                    top = fmaxf(top, acc[i][j][e]);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top > -__builtin_inff() ? top : 0.0f; // of no logits, or of none above -inf
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < C::FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += exp_of(acc[i][j][e] - from);
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

// G of a piece of the vocabulary that begins at `first`, by rows and by columns.
template <typename T> struct TileGradient {
    T *g, *gt;
    uint64_t pitch, pitch_t; // elements
    uint64_t first, vocab;
    const uint32_t *targets;
    const float *lse, *grad, *most;
    template <typename C>
    __device__ __forceinline__ void finish(f32x4 (&acc)[C::FM][C::FN], const Place &at, const Product &p, float *) {
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = at.m + 16 * i;
            if (row >= p.m) continue;
            const uint64_t target = targets[row];
            const bool counts = target < vocab;
            const float from = lse[row], weight = counts ? grad[row] / *most : 0.0f;
#pragma unroll
            for (int j = 0; j < C::FN; ++j) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t n = at.n + 16 * j + e;
                    const float s = exp_of(acc[i][j][e] - from) - (first + n == target ? 1.0f : 0.0f);
                    v[e] = counts ? s * weight : 0.0f;
                    if (n < p.n) {
                        g[row * pitch + n] = (T)v[e];
                        gt[n * pitch_t + row] = (T)v[e];
                    }
                }
            }
        }
    }
};

// scale·(sum + what earlier pieces summed up): to `out`, or on to the next piece.
template <typename T> struct TileOut {
    const float *scale;
    const float *before; // may be null
    float *after;        // may be null: this is the last piece
    T *out;
    uint64_t sum_pitch;
    int64_t out_stride;
    template <typename C>
    __device__ __forceinline__ void finish(f32x4 (&acc)[C::FM][C::FN], const Place &at, const Product &p, float *) {
        const float by = *scale;
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
            const uint64_t row = at.m + 16 * i;
            if (row >= p.m) continue;
#pragma unroll
            for (int j = 0; j < C::FN; ++j) {
                const uint64_t n = at.n + 16 * j;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (n + e >= p.n) continue;
                    float v = acc[i][j][e];
                    if (before) v += before[row * sum_pitch + n + e];
                    if (after) after[row * sum_pitch + n + e] = v;
                    else out[(int64_t)row * out_stride + (int64_t)(n + e)] = (T)(v * by);
                }
            }
        }
    }
};

template <typename T, typename C, typename E>
hx_status launch_tiles(const Product &p, const E &epilogue, hipStream_t stream) {
    const auto kernel = product_kernel<T, C, E>;
    static std::atomic<uint64_t> allowed{0};
    HX_TRY(allow_lds((const void *)kernel, C::kLds, allowed));
    const uint64_t tm = ceil_div(p.m, C::BM), tn = ceil_div(p.n, C::BN);
    if (tm * tn * C::kThreads > 0xFFFFFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "product of %llu tiles exceeds the grid range", (unsigned long long)(tm * tn));
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tm * tn)), dim3(C::kThreads), C::kLds, stream, p, epilogue,
                       (uint32_t)tm, (uint32_t)tn);
    return check_launch("product_kernel");
}
template <typename T, typename E> hx_status launch_product(const Product &p, const E &epilogue, hipStream_t stream) {
    if (p.m == 0 || p.n == 0) return HX_OK;
    switch (product_tile(p.m, p.n)) {
    case ProductTile::k256x256: return launch_tiles<T, Tile<256, 256, 2, 4, 2>>(p, epilogue, stream);
    case ProductTile::k128x128: return launch_tiles<T, Tile<128, 128, 2, 2, 2>>(p, epilogue, stream);
    case ProductTile::k64x64: return launch_tiles<T, Tile<64, 64, 4, 2, 4>>(p, epilogue, stream);
    case ProductTile::k32x64: return launch_tiles<T, Tile<32, 64, 1, 4, 6>>(p, epilogue, stream);
    }
    return HX_OK;
}

// ------------------------------------------------------------------ rows

// Rows at any byte, copied to rows of whole steps with zeros after their ends.
__global__ __launch_bounds__(256) void copy_rows_kernel(const int8_t *from, int64_t stride, uint64_t rows, uint32_t bytes,
                                                       int8_t *to, uint32_t pitch) {
    const uint32_t chunks = pitch / 16;
    for (uint64_t first = (uint64_t)blockIdx.x * 256; first < rows * chunks; first += (uint64_t)gridDim.x * 256) {
        const uint32_t i = (uint32_t)(first % chunks) + threadIdx.x, at = i % chunks * 16;
        const uint64_t r = first / chunks + i / chunks;
        if (r >= rows) return;
        *(u32x4 *)(to + r * pitch + at) = load_bytes(from + (int64_t)r * stride, at, bytes);
    }
}

// to[c][r] = from[r][c], with zeros in the rows that have no target where `targets`
// is given: whatever such a row holds, it adds nothing.
template <typename T>
__global__ __launch_bounds__(256) void transpose_kernel(const T *from, int64_t stride, uint64_t rows, uint64_t cols,
                                                        T *to, uint64_t pitch, const uint32_t *targets, uint64_t vocab) {
    __shared__ T tile[64][65];
    const uint64_t r0 = (uint64_t)blockIdx.x * 64, c0 = (uint64_t)blockIdx.y * 64;
    for (int i = threadIdx.x / 64; i < 64; i += 4) {
        const uint64_t r = r0 + i, c = c0 + threadIdx.x % 64;
        T v = (T)0.0f;
        if (r < rows && c < cols && (!targets || targets[r] < vocab)) v = from[(int64_t)r * stride + (int64_t)c];
        tile[i][threadIdx.x % 64] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x / 64; i < 64; i += 4) {
        const uint64_t c = c0 + i, r = r0 + threadIdx.x % 64;
        if (c < cols && r < rows) to[c * pitch + r] = tile[threadIdx.x % 64][i];
    }
}

// The tiles' sums of a row, joined in one order: 16 rows a block.
__global__ __launch_bounds__(256) void join_stats_kernel(const float2 *stats, const float *picked,
                                                         const uint32_t *targets, uint64_t tiles, uint64_t rows,
                                                         uint64_t vocab, float *loss, float *lse) {
    __shared__ float2 part[16][17];
    const uint64_t row = (uint64_t)blockIdx.x * 16 + threadIdx.x % 16;
    float2 s = {-__builtin_inff(), 0.0f};
    if (row < rows)
        for (uint64_t t = threadIdx.x / 16; t < tiles; t += 16) s = TileStats::join(s, stats[t * rows + row]);
    part[threadIdx.x / 16][threadIdx.x % 16] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || row >= rows) return;
    for (int i = 1; i < 16; ++i) s = TileStats::join(s, part[i][threadIdx.x]);
    const float l = s.x + logf(s.y);
    if (lse) lse[row] = l;
    loss[row] = targets[row] < vocab ? l - picked[row] : 0.0f;
}

// The largest finite |grad| of a row that has a target; 1 where there is none.
__global__ __launch_bounds__(1024) void most_kernel(const float *grad, const uint32_t *targets, uint64_t rows,
                                                    uint64_t vocab, float *most) {
    float top = 0.0f;
    for (uint64_t r = threadIdx.x; r < rows; r += 1024) {
        const float g = fabsf(grad[r]);
        if (targets[r] < vocab && g < __builtin_inff()) top = fmaxf(top, g);
    }
    __shared__ float tops[16];
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    if (lane_id() == 0) tops[threadIdx.x / kWave] = top;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 16; ++i) top = fmaxf(top, tops[i]);
    *most = top > 0.0f ? top : 1.0f;
}

template <typename T>
hx_status copy_rows(const void *from, int64_t stride, uint64_t rows, uint64_t width, void *to, hipStream_t stream) {
    const uint32_t bytes = (uint32_t)(width * sizeof(T)), pitch = (uint32_t)round_up(bytes, kDepth);
    if (rows == 0 || pitch == 0) return HX_OK;
    const uint64_t blocks = std::min<uint64_t>(ceil_div(rows * (pitch / 16), 256), 1 << 22);
    hipLaunchKernelGGL(copy_rows_kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, (const int8_t *)from,
                       stride * (int64_t)sizeof(T), rows, bytes, (int8_t *)to, pitch);
    return check_launch("copy_rows_kernel");
}
template <typename T>
hx_status transpose(const void *from, int64_t stride, uint64_t rows, uint64_t cols, void *to, uint64_t pitch,
                    const uint32_t *targets, uint64_t vocab, hipStream_t stream) {
    if (rows == 0 || cols == 0) return HX_OK;
    hipLaunchKernelGGL(transpose_kernel<T>, dim3((uint32_t)ceil_div(rows, 64), (uint32_t)ceil_div(cols, 64)), dim3(256),
                       0, stream, (const T *)from, stride, rows, cols, (T *)to, pitch, targets, vocab);
    return check_launch("transpose_kernel");
}

template <typename T> hx_status launch(const CrossEntropyArgs &a, void *ws, hipStream_t stream) {
    const CrossEntropyPlan plan = cross_entropy_plan(a);
    char *base = (char *)ws;
    float2 *stats = (float2 *)(base + plan.stats);
    float *picked = (float *)(base + plan.picked);
    Product p{(const int8_t *)a.x, (const int8_t *)a.weight, a.rows, a.vocab, (uint32_t)(a.width * sizeof(T)),
              a.x_stride * (int64_t)sizeof(T), a.weight_stride * (int64_t)sizeof(T)};
    if (plan.copies) {
        HX_TRY(copy_rows<T>(a.x, a.x_stride, a.rows, a.width, base + plan.x, stream));
        HX_TRY(copy_rows<T>(a.weight, a.weight_stride, a.vocab, a.width, base + plan.weight, stream));
        p.a = (const int8_t *)base + plan.x;
        p.b = (const int8_t *)base + plan.weight;
        p.a_stride = p.b_stride = (int64_t)round_up(p.k, kDepth);
    }
    HX_TRY(launch_product<T>(p, TileStats{stats, picked, a.targets}, stream));
    hipLaunchKernelGGL(join_stats_kernel, dim3((uint32_t)ceil_div(a.rows, 16)), dim3(256), 0, stream, stats, picked,
                       a.targets, a.vocab ? plan.tiles_n : 0, a.rows, a.vocab, a.loss, a.lse);
    return check_launch("join_stats_kernel");
}

template <typename T> hx_status launch(const CrossEntropyGradArgs &a, void *ws, hipStream_t stream) {
    const CrossEntropyGradPlan plan = cross_entropy_grad_plan(a);
    char *base = (char *)ws;
    float *most = (float *)base;
    hipLaunchKernelGGL(most_kernel, dim3(1), dim3(1024), 0, stream, a.grad, a.targets, a.rows, a.vocab, most);
    HX_TRY(check_launch("most_kernel"));
    const int64_t size = sizeof(T);
    const uint64_t row_bytes = round_up(a.width * size, kDepth);
    Product logits{(const int8_t *)a.x, nullptr, a.rows, 0, (uint32_t)(a.width * size), a.x_stride * size,
                   a.weight_stride * size};
    if (plan.copies) {
        HX_TRY(copy_rows<T>(a.x, a.x_stride, a.rows, a.width, base + plan.x, stream));
        logits.a = (const int8_t *)base + plan.x;
        logits.a_stride = logits.b_stride = (int64_t)row_bytes;
    }
    if (a.grad_weight)
        HX_TRY(transpose<T>(a.x, a.x_stride, a.rows, a.width, base + plan.x_columns, plan.rows_pitch, a.targets, a.vocab,
                            stream));
    float *sums = (float *)(base + plan.sums);
    T *g = (T *)(base + plan.g), *gt = (T *)(base + plan.g_columns);
    for (uint64_t first = 0; first < a.vocab || first == 0; first += plan.piece) {
        const uint64_t n = std::min<uint64_t>(plan.piece, a.vocab - first);
        const T *w = (const T *)a.weight + (int64_t)first * a.weight_stride;
        if (plan.copies) {
            HX_TRY(copy_rows<T>(w, a.weight_stride, n, a.width, base + plan.weight, stream));
            logits.b = (const int8_t *)base + plan.weight;
        } else {
            logits.b = (const int8_t *)w;
        }
        logits.n = n;
        HX_TRY(launch_product<T>(logits, TileGradient<T>{g, gt, plan.piece_pitch, plan.rows_pitch, first, a.vocab,
                                                         a.targets, a.lse, a.grad, most},
                                 stream));
        if (a.grad_x) {
            HX_TRY(transpose<T>(w, a.weight_stride, n, a.width, base + plan.weight_columns, plan.piece_pitch, nullptr, 0,
                                stream));
            const bool is_last = first + n >= a.vocab;
            const Product p{(const int8_t *)g, (const int8_t *)base + plan.weight_columns, a.rows, a.width,
                            (uint32_t)(n * size), (int64_t)plan.piece_pitch * size, (int64_t)plan.piece_pitch * size};
            HX_TRY(launch_product<T>(p, TileOut<T>{most, first ? sums : nullptr, is_last ? nullptr : sums, (T *)a.grad_x,
                                                   a.width, a.grad_x_stride},
                                     stream));
        }
        if (a.grad_weight) {
            const Product p{(const int8_t *)gt, (const int8_t *)base + plan.x_columns, n, a.width,
                            (uint32_t)(a.rows * size), (int64_t)plan.rows_pitch * size, (int64_t)plan.rows_pitch * size};
            HX_TRY(launch_product<T>(p, TileOut<T>{most, nullptr, nullptr,
                                                   (T *)a.grad_weight + (int64_t)first * a.grad_weight_stride, 0,
                                                   a.grad_weight_stride},
                                     stream));
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
