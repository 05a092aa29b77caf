// Product of 8-bit integers with a scale for each token and channel
// (hx_matmul_i8), for gfx950.
//
// Both forms use the 16 x 16 x 64 integer matrix instruction: lane l of a wave
// holds 16 consecutive bytes of k, from 16·(l / 16) on, of row l % 16 of either
// operand.  The rows of b are its first operand, so lane l ends up with the
// sums of channels 4·(l / 16) + i, i = 0..3, of token l % 16, and a token's four
// channels are stored together.  Sums of integers do not depend on their
// order: every split of k below is exact and gives the same bits.
//
// * Few tokens (skinny): b is read once and straight into registers; the
//   waves of a block take slices of k and add their sums in LDS.
// * Tiles: rows of 128 bytes of a and b go through two LDS buffers in turn.
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kDepth = 128; // bytes of k a step
constexpr int kWaitLoads = 0x0F70; // s_waitcnt vmcnt(0)

__device__ __forceinline__ i32x4v mma(i32x4v b, i32x4v a, i32x4v sum) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, sum, 0, 0, 0);
}

// 16 bytes of a row from `k` on, zeros from `end` on.  Global memory takes
// vectors at any byte address.
__device__ __forceinline__ i32x4v load_bytes(const int8_t *row, uint32_t k, uint32_t end) {
    if (k + 16 <= end) return __builtin_bit_cast(i32x4v, (u32x4)*(const u32x4_any *)(row + k));
    i32x4v v = {0, 0, 0, 0};
    for (uint32_t i = 0; k + i < end; ++i) v[i / 4] |= (int)((uint32_t)(uint8_t)row[k + i] << (8 * (i % 4)));
    return v;
}

typedef bf16 bf16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// Four channels of one token: out[n..n+3] = sum·sa·sb.
template <typename T>
__device__ __forceinline__ void store_scaled(T *row, uint64_t n, uint64_t end, i32x4v sum, float sa, const float *sb) {
    if (n + 4 <= end) {
        const f32x4 s = *(const f32x4_a4 *)(sb + n);
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)sum[i] * sa * s[i];
        if constexpr (sizeof(T) == 4) {
            *(f32x4_a4 *)(row + n) = v;
        } else {
            bf16x4_a2 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (bf16)v[i];
            *(bf16x4_a2 *)(row + n) = r;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < end) row[n + i] = (T)((float)sum[i] * sa * sb[n + i]);
    }
}

// ------------------------------------------------------------------ skinny
// Up to 16·MF tokens; a block takes 16·NF channels, each of its eight waves
// every eighth 128 bytes of k.
constexpr int kSkinnyWaves = 8;

template <typename T, int MF, int NF>
__global__ __launch_bounds__(kSkinnyWaves *kWave) void matmul_skinny_kernel(MatmulArgs p) {
    __shared__ int sums[MF * NF * 4 * kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint64_t n0 = (uint64_t)blockIdx.x * (16 * NF);
    const uint32_t k_end = (uint32_t)p.k, at = lane / 16 * 16;
    for (int i = threadIdx.x; i < MF * NF * 4 * kWave; i += kSkinnyWaves * kWave) sums[i] = 0;
    const int8_t *a[MF], *b[NF];
    uint32_t a_end[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
        const uint64_t m = 16 * i + lane % 16;
        a_end[i] = m < p.m ? k_end : 0; // rows that are not there are zeros
        a[i] = p.a + (int64_t)(m < p.m ? m : 0) * p.a_stride;
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) // channels past the end are summed and dropped
        b[j] = p.b + (int64_t)min(n0 + 16 * j + lane % 16, p.n - 1) * p.b_stride;
    i32x4v acc[MF][NF] = {};
    const uint32_t whole = k_end / kDepth * kDepth;
    for (uint32_t k = wave * kDepth; k < whole; k += kSkinnyWaves * kDepth) {
        i32x4v fb[NF][2], fa[MF][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int j = 0; j < NF; ++j)
                fb[j][s] = __builtin_bit_cast(i32x4v, __builtin_nontemporal_load((const u32x4_any *)(b[j] + k + 64 * s + at)));
#pragma unroll
            for (int i = 0; i < MF; ++i)
                fa[i][s] = a_end[i] ? __builtin_bit_cast(i32x4v, (u32x4)*(const u32x4_any *)(a[i] + k + 64 * s + at))
                                    : i32x4v{0, 0, 0, 0};
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int i = 0; i < MF; ++i) acc[i][j] = mma(fb[j][s], fa[i][s], acc[i][j]);
    }
    // The last, partial 128 bytes: to the wave whose turn it is.
    if (whole < k_end && wave == (int)(whole / kDepth % kSkinnyWaves)) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const i32x4v fb = load_bytes(b[j], whole + 64 * s + at, k_end);
#pragma unroll
                for (int i = 0; i < MF; ++i)
                    acc[i][j] = mma(fb, load_bytes(a[i], whole + 64 * s + at, a_end[i]), acc[i][j]);
            }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) atomicAdd(&sums[((i * NF + j) * 4 + e) * kWave + lane], acc[i][j][e]);
    __syncthreads();
    for (int f = wave; f < MF * NF; f += kSkinnyWaves) {
        const uint64_t m = 16 * (f / NF) + lane % 16, n = n0 + 16 * (f % NF) + lane / 16 * 4;
        if (m >= p.m) continue;
        i32x4v s;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = sums[(f * 4 + e) * kWave + lane];
        store_scaled((T *)p.out + (int64_t)m * p.out_stride, n, p.n, s, p.a_scales[m], p.b_scales);
    }
}

template <typename T, int MF> hx_status launch_skinny(const MatmulArgs &p, hipStream_t stream) {
    const auto run = [&](auto nf) {
        constexpr int NF = decltype(nf)::value;
        hipLaunchKernelGGL((matmul_skinny_kernel<T, MF, NF>), dim3((uint32_t)ceil_div(p.n, 16 * NF)),
                           dim3(kSkinnyWaves * kWave), 0, stream, p);
    };
    if (p.n >= 16 * 2 * 256) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 1>{});
    return check_launch("matmul_skinny_kernel");
}

// ------------------------------------------------------------------- tiles
// BM tokens by BN channels a block of WM x WN waves.  A step's 128 bytes of k
// of each row lie in LDS as eight chunks of 16, chunk c of row r at place
// c ^ (r % 8), so that the 16 rows that a matrix instruction reads at one c
// fall on all banks.  DIRECT loads go from memory to LDS without registers:
// each wave's 64 chunks of an instruction land side by side, and the exchange
// of places is made on the global side.  They need rows whose addresses and
// lengths are multiples of 16; other rows pass through registers.
template <typename T, int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(WM *WN *kWave) void matmul_tiles_kernel(MatmulArgs p, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int kThreads = WM * WN * kWave, kRows = BM + BN, kStage = kRows * kDepth;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int kLoads = kRows * 8 / kThreads; // chunks of 16 bytes a thread and step
    extern __shared__ __align__(16) int8_t lds[]; // two stages
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

    // Blocks go to the eight XCDs in turn: each XCD takes a run of tiles, in
    // strips of eight tiles of m so that its L2 serves both operands.
    const uint32_t total = tiles_m * tiles_n, share = total / 8, rest = total % 8;
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t tile = xcd * share + min(xcd, rest) + turn;
    const uint32_t strip = tile / (8 * tiles_n), in_strip = tile % (8 * tiles_n);
    const uint32_t height = min(8u, tiles_m - 8 * strip);
    const uint64_t m0 = (uint64_t)(8 * strip + in_strip % height) * BM, n0 = (uint64_t)(in_strip / height) * BN;

    const uint32_t k_end = (uint32_t)p.k;
    // A thread's chunk of each row it loads: rows past the operands repeat the
    // last one and are dropped at the end.
    const uint32_t place = threadIdx.x % 8, row0 = DIRECT ? wave * (kLoads * 8) + lane / 8 : threadIdx.x / 8;
    constexpr uint32_t kRowStep = DIRECT ? 8 : kThreads / 8;
    const uint32_t chunk = (place ^ (row0 % 8)) * 16;
    const int8_t *src[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const uint32_t r = row0 + j * kRowStep;
        src[j] = (r < BM ? p.a + (int64_t)min(m0 + r, p.m - 1) * p.a_stride
                         : p.b + (int64_t)min(n0 + (r - BM), p.n - 1) * p.b_stride) + chunk;
    }
    u32x4 held[DIRECT ? 1 : kLoads];

    const auto fetch = [&](uint32_t k, int8_t *stage) {
        if constexpr (DIRECT) {
            if (k + kDepth <= k_end) {
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    __builtin_amdgcn_global_load_lds((const void *)(src[j] + k),
                                                     (lds_void *)(stage + (wave * kLoads + j) * 1024), 16, 0, 0);
            } else { // chunks past the end are zeros
#pragma unroll
                for (int j = 0; j < kLoads; ++j) {
                    if (k + chunk < k_end)
                        __builtin_amdgcn_global_load_lds((const void *)(src[j] + k),
                                                         (lds_void *)(stage + (wave * kLoads + j) * 1024), 16, 0, 0);
                    else *(u32x4 *)(stage + (wave * kLoads + j) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
                held[j] = __builtin_bit_cast(u32x4, load_bytes(src[j] - chunk, k + chunk, k_end));
        }
    };
    const auto settle = [&](int8_t *stage) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
                *(u32x4 *)(stage + (row0 + j * kRowStep) * kDepth + place * 16) = held[j];
        }
    };

    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    const uint32_t swizzled = (lane / 16 ^ (lane % 8)) * 16; // of k bytes 0..63; 64..127: ^ 64
    const uint32_t at_a = (wm + lane % 16) * kDepth + swizzled, at_b = (BM + wn + lane % 16) * kDepth + swizzled;
    i32x4v acc[FM][FN] = {};
    const auto compute = [&](const int8_t *stage) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x4v fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = *(const i32x4v *)(stage + (at_b ^ (64 * s)) + j * (16 * kDepth));
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = *(const i32x4v *)(stage + (at_a ^ (64 * s)) + i * (16 * kDepth));
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
        }
    };

    // The barrier itself does not wait for direct loads.
    const auto sync = [&] {
        if constexpr (DIRECT) __builtin_amdgcn_s_waitcnt(kWaitLoads);
        __syncthreads();
    };
    if (k_end) {
        fetch(0, lds);
        settle(lds);
        sync();
        uint32_t stage = 0;
        for (uint32_t k = 0; k < k_end; k += kDepth, stage ^= 1) {
            int8_t *next = lds + (stage ^ 1) * kStage;
            const bool more = k + kDepth < k_end;
            if (more) fetch(k + kDepth, next);
            compute(lds + stage * kStage);
            if (more) settle(next);
            sync();
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const uint64_t m = m0 + wm + 16 * i + lane % 16;
        if (m >= p.m) continue;
        const float sa = p.a_scales[m];
        T *row = (T *)p.out + (int64_t)m * p.out_stride;
#pragma unroll
        for (int j = 0; j < FN; ++j)
            store_scaled(row, n0 + wn + 16 * j + lane / 16 * 4, p.n, acc[i][j], sa, p.b_scales);
    }
}

template <typename T, int BM, int BN, int WM, int WN, bool DIRECT>
hx_status launch_tiles(const MatmulArgs &p, hipStream_t stream) {
    constexpr uint32_t kLds = 2 * (BM + BN) * kDepth;
    const auto kernel = matmul_tiles_kernel<T, BM, BN, WM, WN, DIRECT>;
    if constexpr (kLds > 65536) {
        static const hipError_t allowed =
            hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
        if (allowed != hipSuccess) return hip_fail(HX_ERR_DISPATCH_FAILED, allowed, "matmul LDS size");
    }
    const uint64_t tm = ceil_div(p.m, BM), tn = ceil_div(p.n, BN);
    if (tm * tn > 0x7FFFFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "matmul of %llu tiles exceeds the grid range", (unsigned long long)(tm * tn));
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tm * tn)), dim3(WM * WN * kWave), kLds, stream, p, (uint32_t)tm,
                       (uint32_t)tn);
    return check_launch("matmul_tiles_kernel");
}

template <typename T> hx_status launch(const MatmulArgs &p, hipStream_t stream) {
    if (p.m <= 16) return launch_skinny<T, 1>(p, stream);
    if (p.m <= 32) return launch_skinny<T, 2>(p, stream);
    if (p.m <= 64) return launch_skinny<T, 4>(p, stream);
    const bool direct = (((uintptr_t)p.a | (uintptr_t)p.b | (uint64_t)p.a_stride | (uint64_t)p.b_stride | p.k) % 16) == 0;
    if (!direct) return launch_tiles<T, 64, 64, 2, 2, false>(p, stream);
    if (ceil_div(p.m, 256) * ceil_div(p.n, 256) >= 200) return launch_tiles<T, 256, 256, 2, 4, true>(p, stream);
    if (ceil_div(p.m, 128) * ceil_div(p.n, 128) >= 200) return launch_tiles<T, 128, 128, 2, 2, true>(p, stream);
    return launch_tiles<T, 64, 64, 2, 2, true>(p, stream);
}

} // namespace

uint64_t matmul_i8_workspace_bytes(const MatmulArgs &) { return 0; }

hx_status launch_matmul_i8(const MatmulArgs &args, void *, hipStream_t stream) {
    if (args.m == 0 || args.n == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, stream) : launch<bf16>(args, stream);
}

} // namespace hx
