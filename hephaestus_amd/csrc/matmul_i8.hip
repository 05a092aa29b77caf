// Product of 8-bit integers with a scale for each token and channel
// (hx_matmul_i8), for gfx950.
//
// Tiles of a and b are staged through LDS in rows of 64 bytes of k and
// multiplied by the 16 x 16 x 64 integer matrix instruction: lane l of a wave
// holds 16 consecutive bytes of k, at 16·(l / 16), of row l % 16 of either
// operand, and the sums of row 4·(l / 16) + i, column l % 16 of the product.
// Rows and bytes outside the operands are staged as zeros, so they add
// nothing.  The sums are exact; the scales are applied to them in f32.
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// 16 bytes of a row from `k` on; zeros past `end`.
__device__ __forceinline__ u32x4 load_bytes(const int8_t *row, uint64_t k, uint64_t end) {
    if (k + 16 <= end) return *(const u32x4_any *)(row + k);
    u32x4 v = {0, 0, 0, 0};
    for (uint32_t i = 0; k + i < end; ++i) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
    return v;
}

template <typename T> __device__ __forceinline__ void store_scaled(T *p, int32_t sum, float sa, float sb) {
    *p = (T)((float)sum * sa * sb);
}

constexpr int kTile = 64;     // rows of a and of b a block
constexpr int kDepth = 64;    // bytes of k a step
constexpr int kPitch = kDepth + 16;

// Four waves, each 32 x 32 of the block's 64 x 64.
template <typename T> __global__ __launch_bounds__(256) void matmul_tile_kernel(MatmulArgs p) {
    __shared__ __align__(16) int8_t as[kTile * kPitch], bs[kTile * kPitch];
    const uint64_t m0 = (uint64_t)blockIdx.y * kTile, n0 = (uint64_t)blockIdx.x * kTile;
    const int lane = lane_id(), wave = threadIdx.x / kWave;
    const int r = threadIdx.x / 4, c = threadIdx.x % 4 * 16;
    const bool a_in = m0 + r < p.m, b_in = n0 + r < p.n;
    const int8_t *ga = p.a + (int64_t)(a_in ? m0 + r : 0) * p.a_stride;
    const int8_t *gb = p.b + (int64_t)(b_in ? n0 + r : 0) * p.b_stride;
    const int wm = wave / 2 * 32, wn = wave % 2 * 32;
    i32x4v acc[2][2] = {};
    for (uint64_t k = 0; k < p.k; k += kDepth) {
        const u32x4 va = load_bytes(ga, k + c, a_in ? p.k : 0), vb = load_bytes(gb, k + c, b_in ? p.k : 0);
        __syncthreads();
        *(u32x4 *)(as + r * kPitch + c) = va;
        *(u32x4 *)(bs + r * kPitch + c) = vb;
        __syncthreads();
        i32x4v fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = *(const i32x4v *)(as + (wm + 16 * i + lane % 16) * kPitch + lane / 16 * 16);
            fb[i] = *(const i32x4v *)(bs + (wn + 16 * i + lane % 16) * kPitch + lane / 16 * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint64_t n = n0 + wn + 16 * j + lane % 16;
        if (n >= p.n) continue;
        const float sb = p.b_scales[n];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t m = m0 + wm + 16 * i + lane / 16 * 4 + e;
                if (m < p.m) store_scaled((T *)p.out + (int64_t)m * p.out_stride + n, acc[i][j][e], p.a_scales[m], sb);
            }
    }
}

template <typename T> hx_status launch(const MatmulArgs &p, hipStream_t stream) {
    const uint64_t gm = ceil_div(p.m, kTile), gn = ceil_div(p.n, kTile);
    if (gm > 65535) return fail(HX_ERR_DISPATCH_FAILED, "matmul of %llu rows exceeds the grid range", (unsigned long long)p.m);
    hipLaunchKernelGGL((matmul_tile_kernel<T>), dim3((uint32_t)gn, (uint32_t)gm), dim3(256), 0, stream, p);
    return check_launch("matmul_tile_kernel");
}

} // namespace

uint64_t matmul_i8_workspace_bytes(const MatmulArgs &) { return 0; }

hx_status launch_matmul_i8(const MatmulArgs &args, void *, hipStream_t stream) {
    if (args.m == 0 || args.n == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, stream) : launch<bf16>(args, stream);
}

} // namespace hx
