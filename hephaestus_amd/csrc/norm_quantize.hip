// RMS norm of rows with the residual's addition and an 8-bit output
// (hx_rms_norm_quantize), for gfx950.
//
// With h = x + r and y = h·rstd·w, the largest |y| is rstd·max|h·w| and
// q = y / (max|y| / 127) = h·w·(127 / max|h·w|): the reciprocal root cancels.
// One sweep over h therefore gives both Σh² and max|h·w|, one combine across
// the row's waves gives both results, and the row is written from the
// registers that it was read into.  Rows too long for the registers are read
// twice.
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

// Scaling of one row from Σh² and max|h·w|.  The maximum is taken of the bits
// of |h·w| as integers: they order as the values do, with infinities and then
// NaN above them, so that neither is lost.
constexpr uint32_t kInfinity = 0x7F800000u;
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }
struct RowScale {
    float scale;   // s
    float up, inv; // q = round(h·w·up·inv)
};
__device__ __forceinline__ RowScale row_scale(float sum, uint32_t bits, float cols, float epsilon) {
    RowScale r;
    const float rstd = 1.0f / sqrtf(sum / cols + epsilon), top = __builtin_bit_cast(float, bits);
    const bool finite = magnitude(sum) < kInfinity && bits < kInfinity;
    r.scale = finite ? (top > 0.0f ? rstd * top / 127.0f : 0.0f) : __builtin_nanf("");
    // 127 / top overflows for the tiniest rows; two factors do not.
    r.up = top < 0x1p-60f ? 0x1p60f : 1.0f;
    r.inv = finite && top > 0.0f ? 127.0f / (top * r.up) : 0.0f;
    return r;
}
__device__ __forceinline__ int quantize(float hw, const RowScale &r) {
    return r.inv > 0.0f ? (int)fminf(fmaxf(rintf(hw * r.up * r.inv), -127.0f), 127.0f) : 0;
}

// Σ and max over the WAVES waves of a row; every wave of the block calls it.
template <int WAVES> __device__ __forceinline__ void combine(float &sum, uint32_t &top) {
    sum = wave_sum(sum);
    top = wave_max(top);
    if constexpr (WAVES > 1) {
        __shared__ float sums[WAVES];
        __shared__ uint32_t tops[WAVES];
        const int wave = threadIdx.x / kWave;
        if (lane_id() == 0) {
            sums[wave] = sum;
            tops[wave] = top;
        }
        __syncthreads();
        sum = 0.0f;
        top = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            sum += sums[i];
            top = max(top, tops[i]);
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void load_row(const T *p, uint32_t c, uint32_t cols, float (&x)[N]) {
    if (c + N <= cols) {
        load_pack(p + c, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = c + i < cols ? (float)p[c + i] : 0.0f;
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T *p, uint32_t c, uint32_t cols, const float (&x)[N]) {
    if (c + N <= cols) {
        store_pack(p + c, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < cols) p[c + i] = (T)x[i];
    }
}

template <int N>
__device__ __forceinline__ void store_bytes(int8_t *p, uint32_t c, uint32_t cols, const float (&hw)[N],
                                            const RowScale &r) {
    uint32_t word[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        word[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) word[i] |= ((uint32_t)quantize(hw[4 * i + j], r) & 0xFFu) << (8 * j);
    }
    if (c + N <= cols) {
        __builtin_memcpy(p + c, word, N);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < cols) p[c + i] = (int8_t)(word[i / 4] >> (8 * (i % 4)));
    }
}

// WAVES waves a row, STEPS vectors a lane; rows of up to WAVES·64·STEPS·N.
template <typename T, int WAVES, int STEPS>
__global__ __launch_bounds__(WAVES *kWave) void norm_rows_kernel(NormArgs a) {
    constexpr int N = Pack16<T>::N;
    const uint64_t row = blockIdx.x;
    const uint32_t cols = (uint32_t)a.cols;
    const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
    const T *res = (const T *)a.residual + (int64_t)row * a.residual_stride;
    const T *w = (const T *)a.weight;
    float h[STEPS][N], hw[STEPS][N];
    float sum = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * WAVES * kWave + threadIdx.x) * N;
        load_row(x, c, cols, h[s]);
        if (a.residual) {
            float r[N];
            load_row(res, c, cols, r);
#pragma unroll
            for (int i = 0; i < N; ++i) h[s][i] += r[i];
        }
        load_row(w, c, cols, hw[s]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum += h[s][i] * h[s][i];
            hw[s][i] *= h[s][i];
            top = max(top, magnitude(hw[s][i]));
        }
    }
    combine<WAVES>(sum, top);
    const RowScale r = row_scale(sum, top, (float)a.cols, a.epsilon);
    if (threadIdx.x == 0) a.scales[row] = r.scale;
    T *ho = (T *)a.residual_out + (int64_t)row * a.residual_out_stride;
    int8_t *q = a.quantized + (int64_t)row * a.quantized_stride;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * WAVES * kWave + threadIdx.x) * N;
        if (c >= cols) continue;
        if (a.residual_out) store_row(ho, c, cols, h[s]);
        store_bytes(q, c, cols, hw[s], r);
    }
}

// Rows of any length, read twice by one block; h is written by the sweep
// that reads it last, so residual_out may lie on x or the residual.
template <typename T> __global__ __launch_bounds__(1024) void norm_long_rows_kernel(NormArgs a) {
    constexpr int N = Pack16<T>::N;
    const uint64_t row = blockIdx.x;
    const uint32_t cols = (uint32_t)a.cols;
    const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
    const T *res = (const T *)a.residual + (int64_t)row * a.residual_stride;
    const T *w = (const T *)a.weight;
    T *ho = (T *)a.residual_out + (int64_t)row * a.residual_out_stride;
    int8_t *q = a.quantized + (int64_t)row * a.quantized_stride;
    const auto sweep = [&](uint32_t c, float (&h)[N], float (&hw)[N]) {
        load_row(x, c, cols, h);
        if (a.residual) {
            float r[N];
            load_row(res, c, cols, r);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] += r[i];
        }
        load_row(w, c, cols, hw);
#pragma unroll
        for (int i = 0; i < N; ++i) hw[i] *= h[i];
    };
    float sum = 0.0f;
    uint32_t top = 0;
    for (uint32_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
        float h[N], hw[N];
        sweep(c, h, hw);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum += h[i] * h[i];
            top = max(top, magnitude(hw[i]));
        }
    }
    combine<16>(sum, top);
    const RowScale r = row_scale(sum, top, (float)a.cols, a.epsilon);
    if (threadIdx.x == 0) a.scales[row] = r.scale;
    for (uint32_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
        float h[N], hw[N];
        sweep(c, h, hw);
        if (a.residual_out) store_row(ho, c, cols, h);
        store_bytes(q, c, cols, hw, r);
    }
}

template <typename T> hx_status launch(const NormArgs &a, hipStream_t stream) {
    constexpr uint64_t N = Pack16<T>::N;
    const uint64_t vectors = ceil_div(a.cols, N);
    const dim3 grid((uint32_t)a.rows);
    if (vectors <= 4 * kWave) hipLaunchKernelGGL((norm_rows_kernel<T, 1, 4>), grid, dim3(kWave), 0, stream, a);
    else if (vectors <= 16 * kWave)
        hipLaunchKernelGGL((norm_rows_kernel<T, 4, 4>), grid, dim3(4 * kWave), 0, stream, a);
    else if (vectors <= 64 * kWave)
        hipLaunchKernelGGL((norm_rows_kernel<T, 16, 4>), grid, dim3(16 * kWave), 0, stream, a);
    else hipLaunchKernelGGL((norm_long_rows_kernel<T>), grid, dim3(1024), 0, stream, a);
    return check_launch("norm_rows_kernel");
}

} // namespace

hx_status launch_norm_quantize(const NormArgs &args, hipStream_t stream) {
    if (args.rows == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, stream) : launch<bf16>(args, stream);
}

} // namespace hx
