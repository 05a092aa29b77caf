// RMS norm of rows with the residual's addition and an 8-bit output
// (hx_rms_norm_quantize), for gfx950.
//
// With h = x + r and y = h·rstd·w, the largest |y| is rstd·max|h·w| and
// q = y / (max|y| / 127) = h·w·(127 / max|h·w|): the reciprocal root cancels.
// One sweep over h therefore gives both Σh² and max|h·w|, one combine across
// the row's waves gives both results, and the row is written from the
// registers that it was read into.  Rows too long for the registers are read
// twice; rows too small for f32 to hold their squares, thrice more (is_tiny).
//
// Memory bounds long inputs: 16384 x 8192 bf16 with a residual, 940 MB, takes
// 156 us, 6.0 TB/s.  One row of 4096 takes 2.7 us, a launch and one wait for
// memory.  Rows of odd width begin anywhere and end in part of a vector: 1000 x 5001
// f32 takes 8.8 us, 2.8 TB/s, and 6932 x 9681 bf16 115 us, 4.1 TB/s, where vectors
// cross the 128-byte lines.
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

// Scaling of one row from Σh² and max|h·w|, or from 1 and max|y|.  The maximum is
// taken of the bits as integers: they order as the magnitudes do, with infinities
// and then NaN above them, so that neither is lost.
constexpr uint32_t kInfinity = 0x7F800000u;
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }
struct RowScale {
    float scale;   // s
    float up, inv; // q = round(h·w·up·inv)
};
__device__ __forceinline__ RowScale scale_of(float rstd, uint32_t bits, bool finite) {
    RowScale r;
    const float top = __builtin_bit_cast(float, bits);
    r.scale = finite ? (top > 0.0f ? rstd * top / 127.0f : 0.0f) : __builtin_nanf("");
    // 127 / top overflows for the tiniest rows; two factors do not.
    r.up = top < 0x1p-60f ? 0x1p60f : 1.0f;
    r.inv = finite && top > 0.0f ? 127.0f / (top * r.up) : 0.0f;
    return r;
}
__device__ __forceinline__ RowScale row_scale(float sum, uint32_t bits, float cols, float epsilon) {
    return scale_of(1.0f / sqrtf(sum / cols + epsilon), bits, magnitude(sum) < kInfinity && bits < kInfinity);
}
__device__ __forceinline__ int quantize(float hw, const RowScale &r) {
    return r.inv > 0.0f ? (int)fminf(fmaxf(rintf(hw * r.up * r.inv), -127.0f), 127.0f) : 0;
}

// Σ and max over a row's lanes: LANES of one wave, or WAVES waves of a block.
template <int LANES> __device__ __forceinline__ void combine_lanes(float &sum, uint32_t &top) {
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) {
        sum += __shfl_xor(sum, d);
        top = max(top, (uint32_t)__shfl_xor((int)top, d));
    }
}
template <int WAVES> __device__ __forceinline__ void combine_waves(float &sum, uint32_t &top) {
    combine_lanes<kWave>(sum, top);
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

// A row in memory, swept by LANES threads: h is written by the sweep that reads it
// last, so residual_out may lie on x or the residual.
template <typename T, int LANES> struct SweptRow {
    static constexpr int N = Pack16<T>::N;
    const NormArgs &a;
    const uint64_t row;
    const uint32_t lane;

    // f(c, h, w) for each vector of the row that is this thread's.
    template <typename F> __device__ __forceinline__ void sweep(F f) const {
        const uint32_t cols = (uint32_t)a.cols;
        const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
        const T *res = (const T *)a.residual + (int64_t)row * a.residual_stride;
        const T *w = (const T *)a.weight;
#pragma unroll 1
        for (uint32_t c = lane * N; c < cols; c += LANES * N) {
            const u32x4 vx = load_part(x, c, cols), vw = load_part(w, c, cols);
            u32x4 vr = {0, 0, 0, 0};
            if (a.residual) vr = load_part(res, c, cols);
            float h[N], r[N], wv[N];
            unpack<T>(place_part<T>(vx, c, cols), h);
            if (a.residual) {
                unpack<T>(place_part<T>(vr, c, cols), r);
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] += r[i];
            }
            unpack<T>(place_part<T>(vw, c, cols), wv);
            f(c, h, wv);
        }
    }
    // Σ(h·up)² and the largest |of(h, w)|.
    template <typename F> __device__ __forceinline__ void total(float up, F of, float &sum, uint32_t &top) const {
        sum = 0.0f;
        top = 0;
        sweep([&](uint32_t, const float(&h)[N], const float(&w)[N]) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sum += h[i] * up * (h[i] * up);
                top = max(top, magnitude(of(h[i], w[i])));
            }
        });
        if constexpr (LANES <= kWave) combine_lanes<LANES>(sum, top);
        else combine_waves<LANES / kWave>(sum, top);
    }
    template <typename F> __device__ __forceinline__ void write(const RowScale &r, F of) const {
        const uint32_t cols = (uint32_t)a.cols;
        if (lane == 0) a.scales[row] = r.scale;
        T *ho = (T *)a.residual_out + (int64_t)row * a.residual_out_stride;
        int8_t *q = a.quantized + (int64_t)row * a.quantized_stride;
        sweep([&](uint32_t c, const float(&h)[N], const float(&w)[N]) {
            float y[N];
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = of(h[i], w[i]);
            if (a.residual_out) store_row(ho, c, cols, h);
            store_bytes(q, c, cols, y, r);
        });
    }
};

// Rows that are read again because f32 cannot hold what the one sweep takes:
// * The squares lose bits or vanish, and epsilon does not outweigh them: the mean
//   has an error of 2^-150 at most, which counts below 2^-120.  They are taken from
//   h·2^100: whole from the least float on, and their mean is below 2^80.
// * h·w loses bits where y does not: the largest is below 2^-100.
// Both take y itself, h·rstd first.
constexpr float kTinyMean = 0x1p-120f, kTinyTop = 0x1p-100f;
__device__ __forceinline__ bool is_tiny(float sum, uint32_t bits, float cols, float epsilon) {
    return bits < kInfinity &&
           (sum / cols + epsilon < kTinyMean || (bits > 0 && bits < __builtin_bit_cast(uint32_t, kTinyTop)));
}
template <typename T, int LANES> __device__ __forceinline__ void write_tiny_row(const SweptRow<T, LANES> &row, float sum) {
    const float cols = (float)row.a.cols, epsilon = row.a.epsilon;
    const float lift = sum / cols + epsilon < kTinyMean ? 0x1p100f : 1.0f;
    uint32_t top;
    float none;
    if constexpr (LANES > kWave) __syncthreads(); // the last sums have been read
    row.total(lift, [](float, float) { return 0.0f; }, sum, top);
    const float mean = sum / cols + epsilon * lift * lift, rstd = mean > 0.0f ? 1.0f / sqrtf(mean) : 0.0f;
    const auto y = [&](float h, float w) { return h * lift * rstd * w; };
    if constexpr (LANES > kWave) __syncthreads();
    row.total(1.0f, y, none, top);
    row.write(scale_of(1.0f, top, magnitude(sum) < kInfinity && top < kInfinity), y);
}

// Rows of up to LANES·STEPS vectors, LANES threads a row.  A block has one row,
// or, where a row has less than four waves, as many as fill four.
template <typename T, int LANES, int STEPS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_rows_kernel(NormArgs a) {
    constexpr int N = Pack16<T>::N, kRows = LANES <= kWave ? 256 / LANES : 1;
    static_assert(LANES <= kWave || LANES >= 256);
    const uint64_t row = kRows > 1 ? (uint64_t)blockIdx.x * kRows + threadIdx.x / LANES : blockIdx.x;
    const uint32_t lane = kRows > 1 ? threadIdx.x % LANES : threadIdx.x;
    if (kRows > 1 && row >= a.rows) return; // a row's lanes leave together
    const uint32_t cols = (uint32_t)a.cols;
    const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
    const T *res = (const T *)a.residual + (int64_t)row * a.residual_stride;
    const T *w = (const T *)a.weight;
    u32x4 vx[STEPS], vr[STEPS], vw[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        vx[s] = load_part(x, c, cols);
        vr[s] = u32x4{0, 0, 0, 0};
        if (a.residual) vr[s] = load_part(res, c, cols);
        vw[s] = load_part(w, c, cols);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        if (c + N <= cols) continue;
        vx[s] = place_part<T>(vx[s], c, cols);
        if (a.residual) vr[s] = place_part<T>(vr[s], c, cols);
        vw[s] = place_part<T>(vw[s], c, cols);
    }
    // h and h·w of a vector, from the registers it was loaded into.
    const auto values = [&](int s, float(&h)[N], float(&hw)[N]) {
        float r[N];
        unpack<T>(vx[s], h);
        unpack<T>(vr[s], r);
        unpack<T>(vw[s], hw);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (a.residual) h[i] += r[i];
            hw[i] *= h[i];
        }
    };
    float sum = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        float h[N], hw[N];
        values(s, h, hw);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum += h[i] * h[i];
            top = max(top, magnitude(hw[i]));
        }
    }
    if constexpr (LANES <= kWave) combine_lanes<LANES>(sum, top);
    else combine_waves<LANES / kWave>(sum, top);
    if (is_tiny(sum, top, (float)a.cols, a.epsilon)) { // the same for all lanes of a row
        write_tiny_row(SweptRow<T, LANES>{a, row, lane}, sum);
        return;
    }
    const RowScale r = row_scale(sum, top, (float)a.cols, a.epsilon);
    if (lane == 0) a.scales[row] = r.scale;
    T *ho = (T *)a.residual_out + (int64_t)row * a.residual_out_stride;
    int8_t *q = a.quantized + (int64_t)row * a.quantized_stride;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        if (c >= cols) continue;
        float h[N], hw[N];
        values(s, h, hw);
        if (a.residual_out) store_row(ho, c, cols, h);
        store_bytes(q, c, cols, hw, r);
    }
}

// Rows of any length, read twice by one block.
template <typename T> __global__ __launch_bounds__(1024) void norm_long_rows_kernel(NormArgs a) {
    const SweptRow<T, 1024> row{a, blockIdx.x, threadIdx.x};
    const auto product = [](float h, float w) { return h * w; };
    float sum;
    uint32_t top;
    row.total(1.0f, product, sum, top);
    if (is_tiny(sum, top, (float)a.cols, a.epsilon)) write_tiny_row(row, sum);
    else row.write(row_scale(sum, top, (float)a.cols, a.epsilon), product);
}

// The rows from `first` on.
template <typename T> NormArgs rows_from(NormArgs a, uint64_t first) {
    const int64_t n = (int64_t)first;
    a.rows -= first;
    a.x = (const T *)a.x + n * a.x_stride;
    if (a.residual) a.residual = (const T *)a.residual + n * a.residual_stride;
    if (a.residual_out) a.residual_out = (T *)a.residual_out + n * a.residual_out_stride;
    a.quantized += n * a.quantized_stride;
    a.scales += n;
    return a;
}

template <typename T> hx_status launch(const NormArgs &a, hipStream_t stream) {
    const uint64_t vectors = ceil_div(a.cols, Pack16<T>::N);
    // A launch has fewer than 2^32 threads: more rows take several.
    constexpr uint64_t kBlocks = 1 << 21;
    const auto run = [&](auto kernel, uint64_t lanes) {
        const uint64_t rows = lanes <= kWave ? 256 / lanes : 1;
        for (uint64_t first = 0; first < a.rows; first += kBlocks * rows) {
            NormArgs part = rows_from<T>(a, first);
            part.rows = min(part.rows, kBlocks * rows);
            hipLaunchKernelGGL(kernel, dim3((uint32_t)ceil_div(part.rows, rows)),
                               dim3((uint32_t)(lanes < 256 ? 256 : lanes)), 0, stream, part);
        }
    };
    // One or two vectors a thread as long as rows allow: a thread that holds
    // more keeps fewer waves on a CU.  Measured (us): 16384 x 128 16 lanes 5.5, 64
    // lanes 10.8; 16384 x 1024 64 lanes 23.5, 256 30.0; 16384 x 4096 512 lanes
    // 77.8, 64 88.8, 1024 100.6; 1 x 4096 512 lanes 2.7, 64 6.1.
    if (vectors <= 16) run(norm_rows_kernel<T, 16, 1>, 16);
    else if (vectors <= 64) run(norm_rows_kernel<T, 64, 1>, 64);
    else if (vectors <= 128) run(norm_rows_kernel<T, 64, 2>, 64);
    else if (vectors <= 256) run(norm_rows_kernel<T, 256, 1>, 256);
    else if (vectors <= 512) run(norm_rows_kernel<T, 512, 1>, 512);
    else if (vectors <= 1024) run(norm_rows_kernel<T, 512, 2>, 512);
    else if (vectors <= 2048) run(norm_rows_kernel<T, 512, 4>, 512);
    else if (vectors <= 4096) run(norm_rows_kernel<T, 1024, 4>, 1024);
    else run(norm_long_rows_kernel<T>, 1024);
    return check_launch("norm_rows_kernel");
}

} // namespace

hx_status launch_norm_quantize(const NormArgs &args, hipStream_t stream) {
    if (args.rows == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, stream) : launch<bf16>(args, stream);
}

} // namespace hx
