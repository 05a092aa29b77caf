// Layer norm of rows with the residual's addition (hx_layer_norm) and its
// backward pass (hx_layer_norm_backward), for gfx950.
//
// Forward: a row lies in the registers of the threads that share it, so that the
// mean and then the squares of what differs from it are taken from one reading.
// The mean that a sum in f32 gives is off by a few roundings; what the differences
// from it sum up to corrects the variance, and the mean where it is far from 0:
//   m' = m + Σd / n,   var = (Σd² - (Σd)² / n) / n,   d = h - m.
//
// Backward, with u = (h - mean)·rstd and t = dy·w of a row:
//   dh = rstd·(t - Σt / n - u·Σ(t·u) / n) + what reaches h past the norm,
//   dw = Σ dy·u,  db = Σ dy   over the rows.
// A block goes through rows and keeps its share of dw and db in registers; the
// blocks' shares are added up by a second launch, in one order.
//
// Memory bounds both: 16384 x 8192 bf16 with a residual takes 192 us forward (5.6 TB/s
// of x, residual, h and out) and 210 us backward (5.1 TB/s and the sums' launch of 6 us),
// where torch's copy of 1 GiB reaches 5.2 TB/s.  A single row of 4096 takes 3.7 us, 3.5 of
// them the kernel's, a launch and one wait for memory; 1000 x 5001 f32 takes 24 us
// backward, 250 blocks of 4 rows whose loads lie off the 128-byte grid, and 6 us of the sums.
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

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

// Sums of up to three values over the threads of a row: LANES of a wave, or a block.
template <int LANES> struct RowSums {
    static constexpr int kWaves = LANES / kWave;
    float (*lds)[3][kWaves]; // two of them, in turn: one is read while the next is written
    uint32_t turn = 0;
    __device__ __forceinline__ RowSums() {
        __shared__ float sums[2][3][kWaves];
        lds = sums;
    }
    template <int N> __device__ __forceinline__ void operator()(float (&v)[N]) {
        static_assert(N <= 3);
#pragma unroll
        for (int d = 1; d < kWave; d *= 2)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], d);
        float(&s)[3][kWaves] = lds[turn];
        turn ^= 1;
        if (lane_id() == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) s[k][threadIdx.x / kWave] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) v[k] += s[k][i];
        }
    }
};
template <int LANES> struct LaneSums {
    template <int N> __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
        for (int d = 1; d < LANES; d *= 2)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], d);
    }
};
template <int LANES> struct SumsOf { using type = RowSums<LANES>; };
template <> struct SumsOf<16> { using type = LaneSums<16>; };
template <> struct SumsOf<64> { using type = LaneSums<64>; };

// ----------------------------------------------------------------- forward

// Mean and (variance + epsilon)^(-1/2) of a row of h·scale.
struct RowStats {
    float scale, mean, rstd;
};
// each(f) calls f(c, h) for the vectors of the row that are this thread's, with
// zeros past its end.
template <typename Each, typename Sums>
__device__ __forceinline__ float scaled_stats(const Each &each, Sums &sums, uint32_t cols, float epsilon,
                                              RowStats &r) {
    float sum[1] = {0.0f};
    each([&](uint32_t, const auto &h) {
        for (float v : h) sum[0] += v * r.scale;
    });
    sums(sum);
    const float mean = sum[0] / cols;
    float far[3] = {0.0f, 0.0f, 0.0f}; // Σd, Σd², Σ|d|
    each([&](uint32_t c, const auto &h) {
        uint32_t at = c;
        for (float v : h) {
            const float d = at++ < cols ? v * r.scale - mean : 0.0f;
            far[0] += d;
            far[1] += d * d;
            far[2] += fabsf(d);
        }
    });
    sums(far);
    const float shift = far[0] / cols;
    // The differences' own roundings, up to 2^-24 of each and often the same in all,
    // leave about that much of Σ|d| / n in the shift, beside a mean near 0 far more than
    // what the first sum was off: of 4096 bf16 elements 7e-7 of the mean against 9e-8
    // (95 of 100 rows).  A shift past 4 times that, or one that is a NaN, goes to the mean.
    r.mean = fabsf(shift) <= 0x1p-22f * (far[2] / cols) ? mean : mean + shift;
    const float var = (far[1] - far[0] * shift) / cols;
    const float m = (var < 0.0f ? 0.0f : var) + epsilon * r.scale * r.scale; // a NaN stays
    r.rstd = m > 0.0f ? 1.0f / sqrtf(m) : m == 0.0f ? 0.0f : __builtin_nanf("");
    return m;
}
// Rows beyond f32 are taken again: sums or squares that overflow from h·2^-100,
// squares that lose bits or vanish, where epsilon does not outweigh them, from
// h·2^100 (an error of 2^-150 in the mean square counts below 2^-120; where the mean
// is large beside such a variance all elements are equal).
template <typename Each, typename Sums>
__device__ __forceinline__ RowStats stats_of(const Each &each, Sums &sums, uint32_t cols, float epsilon) {
    RowStats r{1.0f, 0.0f, 0.0f};
    const float m = scaled_stats(each, sums, cols, epsilon, r);
    if (!(m < __builtin_inff())) r.scale = 0x1p-100f;
    else if (m < 0x1p-120f && fabsf(r.mean) < 0x1p-20f) r.scale = 0x1p100f;
    if (r.scale != 1.0f) scaled_stats(each, sums, cols, epsilon, r); // the same for all threads of a row
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void write_vector(const LayerNormArgs &a, uint64_t row, uint32_t c, const RowStats &r,
                                             const float (&h)[N], const float (&w)[N], const float (&b)[N]) {
    const uint32_t cols = (uint32_t)a.cols;
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = (h[i] * r.scale - r.mean) * r.rstd * w[i] + b[i];
    if (a.residual_out) store_row((T *)a.residual_out + (int64_t)row * a.residual_out_stride, c, cols, h);
    store_row((T *)a.out + (int64_t)row * a.out_stride, c, cols, y);
}
__device__ __forceinline__ void write_stats(const LayerNormArgs &a, uint64_t row, const RowStats &r) {
    if (a.mean) a.mean[row] = r.mean / r.scale;
    if (a.rstd) a.rstd[row] = r.rstd * r.scale;
}

// Rows of up to LANES·STEPS vectors, LANES threads a row.  A block has one row,
// or, where a row has less than four waves, as many as fill four.
template <typename T, int LANES, int STEPS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void layer_norm_kernel(LayerNormArgs a) {
    constexpr int N = Pack16<T>::N, kRows = LANES <= kWave ? 256 / LANES : 1;
    const uint64_t row = kRows > 1 ? (uint64_t)blockIdx.x * kRows + threadIdx.x / LANES : blockIdx.x;
    const uint32_t lane = kRows > 1 ? threadIdx.x % LANES : threadIdx.x;
    if (kRows > 1 && row >= a.rows) return; // a row's lanes leave together
    const uint32_t cols = (uint32_t)a.cols;
    const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
    const T *res = (const T *)a.residual + (int64_t)row * a.residual_stride;
    const T *w = (const T *)a.weight, *b = (const T *)a.bias;
    u32x4 vx[STEPS], vr[STEPS], vw[STEPS], vb[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        vx[s] = load_part(x, c, cols);
        vr[s] = vb[s] = u32x4{0, 0, 0, 0};
        if (a.residual) vr[s] = load_part(res, c, cols);
        vw[s] = load_part(w, c, cols);
        if (a.bias) vb[s] = load_part(b, c, cols);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        if (c + N <= cols) continue;
        vx[s] = place_part<T>(vx[s], c, cols);
        if (a.residual) vr[s] = place_part<T>(vr[s], c, cols);
        vw[s] = place_part<T>(vw[s], c, cols);
        if (a.bias) vb[s] = place_part<T>(vb[s], c, cols);
    }
    const auto value = [&](int s, float(&h)[N]) {
        unpack<T>(vx[s], h);
        if (!a.residual) return;
        float r[N];
        unpack<T>(vr[s], r);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] += r[i];
    };
    const auto each = [&](const auto &f) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t c = ((uint32_t)s * LANES + lane) * N;
            if (c >= cols) continue;
            float h[N];
            value(s, h);
            f(c, h);
        }
    };
    typename SumsOf<LANES>::type sums;
    const RowStats r = stats_of(each, sums, cols, a.epsilon);
    if (lane == 0) write_stats(a, row, r);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        if (c >= cols) continue;
        float h[N], wv[N], bv[N];
        value(s, h);
        unpack<T>(vw[s], wv);
        unpack<T>(vb[s], bv);
        write_vector<T>(a, row, c, r, h, wv, bv);
    }
}

// Rows of any length, read three times by one block: 1024 threads hold no more than 4 vectors
// of x and of the residual each.  1500 x 40000 bf16 with a residual takes 144 us (3.3 TB/s of
// what has to be moved), 2048 x 32768, in registers, 123 (4.4).
template <typename T> __global__ __launch_bounds__(1024) void layer_norm_long_kernel(LayerNormArgs a) {
    constexpr int N = Pack16<T>::N;
    const uint64_t row = blockIdx.x;
    const uint32_t cols = (uint32_t)a.cols;
    const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
    const T *res = (const T *)a.residual + (int64_t)row * a.residual_stride;
    const auto each = [&](const auto &f) {
#pragma unroll 1
        for (uint32_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
            const u32x4 vx = load_part(x, c, cols);
            u32x4 vr = {0, 0, 0, 0};
            if (a.residual) vr = load_part(res, c, cols);
            float h[N], r[N];
            unpack<T>(place_part<T>(vx, c, cols), h);
            if (a.residual) {
                unpack<T>(place_part<T>(vr, c, cols), r);
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] += r[i];
            }
            f(c, h);
        }
    };
    RowSums<1024> sums;
    const RowStats r = stats_of(each, sums, cols, a.epsilon);
    if (threadIdx.x == 0) write_stats(a, row, r);
    each([&](uint32_t c, const float(&h)[N]) { // h is written by the sweep that reads it last
        float wv[N], bv[N];
        unpack<T>(place_part<T>(load_part((const T *)a.weight, c, cols), c, cols), wv);
        u32x4 vb = {0, 0, 0, 0};
        if (a.bias) vb = place_part<T>(load_part((const T *)a.bias, c, cols), c, cols);
        unpack<T>(vb, bv);
        write_vector<T>(a, row, c, r, h, wv, bv);
    });
}

// The rows from `first` on.
template <typename T> LayerNormArgs rows_from(LayerNormArgs a, uint64_t first) {
    const int64_t n = (int64_t)first;
    a.rows -= first;
    a.x = (const T *)a.x + n * a.x_stride;
    if (a.residual) a.residual = (const T *)a.residual + n * a.residual_stride;
    if (a.residual_out) a.residual_out = (T *)a.residual_out + n * a.residual_out_stride;
    a.out = (T *)a.out + n * a.out_stride;
    if (a.mean) a.mean += n;
    if (a.rstd) a.rstd += n;
    return a;
}

template <typename T> hx_status launch(const LayerNormArgs &a, hipStream_t stream) {
    // A launch has fewer than 2^32 threads: more rows take several.
    constexpr uint64_t kBlocks = 1 << 21;
    const auto run = [&](auto kernel, uint64_t lanes) {
        const uint64_t rows = lanes <= kWave ? 256 / lanes : 1;
        for (uint64_t first = 0; first < a.rows; first += kBlocks * rows) {
            LayerNormArgs part = rows_from<T>(a, first);
            part.rows = std::min<uint64_t>(part.rows, kBlocks * rows);
            hipLaunchKernelGGL(kernel, dim3((uint32_t)ceil_div(part.rows, rows)),
                               dim3((uint32_t)(lanes < 256 ? 256 : lanes)), 0, stream, part);
        }
    };
    switch (layer_norm_row(a.cols, sizeof(T))) {
    case NormRow::k16: run(layer_norm_kernel<T, 16, 1>, 16); break;
    case NormRow::k64: run(layer_norm_kernel<T, 64, 1>, 64); break;
    case NormRow::k128: run(layer_norm_kernel<T, 64, 2>, 64); break;
    case NormRow::k256: run(layer_norm_kernel<T, 256, 1>, 256); break;
    case NormRow::k512: run(layer_norm_kernel<T, 512, 1>, 512); break;
    case NormRow::k1024: run(layer_norm_kernel<T, 512, 2>, 512); break;
    case NormRow::k2048: run(layer_norm_kernel<T, 512, 4>, 512); break;
    case NormRow::k4096: run(layer_norm_kernel<T, 1024, 4>, 1024); break;
    case NormRow::kLong: run(layer_norm_long_kernel<T>, 1024); break;
    }
    return check_launch("layer_norm_kernel");
}

// ---------------------------------------------------------------- backward

// Partial sums of dw and db, [blocks][2][cols], to the gradients: 64 columns a
// block, its waves take the blocks in turn.
constexpr int kFoldWaves = 16;
__global__ __launch_bounds__(kFoldWaves *kWave) void layer_norm_fold_kernel(const float *partial, uint32_t blocks,
                                                                           uint32_t cols, float *grad_weight,
                                                                           float *grad_bias) {
    __shared__ float sums[kFoldWaves][kWave];
    const uint32_t c = blockIdx.x * kWave + lane_id(), which = blockIdx.y;
    const int wave = threadIdx.x / kWave;
    float *out = which ? grad_bias : grad_weight;
    if (!out) return;
    float sum = 0.0f;
    if (c < cols)
        for (uint32_t b = wave; b < blocks; b += kFoldWaves) sum += partial[((uint64_t)b * 2 + which) * cols + c];
    sums[wave][lane_id()] = sum;
    __syncthreads();
    if (wave != 0 || c >= cols) return;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kFoldWaves; ++i) sum += sums[i][lane_id()];
    out[c] = sum;
}

template <int N> __device__ __forceinline__ void store_sums(float *p, uint32_t c, uint32_t cols, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        if (c + i + 4 <= cols) {
            *(f32x4_a4 *)(p + c + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + i + e < cols) p[c + i + e] = x[i + e];
        }
    }
}

// Block b goes through the rows of its run, `LANES` threads a row as forward.
template <typename T, int LANES, int STEPS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void layer_norm_grad_kernel(LayerNormGradArgs a,
                                                                                   uint32_t rows_a_block,
                                                                                   float *partial) {
    constexpr int N = Pack16<T>::N, kRows = LANES <= kWave ? 256 / LANES : 1;
    const uint32_t cols = (uint32_t)a.cols, lane = kRows > 1 ? threadIdx.x % LANES : threadIdx.x;
    const uint32_t group = kRows > 1 ? threadIdx.x / LANES : 0;
    const uint64_t first = (uint64_t)blockIdx.x * rows_a_block, end = min(a.rows, first + rows_a_block);
    // Rows of 4 vectors a thread leave no registers for the weight, which lies in LDS, nor to
    // fetch the gradient past the norm ahead: it is asked for while its own row is summed.
    // 2282 x 14976 bf16 takes 81 us so, 159 where registers spilled.
    constexpr bool kAhead = STEPS < 4;
    __shared__ u32x4 weights[kAhead ? 1 : STEPS][LANES];
    u32x4 vw[STEPS];
    float dw[STEPS][N] = {}, db[STEPS][N] = {};
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t c = ((uint32_t)s * LANES + lane) * N;
        vw[s] = place_part<T>(load_part((const T *)a.weight, c, cols), c, cols);
        if constexpr (!kAhead) weights[s][lane] = vw[s]; // read by this lane alone
    }
    const auto weight = [&](int s) { return kAhead ? vw[s] : weights[s][lane]; };
    typename SumsOf<LANES>::type sums;
    struct Row {
        u32x4 x[STEPS], dy[STEPS], past[kAhead ? STEPS : 1];
        float mean, rstd;
    } now, next;
    const auto fetch_past = [&](uint64_t row, u32x4 *past) {
        const T *p = (const T *)a.residual_grad + (int64_t)row * a.residual_grad_stride;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            past[s] = u32x4{0, 0, 0, 0};
            if (a.residual_grad) past[s] = load_part(p, ((uint32_t)s * LANES + lane) * N, cols);
        }
    };
    const auto fetch = [&](uint64_t row, Row &r) {
        const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
        const T *dy = (const T *)a.grad_out + (int64_t)row * a.grad_out_stride;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t c = ((uint32_t)s * LANES + lane) * N;
            r.x[s] = load_part(x, c, cols);
            r.dy[s] = load_part(dy, c, cols);
        }
        if constexpr (kAhead) fetch_past(row, r.past);
        r.mean = a.mean[row];
        r.rstd = a.rstd[row];
    };
    // The next row is on its way while this one is summed.
    if (first + group < end) fetch(first + group, now);
    for (uint64_t row = first + group; row < end; row += kRows, now = next) {
        if (row + kRows < end) fetch(row + kRows, next);
        u32x4(&vx)[STEPS] = now.x, (&vy)[STEPS] = now.dy, late[STEPS], *vp = kAhead ? now.past : late;
        const float mean = now.mean, rstd = now.rstd;
        float st[2] = {0.0f, 0.0f}; // Σt, Σ(t·u)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t c = ((uint32_t)s * LANES + lane) * N;
            vx[s] = place_part<T>(vx[s], c, cols);
            vy[s] = place_part<T>(vy[s], c, cols); // zeros past the row: they add nothing
            float h[N], g[N], w[N];
            unpack<T>(vx[s], h);
            unpack<T>(vy[s], g);
            unpack<T>(weight(s), w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float u = (h[i] - mean) * rstd, t = g[i] * w[i];
                st[0] += t;
                st[1] += t * u;
                dw[s][i] += g[i] * u;
                db[s][i] += g[i];
            }
        }
        if constexpr (!kAhead) fetch_past(row, late);
        sums(st);
        const float mt = st[0] / cols, mtu = st[1] / cols;
        T *out = (T *)a.grad_in + (int64_t)row * a.grad_in_stride;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t c = ((uint32_t)s * LANES + lane) * N;
            if (c >= cols) continue;
            float h[N], g[N], w[N], p[N];
            unpack<T>(vx[s], h);
            unpack<T>(vy[s], g);
            unpack<T>(weight(s), w);
            unpack<T>(place_part<T>(vp[s], c, cols), p);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float u = (h[i] - mean) * rstd;
                g[i] = rstd * (g[i] * w[i] - mt - u * mtu);
                if (a.residual_grad) g[i] += p[i];
            }
            store_row(out, c, cols, g);
        }
    }
    if (!a.grad_weight && !a.grad_bias) return;
    float *mine = partial + (uint64_t)blockIdx.x * 2 * cols;
    if constexpr (kRows > 1) { // the rows' groups join in LDS, one after another
        __shared__ float joined[2][LANES * STEPS * N];
        for (uint32_t turn = 0; turn < kRows; ++turn) {
            if (group == turn)
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const uint32_t at = (s * LANES + lane) * N + i;
                        joined[0][at] = turn ? joined[0][at] + dw[s][i] : dw[s][i];
                        joined[1][at] = turn ? joined[1][at] + db[s][i] : db[s][i];
                    }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < cols; c += 256) {
            mine[c] = joined[0][c];
            mine[cols + c] = joined[1][c];
        }
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t c = ((uint32_t)s * LANES + lane) * N;
            store_sums(mine, c, cols, dw[s]);
            store_sums(mine + cols, c, cols, db[s]);
        }
    }
}

// Rows of any length: dh with two readings of a row by one block, and the sums
// over a run of rows by columns.
template <typename T> __global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(LayerNormGradArgs a) {
    constexpr int N = Pack16<T>::N;
    const uint64_t row = blockIdx.x;
    const uint32_t cols = (uint32_t)a.cols;
    const T *x = (const T *)a.x + (int64_t)row * a.x_stride;
    const T *dy = (const T *)a.grad_out + (int64_t)row * a.grad_out_stride;
    const T *past = (const T *)a.residual_grad + (int64_t)row * a.residual_grad_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    const auto each = [&](const auto &f) { // f(c, t, u)
#pragma unroll 1
        for (uint32_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
            const u32x4 vx = load_part(x, c, cols), vy = load_part(dy, c, cols),
                        vw = load_part((const T *)a.weight, c, cols);
            float u[N], t[N], w[N];
            unpack<T>(place_part<T>(vx, c, cols), u);
            unpack<T>(place_part<T>(vy, c, cols), t);
            unpack<T>(place_part<T>(vw, c, cols), w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                u[i] = (u[i] - mean) * rstd;
                t[i] *= w[i];
            }
            f(c, t, u);
        }
    };
    float st[2] = {0.0f, 0.0f}; // Σt, Σ(t·u)
    each([&](uint32_t, const float(&t)[N], const float(&u)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            st[0] += t[i];
            st[1] += t[i] * u[i];
        }
    });
    RowSums<1024> sums;
    sums(st);
    const float mt = st[0] / cols, mtu = st[1] / cols;
    T *out = (T *)a.grad_in + (int64_t)row * a.grad_in_stride;
    each([&](uint32_t c, const float(&t)[N], const float(&u)[N]) {
        float g[N], p[N];
        u32x4 vp = {0, 0, 0, 0};
        if (a.residual_grad) vp = place_part<T>(load_part(past, c, cols), c, cols);
        unpack<T>(vp, p);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            g[i] = rstd * (t[i] - mt - u[i] * mtu);
            if (a.residual_grad) g[i] += p[i];
        }
        store_row(out, c, cols, g);
    });
}
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_grad_columns_kernel(LayerNormGradArgs a, uint32_t rows_a_block,
                                                                      float *partial) {
    constexpr int N = Pack16<T>::N;
    const uint32_t cols = (uint32_t)a.cols, c = (blockIdx.y * 256 + threadIdx.x) * N;
    if (c >= cols) return;
    const uint64_t first = (uint64_t)blockIdx.x * rows_a_block, end = min(a.rows, first + rows_a_block);
    float dw[N] = {}, db[N] = {};
    for (uint64_t row = first; row < end; ++row) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        float h[N], g[N];
        unpack<T>(place_part<T>(load_part((const T *)a.x + (int64_t)row * a.x_stride, c, cols), c, cols), h);
        unpack<T>(place_part<T>(load_part((const T *)a.grad_out + (int64_t)row * a.grad_out_stride, c, cols), c, cols), g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            dw[i] += g[i] * ((h[i] - mean) * rstd);
            db[i] += g[i];
        }
    }
    float *mine = partial + (uint64_t)blockIdx.x * 2 * cols;
    store_sums(mine, c, cols, dw);
    store_sums(mine + cols, c, cols, db);
}

template <typename T> hx_status launch(const LayerNormGradArgs &a, void *ws, hipStream_t stream) {
    const NormGradSplit split = layer_norm_grad_split(a);
    float *partial = (float *)ws;
    const uint32_t cols = (uint32_t)a.cols;
    const bool sums = a.grad_weight || a.grad_bias;
    const auto run = [&](auto kernel, uint32_t lanes) {
        hipLaunchKernelGGL(kernel, dim3(split.blocks), dim3(lanes < 256 ? 256 : lanes), 0, stream, a,
                           split.rows_a_block, partial);
    };
    if (a.rows > 0 && cols > 0) {
        switch (layer_norm_row(a.cols, sizeof(T))) {
        case NormRow::k16: run(layer_norm_grad_kernel<T, 16, 1>, 16); break;
        case NormRow::k64: run(layer_norm_grad_kernel<T, 64, 1>, 64); break;
        case NormRow::k128: run(layer_norm_grad_kernel<T, 64, 2>, 64); break;
        case NormRow::k256: run(layer_norm_grad_kernel<T, 256, 1>, 256); break;
        case NormRow::k512: run(layer_norm_grad_kernel<T, 512, 1>, 512); break;
        case NormRow::k1024: run(layer_norm_grad_kernel<T, 512, 2>, 512); break;
        case NormRow::k2048: run(layer_norm_grad_kernel<T, 512, 4>, 512); break;
        case NormRow::k4096:
        case NormRow::kLong: {
            // Columns first: grad_in may lie on grad_out.
            if (sums) {
                const uint32_t tiles = (uint32_t)ceil_div(cols, 256 * Pack16<T>::N);
                hipLaunchKernelGGL(layer_norm_grad_columns_kernel<T>, dim3(split.blocks, tiles), dim3(256), 0, stream,
                                   a, split.rows_a_block, partial);
                HX_TRY(check_launch("layer_norm_grad_columns_kernel"));
            }
            constexpr uint64_t kBlocks = 1 << 21;
            for (uint64_t first = 0; first < a.rows; first += kBlocks) {
                LayerNormGradArgs part = a;
                const int64_t n = (int64_t)first;
                part.rows = std::min<uint64_t>(a.rows - first, kBlocks);
                part.x = (const T *)a.x + n * a.x_stride;
                part.grad_out = (const T *)a.grad_out + n * a.grad_out_stride;
                if (a.residual_grad) part.residual_grad = (const T *)a.residual_grad + n * a.residual_grad_stride;
                part.grad_in = (T *)a.grad_in + n * a.grad_in_stride;
                part.mean += n;
                part.rstd += n;
                hipLaunchKernelGGL(layer_norm_grad_long_kernel<T>, dim3((uint32_t)part.rows), dim3(1024), 0, stream,
                                   part);
            }
            break;
        }
        }
        HX_TRY(check_launch("layer_norm_grad_kernel"));
    }
    if (!sums || cols == 0) return HX_OK;
    // No rows: sums of nothing.
    hipLaunchKernelGGL(layer_norm_fold_kernel, dim3((uint32_t)ceil_div(cols, kWave), 2), dim3(kFoldWaves * kWave), 0,
                       stream, partial, a.rows ? split.blocks : 0, cols, a.grad_weight, a.grad_bias);
    return check_launch("layer_norm_fold_kernel");
}

} // namespace

hx_status launch_layer_norm(const LayerNormArgs &args, hipStream_t stream) {
    if (args.rows == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, stream) : launch<bf16>(args, stream);
}

uint64_t layer_norm_grad_workspace_bytes(const LayerNormGradArgs &args) {
    if (!args.grad_weight && !args.grad_bias) return 0;
    return (uint64_t)layer_norm_grad_split(args).blocks * 2 * args.cols * sizeof(float);
}

hx_status launch_layer_norm_grad(const LayerNormGradArgs &args, void *ws, hipStream_t stream) {
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, ws, stream) : launch<bf16>(args, ws, stream);
}

} // namespace hx
