// Linear attention with a decay for each head (hx_linear_attention), for
// gfx950:
//   S_t = e^g·S_{t-1} + k_tᵀ·v_t,   o_t = scale·q_t·S_t.
//
// The recurrence: a block holds 32 columns of one head's state in registers,
// eight lanes of four columns by 32 groups of rows, and steps through the
// tokens.  Each step is a rank-1 update of the lane's own elements and a sum
// over the rows: within the wave by lane exchange, across the four waves
// through LDS (two buffers in turn, so one barrier a token).
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

constexpr int kColumns = 32; // of a state, a block
constexpr int kRowGroups = 32;

// Four columns of a row from column c on.  VEC: the rows are 16-byte aligned
// and the width a multiple of four.
template <bool VEC> __device__ __forceinline__ f32x4 load4(const float *row, uint32_t c, uint32_t width) {
    if constexpr (VEC) return c < width ? *(const f32x4 *)(row + c) : f32x4{0, 0, 0, 0};
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c + i < width) v[i] = row[c + i];
    return v;
}
template <bool VEC> __device__ __forceinline__ void store4(float *row, uint32_t c, uint32_t width, f32x4 v) {
    if constexpr (VEC) {
        if (c < width) *(f32x4 *)(row + c) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c + i < width) row[c + i] = v[i];
}

// Rows of the state a lane: dk at most 32·ROWS.
template <typename T, int ROWS, bool VEC>
__global__ __launch_bounds__(256) void attention_step_kernel(AttentionArgs a) {
    __shared__ f32x4 part[2][4][8];
    const uint32_t h = blockIdx.y, b = blockIdx.z, hk = (uint32_t)(h / (a.heads / a.kv_heads));
    const uint32_t dk = (uint32_t)a.dk, dv = (uint32_t)a.dv;
    const uint32_t c = blockIdx.x * kColumns + threadIdx.x % 8 * 4, group = threadIdx.x / 8;
    const int wave = threadIdx.x / kWave;
    const uint64_t length = a.lengths ? min((uint64_t)a.lengths[b], a.tokens) : a.tokens;
    const T *q = (const T *)a.q + b * a.sq.batch + h * a.sq.head;
    const T *k = (const T *)a.k + b * a.sk.batch + hk * a.sk.head;
    const T *v = (const T *)a.v + b * a.sv.batch + hk * a.sv.head;
    T *out = (T *)a.out + b * a.so.batch + h * a.so.head;
    const float decay = expf(a.log_decay[h]);
    f32x4 s[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const uint32_t row = group + kRowGroups * r;
        s[r] = f32x4{0, 0, 0, 0};
        if (a.state_in && row < dk)
            s[r] = load4<VEC>(a.state_in + b * a.si.batch + h * a.si.head + row * a.si.token, c, dv);
    }
    for (uint64_t t = 0; t < length; ++t) {
        f32x4 vt = {0, 0, 0, 0}, o = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < dv) vt[i] = (float)v[(int64_t)t * a.sv.token + c + i];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const uint32_t row = group + kRowGroups * r;
            if (row >= dk) continue;
            const float kt = (float)k[(int64_t)t * a.sk.token + row], qt = (float)q[(int64_t)t * a.sq.token + row];
            s[r] = decay * s[r] + kt * vt;
            o += qt * s[r];
        }
#pragma unroll
        for (int d = 8; d < kWave; d *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], d);
        f32x4(*buffer)[8] = part[t & 1];
        if (lane_id() < 8) buffer[wave][lane_id()] = o;
        __syncthreads();
        if (threadIdx.x < 8) {
            o = (buffer[0][threadIdx.x] + buffer[1][threadIdx.x]) + (buffer[2][threadIdx.x] + buffer[3][threadIdx.x]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < dv) out[(int64_t)t * a.so.token + c + i] = (T)(o[i] * a.scale);
        }
    }
    for (uint64_t t = length + group; t < a.tokens; t += kRowGroups)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < dv) out[(int64_t)t * a.so.token + c + i] = (T)0.0f;
    if (!a.state_out) return;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const uint32_t row = group + kRowGroups * r;
        if (row < dk) store4<VEC>(a.state_out + b * a.st.batch + h * a.st.head + row * a.st.token, c, dv, s[r]);
    }
}

bool vector_rows(const float *base, const AttentionView &s, uint64_t dv) {
    return base == nullptr || ((uintptr_t)base % 16 == 0 && dv % 4 == 0 && s.batch % 4 == 0 && s.head % 4 == 0 &&
                               s.token % 4 == 0);
}

template <typename T, int ROWS> hx_status launch_step(const AttentionArgs &a, hipStream_t stream) {
    const dim3 grid((uint32_t)ceil_div(a.dv, kColumns), (uint32_t)a.heads, (uint32_t)a.batch);
    if (vector_rows(a.state_in, a.si, a.dv) && vector_rows(a.state_out, a.st, a.dv))
        hipLaunchKernelGGL((attention_step_kernel<T, ROWS, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_step_kernel<T, ROWS, false>), grid, dim3(256), 0, stream, a);
    return check_launch("attention_step_kernel");
}

template <typename T> hx_status launch(const AttentionArgs &a, hipStream_t stream) {
    if (a.dk <= 32) return launch_step<T, 1>(a, stream);
    if (a.dk <= 64) return launch_step<T, 2>(a, stream);
    if (a.dk <= 128) return launch_step<T, 4>(a, stream);
    return launch_step<T, 8>(a, stream);
}

} // namespace

uint64_t linear_attention_workspace_bytes(const AttentionArgs &) { return 0; }

hx_status launch_linear_attention(const AttentionArgs &args, void *, hipStream_t stream) {
    if (args.batch == 0 || args.heads == 0 || args.dv == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, stream) : launch<bf16>(args, stream);
}

} // namespace hx
