// Linear attention with a decay for each head (hx_linear_attention), for
// gfx950:
//   S_t = e^g·S_{t-1} + k_tᵀ·v_t,   o_t = scale·q_t·S_t.
//
// Two forms.  The recurrence, for single tokens: a block holds 32 columns of one head's state in registers,
// eight lanes of four columns by 32 groups of rows, and steps through the
// tokens.  Each step is a rank-1 update of the lane's own elements and a sum
// over the rows: within the wave by lane exchange, across the four waves
// through LDS (two buffers in turn, so one barrier a token).
#include "hx_internal.hpp"
#include "layer_device.hpp"

#include <algorithm>
#include <type_traits>

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

// ------------------------------------------------------------------ chunks
// Prompts, C tokens at a time.  With D = e^g and t, s counted within a chunk
// that holds r tokens and begins with the state S:
//   o_t = scale·(D^(t+1)·q_t·S + Σ_{s<=t} D^(t-s)·(q_t·k_s)·v_s)
//   S  <- D^r·S + Σ_s D^(r-1-s)·k_sᵀ·v_s
// All four products are matrix instructions.  A block takes one head and 16
// columns of v a wave; each wave keeps its columns of S, in f32, in the
// accumulators of the last product, for the whole prompt.
//
// The accumulators of a 16 x 16 product hold, in lane l, column l % 16 and rows
// 4·(l / 16) + i.  An operand holds, in lane l, row or column l % 16 and the
// terms 4·(l / 16) + i of a run of 16.  So what one product leaves is an operand
// of the next without an exchange between lanes, if the products are taken
// transposed: Pᵀ = K·Qᵀ, Oᵀ = Sᵀ·Qᵀ + Vᵀ·Pᵀ.  Only P passes through LDS, because
// every wave needs all of it.
//
// Roundings, where the elements are bf16: an element of P, and of S where a
// query meets it, is rounded to bf16 once.  The sums that go into S are not: a
// weighted value D^(r-1-s)·v is taken as three bf16 terms, which hold 24 bits.
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Four terms of an operand; two of them make the 32 terms of an instruction.
template <typename T> struct Fragment;
template <> struct Fragment<bf16> { using type = bf16x4; };
template <> struct Fragment<float> { using type = f32x4v; };

__device__ __forceinline__ f32x4v mma(const bf16x4 (&a)[2], const bf16x4 (&b)[2], f32x4v c) {
    const bf16x8 x = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7);
    const bf16x8 y = __builtin_shufflevector(b[0], b[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4v mma(const f32x4v (&a)[2], const f32x4v (&b)[2], f32x4v c) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[h][i], b[h][i], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ bf16x4 rounded(f32x4v v, bf16) {
    return bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
}
__device__ __forceinline__ f32x4v rounded(f32x4v v, float) { return v; }
__device__ __forceinline__ f32x4v widened(bf16x4 v) { return f32x4v{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }
__device__ __forceinline__ f32x4v widened(f32x4v v) { return v; }

// v as a sum of TERMS elements: all of a float's bits, for bf16 in three terms
// of eight each.
template <typename T> constexpr int kTerms = sizeof(T) == 2 ? 3 : 1;
__device__ __forceinline__ void split(f32x4v v, bf16x4 (&to)[3]) {
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const s16x4 high = {(short)(__float_as_uint(v[0]) >> 16), (short)(__float_as_uint(v[1]) >> 16),
                            (short)(__float_as_uint(v[2]) >> 16), (short)(__float_as_uint(v[3]) >> 16)};
        to[n] = __builtin_bit_cast(bf16x4, high);
        if (n < 2) v -= widened(to[n]);
    }
}
__device__ __forceinline__ void split(f32x4v v, f32x4v (&to)[1]) { to[0] = v; }

// Eight neighbours of a row in LDS as the two halves of a run of 32 terms.
__device__ __forceinline__ void load_terms(const bf16 *p, bf16x4 (&f)[2]) {
    const bf16x8 v = *(const bf16x8 *)p;
    f[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    f[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
}
__device__ __forceinline__ void load_terms(const float *p, f32x4v (&f)[2]) {
    f[0] = *(const f32x4v *)p;
    f[1] = *(const f32x4v *)(p + 4);
}
// Four terms down a column: rows 4·(l / 16) + i of `tile`, and of its columns
// the (l % 4)-th of the four that begin at `step`·(l % 16 / 4).
__device__ __forceinline__ bf16x4 load_column(const bf16 *tile, int pitch, int step) {
    // The transposing read: lane l names row 4·(l / 16) + l % 16 / 4 and four
    // columns of it, and receives one column of its sixteen lanes' rows.
    const int l = lane_id(), row = l / 16 * 4 + l % 16 / 4;
    return __builtin_bit_cast(bf16x4,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + row * pitch + l % 4 * step)));
}
__device__ __forceinline__ f32x4v load_column(const float *tile, int pitch, int step) {
    const int l = lane_id();
    const float *p = tile + l / 16 * 4 * pitch + l % 16 / 4 * step + l % 4;
    return f32x4v{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
}

// One chunk of a head's rows on its way from memory to LDS: N vectors of 16
// bytes a thread.  Rows from `rows` on and columns from `width` on are zeros.
template <typename T, int ROWS, int COLS, int THREADS> struct Staged {
    static constexpr int V = Pack16<T>::N, kRow = COLS / V, N = (ROWS * kRow + THREADS - 1) / THREADS;
    typedef typename std::conditional<sizeof(T) == 2, u32x4_a2, u32x4_a4>::type Vec;
    u32x4 held[N];
    __device__ __forceinline__ void load(const T *base, int64_t stride, uint32_t rows, uint32_t width) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t at = threadIdx.x + i * THREADS, row = at / kRow, col = at % kRow * V;
            const T *p = base + (int64_t)row * stride + col;
            held[i] = u32x4{0, 0, 0, 0};
            if (row < rows && col + V <= width) {
                held[i] = *(const Vec *)p;
            } else if (row < rows) {
                T part[V];
#pragma unroll
                for (int e = 0; e < V; ++e) part[e] = col + e < width ? p[e] : (T)0.0f;
                __builtin_memcpy(&held[i], part, 16);
            }
        }
    }
    __device__ __forceinline__ void store(T *tile, int pitch) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t at = threadIdx.x + i * THREADS;
            if (N * THREADS == ROWS * kRow || at < ROWS * kRow)
                *(u32x4 *)(tile + at / kRow * pitch + at % kRow * V) = held[i];
        }
    }
};

// A prompt cut into `parts` of `span` tokens each, a multiple of the chunk.
struct Parts {
    uint32_t parts, span;
    float *states; // [batch, heads, parts, dk, dv]: each part's own sum, then the state before it
};

template <typename T, int DK, int NW> struct Chunk {
    static constexpr int C = sizeof(T) == 2 ? 64 : 32, B = C / 16, kThreads = NW * kWave, DV = NW * 16;
    static constexpr int kPad = 16 / sizeof(T); // rows 16 bytes off each other's banks
    static constexpr int kPitch = DK + kPad, kPitchV = DV + kPad;
    static constexpr int kTiles = B * (B + 1) / 2; // of P, on and below the diagonal
    static constexpr int kLds = (2 * C * kPitch + C * kPitchV + kTiles * 4 * kWave) * (int)sizeof(T);
};

// OUTPUTS: the outputs of a part, from the state before it.  Otherwise only the
// part's own sum, from nothing.
template <typename T, int DK, int NW, bool OUTPUTS>
__global__ __launch_bounds__(NW *kWave) void attention_chunk_kernel(AttentionArgs a, Parts parts) {
    using G = Chunk<T, DK, NW>;
    using F = typename Fragment<T>::type;
    constexpr int C = G::C, B = G::B, kPitch = G::kPitch, kPitchV = G::kPitchV;
    extern __shared__ __align__(16) char lds[];
    T *ks = (T *)lds, *vs = ks + C * kPitch, *qs = vs + C * kPitchV;
    F *ps = (F *)(qs + C * kPitch);
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 16, quad = lane / 16;
    const uint32_t part = blockIdx.x % parts.parts, block = blockIdx.x / parts.parts;
    const uint32_t h = blockIdx.y, b = blockIdx.z, hk = (uint32_t)(h / (a.heads / a.kv_heads));
    const uint32_t dk = (uint32_t)a.dk, dv0 = block * G::DV, dv = min((uint32_t)a.dv - dv0, (uint32_t)G::DV);
    const uint32_t tokens = (uint32_t)a.tokens, length = a.lengths ? min(a.lengths[b], tokens) : tokens;
    const uint32_t begin = part * parts.span, end = min(begin + parts.span, length);
    const T *q = (const T *)a.q + b * a.sq.batch + h * a.sq.head;
    const T *k = (const T *)a.k + b * a.sk.batch + hk * a.sk.head;
    const T *v = (const T *)a.v + b * a.sv.batch + hk * a.sv.head + dv0;
    T *out = (T *)a.out + b * a.so.batch + h * a.so.head + dv0;
    const uint32_t vcol = wave * 16 + col; // this lane's column of v and of the state

    // The decay as a power of two a token; minus infinity would make 0·log a NaN.
    const float log2_decay = fmaxf(a.log_decay[h] * 1.44269504f, -1e30f);
    const auto power = [&](int n) { return __builtin_amdgcn_exp2f(log2_decay * (float)n); };

    // Row r of accumulator 2·i + j is dk 32·i + 8·(r / 4) + 4·j + r % 4: two
    // accumulators hold the eight neighbours that a query's lane reads at once.
    f32x4v s[DK / 16] = {};
    const auto state_row = [&](int i, int e) { return (uint32_t)(i / 2 * 32 + quad * 8 + i % 2 * 4 + e); };
    float *saved = parts.states + (((uint64_t)b * a.heads + h) * parts.parts + part) * dk * a.dv + dv0 + vcol;
    if (OUTPUTS && vcol < dv) {
        const float *from = parts.parts > 1 ? saved
                            : a.state_in    ? a.state_in + b * a.si.batch + h * a.si.head + dv0 + vcol
                                            : nullptr;
        const int64_t stride = parts.parts > 1 ? (int64_t)a.dv : a.si.token;
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (from && state_row(i, e) < dk) s[i][e] = from[state_row(i, e) * stride];
    }

    Staged<T, C, DK, G::kThreads> next_q, next_k;
    Staged<T, C, G::DV, G::kThreads> next_v;
    const auto fetch = [&](uint32_t t0) {
        const uint32_t rows = end - t0;
        next_k.load(k + (int64_t)t0 * a.sk.token, a.sk.token, rows, dk);
        next_v.load(v + (int64_t)t0 * a.sv.token, a.sv.token, rows, dv);
        if constexpr (OUTPUTS) next_q.load(q + (int64_t)t0 * a.sq.token, a.sq.token, rows, dk);
    };
    if (begin < end) fetch(begin);
    for (uint32_t t0 = begin; t0 < end; t0 += C) {
        const int rows = (int)min((uint32_t)C, end - t0);
        __syncthreads(); // the last chunk has been read
        next_k.store(ks, kPitch);
        next_v.store(vs, kPitchV);
        if constexpr (OUTPUTS) next_q.store(qs, kPitch);
        __syncthreads();
        if (t0 + C < end) fetch(t0 + C);

        F vf[B]; // this lane's column of v
#pragma unroll
        for (int i = 0; i < B; ++i) vf[i] = load_column(vs + i * 16 * kPitchV + wave * 16, kPitchV, 4);

        if constexpr (OUTPUTS) {
            // Pᵀ tiles (x: rows of k, y: rows of q), the waves in turn.
            int tile = 0;
#pragma unroll
            for (int y = 0; y < B; ++y)
#pragma unroll
                for (int x = 0; x <= y; ++x, ++tile) {
                    if (tile % NW != wave) continue;
                    f32x4v p = {};
#pragma unroll
                    for (int i = 0; i < DK / 32; ++i) {
                        F fk[2], fq[2];
                        load_terms(ks + (x * 16 + col) * kPitch + i * 32 + quad * 8, fk);
                        load_terms(qs + (y * 16 + col) * kPitch + i * 32 + quad * 8, fq);
                        p = mma(fk, fq, p);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int far = (y * 16 + col) - (x * 16 + quad * 4 + e);
                        p[e] = far >= 0 ? p[e] * (power(far) * a.scale) : 0.0f;
                    }
                    ps[tile * kWave + lane] = rounded(p, T{});
                }
            __syncthreads();
            f32x4v o[B];
            int first_bad = C; // the first token whose v is no number, in this lane's column
            for (int again = 0;; ++again) {
#pragma unroll
                for (int y = 0; y < B; ++y) o[y] = f32x4v{};
#pragma unroll
                for (int i = 0; i < DK / 32; ++i) {
                    const F fs[2] = {rounded(s[2 * i], T{}), rounded(s[2 * i + 1], T{})};
#pragma unroll
                    for (int y = 0; y < B; ++y) {
                        F fq[2];
                        load_terms(qs + (y * 16 + col) * kPitch + i * 32 + quad * 8, fq);
                        o[y] = mma(fs, fq, o[y]);
                    }
                }
                float sick = 0.0f;
#pragma unroll
                for (int y = 0; y < B; ++y) {
                    o[y] *= power(y * 16 + col + 1) * a.scale;
#pragma unroll
                    for (int x = 0; x <= y; x += 2) {
                        const F fv[2] = {vf[x], vf[x + 1]};
                        F fp[2] = {ps[(y * (y + 1) / 2 + x) * kWave + lane], F{}};
                        if (x < y) fp[1] = ps[(y * (y + 1) / 2 + x + 1) * kWave + lane];
                        o[y] = mma(fv, fp, o[y]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) sick += o[y][e] * 0.0f;
                }
                // A value that is no number also spoils the tokens before it,
                // whose weights are 0: take it out, and put its mark where
                // it belongs.
                if (again || !__any(!(sick == 0.0f))) break;
#pragma unroll
                for (int x = B - 1; x >= 0; --x) {
                    f32x4v w = widened(vf[x]);
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (!(w[e] * 0.0f == 0.0f)) {
                            first_bad = min(first_bad, x * 16 + quad * 4 + e);
                            w[e] = 0.0f;
                        }
                    vf[x] = rounded(w, T{});
                }
                first_bad = min(first_bad, __shfl_xor(first_bad, 16));
                first_bad = min(first_bad, __shfl_xor(first_bad, 32));
            }
            if (__any(first_bad < C)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int from = __shfl(first_bad, quad * 4 + e); // of the row of o, a column of v
#pragma unroll
                    for (int y = 0; y < B; ++y)
                        if (y * 16 + col >= from) o[y][e] = __builtin_nanf("");
                }
#pragma unroll
                for (int i = 0; i < B; ++i) vf[i] = load_column(vs + i * 16 * kPitchV + wave * 16, kPitchV, 4);
            }
            // Four neighbours of a token's row.
            const uint32_t c = wave * 16 + quad * 4;
#pragma unroll
            for (int y = 0; y < B; ++y) {
                if (y * 16 + col >= rows) continue;
                T *to = out + (int64_t)(t0 + y * 16 + col) * a.so.token + c;
                if (c + 4 <= dv) {
                    const F r = rounded(o[y], T{});
                    __builtin_memcpy(to, &r, sizeof(r));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < dv) to[e] = (T)o[y][e];
                }
            }
        }

        // The state: decayed over the chunk, to the last bit of f32 (the power
        // in two floats), then the chunk's sum.
        const double decayed = exp((double)a.log_decay[h] * rows);
        const float high = (float)decayed, low = (float)(decayed - high);
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = fmaf(s[i][e], high, s[i][e] * low);
        F terms[B][kTerms<T>];
#pragma unroll
        for (int x = 0; x < B; ++x) {
            f32x4v w = widened(vf[x]);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] *= power(max(rows - 1 - (x * 16 + quad * 4 + e), 0));
            split(w, terms[x]);
        }
#pragma unroll
        for (int i = 0; i < DK / 16; ++i)
#pragma unroll
            for (int x = 0; x < B; x += 2) {
                F fk[2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    fk[j] = load_column(ks + (x + j) * 16 * kPitch + i / 2 * 32 + i % 2 * 4, kPitch, 8);
#pragma unroll
                for (int n = kTerms<T> - 1; n >= 0; --n) {
                    const F fv[2] = {terms[x][n], terms[x + 1][n]};
                    s[i] = mma(fk, fv, s[i]);
                }
            }
    }

    if constexpr (OUTPUTS) { // rows past the sequence's end
        const uint32_t until = min(begin + parts.span, tokens);
        for (uint32_t t = max(begin, length) + threadIdx.x / 16; t < until; t += G::kThreads / 16)
            for (uint32_t c = threadIdx.x % 16; c < dv; c += 16) out[(int64_t)t * a.so.token + c] = (T)0.0f;
    }
    if (vcol >= dv) return;
    float *to = !OUTPUTS ? saved
                : parts.parts == 1 && a.state_out ? a.state_out + b * a.st.batch + h * a.st.head + dv0 + vcol
                                                  : nullptr;
    const int64_t stride = OUTPUTS ? a.st.token : (int64_t)a.dv;
#pragma unroll
    for (int i = 0; i < DK / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (to && state_row(i, e) < dk) to[state_row(i, e) * stride] = s[i][e];
}

// The state before each part, from the parts' own sums: one element of the
// state a thread, the parts in order.
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a, Parts parts) {
    const uint32_t n = (uint32_t)(a.dk * a.dv), i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t h = blockIdx.y, b = blockIdx.z, row = i / (uint32_t)a.dv, col = i % (uint32_t)a.dv;
    const uint32_t tokens = (uint32_t)a.tokens, length = a.lengths ? min(a.lengths[b], tokens) : tokens;
    const double log_decay = a.log_decay[h];
    float s = a.state_in ? a.state_in[b * a.si.batch + h * a.si.head + row * a.si.token + col] : 0.0f;
    float *at = parts.states + ((uint64_t)b * a.heads + h) * parts.parts * n + i;
    for (uint32_t p = 0; p < parts.parts; ++p, at += n) {
        const int64_t left = (int64_t)length - (int64_t)p * parts.span, count = min(left, (int64_t)parts.span);
        const double decayed = count > 0 ? exp(log_decay * (double)count) : 1.0; // infinite logs among them
        const float high = (float)decayed, low = (float)(decayed - high), own = *at;
        *at = s;
        s = fmaf(s, high, s * low) + own;
    }
    if (a.state_out) a.state_out[b * a.st.batch + h * a.st.head + row * a.st.token + col] = s;
}

// Columns of v a block: up to 128, in whole waves of 16.
uint32_t block_waves(const AttentionArgs &a) { return a.dv <= 64 ? 4 : 8; }

constexpr uint64_t kStepTokens = 8; // up to here the recurrence
constexpr uint64_t kFullCard = 256; // blocks

Parts parts_of(const AttentionArgs &a) {
    const uint64_t chunk = a.dtype == HX_DTYPE_F32 ? 32 : 64, chunks = ceil_div(a.tokens, chunk);
    const uint64_t blocks = a.batch * a.heads * ceil_div(a.dv, 16 * block_waves(a));
    uint64_t parts = blocks < kFullCard / 2 ? kFullCard / blocks : 1;
    parts = std::min(parts, std::max<uint64_t>(chunks / 4, 1));
    const uint64_t span = ceil_div(chunks, parts) * chunk;
    return Parts{(uint32_t)ceil_div(a.tokens, span), (uint32_t)span, nullptr};
}

template <typename T, int DK, int NW> hx_status launch_chunks(const AttentionArgs &a, void *ws, hipStream_t stream) {
    using G = Chunk<T, DK, NW>;
    const auto run = [&](auto kernel, const Parts &parts) {
        if constexpr (G::kLds > 65536) {
            const hipError_t err =
                hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, G::kLds);
            if (err != hipSuccess) return hip_fail(HX_ERR_DISPATCH_FAILED, err, "attention LDS size");
        }
        const uint64_t x = ceil_div(a.dv, G::DV) * parts.parts;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)x, (uint32_t)a.heads, (uint32_t)a.batch), dim3(G::kThreads), G::kLds,
                           stream, a, parts);
        return check_launch("attention_chunk_kernel");
    };
    Parts parts = parts_of(a);
    parts.states = (float *)ws;
    if (parts.parts > 1) {
        HX_TRY(run(attention_chunk_kernel<T, DK, NW, false>, parts));
        hipLaunchKernelGGL(attention_join_kernel,
                           dim3((uint32_t)ceil_div(a.dk * a.dv, 256), (uint32_t)a.heads, (uint32_t)a.batch), dim3(256),
                           0, stream, a, parts);
        HX_TRY(check_launch("attention_join_kernel"));
    }
    return run(attention_chunk_kernel<T, DK, NW, true>, parts);
}

template <typename T, int NW> hx_status launch_width(const AttentionArgs &a, void *ws, hipStream_t stream) {
    if (a.dk <= 64) return launch_chunks<T, 64, NW>(a, ws, stream);
    if (a.dk <= 128) return launch_chunks<T, 128, NW>(a, ws, stream);
    return launch_chunks<T, 256, NW>(a, ws, stream);
}

bool by_chunks(const AttentionArgs &a) { return a.tokens > kStepTokens && a.dk > 0; }

template <typename T> hx_status launch(const AttentionArgs &a, void *ws, hipStream_t stream) {
    if (by_chunks(a))
        return block_waves(a) == 4 ? launch_width<T, 4>(a, ws, stream) : launch_width<T, 8>(a, ws, stream);
    if (a.dk <= 32) return launch_step<T, 1>(a, stream);
    if (a.dk <= 64) return launch_step<T, 2>(a, stream);
    if (a.dk <= 128) return launch_step<T, 4>(a, stream);
    return launch_step<T, 8>(a, stream);
}

} // namespace

uint64_t linear_attention_workspace_bytes(const AttentionArgs &args) {
    if (args.batch == 0 || args.heads == 0 || args.dv == 0 || !by_chunks(args)) return 0;
    const Parts parts = parts_of(args);
    return parts.parts > 1 ? args.batch * args.heads * parts.parts * args.dk * args.dv * sizeof(float) : 0;
}

hx_status launch_linear_attention(const AttentionArgs &args, void *ws, hipStream_t stream) {
    if (args.batch == 0 || args.heads == 0 || args.dv == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, ws, stream) : launch<bf16>(args, ws, stream);
}

} // namespace hx
