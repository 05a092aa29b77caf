// Linear attention with a decay for each head (hx_linear_attention), for
// gfx950:
//   S_t = e^g·S_{t-1} + k_tᵀ·v_t,   o_t = scale·q_t·S_t.
//
// Two forms.  The recurrence, for a few tokens: a block holds 32 columns of one
// head's state in registers, eight lanes of four columns by 32 groups of rows,
// and steps through the tokens.  Each step is a rank-1 update of the lane's own
// elements and a sum over the rows: within the wave by lane exchange, across the
// four waves through LDS (two buffers in turn, so one barrier a token); the next
// token's elements are on their way meanwhile.  The state's bytes, in and out,
// bound it: 128 sequences of 32 heads of 128 x 128 take 96 us, 5.6 TB/s; 50 of 4
// heads of 256 x 128 10.2.  Blocks of 64 or 128 columns, with whole rows of the
// state side by side but more registers, took 154 and 95 us, and for one
// sequence of 16 heads 6.3 and 6.8 us against 4.7.
//
// Chunks, for prompts: below.
#include "hx_internal.hpp"
#include "layer_device.hpp"

#include <atomic>
#include <type_traits>

namespace hx {
namespace {

// N neighbours of a row of T, in two steps, so that nothing waits for them before
// all loads are under way: where the row ends among them the N that end it are
// loaded, and shifted when they are used.  Past the row's end anything may come.
template <int N, typename T> struct RunOf {
    typedef T type __attribute__((ext_vector_type(N)));
    typedef T loaded __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N, typename T>
__device__ __forceinline__ typename RunOf<N, T>::type load_run(const T *p, uint32_t from, uint32_t end) {
    if (end >= N) return *(const typename RunOf<N, T>::loaded *)(p + min(from, end - N));
    typename RunOf<N, T>::type x = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (from + i < end) x[i] = p[from + i];
    return x;
}
template <int N, typename V> __device__ __forceinline__ V place_run(V x, uint32_t from, uint32_t end) {
    if (from + N <= end || end < N) return x;
    const uint32_t by = from + N - end;
#pragma unroll
    for (int d = 1; d < N; ++d)
#pragma unroll
        for (int i = 0; i + 1 < N; ++i) x[i] = by >= (uint32_t)d ? x[i + 1] : x[i];
    return x;
}

// Four columns of a row of the state from column c on, at any dword.  NT:
// streamed, not kept in the caches.
template <bool NT> __device__ __forceinline__ f32x4 load4(const float *row, uint32_t c, uint32_t width) {
    if (width < 4) return load_run<4>(row, c, width);
    return load_a4<NT>((const f32x4_a4 *)(row + min(c, width - 4)));
}
template <bool NT> __device__ __forceinline__ void store4(float *row, uint32_t c, uint32_t width, f32x4 v) {
    if (c + 4 <= width) {
        store_a4<NT>(v, (f32x4_a4 *)(row + c));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c + i < width) row[c + i] = v[i];
}

// All of the wave's LDS reads and writes have ended when it passes; loads from
// memory may be under way.
__device__ __forceinline__ void meet_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The decay of one token as a float and what its rounding leaves out, so that a
// state keeps the precision of f32 over any number of calls: by the float alone one
// that remembers 2^10 tokens is off by up to 2^-15.  Where the memory is long the
// rest comes from the series of e^g - 1; one of 16 tokens needs none.
struct StepDecay {
    float by, rest;
};
__device__ __forceinline__ StepDecay step_decay(float g) {
    if (!(g > -0.0625f)) return {expf(g), 0.0f};
    const float less = g * (1.0f + g * (1.0f / 2 + g * (1.0f / 6 + g * (1.0f / 24)))), by = 1.0f + less;
    return {by, less - (by - 1.0f)};
}

// A block takes COLUMNS columns of a state, four a lane, and all its rows, ROWS
// neighbours a lane: dk at most ROWS·1024 / COLUMNS.  Registers for four waves a SIMD:
// 32 x 32 heads of 64 x 64 take 8.4 us so and 9.8 without the bound, 50 x 4 of 256 x
// 128 10.8 and 30 (268 registers); streamed states, 128 x 32 heads of 128 x 128,
// 100 and 96.7, so they go without it up to four rows a lane.
template <typename T, int COLUMNS, int ROWS, bool NT>
__global__ __launch_bounds__(256, NT && ROWS < 8 ? 1 : 4) void attention_step_kernel(AttentionArgs a) {
    constexpr int kLanes = COLUMNS / 4; // of a row
    __shared__ f32x4 part[2][4][kLanes];
    const uint32_t h = blockIdx.y, b = blockIdx.z, hk = (uint32_t)(h / (a.heads / a.kv_heads));
    const uint32_t dk = (uint32_t)a.dk, dv = (uint32_t)a.dv;
    const uint32_t c = blockIdx.x * COLUMNS + threadIdx.x % kLanes * 4, row0 = threadIdx.x / kLanes * ROWS;
    const int wave = threadIdx.x / kWave;
    const uint64_t length = a.lengths ? min((uint64_t)a.lengths[b], a.tokens) : a.tokens;
    const T *q = (const T *)a.q + b * a.sq.batch + h * a.sq.head;
    const T *k = (const T *)a.k + b * a.sk.batch + hk * a.sk.head;
    const T *v = (const T *)a.v + b * a.sv.batch + hk * a.sv.head;
    T *out = (T *)a.out + b * a.so.batch + h * a.so.head;
    const float log_decay = a.log_decay[h];
    f32x4 s[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        s[r] = f32x4{0, 0, 0, 0};
        if (a.state_in && row0 + r < dk)
            s[r] = load4<NT>(a.state_in + b * a.si.batch + h * a.si.head + (row0 + r) * a.si.token, c, dv);
    }
    typename RunOf<4, T>::type vt = {};
    typename RunOf<ROWS, T>::type kt = {}, qt = {};
    const auto load = [&](uint64_t t) { // a token's elements, under way while the last one's output is summed
        vt = load_run<4>(v + (int64_t)t * a.sv.token, c, dv);
        kt = load_run<ROWS>(k + (int64_t)t * a.sk.token, row0, dk);
        qt = load_run<ROWS>(q + (int64_t)t * a.sq.token, row0, dk);
    };
    if (length) load(0);
    const StepDecay decay = step_decay(log_decay);
    if (c + 4 > dv)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) s[r] = place_run<4>(s[r], c, dv);
    // rest: what the token's decay takes off besides.  That of all the call's decays
    // goes with its first token; a token of the call itself lacks it, 2^-25 for each
    // of the few that follow.
    const auto token = [&](uint64_t t, auto rest) {
        vt = place_run<4>(vt, c, dv);
        kt = place_run<ROWS>(kt, row0, dk);
        qt = place_run<ROWS>(qt, row0, dk);
        const f32x4 values = {(float)vt[0], (float)vt[1], (float)vt[2], (float)vt[3]};
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            s[r] = decay.by * s[r] + rest(s[r], (float)kt[r] * values);
            // A row past dk adds nothing, whatever the value.
            if (row0 + r < dk) o += (float)qt[r] * s[r];
        }
        if (t + 1 < length) load(t + 1);
#pragma unroll
        for (int d = kLanes; d < kWave; d *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], d);
        f32x4(*buffer)[kLanes] = part[t & 1];
        if (lane_id() < kLanes) buffer[wave][lane_id()] = o;
        meet_lds();
        if (threadIdx.x < kLanes) {
            o = (buffer[0][threadIdx.x] + buffer[1][threadIdx.x]) + (buffer[2][threadIdx.x] + buffer[3][threadIdx.x]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < dv) out[(int64_t)t * a.so.token + c + i] = (T)(o[i] * a.scale);
        }
    };
    if (length) {
        const float rest = decay.rest * (float)length;
        token(0, [&](f32x4 state, f32x4 added) { return rest * state + added; });
    }
    for (uint64_t t = 1; t < length; ++t) token(t, [](f32x4, f32x4 added) { return added; });
    for (uint64_t t = length + threadIdx.x / kLanes; t < a.tokens; t += 256 / kLanes)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < dv) out[(int64_t)t * a.so.token + c + i] = (T)0.0f;
    if (!a.state_out) return;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (row0 + r < dk)
            store4<NT>(a.state_out + b * a.st.batch + h * a.st.head + (row0 + r) * a.st.token, c, dv, s[r]);
}

template <typename T, int COLUMNS, int ROWS> hx_status launch_step(const AttentionArgs &a, hipStream_t stream) {
    const dim3 grid((uint32_t)ceil_div(a.dv, COLUMNS), (uint32_t)a.heads, (uint32_t)a.batch);
    // Streams of four rows a lane are faster with five blocks a CU than with six: 31 KiB
    // of LDS, not used, leave room for five (128 x 32 heads of 128 x 128 96.6 us, 99.2; 40 x
    // 32 31.3, 32.3; of two rows 96.5, 90.4, of one 77.0, 53.1).
    const uint32_t lds = ROWS == 4 ? 31 * 1024 : 0;
    if (attention_streams_state(a))
        hipLaunchKernelGGL((attention_step_kernel<T, COLUMNS, ROWS, true>), grid, dim3(256), lds, stream, a);
    else hipLaunchKernelGGL((attention_step_kernel<T, COLUMNS, ROWS, false>), grid, dim3(256), 0, stream, a);
    return check_launch("attention_step_kernel");
}

template <typename T> hx_status launch_steps(const AttentionArgs &a, hipStream_t stream) {
    if (a.dk <= 32) return launch_step<T, 32, 1>(a, stream);
    if (a.dk <= 64) return launch_step<T, 32, 2>(a, stream);
    if (a.dk <= 128) return launch_step<T, 32, 4>(a, stream);
    return launch_step<T, 32, 8>(a, stream);
}

// ------------------------------------------------------------------ chunks
// Prompts, C tokens at a time.  With D = e^g and t, s counted within a chunk
// that holds r tokens and begins with the state S:
//   o_t = scale·(D^(t+1)·q_t·S + Σ_{s<=t} D^(t-s)·(q_t·k_s)·v_s)
//   S  <- D^r·S + Σ_s D^(r-1-s)·k_sᵀ·v_s
// All four products are matrix instructions.  A block takes one head and 16
// columns of v a wave; each wave keeps its columns of S, in f32, in registers for
// the whole prompt, and adds a chunk's sum to them once: in the accumulators
// of the last product S would be rounded at each instruction (in f32 eight times a
// chunk, an error of 7.8e-7 in the norm after 2048 tokens that are all remembered,
// 1.8e-7 so).
//
// What bounds a block of bf16 is LDS: every wave reads all of q and k, about 4000
// of a chunk's 10000 cycles at 64 tokens of 128 x 128, and then the arithmetic of
// the two and three terms (below).  8 x 32 heads of 128 x 128 over 4096 tokens take
// 306 us, 1.1 GB at 3.6 TB/s; loads and stores alone took 230.  Chunks of 128 tokens
// have no room beside the next one.  In f32 the matrix instructions weigh most, at
// a sixteenth of the rate of bf16: half of the 6.3 us of a chunk of 32 tokens of
// 80 x 96 (5 x 12 heads, up to 1000 tokens: 49 us, and 23 for the parts' sums).
//
// The accumulators of a 16 x 16 product hold, in lane l, column l % 16 and rows
// 4·(l / 16) + i.  An operand holds, in lane l, row or column l % 16 and the
// terms 4·(l / 16) + i of a run of 16.  So what one product leaves is an operand
// of the next without an exchange between lanes, if the products are taken
// transposed: Pᵀ = K·Qᵀ, Oᵀ = Sᵀ·Qᵀ + Vᵀ·Pᵀ.  Only P passes through LDS, because
// every wave needs all of it.
//
// Roundings, where the elements are bf16: an element of P, and of S where a
// query meets it, is taken as two bf16 terms, which hold 16 bits, so that an
// output keeps the 8 bits of its own rounding, as those of single tokens do.  One
// term each took 270 us where these take 302, and made the error of an output in
// the norm 1.4 times as large.  The sums that go into S keep all bits: a weighted
// value D^(r-1-s)·v is three terms.
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

// The same in the two terms that an output needs: the first cut off, so that no
// finite value becomes an infinity, the second rounded.
template <typename T> constexpr int kOutTerms = sizeof(T) == 2 ? 2 : 1;
__device__ __forceinline__ void split_two(f32x4v v, bf16x4 (&to)[2]) {
    const s16x4 high = {(short)(__float_as_uint(v[0]) >> 16), (short)(__float_as_uint(v[1]) >> 16),
                        (short)(__float_as_uint(v[2]) >> 16), (short)(__float_as_uint(v[3]) >> 16)};
    to[0] = __builtin_bit_cast(bf16x4, high);
    to[1] = rounded(v - widened(to[0]), bf16{});
}
__device__ __forceinline__ void split_two(f32x4v v, f32x4v (&to)[1]) { to[0] = v; }

// The same value, which the compiler cannot know: what is computed from it stays
// where it is written, in a branch that is seldom taken, and takes up no
// registers outside.
__device__ __forceinline__ uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Whether an element is an infinity or no number: an exponent of ones, which
// carries into the sign.
template <int N> __device__ __forceinline__ bool not_finite(const bf16x4 (&v)[N]) {
    uint32_t carry = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint2 two = __builtin_bit_cast(uint2, v[n]);
        carry |= ((two.x & 0x7F807F80u) + 0x00800080u) | ((two.y & 0x7F807F80u) + 0x00800080u);
    }
    return (carry & 0x80008000u) != 0;
}
template <int N> __device__ __forceinline__ bool not_finite(const f32x4v (&v)[N]) {
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += v[n][e] * 0.0f;
    return !(sum == 0.0f);
}

// A tile in LDS: rows of WIDTH elements (a power of two) as 16-byte slots.  Slot
// c of row r lies at place c ^ turned(r), so that what is read at once lies on
// different banks: sixteen rows at one slot, and of bf16 tiles that are read
// down columns too, of rows 4·q..4·q + 3 the halves of four slots.  Cycles of a
// wave's instruction with eight waves reading: 16 bytes a lane 6.7 (ROWS, row & 15)
// and 8.2 (else), down columns 8.1 and 6.5; without turning 32 and 16.
template <typename T, int WIDTH, bool ROWS> struct TileOf {
    static constexpr int V = 16 / (int)sizeof(T), kSlots = WIDTH / V, kRow = WIDTH * (int)sizeof(T);
    static_assert(kSlots >= 8 && (kSlots & (kSlots - 1)) == 0);
    static __device__ __forceinline__ uint32_t turned(uint32_t row) {
        if constexpr (kSlots == 8) return (row & 1) << 2 | (row >> 2 & 1) << 1 | (row >> 1 & 1);
        if constexpr (ROWS || sizeof(T) == 4) return row & 15;
        return (row & 3) << 2 | (row >> 2 & 3);
    }
    static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t slot) { // bytes
        return row * kRow + (slot ^ turned(row)) * 16;
    }
};

// Terms 32·i + 8·(l / 16) on, eight neighbours of row l % 16 of the sixteen from
// row `first` on, as the two halves of an operand.
template <int WIDTH, bool ROWS>
__device__ __forceinline__ void load_terms(const char *tile, int first, int i, bf16x4 (&f)[2]) {
    using Tile = TileOf<bf16, WIDTH, ROWS>;
    const int l = lane_id();
    const bf16x8 v = *(const bf16x8 *)(tile + first * Tile::kRow + Tile::place(l % 16, i * 4 + l / 16));
    f[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    f[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
}
template <int WIDTH, bool ROWS>
__device__ __forceinline__ void load_terms(const char *tile, int first, int i, f32x4v (&f)[2]) {
    using Tile = TileOf<float, WIDTH, ROWS>;
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < 2; ++n)
        f[n] = *(const f32x4v *)(tile + first * Tile::kRow + Tile::place(l % 16, i * 8 + l / 16 * 2 + n));
}

// A state S, [dk, columns of v], lies in accumulators of 16 rows each.  Row
// 4·(l / 16) + e of accumulator i is row state_row(i, e) of S; the rows of two
// accumulators, 32·(i / 2) on, are ordered as suits the reads below.
//
// load_state_terms: of row l % 16 of the sixteen from row `first` on, the terms
// that accumulators 2·i and 2·i + 1 hold in this lane.
// load_columns: terms down column l % 16 of the sixteen that accumulator 2·i holds:
// rows 4·(l / 16) + e of each of the BLOCKS sixteens of the tile's rows, then the
// same for accumulator 2·i + 1.
// load_column: the same down column `column` + l % 16.
template <typename T> __device__ __forceinline__ uint32_t state_row(int i, int e) {
    const int q = lane_id() / 16;
    if constexpr (sizeof(T) == 4) return i * 16 + q * 4 + e;
    return i / 2 * 32 + q * 8 + i % 2 * 4 + e;
}
template <int WIDTH>
__device__ __forceinline__ void load_state_terms(const char *tile, int first, int i, bf16x4 (&f)[2]) {
    load_terms<WIDTH, true>(tile, first, i, f);
}
template <int WIDTH>
__device__ __forceinline__ void load_state_terms(const char *tile, int first, int i, f32x4v (&f)[2]) {
    using Tile = TileOf<float, WIDTH, true>;
    const int l = lane_id();
    const uint32_t at = Tile::place(l % 16, i * 8 + l / 16);
    f[0] = *(const f32x4v *)(tile + first * Tile::kRow + at);
    f[1] = *(const f32x4v *)(tile + first * Tile::kRow + (at ^ 64)); // four slots on
}

// The transposing read: lane l names row 4·(l / 16) + l % 16 / 4 and four columns
// of it, and receives one column of its sixteen lanes' rows.  It is written
// out, with its wait, because the compiler puts a wait for all loads that write
// LDS in front of the builtin, those of later chunks among them.
__device__ __forceinline__ uint32_t lds_address(const char *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}
template <int WIDTH, int BLOCKS>
__device__ __forceinline__ void load_columns(const char *tile, int i, bf16x4 (&to)[2 * BLOCKS]) {
    static_assert(BLOCKS == 4);
    using Tile = TileOf<bf16, WIDTH, false>;
    constexpr int kStep = 16 * Tile::kRow;
    const int l = lane_id();
    const uint32_t at = lds_address(tile) + Tile::place(l / 16 * 4 + l % 16 / 4, i * 4 + l % 4);
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%9\n\t"
                 "ds_read_b64_tr_b16 %2, %8 offset:%10\n\tds_read_b64_tr_b16 %3, %8 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:8\n\tds_read_b64_tr_b16 %5, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %6, %8 offset:%13\n\tds_read_b64_tr_b16 %7, %8 offset:%14\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(to[0]), "=&v"(to[1]), "=&v"(to[2]), "=&v"(to[3]), "=&v"(to[4]), "=&v"(to[5]), "=&v"(to[6]),
                   "=&v"(to[7])
                 : "v"(at), "i"(kStep), "i"(2 * kStep), "i"(3 * kStep), "i"(kStep + 8), "i"(2 * kStep + 8),
                   "i"(3 * kStep + 8));
}
template <int WIDTH, int BLOCKS>
__device__ __forceinline__ void load_column(const char *tile, int column, bf16x4 (&to)[BLOCKS]) {
    static_assert(BLOCKS == 4);
    using Tile = TileOf<bf16, WIDTH, false>;
    constexpr int kStep = 16 * Tile::kRow;
    const int l = lane_id(), c = column + l % 4 * 4;
    const uint32_t at = lds_address(tile) + Tile::place(l / 16 * 4 + l % 16 / 4, c / 8) + c % 8 * 2;
    asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%5\n\t"
                 "ds_read_b64_tr_b16 %2, %4 offset:%6\n\tds_read_b64_tr_b16 %3, %4 offset:%7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(to[0]), "=&v"(to[1]), "=&v"(to[2]), "=&v"(to[3])
                 : "v"(at), "i"(kStep), "i"(2 * kStep), "i"(3 * kStep));
}
template <int WIDTH, int BLOCKS>
__device__ __forceinline__ void load_column(const char *tile, int column, f32x4v (&to)[BLOCKS]) {
    using Tile = TileOf<float, WIDTH, false>;
    const int l = lane_id(), at = column + l % 16;
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            to[n][e] = *(const float *)(tile + n * 16 * Tile::kRow + Tile::place(l / 16 * 4 + e, at / 4) + at % 4 * 4);
}
template <int WIDTH, int BLOCKS>
__device__ __forceinline__ void load_columns(const char *tile, int i, f32x4v (&to)[2 * BLOCKS]) {
    f32x4v part[2][BLOCKS];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        load_column<WIDTH, BLOCKS>(tile, i * 32 + j * 16, part[j]);
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n) to[j * BLOCKS + n] = part[j][n];
    }
}

// ROWS rows of a head on their way from memory to a tile, by all threads of the
// block.  Rows from `rows` on and columns from `width` on become zeros.
//
// DIRECT: loads that write LDS without registers, for rows that begin on dwords
// and are whole 16-byte slots.  Every lane loads every time, so that a count of
// loads under way says which have landed: lanes outside the rows load zeros.
// Otherwise through registers.  AGAIN: places and addresses are computed anew for
// each chunk, where the registers do not hold them all: eight waves with keys of
// 128 in bf16 spilled five a lane (8 x 32 heads of 127 x 127 over 2048 tokens 256
// us, 236 so; elsewhere it costs 2 to 5%).
__device__ const uint32_t kZeros[4] = {0, 0, 0, 0};

template <typename T, int ROWS, int WIDTH, bool BY_ROWS, int THREADS, bool DIRECT, bool AGAIN> struct Stager {
    using Tile = TileOf<T, WIDTH, BY_ROWS>;
    static constexpr int V = Tile::V, N = ROWS * Tile::kSlots / THREADS;
    static_assert(N * THREADS == ROWS * Tile::kSlots);
    typedef typename std::conditional<sizeof(T) == 2, u32x4_a2, u32x4_a4>::type Vec;
    uint32_t offset[DIRECT ? N : 1]; // bytes from a chunk's first row
    u32x4 held[DIRECT ? 1 : N];

    // Thread t of a step fills place t % kSlots of row t / kSlots.
    static __device__ __forceinline__ uint32_t row_of(uint32_t t, int i) { return (t + i * THREADS) / Tile::kSlots; }
    static __device__ __forceinline__ uint32_t slot_of(uint32_t t, int i) {
        return t % Tile::kSlots ^ Tile::turned(row_of(t, i));
    }
    __device__ __forceinline__ void begin(int64_t stride) {
        if constexpr (DIRECT)
#pragma unroll
            for (int i = 0; i < N; ++i)
                offset[i] = (row_of(threadIdx.x, i) * (uint32_t)stride + slot_of(threadIdx.x, i) * V) * (uint32_t)sizeof(T);
    }
    __device__ __forceinline__ void load(const T *base, int64_t stride, uint32_t rows, uint32_t width, char *tile) {
        if constexpr (DIRECT) {
            char *wave = tile + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * (kWave * 16);
            const auto put = [&](int i, const void *p) {
                __builtin_amdgcn_global_load_lds(
                    p, (__attribute__((address_space(3))) void *)(wave + i * THREADS * 16), 16, 0, 0);
            };
            if (rows >= ROWS && width == WIDTH) {
#pragma unroll
                for (int i = 0; i < N; ++i) put(i, (const char *)base + offset[i]);
            } else {
                const uint32_t t = here(threadIdx.x);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    put(i, row_of(t, i) < rows && slot_of(t, i) * V < width ? (const char *)base + offset[i]
                                                                          : (const char *)kZeros);
            }
            return;
        }
        const uint32_t t = AGAIN ? here(threadIdx.x) : threadIdx.x;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t row = row_of(t, i), c = slot_of(t, i) * V;
            if constexpr (!DIRECT) {
                held[i] = u32x4{0, 0, 0, 0};
                if (row < rows) held[i] = load_part(base + (int64_t)row * stride, c, width);
            }
        }
    }
    __device__ __forceinline__ void store(char *tile, uint32_t width) const {
        if constexpr (!DIRECT) {
            const uint32_t t = AGAIN ? here(threadIdx.x) : threadIdx.x;
#pragma unroll
            for (int i = 0; i < N; ++i)
                *(u32x4 *)(tile + (t + i * THREADS) * 16) = place_part<T>(held[i], slot_of(t, i) * V, width);
        }
    }
};

// All of the wave's LDS reads and writes and all but its last N transfers of
// memory have ended when it passes.
template <int N> __device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <typename T, int DK, int NW, bool OUTPUTS, bool DIRECT> struct Chunk {
    static constexpr int C = sizeof(T) == 2 ? 64 : 32, B = C / 16, // tokens, and sixteens of them
                          kThreads = NW * kWave, DV = NW * 16;
    static constexpr int WK = DK <= 64 ? 64 : DK <= 128 ? 128 : 256; // rows of q and k in LDS
    static constexpr int kTileK = C * WK * (int)sizeof(T), kTileV = C * DV * (int)sizeof(T);
    static constexpr int kStage = (OUTPUTS ? 2 : 1) * kTileK + kTileV;
    // P, on and below the diagonal.
    static constexpr int kTiles = B * (B + 1) / 2;
    static constexpr int kScores = OUTPUTS ? kTiles * kOutTerms<T> * 4 * kWave * (int)sizeof(T) : 0;
    // Chunks in LDS: one read, the others on their way; two where that lets LDS
    // hold two blocks.
    static constexpr int kHalf = 80 * 1024;
    static constexpr int kRoom = NW == 4 && DK <= 128 && 2 * kStage + kScores <= kHalf ? kHalf : 2 * kHalf;
    static constexpr int S = DIRECT && 3 * kStage + kScores <= kRoom ? 3 : 2;
    static constexpr int kLds = S * kStage + kScores;
    static_assert(kLds <= 160 * 1024);
    // Where LDS holds two blocks of four waves, so must the registers: 1 x 50 heads of
    // 37 x 53 over 4096 tokens take 84 us with one block a CU, 65 with two.  (At dk of
    // 256 they would spill.)
    static constexpr int kWavesPerSimd = NW == 4 && DK <= 128 && 2 * kLds <= 160 * 1024 ? 2 : NW / 4;
};

// OUTPUTS: the outputs of a part, from the state before it.  Otherwise only the
// part's own sum, from nothing.
template <typename T, int DK, int NW, bool OUTPUTS, bool DIRECT>
__global__ __launch_bounds__(NW *kWave, (Chunk<T, DK, NW, OUTPUTS, DIRECT>::kWavesPerSimd)) void attention_chunk_kernel(AttentionArgs a, AttentionParts parts) {
    using G = Chunk<T, DK, NW, OUTPUTS, DIRECT>;
    using F = typename Fragment<T>::type;
    constexpr int C = G::C, B = G::B, S = G::S, WK = G::WK, DV = G::DV;
    extern __shared__ __align__(16) char lds[];
    F *ps = (F *)(lds + S * G::kStage);
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

    // The decay as a power of two a token; minus infinity would make 0·log a NaN,
    // and a NaN has to stay one.
    const float log_decay = a.log_decay[h];
    const float log2_decay = log_decay < -1e30f ? -1e30f : log_decay * 1.44269504f;
    const auto power = [&](int n) { return __builtin_amdgcn_exp2f(log2_decay * (float)n); };

    const uint32_t chunks = begin < end ? (end - begin + C - 1) / C : 0;
    constexpr bool kAgain = !DIRECT && OUTPUTS && sizeof(T) == 2 && DK == 128 && NW == 8;
    Stager<T, C, WK, true, G::kThreads, DIRECT, kAgain> to_q;
    Stager<T, C, WK, false, G::kThreads, DIRECT, kAgain> to_k;
    Stager<T, C, DV, false, G::kThreads, DIRECT, kAgain> to_v;
    to_k.begin(a.sk.token);
    to_v.begin(a.sv.token);
    if constexpr (OUTPUTS) to_q.begin(a.sq.token);
    constexpr int kLoads = to_k.N + to_v.N + (OUTPUTS ? to_q.N : 0); // instructions a chunk
    const auto stage_of = [&](uint32_t n) { return lds + n % S * G::kStage; };
    const auto fetch = [&](uint32_t n) {
        const uint32_t t0 = begin + n * C, rows = end - t0;
        char *stage = stage_of(n);
        to_k.load(k + (int64_t)t0 * a.sk.token, a.sk.token, rows, dk, stage);
        to_v.load(v + (int64_t)t0 * a.sv.token, a.sv.token, rows, dv, stage + G::kTileK);
        if constexpr (OUTPUTS)
            to_q.load(q + (int64_t)t0 * a.sq.token, a.sq.token, rows, dk, stage + G::kTileK + G::kTileV);
    };
    const auto fetch_ahead = [&](uint32_t n) {
        const uint32_t ahead = n + (DIRECT ? S - 1 : 1);
        if (ahead < chunks) fetch(ahead);
    };
    // A chunk's outputs, from their place in LDS as whole rows.
    const auto write_out = [&](uint32_t n) {
        const char *tile = stage_of(n) + G::kTileK;
        const uint32_t t0 = begin + n * C;
        T *rows = out + (int64_t)t0 * a.so.token;
        using ToOut = Stager<T, C, DV, false, G::kThreads, false, false>;
        u32x4 held[ToOut::N];
#pragma unroll
        for (int i = 0; i < ToOut::N; ++i) held[i] = *(const u32x4 *)(tile + (threadIdx.x + i * G::kThreads) * 16);
#pragma unroll
        for (int i = 0; i < ToOut::N; ++i) {
            const uint32_t row = ToOut::row_of(threadIdx.x, i), c = ToOut::slot_of(threadIdx.x, i) * ToOut::V;
            T *to = rows + (int64_t)row * a.so.token + c;
            if (row >= end - t0) continue;
            if (c + ToOut::V <= dv) {
                *(typename ToOut::Vec *)to = held[i];
            } else {
                T part[ToOut::V];
                __builtin_memcpy(part, &held[i], 16);
#pragma unroll
                for (int e = 0; e < ToOut::V; ++e)
                    if (c + e < dv) to[e] = part[e];
            }
        }
    };
    const auto settle = [&](uint32_t n) { // what went through registers
        char *stage = stage_of(n);
        to_k.store(stage, dk);
        to_v.store(stage + G::kTileK, dv);
        if constexpr (OUTPUTS) to_q.store(stage + G::kTileK + G::kTileV, dk);
    };
    if constexpr (DIRECT) {
        for (uint32_t n = 0; n < S - 1 && n < chunks; ++n) fetch(n);
    } else if (chunks) {
        fetch(0);
        settle(0);
    }
    f32x4v s[DK / 16] = {};
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
                if (from && state_row<T>(i, e) < dk) s[i][e] = from[state_row<T>(i, e) * stride];
    }

    // The decay over a chunk, as a float and what its rounding leaves out: the
    // state keeps the precision of f32 however many chunks there are.
    struct Decay {
        float by, rest;
    };
    const auto decay_over = [&](uint32_t rows) {
        const double d = exp((double)log_decay * rows);
        const float by = (float)d;
        return Decay{by, (float)(d - by)};
    };
    const Decay decay = decay_over(C), last_decay = decay_over(chunks ? end - begin - (chunks - 1) * C : 1);
    // Powers of the decay: over 16 tokens; in a whole chunk's last 16 rows, the
    // weight of a row in the state; at a token of the first 16, of the state.
    const float over16 = power(16), query_weight = power(col + 1) * a.scale;
    f32x4v last_weight;
#pragma unroll
    for (int e = 0; e < 4; ++e) last_weight[e] = power(15 - quad * 4 - e);

    // The state has come: or the compiler waits for it in every chunk, and there
    // for all loads under way.
    __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
    for (uint32_t n = 0; n < chunks; ++n) {
        const uint32_t t0 = begin + n * C;
        const int rows = (int)min((uint32_t)C, end - t0);
        // Chunk n has landed once no more is under way than the chunks after it.
        if (DIRECT && n + S - 2 < chunks) meet<(S - 2) * kLoads>();
        else meet<0>();
        if constexpr (OUTPUTS) {
            if (n) write_out(n - 1);
        } else {
            fetch_ahead(n);
        }
        char *ks = stage_of(n), *vs = ks + G::kTileK, *qs = vs + G::kTileV;

        F vf[B]; // this lane's column of v
        load_column<DV, B>(vs, wave * 16, vf);

        f32x4v o[B] = {};
        const auto outputs = [&] {
            // Pᵀ tiles (x: rows of k, y: rows of q), the waves in turn.
#pragma unroll 1
            for (int tile = wave; tile < B * (B + 1) / 2; tile += NW) {
                const int y = (tile >= 1) + (tile >= 3) + (tile >= 6), x = tile - y * (y + 1) / 2;
                f32x4v p = {};
#pragma unroll
                for (int i = 0; i < DK / 32; ++i) {
                    F fk[2], fq[2];
                    load_terms<WK, false>(ks, x * 16, i, fk);
                    load_terms<WK, true>(qs, y * 16, i, fq);
                    p = mma(fk, fq, p);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int far = (y * 16 + col) - (x * 16 + quad * 4 + e);
                    p[e] = far >= 0 ? p[e] * (power(far) * a.scale) : 0.0f;
                }
                F terms[kOutTerms<T>];
                split_two(p, terms);
#pragma unroll
                for (int m = 0; m < kOutTerms<T>; ++m) ps[(m * G::kTiles + tile) * kWave + lane] = terms[m];
            }
            // The state's part of the outputs.
#pragma unroll
            for (int i = 0; i < DK / 32; ++i) {
                F even[kOutTerms<T>], odd[kOutTerms<T>];
                split_two(s[2 * i], even);
                split_two(s[2 * i + 1], odd);
#pragma unroll
                for (int y = 0; y < B; ++y) {
                    F fq[2];
                    load_state_terms<WK>(qs, y * 16, i, fq);
#pragma unroll
                    for (int m = kOutTerms<T> - 1; m >= 0; --m) {
                        const F state[2] = {even[m], odd[m]};
                        o[y] = mma(state, fq, o[y]);
                    }
                }
            }
            float weight = query_weight;
#pragma unroll
            for (int y = 0; y < B; ++y, weight *= over16) o[y] *= weight;
        };
        const auto advance = [&] {
            // The state: decayed over the chunk, and the chunk's sum, which is taken
            // apart so that the state is rounded once a chunk and not at each product.
            const Decay over = rows < C ? last_decay : decay;
            F terms[B][kTerms<T>];
            f32x4v weight = last_weight;
#pragma unroll
            for (int x = B - 1; x >= 0; --x, weight *= over16) {
                if (rows < C) {
                    const int left = rows - 1 - x * 16 - (int)here(quad * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) weight[e] = power(max(left - e, 0));
                }
                split(widened(vf[x]) * weight, terms[x]);
            }
#pragma unroll
            for (int i = 0; i < DK / 16; i += 2) {
                F fk[2 * B];
                load_columns<WK, B>(ks, i / 2, fk);
                f32x4v sum[2] = {};
#pragma unroll
                for (int m = kTerms<T> - 1; m >= 0; --m)
#pragma unroll
                    for (int x = 0; x < B; x += 2) {
                        const F fv[2] = {terms[x][m], terms[x + 1][m]};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const F f[2] = {fk[j * B + x], fk[j * B + x + 1]};
                            sum[j] = mma(f, fv, sum[j]);
                        }
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[i + j][e] = fmaf(s[i + j][e], over.by, fmaf(s[i + j][e], over.rest, sum[j][e]));
            }
        };
        if constexpr (OUTPUTS) outputs();
        advance();

        if constexpr (OUTPUTS) {
            // A value that is no number would also spoil the tokens before it,
            // whose weights are 0: it is taken out, and its mark put where it
            // belongs.
            int first_bad = C; // the first token of one, in this lane's column
            if (__any(not_finite(vf))) {
#pragma unroll
                for (int x = B - 1; x >= 0; --x) {
                    f32x4v w = widened(vf[x]);
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (!(w[e] * 0.0f == 0.0f)) {
                            first_bad = x * 16 + quad * 4 + e;
                            w[e] = 0.0f;
                        }
                    vf[x] = rounded(w, T{});
                }
                first_bad = min(first_bad, __shfl_xor(first_bad, 16));
                first_bad = min(first_bad, __shfl_xor(first_bad, 32));
            }
            meet_lds(); // P is whole, the last chunk's outputs have left LDS
            fetch_ahead(n);
#pragma unroll
            for (int y = 0; y < B; ++y)
#pragma unroll
                for (int x = 0; x <= y; x += 2) {
                    const F fv[2] = {vf[x], vf[x + 1]};
#pragma unroll
                    for (int m = kOutTerms<T> - 1; m >= 0; --m) {
                        const F *p = ps + (m * G::kTiles + y * (y + 1) / 2 + x) * kWave + lane;
                        const F fp[2] = {p[0], x < y ? p[kWave] : F{}};
                        o[y] = mma(fv, fp, o[y]);
                    }
                }
            if (__any(first_bad < C)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int from = __shfl(first_bad, quad * 4 + e); // of the row of o, a column of v
#pragma unroll
                    for (int y = 0; y < B; ++y)
                        if (y * 16 + col >= from) o[y][e] = __builtin_nanf("");
                }
            }
            // The outputs take the place of v, which all waves have read.
#pragma unroll
            for (int y = 0; y < B; ++y) {
                const F r = rounded(o[y], T{});
                const int c = wave * 16 + quad * 4;
                using Tile = TileOf<T, DV, false>;
                *(F *)(vs + Tile::place(y * 16 + col, c / Tile::V) + c % Tile::V * sizeof(T)) = r;
            }
        }

        if (!DIRECT && n + 1 < chunks) settle(n + 1);
    }

    if constexpr (OUTPUTS) {
        if (chunks) {
            meet_lds();
            write_out(chunks - 1);
        }
        // Rows past the sequence's end.
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
            if (to && state_row<T>(i, e) < dk) to[state_row<T>(i, e) * stride] = s[i][e];
}

// The state before each part, from the parts' own sums: V elements of a row of
// the state a thread, the parts in order, sixteen of them loaded together.  V is 4
// where rows are whole fours: 2 x 32 heads of 128 x 128 in four parts take 8.4 us
// so, 12.3 with one element a thread.
template <int V> __global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a, AttentionParts parts) {
    typedef float Values __attribute__((ext_vector_type(V), aligned(4)));
    const uint32_t n = (uint32_t)(a.dk * a.dv), i = (blockIdx.x * 256 + threadIdx.x) * V;
    if (i >= n) return;
    const uint32_t h = blockIdx.y, b = blockIdx.z, row = i / (uint32_t)a.dv, col = i % (uint32_t)a.dv;
    const uint32_t tokens = (uint32_t)a.tokens, length = a.lengths ? min(a.lengths[b], tokens) : tokens;
    float *at = parts.states + ((uint64_t)b * a.heads + h) * parts.parts * n + i;
    constexpr uint32_t kBatch = 16;
    Values own[kBatch] = {};
    const auto load = [&](uint32_t p) {
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
            if (p + k < parts.parts) own[k] = *(const Values *)(at + (uint64_t)(p + k) * n);
    };
    load(0);
    Values s = {};
    if (a.state_in) s = *(const Values *)(a.state_in + b * a.si.batch + h * a.si.head + row * a.si.token + col);
    const double log_decay = a.log_decay[h];
    // Every part but the last with tokens is whole, and those behind it have none:
    // there the state stays as it is, whatever it holds.
    const uint32_t whole = length / parts.span, rest = length % parts.span, used = whole + (rest != 0);
    const double of_whole = exp(log_decay * parts.span), of_rest = exp(log_decay * rest);
    const float whole_high = (float)of_whole, whole_low = (float)(of_whole - whole_high);
    const float rest_high = (float)of_rest, rest_low = (float)(of_rest - rest_high);
    for (uint32_t p = 0;;) {
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) {
            if (p + k >= parts.parts) break;
            *(Values *)(at + (uint64_t)(p + k) * n) = s;
            if (p + k >= used) continue;
            const float high = p + k < whole ? whole_high : rest_high, low = p + k < whole ? whole_low : rest_low;
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] = fmaf(s[e], high, fmaf(s[e], low, own[k][e]));
        }
        if ((p += kBatch) >= parts.parts) break;
        load(p);
    }
    if (a.state_out) *(Values *)(a.state_out + b * a.st.batch + h * a.st.head + row * a.st.token + col) = s;
}

template <typename T, int DK, int NW, bool DIRECT>
hx_status launch_chunks(const AttentionArgs &a, void *ws, hipStream_t stream) {
    AttentionParts parts = attention_parts(a);
    parts.states = (float *)ws;
    const auto run = [&](auto outputs) {
        using G = Chunk<T, DK, NW, decltype(outputs)::value, DIRECT>;
        const auto kernel = attention_chunk_kernel<T, DK, NW, decltype(outputs)::value, DIRECT>;
        static std::atomic<uint64_t> allowed{0};
        HX_TRY(allow_lds((const void *)kernel, G::kLds, allowed));
        const uint64_t x = ceil_div(a.dv, G::DV) * parts.parts;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)x, (uint32_t)a.heads, (uint32_t)a.batch), dim3(G::kThreads), G::kLds,
                           stream, a, parts);
        return check_launch("attention_chunk_kernel");
    };
    if (parts.parts > 1) {
        HX_TRY(run(std::false_type{}));
        const uint32_t wide = a.dv % 4 == 0 ? 4 : 1;
        hipLaunchKernelGGL(wide == 4 ? attention_join_kernel<4> : attention_join_kernel<1>,
                           dim3((uint32_t)ceil_div(a.dk * a.dv, 256 * wide), (uint32_t)a.heads, (uint32_t)a.batch),
                           dim3(256), 0, stream, a, parts);
        HX_TRY(check_launch("attention_join_kernel"));
    }
    return run(std::true_type{});
}

template <typename T, int NW, bool DIRECT> hx_status launch_width(const AttentionArgs &a, void *ws, hipStream_t stream) {
    switch (attention_key_width(a.dk)) {
    case 64: return launch_chunks<T, 64, NW, DIRECT>(a, ws, stream);
    case 96: return launch_chunks<T, 96, NW, DIRECT>(a, ws, stream);
    case 128: return launch_chunks<T, 128, NW, DIRECT>(a, ws, stream);
    default:
        if constexpr (NW == 4) return launch_chunks<T, 256, NW, DIRECT>(a, ws, stream);
    }
    return fail(HX_ERR_DISPATCH_FAILED, "no attention block for keys of width %llu", (unsigned long long)a.dk);
}
template <typename T, bool DIRECT> hx_status launch_chunked(const AttentionArgs &a, void *ws, hipStream_t stream) {
    return attention_waves(a) == 4 ? launch_width<T, 4, DIRECT>(a, ws, stream) : launch_width<T, 8, DIRECT>(a, ws, stream);
}

template <typename T> hx_status launch(const AttentionArgs &a, void *ws, hipStream_t stream) {
    if (attention_by_chunks(a)) {
        return attention_is_direct(a) ? launch_chunked<T, true>(a, ws, stream) : launch_chunked<T, false>(a, ws, stream);
    }
    return launch_steps<T>(a, stream);
}

} // namespace

uint64_t linear_attention_workspace_bytes(const AttentionArgs &args) {
    if (args.batch == 0 || args.heads == 0 || args.dv == 0 || !attention_by_chunks(args)) return 0;
    const AttentionParts parts = attention_parts(args);
    return parts.parts > 1 ? args.batch * args.heads * parts.parts * args.dk * args.dv * sizeof(float) : 0;
}

hx_status launch_linear_attention(const AttentionArgs &args, void *ws, hipStream_t stream) {
    if (args.batch == 0 || args.heads == 0 || args.dv == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, ws, stream) : launch<bf16>(args, ws, stream);
}

} // namespace hx
