// Gated recurrence of each channel along the tokens (hx_gated_recurrence) and its
// backward pass (hx_gated_recurrence_backward), for gfx950.
//
//   f = 1 / (1 + e^-z),  h_t = f_t·h_{t-1} + (1 - f_t)·x_t
// backward, from the last token on, with c the gradient of the state so far:
//   g_t = dy_t + c_t,  c_{t-1} = f_t·g_t,  dx = (1 - f)·g,  dz = f·(1 - f)·g·(h_{t-1} - x)
//
// Both are scans of the maps s -> A·s + B.  A block has 256 bytes of channels, a
// dword a lane, and goes through the tokens in tiles: each of its waves takes a run
// of R tokens from a zero state, the waves' maps meet in LDS, and what came in is added to
// each token by the product of the factors up to it.  The next tile's loads are
// under way meanwhile.  Where sequences and channels are too few to fill the card,
// the tokens are cut into parts: a first launch takes the parts' maps, which
// every block of the second one follows up to its own part.  All sums have one
// order: every run gives the same bits.
//
// Memory bounds the long ones: 8 x 4096 x 4096 bf16 takes 171 us (4.7 TB/s), 1 x 65536 x
// 2048 backward 468 us, of which 160 take the parts' maps, so that the gate and dy are read
// twice (4.6 TB/s of both launches' bytes).  A token of 64 x 4096 takes 3.7 us, a launch and a
// wait.  Short ones in parts are two launches and their waits: 1 x 4406 x 96 backward 23 us.
#include "hx_internal.hpp"
#include "layer_device.hpp"

namespace hx {
namespace {

// V neighbouring channels of a lane: a dword, or one element where rows do not lie
// on dwords.
template <typename T, int V> struct Lane {
    using Raw = typename std::conditional<sizeof(T) * V == 4, uint32_t, uint16_t>::type;
    static __device__ __forceinline__ Raw load(const T *p) { return *(const Raw *)p; }
    static __device__ __forceinline__ void values(Raw r, float (&x)[V]) {
        if constexpr (sizeof(T) == 4) {
            x[0] = __builtin_bit_cast(float, r);
        } else {
            x[0] = __builtin_bit_cast(float, (uint32_t)r << 16);
            if constexpr (V == 2) x[1] = __builtin_bit_cast(float, r & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void store(T *p, const float (&x)[V]) {
        if constexpr (sizeof(T) == 4) {
            *p = x[0];
        } else if constexpr (V == 2) {
            typedef bf16 Two __attribute__((ext_vector_type(2)));
            *(uint32_t *)p = __builtin_bit_cast(uint32_t, Two{(bf16)x[0], (bf16)x[1]});
        } else {
            *p = (bf16)x[0];
        }
    }
};

// s -> A·s as `by`: A where it is below a half, else A - 1, which has the minus sign.  A
// factor near 1 is so applied as s - (1 - A)·s: its own rounding, 2^-25, would be the same
// in every token, or run of tokens, of a steady gate and add up.
__device__ __forceinline__ float apply(float by, float s) {
    return __builtin_fmaf(by, s, __builtin_signbit(by) ? s : 0.0f);
}
// An infinite s makes a NaN of s - (1 - A)·s.  Here only what is finite of it is taken away
// and it stays what it is, as A·s does; two instructions more.  That is for the one
// application a call of a few tokens: where every token has it, 8 x 4096 x 4096 bf16 takes
// 184 us against 172, and 8 waves that join by it, or keep such states apart, 174 to 177
// forward and 338 against 322 backward.
__device__ __forceinline__ float apply_infinite(float by, float s) {
    const bool is_near = __builtin_signbit(by);
    return __builtin_fmaf(by, is_near ? __builtin_amdgcn_fmed3f(s, -__FLT_MAX__, __FLT_MAX__) : s, is_near ? s : 0.0f);
}

// f = 1 / (1 + e^-z), 1 - f, and f as it is applied, from e^-|z|.  For f32 the
// exponential has the rest that the product with log2(e) leaves; a bf16 gate itself is off
// by more.
struct Gate {
    float f, rest, by;
};
template <typename T> __device__ __forceinline__ Gate gate_of(float z) {
    constexpr float kLog2e = 1.44269502f, kLow = 1.92596299e-8f; // their sum is log2(e) to 2^-50
    float e;
    if constexpr (sizeof(T) == 4) {
        const float a = fabsf(z) > 200.0f ? 200.0f : fabsf(z); // e^-200 is nothing; a NaN stays
        const float t = -a * kLog2e, low = __builtin_fmaf(-a, kLog2e, -t) - a * kLow;
        e = __builtin_amdgcn_exp2f(t);
        e = __builtin_fmaf(e, low * 0.693147181f, e);
    } else {
        e = __builtin_amdgcn_exp2f(-fabsf(z) * kLog2e);
    }
    const float near = __builtin_amdgcn_rcpf(1.0f + e), far = e * near;
    return z < 0.0f ? Gate{far, near, far} : Gate{near, far, -far};
}

// The map s -> A·s + b of a run of tokens; 1 - A is kept beside A.
struct Map {
    float a, off, b;
    __device__ __forceinline__ void then(const Gate &g) {
        a = apply(g.by, a);
        off = __builtin_fmaf(g.rest, 1.0f - off, off);
    }
    __device__ __forceinline__ void then_by(float by) {
        a = apply(by, a);
        off = __builtin_signbit(by) ? __builtin_fmaf(-by, 1.0f - off, off) : __builtin_fmaf(-by, 1.0f - off, 1.0f);
    }
    __device__ __forceinline__ float by() const { return off <= 0.5f ? -off : a; }
};

// The maps of parts: [batch][parts][A as it is applied, b][channels].  The place whose map nobody
// needs has the state that comes in as its b.
struct PartMaps {
    float *maps;
    uint32_t parts, span; // tokens of a part
    uint64_t channels;
    __device__ __forceinline__ float *at(uint64_t batch, uint32_t part, uint32_t which) const {
        return maps + ((batch * parts + part) * 2 + which) * channels;
    }
};

// The waves' maps of a tile, in the order in which they follow each other; two
// tiles in turn, so that one barrier a tile is enough.
template <int V, int WAVES> struct TileMaps {
    float by[2][WAVES][V][kWave], b[2][WAVES][V][kWave];
};
// From this wave's map and the state that comes into the tile: the state that comes
// into the wave, and that after the tile.
template <int V, int WAVES>
__device__ __forceinline__ void join_tile(TileMaps<V, WAVES> &m, uint32_t turn, int wave, const Map (&map)[V],
                                          float (&carry)[V], float (&mine)[V]) {
    if constexpr (WAVES == 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            mine[v] = carry[v];
            carry[v] = apply_infinite(map[v].by(), carry[v]) + map[v].b;
        }
    } else {
        const int lane = lane_id();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            m.by[turn][wave][v][lane] = map[v].by();
            m.b[turn][wave][v][lane] = map[v].b;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (w == wave) mine[v] = carry[v];
                carry[v] = apply(m.by[turn][w][v][lane], carry[v]) + m.b[turn][w][v][lane];
            }
    }
}

__device__ __forceinline__ uint64_t length_of(const uint32_t *lengths, uint64_t batch, uint64_t tokens) {
    return lengths ? min((uint64_t)lengths[batch], tokens) : tokens;
}
template <int V> __device__ __forceinline__ void state_at(const float *p, uint64_t c, float (&s)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = p ? p[c + v] : 0.0f;
}
template <int V> __device__ __forceinline__ void put_state(float *p, uint64_t c, const float (&s)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) p[c + v] = s[v];
}

// ----------------------------------------------------------------- forward
// MAPS: the map of each part but the last, and the first state; else the outputs.
template <typename T, int V, int WAVES, int R, bool MAPS>
__global__ __launch_bounds__(WAVES *kWave) void recurrence_kernel(RecurrenceArgs a, PartMaps p) {
    using L = Lane<T, V>;
    __shared__ TileMaps<V, WAVES> maps;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t groups = (uint32_t)((a.channels + kWave * V - 1) / (kWave * V));
    const uint32_t part = blockIdx.x / groups;
    const uint64_t batch = blockIdx.y;
    const uint64_t own = ((uint64_t)(blockIdx.x % groups) * kWave + lane_id()) * V;
    const bool is_there = own < a.channels; // lanes past the end repeat the last ones and store nothing
    const uint64_t c = is_there ? own : a.channels - V;
    const uint64_t n = length_of(a.lengths, batch, a.tokens);
    const uint64_t first = (uint64_t)part * p.span, last = min(a.tokens, first + p.span), end = min(n, last);
    const T *gate = (const T *)a.gate + (int64_t)batch * a.s_gate.batch + c;
    const T *x = (const T *)a.x + (int64_t)batch * a.s_x.batch + c;
    T *out = (T *)a.out + (int64_t)batch * a.s_out.batch + c;
    const float *state = a.state_in ? a.state_in + (int64_t)batch * a.s_state_in : nullptr;

    float carry[V];
    Map total[V]; // of the tiles so far; its b is the carry
#pragma unroll
    for (int v = 0; v < V; ++v) total[v] = Map{1.0f, 0.0f, 0.0f};
    if constexpr (MAPS) {
        if (part == p.parts - 1) {
            state_at(state, c, carry);
            if (wave == 0 && is_there) put_state(p.at(batch, part, 1), c, carry);
            return;
        }
        state_at<V>(nullptr, 0, carry);
    } else if (p.parts > 1) {
        state_at(p.at(batch, p.parts - 1, 1), c, carry);
#pragma unroll 8
        for (uint32_t i = 0; i < part; ++i) {
            float by[V], b[V];
            state_at(p.at(batch, i, 0), c, by);
            state_at(p.at(batch, i, 1), c, b);
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = apply(by[v], carry[v]) + b[v];
        }
    } else {
        state_at(state, c, carry);
    }

    struct Tile {
        typename L::Raw z[R], x[R];
    } now, next;
    const auto fetch = [&](uint64_t t0, Tile &t) {
#pragma unroll
        for (int r = 0; r < R; ++r) { // tokens past the end repeat the last one
            const int64_t token = (int64_t)min(t0 + wave * R + r, end - 1);
            t.z[r] = L::load(gate + token * a.s_gate.token);
            t.x[r] = L::load(x + token * a.s_x.token);
        }
    };
    if (first < end) fetch(first, now);
    uint32_t turn = 0;
    for (uint64_t t0 = first; t0 < end; t0 += WAVES * R, turn ^= 1) {
        if (t0 + WAVES * R < end) fetch(t0 + WAVES * R, next);
        float h[R][V], kept[R][V];
        Map map[V];
#pragma unroll
        for (int v = 0; v < V; ++v) map[v] = Map{1.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool is_token = t0 + wave * R + r < end;
            float z[V], u[V];
            L::values(now.z[r], z);
            L::values(now.x[r], u);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (is_token) {
                    const Gate g = gate_of<T>(z[v]);
                    map[v].b = __builtin_fmaf(g.rest, u[v], apply(g.by, map[v].b));
                    map[v].then(g);
                }
                h[r][v] = map[v].b;
                kept[r][v] = map[v].a;
            }
        }
        float mine[V];
        join_tile<V, WAVES>(maps, turn, wave, map, carry, mine);
        if constexpr (MAPS) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int v = 0; v < V; ++v) total[v].then_by(maps.by[turn][w][v][lane_id()]);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint64_t t = t0 + wave * R + r;
#pragma unroll
                for (int v = 0; v < V; ++v) h[r][v] += kept[r][v] * mine[v];
                if (t < end && is_there) L::store(out + (int64_t)t * a.s_out.token, h[r]);
            }
        }
        now = next;
    }
    if constexpr (MAPS) {
        if (wave == 0 && is_there) {
            float by[V];
#pragma unroll
            for (int v = 0; v < V; ++v) by[v] = total[v].by();
            put_state(p.at(batch, part, 0), c, by);
            put_state(p.at(batch, part, 1), c, carry);
        }
    } else {
        // Rows past a sequence's end.
        const float zeros[V] = {};
        for (uint64_t t = max(first, n) + wave; t < last; t += WAVES)
            if (is_there) L::store(out + (int64_t)t * a.s_out.token, zeros);
        const uint32_t ending = n ? (uint32_t)((n - 1) / p.span) : 0;
        if (a.state_out && part == ending && wave == 0 && is_there)
            put_state(a.state_out + (int64_t)batch * a.s_state_out, c, carry);
    }
}

// ---------------------------------------------------------------- backward
// Tiles and parts from the last token on.  MAPS: the map of each part but the
// first, and the gradient of the last state.
template <typename T, int V, int WAVES, int R, bool MAPS>
__global__ __launch_bounds__(WAVES *kWave) void recurrence_grad_kernel(RecurrenceGradArgs a, PartMaps p) {
    using L = Lane<T, V>;
    __shared__ TileMaps<V, WAVES> maps;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t groups = (uint32_t)((a.channels + kWave * V - 1) / (kWave * V));
    const uint32_t part = blockIdx.x / groups;
    const uint64_t batch = blockIdx.y;
    const uint64_t own = ((uint64_t)(blockIdx.x % groups) * kWave + lane_id()) * V;
    const bool is_there = own < a.channels;
    const uint64_t c = is_there ? own : a.channels - V;
    const uint64_t n = length_of(a.lengths, batch, a.tokens);
    const uint64_t first = (uint64_t)part * p.span, last = min(a.tokens, first + p.span), end = min(n, last);
    const T *gate = (const T *)a.gate + (int64_t)batch * a.s_gate.batch + c;
    const T *x = (const T *)a.x + (int64_t)batch * a.s_x.batch + c;
    const T *h = (const T *)a.h + (int64_t)batch * a.s_h.batch + c;
    const T *dy = (const T *)a.grad_out + (int64_t)batch * a.s_grad_out.batch + c;
    T *dz = (T *)a.grad_gate + (int64_t)batch * a.s_grad_gate.batch + c;
    T *dx = (T *)a.grad_x + (int64_t)batch * a.s_grad_x.batch + c;
    const float *after = a.grad_state_out ? a.grad_state_out + (int64_t)batch * a.s_grad_state_out : nullptr;

    float carry[V], before[V]; // before: the state in front of the first token
    Map total[V];              // of the tiles so far; its b is the carry
#pragma unroll
    for (int v = 0; v < V; ++v) total[v] = Map{1.0f, 0.0f, 0.0f};
    if constexpr (MAPS) {
        if (part == 0) {
            state_at(after, c, carry);
            if (wave == 0 && is_there) put_state(p.at(batch, 0, 1), c, carry);
            return;
        }
        state_at<V>(nullptr, 0, carry);
    } else {
        state_at(a.state_in ? a.state_in + (int64_t)batch * a.s_state_in : nullptr, c, before);
        if (p.parts > 1) {
            state_at(p.at(batch, 0, 1), c, carry);
#pragma unroll 8
            for (uint32_t i = p.parts - 1; i > part; --i) {
                float by[V], b[V];
                state_at(p.at(batch, i, 0), c, by);
                state_at(p.at(batch, i, 1), c, b);
#pragma unroll
                for (int v = 0; v < V; ++v) carry[v] = apply(by[v], carry[v]) + b[v];
            }
        } else {
            state_at(after, c, carry);
        }
    }

    struct Tile {
        typename L::Raw z[R], y[R], x[MAPS ? 1 : R], h[MAPS ? 1 : R];
    } now, next;
    // Token r of this wave in the tile that ends before `hi`; below `first` there is none.
    const auto token_of = [&](uint64_t hi, int r) { return (int64_t)hi - 1 - (wave * R + r); };
    const auto fetch = [&](uint64_t hi, Tile &t) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t token = max(token_of(hi, r), (int64_t)first);
            t.z[r] = L::load(gate + token * a.s_gate.token);
            t.y[r] = L::load(dy + token * a.s_grad_out.token);
            if constexpr (!MAPS) {
                t.x[r] = L::load(x + token * a.s_x.token);
                t.h[r] = L::load(h + max(token - 1, (int64_t)0) * a.s_h.token);
            }
        }
    };
    if (first < end) fetch(end, now);
    uint32_t turn = 0;
    for (int64_t hi = (int64_t)end; hi > (int64_t)first; hi -= WAVES * R, turn ^= 1) {
        if (hi - WAVES * R > (int64_t)first) fetch(hi - WAVES * R, next);
        float g[R][V], kept[R][V];
        Gate gates[R][V];
        Map map[V];
#pragma unroll
        for (int v = 0; v < V; ++v) map[v] = Map{1.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool is_token = token_of(hi, r) >= (int64_t)first;
            float z[V], y[V];
            L::values(now.z[r], z);
            L::values(now.y[r], y);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gates[r][v] = gate_of<T>(z[v]);
                g[r][v] = y[v] + map[v].b;
                kept[r][v] = map[v].a;
                if (is_token) {
                    map[v].b = apply(gates[r][v].by, g[r][v]);
                    map[v].then(gates[r][v]);
                }
            }
        }
        float mine[V];
        join_tile<V, WAVES>(maps, turn, wave, map, carry, mine);
        if constexpr (MAPS) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int v = 0; v < V; ++v) total[v].then_by(maps.by[turn][w][v][lane_id()]);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t t = token_of(hi, r);
                float u[V], prev[V], gz[V], gx[V];
                L::values(now.x[r], u);
                L::values(now.h[r], prev);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    gx[v] = gates[r][v].rest * (g[r][v] + kept[r][v] * mine[v]);
                    gz[v] = gates[r][v].f * gx[v] * ((t == 0 ? before[v] : prev[v]) - u[v]);
                }
                if (t >= (int64_t)first && is_there) {
                    L::store(dz + t * a.s_grad_gate.token, gz);
                    L::store(dx + t * a.s_grad_x.token, gx);
                }
            }
        }
        now = next;
    }
    if constexpr (MAPS) {
        if (wave == 0 && is_there) {
            float by[V];
#pragma unroll
            for (int v = 0; v < V; ++v) by[v] = total[v].by();
            put_state(p.at(batch, part, 0), c, by);
            put_state(p.at(batch, part, 1), c, carry);
        }
    } else {
        const float zeros[V] = {};
        for (uint64_t t = max(first, n) + wave; t < last; t += WAVES)
            if (is_there) {
                L::store(dz + (int64_t)t * a.s_grad_gate.token, zeros);
                L::store(dx + (int64_t)t * a.s_grad_x.token, zeros);
            }
        if (a.grad_state_in && part == 0 && wave == 0 && is_there)
            put_state(a.grad_state_in + (int64_t)batch * a.s_grad_state_in, c, carry);
    }
}

// `count` channels from `first` on.
template <typename T> void shift(const void *&p, uint64_t first) { p = (const T *)p + first; }
template <typename T> void shift(void *&p, uint64_t first) { p = (T *)p + first; }
inline void shift_state(const float *&p, uint64_t first) { p = p ? p + first : nullptr; }
inline void shift_state(float *&p, uint64_t first) { p = p ? p + first : nullptr; }
template <typename T> RecurrenceArgs channels_from(RecurrenceArgs a, uint64_t first, uint64_t count) {
    shift<T>(a.gate, first), shift<T>(a.x, first), shift<T>(a.out, first);
    shift_state(a.state_in, first), shift_state(a.state_out, first);
    a.channels = count;
    return a;
}
template <typename T> RecurrenceGradArgs channels_from(RecurrenceGradArgs a, uint64_t first, uint64_t count) {
    shift<T>(a.gate, first), shift<T>(a.x, first), shift<T>(a.h, first), shift<T>(a.grad_out, first);
    shift<T>(a.grad_gate, first), shift<T>(a.grad_x, first);
    shift_state(a.state_in, first), shift_state(a.grad_state_out, first), shift_state(a.grad_state_in, first);
    a.channels = count;
    return a;
}

template <typename T, int V, typename Args>
hx_status launch_channels(const Args &a, const RecurrenceParts &cut, void *ws, hipStream_t stream) {
    constexpr bool kGrad = std::is_same<Args, RecurrenceGradArgs>::value;
    const PartMaps p{(float *)ws, cut.parts, cut.span, a.channels};
    const dim3 grid((uint32_t)(ceil_div(a.channels, kWave * V) * cut.parts), (uint32_t)a.batch);
    const auto run = [&](auto kernel, uint32_t waves) {
        hipLaunchKernelGGL(kernel, grid, dim3(waves * kWave), 0, stream, a, p);
        return check_launch("recurrence_kernel");
    };
    if constexpr (kGrad) {
        switch (cut.tile) {
        case RecurrenceTile::kOne: return run(recurrence_grad_kernel<T, V, 1, 1, false>, 1);
        case RecurrenceTile::kFew: return run(recurrence_grad_kernel<T, V, 1, 8, false>, 1);
        default:
            if (cut.parts > 1) HX_TRY(run(recurrence_grad_kernel<T, V, 8, 8, true>, 8));
            return run(recurrence_grad_kernel<T, V, 8, 8, false>, 8);
        }
    } else {
        switch (cut.tile) {
        case RecurrenceTile::kOne: return run(recurrence_kernel<T, V, 1, 1, false>, 1);
        case RecurrenceTile::kFew: return run(recurrence_kernel<T, V, 1, 8, false>, 1);
        case RecurrenceTile::kMany:
            if (cut.parts > 1) HX_TRY(run(recurrence_kernel<T, V, 8, 8, true>, 8));
            return run(recurrence_kernel<T, V, 8, 8, false>, 8);
        case RecurrenceTile::kLong: return run(recurrence_kernel<T, V, 8, 16, false>, 8);
        }
    }
    return HX_OK;
}

template <typename T, int V, typename Args> hx_status launch(const Args &a, void *ws, hipStream_t stream) {
    // Blocks of 512 threads, fewer than 2^32 of these in a launch: more channels take
    // several, and far fewer are ever cut into parts.
    constexpr uint64_t kMost = (uint64_t)kWave * V << 22;
    const RecurrenceParts cut = recurrence_parts(a, V, std::is_same<Args, RecurrenceGradArgs>::value);
    for (uint64_t first = 0; first < a.channels; first += kMost)
        HX_TRY((launch_channels<T, V>(channels_from<T>(a, first, std::min(kMost, a.channels - first)), cut, ws, stream)));
    return HX_OK;
}

template <typename Args> hx_status launch_any(const Args &a, void *ws, hipStream_t stream) {
    if (a.batch == 0 || a.channels == 0) return HX_OK;
    if (a.dtype == HX_DTYPE_F32) return launch<float, 1>(a, ws, stream);
    if (recurrence_on_dwords(a)) return launch<bf16, 2>(a, ws, stream);
    return launch<bf16, 1>(a, ws, stream);
}
template <typename Args> uint64_t maps_bytes(const Args &a) {
    if (a.batch == 0 || a.channels == 0) return 0;
    const RecurrenceParts cut = recurrence_parts(a, recurrence_on_dwords(a) && a.dtype != HX_DTYPE_F32 ? 2 : 1,
                                                 std::is_same<Args, RecurrenceGradArgs>::value);
    return cut.parts > 1 ? a.batch * cut.parts * 2 * a.channels * sizeof(float) : 0;
}

} // namespace

uint64_t gated_recurrence_workspace_bytes(const RecurrenceArgs &args) { return maps_bytes(args); }
hx_status launch_gated_recurrence(const RecurrenceArgs &args, void *ws, hipStream_t stream) {
    return launch_any(args, ws, stream);
}
uint64_t gated_recurrence_grad_workspace_bytes(const RecurrenceGradArgs &args) { return maps_bytes(args); }
hx_status launch_gated_recurrence_grad(const RecurrenceGradArgs &args, void *ws, hipStream_t stream) {
    return launch_any(args, ws, stream);
}

} // namespace hx
