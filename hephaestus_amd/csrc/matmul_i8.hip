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
//   waves of a block take slices of k and add their sums in LDS.  The reading of
//   b bounds it: 1 x 4096 x 4096 takes 4.8 us, 3.5 TB/s with the launch; 4097 bytes
//   of k, rows at any byte, 6.1.
// * Tiles: rows of 128 bytes of a and b go through LDS buffers in turn.  The
//   matrix instructions bound large products, 8192 x 8192 x 8192 in 481 us, 2.29
//   PetaOP/s; the reading of b bounds a few tokens more than a skinny one takes,
//   64 x 8192 x 8192 in 15.5 us, 4.4 TB/s.
#include "hx_internal.hpp"
#include "layer_device.hpp"

#include <atomic>
#include <type_traits>

namespace hx {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kDepth = kMatmulDepth;

__device__ __forceinline__ i32x4v mma(i32x4v b, i32x4v a, i32x4v sum) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a, sum, 0, 0, 0);
}

// 16 bytes of a row from `k` on, zeros from `end` on.  Global memory takes
// vectors at any byte address.  The last bytes of a row come as the sixteen that
// end it: read one by one they cost a wait each.
__device__ __forceinline__ i32x4v load_bytes(const int8_t *row, uint32_t k, uint32_t end) {
    if (k + 16 <= end) return __builtin_bit_cast(i32x4v, (u32x4)*(const u32x4_any *)(row + k));
    i32x4v v = {0, 0, 0, 0};
    if (k >= end) return v;
    if (end >= 16) {
        const u32x4 last = *(const u32x4_any *)(row + end - 16);
        return __builtin_bit_cast(i32x4v, __builtin_bit_cast(unsigned __int128, last) >> (8 * (k + 16 - end)));
    }
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

// 16 bytes of a row at any address, from the dwords that hold them, which are
// shifted when they are used: vectors off dwords load at half the rate (7 x 8192 x
// 8192 27.5 us, 16.4 so).  The dword after the first sixteen bytes is read only where
// some of the row's lie in it.
struct AnyBytes {
    u32x4 v;
    uint32_t next;
};
__device__ __forceinline__ AnyBytes load_dwords(const int8_t *p) {
    const int8_t *down = p - ((uintptr_t)p & 3);
    return {*(const u32x4_a4 *)down, *(const uint32_t *)(down + ((uintptr_t)p & 3 ? 16 : 12))};
}
__device__ __forceinline__ i32x4v shift_bytes(const AnyBytes &b, uint32_t by) {
    return i32x4v{(int)__builtin_amdgcn_alignbyte(b.v[1], b.v[0], by), (int)__builtin_amdgcn_alignbyte(b.v[2], b.v[1], by),
                  (int)__builtin_amdgcn_alignbyte(b.v[3], b.v[2], by), (int)__builtin_amdgcn_alignbyte(b.next, b.v[3], by)};
}

// ------------------------------------------------------------------ skinny
// Up to 16·MF tokens; a block takes 16·NF channels, each of its eight waves every
// eighth 128 bytes of k.
constexpr int kSkinnyWaves = 8;

template <typename T, int MF, int NF, bool DWORDS>
__global__ __launch_bounds__(kSkinnyWaves *kWave) void matmul_skinny_kernel(MatmulArgs p) {
    __shared__ int sums[MF * NF * 4 * kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    static_assert(MF * NF <= kSkinnyWaves); // a wave stores one of the fragments
    const uint64_t n0 = (uint64_t)blockIdx.x * (16 * NF);
    const uint32_t k_end = (uint32_t)p.k, at = lane / 16 * 16;
    for (int i = threadIdx.x; i < MF * NF * 4 * kWave; i += kSkinnyWaves * kWave) sums[i] = 0;
    uint32_t a_end[MF]; // rows that are not there are zeros
    const int8_t *a[MF], *b[NF];
#pragma unroll
    for (int f = 0; f < MF; ++f) {
        const uint64_t m = 16 * f + lane % 16;
        a_end[f] = m < p.m ? k_end : 0;
        a[f] = p.a + (int64_t)(m < p.m ? m : 0) * p.a_stride;
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) // channels past the end are summed and dropped
        b[j] = p.b + (int64_t)min(n0 + 16 * j + lane % 16, p.n - 1) * p.b_stride;
    i32x4v acc[MF][NF] = {};
    const uint32_t whole = k_end / kDepth * kDepth;
    constexpr uint32_t kTurn = kSkinnyWaves * kDepth;
    // The next turn's bytes are on their way while this turn is summed.
    using Bytes = typename std::conditional<DWORDS, u32x4, AnyBytes>::type;
    struct Turn {
        Bytes b[NF][2], a[MF][2];
    } now, next;
    const auto load = [](const int8_t *p) {
        if constexpr (DWORDS) return (u32x4)*(const u32x4_a4 *)p;
        else return load_dwords(p);
    };
    const auto whole_of = [](const Bytes &v, const int8_t *row) { // rows of one address modulo 4 throughout
        if constexpr (DWORDS) return __builtin_bit_cast(i32x4v, v);
        else return shift_bytes(v, (uint32_t)(uintptr_t)row & 3);
    };
    const auto fetch = [&](uint32_t k, Turn &t) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int j = 0; j < NF; ++j) t.b[j][s] = load(b[j] + k + 64 * s + at);
#pragma unroll
            for (int f = 0; f < MF; ++f) {
                t.a[f][s] = Bytes{};
                if (a_end[f]) t.a[f][s] = load(a[f] + k + 64 * s + at);
            }
        }
    };
    // Blocks begin at different turns: rows a power of two apart lie on the
    // same memory channels, and blocks in step would all ask the same ones
    // (1 x 4096 x 4096: 7.1 us in step, 5.4 us so).
    const uint32_t first = wave * kDepth, turns = whole > first ? (whole - first + kTurn - 1) / kTurn : 0;
    uint32_t t = turns ? blockIdx.x / 8 % turns : 0;
    if (turns) fetch(first + t * kTurn, now);
    for (uint32_t left = turns; left; --left) {
        t = t + 1 < turns ? t + 1 : 0;
        if (left > 1) fetch(first + t * kTurn, next);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x4v fb[NF];
#pragma unroll
            for (int j = 0; j < NF; ++j) fb[j] = whole_of(now.b[j][s], b[j]);
#pragma unroll
            for (int f = 0; f < MF; ++f) {
                const i32x4v fa = whole_of(now.a[f][s], a[f]);
#pragma unroll
                for (int j = 0; j < NF; ++j) acc[f][j] = mma(fb[j], fa, acc[f][j]);
            }
        }
        now = next;
    }
    // The last, partial 128 bytes: to the wave whose turn it is.
    if (whole < k_end && wave == (int)(whole / kDepth % kSkinnyWaves)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t k = whole + 64 * s + at;
            i32x4v fa[MF], fb[NF];
#pragma unroll
            for (int f = 0; f < MF; ++f) fa[f] = load_bytes(a[f], k, a_end[f]);
#pragma unroll
            for (int j = 0; j < NF; ++j) fb[j] = load_bytes(b[j], k, k_end);
#pragma unroll
            for (int f = 0; f < MF; ++f)
#pragma unroll
                for (int j = 0; j < NF; ++j) acc[f][j] = mma(fb[j], fa[f], acc[f][j]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) atomicAdd(&sums[((f * NF + j) * 4 + e) * kWave + lane], acc[f][j][e]);
    __syncthreads();
    if (wave >= MF * NF) return;
    const uint64_t m = 16 * (wave / NF) + lane % 16;
    if (m >= p.m) return;
    i32x4v s;
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = sums[(wave * 4 + e) * kWave + lane];
    store_scaled((T *)p.out + (int64_t)m * p.out_stride, n0 + 16 * (wave % NF) + lane / 16 * 4, p.n, s, p.a_scales[m],
                 p.b_scales);
}

template <typename T, int MF, bool DWORDS> hx_status launch_skinny(const MatmulArgs &p, hipStream_t stream) {
    const auto run = [&](auto kernel, uint64_t channels) {
        hipLaunchKernelGGL(kernel, dim3((uint32_t)ceil_div(p.n, channels)), dim3(kSkinnyWaves * kWave), 0, stream, p);
    };
    if (skinny_is_wide(p.n)) run(matmul_skinny_kernel<T, MF, 2, DWORDS>, 32);
    else run(matmul_skinny_kernel<T, MF, 1, DWORDS>, 16);
    return check_launch("matmul_skinny_kernel");
}

// ------------------------------------------------------------------- tiles
// BM tokens by BN channels a block.  Its WM x WN waves each take a part of the
// tile; with KG > 1 there are KG such groups, which take the steps of k in turn
// and add their sums in LDS.  A step's 128 bytes of k of each row lie in LDS as
// eight chunks of 16, chunk c of row r at place c ^ (r % 8), so that the 16 rows
// that a matrix instruction reads at one c fall on all banks.
//
// Loads go from memory to LDS without registers, S - 1 steps ahead: each
// wave's 64 chunks of an instruction land side by side, and the exchange of
// places is made on the global side.  They need rows that begin on dwords;
// others are copied to such rows first.
//
// The barrier between steps is written out: all of the wave's LDS reads and
// writes and all but its last N loads have ended when it is passed.
// __syncthreads would wait for every load.
template <int N> __device__ __forceinline__ void step_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <int BM, int BN, int WM, int WN, int KG, int S> struct Tile {
    static constexpr int kWaves = WM * WN, kThreads = kWaves * KG * kWave;
    static constexpr int kRows = BM + BN, kStage = kRows * kDepth, kLds = kStage * S * KG;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    static constexpr int kLoads = kRows * 8 / (kWaves * kWave); // chunks a thread and step
    static_assert(kLds <= 160 * 1024 && kLoads * 8 * kWaves == kRows && (S - 2) * kLoads < 64);
    static_assert(KG == 1 || BM * BN * 4 <= kLds);
};

template <typename T, int BM, int BN, int WM, int WN, int KG, int S>
__global__ __launch_bounds__(WM *WN *KG *kWave, 2) void matmul_tiles_kernel(MatmulArgs p, uint32_t tiles_m,
                                                                        uint32_t tiles_n) {
    using C = Tile<BM, BN, WM, WN, KG, S>;
    constexpr int FM = C::FM, FN = C::FN, kLoads = C::kLoads;
    extern __shared__ __align__(16) int8_t lds[];
    const int lane = lane_id(), block_wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wave = block_wave % C::kWaves, group = block_wave / C::kWaves;
    int8_t *stages = lds + group * (S * C::kStage);

    // Blocks go to the eight XCDs in turn: each XCD takes a run of tiles, in
    // strips of eight tiles of m so that its L2 serves both operands.
    const uint32_t total = tiles_m * tiles_n, share = total / 8, rest = total % 8;
    const uint32_t xcd = blockIdx.x % 8, turn = blockIdx.x / 8;
    const uint32_t tile = xcd * share + min(xcd, rest) + turn;
    const uint32_t strip = tile / (8 * tiles_n), in_strip = tile % (8 * tiles_n);
    const uint32_t height = min(8u, tiles_m - 8 * strip);
    const uint64_t m0 = (uint64_t)(8 * strip + in_strip % height) * BM, n0 = (uint64_t)(in_strip / height) * BN;

    const uint32_t k_end = (uint32_t)p.k, steps = (k_end + kDepth - 1) / kDepth, whole = k_end / kDepth;
    const uint32_t turns = (steps + KG - 1) / KG; // this group's step of turn t: t·KG + group
    // A thread's chunk of each row that it loads: rows past the operands
    // repeat the last one and are dropped at the end.
    const uint32_t row0 = wave * (kLoads * 8) + lane / 8, place = lane % 8, chunk = (place ^ (row0 % 8)) * 16;
    const int8_t *src[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const uint32_t r = row0 + j * 8;
        src[j] = r < BM ? p.a + (int64_t)min(m0 + r, p.m - 1) * p.a_stride
                        : p.b + (int64_t)min(n0 + (r - BM), p.n - 1) * p.b_stride;
    }
    const uint32_t to = wave * (kLoads * 1024); // this wave's first row in a stage

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

    // Whole steps: no branch in the loads.
    const auto fetch = [&](uint32_t t) {
        int8_t *stage = stages + t % S * C::kStage + to;
        const uint32_t k = (t * KG + group) * kDepth + chunk;
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            __builtin_amdgcn_global_load_lds((const void *)(src[j] + k), (lds_void *)(stage + j * 1024), 16, 0, 0);
    };
    // The step of the last, partial 128 bytes: zeros past the end of k.
    const auto fetch_rest = [&](uint32_t t) {
        int8_t *stage = stages + t % S * C::kStage + to;
        for (int j = 0; j < kLoads; ++j)
            *(i32x4v *)(stage + j * 1024 + lane * 16) = load_bytes(src[j], whole * kDepth + chunk, k_end);
    };
    const auto fetch_any = [&](uint32_t t) {
        const uint32_t q = t * KG + group;
        if (q < whole) fetch(t);
        else if (q < steps) fetch_rest(t);
    };
    for (int t = 0; t < S - 1; ++t) fetch_any(t);
    // Step t has landed once no more loads are under way than those of the
    // S - 2 steps behind it.
    const uint32_t mine = whole > (uint32_t)group ? (whole - group + KG - 1) / KG : 0; // whole steps of this group
    uint32_t t = 0;
    for (; t + (S - 1) < mine; ++t) {
        step_barrier<(S - 2) * kLoads>();
        fetch(t + S - 1);
        compute(stages + t % S * C::kStage);
    }
    for (; t < turns; ++t) { // the last ones, not all of them direct loads
        step_barrier<0>();
        if (t + S - 1 < turns) fetch_any(t + S - 1);
        if (t * KG + group < steps) compute(stages + t % S * C::kStage);
    }

    const uint32_t token = wm + lane % 16, channel = wn + lane / 16 * 4; // of the tile, and 16·i, 16·j on
    if constexpr (KG > 1) {
        int *sums = (int *)lds;
        __syncthreads();
        for (int i = threadIdx.x; i < BM * BN; i += C::kThreads) sums[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    atomicAdd(&sums[((wave * FM * FN + i * FN + j) * 4 + e) * kWave + lane], acc[i][j][e]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if ((i * FN + j) % KG != group) continue; // the groups share the fragments
                const uint64_t m = m0 + token + 16 * i;
                if (m >= p.m) continue;
                i32x4v v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = sums[((wave * FM * FN + i * FN + j) * 4 + e) * kWave + lane];
                store_scaled((T *)p.out + (int64_t)m * p.out_stride, n0 + channel + 16 * j, p.n, v, p.a_scales[m],
                             p.b_scales);
            }
    } else {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const uint64_t m = m0 + token + 16 * i;
            if (m >= p.m) continue;
            const float sa = p.a_scales[m];
            T *row = (T *)p.out + (int64_t)m * p.out_stride;
#pragma unroll
            for (int j = 0; j < FN; ++j) store_scaled(row, n0 + channel + 16 * j, p.n, acc[i][j], sa, p.b_scales);
        }
    }
}

template <typename T, int BM, int BN, int WM, int WN, int KG, int S>
hx_status launch_tiles(const MatmulArgs &p, hipStream_t stream) {
    using C = Tile<BM, BN, WM, WN, KG, S>;
    const auto kernel = matmul_tiles_kernel<T, BM, BN, WM, WN, KG, S>;
    static std::atomic<uint64_t> allowed{0};
    HX_TRY(allow_lds((const void *)kernel, C::kLds, allowed));
    const uint64_t tm = ceil_div(p.m, BM), tn = ceil_div(p.n, BN);
    if (tm * tn * C::kThreads > 0xFFFFFFFFull)
        return fail(HX_ERR_DISPATCH_FAILED, "matmul of %llu tiles exceeds the grid range", (unsigned long long)(tm * tn));
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(tm * tn)), dim3(C::kThreads), C::kLds, stream, p, (uint32_t)tm,
                       (uint32_t)tn);
    return check_launch("matmul_tiles_kernel");
}

template <typename T> hx_status launch_tiled(const MatmulArgs &p, hipStream_t stream) {
    switch (matmul_tile(p.m, p.n, p.k)) {
    case MatmulTile::k256x256: return launch_tiles<T, 256, 256, 2, 4, 1, 2>(p, stream);
    case MatmulTile::k128x128Pairs: return launch_tiles<T, 128, 128, 2, 2, 1, 2>(p, stream);
    case MatmulTile::k128x128: return launch_tiles<T, 128, 128, 2, 4, 1, 4>(p, stream);
    case MatmulTile::k96x96: return launch_tiles<T, 96, 96, 2, 2, 2, 3>(p, stream);
    case MatmulTile::k64x64Groups: return launch_tiles<T, 64, 64, 2, 2, 3, 3>(p, stream);
    case MatmulTile::k64x64: return launch_tiles<T, 64, 64, 4, 2, 1, 4>(p, stream);
    case MatmulTile::k64x32Pairs: return launch_tiles<T, 64, 32, 2, 1, 3, 2>(p, stream);
    case MatmulTile::k64x32: return launch_tiles<T, 64, 32, 2, 1, 6, 2>(p, stream);
    case MatmulTile::k32x32Pairs: return launch_tiles<T, 32, 32, 1, 2, 4, 2>(p, stream);
    case MatmulTile::k32x32: return launch_tiles<T, 32, 32, 1, 2, 8, 2>(p, stream);
    case MatmulTile::k32x16: return launch_tiles<T, 32, 16, 1, 1, 8, 3>(p, stream);
    }
    return fail(HX_ERR_DISPATCH_FAILED, "no tile for a matmul of %llu x %llu", (unsigned long long)p.m,
                (unsigned long long)p.n);
}

// ----------------------------------------------------------- rows on dwords
// Rows of a and b at any byte, copied to rows of whole 128 bytes with zeros
// after their ends, sixteen bytes a thread, the rows end to end.  Loading such rows
// through registers in every tile took 29 us for 1000 x 1027 x 4099; the copy and
// then direct loads take 19.7.
__global__ __launch_bounds__(256) void matmul_align_kernel(MatmulArgs p, int8_t *rows, uint32_t pitch) {
    const uint32_t chunks = pitch / 16; // of a row
    for (uint64_t first = (uint64_t)blockIdx.x * 256; first < (p.m + p.n) * chunks; first += (uint64_t)gridDim.x * 256) {
        const uint32_t i = (uint32_t)(first % chunks) + threadIdx.x, at = i % chunks * 16;
        const uint64_t r = first / chunks + i / chunks;
        if (r >= p.m + p.n) return;
        const int8_t *from = r < p.m ? p.a + (int64_t)r * p.a_stride : p.b + (int64_t)(r - p.m) * p.b_stride;
        *(i32x4v *)(rows + r * pitch + at) = load_bytes(from, at, (uint32_t)p.k);
    }
}

// A launch has fewer than 2^32 threads: 16 a channel for a few tokens, up to 12 a
// channel or 2 a token in tiles.  More channels or tokens take several launches.
constexpr uint64_t kMostRows = 1ull << 27;
template <typename T, typename F> hx_status in_parts(const MatmulArgs &p, F run) {
    for (uint64_t m = 0; m < p.m; m += kMostRows)
        for (uint64_t n = 0; n < p.n; n += kMostRows) {
            MatmulArgs part = p;
            part.m = min(p.m - m, kMostRows);
            part.n = min(p.n - n, kMostRows);
            part.a += (int64_t)m * p.a_stride;
            part.b += (int64_t)n * p.b_stride;
            part.a_scales += m;
            part.b_scales += n;
            part.out = (T *)p.out + (int64_t)m * p.out_stride + (int64_t)n;
            HX_TRY(run(part));
        }
    return HX_OK;
}

template <typename T> hx_status launch(MatmulArgs p, void *ws, hipStream_t stream) {
    if (matmul_is_skinny(p))
        return in_parts<T>(p, [&](const MatmulArgs &part) {
            if (!matmul_off_dwords(p)) return launch_skinny<T, 1, true>(part, stream);
            if (p.m <= 16) return launch_skinny<T, 1, false>(part, stream);
            return launch_skinny<T, 2, false>(part, stream);
        });
    if (matmul_needs_copy(p)) {
        const uint32_t pitch = (uint32_t)matmul_copy_pitch(p);
        const uint64_t blocks = min(ceil_div((p.m + p.n) * (pitch / 16), 256), (uint64_t)1 << 22);
        hipLaunchKernelGGL(matmul_align_kernel, dim3((uint32_t)blocks), dim3(256), 0, stream, p, (int8_t *)ws, pitch);
        HX_TRY(check_launch("matmul_align_kernel"));
        p.a = (const int8_t *)ws;
        p.b = p.a + p.m * pitch;
        p.a_stride = p.b_stride = pitch;
        p.k = pitch;
    }
    return in_parts<T>(p, [&](const MatmulArgs &part) { return launch_tiled<T>(part, stream); });
}

} // namespace

uint64_t matmul_i8_workspace_bytes(const MatmulArgs &args) {
    return args.m && args.n && matmul_needs_copy(args) ? (args.m + args.n) * matmul_copy_pitch(args) : 0;
}

hx_status launch_matmul_i8(const MatmulArgs &args, void *ws, hipStream_t stream) {
    if (args.m == 0 || args.n == 0) return HX_OK;
    return args.dtype == HX_DTYPE_F32 ? launch<float>(args, ws, stream) : launch<bf16>(args, ws, stream);
}

} // namespace hx
