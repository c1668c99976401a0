// hx_i8.hip — products of activations and weights in 8 bits, a scale to every row of each.
#include <cmath>

#include "hx_common.h"
#include "hx_i8_rule.h"
#include "hx_wave.h"

namespace hx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A piece holds 16 rows by 64 columns of the weights in the order in which a wave's lanes hold the matrix instruction's operand:
// lane l has row l % 16, columns 16 (l / 16)..+15. A wave's load of one is 1024 bytes in a row.
constexpr int kPieceRows = 16, kPieceCols = 64, kPiece = kPieceRows * kPieceCols;
__host__ __device__ inline int64_t pieces_of(int64_t K) { return (K + kPieceCols - 1) / kPieceCols; }

struct I8Args {
    int64_t M, N, K, ldx, ldy;
    const int8_t *X, *W;
    const float *sx, *sw, *bias;
    void* Y;
    int act;
};

// 16 bytes of a row of X of which `left` are there, zeros behind them
__device__ inline i32x4 load_x(const int8_t* at, int64_t left) {
    i32x4 v = {0, 0, 0, 0};
    if (left >= 16) {
        __builtin_memcpy(&v, at, 16);
    } else if (left > 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < left) v[e / 4] |= (int)((uint32_t)(uint8_t)at[e] << (8 * (e % 4)));
    }
    return v;
}

// What becomes of a sum: exact in 32 bits up to here, one conversion and one product with both scales.
struct Finish {
    float sw, bias;
    __device__ static Finish of(const I8Args& p, int64_t n) {
        const bool in = n < p.N;
        return {in ? p.sw[n] : 0.0f, in && p.bias ? p.bias[n] : 0.0f};
    }
    __device__ float operator()(const I8Args& p, int acc, float sx) const {
        float v = (float)acc * (sx * sw);
        if (p.bias) v += bias;
        return p.act & 1 ? silu(v) : v;
    }
};

// E outputs of a row at `to`, `left` of them inside it
template <int E, typename TO>
__device__ inline void store_outputs(const I8Args& p, TO* to, int64_t left, float (&v)[E]) {
    if (left >= E) {
        if (p.act & 2) {
            const Run<E, TO> old = Run<E, TO>::load(to);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += Storage<TO>::load(&old.v[e]);
        }
        uint32_t w[E * sizeof(TO) / 4];
#pragma unroll
        for (int e = 0; e < (int)(E * sizeof(TO) / 4); ++e) {
            if constexpr (sizeof(TO) == 4)
                w[e] = __float_as_uint(v[e]);
            else
                w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
        }
        if constexpr (sizeof(w) == 16) {  // outputs stream out past what the other tiles still read
            typedef uint32_t anywhere __attribute__((ext_vector_type(4), aligned(2)));
            anywhere v4;
            __builtin_memcpy(&v4, w, 16);
            __builtin_nontemporal_store(v4, (anywhere*)to);
        } else {
            __builtin_memcpy(to, w, sizeof(w));
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < left) {
                if (p.act & 2) v[e] += Storage<TO>::load(to + e);
                Storage<TO>::store(to + e, v[e]);
            }
    }
}

// ------------------------------------------------------------------ few rows
// A block takes 16 NT outputs of 16 MT rows of X, its waves a run of K each, in windows of 256 columns. Pieces of weights come
// straight into the matrix instruction's registers, a window ahead. X comes by memory, 16 lanes to a row's 256 bytes, since
// lanes that each sit in a row of their own cost the L1 a look-up apiece (64 a load), and goes through LDS rows that a wave
// keeps to itself. Sums are whole numbers: the waves' are added in any order to the same bits. Bound by the latency of one round of loads
// and of the joining (1 x 8192 x 2048 4.5 us, 3.7 TB/s of weights) and by X, which every block reads whole (48 x 2048 x 8192 8.5 us).
constexpr int kWindow = 256, kWindowPieces = kWindow / kPieceCols, kXRow = kWindow + 16;

template <int NT, int MT, typename TO>
__global__ __launch_bounds__(512) void linear_i8_rows_kernel(const I8Args p, const int windows, const int per, const int waves) {
    extern __shared__ __align__(16) char lds[];
    constexpr int XR = 4 * MT;  // rows of X that a lane loads from
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, u = lane >> 4;
    const int64_t tiles = (p.N + 15) / 16, t0 = (int64_t)blockIdx.x * NT, m0 = (int64_t)blockIdx.y * (16 * MT), pieces = pieces_of(p.K);
    char* const mine = lds + wave * (16 * MT * kXRow);
    const int8_t* w[NT];
#pragma unroll
    for (int a = 0; a < NT; ++a) w[a] = p.W + (t0 + a < tiles ? t0 + a : tiles - 1) * pieces * kPiece + lane * 16;
    // rows behind the last read the last one; what they give is not stored
    const int8_t* x[XR];
#pragma unroll
    for (int i = 0; i < XR; ++i) x[i] = p.X + (m0 + 4 * i + u < p.M ? m0 + 4 * i + u : p.M - 1) * p.ldx + 16 * r;
    i32x4 acc[NT][MT];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) acc[a][b] = i32x4{0, 0, 0, 0};

    const int first = wave * per, end = first + per < windows ? first + per : windows;
    const int whole = (int)(p.K / kWindow) < end ? (int)(p.K / kWindow) : end;  // windows that lie inside K
    const auto load_rows = [&](int at, i32x4 (&o)[XR]) {
#pragma unroll
        for (int i = 0; i < XR; ++i) __builtin_memcpy(&o[i], x[i] + (int64_t)at * kWindow, 16);
    };
    const auto load_weights = [&](int at, i32x4 (&o)[NT][kWindowPieces]) {
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int k = 0; k < kWindowPieces; ++k) o[a][k] = *reinterpret_cast<const i32x4*>(w[a] + ((int64_t)at * kWindowPieces + k) * kPiece);
    };
    // Lanes read what other lanes of the wave wrote: the compiler cannot tell which (the offset is hidden from it), so that it
    // keeps the accesses in order, and a wave's LDS accesses complete in order.
    const char* from = mine;
    {
        int off = r * kXRow + 16 * u;
        asm("" : "+v"(off));
        from += off;
    }
    const auto stage = [&](const i32x4 (&xs)[XR]) {
#pragma unroll
        for (int i = 0; i < XR; ++i) *reinterpret_cast<i32x4*>(mine + (4 * i + u) * kXRow + 16 * r) = xs[i];
    };
    const auto multiply = [&](const i32x4 (&ws)[NT][kWindowPieces]) {
#pragma unroll
        for (int k = 0; k < kWindowPieces; ++k)
#pragma unroll
            for (int b = 0; b < MT; ++b) {
                const i32x4 xv = *reinterpret_cast<const i32x4*>(from + 16 * b * kXRow + 64 * k);
#pragma unroll
                for (int a = 0; a < NT; ++a) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ws[a][k], xv, acc[a][b], 0, 0, 0);
            }
    };
    i32x4 xs[XR], ws[2][NT][kWindowPieces];
    int at = first;
    if (at < whole) {
        load_weights(at, ws[0]);
        load_rows(at, xs);
        for (; at + 2 <= whole; at += 2) {
            load_weights(at + 1, ws[1]);
            stage(xs);
            load_rows(at + 1, xs);
            multiply(ws[0]);
            const int next = at + 2 < whole ? at + 2 : at;  // the last ones are asked for twice
            load_weights(next, ws[0]);
            stage(xs);
            load_rows(next, xs);
            multiply(ws[1]);
        }
        if (at < whole) {
            stage(xs);
            multiply(ws[0]);
            ++at;
        }
    }
    if (at < end) {  // the window that K ends in
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int k = 0; k < kWindowPieces; ++k) {
                const int64_t piece = (int64_t)at * kWindowPieces + k;
                ws[0][a][k] = piece < pieces ? *reinterpret_cast<const i32x4*>(w[a] + piece * kPiece) : i32x4{0, 0, 0, 0};
            }
#pragma unroll
        for (int i = 0; i < XR; ++i) xs[i] = load_x(x[i] + (int64_t)at * kWindow, p.K - (int64_t)at * kWindow - 16 * r);
        stage(xs);
        multiply(ws[0]);
    }
    __syncthreads();
    // lane (m = r, outputs 4u..4u + 3) of a tile
    int* const sums = (int*)lds;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) *reinterpret_cast<i32x4*>(sums + ((wave * MT + b) * 16 + r) * (16 * NT + 4) + 16 * a + 4 * u) = acc[a][b];
    __syncthreads();
    constexpr int Q = 4 * NT;  // runs of four outputs a row
    for (int o = threadIdx.x; o < 16 * MT * Q; o += blockDim.x) {
        const int row = o / Q, n = o % Q * 4;
        if (m0 + row >= p.M || t0 * 16 + n >= p.N) continue;
        i32x4 s = *reinterpret_cast<const i32x4*>(sums + row * (16 * NT + 4) + n);
        for (int k = 1; k < waves; ++k) s += *reinterpret_cast<const i32x4*>(sums + (k * 16 * MT + row) * (16 * NT + 4) + n);
        const float sx = p.sx[m0 + row];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = Finish::of(p, t0 * 16 + n + e)(p, s[e], sx);
        store_outputs<4>(p, (TO*)p.Y + (m0 + row) * p.ldy + t0 * 16 + n, p.N - t0 * 16 - n, v);
    }
}

// ------------------------------------------------------------------ many rows
// A block's tile is 64 TM rows by 64 TN outputs, four waves in 2 x 2, each TM x TN tiles of 32 x 32. K tiles of 128 columns move
// straight into a two-stage LDS ring: rows of X as 128 bytes with their 16-byte chunks exchanged by row (chunk c of row r
// in place c ^ (r & 7)), so that a fragment's 32 rows meet all banks, pieces of weights as they lie in memory, which is the
// order they are read in. The next fragments are read and a later tile's loads issued between the matrix instructions; the barrier
// of a K tile stands before its last quarter, whose fragments are in registers by then. 8191 x 8192 x 2048 to bf16 with SiLU: 167-183 us, 1.5
// to 1.65 POP/s of the 2.1 that a large library product reaches; a K of 2048 leaves a sixth of the time to first loads and outputs. Needs rows of X that start at
// 16 bytes; columns behind the last whole K tile come straight from memory. Rows behind M and N are the last ones', and not stored.
typedef int i32x16 __attribute__((ext_vector_type(16)));
constexpr int kTileCols = 128;
constexpr int kRsrcWord3 = 0x00020000;  // a raw buffer of 32-bit data without swizzle

template <int TM, int TN, typename TO>
__global__ __launch_bounds__(256) void linear_i8_tiles_kernel(const I8Args p, const int nbx, const int nb) {
    constexpr int BM = 64 * TM, BN = 64 * TN, kA = BM * kTileCols, kStage = (BM + BN) * kTileCols;
    constexpr int kEach = kStage / 1024 / 4;  // loads of 1 KiB a wave issues for a K tile
    constexpr int F = TM + TN;                // fragments of a quarter
    static_assert(TM == TN && TM * TN % F == 0, "waves 0 and 1 load X, 2 and 3 weights");
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, fr = lane & 31, half = lane >> 5;
    // consecutive blocks go to different dies, each with an L2 of its own: a die takes a run of tiles, and walks it in groups of
    // four rows of tiles, so that those in flight share rows of X and columns of weights
    int64_t id = blockIdx.x;
    if (nb % 8 == 0) id = (id % 8) * (nb / 8) + id / 8;
    const int64_t group = id / (4 * nbx), rest = id % (4 * nbx), nby = nb / nbx;
    const int64_t high = nby - 4 * group < 4 ? nby - 4 * group : 4;
    const int64_t m0 = (4 * group + rest % high) * BM, n0 = rest / high * BN;
    const int64_t pieces = pieces_of(p.K), tiles = (p.N + 15) / 16;

    const bool is_x = wave < 2;
    const int8_t* const base = is_x ? p.X + m0 * p.ldx : p.W + n0 / 16 * pieces * kPiece;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)0x7fffffff, kRsrcWord3);
    uint32_t from[16];  // kEach of them (a bound that depends on the template here drops the launch stub on the host)
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int q = (wave & 1) * kEach + j;
        if (is_x) {
            const int row = 8 * q + lane / 8;
            from[j] = (uint32_t)((m0 + row < p.M ? row : p.M - 1 - m0) * p.ldx) + 16 * ((lane % 8) ^ (row & 7));
        } else {
            const int64_t tile = n0 / 16 + q / 2 < tiles ? q / 2 : tiles - 1 - n0 / 16;
            from[j] = (uint32_t)((tile * pieces + q % 2) * kPiece) + lane * 16;
        }
    }
    const auto load = [&](int j, int kt, int stage) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lvoid_t*)(lds + stage * kStage + (wave * kEach + j) * 1024), 16, from[j],
                                                 is_x ? kt * kTileCols : kt * 2 * kPiece, 0, 0);
    };
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // fragment q of quarter s: TM of X, then TN of weights
    const auto frag = [&](int stage, int s, int q) __attribute__((always_inline)) {
        const char* at = lds + stage * kStage;
        return q < TM ? *reinterpret_cast<const i32x4*>(at + (wm * 32 * TM + 32 * q + fr) * kTileCols + (((2 * s + half) ^ (fr & 7)) << 4))
                      : *reinterpret_cast<const i32x4*>(at + kA + ((wn * TN + q - TM) * 2 + fr / 16) * 2 * kPiece + s / 2 * kPiece +
                                                        (2 * (s % 2) + half) * 256 + fr % 16 * 16);
    };
    const int nk = (int)(p.K / kTileCols);
    if (nk > 0) {
        i32x4 f[2][F];
#pragma unroll
        for (int j = 0; j < kEach; ++j) load(j, 0, 0);
        if (nk > 1) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) load(j, 1, 1);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kEach) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll
        for (int q = 0; q < F; ++q) f[0][q] = frag(0, 0, q);
        for (int kt = 0; kt < nk; ++kt) {
            const int stage = kt & 1;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int cur = s & 1, nxt = cur ^ 1;
                // the loads of tile kt + 2 go out over this tile's last quarter and the next one's first
                const int tl = s == 3 ? kt + 2 : kt + 1;
                const bool issue = s == 3 ? tl < nk : s == 0 && kt >= 1 && tl < nk;
                const int j0 = s == 3 ? 0 : kEach / 2;
                if (s == 3 && kt + 1 < nk) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
                for (int q = 0; q < F; ++q) {
#pragma unroll
                    for (int t = q * TM * TN / F; t < (q + 1) * TM * TN / F; ++t)
                        acc[t / TN][t % TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[cur][t / TN], f[cur][TM + t % TN], acc[t / TN][t % TN], 0, 0, 0);
                    // (the last tile's last quarter reads fragments of a stage that no load fills any more, and does not use them)
                    f[nxt][q] = s < 3 ? frag(stage, s + 1, q) : frag(stage ^ 1, 0, q);
                    if (issue) {
#pragma unroll
                        for (int j = q * (kEach / 2) / F; j < (q + 1) * (kEach / 2) / F; ++j) load(j0 + j, tl, tl & 1);
                    }
                }
#pragma unroll
                for (int q = 0; q < F; ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x008, TM * TN / F, 0);  // matrix instructions
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);            // an LDS read
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);            // a load
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    // columns behind the whole K tiles: codes of weights behind K are zero
    for (int64_t k = (int64_t)nk * 2; k < pieces; ++k) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x4 a[TM], b[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int64_t m = m0 + wm * 32 * TM + 32 * i + fr, c = k * kPieceCols + 32 * s + 16 * half;
                a[i] = load_x(p.X + (m < p.M ? m : p.M - 1) * p.ldx + c, p.K - c);
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int64_t t = n0 / 16 + (wn * TN + j) * 2 + fr / 16;
                b[j] = *reinterpret_cast<const i32x4*>(p.W + ((t < tiles ? t : tiles - 1) * pieces + k) * kPiece + (2 * s + half) * 256 + fr % 16 * 16);
            }
#pragma unroll
            for (int t = 0; t < TM * TN; ++t)
                acc[t / TN][t % TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[t / TN], b[t % TN], acc[t / TN][t % TN], 0, 0, 0);
        }
    }
    // Slabs of 32 rows by 64 outputs through LDS rows of the wave's own, and out as rows. The scales are all asked for ahead: with
    // few waves to a SIMD a load between slabs is waited for in full (256 wide, 8191 x 8192 x 2048: 193 -> 175 us).
    constexpr int E = 16 / sizeof(TO), kLanes = 64 / E, kRows = 64 / kLanes;  // elements a lane, lanes a row, rows at a time
    int* const st = (int*)lds + wave * (32 * 68);
    const int c = lane % kLanes * E;
    float sx[TM][32 / kRows];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int h = 0; h < 32 / kRows; ++h) {
            const int64_t m = m0 + wm * 32 * TM + 32 * i + h * kRows + lane / kLanes;
            sx[i][h] = p.sx[m < p.M ? m : p.M - 1];
        }
    Finish fin[TN / 2][E];
#pragma unroll
    for (int jj = 0; jj < TN / 2; ++jj)
#pragma unroll
        for (int e = 0; e < E; ++e) fin[jj][e] = Finish::of(p, n0 + wn * 32 * TN + 64 * jj + c + e);
    __syncthreads();  // the ring's memory is free
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int jj = 0; jj < TN / 2; ++jj) {
            const int64_t n = n0 + wn * 32 * TN + 64 * jj + c;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) st[(8 * (e >> 2) + 4 * half + (e & 3)) * 68 + 32 * j + fr] = acc[i][2 * jj + j][e];
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
            for (int h = 0; h < 32 / kRows; ++h) {
                const int row = h * kRows + lane / kLanes;
                const int64_t m = m0 + wm * 32 * TM + 32 * i + row;
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = fin[jj][e](p, st[row * 68 + c + e], sx[i][h]);
                if (m < p.M && n < p.N) store_outputs<E>(p, (TO*)p.Y + m * p.ldy + n, p.N - n, v);
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        }
    }
}

template <int NT, int MT, typename TO>
int launch_rows(const I8Args& p, hipStream_t s) {
    // waves to a tile of outputs, each with two windows at least: enough of them to fill the chip, no more than share a block's LDS
    const int windows = (int)((p.K + kWindow - 1) / kWindow);
    const int64_t blocks = (p.N + 16 * NT - 1) / (16 * NT), groups = (p.M + 16 * MT - 1) / (16 * MT);
    int waves = 1;
    while (waves < 8 && windows >= 4 * waves && blocks * groups * waves < 4096) waves *= 2;
    constexpr size_t staged = 16 * MT * kXRow, summed = 16 * MT * (16 * NT + 4) * sizeof(int);
    const size_t bytes = waves * (staged > summed ? staged : summed);
    const auto k = linear_i8_rows_kernel<NT, MT, TO>;
    HX_REQUIRE(bytes <= 65536 || grant_dynamic_lds((const void*)k, bytes, 0), HX_ERR_BACKEND, "linear_i8: %zu bytes of LDS not granted", bytes);
    hipLaunchKernelGGL(k, dim3((unsigned)blocks, (unsigned)groups), dim3(64 * waves), bytes, s, p, windows, (windows + waves - 1) / waves, waves);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

template <int T, typename TO>
int launch_tiles(const I8Args& p, hipStream_t s) {
    constexpr size_t bytes = 2 * 128 * T * kTileCols;
    const auto k = linear_i8_tiles_kernel<T, T, TO>;
    HX_REQUIRE(bytes <= 65536 || grant_dynamic_lds((const void*)k, bytes, 0), HX_ERR_BACKEND, "linear_i8: %zu bytes of LDS not granted", bytes);
    const int64_t nbx = (p.N + 64 * T - 1) / (64 * T), nby = (p.M + 64 * T - 1) / (64 * T);
    hipLaunchKernelGGL(k, dim3((unsigned)(nbx * nby)), dim3(256), bytes, s, p, (int)nbx, (int)(nbx * nby));
    HX_LAUNCH_CHECK();
    return HX_OK;
}

template <typename TO>
int launch_i8(const I8Args& p, hipStream_t s) {
    switch (i8_kernel(p.M, p.N, p.K, aligned(p.X, 16) && p.ldx % 16 == 0 && p.ldx < (1 << 22))) {
        case I8Kernel::kTiles256: return launch_tiles<4, TO>(p, s);
        case I8Kernel::kTiles128: return launch_tiles<2, TO>(p, s);
        case I8Kernel::kRows64x32: return launch_rows<2, 4, TO>(p, s);
        case I8Kernel::kRows32x32: return launch_rows<2, 2, TO>(p, s);
        default: return launch_rows<1, 1, TO>(p, s);
    }
}

}  // namespace
}  // namespace hx

extern "C" int hx_i8_quantize(int64_t N, int64_t K, const float* w, void* packed, float* scales) {
    using namespace hx;
    HX_REQUIRE(N >= 0 && K >= 0, HX_ERR_INVALID_DIMENSION, "i8_quantize: negative size");
    if (N == 0) return HX_OK;
    HX_REQUIRE(scales && (K == 0 || (w && packed)), HX_ERR_INVALID_INPUT, "i8_quantize: NULL pointer");
    const int64_t pieces = pieces_of(K);
    memset(packed, 0, (size_t)((N + kPieceRows - 1) / kPieceRows * pieces * kPiece));
    for (int64_t n = 0; n < N; ++n) {
        const float* v = w + n * K;
        float top = 0.0f;
        bool finite = true;
        for (int64_t k = 0; k < K; ++k) {
            finite = finite && std::isfinite(v[k]);
            top = std::fmax(top, std::fabs(v[k]));
        }
        HX_REQUIRE(finite, HX_ERR_INVALID_INPUT, "i8_quantize: row %lld holds a value that is not finite", (long long)n);
        scales[n] = (float)((double)top / 127.0);
        int8_t* to = (int8_t*)packed + n / kPieceRows * pieces * kPiece + n % kPieceRows * 16;
        for (int64_t k = 0; top > 0.0f && k < K; ++k)
            to[k / kPieceCols * kPiece + k % kPieceCols / 16 * 256 + k % 16] = (int8_t)std::nearbyint((double)v[k] * 127.0 / (double)top);
    }
    return HX_OK;
}

extern "C" int hx_linear_i8(int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const float* x_scales, const void* packed,
                            const float* scales, const float* bias, int act, int out_dtype, void* Y, int64_t ldy, void* stream) {
    using namespace hx;
    HX_REQUIRE(M >= 0 && N >= 0 && K >= 0, HX_ERR_INVALID_DIMENSION, "linear_i8: negative size");
    HX_REQUIRE(out_dtype == HX_F32 || out_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "linear_i8: out_dtype %d", out_dtype);
    HX_REQUIRE(act >= 0 && act <= 3, HX_ERR_INVALID_INPUT, "linear_i8: act %d", act);
    if (M == 0 || N == 0) return HX_OK;
    HX_REQUIRE(Y && x_scales && scales && ldy >= N && (K == 0 || (X && packed && ldx >= K)), HX_ERR_INVALID_INPUT,
               "linear_i8: X, x_scales, packed, scales and Y required, ldx >= K, ldy >= N");
    HX_REQUIRE(aligned(packed, 16), HX_ERR_INVALID_INPUT, "linear_i8: packed must be 16-byte aligned");
    HX_REQUIRE(K < (1 << 17) && M <= 64 * (int64_t)65535 && N < (1 << 26), HX_ERR_UNSUPPORTED,
               "linear_i8: K below 2^17 (sums in 32 bits), at most %d rows of X, N below 2^26", 64 * 65535);
    const I8Args p{M, N, K, ldx, ldy, (const int8_t*)X, (const int8_t*)packed, x_scales, scales, bias, Y, act};
    return out_dtype == HX_F32 ? launch_i8<float>(p, as_stream(stream)) : launch_i8<uint16_t>(p, as_stream(stream));
}
