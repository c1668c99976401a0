// hx_w4.hip — 4-bit weights with group scales (OCP MXFP4): rounding on the host, products on the device.
#include <cmath>

#include "hx_common.h"
#include "hx_wave.h"

namespace hx {
namespace {

constexpr int kGroup = HX_W4_GROUP;

// Bytes of a packed row and of a row of scales: whole groups, and whole 16-byte loads of scales.
__host__ __device__ inline int64_t groups_of(int64_t K) { return (K + kGroup - 1) / kGroup; }
__host__ __device__ inline int64_t packed_row(int64_t K) { return groups_of(K) * (kGroup / 2); }
__host__ __device__ inline int64_t scales_row(int64_t K) { return (groups_of(K) + 15) / 16 * 16; }

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWindow = 128;  // elements of K that one 16-byte load per lane covers for 16 rows
constexpr int kAhead = 4;     // windows whose scales one load covers, and whose weights are in flight at once
constexpr int kRowsAtOnce = 32;  // rows of X that one block takes at most
constexpr int kXRow = 2 * kWindow + 16;  // bytes from one staged row of X to the next

struct W4Args {
    int64_t M, N, K, ldx, ldy;
    const uint16_t* X;
    const uint8_t *W, *S;
    const float* bias;
    void* Y;
    int act, windows, per, waves;  // windows of K, how many a wave takes, the waves of a block
};

// Eight codes of a group at its scale as bf16: exact (one significant bit and a power of two), two codes an instruction.
__device__ inline bf16x8 expand8(uint32_t q, float scale) {
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
    union {
        bf16x2 p[4];
        bf16x8 v;
    } u;
    u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
    u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
    u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
    u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
    return u.v;
}

// A block takes 16 NT outputs of at most 4 XR rows of X, its waves a run of windows each. What a wave loads is laid out by
// memory, since the L1 looks up one line a clock and lanes that each sit in a row of their own cost 64 looks a load (47 us
// instead of 34.5 at 5 x 32768 x 8192, whatever the loads in flight), and brought to the matrix instruction's order:
//   weights  lane 4n + j holds row n's group j of a window, 32 codes in 16 bytes. A lane permutation gives (n, j) its
//            place 16j + n, four register swaps turn (lane j, word i) into (lane i, word j), after which instruction i
//            of four takes group i, eight codes a lane under one scale (with the scale inside the expanded weights the
//            groups need no sums of their own);
//   X        16 lanes read a row's 256 bytes of the window and leave them in the wave's own LDS rows, 16 bytes apart
//            from a power of two, so that 16 rows read at one place of theirs meet all banks.
// Rows of X start anywhere: global memory takes 16-byte accesses at any element.
// The next weights are asked for once the registers that take them are read, and no address is kept, which leaves room for two
// blocks of 8 waves to a CU (four waves a SIMD): 1 x 32768 x 8192 33.1 -> 29.7 us, 1 x 8950 x 7360 15.2 -> 12.3. With 32 rows
// of X, or four tiles, they do not hold it (220 bytes spilled): two waves.
template <int NT, int XR, typename TO>
__global__ __launch_bounds__(512, XR > 4 || NT > 2 ? 2 : 4) void linear_w4_kernel(const W4Args p) {
    constexpr int MT = XR < 4 ? 1 : XR / 4, kRows = 4 * XR;  // column tiles of 16, rows of X that are staged
    extern __shared__ float lds[];  // first the waves' rows of X, then [waves][NT][MT][16 m][16 n] sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, j = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * kRows;
    const int64_t G = groups_of(p.K), pr = packed_row(p.K), sr = scales_row(p.K);
    // Rows behind the last read the last one; what they give is not stored. A lane's part of an address is a 32-bit offset
    // from a uniform place.
    const uint8_t *const wb = p.W + n0 * pr, *const sb = p.S + n0 * sr;
    uint32_t w[NT], s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t row = 16 * t + lane / 4, inside = n0 + row < p.N ? row : p.N - 1 - n0;
        w[t] = (uint32_t)(inside * pr) + 16 * (lane % 4);
        s[t] = (uint32_t)(inside * sr);
    }
    const int place = (4 * r + j) * 4;  // the lane that loaded (r, j), in bytes
    char* const xrow = (char*)lds + wave * (kRows * kXRow);
    const int64_t rows = p.M - m0 < kRows ? p.M - m0 : kRows;
    const int rows_in = (int)rows;
    const char* const xb = (const char*)(p.X + m0 * p.ldx);
    uint32_t x[XR];
#pragma unroll
    for (int t = 0; t < XR; ++t) x[t] = (uint32_t)((4 * t + j < rows_in ? 4 * t + j : rows_in - 1) * p.ldx * 2) + 16 * r;
    // Lanes read what other lanes of the wave wrote, which one lane's own addresses do not show. These are hidden from the
    // compiler, so that each may be any that was written, and no read passes a write or a write a read. (Fences of the wave
    // around the writes hold back the loads from global memory as well: 1 x 32768 x 8192 33.4 us against 29.7.)
    const char* xread[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        int from = (16 * t + r < rows_in ? 16 * t + r : rows_in - 1) * kXRow + 16 * j;
        asm("" : "+v"(from));
        xread[t] = xrow + from;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) acc[a][b] = f32x4{0, 0, 0, 0};
    uint32_t top[NT] = {};  // the largest scale byte of each row: 255 is not a number

    // Kept 32 bits wide up to the load, which adds it to a scalar base by itself; 64-bit sums would stay in registers.
    const auto offset = [](uint32_t v) {
        asm("" : "+v"(v));
        return v;
    };
    const auto load_x = [&](int at, u32x4 (&o)[XR]) {
        const char* from = xb + (int64_t)at * (2 * kWindow);
#pragma unroll
        for (int t = 0; t < XR; ++t) __builtin_memcpy(&o[t], from + offset(x[t]), 16);
    };
    // A wave's own rows, and its LDS accesses keep their order: no barrier, and the registers are free for the next window.
    // The compiler keeps it too: it cannot tell what a lane reads (xread) from what it wrote.
    const auto stage = [&](const u32x4 (&xs)[XR]) {
#pragma unroll
        for (int t = 0; t < XR; ++t) *reinterpret_cast<u32x4*>(xrow + (4 * t + j) * kXRow + 16 * r) = xs[t];
    };
    // The window that K ends in: elements from K on are zero. The eight that hold K are loaded ending at K and moved up, so
    // that nothing behind a row is touched; rows of fewer than eight go one by one.
    const auto load_x_end = [&](int at, u32x4 (&o)[XR]) {
        const int left = (int)(p.K - (int64_t)at * kWindow) - 8 * r;
        const int back = left >= 8 ? 0 : 8 - left;
        const char* from = xb + (int64_t)at * (2 * kWindow);
#pragma unroll
        for (int t = 0; t < XR; ++t) {
            unsigned __int128 v = 0;
            if (left > 0) {
                if (p.K >= 8) {
                    __builtin_memcpy(&v, from + x[t] - 2 * back, 16);
                    v >>= 16 * back;
                } else {
                    for (int e = 0; e < left; ++e) v |= (unsigned __int128)*(const uint16_t*)(from + x[t] + 2 * e) << (16 * e);
                }
            }
            __builtin_memcpy(&o[t], &v, 16);
        }
    };
    const auto load_w = [&](int at, bool in, u32x4 (&o)[NT]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
            o[t] = in ? *reinterpret_cast<const u32x4*>(wb + (int64_t)at * (kWindow / 2) + offset(w[t])) : u32x4{0, 0, 0, 0};
    };
    // lane 4n + u: the four scale bytes of row n's window at + u
    const int last = (int)(sr / 4) - 1;
    const auto load_s = [&](int at, uint32_t (&o)[NT]) {
        const int word = at + lane % 4 < last ? at + lane % 4 : last;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] = *reinterpret_cast<const uint32_t*>(sb + (s[t] + word * 4));
    };
    const auto whole_groups = [](auto&) {};
    const auto multiply = [&](u32x4 (&q)[NT], const uint32_t (&sc)[NT], int u, int groups_in, const auto& cut, const auto& refill) {
        const auto moved = [&](uint32_t v) { return __int_as_float(__builtin_amdgcn_ds_bpermute(place, (int)v)); };
        float c[NT][4];
        uint32_t scales[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            c[a][0] = moved(q[a].x);
            c[a][1] = moved(q[a].y);
            c[a][2] = moved(q[a].z);
            c[a][3] = moved(q[a].w);
            swap32(c[a][0], c[a][2]);
            swap32(c[a][1], c[a][3]);
            swap16(c[a][0], c[a][1]);
            swap16(c[a][2], c[a][3]);
            scales[a] = (uint32_t)__builtin_amdgcn_ds_bpermute((4 * r + u) * 4, (int)sc[a]);
            if (groups_in < 4) {  // groups that are not there have no weights and a scale of one
                const uint32_t kept = 0xffffffffu >> (8 * (4 - groups_in));
                scales[a] = (scales[a] & kept) | (0x7f7f7f7fu & ~kept);
            }
        }
        refill(q);
        cut(c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 xv[MT];
#pragma unroll
            for (int b = 0; b < MT; ++b) xv[b] = *reinterpret_cast<const bf16x8*>(xread[b] + 64 * i);
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const uint32_t scale = scales[a] >> (8 * i) & 255;
                top[a] = scale > top[a] ? scale : top[a];
                const bf16x8 wv = expand8(__float_as_uint(c[a][i]), __uint_as_float(scale << 23));
#pragma unroll
                for (int b = 0; b < MT; ++b)
                    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[b], acc[a][b], 0, 0, 0);
            }
        }
    };

    int at = wave * p.per;
    const int end = at + p.per < p.windows ? at + p.per : p.windows;
    const int whole = (int)(p.K / kWindow) < end ? (int)(p.K / kWindow) : end;
    if (at + kAhead <= whole) {
        // a ring of R windows of weights: the one that was multiplied makes room for the one R later. X comes one window
        // ahead, asked for before the weights that follow it: loads return in order.
        constexpr int R = NT > 2 ? kAhead / 2 : kAhead;  // four tiles' registers
        u32x4 q[R][NT], xs[XR];
        uint32_t sc[NT];
        load_s(at, sc);
#pragma unroll
        for (int u = 0; u < R; ++u) load_w(at + u, true, q[u]);
        load_x(at, xs);
        for (; at + 2 * kAhead <= whole; at += kAhead) {
            uint32_t after[NT];
            load_s(at + kAhead, after);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                stage(xs);
                load_x(at + u + 1, xs);
                multiply(q[u % R], sc, u, 4, whole_groups, [&](u32x4 (&o)[NT]) { load_w(at + u + R, true, o); });
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) sc[t] = after[t];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            stage(xs);
            if (u + 1 < kAhead) load_x(at + u + 1, xs);
            multiply(q[u % R], sc, u, 4, whole_groups, [&](u32x4 (&o)[NT]) {
                if (u + R < kAhead) load_w(at + u + R, true, o);
            });
        }
        at += kAhead;
    }
    if (at < end) {  // at most kAhead windows, the last of K perhaps not whole
        u32x4 q[kAhead][NT];
        uint32_t sc[NT];
        load_s(at, sc);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (at + u < end) load_w(at + u, (at + u) * 4 + lane % 4 < G, q[u]);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (at + u >= end) break;
            const int left = (int)(G - (int64_t)(at + u) * 4);
            u32x4 xs[XR];
            if (at + u < whole)
                load_x(at + u, xs);
            else
                load_x_end(at + u, xs);
            stage(xs);
            // K's last group, in its place in the matrix instruction: lane (r, j) holds its codes 8j..8j + 7. Those from K on
            // are zero, whatever the rows hold there, since X's zeros do not cancel an infinity (scale bytes 253 and 254).
            // Cleared in the loaded words instead, registers cost 1 x 8950 x 7360 11.9 -> 13.4 us.
            const auto cut = [&](float (&c)[NT][4]) {
                const int codes = (int)(p.K % kGroup), n = codes - 8 * j;
                if (codes == 0) return;
                const uint32_t kept = n <= 0 ? 0u : n >= 8 ? 0xffffffffu : (1u << (4 * n)) - 1u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t m = i == left - 1 ? kept : 0xffffffffu;
#pragma unroll
                    for (int a = 0; a < NT; ++a) c[a][i] = __uint_as_float(__float_as_uint(c[a][i]) & m);
                }
            };
            multiply(q[u], sc, u, left < 4 ? left : 4, cut, [](auto&) {});
        }
    }
    // a scale that is not a number makes its whole row one: NaN * 0 added to it
#pragma unroll
    for (int a = 0; a < NT; ++a)
        if (__any(top[a] == 255)) {
            const uint32_t bits = top[a] == 255 ? 0x7fc07fc0u : 0u;
            const bf16x8 wv = __builtin_bit_cast(bf16x8, make_uint4(bits, bits, bits, bits));
            const bf16x8 zero = __builtin_bit_cast(bf16x8, make_uint4(0, 0, 0, 0));
#pragma unroll
            for (int b = 0; b < MT; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, zero, acc[a][b], 0, 0, 0);
        }

    __syncthreads();
    // The waves' sums in the order of K, then the epilogue; lane (m = r, 4j..4j+3) holds four outputs of a row of X.
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b)
            *reinterpret_cast<f32x4*>(lds + ((wave * NT + a) * MT + b) * 256 + r * 16 + 4 * j) = acc[a][b];
    __syncthreads();
    TO* y = (TO*)p.Y;
    for (int o = threadIdx.x; o < NT * MT * 256; o += blockDim.x) {
        const int a = o / 16 % NT, row = o / (16 * NT);  // consecutive threads take consecutive outputs
        const int64_t n = n0 + 16 * a + o % 16, m = m0 + row;
        if (n >= p.N || m >= p.M) continue;
        const float* at_o = lds + (a * MT + row / 16) * 256 + row % 16 * 16 + o % 16;
        float v = 0.0f;
        for (int k = 0; k < p.waves; ++k) v += at_o[k * NT * MT * 256];
        if (p.bias) v += p.bias[n];
        if (p.act & 1) v = silu(v);
        TO* to = y + m * p.ldy + n;
        if (p.act & 2) v += Storage<TO>::load(to);
        Storage<TO>::store(to, v);
    }
}

template <int NT, int XR>
int launch_w4(const W4Args& p, bool f32, hipStream_t s) {
    const dim3 grid((unsigned)((p.N + 16 * NT - 1) / (16 * NT)), (unsigned)((p.M + 4 * XR - 1) / (4 * XR)));
    const auto k = f32 ? linear_w4_kernel<NT, XR, float> : linear_w4_kernel<NT, XR, uint16_t>;
    constexpr size_t staged = 4 * XR * kXRow, summed = NT * (XR < 4 ? 1 : XR / 4) * 256 * sizeof(float);
    const size_t bytes = p.waves * (staged > summed ? staged : summed);
    if (bytes > 65536 && !grant_dynamic_lds((const void*)k, bytes, 0)) {
        if constexpr (XR > 4) return launch_w4<NT, XR / 2>(p, f32, s);  // the same sums, X's rows in two blocks
    }
    hipLaunchKernelGGL(k, grid, dim3((unsigned)(64 * p.waves)), bytes, s, p);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

}  // namespace
}  // namespace hx

extern "C" int hx_w4_quantize(int64_t N, int64_t K, const float* w, void* packed, void* scales) {
    using namespace hx;
    HX_REQUIRE(N >= 0 && K >= 0, HX_ERR_INVALID_DIMENSION, "w4_quantize: negative size");
    if (N == 0 || K == 0) return HX_OK;
    HX_REQUIRE(w && packed && scales, HX_ERR_INVALID_INPUT, "w4_quantize: NULL pointer");
    const int64_t G = groups_of(K);
    for (int64_t n = 0; n < N; ++n) {
        uint8_t* q = (uint8_t*)packed + n * packed_row(K);
        uint8_t* s = (uint8_t*)scales + n * scales_row(K);
        memset(q, 0, packed_row(K));
        memset(s, 127, scales_row(K));
        for (int64_t g = 0; g < G; ++g) {
            const float* v = w + n * K + g * kGroup;
            const int len = (int)(K - g * kGroup < kGroup ? K - g * kGroup : kGroup);
            float top = 0.0f;
            bool finite = true;
            for (int k = 0; k < len; ++k) {
                finite = finite && std::isfinite(v[k]);
                top = std::fmax(top, std::fabs(v[k]));
            }
            HX_REQUIRE(finite, HX_ERR_INVALID_INPUT, "w4_quantize: row %lld holds a value that is not finite", (long long)n);
            int e = -125;  // 4 <= top / 2^e < 8, inside the exponents whose weights bf16 holds exactly
            if (top > 0.0f) e = std::ilogb(top) - 2;
            e = e < -125 ? -125 : e > 125 ? 125 : e;
            s[g] = (uint8_t)(e + 127);
            for (int k = 0; k < len; ++k) {
                const float a = std::ldexp(std::fabs(v[k]), -e);
                // how many midpoints lie below: a tie goes to the even code
                int c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
                if (std::signbit(v[k])) c |= 8;
                const int64_t at = g * kGroup + k;
                q[at >> 1] |= (uint8_t)(c << (at & 1 ? 4 : 0));
            }
        }
    }
    return HX_OK;
}

extern "C" int hx_linear_w4(int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx, const void* packed,
                            const void* scales, const float* bias, int act, int out_dtype, void* Y, int64_t ldy,
                            void* stream) {
    using namespace hx;
    HX_REQUIRE(M >= 0 && N >= 0 && K >= 0, HX_ERR_INVALID_DIMENSION, "linear_w4: negative size");
    HX_REQUIRE(out_dtype == HX_F32 || out_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "linear_w4: out_dtype %d", out_dtype);
    HX_REQUIRE(act >= 0 && act <= 3, HX_ERR_INVALID_INPUT, "linear_w4: act %d", act);
    if (M == 0 || N == 0) return HX_OK;
    HX_REQUIRE(Y && ldy >= N && (K == 0 || (X && packed && scales && ldx >= K)), HX_ERR_INVALID_INPUT,
               "linear_w4: X, packed, scales and Y required, ldx >= K, ldy >= N");
    HX_REQUIRE(aligned(packed, 16) && aligned(scales, 16), HX_ERR_INVALID_INPUT,
               "linear_w4: packed and scales must be 16-byte aligned");
    HX_REQUIRE(N < (1 << 30) && M <= kRowsAtOnce * (int64_t)65535 && K < (1 << 26) && ldx < (1 << 26),
               HX_ERR_UNSUPPORTED, "linear_w4: at most %d rows of X, N below 2^30, K and ldx below 2^26", kRowsAtOnce * 65535);
    // How K is cut decides the order of the sums, so it goes by N and K alone: up to 8 waves a tile of 16 outputs while there
    // are fewer than 8 for each of 256 CUs, or 16 where a wave would walk more than 8 windows, none with fewer than two; and
    // up to 4 where each still walks 8. 1 x 8192 x 8192: 8 waves 11.1 us, 4 waves 12.7; 2 x 16384 x 4096: 4 waves 10.7, 8 waves
    // 11.5, 2 waves 12.6; 45 x 14152 x 736: 2 waves 10.4, 4 waves 12.9; 1 x 32768 x 4096: 4 waves 16.8, 2 waves 19.6; 5 x 32768 x
    // 8192: 34.5 and 34.1; 64 x 32768 x 4096: 52.0 and 50.8; 1 x 65536 x 2048: 2 waves 17.3, 1 wave 20.7.
    const int windows = (int)((K + kWindow - 1) / kWindow);
    const int64_t tiles = (N + 15) / 16;
    int waves = 1;
    while (waves < 8 && windows >= 4 * waves && (tiles * waves < 2048 || (windows > 8 * waves && tiles * waves < 4096) ||
                                                   (windows >= 16 * waves && waves < 4)))
        waves *= 2;
    const W4Args p{M, N, K, ldx, ldy, (const uint16_t*)X, (const uint8_t*)packed, (const uint8_t*)scales, bias, Y, act, windows,
                   (windows + waves - 1) / waves, waves};
    const bool f32 = out_dtype == HX_F32;
    hipStream_t s = as_stream(stream);
    // Two or four tiles share a wave's rows of X where it is X that costs: with few tiles it is the idle CUs.
    //   up to 16 rows  1 tile and 2 tiles: 1 x 32768 x 8192 32.5 and 29.8 us, 2 x 16384 x 4096 10.7 and 11.8; 5 x 32768 x 8192
    //       39.1 and 34.5, 8 x 8950 x 7360 15.6 and 18.3; 16 x 8192 x 8192 15.2 and 13.7. 2 and 4: 16 x 32768 x 8192 43 and 36,
    //       16 x 8950 x 7360 20.8 and 18.5; 16 x 8192 x 8192 13.6 and 17.1, 12 x 32768 x 2048 12.9 and 14.2.
    //   more  the registers leave a CU 8 waves in every form, and a round of blocks takes up to 1.6 times as long with twice
    //       the tiles, so they are doubled where that saves a third of the rounds. 1 and 2 tiles: 60 x 4096 x 4096 12.3 and 9.7
    //       (2 rounds and 1), 24 x 8192 x 544 5.8 and 6.4 (1 and 1). 2 and 4: 64 x 8192 x 8192 28 and 22, 64 x 24576 x 8192 67
    //       and 58 (3 and 2), 64 x 4096 x 4096 8.7 and 12.0 (1 and 1). Where the last round is nearly empty the rule misses:
    //       57 x 8950 x 7360 gets four tiles (2 rounds against 3) at 38.4, 36.5 with two.
    const auto rounds = [&](int64_t t) { return ((tiles + t - 1) / t * ((M + kRowsAtOnce - 1) / kRowsAtOnce) * waves + 2047) / 2048; };
    const bool two = M > 16 ? 3 * rounds(2) <= 2 * rounds(1) : M > 8 ? tiles > 256 : tiles >= (M > 4 ? 1024 : 2048);
    const bool four = M > 16 ? 3 * rounds(4) <= 2 * rounds(2) : M > 8 && tiles > 512 && windows > 32;
    if (M <= 4) return two ? launch_w4<2, 1>(p, f32, s) : launch_w4<1, 1>(p, f32, s);
    if (M <= 8) return two ? launch_w4<2, 2>(p, f32, s) : launch_w4<1, 2>(p, f32, s);
    if (M <= 16) return four ? launch_w4<4, 4>(p, f32, s) : two ? launch_w4<2, 4>(p, f32, s) : launch_w4<1, 4>(p, f32, s);
    return four ? launch_w4<4, 8>(p, f32, s) : two ? launch_w4<2, 8>(p, f32, s) : launch_w4<1, 8>(p, f32, s);
}
