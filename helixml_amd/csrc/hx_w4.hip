// hx_w4.hip — 4-bit weights with group scales (OCP MXFP4): rounding on the host, products on the device.
#include <cmath>

#include "hx_common.h"

namespace hx {
namespace {

constexpr int kGroup = HX_W4_GROUP;

// Bytes of a packed row and of a row of scales: whole groups, and whole 16-byte loads of scales.
__host__ __device__ inline int64_t groups_of(int64_t K) { return (K + kGroup - 1) / kGroup; }
__host__ __device__ inline int64_t packed_row(int64_t K) { return groups_of(K) * (kGroup / 2); }
__host__ __device__ inline int64_t scales_row(int64_t K) { return (groups_of(K) + 15) / 16 * 16; }

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;

constexpr int kWindow = 128;  // elements of K that one 16-byte load per lane covers for 16 rows
constexpr int kAhead = 4;     // windows whose weights are in flight at once

struct W4Args {
    int64_t M, N, K, ldx, ldy;
    const uint16_t* X;
    const uint8_t *W, *S;
    const float* bias;
    void* Y;
    int act, windows, per;  // windows of K, and how many a wave takes
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

// A block computes 16 NT outputs of 16 MT rows of X, its waves a run of windows each. Lane (n, j) of a wave holds row n's
// group j of a window, 32 codes in one 16-byte load under one scale; the matrix instruction i of four takes the codes
// 8i..8i+7 of all four groups, and X's elements at the same places as its other operand (K may be summed in any order).
// With the scale inside the expanded weights the groups need no sums of their own. XVEC: 16-byte aligned rows of X.
template <int NT, int MT, bool XVEC, typename TO>
__global__ __launch_bounds__(1024) void linear_w4_kernel(const W4Args p) {
    extern __shared__ float sums[];  // [waves][NT][MT][16 m][16 n]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, j = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const int64_t G = groups_of(p.K), pr = packed_row(p.K), sr = scales_row(p.K);
    // rows behind the last read the last one; what they give is not stored
    const uint8_t *w[NT], *s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + 16 * t + r < p.N ? n0 + 16 * t + r : p.N - 1;
        w[t] = p.W + n * pr + 16 * j;
        s[t] = p.S + n * sr + j;
    }
    const uint16_t* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = m0 + 16 * t + r < p.M ? m0 + 16 * t + r : p.M - 1;
        x[t] = p.X + m * p.ldx + 32 * j;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b) acc[a][b] = f32x4{0, 0, 0, 0};
    uint32_t top[NT] = {};  // the largest scale byte of each row: 255 is not a number

    const auto load_x = [&](int t, int64_t k, int i, bool whole) {
        const uint16_t* at = x[t] + k + 8 * i;
        union {
            uint4 v;
            uint16_t e[8];
        } u;
        if (XVEC && whole) {
            u.v = *reinterpret_cast<const uint4*>(at);
        } else {
            const int64_t left = p.K - (k + 32 * j + 8 * i);  // elements from K on count as zero
#pragma unroll
            for (int e = 0; e < 8; ++e) u.e[e] = whole || e < left ? at[e] : 0;
        }
        return __builtin_bit_cast(bf16x8, u.v);
    };
    const auto window = [&](int64_t k, const uint4 (&q)[NT], const uint32_t (&sb)[NT], bool whole) {
        float scale[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            scale[t] = __uint_as_float(sb[t] << 23);
            top[t] = sb[t] > top[t] ? sb[t] : top[t];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x8 xb[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) xb[t] = load_x(t, k, i, whole);
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const uint32_t c = i == 0 ? q[a].x : i == 1 ? q[a].y : i == 2 ? q[a].z : q[a].w;
                const bf16x8 wv = expand8(c, scale[a]);
#pragma unroll
                for (int b = 0; b < MT; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xb[b], acc[a][b], 0, 0, 0);
            }
        }
    };

    int at = wave * p.per;
    const int end = at + p.per < p.windows ? at + p.per : p.windows;
    const int whole = (int)(p.K / kWindow) < end ? (int)(p.K / kWindow) : end;
    for (; at + kAhead <= whole; at += kAhead) {
        uint4 q[kAhead][NT];
        uint32_t sb[kAhead][NT];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                q[u][t] = *reinterpret_cast<const uint4*>(w[t] + (int64_t)(at + u) * (kWindow / 2));
                sb[u][t] = s[t][(at + u) * 4];
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) window((int64_t)(at + u) * kWindow, q[u], sb[u], true);
    }
    for (; at < end; ++at) {
        uint4 q[NT];
        uint32_t sb[NT];
        const bool in = at < whole || at * 4 + j < G;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            q[t] = in ? *reinterpret_cast<const uint4*>(w[t] + (int64_t)at * (kWindow / 2)) : make_uint4(0, 0, 0, 0);
            sb[t] = in ? s[t][at * 4] : 127;
        }
        window((int64_t)at * kWindow, q, sb, at < whole);
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

    // The waves' sums in the order of K, then the epilogue; lane (m = r, 4j..4j+3) holds four outputs of a row of X.
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b)
            *reinterpret_cast<f32x4*>(sums + ((wave * NT + a) * MT + b) * 256 + r * 16 + 4 * j) = acc[a][b];
    __syncthreads();
    TO* y = (TO*)p.Y;
    for (int o = threadIdx.x; o < NT * MT * 256; o += blockDim.x) {
        const int a = o / 16 % NT, row = o / (16 * NT);  // consecutive threads take consecutive outputs
        const int64_t n = n0 + 16 * a + o % 16, m = m0 + row;
        if (n >= p.N || m >= p.M) continue;
        const float* at_o = sums + (a * MT + row / 16) * 256 + row % 16 * 16 + o % 16;
        float v = 0.0f;
        for (int k = 0; k < waves; ++k) v += at_o[k * NT * MT * 256];
        if (p.bias) v += p.bias[n];
        if (p.act & 1) v = silu(v);
        TO* to = y + m * p.ldy + n;
        if (p.act & 2) v += Storage<TO>::load(to);
        Storage<TO>::store(to, v);
    }
}

template <int NT, int MT>
int launch_w4(const W4Args& p, int waves, bool xvec, bool f32, hipStream_t s) {
    const dim3 grid((unsigned)((p.N + 16 * NT - 1) / (16 * NT)), (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
    const auto k = f32 ? (xvec ? linear_w4_kernel<NT, MT, true, float> : linear_w4_kernel<NT, MT, false, float>)
                       : (xvec ? linear_w4_kernel<NT, MT, true, uint16_t> : linear_w4_kernel<NT, MT, false, uint16_t>);
    hipLaunchKernelGGL(k, grid, dim3(64 * waves), (size_t)waves * NT * MT * 256 * sizeof(float), s, p);
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
    HX_REQUIRE(N < ((int64_t)1 << 34) && M <= 16 * (int64_t)65535 && K < ((int64_t)1 << 31), HX_ERR_UNSUPPORTED,
               "linear_w4: at most %d rows of X, 2^34 outputs and K below 2^31", 16 * 65535);
    // How K is cut decides the order of the sums, so it goes by N and K alone: enough waves for every CU's 16 (256 CUs),
    // none with less than one window.
    const int windows = (int)((K + kWindow - 1) / kWindow);
    const int64_t tiles = (N + 15) / 16;
    int waves = 1;
    while (waves < 16 && waves * 2 <= windows && tiles * waves < 4096) waves *= 2;
    const W4Args p{M, N, K, ldx, ldy, (const uint16_t*)X, (const uint8_t*)packed, (const uint8_t*)scales, bias, Y, act, windows,
                   (windows + waves - 1) / waves};
    const bool xvec = aligned(X, 16) && ldx % 8 == 0, f32 = out_dtype == HX_F32;
    return launch_w4<1, 1>(p, waves, xvec, f32, as_stream(stream));
}
