// hx_i8.hip — products of activations and weights in 8 bits, a scale to every row of each.
#include <cmath>

#include "hx_common.h"
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

// four outputs n.. of row m
template <typename TO>
__device__ inline void finish(const I8Args& p, int64_t m, int64_t n, const i32x4& acc) {
    if (m >= p.M || n >= p.N) return;
    const float sx = p.sx[m];
    TO* to = (TO*)p.Y + m * p.ldy + n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (n + e >= p.N) break;
        float v = (float)acc[e] * (sx * p.sw[n + e]);
        if (p.bias) v += p.bias[n + e];
        if (p.act & 1) v = silu(v);
        if (p.act & 2) v += Storage<TO>::load(to + e);
        Storage<TO>::store(to + e, v);
    }
}

template <typename TO>
__global__ __launch_bounds__(256) void linear_i8_kernel(const I8Args p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, u = lane >> 4;
    const int64_t tile = (int64_t)blockIdx.x * 4 + wave, m0 = (int64_t)blockIdx.y * 64, pieces = pieces_of(p.K);
    if (tile * 16 >= p.N) return;
    const int8_t* w = p.W + tile * pieces * kPiece + lane * 16;
    i32x4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = i32x4{0, 0, 0, 0};
    for (int64_t k = 0; k < pieces; ++k) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(w + k * kPiece);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + 16 * i + r, c = k * 64 + 16 * u;
            const i32x4 b = m < p.M ? load_x(p.X + m * p.ldx + c, p.K - c) : i32x4{0, 0, 0, 0};
            acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc[i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) finish<TO>(p, m0 + 16 * i + r, tile * 16 + 4 * u, acc[i]);
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
    HX_REQUIRE(K < (1 << 17) && M <= 64 * (int64_t)65535 && N < (1 << 28), HX_ERR_UNSUPPORTED,
               "linear_i8: K below 2^17 (sums in 32 bits), at most %d rows of X, N below 2^28", 64 * 65535);
    const I8Args p{M, N, K, ldx, ldy, (const int8_t*)X, (const int8_t*)packed, x_scales, scales, bias, Y, act};
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
    if (out_dtype == HX_F32)
        hipLaunchKernelGGL(linear_i8_kernel<float>, grid, dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL(linear_i8_kernel<uint16_t>, grid, dim3(256), 0, as_stream(stream), p);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
