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

// E2M1: (-1)^s * {0, 0.5, 1, 1.5, 2, 3, 4, 6}.
__device__ inline float e2m1(uint32_t c) {
    const uint32_t e = (c >> 1) & 3, m = c & 1;
    const float v = e == 0 ? 0.5f * m : (float)(1u << (e - 1)) * (1.0f + 0.5f * m);
    return c & 8 ? -v : v;
}

// One wave per (row of X, output): lanes take elements K apart by 64.
template <typename TO>
__global__ __launch_bounds__(256) void linear_w4_kernel(int64_t M, int64_t N, int64_t K, const uint16_t* __restrict__ X,
                                                        int64_t ldx, const uint8_t* __restrict__ W,
                                                        const uint8_t* __restrict__ S, const float* __restrict__ bias,
                                                        int act, TO* __restrict__ Y, int64_t ldy) {
    const int64_t o = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (o >= M * N) return;
    const int64_t m = o / N, n = o - m * N;
    const int lane = threadIdx.x & 63;
    const uint8_t *w = W + n * packed_row(K), *s = S + n * scales_row(K);
    float acc = 0.0f;
    for (int64_t k = lane; k < K; k += 64) {
        const uint32_t c = (w[k >> 1] >> (k & 1 ? 4 : 0)) & 15;
        acc = fmaf(ldexpf(e2m1(c), (int)s[k / kGroup] - 127), Storage<uint16_t>::load(X + m * ldx + k), acc);
    }
    for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, 64);
    if (lane != 0) return;
    if (bias) acc += bias[n];
    if (act & 1) acc = silu(acc);
    TO* y = Y + m * ldy + n;
    if (act & 2) acc += Storage<TO>::load(y);
    Storage<TO>::store(y, acc);
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
    HX_REQUIRE((__int128)M * N < ((__int128)1 << 32), HX_ERR_UNSUPPORTED, "linear_w4: too many outputs");
    dim3 grid((unsigned)((M * N + 3) / 4));
    hipStream_t s = as_stream(stream);
    if (out_dtype == HX_F32)
        hipLaunchKernelGGL(linear_w4_kernel<float>, grid, dim3(256), 0, s, M, N, K, (const uint16_t*)X, ldx,
                           (const uint8_t*)packed, (const uint8_t*)scales, bias, act, (float*)Y, ldy);
    else
        hipLaunchKernelGGL(linear_w4_kernel<uint16_t>, grid, dim3(256), 0, s, M, N, K, (const uint16_t*)X, ldx,
                           (const uint8_t*)packed, (const uint8_t*)scales, bias, act, (uint16_t*)Y, ldy);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
