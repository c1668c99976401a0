// hx_gated.hip — the gated linear recurrence with one state per channel: forward, backward, one token.
//   a = sigmoid(f), i = sigmoid(-f);  h_t = a_t h_{t-1} + i_t x_t;  out = h [silu(z)]
#include "hx_common.h"
#include "hx_wave.h"

namespace hx {
namespace {

constexpr int kChunk = HX_GATED_CHUNK;

// Both gates from one exponential of -|f|, which is at most 1: neither overflows, and the smaller of
// the two is a product, so it keeps its relative accuracy where the other rounds to 1. A state's decay
// over n steps is a product of n gates, in which the reciprocal's error of up to an ulp, always to the
// same side for neighbouring values, would add up: one Newton step, with the rounding error d of 1 + e
// (exact, as e <= 1), leaves that of the last rounding alone.
__device__ inline void gates(float f, float& a, float& i) {
    const float e = fast_exp2(-fabsf(f) * kLog2e);
    const float u = 1.0f + e, d = e - (u - 1.0f), q = fast_rcp(u);
    const float r = fmaf(q, fmaf(-u, q, 1.0f) - d * q, q), s = e * r;
    a = f >= 0.0f ? r : s;
    i = f >= 0.0f ? s : r;
}

// silu(z) and its derivative s (1 + z (1 - s)), s = sigmoid(z), from the same exponential.
__device__ inline void silu_grad(float z, float& v, float& d) {
    float s, t;
    gates(z, s, t);
    v = z * s;
    d = s * fmaf(z, t, 1.0f);
}

// One thread per (batch, channel), in time order.
template <typename T>
__global__ __launch_bounds__(64) void gated_fwd_kernel(int64_t rows, int64_t L, int64_t D, const T* __restrict__ x,
                                                       const T* __restrict__ f, const T* __restrict__ z,
                                                       const float* __restrict__ init, T* __restrict__ out,
                                                       float* __restrict__ last, float* __restrict__ states) {
    const int64_t r = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (r >= rows) return;
    const int64_t b = r / D, d = r - b * D, nc = (L + kChunk - 1) / kChunk;
    float h = init ? init[r] : 0.0f;
    for (int64_t t = 0; t < L; ++t) {
        if (states && t % kChunk == 0) states[(b * nc + t / kChunk) * D + d] = h;
        const int64_t o = (b * L + t) * D + d;
        float a, i;
        gates(Storage<T>::load(f + o), a, i);
        h = fmaf(a, h, i * Storage<T>::load(x + o));
        Storage<T>::store(out + o, z ? h * silu(Storage<T>::load(z + o)) : h);
    }
    if (last) last[r] = h;
}

// One thread per (batch, channel), chunks from the last: a chunk's states before each step are formed
// again from the stored one and kept in LDS.
template <typename T>
__global__ __launch_bounds__(64) void gated_bwd_kernel(int64_t rows, int64_t L, int64_t D, const T* __restrict__ x,
                                                       const T* __restrict__ f, const T* __restrict__ z,
                                                       const float* __restrict__ states, const T* __restrict__ dout,
                                                       const float* __restrict__ dlast, T* __restrict__ dx,
                                                       T* __restrict__ df, T* __restrict__ dz, float* __restrict__ dinit) {
    __shared__ float before[kChunk][64];
    const int64_t r = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (r >= rows) return;
    const int64_t b = r / D, d = r - b * D, nc = (L + kChunk - 1) / kChunk;
    float carry = dlast ? dlast[r] : 0.0f;  // a_{t+1} g_{t+1}
    for (int64_t c = nc - 1; c >= 0; --c) {
        const int64_t t0 = c * kChunk;
        const int n = (int)(L - t0 < kChunk ? L - t0 : kChunk);
        float h = states[(b * nc + c) * D + d];
        for (int k = 0; k < n; ++k) {
            const int64_t o = (b * L + t0 + k) * D + d;
            before[k][threadIdx.x] = h;
            float a, i;
            gates(Storage<T>::load(f + o), a, i);
            h = fmaf(a, h, i * Storage<T>::load(x + o));
        }
        for (int k = n - 1; k >= 0; --k) {
            const int64_t o = (b * L + t0 + k) * D + d;
            const float xv = Storage<T>::load(x + o), hb = before[k][threadIdx.x], dy = Storage<T>::load(dout + o);
            float a, i, dh = dy;
            gates(Storage<T>::load(f + o), a, i);
            if (z) {
                float v, g;
                silu_grad(Storage<T>::load(z + o), v, g);
                Storage<T>::store(dz + o, dy * fmaf(a, hb, i * xv) * g);
                dh = dy * v;
            }
            const float g = dh + carry, gi = g * i;
            Storage<T>::store(dx + o, gi);
            Storage<T>::store(df + o, gi * a * (hb - xv));
            carry = g * a;
        }
    }
    if (dinit) dinit[r] = carry;
}

template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(int64_t n, float* __restrict__ state, const T* __restrict__ x,
                                                         const T* __restrict__ f, const T* __restrict__ z,
                                                         T* __restrict__ out) {
    const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (o >= n) return;
    float a, i;
    gates(Storage<T>::load(f + o), a, i);
    const float h = fmaf(a, state[o], i * Storage<T>::load(x + o));
    state[o] = h;
    Storage<T>::store(out + o, z ? h * silu(Storage<T>::load(z + o)) : h);
}

// dst = src, or zero: what is left of a sequence without steps.
__global__ __launch_bounds__(256) void gated_state_copy_kernel(int64_t n, const float* __restrict__ src,
                                                               float* __restrict__ dst) {
    const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (o < n) dst[o] = src ? src[o] : 0.0f;
}

constexpr int64_t kMaxBlocks = 0x7fffffff;  // of one grid axis

// batch * seqlen * dim elements whose byte offsets fit 63 bits, rows that fit one grid axis.
bool sizes_fit(int64_t batch, int64_t seqlen, int64_t dim) {
    __int128 n = (__int128)batch * dim;
    return n < (__int128)64 * kMaxBlocks && n * (seqlen > 0 ? seqlen : 1) < ((__int128)1 << 60);
}

int copy_state(int64_t rows, const float* src, float* dst, hipStream_t s) {
    if (!dst) return HX_OK;
    hipLaunchKernelGGL(gated_state_copy_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, s, rows, src, dst);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

template <typename T>
int fwd(int64_t batch, int64_t L, int64_t D, const void* x, const void* f, const void* z, const float* init, void* out,
        float* last, float* states, hipStream_t s) {
    const int64_t rows = batch * D;
    hipLaunchKernelGGL(gated_fwd_kernel<T>, dim3((unsigned)((rows + 63) / 64)), dim3(64), 0, s, rows, L, D, (const T*)x,
                       (const T*)f, (const T*)z, init, (T*)out, last, states);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

template <typename T>
int bwd(int64_t batch, int64_t L, int64_t D, const void* x, const void* f, const void* z, const float* states,
        const void* dout, const float* dlast, void* dx, void* df, void* dz, float* dinit, hipStream_t s) {
    const int64_t rows = batch * D;
    hipLaunchKernelGGL(gated_bwd_kernel<T>, dim3((unsigned)((rows + 63) / 64)), dim3(64), 0, s, rows, L, D, (const T*)x,
                       (const T*)f, (const T*)z, states, (const T*)dout, dlast, (T*)dx, (T*)df, (T*)dz, dinit);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

}  // namespace
}  // namespace hx

extern "C" size_t hx_gated_scan_workspace_size(int64_t, int64_t, int64_t, int) { return 0; }
extern "C" size_t hx_gated_scan_bwd_workspace_size(int64_t, int64_t, int64_t, int) { return 0; }

extern "C" int hx_gated_scan_fwd(int64_t batch, int64_t seqlen, int64_t dim, int dtype, const void* x, const void* f,
                                 const void* z, const float* init_state, void* out, float* last_state, float* states,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && seqlen >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "gated_scan: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "gated_scan: dtype %d", dtype);
    if (batch == 0 || dim == 0) return HX_OK;
    HX_REQUIRE(sizes_fit(batch, seqlen, dim), HX_ERR_UNSUPPORTED, "gated_scan: too many elements");
    const size_t need = hx_gated_scan_workspace_size(batch, seqlen, dim, dtype);
    hipStream_t s = as_stream(stream);
    if (seqlen == 0) return copy_state(batch * dim, init_state, last_state, s);
    HX_REQUIRE(x && f && out, HX_ERR_INVALID_INPUT, "gated_scan: x, f and out are required");
    HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), HX_ERR_INVALID_INPUT,
               "gated_scan: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
    return dtype == HX_F32 ? fwd<float>(batch, seqlen, dim, x, f, z, init_state, out, last_state, states, s)
                           : fwd<uint16_t>(batch, seqlen, dim, x, f, z, init_state, out, last_state, states, s);
}

extern "C" int hx_gated_scan_bwd(int64_t batch, int64_t seqlen, int64_t dim, int dtype, const void* x, const void* f,
                                 const void* z, const float* states, const void* dout, const float* dlast, void* dx,
                                 void* df, void* dz, float* dinit, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && seqlen >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "gated_scan_bwd: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "gated_scan_bwd: dtype %d", dtype);
    if (batch == 0 || dim == 0) return HX_OK;
    HX_REQUIRE(sizes_fit(batch, seqlen, dim), HX_ERR_UNSUPPORTED, "gated_scan_bwd: too many elements");
    const size_t need = hx_gated_scan_bwd_workspace_size(batch, seqlen, dim, dtype);
    hipStream_t s = as_stream(stream);
    if (seqlen == 0) return copy_state(batch * dim, dlast, dinit, s);
    HX_REQUIRE(x && f && states && dout && dx && df, HX_ERR_INVALID_INPUT,
               "gated_scan_bwd: x, f, states, dout, dx and df are required");
    HX_REQUIRE((z == nullptr) == (dz == nullptr), HX_ERR_INVALID_INPUT, "gated_scan_bwd: dz goes with z");
    HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), HX_ERR_INVALID_INPUT,
               "gated_scan_bwd: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
    return dtype == HX_F32
               ? bwd<float>(batch, seqlen, dim, x, f, z, states, dout, dlast, dx, df, dz, dinit, s)
               : bwd<uint16_t>(batch, seqlen, dim, x, f, z, states, dout, dlast, dx, df, dz, dinit, s);
}

extern "C" int hx_gated_state_update(int64_t batch, int64_t dim, int dtype, float* state, const void* x, const void* f,
                                     const void* z, void* out, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "gated_state_update: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "gated_state_update: dtype %d", dtype);
    if (batch == 0 || dim == 0) return HX_OK;
    HX_REQUIRE(sizes_fit(batch, 1, dim), HX_ERR_UNSUPPORTED, "gated_state_update: too many elements");
    HX_REQUIRE(state && x && f && out, HX_ERR_INVALID_INPUT, "gated_state_update: state, x, f and out are required");
    const int64_t n = batch * dim;
    dim3 grid((unsigned)((n + 255) / 256));
    if (dtype == HX_F32)
        hipLaunchKernelGGL(gated_step_kernel<float>, grid, dim3(256), 0, as_stream(stream), n, state, (const float*)x,
                           (const float*)f, (const float*)z, (float*)out);
    else
        hipLaunchKernelGGL(gated_step_kernel<uint16_t>, grid, dim3(256), 0, as_stream(stream), n, state,
                           (const uint16_t*)x, (const uint16_t*)f, (const uint16_t*)z, (uint16_t*)out);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
