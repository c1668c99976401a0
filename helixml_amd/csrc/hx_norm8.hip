// hx_norm8.hip — the residual's addition, a root-mean-square norm and rounding to 8 bits with a scale a row, in one pass.
#include "hx_common.h"
#include "hx_wave.h"

namespace hx {
namespace {

struct NormArgs {
    int64_t rows, dim;
    const void *x, *delta;
    int64_t ldx, ldd;
    int ddtype;  // -1: none
    const float* weight;
    float eps;
    void* resid;
    int64_t ldr;
    void* y;
    int64_t ldy;
    float* scales;
};

// With r = x + delta as it is stored and p = r w (exact in 64 bits: two numbers of 24), a row is p / rms(r). In 8 bits its codes
// are round(127 p / max |p|), whatever the norm, and its scale is max |p| / (127 rms). All of it is formed in 64 bits: the
// codes are those of the definition, not of one order of summing, and the rate (half of fp32's) leaves memory the bound.
struct RowSums {
    double squares;
    uint64_t top;  // the largest |p|: the bits of numbers without a sign order as they do, with NaN above all
    __device__ void add(double r, double p) {
        squares = fma(r, r, squares);
        const uint64_t bits = (uint64_t)__double_as_longlong(fabs(p));
        top = bits > top ? bits : top;
    }
    __device__ void join(const RowSums& o) {
        squares += o.squares;
        top = o.top > top ? o.top : top;
    }
};

__device__ inline RowSums over_wave(RowSums s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        RowSums o;
        o.squares = __shfl_xor(s.squares, off, 64);
        o.top = (uint64_t)__shfl_xor((unsigned long long)s.top, off, 64);
        s.join(o);
    }
    return s;
}

enum Kind { kF32 = HX_F32, kBf16 = HX_BF16, kI8 = HX_I8 };

// What a row's elements are multiplied with, and its scale.
struct RowFactor {
    double m, top;
    float scale;
    bool bad;
    template <int KIND>
    static __device__ RowFactor of(const RowSums& s, const NormArgs& p) {
        RowFactor f;
        const double inv = p.weight ? 1.0 / sqrt(s.squares / (double)p.dim + (double)p.eps) : 1.0;
        f.top = __longlong_as_double((long long)s.top);
        f.bad = s.top >= 0x7ff0000000000000ull || !(inv <= 1.7e308);
        if constexpr (KIND == kI8) {
            f.m = f.bad || f.top == 0.0 ? 0.0 : 127.0 / f.top;
            f.scale = f.bad ? __uint_as_float(0x7fc00000u) : (float)(f.top * inv / 127.0);
        } else {
            f.m = inv;
        }
        return f;
    }
    __device__ int code(double p) const {
        if (bad) return 0;
        const double t = p * m;
        double q = rint(t);
        if (fabs(fabs(t - q) - 0.5) < 1e-9) q = rint(p * 127.0 / top);  // a tie of p itself, not of the rounded factor's
        return (int)q;
    }
};

template <int N, typename T>
__device__ inline void load_run(const T* at, int64_t left, float (&v)[N]) {
    if (left >= N) {
        const Run<N, T> r = Run<N, T>::load(at);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = Storage<T>::load(&r.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = e < left ? Storage<T>::load(at + e) : 0.0f;
    }
}
template <int N, typename T>
__device__ inline void store_run(T* at, int64_t left, const T (&v)[N]) {
    if (left >= N) {
        __builtin_memcpy(at, v, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < left) at[e] = v[e];
    }
}
template <typename T> __device__ inline T as_stored(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return Storage<uint16_t>::round(v);
}

// four elements of r from column c on
template <typename TX>
__device__ inline void load_sum(const NormArgs& p, int64_t row, int64_t c, float (&r)[4]) {
    const int64_t left = p.dim - c;
    load_run<4>((const TX*)p.x + row * p.ldx + c, left, r);
    if (p.ddtype >= 0) {
        float d[4];
        if (p.ddtype == HX_F32)
            load_run<4>((const float*)p.delta + row * p.ldd + c, left, d);
        else
            load_run<4>((const uint16_t*)p.delta + row * p.ldd + c, left, d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const TX s = as_stored<TX>(r[e] + d[e]);
            r[e] = Storage<TX>::load(&s);
        }
    }
}
template <typename TX>
__device__ inline void store_sum(const NormArgs& p, int64_t row, int64_t c, const float (&r)[4]) {
    TX s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = as_stored<TX>(r[e]);
    store_run<4>((TX*)p.resid + row * p.ldr + c, p.dim - c, s);
}
template <int KIND>
__device__ inline void store_y(const NormArgs& p, const RowFactor& f, int64_t row, int64_t c, const float (&r)[4], const float (&w)[4]) {
    const int64_t at = row * p.ldy + c, left = p.dim - c;
    if constexpr (KIND == kI8) {
        int8_t q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = (int8_t)f.code((double)r[e] * (double)w[e]);
        store_run<4>((int8_t*)p.y + at, left, q);
    } else {
        using T = std::conditional_t<KIND == kF32, float, uint16_t>;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = as_stored<T>((float)((double)r[e] * (double)w[e] * f.m));
        store_run<4>((T*)p.y + at, left, v);
    }
}

// A row in the registers of THREADS threads, 4 NV elements each: read once, written once.
template <typename TX, int KIND, int THREADS, int NV>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void row_kernel(const NormArgs p) {
    constexpr int kBlock = THREADS < 256 ? 256 : THREADS, kWaves = THREADS / 64;
    const int64_t row = (int64_t)blockIdx.x * (kBlock / THREADS) + threadIdx.x / THREADS;
    const int at = threadIdx.x % THREADS;
    if (THREADS == 64 && row >= p.rows) return;
    float r[NV][4], w[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(i * THREADS + at) * 4;
        load_sum<TX>(p, row, c, r[i]);
        if (p.weight)
            load_run<4>(p.weight + c, p.dim - c, w[i]);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i][e] = 1.0f;
    }
    RowSums s{0.0, 0};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(i * THREADS + at) * 4;
        if (p.resid) store_sum<TX>(p, row, c, r[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s.add(r[i][e], (double)r[i][e] * (double)w[i][e]);
    }
    s = over_wave(s);
    if constexpr (kWaves > 1) {
        __shared__ RowSums part[kWaves];
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
        __syncthreads();
        s = part[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) s.join(part[i]);
    }
    const RowFactor f = RowFactor::of<KIND>(s, p);
#pragma unroll
    for (int i = 0; i < NV; ++i) store_y<KIND>(p, f, row, (int64_t)(i * THREADS + at) * 4, r[i], w[i]);
    if (KIND == kI8 && at == 0) p.scales[row] = f.scale;
}

// Rows of any width: two passes, the second from what the first stored where it stored anything.
template <typename TX, int KIND>
__global__ __launch_bounds__(1024) void wide_row_kernel(const NormArgs p) {
    const int64_t row = blockIdx.x;
    RowSums s{0.0, 0};
    const auto weights = [&](int64_t c, float (&w)[4]) {
        if (p.weight)
            load_run<4>(p.weight + c, p.dim - c, w);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = 1.0f;
    };
    for (int64_t c = threadIdx.x * 4; c < p.dim; c += 4096) {
        float r[4], w[4];
        load_sum<TX>(p, row, c, r);
        weights(c, w);
        if (p.resid) store_sum<TX>(p, row, c, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) s.add(r[e], (double)r[e] * (double)w[e]);
    }
    s = over_wave(s);
    __shared__ RowSums part[16];
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
    __syncthreads();
    s = part[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) s.join(part[i]);
    const RowFactor f = RowFactor::of<KIND>(s, p);
    for (int64_t c = threadIdx.x * 4; c < p.dim; c += 4096) {
        float r[4], w[4];
        if (p.resid)
            load_run<4>((const TX*)p.resid + row * p.ldr + c, p.dim - c, r);
        else
            load_sum<TX>(p, row, c, r);
        weights(c, w);
        store_y<KIND>(p, f, row, c, r, w);
    }
    if (KIND == kI8 && threadIdx.x == 0) p.scales[row] = f.scale;
}

template <typename TX, int KIND>
int launch_rows(const NormArgs& p, hipStream_t s) {
    const dim3 four((unsigned)((p.rows + 3) / 4)), one((unsigned)p.rows);
    if (p.dim <= 512)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 64, 2>), four, dim3(256), 0, s, p);
    else if (p.dim <= 1024)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 64, 4>), four, dim3(256), 0, s, p);
    else if (p.dim <= 2048)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 64, 8>), four, dim3(256), 0, s, p);
    else if (p.dim <= 4096)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 256, 4>), one, dim3(256), 0, s, p);
    else if (p.dim <= 8192)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 256, 8>), one, dim3(256), 0, s, p);
    else if (p.dim <= 16384)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 1024, 4>), one, dim3(1024), 0, s, p);
    else
        hipLaunchKernelGGL((wide_row_kernel<TX, KIND>), one, dim3(1024), 0, s, p);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
template <typename TX>
int launch_kind(const NormArgs& p, int kind, hipStream_t s) {
    return kind == kI8 ? launch_rows<TX, kI8>(p, s) : kind == kF32 ? launch_rows<TX, kF32>(p, s) : launch_rows<TX, kBf16>(p, s);
}

}  // namespace
}  // namespace hx

extern "C" int hx_add_rmsnorm(int64_t rows, int64_t dim, int dtype, const void* x, int64_t ldx, int delta_dtype, const void* delta, int64_t ldd,
                              const float* weight, float eps, void* resid, int64_t ldr, int out_dtype, void* y, int64_t ldy, float* scales,
                              void* stream) {
    using namespace hx;
    HX_REQUIRE(rows >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "add_rmsnorm: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "add_rmsnorm: dtype %d", dtype);
    HX_REQUIRE(!delta || delta_dtype == HX_F32 || delta_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "add_rmsnorm: delta_dtype %d", delta_dtype);
    HX_REQUIRE(out_dtype == HX_F32 || out_dtype == HX_BF16 || out_dtype == HX_I8, HX_ERR_DTYPE_MISMATCH, "add_rmsnorm: out_dtype %d", out_dtype);
    if (rows == 0 || dim == 0) return HX_OK;
    HX_REQUIRE(x && y && (out_dtype != HX_I8 || scales), HX_ERR_INVALID_INPUT, "add_rmsnorm: NULL pointer");
    HX_REQUIRE(ldx >= dim && ldy >= dim && (!delta || ldd >= dim) && (!resid || ldr >= dim), HX_ERR_INVALID_INPUT,
               "add_rmsnorm: a stride is shorter than a row");
    HX_REQUIRE(rows < (1 << 22) || (dim <= 2048 && rows < (1 << 24)), HX_ERR_UNSUPPORTED,
               "add_rmsnorm: fewer than 2^24 rows of up to 2048 elements, 2^22 of more");
    const NormArgs p{rows, dim, x, delta, ldx, ldd, delta ? delta_dtype : -1, weight, eps, resid, ldr, y, ldy, scales};
    return dtype == HX_F32 ? launch_kind<float>(p, out_dtype, as_stream(stream)) : launch_kind<uint16_t>(p, out_dtype, as_stream(stream));
}
