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

// With r = x + delta as it is stored and p = r w, a row is p / rms(r). In 8 bits its codes are round(127 p / max |p|), whatever the
// norm, and its scale is max |p| / (127 rms). The squares are summed in 64 bits, and the codes are those of the definition, not of
// one order of rounding: 127 p / max |p| in 32 bits is off by less than 4e-5 steps, so what lies further than 1e-4 from a border
// is decided by it, and the rest (one element in five thousand) by the exact products, which 64 bits hold (two numbers of 24), and
// the exact sign of their distance from the border.
// The largest of the exact products is sought among the elements that are the largest in 32 bits. Rows whose products leave 32
// bits' range take 64 throughout. Memory bounds it. 32768 x 2048 fp32 with a bf16 delta: 64 bits for every element and a wave a row 207 us,
// a block of four waves a row, 2 x 4 elements a lane (60 registers for 145), 146 (5.1 TB/s); to fp32, every element in 64 bits, 181 (5.2), to
// bf16 151 (5.3). A bf16 stream has fewer bytes for the same arithmetic: with a bf16 delta 111 (4.2 TB/s), without a delta 62 to 65 (3.1).
struct RowSums {
    double squares;
    uint32_t top;  // the largest |p| in 32 bits: the bits of numbers without a sign order as they do, with NaN above all
    __device__ void add(float r, float w) {
        squares = fma((double)r, (double)r, squares);
        const uint32_t bits = __float_as_uint(r * w) & 0x7fffffffu;
        top = bits > top ? bits : top;
    }
    __device__ void join(const RowSums& o) {
        squares += o.squares;
        top = o.top > top ? o.top : top;
    }
    __device__ bool common() const { return top >= 0x0d800000u && top < 0x71800000u; }  // 2^-100 and 2^100
};

// over the THREADS of a row, the same in all of them
template <int THREADS>
__device__ inline RowSums over_row(RowSums v, RowSums* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v.join({__shfl_xor(v.squares, off, 64), (uint32_t)__shfl_xor((int)v.top, off, 64)});
    if constexpr (THREADS > 64) {
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < THREADS / 64; ++i) v.join(part[i]);
    }
    return v;
}
// |p| in 64 bits, as the integer that orders as it does
__device__ inline unsigned long long exact_bits(float r, float w) { return (unsigned long long)__double_as_longlong(fabs((double)r * (double)w)); }
// Where one of four elements is the row's largest in 32 bits (or all are to be looked at), the largest of their exact products.
__device__ inline void find_top(const float (&r)[4], const float (&w)[4], const RowSums& s, unsigned long long* top) {
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t bits = __float_as_uint(r[e] * w[e]) & 0x7fffffffu;
        most = bits > most ? bits : most;
    }
    if (most == s.top || !s.common()) {
        unsigned long long v = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned long long bits = exact_bits(r[e], w[e]);
            v = bits > v ? bits : v;
        }
        atomicMax(top, v);  // whichever order they come in
    }
}
__device__ inline double inverse_rms(const RowSums& s, const NormArgs& p) {
    return p.weight ? 1.0 / sqrt(s.squares / (double)p.dim + (double)p.eps) : 1.0;
}

// round(127 |p| / top), ties to even, of products of 48 bits; by = 127 / top. 127 |p| has up to 55 bits, so its quotient would be rounded
// twice, and an element of half the row's largest go either way. The border above a whole part that is right or one off is exact: 254 |p| -
// (2 whole + 1) top, the second product as a rounded one and its error. Next to a border the difference is a few units of what the
// products are multiples of; elsewhere its sign is plain.
__device__ inline int exact_code(float r, float w, double top, double by) {
    const double rw = (double)r * (double)w, p = fabs(rw), whole = floor(p * by), odd = 2.0 * whole + 1.0, edge = odd * top;
    const double over = fma(254.0, p, -edge) - fma(odd, top, -edge);
    const int code = (int)whole + (over > 0.0 || (over == 0.0 && ((int)whole & 1)));
    return rw < 0.0 ? -code : code;  // (the signs' own bits were held in registers for all elements, 10 more)
}

enum Kind { kF32 = HX_F32, kBf16 = HX_BF16, kI8 = HX_I8 };

// What four elements become. For codes: the largest |p| exactly and 127 over it in 32 bits (0 where that does not serve).
struct RowFactor {
    double top, inv;
    float m32;
    bool zero, fast;
    __device__ static RowFactor of_codes(const RowSums& s, unsigned long long top) {
        RowFactor f;
        f.top = __longlong_as_double((long long)top);
        f.zero = top == 0 || top >= 0x7ff0000000000000ull;
        f.fast = s.common();
        f.m32 = 127.0f / __uint_as_float(s.top);
        f.inv = 0.0;
        return f;
    }
    __device__ static RowFactor of_values(const RowSums& s, const NormArgs& p) {
        RowFactor f{};
        f.inv = inverse_rms(s, p);
        f.m32 = (float)f.inv;
        // (a subnormal product is off by 2^-150, which the factor lifts: to 2^-141 at most, far below half a step of bf16)
        f.fast = s.common() && f.inv >= 0x1p-100 && f.inv <= 0x1p9;
        return f;
    }
    __device__ uint32_t codes(const float (&r)[4], const float (&w)[4]) const {
        int q[4];
        bool border = !fast;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = r[e] * w[e] * m32, whole = rintf(t);
            border |= fabsf(t - whole) > 0.4999f;
            q[e] = (int)whole;
        }
        if (border) {
            const double by = 127.0 / top;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = zero ? 0 : exact_code(r[e], w[e], top, by);
        }
        return (uint32_t)(q[0] & 255) | (uint32_t)(q[1] & 255) << 8 | (uint32_t)(q[2] & 255) << 16 | (uint32_t)q[3] << 24;
    }
};
// a row's scale; NaN where it holds what is not finite (a NaN among the products is above all numbers in `top`), 0 where all of its
// products are zero, also where its squares are and eps is, so that 1 / rms has no value
__device__ inline float scale_of(const RowSums& s, unsigned long long top, const NormArgs& p) {
    if (top == 0) return 0.0f;
    const double inv = inverse_rms(s, p);
    return top >= 0x7ff0000000000000ull || !(inv <= 1.7e308) ? __uint_as_float(0x7fc00000u) : (float)(__longlong_as_double((long long)top) * inv / 127.0);
}

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
        const uint32_t q = f.codes(r, w);
        int8_t v[4];
        __builtin_memcpy(v, &q, 4);
        store_run<4>((int8_t*)p.y + at, left, v);
    } else {
        using T = std::conditional_t<KIND == kF32, float, uint16_t>;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = as_stored<T>(KIND == kBf16 && f.fast ? r[e] * w[e] * f.m32 : (float)((double)r[e] * (double)w[e] * f.inv));
        store_run<4>((T*)p.y + at, left, v);
    }
}

// A row in the registers of THREADS threads, 4 NV elements each: read once, written once.
template <typename TX, int KIND, int THREADS, int NV>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void row_kernel(const NormArgs p) {
    constexpr int kBlock = THREADS < 256 ? 256 : THREADS;
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
        for (int e = 0; e < 4; ++e) s.add(r[i][e], w[i][e]);
    }
    __shared__ RowSums sums[kBlock / 64];
    __shared__ unsigned long long tops[kBlock / THREADS];
    unsigned long long* const top = tops + threadIdx.x / THREADS;
    if (at == 0) *top = 0;
    s = over_row<THREADS>(s, sums);
    if constexpr (KIND == kI8) {
        const auto meet = [] {  // of a row's threads
            if constexpr (THREADS > 64) {
                __syncthreads();
            } else {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");
                __builtin_amdgcn_wave_barrier();
            }
        };
        meet();
#pragma unroll
        for (int i = 0; i < NV; ++i) find_top(r[i], w[i], s, top);
        meet();
        const RowFactor f = RowFactor::of_codes(s, *top);
#pragma unroll
        for (int i = 0; i < NV; ++i) store_y<KIND>(p, f, row, (int64_t)(i * THREADS + at) * 4, r[i], w[i]);
        if (at == 0) p.scales[row] = scale_of(s, *top, p);
    } else {
        const RowFactor f = RowFactor::of_values(s, p);
#pragma unroll
        for (int i = 0; i < NV; ++i) store_y<KIND>(p, f, row, (int64_t)(i * THREADS + at) * 4, r[i], w[i]);
    }
}

// Rows of any width: passes over the row, the later ones from what the first stored where it stored anything. Two blocks a CU, whose 64
// registers the 8-bit form passes by two: 4096 x 20000 bf16 with a bf16 delta 224 us, with one block 316.
template <typename TX, int KIND>
__global__ __launch_bounds__(1024, 8) void wide_row_kernel(const NormArgs p) {
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
        for (int e = 0; e < 4; ++e) s.add(r[e], w[e]);
    }
    __shared__ RowSums sums[16];
    __shared__ unsigned long long top;
    if (threadIdx.x == 0) top = 0;
    s = over_row<1024>(s, sums);
    const auto again = [&](int64_t c, float (&r)[4], float (&w)[4]) {
        if (p.resid)
            load_run<4>((const TX*)p.resid + row * p.ldr + c, p.dim - c, r);
        else
            load_sum<TX>(p, row, c, r);
        weights(c, w);
    };
    if constexpr (KIND == kI8) {
        for (int64_t c = threadIdx.x * 4; c < p.dim; c += 4096) {
            float r[4], w[4];
            again(c, r, w);
            find_top(r, w, s, &top);
        }
        __syncthreads();
    }
    const RowFactor f = KIND == kI8 ? RowFactor::of_codes(s, top) : RowFactor::of_values(s, p);
    for (int64_t c = threadIdx.x * 4; c < p.dim; c += 4096) {
        float r[4], w[4];
        again(c, r, w);
        store_y<KIND>(p, f, row, c, r, w);
    }
    if (KIND == kI8 && threadIdx.x == 0) p.scales[row] = scale_of(s, top, p);
}

template <typename TX, int KIND>
int launch_rows(const NormArgs& p, hipStream_t s) {
    const dim3 four((unsigned)((p.rows + 3) / 4)), one((unsigned)p.rows);
    if (p.dim <= 512)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 64, 2>), four, dim3(256), 0, s, p);
    else if (p.dim <= 1024)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 256, 1>), one, dim3(256), 0, s, p);
    else if (p.dim <= 2048)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 256, 2>), one, dim3(256), 0, s, p);
    else if (p.dim <= 4096)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 256, 4>), one, dim3(256), 0, s, p);
    else if (p.dim <= 8192)
        hipLaunchKernelGGL((row_kernel<TX, KIND, 1024, 2>), one, dim3(1024), 0, s, p);
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
    HX_REQUIRE(!resid || ((resid != x || ldr == ldx) && (resid != delta || (delta_dtype == dtype && ldr == ldd))), HX_ERR_INVALID_INPUT,
               "add_rmsnorm: resid in the place of x or delta needs its type and stride");
    HX_REQUIRE(rows < (1 << 22) || (dim <= 4096 && rows < (1 << 24)), HX_ERR_UNSUPPORTED,
               "add_rmsnorm: fewer than 2^24 rows of up to 4096 elements, 2^22 of more");
    const NormArgs p{rows, dim, x, delta, ldx, ldd, delta ? delta_dtype : -1, weight, eps, resid, ldr, y, ldy, scales};
    return dtype == HX_F32 ? launch_kind<float>(p, out_dtype, as_stream(stream)) : launch_kind<uint16_t>(p, out_dtype, as_stream(stream));
}
