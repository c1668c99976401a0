// hx_logits.hip — penalties for repeated tokens, biases and grammar masks on a decode step's logits.
#include "hx_common.h"

namespace hx {
namespace {

constexpr uint32_t kSeen = 1u << 31;  // the token is in the prompt part; the low bits count the answer

struct LogitsArgs {
    int64_t vocab, ldl, ldh, hist, ldb, lda, ldo;
    int slice;  // tokens of one block, each with a counter in LDS
    const int32_t *history, *lengths, *prompts, *allowed;
    const float *repetition, *frequency, *presence, *bias;
};

__device__ inline float adjusted(float l, uint32_t c, float r, float fq, float pr) {
    if (c) l = l > 0.0f ? l / r : l * r;
    if (c & ~kSeen) l = l - fq * (float)(c & ~kSeen) - pr;
    return l;
}

// Block (slice, row): it counts the row's history for its own tokens in LDS, then walks them once. Counters are whole
// numbers, so the order of the atomic adds changes nothing. Every slice reads the whole history, which is why slices are
// as long as the batch allows; bound by the logits' one read and one write and, for few tokens, by latency.
template <typename T>
__global__ __launch_bounds__(1024) void logits_kernel(const LogitsArgs p, const T* logits, T* out) {
    constexpr int kRun = 16 / sizeof(T);
    extern __shared__ uint4 lds[];
    uint32_t* const counts = reinterpret_cast<uint32_t*>(lds);
    const int64_t b = blockIdx.y, v0 = (int64_t)blockIdx.x * p.slice;
    const int n = (int)(p.vocab - v0 < p.slice ? p.vocab - v0 : p.slice);
    const int tid = threadIdx.x, threads = blockDim.x;
    for (int i = tid; i < p.slice / 4; i += threads) lds[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    int len = (int)p.hist;
    if (p.lengths) len = p.lengths[b] < 0 ? 0 : p.lengths[b] < len ? p.lengths[b] : len;
    const int prompt = p.prompts ? p.prompts[b] : 0;
    const int32_t* const h = p.history + b * p.ldh;
    const auto count = [&](int32_t token, int j) {
        const int64_t v = token - v0;
        if (v < 0 || v >= n) return;
        if (j < prompt)
            atomicOr(&counts[v], kSeen);
        else
            atomicAdd(&counts[v], 1u);
    };
    const int runs = len / 4;
    for (int j = tid; j < runs; j += threads) {
        const Run<4, int32_t> t = Run<4, int32_t>::load(h + 4 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) count(t.v[e], 4 * j + e);
    }
    if (tid < len - 4 * runs) count(h[4 * runs + tid], 4 * runs + tid);
    __syncthreads();

    const float r = p.repetition ? p.repetition[b] : 1.0f, fq = p.frequency ? p.frequency[b] : 0.0f,
                pr = p.presence ? p.presence[b] : 0.0f;
    const T* const from = logits + b * p.ldl + v0;
    T* const to = out + b * p.ldo + v0;
    const float* const bias = p.bias ? p.bias + b * p.ldb + v0 : nullptr;
    const int32_t* const allowed = p.allowed ? p.allowed + b * p.lda + v0 / 32 : nullptr;
    const int whole = n / kRun;
    for (int i = tid; i < whole; i += threads) {
        const int at = i * kRun;
        const Run<kRun, T> in = Run<kRun, T>::load(from + at);
        float l[kRun];
        uint32_t any = 0, c[kRun];
#pragma unroll
        for (int e = 0; e < kRun; ++e) {
            l[e] = Storage<T>::load(&in.v[e]);
            c[e] = counts[at + e];
            any |= c[e];
        }
        if (any) {
#pragma unroll
            for (int e = 0; e < kRun; ++e) l[e] = adjusted(l[e], c[e], r, fq, pr);
        }
        if (bias) {
            const Run<kRun, float> add = Run<kRun, float>::load(bias + at);
#pragma unroll
            for (int e = 0; e < kRun; ++e) l[e] += add.v[e];
        }
        if (allowed) {
            const uint32_t bits = (uint32_t)allowed[at / 32] >> (at % 32);  // a run lies within one word
#pragma unroll
            for (int e = 0; e < kRun; ++e) l[e] = bits >> e & 1 ? l[e] : -INFINITY;
        }
        Run<kRun, T> o;
#pragma unroll
        for (int e = 0; e < kRun; ++e) Storage<T>::store(&o.v[e], l[e]);
        o.store(to + at);
    }
    const int at = whole * kRun + tid;
    if (at < n) {
        float l = adjusted(Storage<T>::load(from + at), counts[at], r, fq, pr);
        if (bias) l += bias[at];
        if (allowed && !((uint32_t)allowed[at / 32] >> (at % 32) & 1)) l = -INFINITY;
        Storage<T>::store(to + at, l);
    }
}

}  // namespace
}  // namespace hx

extern "C" int hx_logits_adjust(int64_t batch, int64_t vocab, int dtype, const void* logits, int64_t ldl,
                                const int32_t* history, int64_t ldh, int64_t history_len, const int32_t* lengths,
                                const int32_t* prompt_lengths, const float* repetition, const float* frequency,
                                const float* presence, const float* bias, int64_t ldb, const int32_t* allowed,
                                int64_t lda, void* out, int64_t ldo, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && vocab >= 0 && history_len >= 0, HX_ERR_INVALID_DIMENSION, "logits_adjust: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "logits_adjust: dtype %d", dtype);
    if (batch == 0 || vocab == 0) return HX_OK;
    HX_REQUIRE(batch <= 65535 && vocab < ((int64_t)1 << 31) && history_len < ((int64_t)1 << 31), HX_ERR_UNSUPPORTED,
               "logits_adjust: at most 65535 rows, vocab and history below 2^31");
    HX_REQUIRE(logits && out && ldl >= vocab && ldo >= vocab, HX_ERR_INVALID_INPUT,
               "logits_adjust: logits and out required, row strides of at least vocab");
    HX_REQUIRE(logits != out || ldl == ldo, HX_ERR_INVALID_INPUT, "logits_adjust: in place needs one row stride");
    HX_REQUIRE(history_len == 0 || (history && ldh >= history_len), HX_ERR_INVALID_INPUT,
               "logits_adjust: history required, row stride of at least history_len");
    HX_REQUIRE(!bias || ldb == 0 || ldb >= vocab, HX_ERR_INVALID_INPUT, "logits_adjust: bias row stride 0 or >= vocab");
    HX_REQUIRE(!allowed || lda == 0 || lda >= (vocab + 31) / 32, HX_ERR_INVALID_INPUT,
               "logits_adjust: allowed row stride 0 or >= ceil(vocab / 32)");
    // Slices of up to 16384 tokens (64 KiB of counters), shorter while there are fewer than two blocks a CU for 256 CUs; a
    // thread for every 16 tokens of the slice or of the history, whichever are more.
    int slice = 256;
    while (slice < 16384 && slice < vocab) slice *= 2;
    while (slice > 2048 && batch * ((vocab + slice - 1) / slice) < 512) slice /= 2;
    int threads = 256;
    while (threads < 1024 && threads * 16 < (slice > history_len ? slice : history_len)) threads *= 2;
    const LogitsArgs p{vocab, ldl, ldh, history_len, ldb, lda, ldo, slice, history, lengths, prompt_lengths, allowed,
                       repetition, frequency, presence, bias};
    const dim3 grid((unsigned)((vocab + slice - 1) / slice), (unsigned)batch);
    const size_t lds = slice * sizeof(uint32_t);
    if (dtype == HX_F32)
        hipLaunchKernelGGL(logits_kernel<float>, grid, dim3(threads), lds, as_stream(stream), p, (const float*)logits, (float*)out);
    else
        hipLaunchKernelGGL(logits_kernel<uint16_t>, grid, dim3(threads), lds, as_stream(stream), p, (const uint16_t*)logits,
                           (uint16_t*)out);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
