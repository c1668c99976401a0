// hx_logits.hip — penalties for repeated tokens, biases and grammar masks on a decode step's logits.
#include "hx_common.h"

namespace hx {
namespace {

constexpr int kSlice = 4096;         // tokens of one block, each with a counter in LDS
constexpr uint32_t kSeen = 1u << 31;  // the token is in the prompt part; the low bits count the answer

struct LogitsArgs {
    int64_t vocab, ldl, ldh, hist, ldb, lda, ldo;
    const int32_t *history, *lengths, *prompts, *allowed;
    const float *repetition, *frequency, *presence, *bias;
};

// Block (slice, row). Counters are whole numbers, so the order of the atomic adds changes nothing.
template <typename T>
__global__ __launch_bounds__(256) void logits_kernel(LogitsArgs p, const T* logits, T* out) {
    __shared__ uint32_t counts[kSlice];
    const int64_t b = blockIdx.y, v0 = (int64_t)blockIdx.x * kSlice;
    const int n = (int)(p.vocab - v0 < kSlice ? p.vocab - v0 : kSlice);
    for (int i = threadIdx.x; i < kSlice; i += 256) counts[i] = 0;
    __syncthreads();
    int64_t len = p.lengths ? p.lengths[b] : p.hist;
    len = len < 0 ? 0 : len > p.hist ? p.hist : len;
    const int64_t prompt = p.prompts ? p.prompts[b] : 0;
    for (int64_t j = threadIdx.x; j < len; j += 256) {
        const int64_t v = (int64_t)p.history[b * p.ldh + j] - v0;
        if (v < 0 || v >= n) continue;
        if (j < prompt)
            atomicOr(&counts[v], kSeen);
        else
            atomicAdd(&counts[v], 1u);
    }
    __syncthreads();
    const float r = p.repetition ? p.repetition[b] : 1.0f, fq = p.frequency ? p.frequency[b] : 0.0f,
                pr = p.presence ? p.presence[b] : 0.0f;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int64_t v = v0 + i;
        float l = Storage<T>::load(logits + b * p.ldl + v);
        const uint32_t c = counts[i];
        if (c) l = l > 0.0f ? l / r : l * r;
        if (c & ~kSeen) l = l - fq * (float)(c & ~kSeen) - pr;
        if (p.bias) l += p.bias[b * p.ldb + v];
        if (p.allowed && !((uint32_t)p.allowed[b * p.lda + v / 32] >> (v % 32) & 1)) l = -INFINITY;
        Storage<T>::store(out + b * p.ldo + v, l);
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
    const LogitsArgs p{vocab, ldl, ldh, history_len, ldb, lda, ldo, history, lengths, prompt_lengths, allowed,
                       repetition, frequency, presence, bias};
    dim3 grid((unsigned)((vocab + kSlice - 1) / kSlice), (unsigned)batch);
    if (dtype == HX_F32)
        hipLaunchKernelGGL(logits_kernel<float>, grid, dim3(256), 0, as_stream(stream), p, (const float*)logits, (float*)out);
    else
        hipLaunchKernelGGL(logits_kernel<uint16_t>, grid, dim3(256), 0, as_stream(stream), p, (const uint16_t*)logits,
                           (uint16_t*)out);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
