// hx_decay.hip — linear attention with one decay per head: whole sequences, their backward pass, one token.
#include "hx_common.h"
#include "hx_wave.h"

namespace hx {
namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ the mathematics
// Every pass over a sequence is one mixing of three operands, tokens counted in the pass's own direction:
//   out_i = ps sum_{j <= i} w^(i-j) (a_i . b_j) c_j + es w^(i+e0) a_i S,     S the state before the first token,
//   S' = w^n S + cs sum_j w^(n-1-j+1-e0) b_j c_j^T                          the state after n tokens
// with w = e^g, g = log_decay[head]:
//   out  a = q, b = k, c = v, forwards, e0 = 1        dq  a = do, b = v, c = k, forwards, e0 = 1 (its state is S^T)
//   dv   a = k, b = q, c = do, backwards, e0 = 0      dk  a = v, b = do, c = q, backwards, e0 = 0 (S^T's adjoint)
// Tokens are taken in chunks: inside a chunk the sum over j is two matrix products around the masked and weighted scores,
// what came before enters through the state. Powers with a negative exponent are never formed, so no decay overflows.
struct MixArgs {
    const void *a, *b, *c;
    int64_t lda, ldb, ldc;  // elements from one token to the next
    int ga, gb, gc;         // heads that share one head of the operand
    int64_t B, L, H;
    int m, n, heads_out;  // channels of a and b, of c and the output
    const float* log_decay;
    const int32_t* lengths;
    const float* init;   // [B, H, dk, dv]: the states before the first token (nullable: zero)
    float* last;         // the states after the last one (nullable)
    float* parts;        // [B, H, segments, dk, dv]: what each segment gives from a zero state, or, chained, the states before segments
    int chained;
    int64_t state;       // elements of a state
    int sm, sn;                // a state's strides along m and n
    float ps, es, cs;
    int e0, back;
    void* out;
    int64_t ldo;
    int64_t seglen;  // tokens of a segment, whole chunks
    int nseg;
};
// Passes of one kind that go out as one launch, their blocks side by side: what they share they find in the L2.
constexpr int kMaxPasses = 3;
struct MixPasses {
    MixArgs p[kMaxPasses];
    int count, slices;
    int64_t b0;  // the first sequence of the launch
};

// w^x for x >= 0 as 2^(x l2); a decay of nothing (g = -inf) keeps w^0 = 1.
__device__ inline float log2_decay(float g) {
    const float l2 = g * kLog2e;
    return l2 < -1e30f ? -1e30f : l2;
}
__device__ inline float power(float l2, int x) { return fast_exp2(l2 * (float)x); }
// The decay of a state over x tokens as v -> v * a + v * b. Near 1 the difference from 1 is what is kept: a factor rounded to
// 24 bits would repeat its error at every chunk, 3e-8 times the chunks that a state lives for.
struct Decay {
    float a, b;
    __device__ Decay(float g, float x) {
        const float y = g * x;  // -inf * 0 is a decay over nothing
        const bool near = x == 0.0f || (y > -0.5f && y < 0.5f);
        a = near ? 1.0f : __expf(y);
        b = near ? (x == 0.0f ? 0.0f : expm1f(y)) : 0.0f;
    }
    // v decayed, and x added
    __device__ float operator()(float v, float x) const { return fmaf(v, a, fmaf(v, b, x)); }
};

// ------------------------------------------------------------------ eight values a lane along a contraction of 32
// Lane (r = lane % 16, u = lane / 16) of an operand holds row (or column) r and the contraction's places 8u..8u + 7: one bf16
// instruction, or eight in fp32 that each contract over u. Any order of the places will do as long as both operands have it.
template <typename T> struct Frag;
template <> struct Frag<uint16_t> {
    bf16x8 v;
};
template <> struct Frag<float> {
    float v[8];
};
__device__ inline f32x4 mma(f32x4 acc, const Frag<uint16_t>& a, const Frag<uint16_t>& b) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ inline f32x4 mma(f32x4 acc, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
    return acc;
}

// fp32 values as a sum of PARTS operands of type T: bf16 keeps 8 bits a part (two leave 2^-17 of the value, three all of fp32's).
template <typename T, int PARTS> struct Split;
template <int PARTS> struct Split<float, PARTS> {
    static constexpr int kParts = 1;
    Frag<float> p[1];
    Split() = default;
    __device__ explicit Split(const float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[0].v[e] = x[e];
    }
};
template <int PARTS> struct Split<uint16_t, PARTS> {
    static constexpr int kParts = PARTS;
    Frag<uint16_t> p[PARTS];
    Split() = default;
    __device__ explicit Split(const float (&x)[8]) {
        float rest[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = pack_bf16x2(rest[2 * i], rest[2 * i + 1]);
                rest[2 * i] -= __uint_as_float(w[i] << 16);
                rest[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
            }
            p[k].v = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
        }
    }
};

// places 8u..8u + 7 of one row of a tile
__device__ inline Frag<uint16_t> row_frag(const uint16_t* at) { return {*reinterpret_cast<const bf16x8*>(at)}; }
__device__ inline Frag<float> row_frag(const float* at) {
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(at + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[4 * i + e] = v[e];
    }
    return f;
}
// places 4u..4u + 3 of two neighbouring groups of 16: how a state's accumulators hold their rows
__device__ inline Frag<uint16_t> pair_frag(const uint16_t* at) {
    const uint2 x = *reinterpret_cast<const uint2*>(at), y = *reinterpret_cast<const uint2*>(at + 16);
    return {__builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, y.x, y.y))};
}
__device__ inline Frag<float> pair_frag(const float* at) {
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(at + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[4 * i + e] = v[e];
    }
    return f;
}
// Eight rows of one column of a tile: rows 8u.. of column r, `at` being what col_at gives for the tile's first row and column.
// bf16 comes through the LDS's transposing read: of 16 lanes each names four neighbours of a row, four lanes to a row, and gets
// four rows of its own column.
template <typename T, int STRIDE>
__device__ inline int col_at(int r, int u) {
    return sizeof(T) == 2 ? (8 * u + r / 4) * STRIDE + r % 4 * 4 : 8 * u * STRIDE + r;
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
template <int STRIDE>
__device__ inline Frag<uint16_t> col_frag(const uint16_t* at) {
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * STRIDE));
    return {__builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7))};
}
template <int STRIDE>
__device__ inline Frag<float> col_frag(const float* at) {
    Frag<float> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = at[e * STRIDE];
    return f;
}
__device__ inline float value(const Frag<uint16_t>& f, int e) {
    const uint4 w = __builtin_bit_cast(uint4, f.v);
    const uint32_t x = e < 2 ? w.x : e < 4 ? w.y : e < 6 ? w.z : w.w;
    return __uint_as_float(e & 1 ? x & 0xffff0000u : x << 16);
}
__device__ inline float value(const Frag<float>& f, int e) { return f.v[e]; }

__device__ inline bool not_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
__device__ inline Frag<uint16_t> finite_only(const Frag<uint16_t>& f) {
    uint4 w = __builtin_bit_cast(uint4, f.v);
    const auto keep = [](uint32_t x) {
        return ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
    };
    return {__builtin_bit_cast(bf16x8, make_uint4(keep(w.x), keep(w.y), keep(w.z), keep(w.w)))};
}
__device__ inline Frag<float> finite_only(Frag<float> f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = not_finite(f.v[e]) ? 0.0f : f.v[e];
    return f;
}
// Rows by columns of T in LDS, 16 bytes apart from a multiple of all banks, and the registers through which a chunk of them comes
// from global memory: a thread has the same 16 bytes of every few rows. Loads go out without a branch, rows and columns that are
// not there reading ones that are; columns behind a row's end are never written to LDS and keep the zeros that it starts with.
// WHOLE: rows end with a whole 16 bytes. Else the last 16 bytes end with the row, and repeat in LDS what stands before them (they
// were moved into place in registers, for which the compiler took scratch memory: training 2 x 19407 x 15 x 57 bf16 1637 -> 608 us).
// Where a slice's first columns are a row's last, what repeats falls into the E elements of padding before them.
template <typename T, int ROWS, int COLS, int THREADS, bool WHOLE>
struct Tile {
    static constexpr int E = 16 / sizeof(T), kStride = COLS + E, kPerRow = (COLS > 128 ? 256 : COLS) / E, kStep = THREADS / kPerRow;
    static constexpr int kEach = (ROWS + kStep - 1) / kStep, kBytes = ROWS * kStride * (int)sizeof(T);
    static_assert(THREADS % kPerRow == 0, "a thread's column is the same in all rows");
    u32x4 reg[kEach];
    int row, col, place, n;
    bool in;
    // columns c0.. of rows of n
    __device__ void begin(int c0, int width) {
        row = threadIdx.x / kPerRow;
        n = width;
        const int want = c0 + threadIdx.x % kPerRow * E, most = WHOLE || n >= E ? n - E : 0;
        in = want < n;
        col = want < most ? want : most;
        place = WHOLE ? threadIdx.x % kPerRow * E : col - c0;
    }
    // A row of fewer than E elements, which only the narrowest tile holds.
    static constexpr bool kNarrow = !WHOLE && COLS <= 64;
    __device__ u32x4 narrow(const T* at) const {
        uint64_t v[2] = {0, 0};
        int k = 0;
        if (sizeof(T) == 2 && (n & 4)) {
            __builtin_memcpy(&v[0], at, 8);
            k = 8;
        }
        if (n & 2) {
            uint64_t x = 0;
            __builtin_memcpy(&x, at + k / sizeof(T), 2 * sizeof(T));
            if (k) v[1] = x;
            else v[0] = x;
            k += 2 * sizeof(T);
        }
        if (n & 1) {
            T x;
            __builtin_memcpy(&x, at + k / sizeof(T), sizeof(T));
            const uint64_t bits = sizeof(T) == 2 ? (uint64_t)x : (uint64_t)__builtin_bit_cast(uint32_t, (float)x);
            if (k < 8) v[0] |= bits << (8 * k);
            else v[1] |= bits << (8 * k - 64);
        }
        return u32x4{(uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32)};
    }
    // Rows shift.. of the tile are tokens of a chunk, ROWS - shift of them, the first (or, backwards, the last) at `first`.
    __device__ void load(const T* first, int64_t ld, int shift, bool back) {
        if (kNarrow && n < E) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                int k = row + i * kStep - shift;
                k = k < 0 ? 0 : k >= ROWS - shift ? ROWS - shift - 1 : k;
                reg[i] = narrow(first + (back ? ROWS - shift - 1 - k : k) * ld);
            }
        } else if (shift == 0 && ROWS % kStep == 0) {  // one offset, and places that are the same for all threads
            const uint32_t off = (uint32_t)((back ? kStep - 1 - row : row) * (int)ld + col);
#pragma unroll
            for (int i = 0; i < kEach; ++i) __builtin_memcpy(&reg[i], first + (back ? kEach - 1 - i : i) * kStep * ld + off, 16);
        } else {
            const int valid = ROWS - shift;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                int k = row + i * kStep - shift;
                k = k < 0 ? 0 : k >= valid ? valid - 1 : k;
                __builtin_memcpy(&reg[i], first + (uint32_t)((back ? valid - 1 - k : k) * (int)ld + col), 16);
            }
        }
    }
    __device__ void store(T* tile, int shift) {
        if (shift) {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (row + i * kStep < shift) reg[i] = u32x4{0, 0, 0, 0};
        }
        if (!in) return;
        T* const to = tile + row * kStride + place;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (ROWS % kStep == 0 || row + i * kStep < ROWS) {
                if constexpr (WHOLE)
                    *reinterpret_cast<u32x4*>(to + i * kStep * kStride) = reg[i];
                else
                    __builtin_memcpy(to + i * kStep * kStride, &reg[i], 16);
            }
    }
    // after store(): whether a value that was stored is not finite
    __device__ bool bad() const {
        if constexpr (sizeof(T) == 2) {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            u16x2 most = {0, 0};  // of the exponents
#pragma unroll
            for (int i = 0; i < kEach; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, reg[i][k] & 0x7f807f80u));
            return in && (most[0] == 0x7f80 || most[1] == 0x7f80);
        } else {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) most = max(most, reg[i][k] & 0x7f800000u);
            return in && most == 0x7f800000u;
        }
    }
};

template <typename T> constexpr int kPParts = sizeof(T) == 2 ? 2 : 1;
// waves to a SIMD that a kernel's LDS leaves room for, as its register bound
template <typename T, int MP, int NW, bool OUT> constexpr int kOccupancy = !OUT ? (MP > 128 ? 2 : 3) : MP > 192 ? (NW == 8 ? 2 : 1) : NW == 8 ? 2 : MP > 64 ? 2 : sizeof(T) == 4 ? 4 : 3;

// One segment of one (sequence, head) through NW waves, 16 columns of the output to each; MP >= m channels of a and b, C tokens
// a chunk. OUT: outputs, of type TO; else only the state that the segment gives from a zero state. A segment's last chunk that
// is not whole stands at its tile's end, zeros before it, where its weights are a whole chunk's.
// A wave keeps 16 columns of the state in accumulators, whose layout (rows 4u.. of a column) is the matrix instruction's operand as it is,
// so the state never passes through LDS. bf16 operands that are formed in fp32 go in as two bf16 parts (scores and the state before a
// chunk, 2^-17 of the value, below an output's rounding) or three (what a chunk adds to the state, which is carried on): one part's
// 2^-9 would show. Chunks of 64 bf16 or 32 fp32 tokens: the scores' share grows with the chunk, the state's falls.
// What bounds it: memory at some 4 TB/s (reading more than writing) for heads of 64 channels, the issue of matrix and LDS instructions of
// its few waves a SIMD for wider ones. 1 x 65536 x 16 x 64 fp32, 1074 MB: segments' states 126-149 us (537 MB), outputs 315-348; 8 x 2048 x 16 x 64
// bf16: 19 and 40, its three gradients 94.
template <typename T, int MP, int C, int NW, bool WHOLE, bool OUT, typename TO>
__global__ __launch_bounds__(64 * NW, (kOccupancy<T, MP, NW, OUT>)) void mix_kernel(const MixPasses all) {
    constexpr int THREADS = 64 * NW, MT = MP / 16, NT = C / 16, KB = C / 32, E = 16 / sizeof(T);
    using TileM = Tile<T, C, MP, THREADS, WHOLE>;
    using TileN = Tile<T, C, 16 * NW, THREADS, WHOLE>;
    constexpr int PS = C + E;  // stride of the scores
    extern __shared__ __align__(16) char lds[];
    T* const tb = (T*)lds;
    T* const tc = (T*)(lds + TileM::kBytes);
    T* const ta = (T*)(lds + TileM::kBytes + TileN::kBytes);
    T* const tp = (T*)(lds + 2 * TileM::kBytes + TileN::kBytes);
    __shared__ int bad_rows[2];  // whether c's tile holds values that are not finite, this chunk's and the next one's
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, u = lane >> 4;

    // Consecutive blocks go to different dies. A die takes all heads of its segments, whose rows are neighbours in memory (a head's own
    // rows stand a whole token apart, which meets few of an L2's channels: 1 x 65536 x 16 x 64 fp32 343 -> 315 us), and passes and
    // slices of a head one after the other.
    const uint32_t inner = (uint32_t)(all.count * all.slices), heads = (uint32_t)all.p[0].H, groups = gridDim.x / (inner * heads);
    const uint32_t dies = groups % 8 == 0 ? 8 : groups % 4 == 0 ? 4 : groups % 2 == 0 ? 2 : 1, die = blockIdx.x % dies;
    uint32_t id = blockIdx.x / dies;
    const uint32_t which = id % inner;
    id /= inner;
    const MixArgs& p = all.p[which / (uint32_t)all.slices];
    const int slice = (int)(which % (uint32_t)all.slices);
    const int h = (int)(id % heads);
    id = id / heads * dies + die;
    const int seg = (int)(id % (uint32_t)p.nseg);
    const int64_t b = all.b0 + id / (uint32_t)p.nseg;
    int64_t len = p.L;
    if (p.lengths) {
        const int64_t given = p.lengths[b];
        len = given < 0 ? 0 : given < len ? given : len;
    }
    const int n0 = slice * 16 * NW;
    const int64_t t0 = seg * p.seglen, t1 = t0 + p.seglen < p.L ? t0 + p.seglen : p.L;
    const int64_t end = t1 < len ? t1 : len;
    const bool back = p.back != 0;

    // token t of the pass is token len - 1 - t of the sequence where it goes backwards
    TileM ra, rb;
    TileN rc;
    ra.begin(0, p.m);
    rb.begin(0, p.m);
    rc.begin(n0, p.n);
    const T* const pa = (const T*)p.a + b * p.L * p.lda + h / p.ga * p.m;
    const T* const pb = (const T*)p.b + b * p.L * p.ldb + h / p.gb * p.m;
    const T* const pc = (const T*)p.c + b * p.L * p.ldc + h / p.gc * p.n;
    const auto load = [&](int64_t t) {
        const int shift = end - t < C ? (int)(C - (end - t)) : 0;
        const int64_t first = back ? len - t - (C - shift) : t;  // the chunk's lowest token
        rb.load(pb + first * p.ldb, p.ldb, shift, back);
        rc.load(pc + first * p.ldc, p.ldc, shift, back);
        if constexpr (OUT) ra.load(pa + first * p.lda, p.lda, shift, back);
    };
    if (t0 < end) load(t0);

    // Columns behind a row's end stay zero, and so do the score tiles above the diagonal that a product over 32 tokens meets.
    if (!WHOLE || p.m < MP || p.n - n0 < 16 * NW) {
        constexpr int kTiles = (OUT ? 2 : 1) * TileM::kBytes + TileN::kBytes;
        for (int i = threadIdx.x; i < kTiles / 16; i += THREADS) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    }
    if constexpr (OUT) {
        for (int i = threadIdx.x; i < kPParts<T> * (NT / 2) * 256; i += THREADS) {
            const int row = i / 16 % 16, t = i / 256 % (NT / 2) * 32, part = i / (NT / 2 * 256);
            tp[part * C * PS + (t + row) * PS + t + 16 + i % 16] = 0;
        }
    }
    const float g = p.log_decay[h], l2 = log2_decay(g);

    // S[mt]: rows 16 mt + 4u..+3 of the state's column n0 + 16 wave + r
    const int64_t state_at = (b * p.H + h) * p.state;
    const int col = n0 + 16 * wave + r, col_in = (col < p.n ? col : p.n - 1) * p.sn;
    f32x4 S[MT];
    const auto each = [&](const float* from, const auto& take) {  // a state's part of this lane, 16 rows at a time
        from += col_in;
        const bool down = p.sm == 1 && p.m % 4 == 0;  // rows are neighbours
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            f32x4 x;
            const int row = 16 * mt + 4 * u;
            if (down) {
                __builtin_memcpy(&x, from + (row < p.m ? row : p.m - 4), 16);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = from[(row + e < p.m ? row + e : p.m - 1) * p.sm];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = row + e < p.m && col < p.n ? x[e] : 0.0f;
            take(mt, x);
        }
    };
    const float* const first = !OUT ? nullptr : p.chained ? p.parts + state_at * p.nseg + seg * p.state : p.init ? p.init + state_at : nullptr;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) S[mt] = f32x4{0, 0, 0, 0};
    if (first) each(first, [&](int mt, const f32x4& x) { S[mt] = x; });
    if (OUT && !p.chained) {  // few segments: those before this one, in turn
        const Decay whole(g, (float)p.seglen);
#pragma unroll 1
        for (int k = 0; k < seg; ++k) {
            const int64_t there = len - k * p.seglen;
            if (there <= 0) break;
            const Decay decay = there >= p.seglen ? whole : Decay(g, (float)there);
            each(p.parts + state_at * p.nseg + k * p.state, [&](int mt, const f32x4& x) {
#pragma unroll
                for (int e = 0; e < 4; ++e) S[mt][e] = decay(S[mt][e], x[e]);
            });
        }
    }
    float* const ends = !OUT ? p.parts + state_at * p.nseg + seg * p.state : seg == p.nseg - 1 && p.last ? p.last + state_at : nullptr;

    // Weights of a lane's places: scores on and off the diagonal, tokens' part of the state, the state's part of outputs. The last
    // and the state's decay are another chunk's only where that is not whole.
    float near[4], off[4], left[KB * 8], entry[NT];
    Decay decay(g, (float)C);
#pragma unroll
    for (int it = 0; it < NT; ++it) entry[it] = p.es * power(l2, 16 * it + r + p.e0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = r - 4 * u - e;
        near[e] = p.ps * power(l2, d < 0 ? 0 : d);
        off[e] = p.ps * power(l2, 16 + d);
    }
#pragma unroll
    for (int i = 0; i < KB * 8; ++i) left[i] = p.cs * power(l2, C - (32 * (i / 8) + 8 * u + i % 8) - p.e0);

    // places of a lane's fragments in the tiles
    const int row_m = r * TileM::kStride + 8 * u, pair_m = r * TileM::kStride + 4 * u, row_p = r * PS + 8 * u;
    const T* const col_b = tb + col_at<T, TileM::kStride>(r, u);
    const T* const col_c = tc + col_at<T, TileN::kStride>(r, u) + 16 * wave;
    const int more = p.n - n0 - 16 * wave - 4 * u;  // columns from this lane's first of the output on
    TO* const po = (TO*)p.out + b * p.L * p.ldo + (int64_t)h * p.n + n0 + 16 * wave;

    if (threadIdx.x == 0) bad_rows[0] = 0;
    int turn = 0;
#pragma unroll 1
    for (int64_t t = t0; t < end; t += C, turn ^= 1) {
        const int shift = end - t < C ? (int)(C - (end - t)) : 0;
        if (shift) {
            decay = Decay(g, (float)(C - shift));
#pragma unroll
            for (int it = 0; it < NT; ++it) {
                const int i = 16 * it + r - shift;
                entry[it] = p.es * power(l2, (i < 0 ? 0 : i) + p.e0);
            }
        }
        lds_barrier();  // the last chunk's tiles are read
        if (threadIdx.x == 0) bad_rows[turn ^ 1] = 0;
        rb.store(tb, shift);
        rc.store(tc, shift);
        if constexpr (OUT) {
            ra.store(ta, shift);
            if (rc.bad()) bad_rows[turn] = 1;
        }
        if (t + C < end) load(t + C);
        lds_barrier();
        f32x4 O[NT];
        if constexpr (OUT) {
            // scores: rows j of b against rows i of a, tiles on and below the diagonal
#pragma unroll
            for (int n = 0; n < (NT * (NT + 1) / 2 + NW - 1) / NW; ++n) {
                const int job = wave + n * NW;
                if (job >= NT * (NT + 1) / 2) break;
                const int it = job < 1 ? 0 : job < 3 ? 1 : job < 6 ? 2 : 3, jt = job - it * (it + 1) / 2;
                f32x4 s = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < MP / 32; ++k)
                    s = mma(s, row_frag(tb + 16 * jt * TileM::kStride + row_m + 32 * k), row_frag(ta + 16 * it * TileM::kStride + row_m + 32 * k));
                const float far = power(l2, 16 * (it > jt ? it - jt - 1 : 0));
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = s[e] * (it == jt ? near[e] : off[e] * far);
                    x[e] = it > jt || r >= 4 * u + e ? x[e] : 0.0f;
                }
                T* const to = tp + (16 * it + r) * PS + 16 * jt + 4 * u;
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
                } else {
                    const uint32_t h0 = pack_bf16x2(x[0], x[1]), h1 = pack_bf16x2(x[2], x[3]);
                    *reinterpret_cast<uint2*>(to) = make_uint2(h0, h1);
                    *reinterpret_cast<uint2*>(to + C * PS) =
                        make_uint2(pack_bf16x2(x[0] - __uint_as_float(h0 << 16), x[1] - __uint_as_float(h0 & 0xffff0000u)),
                                   pack_bf16x2(x[2] - __uint_as_float(h1 << 16), x[3] - __uint_as_float(h1 & 0xffff0000u)));
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            // what came before the chunk, through the state
#pragma unroll
            for (int it = 0; it < NT; ++it) O[it] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < MT / 2; ++k) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = S[2 * k + e / 4][e % 4];
                const Split<T, 2> s(x);
#pragma unroll
                for (int it = 0; it < NT; ++it) {
                    const Frag<T> a = pair_frag(ta + 16 * it * TileM::kStride + pair_m + 32 * k);
#pragma unroll
                    for (int q = 0; q < s.kParts; ++q) O[it] = mma(O[it], s.p[q], a);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int it = 0; it < NT; ++it)
#pragma unroll
                for (int e = 0; e < 4; ++e) O[it][e] *= entry[it];
            lds_barrier();  // the scores are there
        }
        Frag<T> c[KB];
#pragma unroll
        for (int k = 0; k < KB; ++k) c[k] = col_frag<TileN::kStride>(col_c + 32 * k * TileN::kStride);
        if constexpr (OUT) {
            // A masked score does not cancel what is not finite: such values are left out here and added by themselves below.
            const bool bad = bad_rows[turn];
            if (bad) {
#pragma unroll
                for (int k = 0; k < KB; ++k) c[k] = finite_only(c[k]);
            }
#pragma unroll
            for (int it = 0; it < NT; ++it)
#pragma unroll
                for (int k = 0; k <= it / 2; ++k)
#pragma unroll
                    for (int q = 0; q < kPParts<T>; ++q) O[it] = mma(O[it], c[k], row_frag(tp + q * C * PS + 16 * it * PS + row_p + 32 * k));
            if (bad) {
#pragma unroll 1
                for (int j = shift; j < C; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = Storage<T>::load(tc + j * TileN::kStride + 16 * wave + 4 * u + e);
                        if (not_finite(v)) {
#pragma unroll
                            for (int it = 0; it < NT; ++it) {
                                float s = Storage<T>::load(tp + (16 * it + r) * PS + j);
                                if constexpr (sizeof(T) == 2) s += Storage<T>::load(tp + C * PS + (16 * it + r) * PS + j);
                                if (16 * it + r >= j) O[it][e] += s * v;
                            }
                        }
                    }
#pragma unroll
                for (int k = 0; k < KB; ++k) c[k] = col_frag<TileN::kStride>(col_c + 32 * k * TileN::kStride);
            }
            __builtin_amdgcn_sched_barrier(0);
            // rows 4u..+3 of the wave's columns, row 16 it + r of the tile
            TO* const first = po + (back ? len - t - (C - shift) : t) * p.ldo;  // the chunk's lowest token
#pragma unroll
            for (int it = 0; it < NT; ++it) {
                const int i = 16 * it + r - shift;
                TO* const to = first + (uint32_t)((back ? C - shift - 1 - i : i) * (int)p.ldo + 4 * u);
                if (i < 0 || more <= 0) continue;
                if (WHOLE || more >= 4) {
                    if constexpr (sizeof(TO) == 4) {
                        __builtin_memcpy(to, &O[it], 16);
                    } else {
                        // hidden from the compiler, which else carries all tiles through wide vectors (168 registers and 496 bytes spilled
                        // for 143 and none)
                        float x[4] = {O[it][0], O[it][1], O[it][2], O[it][3]};
                        asm("" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
                        const uint2 w = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
                        __builtin_memcpy(to, &w, 8);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (e < more) Storage<TO>::store(to + e, O[it][e]);
                }
            }
        }
        // The state after the chunk: the chunk's part is summed by itself, so that the state is rounded once a chunk.
        if (ends || t + C < end) {
            Split<T, 3> v[KB];
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = value(c[k], e) * left[8 * k + e];
                v[k] = Split<T, 3>(x);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                f32x4 s = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const Frag<T> a = col_frag<TileM::kStride>(col_b + 32 * k * TileM::kStride + 16 * mt);
#pragma unroll
                    for (int q = 0; q < v[k].kParts; ++q) s = mma(s, a, v[k].p[q]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) S[mt][e] = decay(S[mt][e], s[e]);
                if (mt % 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (ends && col < p.n) {
        float* const to = ends + col_in;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * mt + 4 * u + e;
                if (row < p.m) to[row * p.sm] = S[mt][e];
            }
    }
    if constexpr (OUT) {  // rows behind a sequence's length
        const int64_t behind = t0 > end ? t0 : end;
        const int cols = p.n - n0 < 16 * NW ? p.n - n0 : 16 * NW;
        TO* const to = (TO*)p.out + b * p.L * p.ldo + (int64_t)h * p.n + n0;
        for (int64_t i = threadIdx.x; i < (t1 - behind) * cols; i += THREADS) Storage<TO>::store(to + (behind + i / cols) * p.ldo + i % cols, 0.0f);
    }
}

// Many segments' parts to the states before them, in place: of one or two passes. A thread has one element of the state, eight segments'
// loads on their way at once. Each state is read and written once: 64 x 8 x 256 x 256 fp32 for two passes 63 us, 4.3 TB/s; some 4 us at least.
struct ChainArgs {
    const float* init[2];
    float* parts[2];
};
__global__ __launch_bounds__(256) void chain_kernel(int64_t H, int64_t L, int64_t seglen, int nseg, int64_t state, const float* __restrict__ log_decay,
                                                    const int32_t* __restrict__ lengths, const ChainArgs passes) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= state) return;
    const int64_t bh = blockIdx.y, b = bh / H;
    int64_t len = L;
    if (lengths) {
        const int64_t given = lengths[b];
        len = given < 0 ? 0 : given < L ? given : L;
    }
    const float g = log_decay[bh % H];
    const float* const init = passes.init[blockIdx.z];
    float cur = init ? init[bh * state + i] : 0.0f;
    float* at = passes.parts[blockIdx.z] + bh * nseg * state + i;
    const Decay whole(g, (float)seglen);
    constexpr int kAhead = 8;  // segments whose parts are on their way at once
    for (int s0 = 0; s0 < nseg; s0 += kAhead, at += kAhead * state) {
        float e[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) e[k] = s0 + k < nseg ? at[k * state] : 0.0f;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (s0 + k >= nseg) break;
            at[k * state] = cur;
            const int64_t left = len - (s0 + k) * seglen;
            if (left >= seglen)
                cur = whole(cur, e[k]);
            else if (left > 0)
                cur = Decay(g, (float)left)(cur, e[k]);
        }
    }
}

// y[row][h][c] = sum over the heads of a group of x, in their order, rounded once; V neighbouring columns a thread. 65536 rows of 16
// heads x 128 to one: 537 MB in 96-108 us (5.0-5.6 TB/s).
template <typename T, int V>
__global__ __launch_bounds__(256) void group_sum_kernel(int64_t total, int group, int n, const float* __restrict__ x, T* __restrict__ y) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < total; i += (int64_t)gridDim.x * 256 * V) {
        const int64_t rh = (uint64_t)i / (uint32_t)n;
        const float* at = x + rh * (group - 1) * n + i;
        Run<V, float> s = Run<V, float>::load(at);
#pragma unroll 4
        for (int k = 1; k < group; ++k) {
            const Run<V, float> o = Run<V, float>::load(at + (int64_t)k * n);
#pragma unroll
            for (int e = 0; e < V; ++e) s.v[e] += o.v[e];
        }
        Run<V, T> r;
#pragma unroll
        for (int e = 0; e < V; ++e) Storage<T>::store(&r.v[e], s.v[e]);
        r.store(y + i);
    }
}

// ------------------------------------------------------------------ one token
// S = e^g S + k v^T, out = scale q S: a state is read and written once. A block takes 64 columns of one (sequence, head): 16
// threads hold four columns each of a row, 16 rows at a time; the rows' parts of q S are joined in LDS in a fixed order.
// Memory bounds it: 256 x 16 x 128 x 64, 268 MB, 42 us (6.4 TB/s). Columns that do not fill a block's 64 leave its threads idle: 128 x 16
// 17.6 (67 MB, 3.8 TB/s), 128 x 66 63 (4.4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void step_kernel(int64_t H, int dk, int dv, int gq, int gk, int gv, float* __restrict__ state,
                                                   const T* __restrict__ q, int64_t ldq, const T* __restrict__ k, int64_t ldk,
                                                   const T* __restrict__ v, int64_t ldv, const float* __restrict__ log_decay, float scale,
                                                   T* __restrict__ out) {
    const int64_t bh = blockIdx.x, b = bh / H, h = bh % H;
    const int c0 = blockIdx.y * 64 + threadIdx.x % 16 * 4, row = threadIdx.x / 16;
    const T *pq = q + b * ldq + h / gq * dk, *pk = k + b * ldk + h / gk * dk, *pv = v + b * ldv + h / gv * dv;
    const Decay decay(log_decay[h], 1.0f);
    const int left = dv - c0;
    float vv[4], sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) vv[e] = e < left ? Storage<T>::load(pv + c0 + e) : 0.0f;
    float* s = state + bh * dk * dv + c0;
    for (int m = row; m < dk; m += 16) {
        const float qm = Storage<T>::load(pq + m), km = Storage<T>::load(pk + m);
        float* at = s + (int64_t)m * dv;
        if (left >= 4) {
            f32x4 x;
            __builtin_memcpy(&x, at, 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = decay(x[e], km * vv[e]);
                sum[e] = fmaf(qm, x[e], sum[e]);
            }
            __builtin_memcpy(at, &x, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < left) {
                    at[e] = decay(at[e], km * vv[e]);
                    sum[e] = fmaf(qm, at[e], sum[e]);
                }
        }
    }
    __shared__ float part[16][64];
#pragma unroll
    for (int e = 0; e < 4; ++e) part[row][threadIdx.x % 16 * 4 + e] = sum[e];
    __syncthreads();
    const int c = blockIdx.y * 64 + threadIdx.x;
    if (threadIdx.x < 64 && c < dv) {
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) y += part[i][threadIdx.x];
        Storage<T>::store(out + bh * dv + c, y * scale);
    }
}

// ------------------------------------------------------------------ host
constexpr int kMaxChannels = 256;
constexpr int64_t kMaxStride = 1 << 23;  // elements from one token to the next: a chunk's offsets take 32 bits
int chunk_of(int dtype) { return dtype == HX_BF16 ? 64 : 32; }

// Segments that a sequence is cut into where the (sequence, head) pairs leave compute units idle: as many blocks as are
// resident at once, each of two chunks at least, and fewer of large states, which are written and read again for every one. Blocks aimed at,
// in us:
//   64 x 64 channels                   256   512   768  1024  2048
//   fp32 forward   1 x 65536 x 16      649   440   417   397   409      1 x 16384 x 8    86    71    75    77   100
//   fp32 backward  1 x 65536 x 16     1035  1004  1031  1010  1016      8 x 2048 x 16   265   257   284   277   295
//   bf16 forward   1 x 65536 x 16      333   206   208   216   223      8 x 2048 x 16    81    55    54    68    75
//   bf16 backward  1 x 65536 x 16      471   477   480   475   497      8 x 2048 x 16   105   113   125   143   156
// so 1024, 768 and 512 stand where the long sequences take them; a few percent are left at shorter ones, most at a single head (1 x 131072 x
// 1: fp32 forward 172 for 109 with 256). Training, wider heads, 128, 256 and 512 blocks: 1 x 65536 x 16 x 128/64 bf16 (q, k shared) 2342,
// 1598 and 1268; 1 x 16384 x 8 bf16 x 80 295, 249 and 269, x 96 298, 253 and 277, x 128 304, 265 and 301, x 192 682, 662 and 736, x 200 768, 844
// and 983, x 256 822, 899 and 1061. The rule goes by a state's elements: 512 up to 8192, 256 up to 40960 (192 x 192 are
// 36864; 200 x 200, 40000, would do better with 128, as every tile of more than 192 channels does), 128 beyond.
int64_t segments_of(int64_t B, int64_t L, int64_t H, int64_t dk, int64_t dv, int dtype, bool backward, int64_t* seglen) {
    const int64_t C = chunk_of(dtype), chunks = (L + C - 1) / C, pairs = B * H, wide = dk > dv ? dk : dv;
    const int64_t area = dk * dv, large = area <= 8192 ? 512 : area <= 40960 ? 256 : 128;
    const int64_t target = wide > 64 ? large : dtype == HX_F32 ? 1024 : backward ? 512 : 768;
    int64_t want = pairs > 0 ? target / pairs : 1;
    const int64_t most = chunks / 2;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t per = (chunks + want - 1) / want;
    *seglen = (per > 0 ? per : 1) * C;
    const int64_t nseg = chunks > 0 ? (chunks + per - 1) / per : 1;
    return nseg >= 8 ? (nseg + 7) / 8 * 8 : nseg;  // whole rounds of dies, the last ones perhaps without tokens
}
// Up to this many, an output's block goes through the segments before it by itself, which saves the chain's launch but reads a part
// after the other: fewer of large states (training at 2 x 520 x 1 x 168/58 fp32, six segments, 159 us so and 103 chained; 6 x 2048 x 16
// x 128/64 bf16, five, 278 and 285). Not where the last one's state takes the first one's buffer, which another block may yet read.
int64_t few_segments(int64_t dk, int64_t dv) {
    const int64_t few = 40960 / (dk * dv);
    return few < 8 ? few : 8;
}

struct Shape {
    int64_t B, L, H, hq, hk, hv, dk, dv;
    int dtype;
};

int check_shape(const char* what, const Shape& s) {
    HX_REQUIRE(s.B >= 0 && s.L >= 0 && s.H >= 0 && s.hq >= 0 && s.hk >= 0 && s.hv >= 0 && s.dk >= 0 && s.dv >= 0, HX_ERR_INVALID_DIMENSION,
               "%s: negative size", what);
    HX_REQUIRE(s.dtype == HX_F32 || s.dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "%s: dtype %d", what, s.dtype);
    if (s.H == 0) return HX_OK;
    HX_REQUIRE(s.hq > 0 && s.hk > 0 && s.hv > 0 && s.H % s.hq == 0 && s.H % s.hk == 0 && s.H % s.hv == 0, HX_ERR_SHAPE_MISMATCH,
               "%s: q, k and v need heads that divide %lld (%lld, %lld, %lld)", what, (long long)s.H, (long long)s.hq, (long long)s.hk, (long long)s.hv);
    HX_REQUIRE(s.H * (s.dk > s.dv ? s.dk : s.dv) < kMaxStride, HX_ERR_UNSUPPORTED, "%s: tokens of fewer than 2^23 elements", what);
    HX_REQUIRE(s.dk > 0 && s.dv > 0, HX_ERR_INVALID_DIMENSION, "%s: a head without channels", what);
    HX_REQUIRE(s.dk <= kMaxChannels && s.dv <= kMaxChannels, HX_ERR_UNSUPPORTED, "%s: at most %d channels a head", what, kMaxChannels);
    HX_REQUIRE(s.B < (1 << 24) && s.H < (1 << 16) && s.B * s.H < (1 << 24) && s.L < ((int64_t)1 << 40) / (s.B > 0 ? s.B : 1), HX_ERR_UNSUPPORTED,
               "%s: batch * heads below 2^24, heads below 2^16, batch * seqlen below 2^40", what);
    return HX_OK;
}

template <typename T, int MP, int NW, bool WHOLE, bool OUT, typename TO>
int launch_mix_of(MixPasses& a, hipStream_t stream) {
    constexpr int C = sizeof(T) == 2 ? 64 : 32;
    using TileM = Tile<T, C, MP, 64 * NW, WHOLE>;
    using TileN = Tile<T, C, 16 * NW, 64 * NW, WHOLE>;
    constexpr size_t bytes = (OUT ? 2 : 1) * TileM::kBytes + TileN::kBytes + (OUT ? kPParts<T> * C * (C + 16 / sizeof(T)) * sizeof(T) : 0);
    const auto k = mix_kernel<T, MP, C, NW, WHOLE, OUT, TO>;
    HX_REQUIRE(bytes <= 65536 || grant_dynamic_lds((const void*)k, bytes, 16), HX_ERR_BACKEND, "decay_attention: %zu bytes of LDS not granted", bytes);
    const MixArgs& p = a.p[0];
    a.slices = (p.n + 16 * NW - 1) / (16 * NW);
    // A launch holds fewer than 2^32 threads: many short sequences take several, whole sequences to each (one has fewer than 2^16 heads by
    // four slices by three passes, or, cut into segments, some thousand blocks).
    const int64_t each = p.H * p.nseg * a.slices * a.count, most = (((int64_t)1 << 32) / (64 * NW) - 1) / each;
    for (a.b0 = 0; a.b0 < p.B; a.b0 += most) {
        const int64_t count = p.B - a.b0 < most ? p.B - a.b0 : most;
        hipLaunchKernelGGL(k, dim3((unsigned)(count * each)), dim3(64 * NW), bytes, stream, a);
        HX_LAUNCH_CHECK();
    }
    return HX_OK;
}
template <typename T, bool WHOLE, bool OUT, typename TO>
int launch_mix_as(MixPasses& a, hipStream_t s) {
    const MixArgs& p = a.p[0];
    if (p.m <= 64) return launch_mix_of<T, 64, 4, WHOLE, OUT, TO>(a, s);
    if (p.m <= 128) return launch_mix_of<T, 128, 4, WHOLE, OUT, TO>(a, s);
    if (p.m <= 192) return launch_mix_of<T, 192, 4, WHOLE, OUT, TO>(a, s);
    // Eight waves share a tile of m > 192, whose memory leaves room for one block a CU. Training, four and eight waves: 1 x 16384 x 8 x 256 bf16
    // 1132 and 817, 1 x 4096 x 8 x 256 fp32 721 and 588; four do as well or better below: 1 x 16384 x 8 x 192 bf16 664 and 678, 1 x 4096 x
    // 8 x 192 fp32 415 and 502, 1 x 16384 x 8 x 128 bf16 265 and 280 (fp32, 4096 tokens, 205 and 200).
    if (p.n <= 64) return launch_mix_of<T, 256, 4, WHOLE, OUT, TO>(a, s);
    return launch_mix_of<T, 256, 8, WHOLE, OUT, TO>(a, s);
}
template <typename T, bool OUT, typename TO>
int launch_mix(MixPasses& a, hipStream_t s) {
    constexpr int E = 16 / sizeof(T);
    return a.p[0].m % E == 0 && a.p[0].n % E == 0 ? launch_mix_as<T, true, OUT, TO>(a, s) : launch_mix_as<T, false, OUT, TO>(a, s);
}

// What the segments of one or two passes give (b c^T each), and, where there are many, the states before them.
int segment_states(MixPasses a, int dtype, hipStream_t s) {
    const int rc = dtype == HX_F32 ? launch_mix<float, false, float>(a, s) : launch_mix<uint16_t, false, uint16_t>(a, s);
    if (rc != HX_OK || !a.p[0].chained) return rc;
    const MixArgs& p = a.p[0];
    HX_REQUIRE(p.B * p.H < 65536, HX_ERR_UNSUPPORTED, "decay_attention: batch * heads below 2^16 for segments");
    ChainArgs c{};
    for (int i = 0; i < a.count; ++i) c.init[i] = a.p[i].init, c.parts[i] = a.p[i].parts;
    const dim3 grid((unsigned)((p.state + 255) / 256), (unsigned)(p.B * p.H), (unsigned)a.count);
    hipLaunchKernelGGL(chain_kernel, grid, dim3(256), 0, s, p.H, p.L, p.seglen, p.nseg, p.state, p.log_decay, p.lengths, c);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

// The outputs of passes that have their sizes in common.
int outputs(MixPasses a, int dtype, bool out_f32, hipStream_t s) {
    if (dtype == HX_F32) return launch_mix<float, true, float>(a, s);
    return out_f32 ? launch_mix<uint16_t, true, float>(a, s) : launch_mix<uint16_t, true, uint16_t>(a, s);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

template <typename T>
int group_sum(int64_t rows, int64_t H, int64_t heads, int64_t n, const float* x, void* y, hipStream_t s) {
    const int64_t total = rows * heads * n, each = n % 4 == 0 ? 4 : 1, most = (int64_t)1 << 23, want = (total / each + 255) / 256;
    const int64_t blocks = want < most ? want : most;
    hipLaunchKernelGGL((each == 4 ? group_sum_kernel<T, 4> : group_sum_kernel<T, 1>), dim3((unsigned)blocks), dim3(256), 0, s, total, (int)(H / heads), (int)n, x, (T*)y);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

}  // namespace
}  // namespace hx

// bytes of the segments' states of one direction (0 where no sequence is cut)
static size_t hx_state_bytes(int64_t B, int64_t L, int64_t H, int64_t dk, int64_t dv, int dtype, bool backward) {
    int64_t seglen;
    const int64_t nseg = hx::segments_of(B, L, H, dk, dv, dtype, backward, &seglen);
    return nseg > 1 ? hx::round16((size_t)(B * H * nseg * dk * dv * 4)) : 0;
}

extern "C" size_t hx_decay_attention_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t dk, int64_t dv, int dtype) {
    using namespace hx;
    if (check_shape("decay_attention", {batch, seqlen, heads, heads, heads, heads, dk, dv, dtype}) != HX_OK) return 0;
    return batch == 0 || heads == 0 ? 0 : hx_state_bytes(batch, seqlen, heads, dk, dv, dtype, false);
}

extern "C" int hx_decay_attention_fwd(int64_t batch, int64_t seqlen, int64_t heads, int64_t q_heads, int64_t k_heads, int64_t v_heads, int64_t dk,
                                      int64_t dv, int dtype, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                      const float* log_decay, float scale, const int32_t* lengths, const float* init_state, void* out,
                                      float* last_state, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hx;
    const Shape s{batch, seqlen, heads, q_heads, k_heads, v_heads, dk, dv, dtype};
    int rc = check_shape("decay_attention_fwd", s);
    if (rc != HX_OK || batch == 0 || heads == 0) return rc;
    HX_REQUIRE(log_decay && (seqlen == 0 || (out && q && k && v)), HX_ERR_INVALID_INPUT, "decay_attention_fwd: NULL pointer");
    HX_REQUIRE(ldq >= q_heads * dk && ldk >= k_heads * dk && ldv >= v_heads * dv, HX_ERR_INVALID_INPUT, "decay_attention_fwd: a stride is shorter than a token");
    HX_REQUIRE(ldq < kMaxStride && ldk < kMaxStride && ldv < kMaxStride, HX_ERR_UNSUPPORTED, "decay_attention_fwd: strides below 2^23 elements");
    int64_t seglen;
    const int64_t nseg = segments_of(batch, seqlen, heads, dk, dv, dtype, false, &seglen);
    const size_t need = hx_state_bytes(batch, seqlen, heads, dk, dv, dtype, false);
    HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), HX_ERR_INVALID_INPUT,
               "decay_attention_fwd: workspace of %zu bytes (16-byte aligned) required", need);
    MixPasses all{};
    all.count = 1;
    MixArgs& p = all.p[0];
    p.a = q, p.b = k, p.c = v;
    p.lda = ldq, p.ldb = ldk, p.ldc = ldv;
    p.ga = (int)(heads / q_heads), p.gb = (int)(heads / k_heads), p.gc = (int)(heads / v_heads);
    p.B = batch, p.L = seqlen, p.H = heads;
    p.m = (int)dk, p.n = (int)dv;
    p.log_decay = log_decay, p.lengths = lengths;
    p.init = init_state, p.last = last_state, p.parts = (float*)workspace;
    p.chained = nseg > 1 && (nseg > few_segments(dk, dv) || (last_state && last_state == init_state));
    p.state = dk * dv, p.sm = (int)dv, p.sn = 1;
    p.ps = p.es = scale, p.cs = 1.0f, p.e0 = 1, p.back = 0;
    p.out = out, p.ldo = heads * dv;
    p.seglen = seglen, p.nseg = (int)nseg;
    if (nseg > 1) {
        rc = segment_states(all, dtype, as_stream(stream));
        if (rc != HX_OK) return rc;
    }
    return outputs(all, dtype, false, as_stream(stream));
}

// bytes of the fp32 gradients of an operand that heads share
static size_t hx_shared_bytes(int64_t rows, int64_t H, int64_t heads, int64_t n) { return heads == H ? 0 : hx::round16((size_t)(rows * H * n * 4)); }

extern "C" size_t hx_decay_attention_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t q_heads, int64_t k_heads,
                                                        int64_t v_heads, int64_t dk, int64_t dv, int dtype) {
    using namespace hx;
    if (check_shape("decay_attention_bwd", {batch, seqlen, heads, q_heads, k_heads, v_heads, dk, dv, dtype}) != HX_OK) return 0;
    if (batch == 0 || heads == 0) return 0;
    const int64_t rows = batch * seqlen;
    return 2 * hx_state_bytes(batch, seqlen, heads, dk, dv, dtype, true) + hx_shared_bytes(rows, heads, q_heads, dk) +
           hx_shared_bytes(rows, heads, k_heads, dk) + hx_shared_bytes(rows, heads, v_heads, dv);
}

extern "C" int hx_decay_attention_bwd(int64_t batch, int64_t seqlen, int64_t heads, int64_t q_heads, int64_t k_heads, int64_t v_heads, int64_t dk,
                                      int64_t dv, int dtype, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                      const float* log_decay, float scale, const int32_t* lengths, const float* init_state, const void* dout,
                                      const float* dlast, void* dq, void* dk_out, void* dv_out, float* dinit, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    using namespace hx;
    const Shape sh{batch, seqlen, heads, q_heads, k_heads, v_heads, dk, dv, dtype};
    int rc = check_shape("decay_attention_bwd", sh);
    if (rc != HX_OK || batch == 0 || heads == 0) return rc;
    HX_REQUIRE(log_decay && (seqlen == 0 || (q && k && v && dout && dq && dk_out && dv_out)), HX_ERR_INVALID_INPUT, "decay_attention_bwd: NULL pointer");
    HX_REQUIRE(ldq >= q_heads * dk && ldk >= k_heads * dk && ldv >= v_heads * dv, HX_ERR_INVALID_INPUT, "decay_attention_bwd: a stride is shorter than a token");
    HX_REQUIRE(ldq < kMaxStride && ldk < kMaxStride && ldv < kMaxStride, HX_ERR_UNSUPPORTED, "decay_attention_bwd: strides below 2^23 elements");
    const size_t need = hx_decay_attention_bwd_workspace_size(batch, seqlen, heads, q_heads, k_heads, v_heads, dk, dv, dtype);
    HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), HX_ERR_INVALID_INPUT,
               "decay_attention_bwd: workspace of %zu bytes (16-byte aligned) required", need);
    hipStream_t s = as_stream(stream);
    int64_t seglen;
    const int64_t nseg = segments_of(batch, seqlen, heads, dk, dv, dtype, true, &seglen), rows = batch * seqlen;
    const size_t state_bytes = hx_state_bytes(batch, seqlen, heads, dk, dv, dtype, true);
    char* at = (char*)workspace;
    float *const before = (float*)at, *const behind = (float*)(at + state_bytes);  // states before segments, their adjoints behind
    at += 2 * state_bytes;
    const int gq = (int)(heads / q_heads), gk = (int)(heads / k_heads), gv = (int)(heads / v_heads);
    struct Operand {
        const void* p;
        int64_t ld;
        int group;
    };
    const Operand Q{q, ldq, gq}, K{k, ldk, gk}, V{v, ldv, gv}, D{dout, heads * dv, 1};
    const bool in_place = dinit && (dinit == dlast || dinit == init_state), chained = nseg > 1 && (nseg > few_segments(dk, dv) || in_place);
    const auto mixing = [&](const Operand& a, const Operand& b, const Operand& c, bool transposed, bool back, float* last) {
        MixArgs p{};
        p.B = batch, p.L = seqlen, p.H = heads;
        p.log_decay = log_decay, p.lengths = lengths;
        p.init = back ? dlast : init_state, p.last = last, p.parts = back ? behind : before, p.chained = chained;
        p.state = dk * dv;
        p.seglen = seglen, p.nseg = (int)nseg;
        p.a = a.p, p.b = b.p, p.c = c.p, p.lda = a.ld, p.ldb = b.ld, p.ldc = c.ld, p.ga = a.group, p.gb = b.group, p.gc = c.group;
        p.m = (int)(transposed ? dv : dk), p.n = (int)(transposed ? dk : dv);
        p.sm = transposed ? 1 : (int)dv, p.sn = transposed ? (int)dv : 1;
        p.back = back, p.e0 = back ? 0 : 1;
        p.ps = scale, p.es = back ? 1.0f : scale, p.cs = back ? scale : 1.0f;
        return p;
    };
    if (nseg > 1) {
        MixPasses both{};
        both.count = 2;
        both.p[0] = mixing(Q, K, V, false, false, nullptr);
        both.p[1] = mixing(K, Q, D, false, true, nullptr);
        rc = segment_states(both, dtype, s);
        if (rc != HX_OK) return rc;
    }
    // dq, dk and dv as they are to be, or in 32 bits and head by head where heads share an operand. Passes with the same sizes
    // and type go out together; where dinit's buffer is dlast's or init_state's, the pass that writes it goes last.
    struct Gradient {
        MixArgs p;
        void* out;
        int64_t heads;
    };
    Gradient grads[3] = {{mixing(D, V, K, true, false, nullptr), dq, q_heads}, {mixing(V, D, Q, true, true, nullptr), dk_out, k_heads},
                         {mixing(K, Q, D, false, true, dinit), dv_out, v_heads}};
    bool wide[3];
    for (int i = 0; i < 3; ++i) {
        Gradient& x = grads[i];
        wide[i] = x.heads != heads;
        x.p.out = wide[i] ? (void*)at : x.out;
        x.p.ldo = heads * x.p.n;
        if (wide[i]) at += hx_shared_bytes(rows, heads, x.heads, x.p.n);
    }
    for (int i = 0; i < 3;) {
        MixPasses all{};
        int j = i;
        for (; j < 3 && grads[j].p.m == grads[i].p.m && grads[j].p.n == grads[i].p.n && wide[j] == wide[i] && !(j == 2 && j > i && in_place); ++j)
            all.p[all.count++] = grads[j].p;
        rc = outputs(all, dtype, wide[i], s);
        if (rc != HX_OK) return rc;
        i = j;
    }
    for (int i = 0; i < 3 && rows > 0; ++i)
        if (wide[i]) {
            const int64_t n = grads[i].p.n;
            rc = dtype == HX_F32 ? group_sum<float>(rows, heads, grads[i].heads, n, (const float*)grads[i].p.out, grads[i].out, s)
                                 : group_sum<uint16_t>(rows, heads, grads[i].heads, n, (const float*)grads[i].p.out, grads[i].out, s);
            if (rc != HX_OK) return rc;
        }
    return HX_OK;
}

extern "C" int hx_decay_attention_step(int64_t batch, int64_t heads, int64_t q_heads, int64_t k_heads, int64_t v_heads, int64_t dk, int64_t dv,
                                       int dtype, float* state, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                       const float* log_decay, float scale, void* out, void* stream) {
    using namespace hx;
    const Shape s{batch, 1, heads, q_heads, k_heads, v_heads, dk, dv, dtype};
    int rc = check_shape("decay_attention_step", s);
    if (rc != HX_OK || batch == 0 || heads == 0) return rc;
    HX_REQUIRE(log_decay && out && state && q && k && v, HX_ERR_INVALID_INPUT, "decay_attention_step: NULL pointer");
    HX_REQUIRE(ldq >= q_heads * dk && ldk >= k_heads * dk && ldv >= v_heads * dv, HX_ERR_INVALID_INPUT, "decay_attention_step: a stride is shorter than a token");
    HX_REQUIRE(ldq < kMaxStride && ldk < kMaxStride && ldv < kMaxStride, HX_ERR_UNSUPPORTED, "decay_attention_step: strides below 2^23 elements");
    const dim3 grid((unsigned)(batch * heads), (unsigned)((dv + 63) / 64));
    const int gq = (int)(heads / q_heads), gk = (int)(heads / k_heads), gv = (int)(heads / v_heads);
    if (dtype == HX_F32)
        hipLaunchKernelGGL(step_kernel<float>, grid, dim3(256), 0, as_stream(stream), heads, (int)dk, (int)dv, gq, gk, gv, state, (const float*)q, ldq,
                           (const float*)k, ldk, (const float*)v, ldv, log_decay, scale, (float*)out);
    else
        hipLaunchKernelGGL(step_kernel<uint16_t>, grid, dim3(256), 0, as_stream(stream), heads, (int)dk, (int)dv, gq, gk, gv, state, (const uint16_t*)q, ldq,
                           (const uint16_t*)k, ldk, (const uint16_t*)v, ldv, log_decay, scale, (uint16_t*)out);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
