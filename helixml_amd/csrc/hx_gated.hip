// hx_gated.hip — the gated linear recurrence with one state per channel: forward, backward, one token.
//   a = sigmoid(f), i = sigmoid(-f);  h_t = a_t h_{t-1} + i_t x_t;  out = h [silu(z)]
#include <type_traits>

#include "hx_common.h"

namespace hx {
namespace {

// Both gates from one exponential of -|f|, which is at most 1: neither overflows, and the smaller of
// the two is a product, so it keeps its relative accuracy where the other rounds to 1. A state's decay
// over n steps is a product of n gates, in which the reciprocal's error of up to an ulp, always to the
// same side for neighbouring values, would add up: one Newton step leaves that of the last rounding.
__device__ inline void gates(float f, float& a, float& i) {
    const float e = fast_exp2(-fabsf(f) * kLog2e);
    const float u = 1.0f + e, q = fast_rcp(u);
    const float r = fmaf(q, fmaf(-u, q, 1.0f), q), s = e * r;
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

// ------------------------------------------------------------------ tiles
// A block owns a tile of kTile steps x 64 channels of one sequence. Lane (half, c) of wave w holds channels
// 2c and 2c+1 of the S consecutive steps of part p = 2w + half, so a row of the tile is one 128-byte (bf16)
// or 256-byte (fp32) run and every element is read once and stays in registers. A part is the affine map
// h -> A h + H (A the product of its gates); the tile's parts are joined in LDS and the tiles of a sequence
// through the workspace (see Chain): a tile publishes its map as soon as it has it.
constexpr int kTile = HX_GATED_CHUNK, kWidth = 64;  // a tile's entry state is one of `states`
// Steps of a lane: as many as fit the registers of four waves a SIMD, since a tile of fewer waves has fewer parts to join
// and a CU holds more such tiles. bf16 forward 16 (tiles of 4 waves) against 8 (of 8): 1 x 65536 x 2048 184 us against 204
// ungated, 242 against 256 gated; 8 x 2048 x 1536 42 against 44, 51 against 53; one tile to a sequence, 3 x 124 x 899, 6.9
// against 5.9. With 16, fp32 spills: 348 us against 300 ungated at 1 x 65536 x 2048. The backward pass holds twice as much.
// (Registers for six waves a SIMD: fp32 with z spills 100 bytes a lane, 8 x 2048 x 1536 136 us against 87.)
template <typename T> constexpr int kForwardSteps = sizeof(T) == 2 ? 16 : 8;
constexpr int kBackwardSteps = 8;
template <int S> constexpr int kWaves = kTile / (2 * S);

// Two neighbouring channels as they are stored, at any address that an element may have: rows of odd width start anywhere.
template <typename T> struct Pair;
template <> struct Pair<float> {
    using raw = float2;
    __device__ static inline raw make(float a, float b) { return make_float2(a, b); }
    __device__ static inline float lo(raw r) { return r.x; }
    __device__ static inline float hi(raw r) { return r.y; }
    __device__ static inline raw pack(float a, float b) { return make_float2(a, b); }
    // Keeps the stored form in registers: what was computed from it before is not carried along to be used again.
    __device__ static inline void hold(raw& r) { asm("" : "+v"(r.x), "+v"(r.y)); }
};
template <> struct Pair<uint16_t> {
    using raw = uint32_t;
    __device__ static inline raw make(uint16_t a, uint16_t b) { return (uint32_t)b << 16 | a; }
    __device__ static inline float lo(raw r) { return __uint_as_float(r << 16); }
    __device__ static inline float hi(raw r) { return __uint_as_float(r & 0xffff0000u); }
    __device__ static inline raw pack(float a, float b) { return pack_bf16x2(a, b); }
    __device__ static inline void hold(raw& r) { asm("" : "+v"(r)); }
};

// Where a lane's elements lie. EVEN: an even number of channels, so that every pair is whole.
template <typename T, bool EVEN, int S>
struct Place {
    using raw = typename Pair<T>::raw;
    int64_t row;   // of the wave's first step, its first channel (uniform)
    int64_t D;
    uint32_t off;  // the lane's part and channel from there
    int steps;     // of this lane that lie inside the sequence, none for channels behind the last
    bool second;   // the pair's second channel exists

    __device__ Place(int64_t b, int64_t t0, int64_t c0, int wave, int lane, int64_t L, int64_t dim) : D(dim) {
        const int half = lane >> 5, c = (lane & 31) * 2;
        row = (b * L + t0 + wave * 2 * S) * D + c0;
        off = (uint32_t)(half * S * D + c);
        const int64_t left = L - t0 - (wave * 2 + half) * S;
        steps = c0 + c < D ? (int)(left < 0 ? 0 : left < S ? left : S) : 0;
        second = EVEN || c0 + c + 1 < D;
    }
    __device__ inline raw load(const T* base, int j) const {
        const T* p = base + (row + j * D);
        raw r;
        if (second)
            __builtin_memcpy(&r, p + off, sizeof(r));
        else
            r = Pair<T>::make(p[off], 0);
        return r;
    }
    __device__ inline void store(T* base, int j, float a, float b) const {
        T* p = base + (row + j * D);
        if (second) {
            const raw r = Pair<T>::pack(a, b);
            __builtin_memcpy(p + off, &r, sizeof(r));
        } else {
            Storage<T>::store(p + off, a);
        }
    }
    __device__ inline bool whole() const { return __all(steps == S); }  // the wave's rows are all there
    // All of the tile's loads of one operand, for the steps that exist.
    __device__ inline void load_all(const T* base, raw (&r)[S]) const {
        if (whole()) {
#pragma unroll
            for (int j = 0; j < S; ++j) r[j] = load(base, j);
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j) r[j] = j < steps ? load(base, j) : raw{};
        }
    }
};

// The workspace: tickets, then 64-bit words, all ones while there is nothing: one for each tile and channel, the tile's
// map (A, H); one for each group of kGroup tiles, the group's map, then its exit state (kExit, h). Each word is written
// whole and says itself what it is, so no fence is needed, only that readers and writers meet beyond the L2 of their XCD
// (agent scope).
//   entry of a tile  = the maps of the tiles before it in its group, applied in turn to the group's entry;
//   exit of a group  = the group's map (its tiles' maps joined in turn) applied to the group's entry;
//   entry of a group = the nearest exit that is there, and the maps of the groups after it applied in turn.
// What is applied to what does not depend on which words were there first, so neither do the bits.
struct Chain {
    uint32_t* tickets;
    unsigned long long *tiles_at, *groups_at;
    int tiles;       // of one sequence
    uint32_t lanes;  // sequences x column tiles
    uint32_t together;  // neighbouring columns that share a counter
};
constexpr unsigned long long kAbsent = ~0ull;
constexpr uint32_t kExit = 0xfffffffeu, kNaN = 0x7fc00000u;
constexpr int kGroup = 16;
// A wait ends by itself where the workspace is misused (two calls at once): some 10^5 looks of about a microsecond.
constexpr int kLooks = 1 << 17;

// The first word of row k (of tiles or groups) in a column: uniform, so that a lane's part of an address is its number.
__device__ inline unsigned long long* words_of(unsigned long long* words, const Chain& c, int k, uint32_t col) {
    return words + ((size_t)k * c.lanes + col) * kWidth;
}
__device__ inline void publish(unsigned long long* word, uint32_t lo, float hi) {
    __hip_atomic_store(word, (unsigned long long)__float_as_uint(hi) << 32 | lo, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void publish_map(unsigned long long* word, float A, float H) {
    const uint32_t u = __float_as_uint(A);
    publish(word, u >= kExit ? kNaN : u, H);  // no NaN passes for a tag
}
__device__ inline unsigned long long look_at(const unsigned long long* word) {
    return __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float map_a(unsigned long long m) { return __uint_as_float((uint32_t)m); }
__device__ inline float map_h(unsigned long long m) { return __uint_as_float((uint32_t)(m >> 32)); }

// What the block's waves have seen: the maps of the tiles before theirs in the group, the words of the W groups
// before it.
template <int W>
struct Looked {
    unsigned long long tiles[kGroup][kWidth], groups[W][kWidth];
    int found[W];
};
constexpr int kNoMap = 1, kGroupExit = 2, kGroupAbsent = 4;

// The state that tile k of a chain starts from, in wave 0's lanes; `first` is the chain's own, (A, H) the tile's map. The
// W waves look together, a share of the tiles and one group each: the maps of a group are all there about when the tile's own
// is, and a chain of many tiles moves on by W groups a look: 16384 steps, or 8192 in the bf16 forward, whose blocks have
// four waves (a window apart from the waves was not measured). 1 x 42983 x 70 bf16 takes 26 us; with a window of 8 tiles
// and an exit state for every tile it took 73.
template <int W>
__device__ inline float entry_of(const Chain& c, int k, uint32_t col, int wave, int lane, float first, float A, float H,
                                 Looked<W>& seen) {
    constexpr int kMine = kGroup / W;
    const int group = k / kGroup, place = k % kGroup;
    const bool closes = place == kGroup - 1 && k + 1 < c.tiles;
    if (wave == 0 && k + 1 < c.tiles) {
        // `first` has arrived before anyone can go on from this tile: the chain's last tile may write its place
        asm volatile("" : "+v"(first)::"memory");
        publish_map(words_of(c.tiles_at, c, k, col) + lane, A, H);
    }
    float GA = 1.0f, GH = 0.0f;
    bool mapped = false, ok = false, held = false;
    int start = -1;
    for (int look = 0; look < kLooks; ++look) {
        int found = 0;
        unsigned long long m[kMine], w = 0;
        const int from = group - W + wave;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (!held && wave * kMine + i < place) m[i] = look_at(words_of(c.tiles_at, c, k - place + wave * kMine + i, col) + lane);
        if (from >= 0) w = look_at(words_of(c.groups_at, c, from, col) + lane);
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (!held && wave * kMine + i < place) {
                if (__any(m[i] == kAbsent)) found = kNoMap;
                seen.tiles[wave * kMine + i][lane] = m[i];
            }
        held = found == 0;
        if (from >= 0) {
            if (__all((uint32_t)w == kExit)) found |= kGroupExit;
            if (__any(w == kAbsent)) found |= kGroupAbsent;
            seen.groups[wave][lane] = w;
        }
        if (lane == 0) seen.found[wave] = found;
        __syncthreads();
        int absent = -1;
        bool maps = true;
        start = -1;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int f = seen.found[i];
            maps = maps && !(f & kNoMap);
            if (f & kGroupExit) start = i;
            if (f & kGroupAbsent) absent = i;
        }
        if (maps && closes && !mapped) {
            mapped = true;
            if (wave == 0) {
#pragma unroll 4
                for (int i = 0; i < kGroup - 1; ++i) {
                    const unsigned long long t = seen.tiles[i][lane];
                    GH = fmaf(map_a(t), GH, map_h(t));
                    GA *= map_a(t);
                }
                GH = fmaf(A, GH, H);
                GA *= A;
                publish_map(words_of(c.groups_at, c, group, col) + lane, GA, GH);
            }
        }
        ok = maps && (start > absent || (absent < 0 && group <= W));  // or the look reaches the chain's start
        if (ok) break;
        __syncthreads();
        __builtin_amdgcn_s_sleep(1);
    }
    if (wave != 0) return 0.0f;
    float e = ok ? first : __uint_as_float(kNaN);
    if (ok)
        for (int i = start >= 0 ? start : W - (group < W ? group : W); i < W; ++i) {
            const unsigned long long g = seen.groups[i][lane];
            e = (uint32_t)g == kExit ? map_h(g) : fmaf(map_a(g), e, map_h(g));
        }
    if (closes) publish(words_of(c.groups_at, c, group, col) + lane, kExit, fmaf(GA, e, GH));
#pragma unroll 4
    for (int i = 0; i < place; ++i) {
        const unsigned long long t = seen.tiles[i][lane];
        e = fmaf(map_a(t), e, map_h(t));
    }
    return e;
}

// Which tile this block takes: tickets are handed out in the order in which blocks start, tile 0 of every column first, so
// what a block waits for is always held by a block that has started. Adding to one word takes the chip about 13.5 ns a
// block, all blocks in turn (1 x 65536 x 2048 bf16 took 227 us for it alone), so the columns are dealt in runs to up to
// kCounters words of lines of their own; a column's tiles all come from one of them. Runs of kTogether neighbours, since
// columns that drift apart share no DRAM page: 1 x 65536 x 2048 fp32 335 us with runs of one, 310 from four on; bf16 230,
// 208 with four, 204 with eight, 226 with all 32 columns on one word; 1 x 1999 x 768 11.5, 11.8, 12.2 and 12.9. Narrower
// sequences have their own: 4 x 25945 x 98 bf16 31 us, 41 with four sequences to a word; 15 x 3568 x 68 18.5 and 17.6.
constexpr uint32_t kCounters = 64, kCounterStride = 32, kTogether = 8;
__device__ inline bool take_unit(const Chain& c, uint32_t& shared_ticket, int& k, uint32_t& col) {
    const uint32_t unit = blockIdx.y * gridDim.x + blockIdx.x;
    k = (int)(unit / c.lanes);
    col = unit - (uint32_t)k * c.lanes;
    if (k >= c.tiles) return false;
    if (c.tiles > 1) {
        const uint32_t mine = col / c.together, first = mine * c.together;
        if (threadIdx.x == 0) shared_ticket = atomicAdd(c.tickets + mine * kCounterStride, 1u);
        __syncthreads();
        const uint32_t ticket = __builtin_amdgcn_readfirstlane(shared_ticket);
        const uint32_t columns = c.lanes - first < c.together ? c.lanes - first : c.together;
        k = (int)(ticket / columns);
        col = first + ticket - (uint32_t)k * columns;
    }
    return k < c.tiles;
}

struct FwdArgs {
    int64_t L, D;
    const void *x, *f, *z;
    const float* init;
    void* out;
    float *last, *states;
    uint32_t cols;  // column tiles of one sequence
    Chain chain;
};

template <typename T, bool EVEN, bool GATE>
__global__ __launch_bounds__(64 * kWaves<kForwardSteps<T>>, 4) void gated_fwd_kernel(const FwdArgs p) {
    constexpr int kSteps = kForwardSteps<T>, W = kWaves<kSteps>, kParts = 2 * W;
    __shared__ float2 maps[kParts][kWidth];
    __shared__ float entries[kParts][kWidth];
    __shared__ Looked<W> seen;
    __shared__ uint32_t shared_ticket;
    int k;
    uint32_t col;
    if (!take_unit(p.chain, shared_ticket, k, col)) return;
    const int64_t b = col / p.cols, c0 = (int64_t)(col - (uint32_t)b * p.cols) * kWidth;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Place<T, EVEN, kSteps> at(b, (int64_t)k * kTile, c0, wave, lane, p.L, p.D);
    typename Pair<T>::raw rf[kSteps], rx[kSteps], rz[kSteps];
    at.load_all((const T*)p.f, rf);
    at.load_all((const T*)p.x, rx);
    if (GATE) at.load_all((const T*)p.z, rz);

    float a0[kSteps], a1[kSteps], b0[kSteps], b1[kSteps];
    float A0 = 1.0f, A1 = 1.0f, H0 = 0.0f, H1 = 0.0f;
    const auto open = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float i0, i1;
            gates(Pair<T>::lo(rf[j]), a0[j], i0);
            gates(Pair<T>::hi(rf[j]), a1[j], i1);
            b0[j] = i0 * Pair<T>::lo(rx[j]);
            b1[j] = i1 * Pair<T>::hi(rx[j]);
            if (!decltype(whole)::value && j >= at.steps) {  // a step that is not there changes nothing
                a0[j] = a1[j] = 1.0f;
                b0[j] = b1[j] = 0.0f;
            }
            H0 = fmaf(a0[j], H0, b0[j]);
            H1 = fmaf(a1[j], H1, b1[j]);
            A0 *= a0[j];
            A1 *= a1[j];
        }
    };
    if (at.whole())
        open(std::true_type{});
    else
        open(std::false_type{});
    const int part = wave * 2 + (lane >> 5), c = (lane & 31) * 2;
    *reinterpret_cast<float4*>(&maps[part][c]) = make_float4(A0, H0, A1, H1);
    __syncthreads();
    const bool in = c0 + lane < p.D;
    const int64_t r = b * p.D + c0 + lane;
    float A = 1.0f, H = 0.0f, e = 0.0f;
    if (wave == 0) {
        if (in && p.init) e = p.init[r];
#pragma unroll 4
        for (int s = 0; s < kParts; ++s) {
            const float2 m = maps[s][lane];
            H = fmaf(m.x, H, m.y);
            A *= m.x;
        }
    }
    if (p.chain.tiles > 1) e = entry_of<W>(p.chain, k, col, wave, lane, e, A, H, seen);
    if (wave == 0) {
        if (in && p.states) p.states[(b * p.chain.tiles + k) * p.D + c0 + lane] = e;
        if (in && p.last && k + 1 == p.chain.tiles) p.last[r] = fmaf(A, e, H);
#pragma unroll 4
        for (int s = 0; s < kParts; ++s) {
            const float2 m = maps[s][lane];
            entries[s][lane] = e;
            e = fmaf(m.x, e, m.y);
        }
    }
    __syncthreads();
    const float2 start = *reinterpret_cast<const float2*>(&entries[part][c]);
    float h0 = start.x, h1 = start.y;
    if (GATE) {  // silu(z) is formed here, not carried through the wait
#pragma unroll
        for (int j = 0; j < kSteps; ++j) Pair<T>::hold(rz[j]);
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
        h0 = fmaf(a0[j], h0, b0[j]);
        h1 = fmaf(a1[j], h1, b1[j]);
        if (j < at.steps)
            at.store((T*)p.out, j, GATE ? h0 * silu(Pair<T>::lo(rz[j])) : h0, GATE ? h1 * silu(Pair<T>::hi(rz[j])) : h1);
    }
}

struct BwdArgs {
    int64_t L, D;
    const void *x, *f, *z, *dout;
    const float *states, *dlast;
    void *dx, *df, *dz;
    float* dinit;
    uint32_t cols;
    Chain chain;
};

// The tiles from the last one back. The carry c_t = a_t g_t obeys c_t = a_t c_{t+1} + a_t dh_t, so parts and tiles
// are affine maps again, with the same A. h is formed from `states` for the tile alone, without waiting.
template <typename T, bool EVEN, bool GATE>
__global__ __launch_bounds__(64 * kWaves<kBackwardSteps>, 4) void gated_bwd_kernel(const BwdArgs p) {
    constexpr int kSteps = kBackwardSteps, W = kWaves<kSteps>, kParts = 2 * W;
    __shared__ float maps_a[kParts][kWidth], maps_h[kParts][kWidth], maps_g[kParts][kWidth];
    __shared__ Looked<W> seen;
    __shared__ uint32_t shared_ticket;
    int k;
    uint32_t col;
    if (!take_unit(p.chain, shared_ticket, k, col)) return;
    const int tile = p.chain.tiles - 1 - k;
    const int64_t b = col / p.cols, c0 = (int64_t)(col - (uint32_t)b * p.cols) * kWidth;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Place<T, EVEN, kSteps> at(b, (int64_t)tile * kTile, c0, wave, lane, p.L, p.D);
    typename Pair<T>::raw rf[kSteps], rx[kSteps], rz[kSteps], rd[kSteps];
    at.load_all((const T*)p.f, rf);
    at.load_all((const T*)p.x, rx);
    at.load_all((const T*)p.dout, rd);
    if (GATE) at.load_all((const T*)p.z, rz);

    float a0[kSteps], a1[kSteps], i0[kSteps], i1[kSteps];
    float A0 = 1.0f, A1 = 1.0f, H0 = 0.0f, H1 = 0.0f, G0 = 0.0f, G1 = 0.0f;
    const auto open = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            gates(Pair<T>::lo(rf[j]), a0[j], i0[j]);
            gates(Pair<T>::hi(rf[j]), a1[j], i1[j]);
            if (!decltype(whole)::value && j >= at.steps) {
                a0[j] = a1[j] = 1.0f;
                i0[j] = i1[j] = 0.0f;
            }
            H0 = fmaf(a0[j], H0, i0[j] * Pair<T>::lo(rx[j]));
            H1 = fmaf(a1[j], H1, i1[j] * Pair<T>::hi(rx[j]));
            A0 *= a0[j];
            A1 *= a1[j];
        }
    };
    if (at.whole())
        open(std::true_type{});
    else
        open(std::false_type{});
#pragma unroll
    for (int j = kSteps - 1; j >= 0; --j) {
        float d0 = Pair<T>::lo(rd[j]), d1 = Pair<T>::hi(rd[j]);
        if (GATE) {
            d0 *= silu(Pair<T>::lo(rz[j]));
            d1 *= silu(Pair<T>::hi(rz[j]));
        }
        G0 = a0[j] * (G0 + d0);
        G1 = a1[j] * (G1 + d1);
    }
    const int part = wave * 2 + (lane >> 5), c = (lane & 31) * 2;
    *reinterpret_cast<float2*>(&maps_a[part][c]) = make_float2(A0, A1);
    *reinterpret_cast<float2*>(&maps_h[part][c]) = make_float2(H0, H1);
    *reinterpret_cast<float2*>(&maps_g[part][c]) = make_float2(G0, G1);
    __syncthreads();
    // Wave 0 joins the carries, wave 1 meanwhile the states; each leaves its parts' entry values where the maps were that
    // only it reads.
    const bool in = c0 + lane < p.D;
    const int64_t r = b * p.D + c0 + lane;
    float A = 1.0f, G = 0.0f, e = 0.0f;
    if (wave == 0) {
        if (in && p.dlast) e = p.dlast[r];
#pragma unroll 4
        for (int s = kParts - 1; s >= 0; --s) {
            const float m = maps_a[s][lane];
            G = fmaf(m, G, maps_g[s][lane]);
            A *= m;
        }
    } else if (wave == 1) {
        float h = in ? p.states[(b * p.chain.tiles + tile) * p.D + c0 + lane] : 0.0f;
#pragma unroll 4
        for (int s = 0; s < kParts; ++s) {
            const float m = maps_h[s][lane];
            maps_h[s][lane] = h;
            h = fmaf(maps_a[s][lane], h, m);
        }
    }
    if (p.chain.tiles > 1) e = entry_of<W>(p.chain, k, col, wave, lane, e, A, G, seen);
    if (wave == 0) {
        if (in && p.dinit && tile == 0) p.dinit[r] = fmaf(A, e, G);
#pragma unroll 4
        for (int s = kParts - 1; s >= 0; --s) {
            const float g = maps_g[s][lane];
            maps_g[s][lane] = e;
            e = fmaf(maps_a[s][lane], e, g);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
        Pair<T>::hold(rx[j]);
        Pair<T>::hold(rd[j]);
        if (GATE) Pair<T>::hold(rz[j]);
    }
    const float2 eh = *reinterpret_cast<const float2*>(&maps_h[part][c]);
    const float2 eg = *reinterpret_cast<const float2*>(&maps_g[part][c]);
    // dout and z were kept as stored, and silu(z) is formed again with its derivative: 32 registers less at the wait
    float h0[kSteps], h1[kSteps], d0[kSteps], d1[kSteps];  // the state before each step, dh
    float n0 = eh.x, n1 = eh.y;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
        h0[j] = n0;
        h1[j] = n1;
        n0 = fmaf(a0[j], n0, i0[j] * Pair<T>::lo(rx[j]));
        n1 = fmaf(a1[j], n1, i1[j] * Pair<T>::hi(rx[j]));
        d0[j] = Pair<T>::lo(rd[j]);
        d1[j] = Pair<T>::hi(rd[j]);
        if (GATE) {
            float v0, v1, s0, s1;
            silu_grad(Pair<T>::lo(rz[j]), v0, s0);
            silu_grad(Pair<T>::hi(rz[j]), v1, s1);
            if (j < at.steps) at.store((T*)p.dz, j, d0[j] * n0 * s0, d1[j] * n1 * s1);
            d0[j] *= v0;
            d1[j] *= v1;
        }
    }
    float g0 = eg.x, g1 = eg.y;
#pragma unroll
    for (int j = kSteps - 1; j >= 0; --j) {
        g0 += d0[j];
        g1 += d1[j];
        const float q0 = g0 * i0[j], q1 = g1 * i1[j];
        if (j < at.steps) {
            at.store((T*)p.dx, j, q0, q1);
            at.store((T*)p.df, j, q0 * a0[j] * (h0[j] - Pair<T>::lo(rx[j])), q1 * a1[j] * (h1[j] - Pair<T>::hi(rx[j])));
        }
        g0 *= a0[j];
        g1 *= a1[j];
    }
}

// Every word of the workspace absent, the tickets at their start.
constexpr size_t kTicketBytes = kCounters * kCounterStride * sizeof(uint32_t);
__global__ __launch_bounds__(256) void gated_chain_clear_kernel(uint4* ws, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const uint32_t v = i < (int64_t)(kTicketBytes / sizeof(uint4)) ? 0 : 0xffffffffu;
        ws[i] = make_uint4(v, v, v, v);
    }
}

// One token: four channels a thread (16 bytes of state), bound by the state's read and write; the last n % 4 channels
// one a thread. 256 x 4096 fp32: 5.2 us, one channel a thread 5.5.
template <typename T, int N>
__device__ inline void step_run(int64_t o, float* state, const T* x, const T* f, const T* z, T* out) {
    const Run<N, T> xv = Run<N, T>::load(x + o), fv = Run<N, T>::load(f + o);
    Run<N, T> zv, y;
    if (z) zv = Run<N, T>::load(z + o);
    Run<N, float> h = Run<N, float>::load(state + o);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        float a, i;
        gates(Storage<T>::load(&fv.v[e]), a, i);
        h.v[e] = fmaf(a, h.v[e], i * Storage<T>::load(&xv.v[e]));
        Storage<T>::store(&y.v[e], z ? h.v[e] * silu(Storage<T>::load(&zv.v[e])) : h.v[e]);
    }
    h.store(state + o);
    y.store(out + o);
}
template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(int64_t n, float* state, const T* x, const T* f, const T* z,
                                                         T* out) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, runs = n / 4;
    if (t < runs)
        step_run<T, 4>(4 * t, state, x, f, z, out);
    else if (t - runs < n - 4 * runs)
        step_run<T, 1>(4 * runs + (t - runs), state, x, f, z, out);
}

// dst = src, or zero: what is left of a sequence without steps. Both may be one buffer.
__global__ __launch_bounds__(256) void gated_state_copy_kernel(int64_t n, const float* src, float* dst) {
    for (int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x; o < n; o += (int64_t)gridDim.x * 256) dst[o] = src ? src[o] : 0.0f;
}

// A grid axis counts its threads in 32 bits: kernels over many elements loop, kernels over many tiles take two axes.
constexpr int64_t kMaxBlocks = 0x7fffffff, kAxis = 1 << 20;
inline dim3 looped(int64_t n) {
    const int64_t blocks = (n + 255) / 256;
    return dim3((unsigned)(blocks < kAxis ? blocks : kAxis));
}

struct Shape {
    int64_t batch, L, D, cols, tiles, units;
    Shape(int64_t batch_, int64_t L_, int64_t D_)
        : batch(batch_), L(L_), D(D_), cols(D_ / kWidth + (D_ % kWidth != 0)), tiles(L_ / kTile + (L_ % kTile != 0)),
          units(fits() ? batch_ * cols * tiles : 0) {}
    // Byte offsets of 63 bits, a lane's offset inside its wave's rows of 32, one block a tile.
    bool fits() const {
        return batch < kMaxBlocks && D < (1 << 26) && L < ((int64_t)1 << 37) &&
               (__int128)batch * cols * (tiles > 0 ? tiles : 1) < kMaxBlocks && (__int128)batch * L * D < ((__int128)1 << 60);
    }
    dim3 grid() const {
        const int64_t x = units < kAxis ? units : kAxis;
        return dim3((unsigned)x, (unsigned)((units + x - 1) / x));
    }
    int64_t together() const {
        const int64_t share = (batch * cols + kCounters - 1) / kCounters;
        const int64_t near = cols < kTogether ? cols : kTogether;
        return share > near ? share : near;
    }
    // The tickets, a word per channel of each tile and group; one tile waits for nobody
    int64_t groups() const { return (tiles + kGroup - 1) / kGroup; }
    size_t workspace() const { return tiles > 1 ? kTicketBytes + ((size_t)units + groups() * batch * cols) * kWidth * 8 : 0; }
    Chain chain(void* ws) const {
        unsigned long long* const words = (unsigned long long*)((char*)ws + kTicketBytes);
        return Chain{(uint32_t*)ws, words, words + (size_t)units * kWidth, (int)tiles, (uint32_t)(batch * cols),
                     (uint32_t)together()};
    }
};

int clear_chain(const Shape& g, void* ws, hipStream_t s) {
    if (g.tiles <= 1) return HX_OK;
    const int64_t n = (int64_t)(g.workspace() / 16);
    hipLaunchKernelGGL(gated_chain_clear_kernel, looped(n), dim3(256), 0, s, (uint4*)ws, n);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

int copy_state(int64_t rows, const float* src, float* dst, hipStream_t s) {
    if (!dst) return HX_OK;
    hipLaunchKernelGGL(gated_state_copy_kernel, looped(rows), dim3(256), 0, s, rows, src, dst);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

template <typename T>
int fwd(const Shape& g, const FwdArgs& p, hipStream_t s) {
    const auto k = g.D % 2 == 0 ? (p.z ? gated_fwd_kernel<T, true, true> : gated_fwd_kernel<T, true, false>)
                             : (p.z ? gated_fwd_kernel<T, false, true> : gated_fwd_kernel<T, false, false>);
    hipLaunchKernelGGL(k, g.grid(), dim3(64 * kWaves<kForwardSteps<T>>), 0, s, p);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

template <typename T>
int bwd(const Shape& g, const BwdArgs& p, hipStream_t s) {
    const auto k = g.D % 2 == 0 ? (p.z ? gated_bwd_kernel<T, true, true> : gated_bwd_kernel<T, true, false>)
                             : (p.z ? gated_bwd_kernel<T, false, true> : gated_bwd_kernel<T, false, false>);
    hipLaunchKernelGGL(k, g.grid(), dim3(64 * kWaves<kBackwardSteps>), 0, s, p);
    HX_LAUNCH_CHECK();
    return HX_OK;
}

size_t workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int dtype) {
    if (batch <= 0 || seqlen <= 0 || dim <= 0 || (dtype != HX_F32 && dtype != HX_BF16)) return 0;
    const Shape g(batch, seqlen, dim);
    return g.fits() ? g.workspace() : 0;
}

}  // namespace
}  // namespace hx

extern "C" size_t hx_gated_scan_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int dtype) {
    return hx::workspace_size(batch, seqlen, dim, dtype);
}
extern "C" size_t hx_gated_scan_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int dtype) {
    return hx::workspace_size(batch, seqlen, dim, dtype);
}

extern "C" int hx_gated_scan_fwd(int64_t batch, int64_t seqlen, int64_t dim, int dtype, const void* x, const void* f,
                                 const void* z, const float* init_state, void* out, float* last_state, float* states,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && seqlen >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "gated_scan: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "gated_scan: dtype %d", dtype);
    if (batch == 0 || dim == 0) return HX_OK;
    const Shape g(batch, seqlen, dim);
    HX_REQUIRE(g.fits(), HX_ERR_UNSUPPORTED, "gated_scan: too many elements");
    const size_t need = g.workspace();
    hipStream_t s = as_stream(stream);
    if (seqlen == 0) return copy_state(batch * dim, init_state, last_state, s);
    HX_REQUIRE(x && f && out, HX_ERR_INVALID_INPUT, "gated_scan: x, f and out are required");
    HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), HX_ERR_INVALID_INPUT,
               "gated_scan: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
    if (int rc = clear_chain(g, workspace, s)) return rc;
    const FwdArgs p{seqlen, dim, x, f, z, init_state, out, last_state, states, (uint32_t)g.cols, g.chain(workspace)};
    return dtype == HX_F32 ? fwd<float>(g, p, s) : fwd<uint16_t>(g, p, s);
}

extern "C" int hx_gated_scan_bwd(int64_t batch, int64_t seqlen, int64_t dim, int dtype, const void* x, const void* f,
                                 const void* z, const float* states, const void* dout, const float* dlast, void* dx,
                                 void* df, void* dz, float* dinit, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && seqlen >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "gated_scan_bwd: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "gated_scan_bwd: dtype %d", dtype);
    if (batch == 0 || dim == 0) return HX_OK;
    const Shape g(batch, seqlen, dim);
    HX_REQUIRE(g.fits(), HX_ERR_UNSUPPORTED, "gated_scan_bwd: too many elements");
    const size_t need = g.workspace();
    hipStream_t s = as_stream(stream);
    if (seqlen == 0) return copy_state(batch * dim, dlast, dinit, s);
    HX_REQUIRE(x && f && states && dout && dx && df, HX_ERR_INVALID_INPUT,
               "gated_scan_bwd: x, f, states, dout, dx and df are required");
    HX_REQUIRE((z == nullptr) == (dz == nullptr), HX_ERR_INVALID_INPUT, "gated_scan_bwd: dz goes with z");
    HX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), HX_ERR_INVALID_INPUT,
               "gated_scan_bwd: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
    if (int rc = clear_chain(g, workspace, s)) return rc;
    const BwdArgs p{seqlen, dim, x, f, z, dout, states, dlast, dx, df, dz, dinit, (uint32_t)g.cols, g.chain(workspace)};
    return dtype == HX_F32 ? bwd<float>(g, p, s) : bwd<uint16_t>(g, p, s);
}

extern "C" int hx_gated_state_update(int64_t batch, int64_t dim, int dtype, float* state, const void* x, const void* f,
                                     const void* z, void* out, void* stream) {
    using namespace hx;
    HX_REQUIRE(batch >= 0 && dim >= 0, HX_ERR_INVALID_DIMENSION, "gated_state_update: negative size");
    HX_REQUIRE(dtype == HX_F32 || dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "gated_state_update: dtype %d", dtype);
    if (batch == 0 || dim == 0) return HX_OK;
    HX_REQUIRE((__int128)batch * dim < ((__int128)1 << 33), HX_ERR_UNSUPPORTED, "gated_state_update: too many elements");
    HX_REQUIRE(state && x && f && out, HX_ERR_INVALID_INPUT, "gated_state_update: state, x, f and out are required");
    const int64_t n = batch * dim, threads = n / 4 + n % 4;
    dim3 grid((unsigned)((threads + 255) / 256));
    if (dtype == HX_F32)
        hipLaunchKernelGGL(gated_step_kernel<float>, grid, dim3(256), 0, as_stream(stream), n, state, (const float*)x,
                           (const float*)f, (const float*)z, (float*)out);
    else
        hipLaunchKernelGGL(gated_step_kernel<uint16_t>, grid, dim3(256), 0, as_stream(stream), n, state,
                           (const uint16_t*)x, (const uint16_t*)f, (const uint16_t*)z, (uint16_t*)out);
    HX_LAUNCH_CHECK();
    return HX_OK;
}
