// The steps around attention that move q, k and v rows: rotary positions (fa_rope), filling a KV cache
// with the rotation on the way (fa_cache_append) and reading a 4-bit cache back (fa_cache_read_u4).
//
// The reference has none of them: its programs start from Q, K and V (src/demo.cu:28-70).
//
// All three read every element once and write it once.  A row of D elements is covered by D / 8 lanes with one 16-byte
// access each, so that a warp's access is two (D = 128) or four whole rows.  A thread keeps to one token and walks heads, so
// cos and sin of its 8 elements are read once, from a table in shared memory that the block computes for its tokens: in 64
// bits, which costs 30 operations of the 64-bit pipe a pair and token, 2 for each 16 bytes moved.
#include <cmath>
#include <cuda_fp8.h>

#include "fast_div.h"
#include "host_common.h"
#include "ptx.cuh"
#include "u4.cuh"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kMaxPairs = 64;

// What a kernel gets of fa_rotary: each pair's turns per position as a 64-bit fraction of a turn.  position * turns modulo
// 2^64 is the exact fraction of a turn that the position has come to, for any 32-bit position: nothing is lost to
// the whole turns, which in 32-bit floating point cost far positions their angle (position 10^6: 0.06 rad).
struct Rotary {
    unsigned long long turns[kMaxPairs];
    double amplitude;
    float minus_zero[2];                 // both -0, known to the host alone (see F2)
    int dim;                             // elements that turn; 0: none
};

__device__ __forceinline__ void cos_sin(const Rotary& r, int position, int pair, bool inverse, float* c, float* s) {
    const long long frac = (long long)((unsigned long long)(long long)position * r.turns[pair]);   // of a turn, times 2^64
    double sd, cd;
    sincospi((double)frac * 0x1p-63, &sd, &cd);
    *c = (float)(cd * r.amplitude);
    *s = (float)((inverse ? -sd : sd) * r.amplitude);
}

// Two 32-bit operations at a time, each rounded by itself.  A product that is added to something is written as a b + (-0)
// with the -0 from the kernel's arguments: mul.rn.f32x2 and add.rn.f32x2 came out as one multiply-add with one rounding
// (1e-4 of fp16 results another, and with them levels of a 4-bit cache), unlike their forms for one value.
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ explicit F2(const float2& f) : F2(f.x, f.y) {}
    __device__ __forceinline__ float2 get() const {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ F2 operator*(const F2& a, const F2& b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 product(const F2& a, const F2& b, const F2& minus_zero) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(minus_zero.v));
    return r;
}
__device__ __forceinline__ F2 operator+(const F2& a, const F2& b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// A thread's part of a row: 8 elements from `lane * 8` on, turned.  With the half layout its partners lie in the lane
// `partner`; `s` comes with the sign of its half.  Neighbouring pairs: c is (cos, cos), s is (-sin, sin).
template <bool BF16, bool INTER>
struct Turn {
    F2 c[4], s[4];
    int partner;
    bool on;
    // `table`: cos and sin of the thread's token, pair by pair
    template <int LPR>
    __device__ __forceinline__ void load(const float2* table, int lane, int dim) {
        on = lane * 8 < dim;
        partner = lane;
        if (!on) return;
        if constexpr (INTER) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 cs = table[lane * 4 + e];
                c[e] = F2(cs.x, cs.x);
                s[e] = F2(-cs.y, cs.y);
            }
        } else {
            const int half = dim / 16;                     // lanes of the first halves
            const bool second = lane >= half;
            partner = second ? lane - half : lane + half;
            const int p = (second ? lane - half : lane) * 8;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 a = table[p + 2 * e], b = table[p + 2 * e + 1];
                c[e] = F2(a.x, b.x);
                s[e] = second ? F2(a.y, b.y) : F2(-a.y, -b.y);
            }
        }
    }
    // All lanes of the warp call this.  Products and sums are rounded one by one, so that a value is the same
    // wherever it is computed: a cache in 4 bits takes its levels from it.
    template <int LPR>
    __device__ __forceinline__ uint4 apply(const uint4& x, const Rotary& rot) const {
        const F2 mz(rot.minus_zero[0], rot.minus_zero[1]);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = unpack16<BF16>(w[i]);
            float2 r;
            if constexpr (INTER) r = (product(F2(f), c[i], mz) + product(F2(f.y, f.x), s[i], mz)).get();
            else r = (product(F2(f), c[i], mz) + product(F2(unpack16<BF16>(__shfl_sync(0xffffffffu, w[i], partner, LPR))), s[i], mz)).get();
            y[i] = pack16<BF16>(r.x, r.y);
        }
        return on ? make_uint4(y[0], y[1], y[2], y[3]) : x;
    }
};

__device__ __forceinline__ uint4 ld_row_16(const uint16_t* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

// ------------------------------------------------------------------------------------------ fa_rope
struct RopeTensor {
    const uint16_t* in;
    uint16_t* out;
    fa_strides is, os;
};
struct RopeArgs {
    RopeTensor q, k;
    Rotary rot;
    int hq, heads, seq_len, tiles;       // heads of q and k together, token tiles of a sequence
    int tokens;                          // of a block: a power of two
    int splits;                          // blocks that share a tile's heads
    const int* positions;
    int positions_stride, position_offset;
    bool inverse;
};

// Blocks of 8 or 16 tokens of a sequence and, while SMs are idle, parts of the heads; kUnroll rows a thread under way.  HBM bounds
// it: bf16 B=2 Hq=32 Hkv=8 S=4096 D=128, half of the head turned, 168 MB in 31 us, 5.4 TB/s.
template <int D, bool BF16, bool INTER>
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int LPR = D / 8, SLOTS = kThreads / LPR;
    extern __shared__ float2 table[];                       // [tokens][dim / 2]
    const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
    const int b = tile / a.tiles, s0 = (tile - b * a.tiles) * a.tokens;
    const int pairs = a.rot.dim / 2;
    if (a.positions != nullptr) grid_dependency_wait();     // known positions: the table overlaps the kernel before
    for (int i = threadIdx.x; i < a.tokens * pairs; i += kThreads) {
        const int t = i / pairs, s = min(s0 + t, a.seq_len - 1);
        const int pos = a.positions == nullptr ? s + a.position_offset : a.positions[(long long)b * a.positions_stride + s];
        float2 cs;
        cos_sin(a.rot, pos, i - t * pairs, a.inverse, &cs.x, &cs.y);
        table[i] = cs;
    }
    grid_dependency_wait();
    grid_launch_dependents();
    __syncthreads();
    const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const int t = slot & (a.tokens - 1), step = SLOTS / a.tokens;
    const int s = s0 + t;
    Turn<BF16, INTER> turn;
    turn.template load<LPR>(table + t * pairs, lane, a.rot.dim);
    const int per = (a.heads + a.splits - 1) / a.splits, h_end = min(a.heads, (split + 1) * per);
    for (int h0 = split * per; h0 < h_end; h0 += step * kUnroll) {
        uint4 x[kUnroll];
        bool live[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int h = h0 + u * step + slot / a.tokens;
            live[u] = h < h_end && s < a.seq_len;
            x[u] = make_uint4(0, 0, 0, 0);
            if (live[u]) {
                const RopeTensor& r = h < a.hq ? a.q : a.k;
                x[u] = ld_row_16(r.in + b * r.is.batch + (h < a.hq ? h : h - a.hq) * r.is.head + s * r.is.row + lane * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int h = h0 + u * step + slot / a.tokens;
            const uint4 y = turn.template apply<LPR>(x[u], a.rot);
            if (live[u]) {
                const RopeTensor& r = h < a.hq ? a.q : a.k;
                *reinterpret_cast<uint4*>(r.out + b * r.os.batch + (h < a.hq ? h : h - a.hq) * r.os.head + s * r.os.row + lane * 8) = y;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ fa_cache_append
struct AppendArgs {
    const uint16_t *q, *k, *v;
    void* q_out;
    uint8_t *k_cache, *v_cache;
    __half2 *k_params, *v_params;
    long long q_stride, k_stride, v_stride;
    Rotary rot;
    int hq, hkv, n_tokens, n_all, seq_len_kv;    // tokens of a sequence, of all
    int tokens, splits;                          // as in RopeArgs
    CacheMap map;
    long long block_stride, head_stride, row_stride;          // bytes
    long long p_block_stride, p_head_stride, p_row_stride;    // pairs
    const int *seq_lens, *num_new, *positions;
    const float *q_scale, *k_scale, *v_scale;
    FastDiv by_tokens, by_pairs, by_splits, by_group, by_hkv;
};

struct Token {
    int b, row, position;
    bool live;                                   // is stored
};
__device__ __forceinline__ Token token(const AppendArgs& a, int n) {
    Token r;
    r.b = a.by_tokens.quot(n);
    const int t = n - r.b * a.n_tokens;
    r.row = sequence_length(a.seq_lens, r.b, a.seq_len_kv) - a.n_tokens + t;
    r.live = r.row >= 0 && (a.num_new == nullptr || a.n_tokens - t <= a.num_new[r.b]);     // any number: nothing is taken from it
    r.position = a.positions == nullptr ? r.row : a.positions[n];
    return r;
}

__device__ __forceinline__ uint32_t e4m3x4(float2 a, float2 b) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// 8 elements as e4m3 codes of value * inv.
template <bool BF16>
__device__ __forceinline__ uint2 to_e4m3(const uint4& x, float inv) {
    const F2 i(inv, inv);
    return make_uint2(e4m3x4((F2(unpack16<BF16>(x.x)) * i).get(), (F2(unpack16<BF16>(x.y)) * i).get()),
                      e4m3x4((F2(unpack16<BF16>(x.z)) * i).get(), (F2(unpack16<BF16>(x.w)) * i).get()));
}
template <bool BF16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 8 elements as 4-bit codes; the 8 lanes of a group of 64 call this together.  Returns the codes, and scale and
// offset in every lane.  An element past +-65504 gets the code of the border: its difference from the offset is clamped.
template <bool BF16>
__device__ __forceinline__ uint32_t to_u4(const uint4& x, __half2* param) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t lo2 = min2_nan<BF16>(min2_nan<BF16>(w[0], w[1]), min2_nan<BF16>(w[2], w[3]));
    uint32_t hi2 = max2_nan<BF16>(max2_nan<BF16>(w[0], w[1]), max2_nan<BF16>(w[2], w[3]));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo2 = min2_nan<BF16>(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
        hi2 = max2_nan<BF16>(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
    }
    const float2 l = unpack16<BF16>(lo2), h = unpack16<BF16>(hi2);
    const float lo = max_nan(min_nan(min_nan(l.x, l.y), kU4Max), -kU4Max), hi = max_nan(min_nan(max_nan(h.x, h.y), kU4Max), -kU4Max);
    const __half z16 = __float2half_rn(lo);
    const float z = __half2float(z16);
    const __half s16 = __float2half_rn(__fmul_rn(__fsub_rn(hi, z), 1.0f / 15.0f));
    const float s = __half2float(s16), inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
    // round to a whole number, ties to even, by adding 1.5 * 2^23: the code is in the last bits; 16 a + b of the bits then
    // strings the codes together, with the constant's share taken off at the end
    constexpr float kRound = 12582912.0f;
    constexpr uint32_t kBits = 0x4B400000u;
    const F2 minus_z(-z, -z), inv2(inv, inv), round2(kRound, kRound);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 3; i >= 0; i--) {
        const float2 c = ((F2(unpack16<BF16>(w[i])) + minus_z) * inv2).get();
        const float2 r = (F2(fminf(fmaxf(c.x, 0.0f), 15.0f), fminf(fmaxf(c.y, 0.0f), 15.0f)) + round2).get();
        codes = (codes * 16u + __float_as_uint(r.y)) * 16u + __float_as_uint(r.x);
    }
    constexpr uint32_t kShare = kBits * 0x11111111u;
    *param = __halves2half2(s16, z16);
    return codes - kShare;
}

// A thread keeps to one token and walks its heads, those of q, then k, then v, kAppendUnroll at a time; the next ones are
// loaded before these are used, the first ones before the block computes its cos and sin.  What bounds it is the chain
// of loads that a block waits for, one after the other (lengths, page, rows), and then the 165 instructions that 16 bytes of a
// row cost: small blocks of few tokens, 8 of them an SM (512 tokens to 8 sequences, Hq=32 Hkv=8 D=128, e4m3 / 4-bit with its read
// back, us in a graph: 256 threads and 8 tokens 22.7 / 29.9, 128 and 2 20.0 / 26.6; one token to 16 sequences 3.3, 2.8; the scales
// of e4m3 inverted once a block instead of once a row 20.3 -> 19.6).
constexpr int kAppendThreads = 128, kAppendUnroll = 2;
template <int D, bool BF16, bool INTER, int CACHE>
__global__ void __launch_bounds__(kAppendThreads, 8) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int LPR = D / 8, SLOTS = kAppendThreads / LPR, U = kAppendUnroll;
    extern __shared__ float2 table[];                       // [tokens][dim / 2]
    const int tile = a.by_splits.quot(blockIdx.x), split = (int)blockIdx.x - tile * a.splits, n0 = tile * a.tokens;
    const int pairs = a.rot.dim / 2, hqk = a.hq + a.hkv, heads = hqk + a.hkv;
    const int per = (heads + a.splits - 1) / a.splits, h_begin = split * per, h_end = min(heads, h_begin + per);
    const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const int t = slot & (a.tokens - 1), step = SLOTS / a.tokens, mine = slot / a.tokens, n = n0 + t;
    grid_dependency_wait();
    grid_launch_dependents();
    const bool in = n < a.n_all;
    const Token tk = token(a, min(n, a.n_all - 1));
    const bool live = in && tk.live;

    // groups of heads of one kind: 0 q, 1 k, 2 v, [h0, end) of that kind left
    struct Group {
        int kind, h0, end;
    };
    auto begin_kind = [&](int kind) {
        Group g;
        do {
            const int base = kind == 0 ? 0 : kind == 1 ? a.hq : hqk;
            g.kind = kind;
            g.h0 = max(h_begin - base, 0);
            g.end = min(h_end - base, kind == 0 ? a.hq : a.hkv);
        } while (g.h0 >= g.end && ++kind < 3);
        g.kind = kind;
        return g;
    };
    auto load = [&](const Group& g, uint4 (&x)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = make_uint4(0, 0, 0, 0);
        if (g.kind > 2 || !live) return;
        const uint16_t* p = (g.kind == 0 ? a.q + n * a.q_stride : g.kind == 1 ? a.k + n * a.k_stride : a.v + n * a.v_stride) + (g.h0 + mine) * D + lane * 8;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (g.h0 + mine + u * step < g.end) x[u] = ld_row_16(p + u * step * D);
    };
    Group g = begin_kind(0);
    uint4 x[U];
    load(g, x);
    if (h_begin < hqk)                                      // not v alone
        for (int i = threadIdx.x; i < a.tokens * pairs; i += kAppendThreads) {
            const int ti = a.by_pairs.quot(i);
            float2 cs;
            cos_sin(a.rot, token(a, min(n0 + ti, a.n_all - 1)).position, i - ti * pairs, false, &cs.x, &cs.y);
            table[i] = cs;
        }
    // e4m3: 1 / scale of the block's tokens, those of q, k and v for each KV head
    float* inv = reinterpret_cast<float*>(table + a.tokens * pairs);
    if constexpr (CACHE == FA_CACHE_E4M3)
        for (int i = threadIdx.x; i < a.tokens * 3 * a.hkv; i += kAppendThreads) {
            const int y = a.by_hkv.quot(i), h = i - y * a.hkv, ti = y / 3, kind = y - ti * 3;
            const float* scale = kind == 0 ? a.q_scale : kind == 1 ? a.k_scale : a.v_scale;
            inv[i] = scale == nullptr ? 0.0f : __frcp_rn(scale[a.by_tokens.quot(min(n0 + ti, a.n_all - 1)) * a.hkv + h]);
        }
    CacheRow at = {-1, 0};
    if (live) at = cache_row(a.map, tk.b, tk.row);
    __syncthreads();
    Turn<BF16, INTER> turn;
    turn.template load<LPR>(table + t * pairs, lane, a.rot.dim);
    inv += t * 3 * a.hkv;
    const bool store = live && at.block >= 0;
    constexpr int kLaneBytes = CACHE == FA_CACHE_U4 ? 4 : CACHE == FA_CACHE_E4M3 ? 8 : 16;
    const long long row = at.block * a.block_stride + at.in_block * a.row_stride + lane * kLaneBytes;
    const long long prow = CACHE == FA_CACHE_U4 ? at.block * a.p_block_stride + at.in_block * a.p_row_stride + lane / 8 : 0;

    while (g.kind <= 2) {
        Group next = g;
        next.h0 += step * U;
        if (next.h0 >= next.end) next = begin_kind(g.kind + 1);
        uint4 x_next[U];
        load(next, x_next);
        if (g.kind == 0) {
            uint8_t* p = static_cast<uint8_t*>(a.q_out) + (((long long)n * a.hq + g.h0 + mine) * D + lane * 8) * (CACHE == FA_CACHE_E4M3 ? 1 : 2);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint4 y = turn.template apply<LPR>(x[u], a.rot);
                const int h = g.h0 + mine + u * step;
                if (h < g.end && in) {
                    if constexpr (CACHE == FA_CACHE_E4M3) {
                        *reinterpret_cast<uint2*>(p + u * step * D) = live ? to_e4m3<BF16>(y, inv[a.by_group.quot(h)]) : make_uint2(0, 0);
                    } else {
                        *reinterpret_cast<uint4*>(p + u * step * D * 2) = live ? y : make_uint4(0, 0, 0, 0);    // turned zeros may be -0
                    }
                }
            }
        } else {
            uint8_t* cache = (g.kind == 2 ? a.v_cache : a.k_cache) + row;
            [[maybe_unused]] __half2* params = (g.kind == 2 ? a.v_params : a.k_params) + prow;
            [[maybe_unused]] const float* kv_inv = inv + g.kind * a.hkv;
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint4 y = x[u];
                if (g.kind == 1) y = turn.template apply<LPR>(y, a.rot);
                const int h = g.h0 + mine + u * step;
                const bool put = store && h < g.end;
                if constexpr (CACHE == FA_CACHE_U4) {
                    __half2 param;
                    const uint32_t codes = to_u4<BF16>(y, &param);           // lanes of a row agree on `put`; all take part
                    if (put) {
                        *reinterpret_cast<uint32_t*>(cache + h * a.head_stride) = codes;
                        if ((lane & 7) == 0) params[h * a.p_head_stride] = param;
                    }
                } else if (put) {
                    if constexpr (CACHE == FA_CACHE_E4M3) *reinterpret_cast<uint2*>(cache + h * a.head_stride) = to_e4m3<BF16>(y, kv_inv[h]);
                    else *reinterpret_cast<uint4*>(cache + h * a.head_stride) = y;
                }
            }
        }
        g = next;
#pragma unroll
        for (int u = 0; u < U; u++) x[u] = x_next[u];
    }
}

// ------------------------------------------------------------------------------------------ fa_cache_read_u4
struct ReadArgs {
    const uint8_t *k, *v;
    const __half2 *kp, *vp;
    uint16_t *k_out, *v_out;
    long long o_batch, o_row, o_head;                         // elements between the outputs' sequences, rows and heads
    long long remainder;                                      // elements from a value to its remainder
    int hkv, seq_len_kv, n_rows, tiles;
    CacheMap map;
    long long block_stride, head_stride, row_stride;          // bytes
    long long p_block_stride, p_head_stride, p_row_stride;    // pairs
    const int *seq_lens, *first_rows;
};

template <bool BF16>
__device__ __forceinline__ uint4 from_u4(uint32_t codes, __half2 param) {
    const float s = __low2float(param), z = __high2float(param);
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = fmaf(s, (float)((codes >> (8 * i)) & 15u), z), b = fmaf(s, (float)((codes >> (8 * i + 4)) & 15u), z);
        // fp16: at most 65504 at either end (a scale rounded up: -65504 + 15 * 8736 = 65536, and the same with the signs turned)
        if constexpr (BF16) y[i] = pack16<true>(a, b);
        else asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(y[i]) : "f"(b), "f"(a));
    }
    return make_uint4(y[0], y[1], y[2], y[3]);
}

// What is left of the values beside their fp16 forms y, in fp16 (2^-22 of a value, at least 2^-25).
__device__ __forceinline__ uint4 remainder_u4(uint32_t codes, __half2 param, const uint4& y) {
    const float s = __low2float(param), z = __high2float(param);
    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 h = unpack16<false>(w[i]);
        const float a = fmaf(s, (float)((codes >> (8 * i)) & 15u), z), b = fmaf(s, (float)((codes >> (8 * i + 4)) & 15u), z);
        // a value past fp16 counts as the largest: nothing is left of it
        r[i] = pack16<false>(max_nan(min_nan(a, kU4Max), -kU4Max) - h.x, max_nan(min_nan(b, kU4Max), -kU4Max) - h.y);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// A block takes kUnroll groups of consecutive rows of one head: the codes and pairs of consecutive rows lie together where the cache
// is laid out for attention, and what it writes are whole rows either way.  HBM bounds it, by its writes: 4 sequences of 16384 rows,
// Hkv=8 D=128, 344 MB in 57 us, 6.0 TB/s.
// COPY, for attention of many tokens: rows that a sequence does not have stay as they are, instead of zero; REMAINDER: what is left of a
// value goes a.remainder elements behind it.
template <int D, bool BF16, bool COPY, bool REMAINDER>
__global__ void __launch_bounds__(kThreads) read_u4_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int LPR = D / 8, SLOTS = kThreads / LPR;
    const int lane = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const int bh = blockIdx.x / a.tiles, tile = blockIdx.x - bh * a.tiles;
    const int b = bh / a.hkv, h = bh - b * a.hkv;
    grid_dependency_wait();
    grid_launch_dependents();
    const int len = sequence_length(a.seq_lens, b, a.seq_len_kv);
    const int first = a.first_rows == nullptr ? 0 : a.first_rows[b];
    uint32_t kc[kUnroll], vc[kUnroll];
    __half2 kp[kUnroll], vp[kUnroll];
    bool live[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
        const int n = (tile * kUnroll + u) * SLOTS + slot;
        const long long row = (long long)first + n;
        kc[u] = vc[u] = 0;
        kp[u] = vp[u] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
        live[u] = row >= 0 && row < len;
        if (n < a.n_rows && live[u]) {
            const CacheRow at = cache_row(a.map, b, (int)row);
            if (at.block >= 0) {
                const long long o = at.block * a.block_stride + h * a.head_stride + at.in_block * a.row_stride + lane * 4;
                const long long p = at.block * a.p_block_stride + h * a.p_head_stride + at.in_block * a.p_row_stride + lane / 8;
                kc[u] = *reinterpret_cast<const uint32_t*>(a.k + o);
                vc[u] = *reinterpret_cast<const uint32_t*>(a.v + o);
                kp[u] = a.kp[p];
                vp[u] = a.vp[p];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
        const int n = (tile * kUnroll + u) * SLOTS + slot;
        if (n < a.n_rows && (live[u] || !COPY)) {
            const long long o = b * a.o_batch + n * a.o_row + h * a.o_head + lane * 8;
            const uint4 k = from_u4<BF16>(kc[u], kp[u]), v = from_u4<BF16>(vc[u], vp[u]);
            *reinterpret_cast<uint4*>(a.k_out + o) = k;
            *reinterpret_cast<uint4*>(a.v_out + o) = v;
            if constexpr (REMAINDER) {
                *reinterpret_cast<uint4*>(a.k_out + o + a.remainder) = remainder_u4(kc[u], kp[u], k);
                *reinterpret_cast<uint4*>(a.v_out + o + a.remainder) = remainder_u4(vc[u], vp[u], v);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ host
int make_rotary(const fa_rotary& r, int d_head, bool optional, Rotary* out) {
    *out = Rotary{};
    out->minus_zero[0] = out->minus_zero[1] = -0.0f;
    if (r.rotary_dim < 0) return FA_ERR_INVALID_ARGUMENT;
    if (r.rotary_dim == 0) return optional ? FA_OK : FA_ERR_INVALID_ARGUMENT;
    if (r.rotary_dim > d_head || r.rotary_dim % 16 != 0) return FA_ERR_UNSUPPORTED;
    if (r.inv_freq == nullptr || !std::isfinite(r.amplitude) || (r.interleaved != 0 && r.interleaved != 1)) return FA_ERR_INVALID_ARGUMENT;
    const long double turns = 1.0L / 6.283185307179586476925286766559L;
    for (int i = 0; i < r.rotary_dim / 2; i++) {
        if (!std::isfinite(r.inv_freq[i])) return FA_ERR_INVALID_ARGUMENT;
        long double f = r.inv_freq[i] * turns;
        if (f < 0.0L || f >= 1.0L) f -= std::floor(f);       // whole turns are none
        out->turns[i] = f >= 1.0L ? 0ull : (unsigned long long)(f * 18446744073709551616.0L);
    }
    out->amplitude = r.amplitude;
    out->dim = r.rotary_dim;
    return FA_OK;
}

// Blocks that share a tile's heads.  A block computes cos and sin for all of its tokens, so few blocks with many heads
// are better until the GPU has idle SMs: two blocks an SM.
int head_splits(long long tiles, int heads, int rows_at_once, int sm_count) {
    const long long want = (2ll * sm_count + tiles - 1) / tiles;
    const int most = (heads + rows_at_once - 1) / rows_at_once;
    return want < 1 ? 1 : want > most ? most : (int)want;
}
int pow2_at_least(int n, int most) {
    int p = 1;
    while (p < n && p < most) p *= 2;
    return p;
}

bool strides_ok(const fa_strides& s) { return s.batch >= 0 && s.head >= 0 && s.row >= 0; }
// A tensor that is its own result: every row is read before it is written if both lie in the same places.
bool in_place_ok(const void* in, const void* out, const fa_strides& is, const fa_strides& os, int batch, int heads, int seq_len) {
    return in != out || ((batch == 1 || is.batch == os.batch) && (heads == 1 || is.head == os.head) && (seq_len == 1 || is.row == os.row));
}
// Results whose rows do not fall together by a stride of 0 (what is read may: an expanded tensor).
bool rows_apart(const fa_strides& s, int batch, int heads, int seq_len) {
    return (batch == 1 || s.batch > 0) && (heads == 1 || s.head > 0) && (seq_len == 1 || s.row > 0);
}
bool strides_aligned(const fa_strides& s) { return s.batch % 8 == 0 && s.head % 8 == 0 && s.row % 8 == 0; }
fa_strides or_dense(const fa_strides& s, int heads, int seq_len, int d_head) {
    if (s.batch || s.head || s.row) return s;
    return {(long long)heads * seq_len * d_head, (long long)seq_len * d_head, d_head};
}

template <int D, bool BF16, bool INTER>
int run_rope(const RopeArgs& a, unsigned blocks, cudaStream_t stream) {
    return launch_dependent(rope_kernel<D, BF16, INTER>, blocks, kThreads, (size_t)a.tokens * (a.rot.dim / 2) * sizeof(float2), stream, 1, a);
}
template <int D, bool BF16, bool INTER, int CACHE>
int run_append(const AppendArgs& a, unsigned blocks, cudaStream_t stream) {
    const size_t smem = (size_t)a.tokens * ((a.rot.dim / 2) * sizeof(float2) + (CACHE == FA_CACHE_E4M3 ? 3 * a.hkv * sizeof(float) : 0));
    return launch_dependent(append_kernel<D, BF16, INTER, CACHE>, blocks, kAppendThreads, smem, stream, 1, a);
}
template <int D, bool BF16, bool INTER>
int run_append_to(const AppendArgs& a, int cache, unsigned blocks, cudaStream_t stream) {
    if (cache == FA_CACHE_U4) return run_append<D, BF16, INTER, FA_CACHE_U4>(a, blocks, stream);
    if constexpr (D == 128)
        if (cache == FA_CACHE_E4M3) return run_append<D, BF16, INTER, FA_CACHE_E4M3>(a, blocks, stream);
    return run_append<D, BF16, INTER, FA_CACHE_16BIT>(a, blocks, stream);
}

template <int D>
int run_read_u4(const ReadArgs& a, bool bf, bool copy, unsigned blocks, cudaStream_t stream) {
    auto kernel = !copy ? (bf ? read_u4_kernel<D, true, false, false> : read_u4_kernel<D, false, false, false>)
                        : a.remainder != 0 ? read_u4_kernel<D, false, true, true> : read_u4_kernel<D, false, true, false>;
    return launch_dependent(kernel, blocks, kThreads, 0, stream, 1, a);
}

}  // namespace

// Checks a layout and gives where the rows lie; strides in bytes (`elem` bytes an element, half a byte: elem = 0).
int check_layout(const fa_cache_layout& l, int cache, int d_head, int seq_len_kv, int elem, CacheMap* map) {
    const long long unit = cache == FA_CACHE_U4 ? 1 : elem, row = cache == FA_CACHE_U4 ? d_head / 2 : (long long)d_head * elem;
    if (l.block_stride <= 0 || l.head_stride <= 0 || l.row_stride * unit < row) return FA_ERR_INVALID_ARGUMENT;
    if (l.block_stride * unit % 16 || l.head_stride * unit % 16 || l.row_stride * unit % 16) return FA_ERR_MISALIGNED;
    if (cache == FA_CACHE_U4) {
        const int pairs = d_head / kU4Group;
        if (l.param_block_stride <= 0 || l.param_head_stride <= 0 || l.param_row_stride < pairs) return FA_ERR_INVALID_ARGUMENT;
        if (l.param_block_stride % pairs || l.param_head_stride % pairs || l.param_row_stride % pairs) return FA_ERR_MISALIGNED;
    }
    *map = CacheMap{nullptr, 0, -1, 0};
    if (l.block_table != nullptr) {
        const int ps = l.page_size;
        if (ps < 16 || (ps & (ps - 1)) != 0 || l.num_pages <= 0) return FA_ERR_INVALID_ARGUMENT;
        if ((long long)l.block_table_stride * ps < seq_len_kv) return FA_ERR_INVALID_ARGUMENT;
        int shift = 0;
        while ((1 << shift) < ps) shift++;
        *map = CacheMap{l.block_table, l.block_table_stride, shift, l.num_pages};
    }
    return FA_OK;
}

}  // namespace fa

using namespace fa;

FA_EXPORT int fa_rope(const fa_rope_args* p) {
    if (!p || !p->q || !p->q_out) return FA_ERR_INVALID_ARGUMENT;
    if (p->batch_size <= 0 || p->num_q_heads <= 0 || p->num_kv_heads < 0 || p->seq_len <= 0) return FA_ERR_INVALID_ARGUMENT;
    if ((long long)p->num_q_heads + p->num_kv_heads > 1 << 24 || p->seq_len > 0x7FFFFFFF - 64) return FA_ERR_INVALID_ARGUMENT;
    if ((p->num_kv_heads > 0) != (p->k != nullptr) || (p->k != nullptr) != (p->k_out != nullptr)) return FA_ERR_INVALID_ARGUMENT;
    if (p->inverse != 0 && p->inverse != 1) return FA_ERR_INVALID_ARGUMENT;
    if (p->positions_stride < 0 || (long long)p->position_offset + p->seq_len - 1 > 0x7FFFFFFFll) return FA_ERR_INVALID_ARGUMENT;
    if (!strides_ok(p->q_strides) || !strides_ok(p->k_strides) || !strides_ok(p->q_out_strides) || !strides_ok(p->k_out_strides))
        return FA_ERR_INVALID_ARGUMENT;
    if (!rows_apart(or_dense(p->q_out_strides, p->num_q_heads, p->seq_len, p->d_head), p->batch_size, p->num_q_heads, p->seq_len) ||
        (p->k && !rows_apart(or_dense(p->k_out_strides, p->num_kv_heads, p->seq_len, p->d_head), p->batch_size, p->num_kv_heads, p->seq_len)))
        return FA_ERR_INVALID_ARGUMENT;
    if (p->d_head != 64 && p->d_head != 128) return FA_ERR_UNSUPPORTED;
    if (p->dtype != FA_DTYPE_F16 && p->dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
    RopeArgs a;
    int rc = make_rotary(p->rotary, p->d_head, false, &a.rot);
    if (rc != FA_OK) return rc;
    if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->q_out) || !aligned16(p->k_out)) return FA_ERR_MISALIGNED;
    if (!strides_aligned(p->q_strides) || !strides_aligned(p->k_strides) || !strides_aligned(p->q_out_strides) || !strides_aligned(p->k_out_strides))
        return FA_ERR_MISALIGNED;
    a.q = {static_cast<const uint16_t*>(p->q), static_cast<uint16_t*>(p->q_out), or_dense(p->q_strides, p->num_q_heads, p->seq_len, p->d_head),
           or_dense(p->q_out_strides, p->num_q_heads, p->seq_len, p->d_head)};
    a.k = {static_cast<const uint16_t*>(p->k), static_cast<uint16_t*>(p->k_out), or_dense(p->k_strides, p->num_kv_heads, p->seq_len, p->d_head),
           or_dense(p->k_out_strides, p->num_kv_heads, p->seq_len, p->d_head)};
    if (!in_place_ok(p->q, p->q_out, a.q.is, a.q.os, p->batch_size, p->num_q_heads, p->seq_len) ||
        (p->k && !in_place_ok(p->k, p->k_out, a.k.is, a.k.os, p->batch_size, p->num_kv_heads, p->seq_len)))
        return FA_ERR_INVALID_ARGUMENT;
    DeviceState* st = device_state();
    if (!st) return FA_ERR_CUDA;
    if (st->cc_major != 10) return FA_ERR_NOT_SM100;
    a.hq = p->num_q_heads;
    a.heads = p->num_q_heads + p->num_kv_heads;
    a.seq_len = p->seq_len;
    // 8 tokens a block, and with d_head 64 16 where that leaves blocks enough: then either has two heads of a token at a time, 8 a turn
    // of the loop, of which a last turn wastes fewer than of 16 (us in a graph, 8 / 16: B=4 Hq=32 Hkv=8 S=4096 37.6 / 35.4, B=8 H=12
    // 50.2 / 44.9; with too few blocks, B=1 Hq=32 Hkv=8 S=4096, 11.3 / 12.2)
    const int slots = kThreads / (p->d_head / 8);
    const bool many = (long long)p->batch_size * ((p->seq_len + slots / 2 - 1) / (slots / 2)) >= 2ll * st->sm_count;
    a.tokens = pow2_at_least(p->seq_len, many ? slots / 2 : 8);
    a.tiles = (p->seq_len + a.tokens - 1) / a.tokens;
    const long long tiles = (long long)a.tiles * p->batch_size;
    a.splits = head_splits(tiles, a.heads, slots / a.tokens, st->sm_count);
    a.positions = p->positions;
    a.positions_stride = p->positions_stride;
    a.position_offset = p->position_offset;
    a.inverse = p->inverse != 0;
    if (tiles * a.splits > 0x7FFFFFFFll) return FA_ERR_INVALID_ARGUMENT;
    const unsigned blocks = (unsigned)(tiles * a.splits);
    cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
    const bool bf = p->dtype == FA_DTYPE_BF16, inter = p->rotary.interleaved != 0;
    if (p->d_head == 64)
        return bf ? (inter ? run_rope<64, true, true>(a, blocks, stream) : run_rope<64, true, false>(a, blocks, stream))
                  : (inter ? run_rope<64, false, true>(a, blocks, stream) : run_rope<64, false, false>(a, blocks, stream));
    return bf ? (inter ? run_rope<128, true, true>(a, blocks, stream) : run_rope<128, true, false>(a, blocks, stream))
              : (inter ? run_rope<128, false, true>(a, blocks, stream) : run_rope<128, false, false>(a, blocks, stream));
}

FA_EXPORT int fa_rope_inv_freq(const fa_rope_scaling* s, int rotary_dim, double* inv_freq, float* amplitude) {
    if (!s || !inv_freq) return FA_ERR_INVALID_ARGUMENT;
    if (rotary_dim <= 0 || rotary_dim % 16 != 0 || rotary_dim > 2 * kMaxPairs) return FA_ERR_UNSUPPORTED;
    if (s->kind < FA_ROPE_PLAIN || s->kind > FA_ROPE_SMOOTH) return FA_ERR_UNSUPPORTED;
    if (!(s->base > 1.0) || !std::isfinite(s->base)) return FA_ERR_INVALID_ARGUMENT;
    if (s->kind != FA_ROPE_PLAIN && (!(s->factor >= 1.0) || !std::isfinite(s->factor))) return FA_ERR_INVALID_ARGUMENT;
    const bool mixed = s->kind == FA_ROPE_PARTS || s->kind == FA_ROPE_SMOOTH;
    if (mixed && (!(s->original_length > 0.0) || !std::isfinite(s->original_length) || !(s->slow > 0.0) || !(s->fast > s->slow) || !std::isfinite(s->fast)))
        return FA_ERR_INVALID_ARGUMENT;
    const double two_pi = 6.283185307179586476925286766559, r = rotary_dim;
    const double base = s->kind == FA_ROPE_BASE ? s->base * std::pow(s->factor, r / (r - 2.0)) : s->base;
    // index at which a pair makes `turns` turns over the original length
    auto index_of = [&](double turns) { return r * std::log(s->original_length / (turns * two_pi)) / (2.0 * std::log(base)); };
    double lo = 0.0, hi = 0.0;
    if (s->kind == FA_ROPE_PARTS) {
        lo = std::fmax(std::floor(index_of(s->fast)), 0.0);
        hi = std::fmin(std::ceil(index_of(s->slow)), r - 1.0);
        if (hi - lo < 1e-3) hi = lo + 1e-3;                  // a step instead of a ramp
    }
    for (int i = 0; i < rotary_dim / 2; i++) {
        const double f = std::pow(base, -2.0 * i / r);
        double keep = s->kind == FA_ROPE_LINEAR ? 0.0 : 1.0;
        if (s->kind == FA_ROPE_PARTS) keep = 1.0 - std::fmin(std::fmax((i - lo) / (hi - lo), 0.0), 1.0);
        if (s->kind == FA_ROPE_SMOOTH) keep = std::fmin(std::fmax((s->original_length * f / two_pi - s->slow) / (s->fast - s->slow), 0.0), 1.0);
        inv_freq[i] = keep == 1.0 ? f : keep * f + (1.0 - keep) * f / s->factor;
    }
    if (amplitude) *amplitude = s->kind == FA_ROPE_PARTS ? (float)(0.1 * std::log(s->factor) + 1.0) : 1.0f;
    return FA_OK;
}

FA_EXPORT int fa_cache_append(const fa_cache_append_args* p) {
    if (!p || !p->k || !p->v || !p->k_cache || !p->v_cache) return FA_ERR_INVALID_ARGUMENT;
    if (p->batch_size <= 0 || p->num_tokens <= 0 || p->num_kv_heads <= 0 || p->num_q_heads < 0 || p->seq_len_kv <= 0) return FA_ERR_INVALID_ARGUMENT;
    if ((p->q != nullptr) != (p->num_q_heads > 0) || (p->q != nullptr) != (p->q_out != nullptr)) return FA_ERR_INVALID_ARGUMENT;
    if (p->num_q_heads % p->num_kv_heads != 0 || p->num_tokens > p->seq_len_kv) return FA_ERR_INVALID_ARGUMENT;
    if (p->q_token_stride < 0 || p->k_token_stride < 0 || p->v_token_stride < 0) return FA_ERR_INVALID_ARGUMENT;
    if (p->d_head != 64 && p->d_head != 128) return FA_ERR_UNSUPPORTED;
    if (p->dtype != FA_DTYPE_F16 && p->dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
    if (p->cache != FA_CACHE_16BIT && p->cache != FA_CACHE_E4M3 && p->cache != FA_CACHE_U4) return FA_ERR_UNSUPPORTED;
    if (p->cache == FA_CACHE_E4M3) {
        if (p->d_head != 128 || p->num_kv_heads > 1024) return FA_ERR_UNSUPPORTED;     // their scales lie in 48 KB of shared memory
        if (!p->k_scale || !p->v_scale || (p->q && !p->q_scale)) return FA_ERR_INVALID_ARGUMENT;
    }
    if (p->cache == FA_CACHE_U4 && (!p->k_params || !p->v_params)) return FA_ERR_INVALID_ARGUMENT;
    const long long n_all = (long long)p->batch_size * p->num_tokens;
    if (n_all > 0x7FFFFFFFll || n_all * (p->num_q_heads + 2ll * p->num_kv_heads) > 0x7FFFFFFFll) return FA_ERR_INVALID_ARGUMENT;
    const int heads = p->num_q_heads + 2 * p->num_kv_heads;
    AppendArgs a;
    int rc = make_rotary(p->rotary, p->d_head, true, &a.rot);
    if (rc != FA_OK) return rc;
    const int elem = p->cache == FA_CACHE_E4M3 ? 1 : 2;
    const long long unit = p->cache == FA_CACHE_U4 ? 1 : elem;
    if ((rc = check_layout(p->layout, p->cache, p->d_head, p->seq_len_kv, elem, &a.map)) != FA_OK) return rc;
    if (p->q_token_stride % 8 || p->k_token_stride % 8 || p->v_token_stride % 8) return FA_ERR_MISALIGNED;
    if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->q_out) || !aligned16(p->k_cache) || !aligned16(p->v_cache) ||
        !aligned16(p->k_params) || !aligned16(p->v_params))
        return FA_ERR_MISALIGNED;
    const long long dense_kv = (long long)p->num_kv_heads * p->d_head, dense_q = (long long)p->num_q_heads * p->d_head;
    a.q_stride = p->q_token_stride ? p->q_token_stride : dense_q;
    a.k_stride = p->k_token_stride ? p->k_token_stride : dense_kv;
    a.v_stride = p->v_token_stride ? p->v_token_stride : dense_kv;
    if (a.q_stride < dense_q || a.k_stride < dense_kv || a.v_stride < dense_kv) return FA_ERR_INVALID_ARGUMENT;
    if (p->q && p->q == p->q_out && (p->cache == FA_CACHE_E4M3 || (n_all > 1 && a.q_stride != dense_q))) return FA_ERR_INVALID_ARGUMENT;
    DeviceState* st = device_state();
    if (!st) return FA_ERR_CUDA;
    if (st->cc_major != 10) return FA_ERR_NOT_SM100;
    a.q = static_cast<const uint16_t*>(p->q);
    a.k = static_cast<const uint16_t*>(p->k);
    a.v = static_cast<const uint16_t*>(p->v);
    a.q_out = p->q_out;
    a.k_cache = static_cast<uint8_t*>(p->k_cache);
    a.v_cache = static_cast<uint8_t*>(p->v_cache);
    a.k_params = static_cast<__half2*>(p->k_params);
    a.v_params = static_cast<__half2*>(p->v_params);
    a.hq = p->num_q_heads;
    a.hkv = p->num_kv_heads;
    a.n_tokens = p->num_tokens;
    a.n_all = (int)n_all;
    a.seq_len_kv = p->seq_len_kv;
    // Tokens of a block: a power of two, 2 to 8, such that the KV heads fill a turn of a token's threads (8 heads of 2 tokens with d_head
    // 128, of 4 with 64); fewer while that leaves SMs idle.  (us in a graph, 2 tokens / this, 8 x 512 tokens: D=64 Hq=32 Hkv=8
    // 4-bit 15.2 / 12.7, Hq=12 Hkv=4 12.9 / 8.2; D=128 Hq=16 Hkv=1 15.1 / 12.6; 8 also with Hq=32 Hkv=8 D=64 13.9, 16 with Hq=8 Hkv=1
    // D=64 7.2 where 8 take 6.1.)
    const int slots = kAppendThreads / (p->d_head / 8);
    const int fill = pow2_at_least((slots * kAppendUnroll + p->num_kv_heads - 1) / p->num_kv_heads, 8);
    a.tokens = pow2_at_least((int)((n_all + 2 * st->sm_count - 1) / (2 * st->sm_count)), fill > 2 ? fill : 2);
    const long long tiles = (n_all + a.tokens - 1) / a.tokens;
    a.splits = head_splits(tiles, heads, slots / a.tokens, st->sm_count);
    a.block_stride = p->layout.block_stride * unit;
    a.head_stride = p->layout.head_stride * unit;
    a.row_stride = p->layout.row_stride * unit;
    a.p_block_stride = p->layout.param_block_stride;
    a.p_head_stride = p->layout.param_head_stride;
    a.p_row_stride = p->layout.param_row_stride;
    a.seq_lens = p->layout.seq_lens;
    a.num_new = p->num_new;
    a.positions = p->positions;
    a.q_scale = p->q_scale;
    a.k_scale = p->k_scale;
    a.v_scale = p->v_scale;
    a.by_tokens = FastDiv(a.n_tokens);
    a.by_pairs = FastDiv(a.rot.dim > 0 ? a.rot.dim / 2 : 1);
    a.by_splits = FastDiv(a.splits);
    a.by_group = FastDiv(a.hq > 0 ? a.hq / a.hkv : 1);
    a.by_hkv = FastDiv(a.hkv);
    const unsigned blocks = (unsigned)(tiles * a.splits);
    cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
    const bool bf = p->dtype == FA_DTYPE_BF16, inter = p->rotary.interleaved != 0;
    if (p->d_head == 64)
        return bf ? (inter ? run_append_to<64, true, true>(a, p->cache, blocks, stream) : run_append_to<64, true, false>(a, p->cache, blocks, stream))
                  : (inter ? run_append_to<64, false, true>(a, p->cache, blocks, stream) : run_append_to<64, false, false>(a, p->cache, blocks, stream));
    return bf ? (inter ? run_append_to<128, true, true>(a, p->cache, blocks, stream) : run_append_to<128, true, false>(a, p->cache, blocks, stream))
              : (inter ? run_append_to<128, false, true>(a, p->cache, blocks, stream) : run_append_to<128, false, false>(a, p->cache, blocks, stream));
}

// Rows of a 4-bit cache in 16 bits at any strides: fa_cache_read_u4, and the copies that attention of many tokens works on.
static int launch_read_u4(const fa_cache_read_args& p, long long o_batch, long long o_row, long long o_head, bool copy, long long remainder) {
    ReadArgs a;
    const int rc = check_layout(p.layout, FA_CACHE_U4, p.d_head, p.seq_len_kv, 0, &a.map);
    if (rc != FA_OK) return rc;
    const int slots = kThreads / (p.d_head / 8);
    const long long tiles = ((long long)p.num_rows + slots * kUnroll - 1) / (slots * kUnroll);
    const long long blocks = tiles * p.batch_size * p.num_kv_heads;
    if (blocks > 0x7FFFFFFFll || (long long)p.num_rows + slots * kUnroll > 0x7FFFFFFFll) return FA_ERR_INVALID_ARGUMENT;
    a.k = static_cast<const uint8_t*>(p.k_cache);
    a.v = static_cast<const uint8_t*>(p.v_cache);
    a.kp = static_cast<const __half2*>(p.k_params);
    a.vp = static_cast<const __half2*>(p.v_params);
    a.k_out = static_cast<uint16_t*>(p.k_out);
    a.v_out = static_cast<uint16_t*>(p.v_out);
    a.o_batch = o_batch;
    a.o_row = o_row;
    a.o_head = o_head;
    a.remainder = remainder;
    a.hkv = p.num_kv_heads;
    a.seq_len_kv = p.seq_len_kv;
    a.n_rows = p.num_rows;
    a.tiles = (int)tiles;
    a.block_stride = p.layout.block_stride;
    a.head_stride = p.layout.head_stride;
    a.row_stride = p.layout.row_stride;
    a.p_block_stride = p.layout.param_block_stride;
    a.p_head_stride = p.layout.param_head_stride;
    a.p_row_stride = p.layout.param_row_stride;
    a.seq_lens = p.layout.seq_lens;
    a.first_rows = p.first_rows;
    const bool bf = p.dtype == FA_DTYPE_BF16;
    if (p.d_head == 64) return run_read_u4<64>(a, bf, copy, (unsigned)blocks, static_cast<cudaStream_t>(p.stream));
    return run_read_u4<128>(a, bf, copy, (unsigned)blocks, static_cast<cudaStream_t>(p.stream));
}

int fa::launch_copy_u4(const fa_cache_read_args& p, long long o_batch, long long o_row, long long o_head, long long remainder) {
    return launch_read_u4(p, o_batch, o_row, o_head, true, remainder);
}

FA_EXPORT int fa_cache_read_u4(const fa_cache_read_args* p) {
    if (!p || !p->k_cache || !p->k_params || !p->v_cache || !p->v_params || !p->k_out || !p->v_out) return FA_ERR_INVALID_ARGUMENT;
    if (p->batch_size <= 0 || p->num_kv_heads <= 0 || p->seq_len_kv <= 0 || p->num_rows <= 0) return FA_ERR_INVALID_ARGUMENT;
    if (p->d_head != 64 && p->d_head != 128) return FA_ERR_UNSUPPORTED;
    if (p->dtype != FA_DTYPE_F16 && p->dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
    if ((long long)p->num_rows + 256 > 0x7FFFFFFFll) return FA_ERR_INVALID_ARGUMENT;
    CacheMap map;
    const int rc = check_layout(p->layout, FA_CACHE_U4, p->d_head, p->seq_len_kv, 0, &map);
    if (rc != FA_OK) return rc;
    if (!aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->k_params) || !aligned16(p->v_params) || !aligned16(p->k_out) || !aligned16(p->v_out))
        return FA_ERR_MISALIGNED;
    DeviceState* st = device_state();
    if (!st) return FA_ERR_CUDA;
    if (st->cc_major != 10) return FA_ERR_NOT_SM100;
    const long long row = (long long)p->num_kv_heads * p->d_head;
    return launch_read_u4(*p, row * p->num_rows, row, p->d_head, false, 0);
}
