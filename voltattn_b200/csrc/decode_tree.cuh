// Attention of a tree of drafted tokens over a paged, quantized KV cache: the
// verification step of speculative decoding (no reference counterpart; the
// reference decodes one token at a time).
//
// Sequence b has lens[b] rows in its cache, of which the last n = nodes[b] are
// the drafted tokens'; ctx = lens[b] - n. Node i of sequence b sees the rows
//   A(b, i) = [0, ctx)  and  ctx + j for every bit j < n of mask[b][i]
// and for every query head h, with KV head h / G,
//   out[b][i][h] = sum_{p in A} w_p V_p / sum_{p in A} w_p,   w_p = exp(q . K_p / sqrt(D))
// in the running form of a softmax; a row that sees nothing gives 0.
//
// All G * Q query rows of a (sequence, KV head) read the same cache rows, so
// a CTA takes a tile of 16 query rows (row r: node r / G, query head
// r % G of the group) over a range of the sequence's positions, and streams
// the codes once. Its four warps take blocks of positions in turn, each with
// its own running statistics and its own ring of shared-memory stages that one
// lane set fills by bulk copies; they merge at the end, and the last CTA of a
// row tile merges the ranges.
//
// The products run on mma.sync m16n8k16 straight from the codes: a code is
// placed into an fp16 mantissa with a shift and a bit operation, the result is
// exact, and no scale is multiplied in fp16.
//   S = Q K^T: the K scale of (row, 64-dim group) multiplies the group's fp32
//     partial score. The offset of the placed codes (x = offset + code * step)
//     is taken off as -offset * sum(q) in the accumulator's initial value.
//   O += P V: the V scale multiplies the fp32 weight before its one rounding to
//     fp16 (P' = fp16(w * scale), one P' per group).
// The rounding of P' is the only one below 32 bits: it is relative (2^-11) down to 2^-14. The
// exponent's reference of a query row is the most of score + floor(log2) of the position's own (larger) V scale
// over the positions that it sees, set where P' of that position is 2^11, and left while that
// grows by no more than kTreeLag (log2): a row's largest P' lies in [2^11, 2^16). P' of the other
// positions, and of the group of smaller scales, lie below it by the ratio of weights and scales.
//
// Rows that a query row does not see have no influence at all on it: their
// scores are replaced, their weights selected to 0 before the scale (which may
// be anything, nan included) is applied, and float formats' rows past the end
// are cleared. A drafted float row with inf or nan entries reaches only the rows
// that see it (`special` below).
//
// Bound by instruction issue and the latency between dependent instructions: 27 warp-instructions a
// position and tile for q8+, start and merge included, with three CTAs of 168 registers an SM, issue
// slots 50 % busy. 16 query rows because 32 spill far more at that count (these spill 4 to 52 bytes at D = 128),
// and two CTAs of more registers were slower; four CTAs of 128 registers took 183 us where this took 113.
// Measured: 16 sequences of 1024 to 8192 rows, q8+, 16 nodes, 32 query / 8 KV heads, 101 us
// (the cache at the copy rate would take 26); one sequence of 1024, q4+, 8 nodes, 10.6 us.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "formats.cuh"
#include "prefill_tc.cuh"

namespace va {

struct TreeParams {
    const uint8_t* K;
    const uint8_t* V;
    const __half* scK;
    const __half* scV;
    const __half* q;
    __half* out;
    const unsigned long long* mask;  // [B][Q]
    const int* lens;                 // [B]
    const int* nodes;                // [B] or null (Q each)
    const int* table;                // [B][max_pages]
    float* ws_o;                     // [B*Hkv][R][S][D] partial outputs
    float* ws_ml;                    // [B*Hkv][R][S][2] reference and sum
    unsigned* counters;              // [B*Hkv*tiles]
    long long qs_b, qs_t, qs_h;      // element strides of q and out: sequence, node, head
    long long os_b, os_t, os_h;
    int B, Hkv, G, Q, R, tiles, S;
    int max_pages, page_rows, num_pages;
    // pos / page_rows = (umulhi(pos, page_mul) + pos) >> page_shift for 0 <= pos < 2^31
    unsigned page_mul, page_shift;
    unsigned g_mul, g_shift;  // r / G likewise
    // node of query row r
    __device__ __forceinline__ int node_of(int r) const { return (int)((__umulhi((unsigned)r, g_mul) + (unsigned)r) >> g_shift); }
};

// Splits of a sequence of len rows: whole units of kTreeUnit rows, at most S.
constexpr int kTreeUnit = 128;
constexpr int kTreeMaxSplits = 128;
__device__ __forceinline__ int tree_chunk(int len, int S) {
    const int units = (len + kTreeUnit - 1) / kTreeUnit;
    return max(1, (units + S - 1) / S) * kTreeUnit;
}

template <Kind K, int kDim>
struct TreeCfg {
    static constexpr Kind kKind = K;
    static constexpr int kD = kDim;
    static constexpr int kRows = 16;              // query rows of a CTA
    static constexpr int kNG = kDim / 64;         // scale groups
    static constexpr bool kScaled = !(K == Kind::F16 || K == Kind::BF16);
    static constexpr bool kFloat = is_float_kind(K);  // rows that can hold inf / nan
    static constexpr int kRb = kDim * KindTraits<K>::kBits / 8;
    static constexpr int kSb = kScaled ? 2 * kNG : 0;
    // positions of a block: 32, or 16 where 32 rows of 256 bytes would leave
    // room for one CTA per SM only
    static constexpr int kPb = (kScaled || kDim == 64) ? 32 : 16;
    static constexpr int kWarps = 4;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kOffV = kPb * kRb;
    static constexpr int kOffSK = 2 * kPb * kRb;
    static constexpr int kOffSV = kOffSK + kPb * kSb;
    static constexpr int kTx = kOffSV + kPb * kSb;
    static constexpr int kStageBytes = (kTx + 127) / 128 * 128;
    static constexpr int kStages = kStageBytes > 8000 ? 2 : kStageBytes > 5000 ? 3 : 4;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kOStride = kDim + 4;     // floats of a merged row
    static constexpr int kMerge = kWarps * kRows * kOStride * 4;
    static constexpr int kBig = kRing > kMerge ? kRing : kMerge;
    // + barriers, masks, (ref, l) of every warp and row, the ticket
    static constexpr int kSmemBytes = kBig + kWarps * kStages * 8 + kRows * 8 + kWarps * kRows * 8 + 16;
    static constexpr int kMinCtas = 3;
    static_assert(kRows * (kTreeMaxSplits + 1) * 4 <= kBig, "the merge of the ranges fits before the barriers");
};

__device__ __forceinline__ void mma_f16_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same with the accumulator's initial values (rows g and g + 8) in c0, c1.
__device__ __forceinline__ void mma_f16_16816_init(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float c0,
                                                   float c1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, "
        "%11, %11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t bf2_to_h2(uint32_t w) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    return h2_bits(__float22half2_rn(f));
}
__device__ __forceinline__ uint32_t f8x2_to_h2(uint32_t b) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(b & 0xFFFFu), __NV_E4M3);
    return (uint32_t)r.x | ((uint32_t)r.y << 16);
}

// What a placed K code stands for: x = kOffset + code / kInvStep, code = the
// signed code. q4: 1 + nibble / 64; q3: 1 + field / 8; q8: 1024 + byte.
template <Kind K>
struct TreeCode {
    static constexpr float kOffset = K == Kind::Q4 ? 1.125f : K == Kind::Q3 ? 1.5f : K == Kind::Q8 ? 1152.f : 0.f;
    static constexpr float kInvStep = K == Kind::Q4 ? 64.f : K == Kind::Q3 ? 8.f : 1.f;
};

// Eight 3-bit fields of a (low halves) and b (high halves) placed at bits 7..9
// of an fp16 1.0: lo = their bits 0..15, hi = their bits 9..23 (fields 3..7).
__device__ __forceinline__ void q3_place(uint32_t a, uint32_t b, uint32_t* h) {
    constexpr uint32_t kM = 0x03800380u, kOne = 0x3C003C00u;
    const uint32_t lo = __byte_perm(a, b, 0x5410), hi = __byte_perm(a >> 9, b >> 9, 0x5410);
    h[0] = ((lo << 7) & kM) | kOne;
    h[1] = ((lo << 4) & kM) | kOne;
    h[2] = ((lo << 1) & kM) | kOne;
    h[3] = ((lo >> 2) & kM) | kOne;
    h[4] = ((lo >> 5) & kM) | kOne;
    h[5] = ((hi << 1) & kM) | kOne;
    h[6] = ((hi >> 2) & kM) | kOne;
    h[7] = ((hi >> 5) & kM) | kOne;
}

// Sixteen consecutive dims (chunk t of group gr) of a K row in shared memory
// as eight fp16 pairs. Pair i holds the dims k_dim(i, 0), k_dim(i, 1) of the
// chunk; the query is loaded in the same order.
template <Kind K>
__device__ __forceinline__ constexpr int k_dim(int i, int e) {
    return K == Kind::Q4 ? 8 * (i >> 2) + (i & 3) + 4 * e : K == Kind::Q3 ? i + 8 * e : 2 * i + e;
}

template <Kind K>
__device__ __forceinline__ void k_chunk(const uint8_t* row, int gr, int t, uint32_t* h) {
    if constexpr (K == Kind::F16 || K == Kind::BF16) {
        const uint4* p = reinterpret_cast<const uint4*>(row + 128 * gr + 32 * t);
        const uint4 a = p[0], b = p[1];
        h[0] = a.x; h[1] = a.y; h[2] = a.z; h[3] = a.w;
        h[4] = b.x; h[5] = b.y; h[6] = b.z; h[7] = b.w;
        if constexpr (K == Kind::BF16) {
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = bf2_to_h2(h[i]);
        }
    } else if constexpr (K == Kind::Q8 || K == Kind::F8) {
        const uint4 a = *reinterpret_cast<const uint4*>(row + 64 * gr + 16 * t);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (K == Kind::Q8) {
                const uint32_t u = w[i] ^ 0x80808080u;
                h[2 * i] = __byte_perm(u, 0x64646464u, 0x4140);
                h[2 * i + 1] = __byte_perm(u, 0x64646464u, 0x4342);
            } else {
                h[2 * i] = f8x2_to_h2(w[i]);
                h[2 * i + 1] = f8x2_to_h2(w[i] >> 16);
            }
        }
    } else if constexpr (K == Kind::Q4) {
        constexpr uint32_t kM = 0x00F000F0u, kOne = 0x3C003C00u;
        const uint2 a = *reinterpret_cast<const uint2*>(row + 32 * gr + 8 * t);
        const uint32_t w[2] = {a.x, a.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            h[4 * i + 0] = ((w[i] << 4) & kM) | kOne;
            h[4 * i + 1] = (w[i] & kM) | kOne;
            h[4 * i + 2] = ((w[i] >> 4) & kM) | kOne;
            h[4 * i + 3] = ((w[i] >> 8) & kM) | kOne;
        }
    } else {
        // bytes 6 t .. 6 t + 5 of the group's 24: two aligned words, shifted by 16 for odd t
        const uint32_t* p = reinterpret_cast<const uint32_t*>(row + 24 * gr + ((6 * t) & ~3));
        const uint32_t sh = (t & 1) * 16;
        const uint32_t w0 = p[0], w1 = p[1];
        const uint32_t lo = __funnelshift_r(w0, w1, sh), hi = w1 >> sh;
        q3_place(lo, (lo >> 24) | (hi << 8), h);
    }
}

// Dims 8 g .. 8 g + 7 of group gr of two V rows as pairs (row a, row b): pair i
// is dim 8 g + i, the code times v_step(i), exact: packed codes are placed where
// they lie in the word, so the step differs between dims (a factor of the
// output's column, applied once at the end) and no shift is spent on them.
template <Kind K>
__host__ __device__ constexpr float v_step(int i) {
    // q4: nibbles 0, 2 of a half word (after one shift by 8) at bits 0..3, nibbles 1, 3 at bits 4..7;
    // q3: fields 0, 3, 6 at bits 0..2, fields 1, 4, 7 at 3..5, fields 2, 5 at 6..8
    return K == Kind::Q4 ? ((i & 1) ? 64.f : 1024.f) : K == Kind::Q3 ? (i % 3 == 0 ? 1024.f : i % 3 == 1 ? 128.f : 16.f) : 1.f;
}

template <Kind K>
__device__ __forceinline__ void v_pairs(const uint8_t* ra, const uint8_t* rb, int gr, int g, uint32_t* h) {
    if constexpr (K == Kind::F16 || K == Kind::BF16) {
        const uint4 a4 = *reinterpret_cast<const uint4*>(ra + 128 * gr + 16 * g);
        const uint4 b4 = *reinterpret_cast<const uint4*>(rb + 128 * gr + 16 * g);
        uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (K == Kind::BF16) {
                a[i] = bf2_to_h2(a[i]);
                b[i] = bf2_to_h2(b[i]);
            }
            h[2 * i] = __byte_perm(a[i], b[i], 0x5410);
            h[2 * i + 1] = __byte_perm(a[i], b[i], 0x7632);
        }
    } else if constexpr (K == Kind::Q8 || K == Kind::F8) {
        const uint2 a2 = *reinterpret_cast<const uint2*>(ra + 64 * gr + 8 * g);
        const uint2 b2 = *reinterpret_cast<const uint2*>(rb + 64 * gr + 8 * g);
        const uint32_t a[2] = {a2.x, a2.y}, b[2] = {b2.x, b2.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t lo = __byte_perm(a[i], b[i], 0x5140), hi = __byte_perm(a[i], b[i], 0x7362);
            if constexpr (K == Kind::Q8) {
                const __half2 off = __float2half2_rn(1152.f);
                lo ^= 0x80808080u;
                hi ^= 0x80808080u;
                h[4 * i + 0] = h2_bits(__hsub2(bits_h2(__byte_perm(lo, 0x64646464u, 0x4140)), off));
                h[4 * i + 1] = h2_bits(__hsub2(bits_h2(__byte_perm(lo, 0x64646464u, 0x4342)), off));
                h[4 * i + 2] = h2_bits(__hsub2(bits_h2(__byte_perm(hi, 0x64646464u, 0x4140)), off));
                h[4 * i + 3] = h2_bits(__hsub2(bits_h2(__byte_perm(hi, 0x64646464u, 0x4342)), off));
            } else {
                h[4 * i + 0] = f8x2_to_h2(lo);
                h[4 * i + 1] = f8x2_to_h2(lo >> 16);
                h[4 * i + 2] = f8x2_to_h2(hi);
                h[4 * i + 3] = f8x2_to_h2(hi >> 16);
            }
        }
    } else if constexpr (K == Kind::Q4) {
        constexpr uint32_t kOne = 0x3C003C00u;
        const __half2 off0 = __float2half2_rn(1.f + 8.f / 1024.f), off1 = __float2half2_rn(1.f + 8.f / 64.f);
        const uint32_t a = *reinterpret_cast<const uint32_t*>(ra + 32 * gr + 4 * g);
        const uint32_t b = *reinterpret_cast<const uint32_t*>(rb + 32 * gr + 4 * g);
        const uint32_t w[2] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632)};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = w[i] >> 8;
            h[4 * i + 0] = h2_bits(__hsub2(bits_h2((w[i] & 0x000F000Fu) | kOne), off0));
            h[4 * i + 1] = h2_bits(__hsub2(bits_h2((w[i] & 0x00F000F0u) | kOne), off1));
            h[4 * i + 2] = h2_bits(__hsub2(bits_h2((u & 0x000F000Fu) | kOne), off0));
            h[4 * i + 3] = h2_bits(__hsub2(bits_h2((u & 0x00F000F0u) | kOne), off1));
        }
    } else {
        constexpr uint32_t kOne = 0x3C003C00u;
        const __half2 off[3] = {__float2half2_rn(1.f + 4.f / 1024.f), __float2half2_rn(1.f + 4.f / 128.f),
                                __float2half2_rn(1.f + 4.f / 16.f)};
        constexpr uint32_t kM[3] = {0x00070007u, 0x00380038u, 0x01C001C0u};
        // bytes 3 g .. 3 g + 2 of the group's 24; the second word only where they straddle
        const int o = 24 * gr + ((3 * g) & ~3);
        const uint32_t sh = 8u * ((3 * g) & 3);
        const uint32_t* pa = reinterpret_cast<const uint32_t*>(ra + o);
        const uint32_t* pb = reinterpret_cast<const uint32_t*>(rb + o);
        const int two = sh > 8 ? 1 : 0;  // (else the first word again: its bits are not used)
        const uint32_t a = __funnelshift_r(pa[0], pa[two], sh);
        const uint32_t b = __funnelshift_r(pb[0], pb[two], sh);
        const uint32_t lo = __byte_perm(a, b, 0x5410), hi = __byte_perm(a >> 9, b >> 9, 0x5410), up = hi >> 9;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t w = i < 3 ? lo : i < 6 ? hi : up;
            h[i] = h2_bits(__hsub2(bits_h2((w & kM[i % 3]) | kOne), off[i % 3]));
        }
    }
}

// One dim of a float row (f16 / bf16 / f8 codes) in shared memory.
template <Kind K>
__device__ __forceinline__ float v_one(const uint8_t* row, int d) {
    if constexpr (K == Kind::F16) return __half2float(reinterpret_cast<const __half*>(row)[d]);
    else if constexpr (K == Kind::BF16) return __half2float(__float2half_rn(__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[d])));
    else return __low2float(bits_h2(f8x2_to_h2(row[d])));
}

// Clears the halves of an fp16 pair that are not finite; true if there were any.
__device__ __forceinline__ bool clear_not_finite(uint32_t& u) {
    bool any = false;
    if ((u & 0x7C00u) == 0x7C00u) u &= 0xFFFF0000u, any = true;
    if ((u & 0x7C000000u) == 0x7C000000u) u &= 0xFFFFu, any = true;
    return any;
}

// floor(log2) of a position's V scales (one, or two and the larger counts) for the exponents'
// reference: whole, so that the position that sets a reference has a power of two as its weight and
// its P' (the scales, then) need no rounding. Infinite and nan ones, which make what they scale
// infinite or nan whatever the reference is, count as fp16's largest; 0, which gives no P' at all, as
// less than its least.
__device__ __forceinline__ float tree_scale_log2(__half2 v) {
    v = __habs2(v);
    const __half m = __hmin(__hmax(__low2half(v), __high2half(v)), __ushort_as_half((unsigned short)0x7BFF));
    return fmaxf((float)((int)(__float_as_uint(__half2float(m)) >> 23) - 127), -25.f);
}
// A row's reference is set where its largest P' is in [2^kTreeBase, 2^(kTreeBase + 1)), and left while
// that stays below 2^(kTreeBase + kTreeLag + 1); fp16 ends just below 2^16. A shorter way to go keeps more of
// the heaviest positions at exact weights, and moves O more often (kTreeLag 2: 103 us where this takes 101).
constexpr float kTreeBase = 11.f, kTreeLag = 3.9f;

// The last range of a row tile merges all of them, in order: first the weights of
// every (row, range) into shared memory (kRows * (kTreeMaxSplits + 1) floats), then the
// outputs with the loads of several rows in flight. kThreads threads take part.
template <int D, int kRows, int kThreads, class Store>
__device__ __forceinline__ void tree_merge(const TreeParams& p, int stream, int r0, int rows, int nsplit, float* sw,
                                           int tid, const Store& store_out) {
    float* sl = sw + kRows * kTreeMaxSplits;  // [kRows] sums
    // some lanes a row, four ranges in flight a lane; the first four are loaded once
    constexpr int kPer = kThreads / kRows >= 8 ? 8 : kThreads / kRows >= 4 ? 4 : 2;
    const int sub = tid % kPer;
#pragma unroll 1
    for (int at = tid / kPer; at < (rows + 15 & ~15); at += kThreads / kPer) {  // (whole warps)
        const int row = min(at, rows - 1);
        const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + ((size_t)stream * p.R + r0 + row) * p.S;
        float2 w[4];
        const auto load = [&](int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = i + kPer * k < nsplit ? __ldcg(ml + i + kPer * k) : make_float2(kNegMax, 0.f);
        };
        float mx = kNegMax, sum = 0.f;
#pragma unroll 1
        for (int i = sub + (nsplit - 1) / (4 * kPer) * (4 * kPer); i >= 0; i -= 4 * kPer) {
            load(i);
            mx = fmaxf(mx, fmaxf(fmaxf(w[0].x, w[1].x), fmaxf(w[2].x, w[3].x)));
        }
#pragma unroll
        for (int off = kPer / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
#pragma unroll 1
        for (int i = sub;;) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float a = fast_exp2(w[k].x - mx);
                sum = fmaf(w[k].y, a, sum);
                if (i + kPer * k < nsplit) sw[row * kTreeMaxSplits + i + kPer * k] = a;
            }
            i += 4 * kPer;
            if (i - sub >= nsplit) break;
            load(i);
        }
#pragma unroll
        for (int off = kPer / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (sub == 0) sl[row] = sum;
    }
    named_barrier_sync(1, kThreads);
    constexpr int Q4 = D / 4;
    static_assert(kThreads % Q4 == 0, "a thread keeps its column");
    constexpr int kRowStep = kThreads / Q4, kItems = 4, kAhead = kRows == 16 ? 4 : 2;
    const int c = tid % Q4;
    for (int rw = tid / Q4; rw < rows; rw += kItems * kRowStep) {
        float4 v[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4* src = reinterpret_cast<const float4*>(p.ws_o + ((size_t)stream * p.R + r0) * p.S * D) + c;
#pragma unroll 1
        for (int s0 = 0; s0 < nsplit; s0 += kAhead) {
            float4 u[kAhead][kItems];
#pragma unroll
            for (int z = 0; z < kAhead; ++z)
#pragma unroll
                for (int k = 0; k < kItems; ++k) {
                    const int row = min(rw + k * kRowStep, rows - 1), s = min(s0 + z, nsplit - 1);
                    u[z][k] = __ldcg(src + ((size_t)row * p.S + s) * Q4);
                }
#pragma unroll
            for (int z = 0; z < kAhead; ++z) {
                const bool on = s0 + z < nsplit;  // (a weight of 0 is not enough: the values may be infinite)
#pragma unroll
                for (int k = 0; k < kItems; ++k) {
                    const int row = min(rw + k * kRowStep, rows - 1);
                    const float a = on ? sw[row * kTreeMaxSplits + s0 + z] : 0.f;
                    v[k].x = fmaf(on ? u[z][k].x : 0.f, a, v[k].x);
                    v[k].y = fmaf(on ? u[z][k].y : 0.f, a, v[k].y);
                    v[k].z = fmaf(on ? u[z][k].z : 0.f, a, v[k].z);
                    v[k].w = fmaf(on ? u[z][k].w : 0.f, a, v[k].w);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int row = rw + k * kRowStep;
            if (row < rows) store_out(r0 + row, c, v[k], sl[row] == 0.f ? 0.f : 1.f / sl[row]);
        }
    }
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, C::kMinCtas) decode_tree_kernel(const TreeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int D = C::kD, NG = C::kNG, PB = C::kPb;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBig);
    unsigned long long* s_mask = reinterpret_cast<unsigned long long*>(bars + C::kWarps * C::kStages);
    float2* s_ml = reinterpret_cast<float2*>(s_mask + C::kRows);
    unsigned* s_ticket = reinterpret_cast<unsigned*>(s_ml + C::kWarps * C::kRows);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int tile = (int)blockIdx.x / p.S, split = (int)blockIdx.x - tile * p.S;
    const int stream = (int)(blockIdx.y + blockIdx.z * gridDim.y);
    if (stream >= p.B * p.Hkv) return;
    const int b = stream / p.Hkv, hk = stream - b * p.Hkv;
    const int r0 = tile * C::kRows;

    grid_dependency_wait();
    const long long cap = (long long)p.max_pages * p.page_rows;
    const int len = (int)max(0ll, min((long long)load_global(p.lens + b), cap));
    const int n = max(0, min(min(p.nodes ? load_global(p.nodes + b) : p.Q, p.Q), len));
    const int ctx = len - n;
    const int chunk = tree_chunk(len, p.S);
    const int nsplit = max(1, (len + chunk - 1) / chunk);
    if (split >= nsplit) return;
    const int p0 = split * chunk, p1 = min(len, p0 + chunk);
    const bool dead = p.node_of(r0) >= n;  // every row of the tile is past the sequence's nodes
    if (dead && split > 0) return;

    uint8_t* ring = smem + warp * (C::kStages * C::kStageBytes);
    uint64_t* bar = bars + warp * C::kStages;
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < C::kStages; ++s) mbar_init(bar + s, 1);
        fence_mbar_init();
    }
    if (tid < C::kRows) {
        const int r = r0 + tid, node = p.node_of(r);
        s_mask[tid] = (r < p.R && node < n) ? load_global(p.mask + (size_t)b * p.Q + node) : 0ull;
    }
    __syncthreads();

    // this warp's blocks: warp, warp + 4, ... of the range's PB-row blocks
    const int nblk = dead ? 0 : (p1 - p0 + PB - 1) / PB;
    const int mine = nblk > warp ? (nblk - warp + C::kWarps - 1) / C::kWarps : 0;
    const uint64_t policy = l2_policy_evict_first();
    const int* trow = p.table + (size_t)b * p.max_pages;
    // rows of one copy: the whole block when it lies inside a page, else runs of 8.
    // Lane 4 r + k copies run r of buffer k (K, V and their scales): its source at
    // page 0 and the bytes of a page and of a row there
    const bool whole = p.page_rows % PB == 0;
    const int run = whole ? PB : 8, nrun = PB / run;
    const int buf = lane & 3, run_at = (lane >> 2) * run;
    const int lane_row = buf < 2 ? C::kRb : C::kSb;
    const uint32_t lane_bytes = (uint32_t)(run * lane_row);
    const bool copies = lane < 4 * nrun && lane_bytes > 0;
    const uint8_t* lane_src = buf == 0   ? p.K
                              : buf == 1 ? p.V
                              : buf == 2 ? reinterpret_cast<const uint8_t*>(p.scK)
                                         : reinterpret_cast<const uint8_t*>(p.scV);
    lane_src += (size_t)hk * p.page_rows * lane_row;
    const long long lane_page = (long long)p.Hkv * p.page_rows * lane_row;
    uint8_t* lane_dst = ring + (buf == 0 ? 0 : buf == 1 ? C::kOffV : buf == 2 ? C::kOffSK : C::kOffSV) + run_at * lane_row;
    const auto issue = [&](int i, int s) {
        if (lane == 0) mbar_arrive_expect_tx(bar + s, C::kTx);
        __syncwarp();
        if (copies) {
            const int pos = p0 + (warp + i * C::kWarps) * PB + run_at;
            const int pi = (int)((__umulhi((unsigned)pos, p.page_mul) + (unsigned)pos) >> p.page_shift);
            int pg = pi < p.max_pages ? load_global(trow + pi) : 0;
            pg = (unsigned)pg < (unsigned)p.num_pages ? pg : 0;
            bulk_g2s(lane_dst + s * C::kStageBytes, lane_src + pg * lane_page + (long long)(pos - pi * p.page_rows) * lane_row,
                     lane_bytes, bar + s, policy);
        }
    };
#pragma unroll 1
    for (int i = 0; i < min(C::kStages, mine); ++i) issue(i, i);

    // the query rows as A fragments, 16 dims (64 gr + 16 t ..) of rows g and
    // g + 8 per lane, in the order of k_chunk's pairs; sums of q per group
    uint32_t qa[NG][4][4];
    float qsum[NG][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = r0 + g + 8 * e;
            const int node = p.node_of(r);
            const bool ok = r < p.R && node < n;
            const __half* src = p.q + b * p.qs_b + (ok ? node : 0) * p.qs_t + (long long)(hk * p.G + (ok ? r - node * p.G : 0)) * p.qs_h;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                uint4 v[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
                if (ok) {
                    const uint4* s4 = reinterpret_cast<const uint4*>(src + 64 * gr + 16 * t);
                    v[0] = load_global(s4);
                    v[1] = load_global(s4 + 1);
                }
                const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    constexpr Kind KK = C::kKind;
                    const int d0 = k_dim<KK>(i, 0), d1 = k_dim<KK>(i, 1);
                    const uint32_t sel = ((d0 & 1) ? 0x32u : 0x10u) | ((d1 & 1) ? 0x7600u : 0x5400u);
                    qa[gr][i >> 1][e + 2 * (i & 1)] = __byte_perm(w[d0 >> 1], w[d1 >> 1], sel);
                    const float2 f = __half22float2(bits_h2(w[i]));
                    sum += f.x + f.y;
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                qsum[gr][e] = -TreeCode<C::kKind>::kOffset * sum;
            }
        }

    float o[NG][8][4];
#pragma unroll
    for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[gr][i][k] = 0.f;
    float ref[2] = {kNegMax, kNegMax}, l[2] = {0.f, 0.f};  // rows g and g + 8
    // scores in log2 units per unit of the raw product
    const float c2 = rsqrtf((float)D) * kLog2e * TreeCode<C::kKind>::kInvStep;

    // One block of positions in stage st. tail: it holds drafted rows or the end
    // of the sequence (two instantiations: the others spend nothing on masks).
    const auto block = [&](auto is_tail, const uint8_t* st, int pb) {
        constexpr bool tail = decltype(is_tail)::value;
        constexpr int NT = PB / 8;  // 8-position tiles of S
        // scores, then weights: row g + 8 r, this lane's positions t + 8 (nt & 1) (.x) and + 4 (.y) of
        // the 16 of tiles nt, nt ^ 1
        float2 x[NT][2];
        __half2 vmax = __float2half2_rn(0.f);
        [[maybe_unused]] uint32_t vsc[NT][2];  // V scales of the two positions (both groups)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // S of 8 positions: lane g decodes row (g >> 1) + 4 (g & 1) (+ 8 for odd tiles) of the 16
            const uint8_t* krow = st + (16 * (nt >> 1) + (g >> 1) + 4 * (g & 1) + 8 * (nt & 1)) * C::kRb;
            float acc[NG][4];
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                uint32_t h[8];
                k_chunk<C::kKind>(krow, gr, t, h);
                float* a = acc[C::kScaled ? gr : 0];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k == 0 && (C::kScaled || gr == 0))
                        mma_f16_16816_init(a, qa[gr][k], h[0], h[1], C::kFloat ? 0.f : qsum[gr][0],
                                           C::kFloat ? 0.f : qsum[gr][1]);
                    else mma_f16_16816(a, qa[gr][k], h[2 * k], h[2 * k + 1]);
                }
            }
            [[maybe_unused]] float2 ks[NG];
            if constexpr (C::kScaled) {
                float2 f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int pr = 16 * (nt >> 1) + t + 4 * e + 8 * (nt & 1);
                    uint32_t k;
                    if constexpr (NG == 2) {
                        k = *reinterpret_cast<const uint32_t*>(st + C::kOffSK + 4 * pr);
                        vsc[nt][e] = *reinterpret_cast<const uint32_t*>(st + C::kOffSV + 4 * pr);
                    } else {
                        k = *reinterpret_cast<const uint16_t*>(st + C::kOffSK + 2 * pr);
                        vsc[nt][e] = *reinterpret_cast<const uint16_t*>(st + C::kOffSV + 2 * pr);
                    }
                    f[e] = __half22float2(bits_h2(k));
                    if constexpr (tail) {
                        if (pb + pr >= len) vsc[nt][e] = 0u;
                    }
                    vmax = __hmax2(vmax, __habs2(bits_h2(vsc[nt][e])));
                }
                ks[0] = make_float2(f[0].x, f[1].x);
                if constexpr (NG == 2) ks[NG - 1] = make_float2(f[0].y, f[1].y);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float2 v = make_float2(acc[0][2 * r], acc[0][2 * r + 1]);
                if constexpr (C::kScaled) {
                    v = fmul2(v, ks[0]);
                    if constexpr (NG == 2) v = ffma2(make_float2(acc[NG - 1][2 * r], acc[NG - 1][2 * r + 1]), ks[NG - 1], v);
                }
                x[nt][r] = v;
            }
        }
        uint32_t seen[2];  // which of this lane's columns a row sees (bit 2 nt + e)
        if constexpr (tail) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const unsigned long long mk = s_mask[g + 8 * r];
                uint32_t bits = 0;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = pb + 16 * (nt >> 1) + t + 4 * e + 8 * (nt & 1) - ctx;
                        const bool v = j < 0 || (j < n && ((mk >> (j & 63)) & 1ull));
                        bits |= (v ? 1u : 0u) << (2 * nt + e);
                        if (!v) (e ? x[nt][r].y : x[nt][r].x) = kNegMax;
                    }
                seen[r] = bits;
            }
        }
        // running reference: the most of score + own V scale's exponent over the columns that the row
        // sees. This lane's largest score with its largest scale is no less; only where one exceeds
        // a row's reference by more than kTreeLag are the row's columns looked at one by one. Nothing of
        // other rows, or of columns that the row does not see, enters a reference.
        float ev = -kTreeBase;
        if constexpr (C::kScaled) {
            ev += tree_scale_log2(vmax);
        }
        float want[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float bm = fmaxf(x[0][r].x, x[0][r].y);
#pragma unroll
            for (int nt = 1; nt < NT; ++nt) bm = fmax3f(bm, x[nt][r].x, x[nt][r].y);
            want[r] = fmaf(bm, c2, ev);
            // (columns that the row does not see at all leave the reference)
            if (tail && bm == kNegMax) want[r] = kNegMax;
        }
        if (__any_sync(0xffffffffu, want[0] > ref[0] + kTreeLag || want[1] > ref[1] + kTreeLag)) {
            float own[2] = {want[0], want[1]};
            if constexpr (C::kScaled) {
                own[0] = own[1] = kNegMax;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float le = tree_scale_log2(bits_h2(vsc[nt][e])) - kTreeBase;
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float y = fmaf(e ? x[nt][r].y : x[nt][r].x, c2, le);
                            if (!tail || ((seen[r] >> (2 * nt + e)) & 1u)) own[r] = fmaxf(own[r], y);
                        }
                    }
            }
            float corr[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                own[r] = fmaxf(own[r], __shfl_xor_sync(0xffffffffu, own[r], 1));
                own[r] = fmaxf(own[r], __shfl_xor_sync(0xffffffffu, own[r], 2));
                const float nr = own[r] > ref[r] + kTreeLag ? own[r] : ref[r];
                corr[r] = fast_exp2(ref[r] - nr);
                ref[r] = nr;
                l[r] *= corr[r];
            }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    o[gr][k][0] *= corr[0];
                    o[gr][k][1] *= corr[0];
                    o[gr][k][2] *= corr[1];
                    o[gr][k][3] *= corr[1];
                }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float2 cc = make_float2(c2, c2), nr = make_float2(-ref[r], -ref[r]);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float2 y = ffma2(x[nt][r], cc, nr);
                float2 w = make_float2(fast_exp2(y.x), fast_exp2(y.y));
                if constexpr (tail) {
                    w.x = (seen[r] >> (2 * nt)) & 1u ? w.x : 0.f;
                    w.y = (seen[r] >> (2 * nt + 1)) & 1u ? w.y : 0.f;
                }
                x[nt][r] = w;
                sum = fadd2(sum, w);
            }
            l[r] += sum.x + sum.y;
        }
        // O += P' V, 16 positions at a time
        bool special = false;
#pragma unroll
        for (int j = 0; j < PB / 16; ++j) {
            const uint8_t* vb = st + C::kOffV + (16 * j + t) * C::kRb;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                uint32_t pa[4];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int nt = 2 * j + hf;
                    float2 s = make_float2(1.f, 1.f);
                    if constexpr (C::kScaled)
                        s = make_float2(__half2float(gr ? __high2half(bits_h2(vsc[nt][0])) : __low2half(bits_h2(vsc[nt][0]))),
                                        __half2float(gr ? __high2half(bits_h2(vsc[nt][1])) : __low2half(bits_h2(vsc[nt][1]))));
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float2 w = x[nt][r];
                        if constexpr (C::kScaled) {
                            w = fmul2(w, s);
                            if constexpr (tail) {  // an unseen row's scale may be nan
                                if (!((seen[r] >> (2 * nt)) & 1u)) w.x = 0.f;
                                if (!((seen[r] >> (2 * nt + 1)) & 1u)) w.y = 0.f;
                            }
                        }
                        pa[2 * hf + r] = h2_bits(__floats2half2_rn(w.x, w.y));
                    }
                }
                uint32_t h0[8], h1[8];
                v_pairs<C::kKind>(vb, vb + 4 * C::kRb, gr, g, h0);
                v_pairs<C::kKind>(vb + 8 * C::kRb, vb + 12 * C::kRb, gr, g, h1);
                if constexpr (C::kFloat && tail) {
                    const int q0 = pb + 16 * j + t;
                    const uint32_t k0 = (q0 < len ? 0xFFFFu : 0u) | (q0 + 4 < len ? 0xFFFF0000u : 0u);
                    const uint32_t k1 = (q0 + 8 < len ? 0xFFFFu : 0u) | (q0 + 12 < len ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {  // entries that are not finite are left to `special`
                        h0[k] &= k0;
                        h1[k] &= k1;
                        special |= clear_not_finite(h0[k]) | clear_not_finite(h1[k]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) mma_f16_16816(o[gr][k], pa, h0[k], h1[k]);
            }
        }
        if constexpr (C::kFloat && tail) {
            // inf and nan entries of the block's rows, added to the rows that see them: what a
            // positive weight times such an entry gives
            if (__any_sync(0xffffffffu, special)) {
                for (int pr = 0; pr < PB; ++pr) {
                    const int j = pb + pr - ctx;
                    if (j >= n) break;
                    const uint8_t* vr = st + C::kOffV + pr * C::kRb;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if (!(j < 0 || ((s_mask[g + 8 * r] >> (j & 63)) & 1ull))) continue;
#pragma unroll
                        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
                            for (int k = 0; k < 8; ++k)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float v = v_one<C::kKind>(vr, 64 * gr + 16 * t + 8 * e + k);
                                    if (!(fabsf(v) <= 65504.f)) o[gr][k][2 * r + e] += v;
                                }
                    }
                }
            }
        }
    };
    bool failed = false;
    int done = 0;
    uint32_t phase = 0;
    for (int i = 0, s = 0; i < mine; ++i) {
        done = i;
        if (!mbar_wait_bounded(bar + s, phase)) {
            failed = true;
            if (lane == 0) report_error(kErrFullWait);
            break;
        }
        const int pb = p0 + (warp + i * C::kWarps) * PB;
        if (pb + PB > ctx) block(std::true_type{}, ring + s * C::kStageBytes, pb);
        else block(std::false_type{}, ring + s * C::kStageBytes, pb);
        __syncwarp();
        if (i + C::kStages < mine) issue(i + C::kStages, s);
        if (++s == C::kStages) s = 0, phase ^= 1u;
    }
    if (failed) {
        // let the copies in flight land (bounded) before the shared memory is given back
        for (int k = done; k < min(done + C::kStages, mine); ++k)
            (void)mbar_wait_bounded(bar + k % C::kStages, (uint32_t)(k / C::kStages) & 1u);
    }
    if (__syncthreads_or(failed)) return;

    // merge the four warps: o and (ref, l) through shared memory
    float* so = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float sum = l[r];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = g + 8 * r;
            if (t == 0) s_ml[warp * C::kRows + row] = make_float2(ref[r], sum);
            float* dst = so + (size_t)(warp * C::kRows + row) * C::kOStride;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int k = 0; k < 8; k += 4)
                        *reinterpret_cast<float4*>(dst + 64 * gr + 16 * t + 8 * e + k) =
                            make_float4(o[gr][k][2 * r + e] * v_step<C::kKind>(k),
                                        o[gr][k + 1][2 * r + e] * v_step<C::kKind>(k + 1),
                                        o[gr][k + 2][2 * r + e] * v_step<C::kKind>(k + 2),
                                        o[gr][k + 3][2 * r + e] * v_step<C::kKind>(k + 3));
        }
    __syncthreads();
    grid_launch_dependents();
    constexpr int Q4 = D / 4;  // float4 columns of a row
    const bool direct = nsplit == 1 || dead;
    const auto store_out = [&](int r, int c, float4 v, float inv) {
        const int node = p.node_of(r);
        __half* dst = p.out + b * p.os_b + node * p.os_t + (long long)(hk * p.G + (r - node * p.G)) * p.os_h + 4 * c;
        const bool live = node < n && inv != 0.f;
        const __half2 a = __floats2half2_rn(live ? v.x * inv : 0.f, live ? v.y * inv : 0.f);
        const __half2 d = __floats2half2_rn(live ? v.z * inv : 0.f, live ? v.w * inv : 0.f);
        *reinterpret_cast<uint2*>(dst) = make_uint2(h2_bits(a), h2_bits(d));
    };
#pragma unroll 1
    for (int i = tid; i < C::kRows * Q4; i += C::kThreads) {
        const int row = i / Q4, c = i - row * Q4, r = r0 + row;
        if (r >= p.R) break;
        float mx = kNegMax, sum = 0.f;
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) mx = fmaxf(mx, s_ml[w * C::kRows + row].x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) {
            const float2 ml = s_ml[w * C::kRows + row];
            const float a = fast_exp2(ml.x - mx);
            const float4 u = *reinterpret_cast<const float4*>(so + (size_t)(w * C::kRows + row) * C::kOStride + 4 * c);
            sum = fmaf(ml.y, a, sum);
            v.x = fmaf(u.x, a, v.x);
            v.y = fmaf(u.y, a, v.y);
            v.z = fmaf(u.z, a, v.z);
            v.w = fmaf(u.w, a, v.w);
        }
        if (direct) {
            store_out(r, c, v, sum == 0.f ? 0.f : 1.f / sum);
        } else {
            const size_t slot = ((size_t)stream * p.R + r) * p.S + split;
            __stcg(reinterpret_cast<float4*>(p.ws_o + slot * D + 4 * c), v);
            if (c == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml + slot * 2), make_float2(mx, sum));
        }
    }
    if (direct) return;
    __syncthreads();
    unsigned* counter = p.counters + (size_t)stream * p.tiles + tile;
    if (tid == 0) *s_ticket = atomic_add_acq_rel_gpu(counter, 1u);
    __syncthreads();
    if (*s_ticket != (unsigned)(nsplit - 1)) return;
    if (tid == 0) store_relaxed_gpu(counter, 0u);
    tree_merge<D, C::kRows, C::kThreads>(p, stream, r0, min(C::kRows, p.R - r0), nsplit, reinterpret_cast<float*>(smem),
                                         tid, store_out);
}

}  // namespace va
