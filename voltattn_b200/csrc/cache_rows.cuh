// Rows of a paged KV cache: K/V rows of packed tokens quantized into their
// pages, and the rows of accepted drafted tokens moved together. No reference
// counterpart: the reference quantizes a whole contiguous cache once
// (src/voltattn.cu:705-745), whose arithmetic the first keeps.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "quantize.cuh"

namespace va {

// BITS of 16-bit rows in bf16 (16: fp16; 8, 4, 3 and kBitsF8 as in quantize.cuh).
constexpr int kBitsBf16 = -16;

struct AppendParams {
    const void* k;
    const void* v;
    long long kt, kh, vt, vh;  // element strides of a token and of a head
    uint8_t* K;
    uint8_t* V;
    __half* scK;
    __half* scV;
    const int* table;
    const int* cu;   // [B + 1] first token of each sequence
    const int* pos;  // [B] row of a sequence's first token
    int T, B, Hkv, D, max_pages, page_rows, num_pages;
    unsigned page_mul, page_shift;  // as TreeParams
};

// Eight consecutive elements of a token's row as they lie in memory, and in fp32.
template <class T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* src) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = load_global(reinterpret_cast<const uint4*>(src) + i);
    return r;
}
template <class T>
__device__ __forceinline__ void to_fp32(const Raw8<T>& r, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else {
        const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 f;
            if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// Sequence of a token: the number of sequences that end at or before it, 32
// ends per step. All lanes of the warp ask for the same token.
__device__ __forceinline__ int token_sequence(const int* cu, int B, int token, int lane) {
    int seq = 0;
    for (int k = 0; k < B; k += 32) {
        const bool past = k + lane < B && load_global(cu + k + lane + 1) <= token;
        const int c = __popc(__ballot_sync(0xffffffffu, past));
        seq += c;
        if (c < 32) break;
    }
    return seq;
}

// The code of va_quantize, by its division: a real call, so that the rare elements that
// need it cost the others a branch and not 25 predicated instructions each.
static __device__ __noinline__ int quantize_exact(float x, float s, int lim) {
    return max(-lim, min(lim, lrint_narrow(__fdiv_rn(x, s))));
}

// The larger of two values, nan if either is.
__device__ __forceinline__ float fmax_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// bits[i] = the fp32 pattern of 1.5 * 2^23 + kBias + code i, code = rint(x / s) clamped to
// [-kLim, kLim] as va_quantize has it, without a division per element: inv = 1 / s to one
// ulp (2^-23) once a group, y = x * inv, and adding 1.5 * 2^23 (+ an even bias) rounds y to an
// integer, half to even. y is within 1.6 * 2^-23 |y| of x / s and the rounded quotient within
// 2^-24 |y|: below 2.6e-7 * (kLim + 1) together, kMargin; so the nearest integer is the
// same unless y is that close to a half. With |y| < kLim + 0.49 in the whole group no
// clamp acts. An element that is close to a half or nan, and groups of other sizes (scales
// that under- or overflowed fp16), take the division.
template <int kLim, int kBias>
__device__ __forceinline__ void quantize_codes(const float (&x)[8], float amax, float s, float inv, uint32_t (&bits)[8]) {
    constexpr float kRound = 12582912.f + (float)kBias, kMargin = 2.6e-7f * (float)(kLim + 1);
    float far = 0.f, y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = x[i] * inv;
        const float t = __fadd_rn(y[i], kRound);
        far = fmax_nan(far, fabsf(y[i] - __fadd_rn(t, -kRound)));
        bits[i] = __float_as_uint(t);
    }
    const bool plain = amax * inv < (float)kLim + 0.49f;
    if (!(plain && far < 0.5f - kMargin)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = fabsf(y[i] - __fadd_rn(__uint_as_float(bits[i]), -kRound));
            if (!(plain && d < 0.5f - kMargin))
                bits[i] = 0x4B400000u + (uint32_t)(kBias + quantize_exact(x[i], s, kLim));
        }
    }
}

// The group scale of va_quantize, amax > 0 ? amax / lim : 1 rounded to fp32, then to
// fp16. The product with 1 / lim is within 2 fp32 ulps of the quotient, so both round to the
// same fp16 unless it lies that close to the middle of two of them: those (about one in
// 1000), and results outside fp16's normal range, take the division.
template <int kLim>
__device__ __forceinline__ __half group_scale(float amax) {
    const float q = amax * (1.f / (float)kLim);
    const uint32_t low = __float_as_uint(q) & 0x1FFFu;
    if (low - 0xFF8u <= 16u || !(q > 6.2e-5f && q < 65000.f))
        return __float2half_rn(amax > 0.f ? __fdiv_rn(amax, (float)kLim) : 1.f);
    return __float2half_rn(q);
}

// One 64-element group from registers, eight consecutive elements per thread (8 lanes a
// group, lane-aligned): scale and codes as quantize_group_values, at `codes` + the
// group's bytes and *scale. All 32 lanes call it.
template <int BITS>
__device__ __forceinline__ void quantize_group_packed(const float (&v)[8], bool active, int part, uint8_t* codes,
                                                      __half* scale) {
    constexpr int lim = BITS == 8 ? 127 : BITS == 4 ? 7 : 3;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));  // fmaxf drops nan operands
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const __half hs = group_scale<lim>(amax);
    const float sh = __half2float(hs);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sh));
    uint32_t c[8];
    quantize_codes<lim, BITS == 8 ? 0 : lim + 1>(v, amax, sh, inv, c);
    if constexpr (BITS == 8) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
        if (active) reinterpret_cast<uint2*>(codes)[part] = make_uint2(w[0], w[1]);
    } else {
        // sum of 2^(BITS i) * (field + the pattern of 1.5 * 2^23), less the patterns' share
        uint32_t w = 0, base = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w += c[i] * (1u << (BITS * i));
            base += 0x4B400000u * (1u << (BITS * i));
        }
        w -= base;
        if constexpr (BITS == 4) {
            if (active) reinterpret_cast<uint32_t*>(codes)[part] = w;
        } else {
            // eight 24-bit pieces as six words: word i begins s bits into piece a
            const int a = (4 * part) / 3, s = 32 * part - 24 * a, lane0 = (threadIdx.x & 31) - part;
            const uint32_t lo = __shfl_sync(0xffffffffu, w, lane0 + (a & 7));
            const uint32_t hi = __shfl_sync(0xffffffffu, w, lane0 + ((a + 1) & 7));
            if (active && part < 6) reinterpret_cast<uint32_t*>(codes)[part] = (lo >> s) | (hi << (24 - s));
        }
    }
    if (active && part == 0) *scale = hs;
}

// A work item is two quads of one token's 64-element groups of K or V (blockIdx.y), 8
// lanes a group. A warp takes items w, w + W, ... and loads the next one (its sequence, its
// page, its elements: four dependent loads) before it quantizes the current one. Bound by the
// quantizer's instructions on prompts (issue slots 70 % busy, DRAM 27 %): 12 prompts of 301 to 4099
// tokens, fp16 to q8+, 8 heads of 128: 55 us, 3.1 TB/s (a division an element: 108 us); 32
// drafts of 7 to 16 tokens: 3.6 us, a launch's latency. (fp32 rows to packed codes spill 40 to 72 bytes at 80
// registers.)
template <int BITS, class T>
__global__ void __launch_bounds__(256, 3) append_packed_kernel(const AppendParams p) {
    constexpr int kBatch = 2;
    constexpr int kBytes = kGroup * (BITS == kBitsF8 ? 8 : BITS == kBitsBf16 ? 16 : BITS) / 8;  // of a group's codes
    const int lane = threadIdx.x & 31, part = lane & 7;
    const int ng = p.D / kGroup, groups = p.Hkv * ng;
    const unsigned per = (unsigned)(groups + 4 * kBatch - 1) / (4 * kBatch);  // items of a token
    const unsigned warps = gridDim.x * (blockDim.x >> 5), step_t = warps / per, step_s = warps - step_t * per;
    const bool is_v = blockIdx.y != 0;
    const long long head = is_v ? p.vh : p.kh, token_step = is_v ? p.vt : p.kt;
    const long long head_groups = (long long)p.page_rows * ng;
    const T* x = static_cast<const T*>(is_v ? p.v : p.k) + part * 8;
    uint8_t* const codes = is_v ? p.V : p.K;
    __half* const scales = is_v ? p.scV : p.scK;
    struct Item {
        Raw8<T> raw[kBatch];
        long long g0;  // the row's first group in the pool; < 0: nothing to do
        int grp;       // this lane's first group of the row
    };
    const auto load = [&](unsigned token, unsigned sub) {
        Item m;
        m.g0 = -1;
        if (token >= (unsigned)p.T) return m;
        m.grp = (int)sub * 4 * kBatch + (lane >> 3);
        const int seq = token_sequence(p.cu, p.B, (int)token, lane);
        if (seq >= p.B) return m;
        const int i = (int)token - load_global(p.cu + seq), at = load_global(p.pos + seq);
        const long long row = (long long)at + i;
        if (i < 0 || at < 0 || row >= (long long)p.max_pages * p.page_rows) return m;
        const int pi = (int)((__umulhi((unsigned)row, p.page_mul) + (unsigned)row) >> p.page_shift);  // (rows fit 31 bits)
        const int pg = load_global(p.table + (size_t)seq * p.max_pages + pi);
        if (pg < 0 || pg >= p.num_pages) return m;
        m.g0 = ((long long)pg * p.Hkv * p.page_rows + ((int)row - pi * p.page_rows)) * ng;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int grp = m.grp + 4 * k, h = ng == 2 ? grp >> 1 : grp;
            m.raw[k] = Raw8<T>{};
            if (grp < groups) m.raw[k] = load8(x + token * token_step + h * head + (grp - h * ng) * kGroup);
        }
        return m;
    };
    grid_dependency_wait();
    grid_launch_dependents();
    const unsigned w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    unsigned token = w / per, sub = w - token * per;
    Item cur = load(token, sub);
    while (token < (unsigned)p.T) {
        token += step_t;
        sub += step_s;
        if (sub >= per) sub -= per, ++token;
        const Item next = load(token, sub);
        if (cur.g0 >= 0) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int grp = cur.grp + 4 * k, h = ng == 2 ? grp >> 1 : grp;
                const bool active = grp < groups;
                const long long g = cur.g0 + h * head_groups + (grp - h * ng);
                float v[8];
                to_fp32(cur.raw[k], v);
                if constexpr (BITS == 16 || BITS == kBitsBf16) {
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (BITS == 16) {
                            const __half2 y = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
                            o[e] = *reinterpret_cast<const uint32_t*>(&y);
                        } else {
                            const __nv_bfloat162 y = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                            o[e] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                    }
                    if (active) reinterpret_cast<uint4*>(codes + g * kBytes)[part] = make_uint4(o[0], o[1], o[2], o[3]);
                } else if constexpr (BITS == kBitsF8) {
                    quantize_group_values<BITS>(v, active, part, g * kGroup + part * 8, g, codes, scales);
                } else {
                    quantize_group_packed<BITS>(v, active, part, codes + g * kBytes, scales + g);
                }
            }
        }
        cur = next;
    }
}

struct AcceptParams {
    uint8_t* K;
    uint8_t* V;
    uint8_t* scK;
    uint8_t* scV;
    const int* table;
    const int* lens;
    const int* nodes;
    const int* path;      // [B][P]
    const int* accepted;  // [B]
    int* new_lens;        // [B]
    long long layer_rows;  // rows of one layer's pool
    int P, Hkv, max_pages, page_rows, num_pages, rb, sb;
};

constexpr int kAcceptMax = 64;     // path entries
constexpr int kAcceptThreads = 128;

// CTA (KV head, sequence, layer): row ctx + path[i] of the sequence to row
// ctx + i, i < accepted. path ascends, so path[i] >= i: no row that is still to
// be read is written by an earlier chunk, and inside a chunk all reads come
// before the writes. Entries that do not ascend inside [0, nodes) end the path.
template <class W>
__device__ __forceinline__ void accept_move(uint8_t* base, int row_bytes, const long long* src, const long long* dst,
                                            int n) {
    const int per = row_bytes / (int)sizeof(W);
    constexpr int kHold = 4;
    for (int c = 0; c < n * per; c += kAcceptThreads * kHold) {
        W hold[kHold];
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
            const int x = c + k * kAcceptThreads + (int)threadIdx.x;
            if (x < n * per && src[x / per] >= 0)
                hold[k] = *reinterpret_cast<const W*>(base + src[x / per] * row_bytes + (x % per) * sizeof(W));
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
            const int x = c + k * kAcceptThreads + (int)threadIdx.x;
            if (x < n * per && src[x / per] >= 0)
                *reinterpret_cast<W*>(base + dst[x / per] * row_bytes + (x % per) * sizeof(W)) = hold[k];
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kAcceptThreads) accept_tree_kernel(const AcceptParams p);

}  // namespace va
