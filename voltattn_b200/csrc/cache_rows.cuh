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
};

template <class T>
__device__ __forceinline__ void load8(const T* src, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4* p = reinterpret_cast<const float4*>(src);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
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
        const bool past = k + lane < B && __ldg(cu + k + lane + 1) <= token;
        const int c = __popc(__ballot_sync(0xffffffffu, past));
        seq += c;
        if (c < 32) break;
    }
    return seq;
}

// A warp quantizes four 64-element groups of one token at a time (8 lanes a
// group), K's groups of all heads before V's; its sequence and page are looked
// up once per token.
template <int BITS, class T>
__global__ void __launch_bounds__(256) append_packed_kernel(const AppendParams p) {
    const int lane = threadIdx.x & 31;
    const int ng = p.D / kGroup, side_groups = p.Hkv * ng;
    const int quads = (2 * side_groups + 3) / 4;
    const long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    grid_dependency_wait();
    grid_launch_dependents();
    if (w >= (long long)p.T * quads) return;
    const int token = (int)(w / quads), quad = (int)(w - (long long)token * quads);
    const int seq = token_sequence(p.cu, p.B, token, lane);
    if (seq >= p.B) return;
    const int i = token - __ldg(p.cu + seq), at = __ldg(p.pos + seq);
    const long long row = (long long)at + i;
    if (i < 0 || at < 0 || row >= (long long)p.max_pages * p.page_rows) return;
    const int pi = (int)(row / p.page_rows);
    const int pg = __ldg(p.table + (size_t)seq * p.max_pages + pi);
    if (pg < 0 || pg >= p.num_pages) return;
    const int grp = quad * 4 + (lane >> 3), part = lane & 7;
    const bool active = grp < 2 * side_groups;
    const bool is_v = grp >= side_groups;
    const int sg = active ? grp - (is_v ? side_groups : 0) : 0;
    const int h = sg / ng, gi = sg - h * ng;
    const T* src = is_v ? static_cast<const T*>(p.v) + token * p.vt + h * p.vh
                        : static_cast<const T*>(p.k) + token * p.kt + h * p.kh;
    float v[8];
    load8(src + gi * kGroup + part * 8, v);
    const long long r = ((long long)pg * p.Hkv + h) * p.page_rows + (row - (long long)pi * p.page_rows);
    uint8_t* codes = is_v ? p.V : p.K;
    const long long e0 = r * p.D + gi * kGroup + part * 8;
    if constexpr (BITS == 16 || BITS == kBitsBf16) {
        if (!active) return;
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (BITS == 16) {
                const __half2 x = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
                o[k] = *reinterpret_cast<const uint32_t*>(&x);
            } else {
                const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                o[k] = *reinterpret_cast<const uint32_t*>(&x);
            }
        }
        *reinterpret_cast<uint4*>(codes + e0 * 2) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
        quantize_group_values<BITS>(v, active, part, e0, r * ng + gi, codes, is_v ? p.scV : p.scK);
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
