// Pages of a paged KV cache: sequences forked, reordered and freed with their
// last pages copied (fork), and the pages in use moved to the front of the
// pool (compact). No reference counterpart: the reference's cache is one
// contiguous buffer of one sequence.
//
// refs[p] counts the table entries that hold page p; 0 is a free page. All
// results are the same from run to run: pages are given out lowest number
// first, in the order (sequence, place), and counts are sums of integers.
#pragma once

#include "common.cuh"

namespace va {

constexpr int kPlanThreads = 1024;

// The four buffers of a pool of `layers` layers, each [num_pages][page bytes].
struct PoolView {
    uint8_t* base[4];      // K, V, scK, scV (null: absent)
    int row_bytes[4];      // per row
    int Hkv, page_rows, num_pages, layers;
};

struct ForkParams {
    PoolView pool;
    const int* refs;
    const int* table;   // [Bin][max_pages]
    const int* lens;    // [Bin]
    const int* parent;  // [Bout]
    int* new_refs;
    int* new_table;     // [Bout][max_pages]
    int* new_lens;
    int* shortage;
    int* free_list;     // workspace [num_pages]: the free pages to give out, past the first kFreeHere
    int* copy;          // workspace [3][Bout]: from, to, rows
    int Bin, Bout, max_pages, reserve;
};

struct CompactParams {
    PoolView pool;
    const int* refs;
    const int* table;   // [B][max_pages]
    int* new_refs;
    int* new_table;
    int* used;
    int* map;           // workspace [num_pages]: where a moved page went
    int* from;          // workspace [num_pages]
    int* to;            // workspace [num_pages]
    int* count;         // workspace [1]
    long long entries;  // B * max_pages
};

// Exclusive prefix sum of one value per thread over the CTA; s: 33 ints.
__device__ __forceinline__ int block_scan(int v, int* s, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s[warp] = x;
    __syncthreads();
    if (warp == 0) {
        const int nw = blockDim.x >> 5;
        int y = lane < nw ? s[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        s[lane] = y;
    }
    __syncthreads();
    const int before = warp ? s[warp - 1] : 0;
    total = s[(blockDim.x >> 5) - 1];
    __syncthreads();
    return before + x - v;
}

__device__ __forceinline__ int valid_page(int e, int num_pages) { return e >= 0 && e < num_pages ? e : -1; }

}  // namespace va
