// Tree attention over a paged cache on the Blackwell tensor cores: the
// operator of decode_tree.cuh (its mathematics, masks, splits and slots) for many
// query rows, with tcgen05.mma and accumulators in tensor memory.
//
// One CTA per SM, each with an equal window of the call's blocks of positions (with S = 1 a CTA per
// tile of query rows): the ranges in it, of one (sequence, KV head, tile) each, one after the other.
// 23 warps:
//   warps 0-15   softmax: thread (group w, half hf, row r) has 32 of the 64 positions of
//                query row r (TMEM lane r) in the jobs of group w;
//   warps 16, 17  producers of K tiles, 18, 19 of V tiles: codes -> exact fp16 codes in
//                swizzled tiles (fp16 rows: warps 16-19 mend the V tiles of the last blocks);
//   warp 20      one elected lane issues the S products, warp 22 the P V products (one
//                warp for both made each wait for the other's barriers);
//   warp 21      copies: blocks of codes and scales into a ring, several ahead (fp16
//                rows by tensor copies straight into the swizzled tiles).
// A job is one block of 64 positions against 128 query rows; the groups take the jobs in
// turn, so one group's exponentials run under the other's loads and exchange. kTwo = false
// (up to 128 query rows): job j is block j, one O, and the groups hand the rows' references
// on from job to job. kTwo = true (up to 256): jobs 2 i, 2 i + 1 are block i against
// rows 0..127 and 128..255, group w has rows and O of its own, and a decoded tile serves
// twice. TMEM holds the O's and kNS buffers of scores, job j's in buffer j % kNS.
//
// Per job j:
//   S_g = Q_g K_g^T (M = 128 rows, N = 64 positions) for each 64-dim group g, in
//     TMEM. The K tile holds the exact codes (times a power of two), so the group
//     scales multiply fp32 scores, as in decode_tree.cuh;
//   the softmax threads load their scores, x = S_0 k_0 + S_1 k_1, exchange the row's
//     maximum, and write P'_g = fp16(w v_g) over the scores;
//   O_g += P'_g V_g (A = P' read from TMEM, B = the V tile read MN-major).
// S(j + kNS) overwrites the buffer of job j once PV(j) has completed; the MMAs of one
// thread complete in issue order, so a completed PV(j) implies every earlier one.
// O is rescaled only when a row's reference, the most of score + own V scale (log2) that it
// sees, grows by more than kTcLag: a row's largest P' stays in [2^10, 2^16), its one rounding
// relative (with two groups, that of the group with the larger scale).
//
// The K and V tiles are the canonical 128-byte-swizzled layout, one panel of 64
// rows per 64-dim group. Packed codes are placed two dims apart by 4 in each
// 32-bit word ((0, 4), (1, 5), ...), which costs no byte permutes; Q's columns are
// stored in the same order and the output's are put back.
//
// Bound by what the roles share: issue slots (60 % busy) and shared memory. A block of 64
// positions against 128 rows takes 1.32 us and 5650 warp-instructions, start and merge included. In
// copies with parts cut out (303 us before the windows): no loads of scales 270, no stores of decoded
// tiles 261, a quarter of the MMAs 293, no exponentials 295. 736 threads leave 80 registers each: the
// softmax spills 28 to 172 bytes at D = 128 (20 to 116 at 64), and where it does decides a few percent.
// Measured: 8 sequences of 16384 to 32768 rows, q4+, 32 nodes, 32 query / 8 KV heads, 232 us, 470
// TFLOP/s (598 us in tiles of 16); 16 of 2048 to 8192, f16+, 64 nodes, 32 / 4 heads, 146 us, 627
// TFLOP/s, in a loop of seconds at the 1000 W power cap, 121 to 124 in a burst.
#pragma once

#include "decode_tree.cuh"
#include "prefill_tc.cuh"

namespace va {

template <Kind K, int kDim, bool kTwoTiles>
struct TreeTcCfg {
    static constexpr Kind kKind = K;
    static constexpr int kD = kDim;
    static constexpr bool kTwo = kTwoTiles;
    static constexpr int kRows = kTwoTiles ? 256 : 128;
    static constexpr int kNG = kDim / 64;
    static constexpr bool kScaled = !(K == Kind::F16 || K == Kind::BF16);
    static constexpr bool kFloat = is_float_kind(K);
    static constexpr bool kPairs4 = K == Kind::Q4 || K == Kind::Q3;  // dims (p, p + 4) in a word
    static constexpr int kSG = kScaled ? kNG : 1;  // score accumulators, weight copies
    static constexpr int kRb = kDim * KindTraits<K>::kBits / 8;
    static constexpr int kNb = 64;                 // positions of a block
    static constexpr int kSw = 64 * kSG;           // TMEM columns of a buffer of scores
    static constexpr int kNS = kSG == 2 ? (kTwoTiles ? 2 : 3) : 4;
    static constexpr int kOCols = kTwoTiles ? 256 : 128;  // TMEM: O, then the scores
    static_assert(kOCols + kNS * kSw <= 512, "tensor memory");
    static constexpr int kProducers = 128;
    static constexpr int kThreads = 23 * 32;
    static constexpr int kQTile = 128 * kDim * 2;
    static constexpr int kTile = kNb * kDim * 2;   // one K or V tile
    static constexpr bool kDirect = K == Kind::F16;  // tiles by tensor copies
    static constexpr int kKS = kDirect ? (kTwoTiles ? 3 : 4) : 2;
    static constexpr int kVS = kKS;
    static constexpr int kOffK = (kTwoTiles ? 2 : 1) * kQTile;
    static constexpr int kOffV = kOffK + kKS * kTile;
    static constexpr int kOffRaw = kOffV + kVS * kTile;        // ring of blocks as they lie in the cache
    static constexpr int kSb = kScaled ? 2 * kNG : 0;
    static constexpr int kRawV = kNb * kRb, kRawSK = 2 * kNb * kRb, kRawSV = kRawSK + kNb * kSb;
    static constexpr int kRawTx = kRawSV + kNb * kSb;
    static constexpr int kRawStage = (kRawTx + 127) / 128 * 128;
    // what follows the ring: scales as floats [8 slots][K, V][kNG][64] and log2 [64], masks,
    // [2][2][2][128] maxima or sums, [2][128] references, barriers, TMEM slot, fail, special, ticket, plan, two ranges
    static constexpr int kScaleSlots = 8;
    static constexpr int kScaleSlot = (2 * kNG + 1) * kNb * 4;
    static constexpr int kScaleV = kNG * kNb * 4;  // where a slot's V scales begin, and their log2
    static constexpr int kScaleLog = 2 * kScaleV;
    static constexpr int kScaleBytes = kScaled ? kScaleSlots * kScaleSlot : 0;
    static constexpr int kRest = kScaleBytes + kRows * 8 + 5120 + 512 + 192;
    static constexpr int kRoom = (227 * 1024 - 1024 - kOffRaw - kRest) / kRawStage;
    static constexpr int kRawStages = kDirect ? 1 : kRoom < 8 ? kRoom : 8;
    // (the merge of the ranges takes the front of shared memory: what follows stays past it)
    static constexpr int kStageRow = kDim + 4;  // floats of a row of the epilogue's stage, there as well
    static constexpr int kMergeBytes =
        (kRows * (kTreeMaxSplits + 1 > kStageRow ? kTreeMaxSplits + 1 : kStageRow) * 4 + 127) / 128 * 128;
    static constexpr int kRingEnd = kOffRaw + (kDirect ? 0 : kRawStages * kRawStage);
    static constexpr int kOffScales = kRingEnd > kMergeBytes ? kRingEnd : kMergeBytes;
    static constexpr int kOffMask = kOffScales + kScaleBytes;
    static constexpr int kOffMl = kOffMask + kRows * 8;
    static constexpr int kOffBars = kOffMl + 5120;
    static constexpr int kBars = 2 * kKS + 3 * kVS + 3 * kNS + 4 + 3 + kScaleSlots + 2 * kRawStages;
    static constexpr int kOffMisc = kOffBars + kBars * 8;
    static constexpr int kSmemBytes = 1024 + kOffMisc + 192;
    static_assert((kDirect || kRawStages >= 2) && kBars * 8 <= 512, "two blocks in flight");
    static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM");
};

// Placed K codes: the code / kTcInvStep.
template <Kind K>
__host__ __device__ constexpr float tc_k_inv_step() {
    return K == Kind::Q4 ? 64.f : K == Kind::Q3 ? 128.f : 1.f;
}
// Placed V codes: the code of pair p (dims p, p + 4) / this.
template <Kind K>
__host__ __device__ constexpr float tc_v_step(int p) {
    return K == Kind::Q4 ? ((p & 1) ? 64.f : 1024.f)
                         : K == Kind::Q3 ? (p == 1 ? 128.f : p == 2 ? 16.f : 1024.f) : 1.f;
}

// The codes of kDim / 4 consecutive dims of one row in shared memory (quarter q).
template <Kind K, int kDim>
struct TcRaw {
    static constexpr int kDims = kDim / 4;
    static constexpr int kWords = K == Kind::Q3 ? (kDims == 32 ? 3 : 2) : kDims * KindTraits<K>::kBits / 32;
    uint32_t w[kWords];
};

template <Kind K, int kDim>
__device__ __forceinline__ void tc_load(TcRaw<K, kDim>& r, const uint8_t* row, int q) {
    constexpr int kBytes = TcRaw<K, kDim>::kDims * KindTraits<K>::kBits / 8;
    if constexpr (K == Kind::Q3) {
        // 12 bytes of 4-byte alignment, or the two words around 6
        const uint32_t* p = reinterpret_cast<const uint32_t*>(row + ((q * kBytes) & ~3));
#pragma unroll
        for (int i = 0; i < TcRaw<K, kDim>::kWords; ++i) r.w[i] = p[i];
        if constexpr (kBytes == 6) {
            const uint32_t sh = (q & 1) * 16;
            r.w[0] = __funnelshift_r(r.w[0], r.w[1], sh);
            r.w[1] >>= sh;
        }
    } else if constexpr (kBytes == 8) {
        const uint2 v = reinterpret_cast<const uint2*>(row)[q];
        r.w[0] = v.x;
        r.w[1] = v.y;
    } else {
        const uint4* p = reinterpret_cast<const uint4*>(row) + q * (kBytes / 16);
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) {
            const uint4 v = p[i];
            r.w[4 * i] = v.x;
            r.w[4 * i + 1] = v.y;
            r.w[4 * i + 2] = v.z;
            r.w[4 * i + 3] = v.w;
        }
    }
}

// Eight dims (chunk j of the slice) as fp16, centred: exact.
template <Kind K, int kDim, bool kIsV>
__device__ __forceinline__ uint4 tc_convert(const TcRaw<K, kDim>& r, int j) {
    constexpr uint32_t kOne = 0x3C003C00u;
    uint32_t h[4] = {};
    if constexpr (K == Kind::F16) {
        return make_uint4(r.w[4 * j], r.w[4 * j + 1], r.w[4 * j + 2], r.w[4 * j + 3]);
    } else if constexpr (K == Kind::BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = bf2_to_h2(r.w[4 * j + i]);
    } else if constexpr (K == Kind::F8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = f8x2_to_h2(r.w[2 * j + (i >> 1)] >> (16 * (i & 1)));
    } else if constexpr (K == Kind::Q8) {
        const __half2 off = __float2half2_rn(1152.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = r.w[2 * j + (i >> 1)] ^ 0x80808080u;
            h[i] = h2_bits(__hsub2(bits_h2(__byte_perm(u, 0x64646464u, (i & 1) ? 0x4342 : 0x4140)), off));
        }
    } else if constexpr (K == Kind::Q4) {
        const uint32_t w = r.w[j];
        const __half2 o64 = __float2half2_rn(1.f + 8.f / 64.f), o1024 = __float2half2_rn(1.f + 8.f / 1024.f);
        if constexpr (kIsV) {
            const uint32_t u = w >> 8;
            h[0] = h2_bits(__hsub2(bits_h2((w & 0x000F000Fu) | kOne), o1024));
            h[1] = h2_bits(__hsub2(bits_h2((w & 0x00F000F0u) | kOne), o64));
            h[2] = h2_bits(__hsub2(bits_h2((u & 0x000F000Fu) | kOne), o1024));
            h[3] = h2_bits(__hsub2(bits_h2((u & 0x00F000F0u) | kOne), o64));
        } else {
            h[0] = h2_bits(__hsub2(bits_h2(((w << 4) & 0x00F000F0u) | kOne), o64));
            h[1] = h2_bits(__hsub2(bits_h2((w & 0x00F000F0u) | kOne), o64));
            h[2] = h2_bits(__hsub2(bits_h2(((w >> 4) & 0x00F000F0u) | kOne), o64));
            h[3] = h2_bits(__hsub2(bits_h2(((w >> 8) & 0x00F000F0u) | kOne), o64));
        }
    } else {
        // bits 24 j .. 24 j + 23 of the slice: fields 0..3 to the low half, 4..7 to the high one
        const int i0 = (24 * j) >> 5, sh = (24 * j) & 31;
        const uint32_t w = sh > 8 && i0 + 1 < TcRaw<K, kDim>::kWords ? __funnelshift_r(r.w[i0], r.w[i0 + 1], sh) : r.w[i0] >> sh;
        const uint32_t u = __byte_perm(w, w >> 12, 0x5410);
        const __half2 o128 = __float2half2_rn(1.f + 4.f / 128.f);
        if constexpr (kIsV) {
            const __half2 o1024 = __float2half2_rn(1.f + 4.f / 1024.f), o16 = __float2half2_rn(1.f + 4.f / 16.f);
            h[0] = h2_bits(__hsub2(bits_h2((u & 0x00070007u) | kOne), o1024));
            h[1] = h2_bits(__hsub2(bits_h2((u & 0x00380038u) | kOne), o128));
            h[2] = h2_bits(__hsub2(bits_h2((u & 0x01C001C0u) | kOne), o16));
            h[3] = h2_bits(__hsub2(bits_h2(((u >> 9) & 0x00070007u) | kOne), o1024));
        } else {
            h[0] = h2_bits(__hsub2(bits_h2(((u << 3) & 0x00380038u) | kOne), o128));
            h[1] = h2_bits(__hsub2(bits_h2((u & 0x00380038u) | kOne), o128));
            h[2] = h2_bits(__hsub2(bits_h2(((u >> 3) & 0x00380038u) | kOne), o128));
            h[3] = h2_bits(__hsub2(bits_h2(((u >> 6) & 0x00380038u) | kOne), o128));
        }
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
}

// 16 consecutive fp32 columns of this thread's TMEM lane, without the wait (as
// tmem_ld32_nowait), and the tie to it.
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_tie16(uint32_t* r) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]));
}

// True in one lane of the (converged) warp. The values around it stay warp-uniform,
// so the operands of the MMAs need no move from vector to uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

// Four floats of shared memory. Not volatile: the compiler may move the load over
// stores (the caller's address comes out of a statement that follows the wait).
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 v;
    asm("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// The same for eight fp16 values.
__device__ __forceinline__ bool clear_not_finite(uint4& v) {
    return clear_not_finite(v.x) | clear_not_finite(v.y) | clear_not_finite(v.z) | clear_not_finite(v.w);
}

// fp16 rows: the V tiles of blocks that hold drafted rows or the end are mended where
// they landed (rows past the end cleared, entries that are not finite too), and every
// tile is passed on to the MMAs. 128 threads: thread (row, half of the dims).
template <class C>
__device__ __forceinline__ void tree_tc_fix_v(int p0, int len, int ctx, int nblk, uint8_t* smem, uint64_t* vraw,
                                              uint64_t* vfull, volatile int* special, volatile int* fail) {
    const int t = (int)threadIdx.x - 512, lane = t & 31, row = t >> 1;
    for (int i = 0; i < nblk; ++i) {
        const int s = i % C::kVS, pb = p0 + i * C::kNb;
        if (!mbar_wait_bounded(vraw + s, (uint32_t)(i / C::kVS) & 1u)) {
            if (lane == 0) report_error(kErrFullWait);
            *fail = 1;
            return;
        }
        if (pb + C::kNb > ctx && pb + row >= ctx) {
            uint8_t* tile = smem + C::kOffV + s * C::kTile;
            for (int c = (t & 1) * (C::kD / 16); c < ((t & 1) + 1) * (C::kD / 16); ++c) {
                uint4* at = reinterpret_cast<uint4*>(tile + (c >> 3) * (C::kNb * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
                uint4 v = *at;
                if (pb + row >= len) *at = make_uint4(0u, 0u, 0u, 0u);
                else if (clear_not_finite(v)) *special = 1, *at = v;
            }
            fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(vfull + s);
    }
}

// Rows of a block's copies: the most of 64, 32, 16 and 8 that divide a page's, so that no
// copy leaves its page.
__host__ __device__ constexpr int tree_tc_run(int page_rows) {
    return page_rows % 64 == 0 ? 64 : page_rows % 32 == 0 ? 32 : page_rows % 16 == 0 ? 16 : 8;
}

// A CTA's share of the call (splits allowed), and the part of it that comes next.
struct TreeTcPlan {
    int window, at, end;  // cost units
    int more;             // whether there is a range at `at`
    int b0, base;         // the 32 sequences that held the last one, and the units before them
};
struct TreeTcRange {
    int b, hk, tile, len, n;    // rows of the sequence, drafted ones
    int p0, p1, part, parts;    // positions [p0, p1): one of the tile's parts (parts = 0: no work)
};

// The work in a line: sequences, their KV heads, their tiles of query rows, each tile
// its sequence's blocks of 64 positions. CTA i takes the i-th window of it, so every CTA
// has the same number of blocks whatever the lengths (a range per CTA in proportion to its
// sequence's length left the SMs idle for a third of the call). A tile counts kTcFixed blocks more
// than it has, about what starting and writing it takes (6 to 14 measure the same); one
// without live rows counts 1. Windows are long enough that none of a tile's blocks need more
// than S of them.
constexpr int kTcFixed = 8, kTcMinWindow = 8;

struct TreeTcSeq {
    int len, n, blocks, live_tiles;
    int cost;  // of one KV head
};
template <class C>
__device__ __forceinline__ TreeTcSeq tree_tc_seq(const TreeParams& p, int b) {
    const long long cap = (long long)p.max_pages * p.page_rows;
    TreeTcSeq q;
    q.len = (int)max(0ll, min((long long)load_global(p.lens + b), cap));
    q.n = max(0, min(min(p.nodes ? load_global(p.nodes + b) : p.Q, p.Q), q.len));
    q.blocks = (int)(((unsigned)q.len + C::kNb - 1) / C::kNb);
    q.live_tiles = (min(p.R, q.n * p.G) + C::kRows - 1) / C::kRows;
    q.cost = q.live_tiles * (q.blocks + kTcFixed) + (p.tiles - q.live_tiles);
    return q;
}

// (one warp) The sequence that position `at` of the line lies in, and the range that the
// CTA's window has of its tile from there on.
template <class C>
__device__ __forceinline__ void tree_tc_take(const TreeParams& p, const TreeTcSeq& q, int b, int base, int upto, int at, int window,
                                             int end, TreeTcPlan* plan, TreeTcRange* range) {
    const int y0 = at - (upto - q.cost * p.Hkv);
    if (y0 < 0 || upto <= at) return;  // one lane's sequence has it
    const int each = q.blocks + kTcFixed, hk = y0 / q.cost, y = y0 - hk * q.cost, live = q.live_tiles * each;
    TreeTcRange r = {b, hk, q.live_tiles + y - live, q.len, q.n, 0, 0, 0, 1};
    int next = at + 1;
    if (y < live) {
        r.tile = y / each;
        const int first = at - (y - r.tile * each) + kTcFixed;  // where its blocks begin
        next = min(end, first + q.blocks);
        r.p0 = max(0, at - first) * C::kNb;
        r.p1 = (int)min((long long)max(0, next - first) * C::kNb, (long long)q.len);
        // (a window that ends before the tile's blocks leaves it to the next)
        const int w0 = first / window;
        r.part = (int)blockIdx.x - w0;
        r.parts = next > first ? (first + q.blocks - 1) / window - w0 + 1 : 0;
    }
    *range = r;
    plan->at = next;
    plan->b0 = b & ~31;
    plan->base = base;
}

// inclusive sums over the lanes
__device__ __forceinline__ int tree_tc_scan(int x, int lane) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += up;
    }
    return x;
}

// (one warp) The next range of the CTA's window.
template <class C>
__device__ __forceinline__ void tree_tc_next(const TreeParams& p, int lane, TreeTcPlan* plan, TreeTcRange* range) {
    const int window = plan->window, at = plan->at, end = plan->end;
    int base = plan->base, b0 = plan->b0;
    __syncwarp();
    if (lane == 0) plan->more = at < end;
    for (; at < end && base <= at && b0 < p.B; b0 += 32) {
        TreeTcSeq q = {0, 0, 0, 0, 0};
        if (b0 + lane < p.B) q = tree_tc_seq<C>(p, b0 + lane);
        const int upto = tree_tc_scan(q.cost * p.Hkv, lane) + base;
        tree_tc_take<C>(p, q, b0 + lane, base, upto, at, window, end, plan, range);
        base = __shfl_sync(0xffffffffu, upto, 31);
    }
}

// (one warp) The CTA's window, and its first range.
template <class C>
__device__ __forceinline__ void tree_tc_plan(const TreeParams& p, int lane, TreeTcPlan* plan, TreeTcRange* range) {
    int total = 0, most = 0;
    TreeTcSeq q;
    int upto;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        q = {0, 0, 0, 0, 0};
        if (b0 + lane < p.B) q = tree_tc_seq<C>(p, b0 + lane);
        upto = tree_tc_scan(q.cost * p.Hkv, lane) + total;
        total = __shfl_sync(0xffffffffu, upto, 31);
        most = max(most, q.blocks);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    const int grid = (int)gridDim.x;
    const int window = max(max((total - 1) / grid + 1, (most + p.S - 2) / (p.S - 1)), kTcMinWindow);
    // (the product fits: at least one CTA before this one had a window of its own, or it is past the end)
    const bool some = (long long)blockIdx.x * window < total;
    const int at = some ? (int)blockIdx.x * window : total, end = min((long long)total, (long long)at + window);
    if (lane == 0) {
        plan->window = window;
        plan->at = at;
        plan->end = end;
        plan->more = some;
        plan->b0 = plan->base = 0;
    }
    __syncwarp();
    if (!some) return;
    if (p.B <= 32) tree_tc_take<C>(p, q, lane, 0, upto, at, window, end, plan, range);
    else tree_tc_next<C>(p, lane, plan, range);
}

// As kTreeBase and kTreeLag: a move costs more here, O's way through registers.
constexpr float kTcBase = 10.f, kTcLag = 4.9f;

// Four columns of query row r of a (sequence, KV head).
struct TreeTcStore {
    const TreeParams& p;
    int b, hk, n;
    __device__ __forceinline__ void operator()(int r, int c, float4 v, float inv) const {
        const int node = p.node_of(r);
        __half* dst = p.out + b * p.os_b + node * p.os_t + (long long)(hk * p.G + (r - node * p.G)) * p.os_h + 4 * c;
        const bool on = node < n && inv != 0.f;
        const __half2 x = __floats2half2_rn(on ? v.x * inv : 0.f, on ? v.y * inv : 0.f);
        const __half2 y = __floats2half2_rn(on ? v.z * inv : 0.f, on ? v.w * inv : 0.f);
        *reinterpret_cast<uint2*>(dst) = make_uint2(h2_bits(x), h2_bits(y));
    }
};

// One range of a tile's positions; false: a wait gave up.
template <class C>
__device__ __forceinline__ bool tree_tc_range(const TreeParams& p, const CUtensorMap& tmK, const CUtensorMap& tmV, uint8_t* smem,
                                              int slot, bool final) {
    constexpr int D = C::kD, NG = C::kNG, NB = C::kNb, KS = C::kKS, VS = C::kVS, SG = C::kSG, NS = C::kNS;
    constexpr Kind KK = C::kKind;
    unsigned long long* s_mask = reinterpret_cast<unsigned long long*>(smem + C::kOffMask);
    float* s_xch = reinterpret_cast<float*>(smem + C::kOffMl);  // [2][2][2][128]
    float* s_ref = s_xch + 1024;                                // [2][128]
    uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
    uint64_t *kempty = kfull + KS, *vfull = kempty + KS, *vempty = vfull + VS, *sfull = vempty + VS;
    uint64_t *pfull = sfull + NS, *pvdone = pfull + NS, *refbar = pvdone + NS, *fin = refbar + 4, *scfull = fin + 2;
    uint64_t *rfull = scfull + C::kScaleSlots, *rempty = rfull + C::kRawStages, *vraw = rempty + C::kRawStages;
    uint64_t* qfull = vraw + VS;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
    volatile int* fail = reinterpret_cast<volatile int*>(tslot + 1);
    volatile int* special = fail + 1;
    unsigned* s_ticket = tslot + 3;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    TreeTcPlan* plan = reinterpret_cast<TreeTcPlan*>(smem + C::kOffMisc + 64);
    TreeTcRange* ranges = reinterpret_cast<TreeTcRange*>(plan + 1);
    const TreeTcRange now = ranges[slot];
    const int b = now.b, hk = now.hk, r0 = now.tile * C::kRows, len = now.len, n = now.n, ctx = len - n;
    const int p0 = now.p0, p1 = now.p1;
    const int live = min(p.R, n * p.G) - r0;  // rows of the tile that belong to a node; none: zeros
    __syncthreads();

    if (live <= 0 || now.parts == 0) {  // (no rows of a node; or no blocks in this window)
        const TreeTcStore store_out = {p, b, hk, n};
        const int rows_here = min(C::kRows, p.R - r0);
        for (int i = now.parts ? tid : rows_here * D; i < rows_here * (D / 4); i += C::kThreads)
            store_out(r0 + i / (D / 4), i % (D / 4), make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
        if (warp == 21) tree_tc_next<C>(p, lane, plan, ranges + 1 - slot);
        return true;
    }

    const int nblk = (p1 - p0 + NB - 1) / NB;
    const int njobs = C::kTwo ? 2 * nblk : nblk;
    if (tid == 0) {
        for (int i = 0; i < KS; ++i) mbar_init(kfull + i, C::kDirect ? 1 : 2), mbar_init(kempty + i, 1);
        for (int i = 0; i < VS; ++i) mbar_init(vfull + i, C::kDirect ? C::kProducers / 32 : 2), mbar_init(vempty + i, 1);
        for (int i = 0; i < NS; ++i) mbar_init(sfull + i, 1), mbar_init(pfull + i, 8), mbar_init(pvdone + i, 1);
        for (int i = 0; i < 4; ++i) mbar_init(refbar + i, 2);
        mbar_init(fin, 1);
        mbar_init(fin + 1, 1);
        mbar_init(qfull, 1);
        for (int i = 0; i < C::kScaleSlots; ++i) mbar_init(scfull + i, 1);
        for (int i = 0; i < C::kRawStages; ++i) mbar_init(rfull + i, 1), mbar_init(rempty + i, C::kProducers / 32);
        for (int i = 0; i < VS; ++i) mbar_init(vraw + i, 1);
        *special = 0;
        fence_mbar_init();
    }
    const int* trow = p.table + (size_t)b * p.max_pages;
    const auto page_of = [&](int pos, int& off) {
        const int pi = (int)((__umulhi((unsigned)pos, p.page_mul) + (unsigned)pos) >> p.page_shift);
        off = pos - pi * p.page_rows;
        const int pg = pi < p.max_pages ? load_global(trow + pi) : 0;
        return (unsigned)pg < (unsigned)p.num_pages ? pg : 0;
    };
    __syncthreads();
    const uint32_t tbase = *tslot;
    const uint32_t sbase = smem_u32(smem);

    // softmax threads: the reference (log2 units) and their half's sum
    float m_ref = kNegMax, l_sum = 0.f;
    const int set = warp >> 3, hf = (warp >> 2) & 1, row = tid & 127, quad = warp & 3;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    if (warp < 16) {
        // ---- softmax -------------------------------------------------------------
        // first the query rows into shared memory in the tiles' order of dims (all loads of a
        // thread before its stores), and their masks
        {
            constexpr int kPer = C::kRows * (D / 8) / 512;
            uint4 v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int x = tid + 512 * i, qr = x / (D / 8), c = x - qr * (D / 8);
                v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (qr < live) {
                    const int r = r0 + qr, node = p.node_of(r);
                    v[i] = load_global(reinterpret_cast<const uint4*>(p.q + b * p.qs_b + node * p.qs_t +
                                                                (long long)(hk * p.G + (r - node * p.G)) * p.qs_h) + c);
                }
            }
            const unsigned long long in_tree = n >= 64 ? ~0ull : (1ull << n) - 1ull;
            if (tid < C::kRows) s_mask[tid] = tid < live ? load_global(p.mask + (size_t)b * p.Q + p.node_of(r0 + tid)) & in_tree : 0ull;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int x = tid + 512 * i, qr = x / (D / 8), c = x - qr * (D / 8), rr = qr & 127;
                if constexpr (C::kPairs4)
                    v[i] = make_uint4(__byte_perm(v[i].x, v[i].z, 0x5410), __byte_perm(v[i].x, v[i].z, 0x7632),
                                      __byte_perm(v[i].y, v[i].w, 0x5410), __byte_perm(v[i].y, v[i].w, 0x7632));
                *reinterpret_cast<uint4*>(smem + (qr >> 7) * C::kQTile + (c >> 3) * 16384 + rr * 128 +
                                          (((c & 7) ^ (rr & 7)) << 4)) = v[i];
            }
            fence_proxy_async_smem();
            named_barrier_sync(1, 512);
            if (tid == 0) mbar_arrive(qfull);
        }
        const float c2 = rsqrtf((float)D) * kLog2e * tc_k_inv_step<KK>();
        const int w = set;
        // A quadrant's two warps meet at a barrier in every job, which has no limit of its own: one that
        // gives up a wait still comes to it for the jobs from `from` on, so that the other one ends too
        const bool live_quad = (C::kTwo ? w * 128 : 0) + quad * 32 < live;
        const auto give_up = [&](int from) {
            if (lane == 0) report_error(kErrFullWait);
            *fail = 1;
            if (live_quad)
                for (int k = from; k < njobs; k += 2) named_barrier_sync(2 + w * 4 + quad, 64);
        };
        for (int j = w; j < njobs; j += 2) {
            const int blk = C::kTwo ? j >> 1 : j, sb = j % NS;
            const uint32_t ph = (uint32_t)(j / NS) & 1u;
            const int pb = p0 + blk * NB;
            bool ok = mbar_wait_fast(sfull + sb, ph);
            // (block i + 8's scales overwrite block i's: its K tile waits for S(i + 6), issued
            // after block i + 2's products at the least, so this phase is not passed twice)
            if constexpr (C::kScaled)
                ok = ok && mbar_wait_fast(scfull + blk % C::kScaleSlots, (uint32_t)(blk / C::kScaleSlots) & 1u);
            if (__any_sync(0xffffffffu, !ok)) {
                give_up(j);
                break;
            }
            tc05_fence_after();
            // a quadrant without live rows only keeps the barriers' count
            if (live_quad) {
                uint32_t sc = sbase + C::kOffScales + (blk % C::kScaleSlots) * C::kScaleSlot;
                asm volatile("" : "+r"(sc));  // the loads of scales come after the waits
                const uint32_t tS = tbase + C::kOCols + sb * C::kSw + lane_addr, tO = tbase + (C::kTwo ? w * 128 : 0) + lane_addr;
                float x[32];
                // their maximum; with scales, of score (log2 units) + the log2 of the position's V
                // scale, taken as the scores come: in a pass of its own it held more registers (16
                // sequences of 1000 to 4000 rows, q8+, 256 query rows: 166 us against 136)
                float b0 = kNegMax, b1 = kNegMax;
                const auto raise = [&](uint32_t scales, int c, float2 u, float2 v) {
                    if constexpr (C::kScaled) {
                        const float4 lv = lds_f4(scales + C::kScaleLog + 4 * (32 * hf + c));
                        u = ffma2(u, make_float2(c2, c2), make_float2(lv.x, lv.y));
                        v = ffma2(v, make_float2(c2, c2), make_float2(lv.z, lv.w));
                    }
                    b0 = fmax3f(b0, u.x, u.y);
                    b1 = fmax3f(b1, v.x, v.y);
                };
#pragma unroll
                for (int cb = 0; cb < 32; cb += 16) {
                    uint32_t s0[16], s1[16];
                    tmem_ld16_nowait(tS + 32 * hf + cb, s0);
                    if constexpr (SG == 2) tmem_ld16_nowait(tS + 64 + 32 * hf + cb, s1);
                    tmem_wait_ld_only();
                    tmem_tie16(s0);
                    if constexpr (SG == 2) tmem_tie16(s1);
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        float2 u = make_float2(__uint_as_float(s0[c]), __uint_as_float(s0[c + 1]));
                        float2 v = make_float2(__uint_as_float(s0[c + 2]), __uint_as_float(s0[c + 3]));
                        if constexpr (C::kScaled) {
                            const float4 k0 = lds_f4(sc + 4 * (32 * hf + cb + c));
                            u = fmul2(u, make_float2(k0.x, k0.y));
                            v = fmul2(v, make_float2(k0.z, k0.w));
                            if constexpr (SG == 2) {
                                const float4 k1 = lds_f4(sc + 4 * (NB + 32 * hf + cb + c));
                                u = ffma2(make_float2(__uint_as_float(s1[c]), __uint_as_float(s1[c + 1])),
                                          make_float2(k1.x, k1.y), u);
                                v = ffma2(make_float2(__uint_as_float(s1[c + 2]), __uint_as_float(s1[c + 3])),
                                          make_float2(k1.z, k1.w), v);
                            }
                        }
                        x[cb + c] = u.x;
                        x[cb + c + 1] = u.y;
                        x[cb + c + 2] = v.x;
                        x[cb + c + 3] = v.y;
                        raise(sc, cb + c, u, v);
                    }
                }
                // which of its 32 columns the row sees
                const bool tail = pb + NB > ctx;
                uint32_t vis = 0xFFFFFFFFu;
                if (tail) {
                    const unsigned long long mk = s_mask[(C::kTwo ? w * 128 : 0) + row];
                    const int d = ctx - pb;  // < 64
                    const unsigned long long all = d > 0 ? (mk << d) | ((1ull << d) - 1ull) : -d < 64 ? mk >> -d : 0ull;
                    vis = (uint32_t)(all >> (32 * hf));
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(vis >> c & 1u)) x[c] = kNegMax;
                }
                if (tail) {
                    b0 = b1 = kNegMax;
                    // (sc once more: the compiler would hold all log2 loaded above until here)
                    uint32_t again = sbase + C::kOffScales + (blk % C::kScaleSlots) * C::kScaleSlot;
                    asm volatile("" : "+r"(again));
#pragma unroll
                    for (int c = 0; c < 32; c += 4) raise(again, c, make_float2(x[c], x[c + 1]), make_float2(x[c + 2], x[c + 3]));
                }
                // the row's maximum over both halves; their barrier also puts every load of S
                // before the stores of P' below
                float* xch = s_xch + w * 512 + (j >> 1 & 1) * 256;
                xch[hf * 128 + row] = fmaxf(b0, b1);
                named_barrier_sync(2 + w * 4 + quad, 64);
                const float bm = fmaxf(fmaxf(b0, b1), xch[(1 - hf) * 128 + row]);
                // (a score far below any product of finite numbers: the row sees none of the block)
                const float want = bm < -1e37f ? kNegMax : C::kScaled ? bm - kTcBase : fmaf(bm, c2, -kTcBase);
                // the reference that O has so far: the row's own (two tiles), or what the other
                // group left after job j - 1 (two slots, each rewritten two jobs on, after both
                // halves have read it)
                float oref = m_ref;
                if constexpr (!C::kTwo) {
                    if (j > 0) {
                        ok = mbar_wait_fast(refbar + quad, (uint32_t)(j - 1) & 1u);
                        oref = s_ref[((j - 1) & 1) * 128 + row];
                    }
                }
                const float nref = want > oref + kTcLag ? want : oref;
                if constexpr (!C::kTwo) {
                    if (hf == 0) s_ref[(j & 1) * 128 + row] = nref;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(refbar + quad);
                }
                l_sum *= fast_exp2(m_ref - nref);
                m_ref = nref;
                const int prev = j - (C::kTwo ? 2 : 1);  // the last job into this O
                if (__any_sync(0xffffffffu, nref != oref) && prev >= 0) {
                    // this half of the row's O, once its earlier products are in
                    ok = ok && mbar_wait_fast(pvdone + prev % NS, (uint32_t)(prev / NS) & 1u);
                    tc05_fence_after();
                    const float corr = fast_exp2(oref - nref);
#pragma unroll 1
                    for (int cb = 0; cb < D / 2; cb += 16) {
                        uint32_t o[16];
                        tmem_ld16_nowait(tO + hf * (D / 2) + cb, o);
                        tmem_wait_ld_only();
                        tmem_tie16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                        tmem_st16_u(tO + hf * (D / 2) + cb, o);
                    }
                }
                if (__any_sync(0xffffffffu, !ok)) {
                    give_up(j + 2);
                    break;
                }
                float2 sum = make_float2(0.f, 0.f);
                // (two instantiations: only blocks with drafted rows or the end select)
                const auto weights = [&](auto is_tail) {
                    constexpr bool kTail = decltype(is_tail)::value;
                    const float2 sc2 = make_float2(c2, c2), nm = make_float2(-nref, -nref);
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        const float2 y = ffma2(make_float2(x[c], x[c + 1]), sc2, nm);
                        float2 e = make_float2(fast_exp2(y.x), fast_exp2(y.y));
                        if constexpr (kTail) {
                            if (!(vis >> c & 1u)) e.x = 0.f;
                            if (!(vis >> (c + 1) & 1u)) e.y = 0.f;
                        }
                        sum = fadd2(sum, e);
                        x[c] = e.x;
                        x[c + 1] = e.y;
                    }
#pragma unroll
                    for (int g = 0; g < SG; ++g) {
                        uint32_t h[16];  // P'_g, pairs of positions
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            float2 u = make_float2(x[c], x[c + 1]), v = make_float2(x[c + 2], x[c + 3]);
                            if constexpr (C::kScaled) {
                                const float4 f = lds_f4(sc + C::kScaleV + 4 * (g * NB + 32 * hf + c));
                                u = fmul2(u, make_float2(f.x, f.y));
                                v = fmul2(v, make_float2(f.z, f.w));
                                if constexpr (kTail) {  // an unseen row's scale may be nan
                                    if (!(vis >> c & 1u)) u.x = 0.f;
                                    if (!(vis >> (c + 1) & 1u)) u.y = 0.f;
                                    if (!(vis >> (c + 2) & 1u)) v.x = 0.f;
                                    if (!(vis >> (c + 3) & 1u)) v.y = 0.f;
                                }
                            }
                            h[c / 2] = h2_bits(__floats2half2_rn(u.x, u.y));
                            h[c / 2 + 1] = h2_bits(__floats2half2_rn(v.x, v.y));
                        }
                        tmem_st16_u(tS + 32 * g + 16 * hf, h);
                    }
                };
                if (tail) weights(std::true_type{});
                else weights(std::false_type{});
                l_sum += sum.x + sum.y;
                tmem_wait_st();
            }
            tc05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull + sb);
        }
        if (!*fail && !mbar_wait_fast(pvdone + (njobs - 1) % NS, (uint32_t)((njobs - 1) / NS) & 1u)) {  // every MMA of the CTA
            if (lane == 0) report_error(kErrFullWait);
            *fail = 1;
        }
        tc05_fence_after();
    } else if (C::kDirect && warp < 20) {
        tree_tc_fix_v<C>(p0, len, ctx, nblk, smem, vraw, vfull, special, fail);
    } else if (!C::kDirect && warp < 20) {
        // ---- producers: a thread takes four slices (row, quarter of the dims) of a tile -------
        const bool is_v = warp >= 18;
        const int pw = warp & 1;
        // lane bits: quarter bit 0, row bits 0..1, quarter bit 1, row bit 2: eight
        // neighbouring lanes store to eight different 16-byte banks
        const int q = (lane & 1) | ((lane >> 2) & 2), row0 = pw * 32 + ((lane >> 1) & 3) + ((lane >> 4) << 2);
        using Raw = TcRaw<KK, D>;
        constexpr int kChunks = Raw::kDims / 8;
        // where its chunks of row row0 go in a tile (rows 8 apart: 1024 bytes, the same phase)
        int to[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int c = q * kChunks + j;
            to[j] = (c >> 3) * (NB * 128) + row0 * 128 + (((c & 7) ^ (row0 & 7)) << 4);
        }
        bool ok = true;
        for (int i = 0; i < nblk; ++i) {
            const int rs = i % C::kRawStages;
            ok = mbar_wait_bounded(rfull + rs, (uint32_t)(i / C::kRawStages) & 1u);
            if (!ok) break;
            const uint8_t* raw = smem + C::kOffRaw + rs * C::kRawStage;
            if (!is_v) {
                const int s = i % KS;
                ok = i < KS || mbar_wait_bounded(kempty + s, (uint32_t)(i / KS - 1) & 1u);
                if (!ok) break;
                if (C::kScaled && pw == (i & 1)) {  // the block's scales: two positions a lane
                    float* sk = reinterpret_cast<float*>(smem + C::kOffScales + (i % C::kScaleSlots) * C::kScaleSlot);
                    float* sv = sk + C::kScaleV / 4;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int at = lane + 32 * e;
                        uint32_t ks, vs;
                        if constexpr (NG == 2) {
                            ks = reinterpret_cast<const uint32_t*>(raw + C::kRawSK)[at];
                            vs = reinterpret_cast<const uint32_t*>(raw + C::kRawSV)[at];
                        } else {
                            ks = reinterpret_cast<const uint16_t*>(raw + C::kRawSK)[at];
                            vs = reinterpret_cast<const uint16_t*>(raw + C::kRawSV)[at];
                        }
                        const float2 fk = __half22float2(bits_h2(ks)), fv = __half22float2(bits_h2(vs));
                        sk[at] = fk.x;
                        sv[at] = fv.x;
                        if constexpr (NG == 2) sk[NB + at] = fk.y, sv[NB + at] = fv.y;
                        sk[C::kScaleLog / 4 + at] = tree_scale_log2(bits_h2(vs));
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(scfull + i % C::kScaleSlots);
                }
                uint8_t* tile_at = smem + C::kOffK + s * C::kTile;
#pragma unroll
                for (int h = 0; h < 4; h += 2) {
                    Raw r[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) tc_load<KK, D>(r[e], raw + (row0 + 8 * (h + e)) * C::kRb, q);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < kChunks; ++j)
                            *reinterpret_cast<uint4*>(tile_at + to[j] + 1024 * (h + e)) = tc_convert<KK, D, false>(r[e], j);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(kfull + s);
                    mbar_arrive(rempty + rs);
                }
            } else {
                const int s = i % VS;
                ok = i < VS || mbar_wait_bounded(vempty + s, (uint32_t)(i / VS - 1) & 1u);
                if (!ok) break;
                uint8_t* tile_at = smem + C::kOffV + s * C::kTile;
#pragma unroll
                for (int h = 0; h < 4; h += 2) {
                    Raw r[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        tc_load<KK, D>(r[e], raw + C::kRawV + (row0 + 8 * (h + e)) * C::kRb, q);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = p0 + i * NB + row0 + 8 * (h + e);
#pragma unroll
                        for (int j = 0; j < kChunks; ++j) {
                            uint4 v = tc_convert<KK, D, true>(r[e], j);
                            if constexpr (C::kFloat) {
                                // rows past the end are cleared; entries of drafted rows that are not finite
                                // are left to the epilogue, which adds them to the rows that see them
                                if (pos >= len) v = make_uint4(0u, 0u, 0u, 0u);
                                else if (pos >= ctx && clear_not_finite(v)) *special = 1;
                            }
                            *reinterpret_cast<uint4*>(tile_at + to[j] + 1024 * (h + e)) = v;
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(vfull + s);
                    mbar_arrive(rempty + rs);
                }
            }
        }
        if (!ok) {
            if (lane == 0) report_error(kErrEmptyWait);
            *fail = 1;
        }
    } else if (C::kDirect && warp == 21) {
        // ---- copies of fp16 rows: tensor copies of 64 dims by the block's rows inside a
        // page into the swizzled tiles; lane = run + 8 * group
        const int run = tree_tc_run(p.page_rows), at = (lane & 7) * run, g = lane >> 3;
        const bool copies = at < NB && g < NG;
        int i = 0;
        bool ok = true;
        for (; ok && i < nblk; ++i) {
            int off = 0, pg = 0;
            if (copies) pg = page_of(p0 + i * NB + at, off);
            const int y = (int)(((long long)pg * p.Hkv + hk) * p.page_rows + off);
            const uint32_t o = g * (NB * 128) + at * 128;
            const int ks = i % KS, vs = i % VS;
            ok = i < KS || mbar_wait_bounded(kempty + ks, (uint32_t)(i / KS - 1) & 1u);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(kfull + ks, C::kTile);
            __syncwarp();
            if (copies) pf_tma_2d(sbase + C::kOffK + ks * C::kTile + o, &tmK, 64 * g, y, kfull + ks);
            ok = i < VS || mbar_wait_bounded(vempty + vs, (uint32_t)(i / VS - 1) & 1u);
            if (!ok) {
                (void)mbar_wait_bounded(kfull + ks, (uint32_t)(i / KS) & 1u);
                break;
            }
            if (lane == 0) mbar_arrive_expect_tx(vraw + vs, C::kTile);
            __syncwarp();
            if (copies) pf_tma_2d(sbase + C::kOffV + vs * C::kTile + o, &tmV, 64 * g, y, vraw + vs);
        }
        if (!ok) {
            if (lane == 0) report_error(kErrEmptyWait);
            *fail = 1;
        }
        // the copies in flight land (bounded) before the shared memory is given back
        for (int k = max(0, i - VS); k < i; ++k)
            if (!mbar_wait_bounded(kfull + k % KS, (uint32_t)(k / KS) & 1u) ||
                !mbar_wait_bounded(vraw + k % VS, (uint32_t)(k / VS) & 1u))
                *fail = 1;
    } else if (!C::kDirect && warp == 21) {
        // ---- copies: lane 4 r + k brings run r of buffer k (K, V, their scales)
        const int run = tree_tc_run(p.page_rows), nrun = NB / run, buf = lane & 3, at = (lane >> 2) * run;
        const int rb = buf < 2 ? C::kRb : C::kSb;
        const uint32_t bytes = (uint32_t)(run * rb);
        const bool copies = lane < 4 * nrun && bytes > 0;
        const uint8_t* src = buf == 0   ? p.K
                             : buf == 1 ? p.V
                             : buf == 2 ? reinterpret_cast<const uint8_t*>(p.scK)
                                        : reinterpret_cast<const uint8_t*>(p.scV);
        const int dst = C::kOffRaw + (buf == 0 ? 0 : buf == 1 ? C::kRawV : buf == 2 ? C::kRawSK : C::kRawSV) + at * rb;
        const uint64_t policy = l2_policy_evict_first();
        int i = 0;
        for (; i < nblk; ++i) {
            const int rs = i % C::kRawStages, u = i / C::kRawStages;
            if (u > 0 && !mbar_wait_bounded(rempty + rs, (uint32_t)(u - 1) & 1u)) {
                if (lane == 0) report_error(kErrEmptyWait);
                *fail = 1;
                break;
            }
            if (lane == 0) mbar_arrive_expect_tx(rfull + rs, C::kRawTx);
            __syncwarp();
            if (copies) {
                int off;
                const int pg = page_of(p0 + i * NB + at, off);
                bulk_g2s(smem + dst + rs * C::kRawStage, src + (((size_t)pg * p.Hkv + hk) * p.page_rows + off) * rb, bytes,
                         rfull + rs, policy);
            }
        }
        // the copies in flight land (bounded) before the shared memory is given back
        for (int k = max(0, i - C::kRawStages); k < i; ++k)
            if (!mbar_wait_bounded(rfull + k % C::kRawStages, (uint32_t)(k / C::kRawStages) & 1u)) *fail = 1;
    } else {
        // ---- the MMA warps: one elected lane of each issues ---------------------------
        constexpr uint32_t kIdescS = umma_idesc_f16(128, NB, false);
        constexpr uint32_t kIdescO = umma_idesc_f16(128, C::kScaled ? 64 : D, true);
        const uint32_t ub = __shfl_sync(0xffffffffu, sbase, 0), ut = __shfl_sync(0xffffffffu, tbase, 0);
        // descriptors differ in their start addresses only (16-byte units, no carry out of them)
        const uint64_t dq = umma_desc_sw128(ub, 16, 1024), dk = umma_desc_sw128(ub + C::kOffK, 16, 1024);
        const uint64_t dv = umma_desc_sw128(ub + C::kOffV, NB * 128, 1024);
        const auto issue_s = [&](int j) {
            const int w = j & 1, i = C::kTwo ? j >> 1 : j, s = i % KS, sb = j % NS;
            if (!mbar_wait_fast(kfull + s, (uint32_t)(i / KS) & 1u)) return false;
            // (job j - NS, the buffer's last)
            if (j >= NS && !mbar_wait_fast(pvdone + sb, (uint32_t)(j / NS - 1) & 1u)) return false;
            tc05_fence_after();
            const uint64_t qa = dq + (C::kTwo ? w * (C::kQTile / 16) : 0), ka = dk + s * (C::kTile / 16);
            const uint32_t d = ut + C::kOCols + sb * C::kSw;
            if (elect_one()) {
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_f16(d + (C::kScaled ? 64 * g : 0), qa + (g * 16384 + kk * 32) / 16, ka + (g * (NB * 128) + kk * 32) / 16,
                                 kIdescS, kk > 0 || (!C::kScaled && g > 0));
                umma_commit(sfull + sb);
                if (!C::kTwo || w == 1) umma_commit(kempty + s);
            }
            __syncwarp();
            return true;
        };
        const auto issue_pv = [&](int j) {
            const int w = j & 1, i = C::kTwo ? j >> 1 : j, s = i % VS, sb = j % NS;
            if (!mbar_wait_fast(vfull + s, (uint32_t)(i / VS) & 1u)) return false;
            if (!mbar_wait_fast(pfull + sb, (uint32_t)(j / NS) & 1u)) return false;
            tc05_fence_after();
            const uint64_t va = dv + s * (C::kTile / 16);
            const uint32_t o = ut + (C::kTwo ? w * 128 : 0), a = ut + C::kOCols + sb * C::kSw;
            const bool more = j >= (C::kTwo ? 2 : 1);  // O holds earlier products
            if (elect_one()) {
#pragma unroll
                for (int g = 0; g < SG; ++g)
#pragma unroll
                    for (int kk = 0; kk < NB / 16; ++kk)
                        umma_f16_ts(o + 64 * g, a + 32 * g + 8 * kk, va + (g * (NB * 128) + kk * 2048) / 16, kIdescO,
                                    more || kk > 0);
                if (!C::kTwo || w == 1) umma_commit(vempty + s);
                umma_commit(pvdone + sb);
            }
            __syncwarp();
            return true;
        };
        bool ok = true;
        if (warp == 20) {
            ok = mbar_wait_fast(qfull, 0);
            for (int j = 0; ok && j < njobs; ++j) ok = issue_s(j);
            for (int i = max(0, nblk - KS); ok && i < nblk; ++i) ok = mbar_wait_fast(kempty + i % KS, (uint32_t)(i / KS) & 1u);
        } else {
            for (int j = 0; ok && j < njobs; ++j) ok = issue_pv(j);
            for (int i = max(0, nblk - VS); ok && i < nblk; ++i) ok = mbar_wait_fast(vempty + i % VS, (uint32_t)(i / VS) & 1u);
        }
        if (!ok) {  // every MMA issued so far ends before the tensor memory is given back
            if (lane == 0) report_error(kErrFullWait);
            *fail = 1;
            if (elect_one()) umma_commit(fin + (warp == 22));
            (void)mbar_wait_bounded(fin + (warp == 22), 0);
        }
        __syncwarp();
    }
    tc05_fence_before();
    __syncthreads();
    tc05_fence_after();
    if (*fail) return false;
    // (every arrival has come: the warps above waited for the commits' as well)
    if (tid < C::kBars) mbar_inval(kfull + tid);
    if (final) grid_launch_dependents();

    // ---- epilogue: a thread's row, its part of the dims: half of them (two tiles: of its
    // group's tile) or a quarter
    // (read again: not held in registers over the loops)
    const volatile TreeTcRange* was = ranges + slot;
    const TreeTcStore store_out = {p, was->b, was->hk, was->n};
    const int stream = store_out.b * p.Hkv + store_out.hk, tile0 = was->tile, r0e = tile0 * C::kRows, split = was->part, nsplit = was->parts;
    const int rows_here = min(C::kRows, p.R - r0e), rows_live = min(p.R, store_out.n * p.G) - r0e;
    const bool direct = nsplit == 1;
    float* stage = reinterpret_cast<float*>(smem);
    if (warp < 16) {
        s_xch[(set * 2 + hf) * 128 + row] = l_sum;
        if (hf == 0) s_xch[512 + set * 128 + row] = m_ref;
        named_barrier_sync(1, 512);
        const auto sum_of = [&](int w) { return s_xch[w * 256 + row] + s_xch[w * 256 + 128 + row]; };
        const int qr = (C::kTwo ? set * 128 : 0) + row, r = r0e + qr;
        const bool on = (C::kTwo ? set * 128 : 0) + quad * 32 < rows_live;  // (the same for the whole warp)
        const int w0 = C::kTwo ? set : 0;
        float mx = s_xch[512 + w0 * 128 + row], sum = sum_of(w0);
        if constexpr (!C::kTwo) {  // O has the last reference, the larger; the sums each group's own
            const float m0 = mx, m1 = s_xch[512 + 128 + row];
            mx = fmaxf(m0, m1);
            sum = sum * fast_exp2(m0 - mx) + sum_of(1) * fast_exp2(m1 - mx);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float scale = direct ? on && qr < rows_live ? inv : 0.f : 1.f;  // (0: rows of no node, or that see nothing)
        float* mine = stage + qr * C::kStageRow;
        constexpr int kCols = C::kTwo ? D / 2 : D / 4;
        const int c0 = C::kTwo ? hf * kCols : (set * 2 + hf) * kCols;
#pragma unroll 1
        for (int cb = c0; cb < c0 + kCols; cb += 16) {
            __syncwarp();
            float o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0.f;
            if (on) {
                uint32_t u[16];
                tmem_ld16_nowait(tbase + w0 * 128 + lane_addr + cb, u);
                tmem_wait_ld_only();
                tmem_tie16(u);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(u[i]);
            }
            if constexpr (C::kFloat) {
                if (*special && qr < rows_live) {
                    const unsigned long long mk = s_mask[qr];
                    for (int j = max(0, p0 - ctx); j < n && ctx + j < p1; ++j) {
                        if (!(mk >> j & 1ull)) continue;
                        int off;
                        const int pg = page_of(ctx + j, off);
                        const uint8_t* vr = p.V + (((size_t)pg * p.Hkv + hk) * p.page_rows + off) * C::kRb;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = v_one<KK>(vr, cb + i);
                            if (!(fabsf(x) <= 65504.f)) o[i] += x;
                        }
                    }
                }
            }
            if (qr >= rows_here) continue;
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
                float v[8];
#pragma unroll
                for (int d = 0; d < 8; ++d)
                    v[d] = C::kPairs4 ? o[i + 2 * (d & 3) + (d >> 2)] * tc_v_step<KK>(d & 3) : o[i + d];
#pragma unroll
                for (int d = 0; d < 8; ++d) v[d] = scale != 0.f ? v[d] * scale : 0.f;
                *reinterpret_cast<float4*>(mine + cb + i) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(mine + cb + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
        if (!direct && on && c0 == 0 && qr < rows_here)
            __stcg(reinterpret_cast<float2*>(p.ws_ml) + ((size_t)stream * p.R + r) * p.S + split, make_float2(mx, sum));
    } else if (warp == 21) {
        tree_tc_next<C>(p, lane, plan, ranges + 1 - slot);
    }
    tc05_fence_before();
    __syncthreads();
    tc05_fence_after();
    // a row at a time: rows' stores by the threads that hold them took 4 us more a range
#pragma unroll 4
    for (int i = tid; i < rows_here * (D / 4); i += C::kThreads) {
        const int qr = i / (D / 4), c = i - qr * (D / 4);
        const float4 v = *reinterpret_cast<const float4*>(stage + qr * C::kStageRow + 4 * c);
        if (direct) store_out(r0e + qr, c, v, 1.f);
        else if (qr < rows_live) __stcg(reinterpret_cast<float4*>(p.ws_o + (((size_t)stream * p.R + r0e + qr) * p.S + split) * D) + c, v);
    }
    if (direct) return true;
    __syncthreads();
    unsigned* counter = p.counters + (size_t)stream * p.tiles + tile0;
    if (tid == 0) *s_ticket = atomic_add_acq_rel_gpu(counter, 1u);
    __syncthreads();
    if (*s_ticket != (unsigned)(nsplit - 1)) return true;
    if (tid == 0) store_relaxed_gpu(counter, 0u);
    tree_merge<D, C::kRows, C::kThreads>(p, stream, r0e, min(rows_here, rows_live), nsplit, reinterpret_cast<float*>(smem), tid, store_out);
    for (int i = tid; i < (rows_here - min(rows_here, rows_live)) * (D / 4); i += C::kThreads)
        store_out(r0e + rows_live + i / (D / 4), i % (D / 4), make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
    return true;
}

template <class C>
__global__ void __launch_bounds__(C::kThreads, 1) decode_tree_tc_kernel(const TreeParams p,
                                                                           const __grid_constant__ CUtensorMap tmK,
                                                                           const __grid_constant__ CUtensorMap tmV) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    // (an offset, not a rounded address: the compiler keeps seeing shared memory)
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
    TreeTcPlan* plan = reinterpret_cast<TreeTcPlan*>(smem + C::kOffMisc + 64);
    TreeTcRange* range = reinterpret_cast<TreeTcRange*>(plan + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == 20) tmem_alloc(tslot, 512);
    if (tid == 0) tslot[1] = 0u;  // no wait has given up
    grid_dependency_wait();
    if (warp == 0) {
        if (p.S > 1) {
            tree_tc_plan<C>(p, lane, plan, range);
        } else if (lane == 0) {  // a whole tile a CTA
            const int stream = (int)(blockIdx.x / p.tiles), b = stream / p.Hkv;
            const TreeTcSeq q = tree_tc_seq<C>(p, b);
            *range = {b, stream - b * p.Hkv, (int)blockIdx.x - stream * p.tiles, q.len, q.n, 0, q.len, 0, 1};
            *plan = {0, 0, 0, 1, 0, 0};
        }
    }
    tc05_fence_before();
    __syncthreads();
    tc05_fence_after();
    for (int slot = 0; plan->more; slot ^= 1) {
        if (!tree_tc_range<C>(p, tmK, tmV, smem, slot, plan->at >= plan->end)) break;
        // what this range left in shared memory by plain stores comes before the next one's copies
        fence_proxy_async_smem();
        __syncthreads();
    }
    __syncthreads();
    if (warp == 20) tmem_dealloc(*tslot, 512);
}

}  // namespace va
