// Kernels and launchers of the cache's rows and pages (cache_rows.cuh, pages.cuh).
#include <algorithm>
#include <climits>

#include "cache_rows.cuh"
#include "launch.cuh"
#include "pages.cuh"

namespace va {

__global__ void __launch_bounds__(kAcceptThreads) accept_tree_kernel(const AcceptParams p) {
    __shared__ long long src[kAcceptMax], dst[kAcceptMax];
    __shared__ int s_n;
    grid_dependency_wait();
    const int hk = blockIdx.x, b = blockIdx.y;
    const long long cap = (long long)p.max_pages * p.page_rows;
    const int len = (int)max(0ll, min((long long)load_global(p.lens + b), cap));
    const int nodes = max(0, min(load_global(p.nodes + b), len));
    const int ctx = len - nodes;
    if (threadIdx.x < 32) {
        const int want = max(0, min(load_global(p.accepted + b), p.P));
        int n = want;
        for (int c = 0; c < want; c += 32) {
            const int i = c + (int)threadIdx.x;
            bool bad = false;
            if (i < want) {
                const int x = load_global(p.path + (size_t)b * p.P + i);
                bad = x < 0 || x >= nodes || (i > 0 && x <= load_global(p.path + (size_t)b * p.P + i - 1));
            }
            const unsigned m = __ballot_sync(0xffffffffu, bad);
            if (m) {
                n = c + __ffs(m) - 1;
                break;
            }
        }
        if (threadIdx.x == 0) {
            s_n = n;
            if (hk == 0 && blockIdx.z == 0) p.new_lens[b] = ctx + n;
        }
    }
    __syncthreads();
    const int n = s_n;
    const int* trow = p.table + (size_t)b * p.max_pages;
    const auto place = [&](int row) -> long long {
        const int pi = row / p.page_rows;
        const int pg = pi < p.max_pages ? valid_page(load_global(trow + pi), p.num_pages) : -1;
        return pg < 0 ? -1
                      : blockIdx.z * p.layer_rows + ((long long)pg * p.Hkv + hk) * p.page_rows + (row - pi * p.page_rows);
    };
    for (int i = threadIdx.x; i < n; i += kAcceptThreads) {
        const int x = load_global(p.path + (size_t)b * p.P + i);
        const long long s = place(ctx + x), d = place(ctx + i);
        // a row in place, or one whose page does not exist, is left
        src[i] = (x == i || d < 0) ? -1 : s;
        dst[i] = d;
    }
    __syncthreads();
    grid_launch_dependents();
    accept_move<uint2>(p.K, p.rb, src, dst, n);
    accept_move<uint2>(p.V, p.rb, src, dst, n);
    if (p.sb == 4) {
        accept_move<uint32_t>(p.scK, p.sb, src, dst, n);
        accept_move<uint32_t>(p.scV, p.sb, src, dst, n);
    } else if (p.sb == 2) {
        accept_move<uint16_t>(p.scK, p.sb, src, dst, n);
        accept_move<uint16_t>(p.scV, p.sb, src, dst, n);
    }
}

// The plan of a fork: tables, lengths, counts, and which rows are to be copied
// (copied by fork_copy_kernel). One CTA: the work is a pass over refs and two over the
// tables, each bound by the latency of its loads, so parents and lengths are kept in
// shared memory and a warp has the first 32 entries of kAhead sequences in flight. 96 new
// sequences of 200 to 1500 rows: about 14 us.
constexpr int kAhead = 2;
constexpr int kFreeHere = 1024;  // free pages kept in shared memory (further ones in free_list)
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const ForkParams p) {
    extern __shared__ int sm[];
    int* kids = sm;              // [Bin]
    int* first = kids + p.Bin;   // [Bin]
    int* lens = first + p.Bin;   // [Bin]
    int* full = lens + p.Bin;    // [Bin] full pages
    int* need = full + p.Bin;    // [Bin] pages of lens + reserve rows
    int* base = need + p.Bin;    // [Bout]
    int* from_seq = base + p.Bout;  // [Bout] parent, or -1
    __shared__ int scan[33], free_here[kFreeHere];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = kPlanThreads / 32;
    const int num_pages = p.pool.num_pages, pr = p.pool.page_rows;
    grid_dependency_wait();
    const long long cap = (long long)p.max_pages * pr;
    for (int s = tid; s < p.Bin; s += kPlanThreads) {
        kids[s] = 0;
        first[s] = INT_MAX;
        const int len = (int)max(0ll, min((long long)load_global(p.lens + s), cap));
        lens[s] = len;
        full[s] = len / pr;
        // (the rest of a page, a page and a reserve below 2^31: 32 bits)
        need[s] = (int)min((unsigned)p.max_pages, (unsigned)full[s] + ((unsigned)(len - full[s] * pr) + p.reserve + pr - 1) / pr);
    }
    for (int i = tid; i < p.Bout; i += kPlanThreads) {
        const int s = load_global(p.parent + i);
        from_seq[i] = s >= 0 && s < p.Bin ? s : -1;
    }
    for (int i = tid; i < num_pages; i += kPlanThreads) p.new_refs[i] = load_global(p.refs + i);
    __syncthreads();
    for (int i = tid; i < p.Bout; i += kPlanThreads)
        if (from_seq[i] >= 0) {
            atomicAdd(kids + from_seq[i], 1);
            atomicMin(first + from_seq[i], i);
        }
    __syncthreads();
    // a new sequence: its parent, its length, how many pages it shares and needs
    struct Child {
        int s, len, full, need;
        bool keep;
    };
    const auto child = [&](int i) {
        Child c;
        c.s = i < p.Bout ? from_seq[i] : -1;
        c.len = c.s >= 0 ? lens[c.s] : 0;
        c.full = c.s >= 0 ? full[c.s] : 0;
        c.need = c.s >= 0 ? need[c.s] : 0;
        c.keep = c.s >= 0 && first[c.s] == i;
        return c;
    };
    const auto held = [&](const Child& c, int j) {
        if (c.s < 0 || j >= p.max_pages || !(c.keep || j < c.full)) return -1;
        return valid_page(load_global(p.table + (size_t)c.s * p.max_pages + j), num_pages);
    };
    for (int i0 = warp; i0 < p.Bout; i0 += kWarps * kAhead) {
        Child c[kAhead];
        int e[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            c[u] = child(i0 + u * kWarps);
            e[u] = held(c[u], lane);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            int n = 0;
            for (int j = lane; j - lane < c[u].need; j += 32)
                n += __popc(__ballot_sync(0xffffffffu, j < c[u].need && (j < 32 ? e[u] : held(c[u], j)) < 0));
            if (lane == 0 && i0 + u * kWarps < p.Bout) base[i0 + u * kWarps] = n;
        }
    }
    // counts of the pages that the old tables hold
    for (int s0 = warp; s0 < p.Bin; s0 += kWarps * kAhead) {
        int e[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = s0 + u * kWarps;
            e[u] = s < p.Bin && lane < p.max_pages ? load_global(p.table + (size_t)s * p.max_pages + lane) : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int s = s0 + u * kWarps;
            if (s >= p.Bin) break;
            const int shared = kids[s] - 1, own = kids[s] > 0 ? 0 : -1;
            for (int j = lane; j < p.max_pages; j += 32) {
                const int pg = valid_page(j < 32 ? e[u] : load_global(p.table + (size_t)s * p.max_pages + j), num_pages);
                const int d = j < full[s] ? shared : own;
                if (pg >= 0 && d != 0) atomicAdd(p.new_refs + pg, d);
            }
        }
    }
    __syncthreads();
    int total = 0;
    for (int c0 = 0; c0 < p.Bout; c0 += kPlanThreads) {
        const int i = c0 + tid;
        int sum;
        const int before = block_scan(i < p.Bout ? base[i] : 0, scan, sum);
        if (i < p.Bout) base[i] = total + before;
        total += sum;
    }
    __syncthreads();
    // the `total` lowest free pages
    int found = 0;
    for (int c0 = 0; c0 < num_pages && found < total; c0 += 4 * kPlanThreads) {
        unsigned f = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int pg = c0 + 4 * tid + k;
            if (pg < num_pages && load_global(p.refs + pg) == 0) f |= 1u << k;
        }
        int sum;
        int at = found + block_scan(__popc(f), scan, sum);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (f >> k & 1u) {
                if (at < kFreeHere) free_here[at] = c0 + 4 * tid + k;
                else if (at < total) p.free_list[at] = c0 + 4 * tid + k;
                ++at;
            }
        found += sum;
    }
    found = min(found, total);
    __syncthreads();
    if (tid == 0) *p.shortage = total - found;
    for (int i0 = warp; i0 < p.Bout; i0 += kWarps * kAhead) {
        Child cs[kAhead];
        int es[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            cs[u] = child(i0 + u * kWarps);
            es[u] = held(cs[u], lane);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * kWarps;
            if (i >= p.Bout) break;
            const Child& c = cs[u];
            const int part = c.full, rest = c.len - part * pr;
            int at = base[i];
            bool lost = false;
            int from = -1, to = -1;
            for (int j = lane; j - lane < p.max_pages; j += 32) {
                const int h = j < 32 ? es[u] : held(c, j);
                const bool ask = j < c.need && h < 0;
                const unsigned m = __ballot_sync(0xffffffffu, ask);
                const int rank = at + __popc(m & ((1u << lane) - 1u));
                at += __popc(m);
                int e = h;
                if (ask && rank < found) {
                    e = rank < kFreeHere ? free_here[rank] : p.free_list[rank];
                    atomicAdd(p.new_refs + e, 1);
                    if (j == part && rest > 0 && !c.keep) {
                        from = valid_page(load_global(p.table + (size_t)c.s * p.max_pages + j), num_pages);
                        to = e;
                    }
                } else if (ask && j == part && rest > 0) {
                    lost = true;
                }
                if (j < p.max_pages) p.new_table[(size_t)i * p.max_pages + j] = e;
            }
            lost = __any_sync(0xffffffffu, lost);
            const unsigned who = __ballot_sync(0xffffffffu, to >= 0);
            if (who) {
                from = __shfl_sync(0xffffffffu, from, __ffs(who) - 1);
                to = __shfl_sync(0xffffffffu, to, __ffs(who) - 1);
            }
            if (lane == 0) {
                p.new_lens[i] = lost ? part * pr : c.len;
                p.copy[i] = from;
                p.copy[p.Bout + i] = to;
                p.copy[2 * p.Bout + i] = from >= 0 && to >= 0 ? (rest + 7) & ~7 : 0;
            }
        }
    }
}

// CTA (new sequence, layer, KV head): the used rows of its parent's last page
// into its own, in blocks of eight (16-byte words in every format), K and V with four
// loads in flight a thread. 96 sequences x 4 layers x 8 heads of f16+ pages: about 13 us, the copied
// bytes at the copy rate 10.
constexpr int kCopyThreads = 256;
__global__ void __launch_bounds__(kCopyThreads) fork_copy_kernel(const ForkParams p) {
    grid_dependency_wait();
    const int i = blockIdx.x;
    const int rows = p.copy[2 * p.Bout + i];
    if (rows == 0) return;
    const long long from = p.copy[i], to = p.copy[p.Bout + i];
    const long long layer = (long long)blockIdx.y * p.pool.num_pages;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!p.pool.base[k]) continue;
        const size_t head = (size_t)p.pool.page_rows * p.pool.row_bytes[k];
        const uint4* src = reinterpret_cast<const uint4*>(p.pool.base[k] + ((layer + from) * p.pool.Hkv + blockIdx.z) * head);
        uint4* dst = reinterpret_cast<uint4*>(p.pool.base[k] + ((layer + to) * p.pool.Hkv + blockIdx.z) * head);
        const int n = rows / 8 * (p.pool.row_bytes[k] / 2);  // (rows: a multiple of 8; their bytes may pass 2^31)
        for (int x = threadIdx.x; x < n; x += 4 * kCopyThreads) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x + j * kCopyThreads < n) v[j] = load_global(src + x + j * kCopyThreads);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x + j * kCopyThreads < n) dst[x + j * kCopyThreads] = v[j];
        }
    }
}

// The plan of a compaction: n pages in use; the m-th used page at or past n
// goes to the m-th free page below n.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactParams p) {
    __shared__ int scan[33];
    const int tid = threadIdx.x, num_pages = p.pool.num_pages;
    grid_dependency_wait();
    int mine = 0;
    for (int i = tid; i < num_pages; i += kPlanThreads) mine += load_global(p.refs + i) > 0;
    int n;
    block_scan(mine, scan, n);
    int holes = 0, movers = 0;
    for (int c0 = 0; c0 < num_pages; c0 += 4 * kPlanThreads) {
        unsigned hole = 0, move = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int pg = c0 + 4 * tid + k;
            if (pg < num_pages) {
                const int r = load_global(p.refs + pg);
                if (pg < n) {
                    if (r > 0) p.new_refs[pg] = r;
                    else hole |= 1u << k;
                } else {
                    p.new_refs[pg] = 0;
                    if (r > 0) move |= 1u << k;
                }
            }
        }
        int sum;  // both counts of a chunk fit 16 bits
        const int at = block_scan(__popc(hole) | __popc(move) << 16, scan, sum);
        int h = holes + (at & 0xFFFF), m = movers + (at >> 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (hole >> k & 1u) p.to[h++] = c0 + 4 * tid + k;
            if (move >> k & 1u) p.from[m++] = c0 + 4 * tid + k;
        }
        holes += sum & 0xFFFF;
        movers += sum >> 16;
    }
    __syncthreads();
    for (int i = tid; i < movers; i += kPlanThreads) {
        const int f = p.from[i], t = p.to[i];
        p.new_refs[t] = load_global(p.refs + f);
        p.map[f] = t;
    }
    if (tid == 0) {
        *p.used = n;
        *p.count = movers;
    }
}

// The moved pages' bytes (chunks of kMoveChunk 16-byte words, over all CTAs) and
// the tables' entries. Bound by HBM: 1400 pages of 64 rows, q4+, 8 heads, 4 layers move in 143 us with
// the plan, 5.4 TB/s.
constexpr int kMoveThreads = 256, kMoveWords = 4 * kMoveThreads;
__global__ void __launch_bounds__(kMoveThreads) compact_move_kernel(const CompactParams p) {
    grid_dependency_wait();
    const int n = *p.used, moved = *p.count;
    const PoolView& v = p.pool;
    for (int k = 0; k < 4; ++k) {
        if (!v.base[k]) continue;
        const long long words = (long long)v.Hkv * v.page_rows * v.row_bytes[k] / 16;  // of a page
        const long long per = (words + kMoveWords - 1) / kMoveWords;
        const long long total = (long long)moved * v.layers * per;
        for (long long u = blockIdx.x; u < total; u += gridDim.x) {
            const long long i = u / per, c = u - i * per;
            const int layer = (int)(i / moved), m = (int)(i - (long long)layer * moved);
            const uint4* src = reinterpret_cast<const uint4*>(v.base[k]) + ((long long)layer * v.num_pages + p.from[m]) * words;
            uint4* dst = reinterpret_cast<uint4*>(v.base[k]) + ((long long)layer * v.num_pages + p.to[m]) * words;
            const long long w0 = c * kMoveWords + threadIdx.x;
            uint4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (w0 + j * kMoveThreads < words) x[j] = load_global(src + w0 + j * kMoveThreads);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (w0 + j * kMoveThreads < words) dst[w0 + j * kMoveThreads] = x[j];
        }
    }
    for (long long i = (long long)blockIdx.x * kMoveThreads + threadIdx.x; i < p.entries;
         i += (long long)gridDim.x * kMoveThreads) {
        const int e = load_global(p.table + i);
        p.new_table[i] = e >= n && e < v.num_pages && load_global(p.refs + e) > 0 ? p.map[e] : e;
    }
}

namespace host {

namespace {
// A launch that may start its prologue while the one before it in the stream ends.
template <class P>
int launch_pdl(void (*kernel)(const P), dim3 grid, int threads, size_t smem, cudaStream_t st, const P& p) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VA_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return VA_OK;
}

template <class T>
int launch_append_in(int bits, const AppendParams& p, cudaStream_t st) {
    // a warp to every item (half of a 16-group token's K or V) up to three 8-warp CTAs an SM
    // for each side, twice what fits at a time; beyond that the warps loop
    int dev;
    const int rc = current_device(&dev);
    if (rc) return rc;
    const long long items = (long long)p.T * ((p.Hkv * (p.D / kGroup) + 7) / 8);
    const dim3 grid((unsigned)std::min<long long>((items + 7) / 8, (long long)sm_count(dev) * 3), 2);
    switch (bits) {
        case 16: return launch_pdl(append_packed_kernel<16, T>, grid, 256, 0, st, p);
        case kBitsBf16: return launch_pdl(append_packed_kernel<kBitsBf16, T>, grid, 256, 0, st, p);
        case kBitsF8: return launch_pdl(append_packed_kernel<kBitsF8, T>, grid, 256, 0, st, p);
        case 8: return launch_pdl(append_packed_kernel<8, T>, grid, 256, 0, st, p);
        case 4: return launch_pdl(append_packed_kernel<4, T>, grid, 256, 0, st, p);
        default: return launch_pdl(append_packed_kernel<3, T>, grid, 256, 0, st, p);
    }
}
}  // namespace

int launch_append_packed(int fmt, int in_type, const AppendParams& p, cudaStream_t st) {
    const int bits = fmt == VA_BF16P ? kBitsBf16 : fmt == VA_F8P ? kBitsF8 : va_fmt_bits(fmt);
    if (in_type == VA_FP32) return launch_append_in<float>(bits, p, st);
    if (in_type == VA_FP16) return launch_append_in<__half>(bits, p, st);
    return launch_append_in<__nv_bfloat16>(bits, p, st);
}

int launch_accept_tree(const AcceptParams& p, int B, int layers, cudaStream_t st) {
    return launch_pdl(accept_tree_kernel, dim3((unsigned)p.Hkv, (unsigned)B, (unsigned)layers), kAcceptThreads, 0, st, p);
}

int launch_fork_pages(const ForkParams& p, cudaStream_t st) {
    int dev;
    int rc = current_device(&dev);
    if (rc) return rc;
    const size_t smem = sizeof(int) * (5 * (size_t)p.Bin + 2 * p.Bout);
    if (smem > 40 * 1024)  // (4 KB more are static; at most 7 * 4000 entries)
        VA_CUDA(cudaFuncSetAttribute(fork_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024));
    rc = launch_pdl(fork_plan_kernel, dim3(1), kPlanThreads, smem, st, p);
    if (rc) return rc;
    return launch_pdl(fork_copy_kernel, dim3((unsigned)p.Bout, (unsigned)p.pool.layers, (unsigned)p.pool.Hkv),
                      kCopyThreads, 0, st, p);
}

int launch_compact_pages(const CompactParams& p, cudaStream_t st) {
    int dev;
    int rc = current_device(&dev);
    if (rc) return rc;
    rc = launch_pdl(compact_plan_kernel, dim3(1), kPlanThreads, 0, st, p);
    if (rc) return rc;
    return launch_pdl(compact_move_kernel, dim3((unsigned)(sm_count(dev) * 8)), kMoveThreads, 0, st, p);
}

}  // namespace host
}  // namespace va
