// Launcher of decode_tree_kernel, instantiated per head dimension in
// launch_tree_d*.cu.
#pragma once

#include <algorithm>
#include <mutex>

#include "decode_tree.cuh"
#include "decode_tree_tc.cuh"
#include "launch.cuh"

namespace va {
namespace host {

template <class C, class... Maps>
int launch_tree_cfg(void (*kernel)(const TreeParams, const Maps...), const TreeParams& p, dim3 grid, cudaStream_t st,
                    const Maps&... maps) {
    int dev;
    int rc = current_device(&dev);
    if (rc) return rc;
    static bool attr_set[kMaxDevices] = {false};
    static std::mutex mu;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!attr_set[dev]) {
            VA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
            attr_set[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VA_CUDA(cudaLaunchKernelEx(&cfg, kernel, p, maps...));
    return VA_OK;
}

// x: the splits and tiles of one (sequence, KV head), which read the same rows, next to
// one another; y, z: the (sequence, KV head) pairs
inline dim3 tree_grid(const TreeParams& p) {
    const unsigned streams = (unsigned)(p.B * p.Hkv), y = std::min(streams, 65535u);
    return dim3((unsigned)(p.tiles * p.S), y, (streams + y - 1) / y);
}

template <class C>
int launch_tree_tc(const TreeParams& p, cudaStream_t st) {
    CUtensorMap tmK = {}, tmV = {};
    if constexpr (C::kDirect) {  // boxes of a block's rows inside a page
        const long long rows = (long long)p.num_pages * p.Hkv * p.page_rows;
        if (rows >= (1ll << 31)) return VA_ERR_TOO_LARGE;
        const int box = tree_tc_run(p.page_rows);
        int rc = encode_f16_rows_map(&tmK, p.K, rows, box, C::kD);
        if (!rc) rc = encode_f16_rows_map(&tmV, p.V, rows, box, C::kD);
        if (rc) return rc;
    }
    int dev;
    const int rc = current_device(&dev);
    if (rc) return rc;
    // splits: one CTA per SM, each with a window of the work; without: a CTA per tile
    const long long items = (long long)p.B * p.Hkv * p.tiles;
    if (items > 0x7FFFFFFFll) return VA_ERR_TOO_LARGE;
    TreeParams q = p;
    if (items * ((long long)p.max_pages * p.page_rows / C::kNb + 1 + kTcFixed) > 0x7FFFFFFFll) q.S = 1;  // (32-bit windows)
    const long long ctas = q.S > 1 ? std::min((long long)sm_count(dev), items * q.S) : items;
    return launch_tree_cfg<C>(decode_tree_tc_kernel<C>, q, dim3((unsigned)ctas), st, tmK, tmV);
}

template <int D>
int launch_tree_dim(int fmt, const TreeParams& p, int rows, cudaStream_t st) {
#define VA_TREE_KIND(kind)                                                                               \
    do {                                                                                                 \
        if (rows == 16) return launch_tree_cfg<TreeCfg<kind, D>>(decode_tree_kernel<TreeCfg<kind, D>>, p, tree_grid(p), st); \
        if (rows == 128) return launch_tree_tc<TreeTcCfg<kind, D, false>>(p, st);                        \
        return launch_tree_tc<TreeTcCfg<kind, D, true>>(p, st);                                          \
    } while (0)
    switch (fmt) {
        case VA_F16P: VA_TREE_KIND(Kind::F16);
        case VA_BF16P: VA_TREE_KIND(Kind::BF16);
        case VA_F8P: VA_TREE_KIND(Kind::F8);
        case VA_Q8P: VA_TREE_KIND(Kind::Q8);
        case VA_Q4P: VA_TREE_KIND(Kind::Q4);
        case VA_Q3P: VA_TREE_KIND(Kind::Q3);
        default: return VA_ERR_UNSUPPORTED;
    }
#undef VA_TREE_KIND
}

}  // namespace host
}  // namespace va
