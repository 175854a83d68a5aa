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

template <class C>
int launch_tree_cfg(void (*kernel)(const TreeParams), const TreeParams& p, cudaStream_t st) {
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
    cfg.gridDim = dim3((unsigned)((long long)p.B * p.Hkv * p.tiles * p.S));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VA_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return VA_OK;
}

template <int D>
int launch_tree_dim(int fmt, const TreeParams& p, int rows, cudaStream_t st) {
#define VA_TREE_CFG(kernel, ...) return launch_tree_cfg<__VA_ARGS__>(kernel<__VA_ARGS__>, p, st)
#define VA_TREE_KIND(kind)                                                                       \
    do {                                                                                         \
        if (rows == 16) VA_TREE_CFG(decode_tree_kernel, TreeCfg<kind, D, 1>);                    \
        if (rows == 32) VA_TREE_CFG(decode_tree_kernel, TreeCfg<kind, D, 2>);                    \
        if (rows == 128) VA_TREE_CFG(decode_tree_tc_kernel, TreeTcCfg<kind, D, false>);          \
        VA_TREE_CFG(decode_tree_tc_kernel, TreeTcCfg<kind, D, true>);                            \
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
#undef VA_TREE_CFG
}

}  // namespace host
}  // namespace va
