// Kernel instantiations of the 8-bit decode for one code type and one group of head dims, and their launch: included by
// decode_q8_<codes>_<dims>.cu so that they compile side by side.
#pragma once

#include <atomic>

#include "decode_q8.cuh"

namespace ftk {

template <typename KV, int D, int NBK, bool SPLIT>
cudaError_t q8_launch_one(const CUtensorMap& mk, const CUtensorMap& mv, const Q8Params& p, cudaStream_t cs) {
    // warps per 64-row tile: with two a warp has 32 rows to overlap work over (one: 53 us instead of 49 for 32 x 4096 rows
    // of 128, too many registers; four: 50, and 94 instead of 90 for ragged ones); wide heads have work enough in 16 rows (256:
    // 51 us instead of 57)
    constexpr int WPT = D >= 192 ? 4 : 2;
    // a function attribute, not a stream operation: legal while the stream is captured. Set once per device.
    static std::atomic<unsigned long long> done{0};
    if (!(done.load(std::memory_order_relaxed) >> p.device & 1ull)) {
        const cudaError_t e = cudaFuncSetAttribute(decode_q8_kernel<KV, D, NBK, SPLIT, WPT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (Q8Cfg<D, NBK, SPLIT, WPT>::SMEM_BYTES));
        if (e != cudaSuccess) return e;
        done.fetch_or(1ull << p.device, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.ncta);
    cfg.blockDim = dim3(Q8_THREADS);
    cfg.dynamicSmemBytes = (Q8Cfg<D, NBK, SPLIT, WPT>::SMEM_BYTES);
    cfg.stream = cs;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, decode_q8_kernel<KV, D, NBK, SPLIT, WPT>, mk, mv, p);
}

template <typename KV, int D>
cudaError_t q8_launch_dim(const CUtensorMap& mk, const CUtensorMap& mv, const Q8Params& p, int nbk, bool split, cudaStream_t cs) {
    if constexpr (D <= 128) {
        if (nbk == 2) return split ? q8_launch_one<KV, D, 2, true>(mk, mv, p, cs) : q8_launch_one<KV, D, 2, false>(mk, mv, p, cs);
    }
    return split ? q8_launch_one<KV, D, 1, true>(mk, mv, p, cs) : q8_launch_one<KV, D, 1, false>(mk, mv, p, cs);
}

}  // namespace ftk
