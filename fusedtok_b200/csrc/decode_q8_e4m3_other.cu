// 8-bit decode kernels: e4m3 codes, head dims 80, 96 and 192.
#include "decode_q8_launch.cuh"

namespace ftk {
cudaError_t q8_launch_e4m3_other(const CUtensorMap& mk, const CUtensorMap& mv, const Q8Params& p, int nbk, bool split, cudaStream_t cs) {
    if (p.D == 80) return q8_launch_dim<__nv_fp8_e4m3, 80>(mk, mv, p, nbk, split, cs);
    if (p.D == 96) return q8_launch_dim<__nv_fp8_e4m3, 96>(mk, mv, p, nbk, split, cs);
    return q8_launch_dim<__nv_fp8_e4m3, 192>(mk, mv, p, nbk, split, cs);
}
}  // namespace ftk
