// 8-bit decode kernels: int8 codes, head dims 64, 128 and 256.
#include "decode_q8_launch.cuh"

namespace ftk {
cudaError_t q8_launch_int8_pow2(const CUtensorMap& mk, const CUtensorMap& mv, const Q8Params& p, int nbk, bool split, cudaStream_t cs) {
    if (p.D == 64) return q8_launch_dim<int8_t, 64>(mk, mv, p, nbk, split, cs);
    if (p.D == 128) return q8_launch_dim<int8_t, 128>(mk, mv, p, nbk, split, cs);
    return q8_launch_dim<int8_t, 256>(mk, mv, p, nbk, split, cs);
}
}  // namespace ftk
