// The warp-level kernels of packed_mma.cuh for float operands.
#include "packed_mma.cuh"

namespace so3lr {
template void packed_forward_mma<float>(cudaStream_t, const PackedArgs&, int);
template void packed_forward_split<float>(cudaStream_t, const PackedArgs&, int, int, bool);
template void packed_dq_mma<float>(cudaStream_t, const PackedArgs&, int);
template void packed_dkv_mma<float>(cudaStream_t, const PackedArgs&, int);
template void packed_delta<float>(cudaStream_t, const PackedArgs&, int);
}  // namespace so3lr
