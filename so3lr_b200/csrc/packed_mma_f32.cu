// The warp-level kernels of packed_mma.cuh for float operands.
#include "packed_mma.cuh"

namespace so3lr {
template int packed_forward_mma<float>(cudaStream_t, const PackedArgs&, int);
template int packed_forward_split<float>(cudaStream_t, const PackedArgs&, int, int, bool);
template int packed_dq_mma<float>(cudaStream_t, const PackedArgs&, int);
template int packed_dkv_mma<float>(cudaStream_t, const PackedArgs&, int);
template int packed_delta<float>(cudaStream_t, const PackedArgs&, const int4*, int, const int4*, int);
template int packed_join<float>(cudaStream_t, const PackedArgs&);
template int packed_sum<float>(cudaStream_t, const PackedArgs&, int, int);
}  // namespace so3lr
