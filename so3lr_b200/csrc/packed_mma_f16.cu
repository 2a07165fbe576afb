// The warp-level kernels of packed_mma.cuh for __half operands.
#include "packed_mma.cuh"

namespace so3lr {
template int packed_forward_mma<__half>(cudaStream_t, const PackedArgs&, int);
template int packed_forward_split<__half>(cudaStream_t, const PackedArgs&, int, int, bool);
template int packed_dq_mma<__half>(cudaStream_t, const PackedArgs&, int);
template int packed_dkv_mma<__half>(cudaStream_t, const PackedArgs&, int);
template int packed_delta<__half>(cudaStream_t, const PackedArgs&, const int4*, int, const int4*, int);
template int packed_join<__half>(cudaStream_t, const PackedArgs&);
template int packed_sum<__half>(cudaStream_t, const PackedArgs&, int, int);
}  // namespace so3lr
