// The 4-bit products' kernels for f32 rows (q4_matvec.cuh).
#include "q4_matvec.cuh"

namespace vfmoe {

int launch_q4_f32(const Q4Args &a, cudaStream_t st) { return q4::launch_type<VFMOE_DT_F32>(a, st); }

}  // namespace vfmoe
