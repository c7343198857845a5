// The 4-bit products' kernels for bf16 rows (q4_matvec.cuh).
#include "q4_matvec.cuh"

namespace vfmoe {

int launch_q4_bf16(const Q4Args &a, cudaStream_t st) { return q4::launch_type<VFMOE_DT_BF16>(a, st); }

}  // namespace vfmoe
