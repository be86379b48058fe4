// The dense GEMM's plain launches (kernels in exl3_gemm_body.h).
#include "exl3_gemm_body.h"

namespace exl3 {

hipError_t run_gemm(int fam, const GemmArgs &a, hipStream_t s) { return launch_gemm<false>(fam, a, nullptr, s); }

}  // namespace exl3
