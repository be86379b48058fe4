// The dense GEMM's launches with an epilogue (kernels in exl3_gemm_body.h).
#include "exl3_gemm_body.h"

namespace exl3 {

hipError_t run_gemm_epilogue(int fam, const GemmArgs &a, const EpilogueArgs &e, hipStream_t s) {
    if (a.groups != 1) return hipErrorInvalidValue;
    return launch_gemm<true>(fam, a, &e, s);
}

}  // namespace exl3
