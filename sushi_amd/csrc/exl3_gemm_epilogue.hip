// The dense GEMM's launches with an epilogue (kernels in exl3_gemm_body.h).
#include "exl3_gemm_body.h"

namespace exl3 {

hipError_t run_gemm_epilogue(int fam, const GemmArgs &a, const EpilogueArgs &e, const GemmSplit &split, hipStream_t s) {
    if (a.groups != 1 || (split.part && (split.splits < 1 || split.splits > a.in / 128))) return hipErrorInvalidValue;
    const GemmEpilogue ge{e, split};
    return launch_gemm<true>(fam, a, &ge, s);
}

}  // namespace exl3
