// Trellis GEMV with an epilogue, codebook family FAM_MCG (kernel body in exl3_gemv_body.h).
#define EXL3_GEMV_EPILOGUE_FAM FAM_MCG
#include "exl3_gemv_body.h"
