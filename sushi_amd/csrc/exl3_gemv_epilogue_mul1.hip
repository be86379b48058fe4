// Trellis GEMV with an epilogue, codebook family FAM_MUL1 (kernel body in exl3_gemv_body.h).
#define EXL3_GEMV_EPILOGUE_FAM FAM_MUL1
#include "exl3_gemv_body.h"
