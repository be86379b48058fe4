// Trellis GEMV with an epilogue, codebook family FAM_3INST (kernel body in exl3_gemv_body.h).
#define EXL3_GEMV_EPILOGUE_FAM FAM_3INST
#include "exl3_gemv_body.h"
