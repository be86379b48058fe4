// Trellis GEMV with an epilogue, codebook family FAM_PAIR (kernel body in exl3_gemv_body.h).
#define EXL3_GEMV_EPILOGUE_FAM FAM_PAIR
#include "exl3_gemv_body.h"
