#define BEAM_T __bf16
#include "gemm_mx_inst.h"
