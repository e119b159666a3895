#define BEAM_T _Float16
#include "gemm_mx_inst.h"
