#define BEAM_T __bf16
#include "gated_inst.h"
