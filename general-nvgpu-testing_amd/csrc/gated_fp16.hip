#define BEAM_T _Float16
#include "gated_inst.h"
