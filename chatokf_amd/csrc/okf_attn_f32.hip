// okf_attn_f32.hip -- prompt attention over f32 inputs.
#define OKF_ATTN_TYPE float
#include "okf_attn_run.h"
