// okf_attn_f16.hip -- prompt attention over f16 inputs.
#define OKF_ATTN_TYPE _Float16
#include "okf_attn_run.h"
