// okf_attn_bf16.hip -- prompt attention over bf16 inputs.
#define OKF_ATTN_TYPE __bf16
#include "okf_attn_run.h"
