// okf_delta_bf16.hip -- the gated delta rule over bf16 inputs.
#define OKF_DELTA_TYPE __bf16
#include "okf_delta_run.h"
