// okf_delta_f16.hip -- the gated delta rule over f16 inputs.
#define OKF_DELTA_TYPE _Float16
#include "okf_delta_run.h"
