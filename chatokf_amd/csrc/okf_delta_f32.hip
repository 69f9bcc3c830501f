// okf_delta_f32.hip -- the gated delta rule over f32 inputs.
#define OKF_DELTA_TYPE float
#include "okf_delta_run.h"
