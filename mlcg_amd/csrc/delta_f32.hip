// The gated delta rule (delta.h) for fp32 elements.
#define MLCG_DELTA_TYPE float
#include "delta.h"
