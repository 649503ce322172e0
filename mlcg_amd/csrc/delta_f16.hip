// The gated delta rule (delta.h) for fp16 elements.
#define MLCG_DELTA_TYPE _Float16
#include "delta.h"
