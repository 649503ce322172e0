// The gated delta rule (delta.h) for bf16 elements.
#define MLCG_DELTA_TYPE __bf16
#include "delta.h"
