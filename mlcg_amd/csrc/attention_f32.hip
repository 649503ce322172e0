// The attention kernels (attention.h) for fp32 elements.
#define MLCG_ATTENTION_TYPE float
#include "attention.h"
