// The attention kernels (attention.h) for bf16 elements.
#define MLCG_ATTENTION_TYPE __bf16
#include "attention.h"
