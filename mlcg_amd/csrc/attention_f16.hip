// The attention kernels (attention.h) for fp16 elements.
#define MLCG_ATTENTION_TYPE _Float16
#include "attention.h"
