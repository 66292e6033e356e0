#define MIA_ATTENTION_TYPE __bf16
#include "attention_kernels.h"
