#define MIA_ATTENTION_TYPE float
#include "attention_kernels.h"
