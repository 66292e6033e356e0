#define MIA_LINEAR_TYPE __bf16
#include "linear_kernels.h"
