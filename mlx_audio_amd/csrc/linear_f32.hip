#define MIA_LINEAR_TYPE float
#include "linear_kernels.h"
