#define MIA_LINEAR_TYPE _Float16
#include "linear_kernels.h"
