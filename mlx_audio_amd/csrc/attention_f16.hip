#define MIA_ATTENTION_TYPE _Float16
#include "attention_kernels.h"
