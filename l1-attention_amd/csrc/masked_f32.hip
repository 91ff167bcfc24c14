// Masked L1 attention for float rows.
#include "masked_kernels.h"

L1_MASKED_TABLE(l1_masked_f32, float)
