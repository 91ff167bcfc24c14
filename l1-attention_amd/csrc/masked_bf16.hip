// Masked L1 attention for __bf16 rows.
#include "masked_kernels.h"

L1_MASKED_TABLE(l1_masked_bf16, __bf16)
