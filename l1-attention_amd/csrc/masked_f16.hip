// Masked L1 attention for _Float16 rows.
#include "masked_kernels.h"

L1_MASKED_TABLE(l1_masked_f16, _Float16)
