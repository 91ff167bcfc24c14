// Arguments of the masked L1 attention kernels, passed by value.
#pragma once
#include <stdint.h>
#include "../../include/l1attn_hip.h"

#define L1_MASKED_HEADS 256  // slopes travel with the kernel arguments

struct L1MaskedArgs {
	int B, T, S, H, Hk, W, Wv;
	int causal, has_slopes;
	int vec;              // which rows may be read in whole vectors: 1 q, 2 k, 4 v, 8 d_o
	float cap, icap, rw;  // rw = 1/sqrt(W)
	const int32_t* doc;
	const int32_t* prefix;
	float slopes[L1_MASKED_HEADS];
};
