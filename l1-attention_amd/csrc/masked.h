// Masked L1 attention: the kernels' arguments, passed by value, and what masked.hip calls of the files of each type.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/l1attn_hip.h"

#define L1_MASKED_HEADS 256  // slopes travel with the kernel arguments

struct L1MaskedArgs {
	int B, T, S, H, Hk, W, Wv;
	int causal, has_slopes;
	int vec;              // which rows may be read in whole vectors of 16 bytes: 1 q, 2 k, 4 v, 8 d_o (o in the forward)
	float cap, icap, rw;  // rw = 1/sqrt(W)
	const int32_t* doc;
	const int32_t* prefix;
	void* rest;           // what the rounding of o to 16 bits left out, NULL where it is not wanted
	float slopes[L1_MASKED_HEADS];
};

// how a launch is cut: waves of a workgroup (32 rows each), workgroups that share the other side's tiles among them
struct L1MaskedPlan { int waves, splits; };

struct L1MaskedTable {
	int (*fwd)(L1MaskedArgs&, const L1MaskedPlan&, const void* q, const void* k, const void* v, void* o, float* lse, float* part, hipStream_t);
	int (*rows)(const void* d_o, const void* o, const void* rest, float* D, int64_t rows, int Wv, hipStream_t);
	int (*side_q)(L1MaskedArgs&, const L1MaskedPlan&, const void* q, const void* k, const void* v, const void* d_o, const float* lse, const float* D, void* dq,
	              float* part, hipStream_t);
	int (*side_k)(L1MaskedArgs&, const L1MaskedPlan&, const void* q, const void* k, const void* v, const void* d_o, const float* lse, const float* D, void* dk,
	              void* dv, float* part, hipStream_t);
	int (*lds)(int W, int Wv, int waves, bool backward, bool weigh);
};

const L1MaskedTable& l1_masked_f32();
const L1MaskedTable& l1_masked_f16();
const L1MaskedTable& l1_masked_bf16();
