// The soft cap of a logit for 16-bit rows, of the masked attention and of the attention over the cache: cap * tanh(y), y = a / cap.
//
// tanh as (e - 1) / (e + 1), e = exp(2y), is off by 2^-23 absolutely.  From |y| = 1/8 on that is 2^-20 of the logit; below, it
// would be multiplied by the cap and become all there is left of the logit (1.5 at a cap of 1e8).  There the series
// y (1 - y^2/3 + 2 y^4/15 - 17 y^6/315) is taken, whose next term is 2^-29 of the first: times the cap it is a times the sum, and
// no rounding grows with the cap.  The series is worked out where a lane of the wave needs it only: for caps of the logits' own
// size that is hardly ever (138 -> 152 us with it for every pair, 16 sequences of 8192 to 32768 tokens, 16 rows, cap 20).
#pragma once
#include <hip/hip_runtime.h>

constexpr float kCapSeries = 0.125f;  // below this |y|

// 1 / cap as the kernels take it: finite, since a distance of zero is multiplied by it (and by 2 log2(e) besides).  Below a cap of
// 1e-38 it is not the reciprocal any more, and the capped logits, no larger than the cap, are nothing beside the no-op's.
static inline float l1_icap(float cap) { return cap > 1e-38f ? 1.f / cap : cap > 0.f ? 1e38f : 0.f; }

// tanh(y), and in d its derivative as 4 e / (1 + e)^2: 1 - tanh^2 has none of its digits left where the cap is a fraction of the logits
__device__ __forceinline__ float l1_tanh_far(float y, float& d)
{
	const float e = __builtin_amdgcn_exp2f(y * 2.885390082f), r = __builtin_amdgcn_rcpf(e + 1.f);
	d = 4.f * e * r * r;
	return (e - 1.f) * r;
}

// tanh(y) / y
__device__ __forceinline__ float l1_tanh_near(float y)
{
	const float y2 = y * y;
	return __builtin_fmaf(y2, __builtin_fmaf(y2, __builtin_fmaf(y2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
}
