// 16-bit codes of 16-bit rows, on one grid for both sides of a distance: sums of |difference| of codes (v_sad_u16) stand for sums of
// |difference| of values, in the masked attention and in the attention over the cache.
//
// A value x of column w becomes round(x / u + shift + delta_w), u = a 65533rd of the range.  A code is off by half a step at most,
// a difference by a step: u * sqrt(1/6) rms, if the roundings of the W columns have nothing to do with each other, so that a logit
// moves by u * sqrt(1/6) = 0.41 u rms, whatever W.  The offsets delta_w see to that: without them rows whose columns repeat few
// values round alike everywhere, and a logit moves by up to sqrt(W) u (11 u at W 128; 4.6 u rms for rows of one value).  They are
// frac(3 e / 8) + frac(0.618 c) of the e-th column of the c-th eight: spread evenly over the columns of any eight, of every second,
// fourth, eighth and sixteenth column, and of any block of them.  For rows of one value, of values that repeat with a period of 2 to
// 32, of 2 to 32 blocks, of two values in any order, W 16 to 128: 0.41 u rms at most, 1.8 u the largest of 4000 draws each (2.7 u is
// allowed below).  Rows made to fit the offsets could still agree, up to sqrt(W) u.
//
// Widest range for which codes are taken: 2.7 u is the type's half step, 2^-11 (float16) or 2^-8 (bfloat16) of a weight: 12 and 96.
#pragma once
#include <hip/hip_runtime.h>

template <typename ST> inline constexpr float kCodeRange = 12.f;
template <> inline constexpr float kCodeRange<__bf16> = 96.f;
constexpr float kCodeSteps = 65533.f;  // of the range; the offsets are less than two steps

// delta of the e-th column of the c-th eight, as a part of 65535 steps
__device__ __forceinline__ float l1_code_eight(int c) { return __builtin_amdgcn_fractf(0.618034f * c) * (1.f / 65535.f); }
__device__ __forceinline__ constexpr float l1_code_column(int e) { return (float)(3 * e & 7) * (1.f / (8.f * 65535.f)); }
