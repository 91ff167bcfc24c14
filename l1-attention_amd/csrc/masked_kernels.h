// Masked L1 attention for gfx950, forward and backward, float32 / float16 / bfloat16, grouped key heads:
//
//   a[t,s] = -1/sqrt(W) * sum_w |q[t,w] - k[s,w]|         c = cap * tanh(a / cap)      (cap > 0, else c = a)
//   x[t,s] = c - slope[h] * |i - s|                        i = S - T + t, the query's place among the S tokens
//   p[t,s] = exp(x) / (1 + sum_s exp(x))                   over the visible s; the 1 is the no-op logit
//   o[t]   = sum_s p[t,s] * v[s]
//   visible: (not causal or s <= i or s < prefix[b]) and (no documents or doc[b,s] == doc[b,i] >= 0)
//
// Every logit is <= 0 (slopes are not negative) and the no-op logit is 0, so a row needs no running maximum: exp(x) <= 1,
// the denominator is >= 1, partial sums over pieces of the keys add up, and a row that sees nothing comes out as zero.
//
// One wavefront owns 32 rows ("owners": queries in the forward and in the gradient of q, keys in that of k and v) and walks
// the other side ("stream") in tiles of 64 rows (16-bit forward) or 32 (backward and float32, whose registers would spill far more at
// 64), which the waves of a workgroup share through LDS.  Three parts of a tile use
// three maps of its pairs onto the lanes, joined by a wave-private LDS scratch:
//   distances  lane (i,j) = (lane & 7, lane >> 3) holds owners i + 8a (a < 4) and stream rows j + 8b (b < 8 or 4): 12 LDS reads
//              of 16 bytes feed 32 pairs at b < 8; |q - k| is no contraction, so this is vector-ALU work
//   products   p*v, do*v: matrix instructions; column order of a tile: c = 32*(b/4) + 4*j + b%4, so that a lane's four values
//              of one half of the tile are neighbours
//   signs      lane = column w; the 32 owners' sums live in registers, the score gradients come as broadcast LDS reads
// LDS reads are issued one step ahead of their use, held there by scheduling barriers: left alone, the compiler puts each read
// right before its use, and waits (signs: 12.9 -> 6.6 cycles per 64 pair-elements, float32 distances: 6.7 -> 5.2, at two waves
// a SIMD and 2.4 GHz; the instructions alone are 5.2 and 5.2).
//
// 16-bit inputs: distances are sums of |difference| of 16-bit codes (v_sad_u16: two pair-elements an instruction; 2.5 cycles per
// 64 pair-elements against 5.2 in float32).  The codes are a grid over the range [lo, hi] of the workgroup's owner rows; a stream
// value x outside of it counts as |x - clip(x)|, summed per stream row, plus the code of clip(x): for an owner q within
// the range |q - x| = |q - clip(x)| + |clip(x) - x|.  What the codes' roundings do to a logit, and the widest range hi - lo that
// they are taken for: codes.h.  A workgroup whose owners spread further (or are not finite) takes float32 distances, half of the
// columns at a time.  Signs do not go by these codes but by the bits of the values themselves, as integers in order: sign(q - k)
// is exact.
//
// What bounds it: the vector ALU's issue, with about a quarter of the time waits (1.8 waves a SIMD: sums, codes and tiles fill the
// registers; one above widths of 64).  The gradients of k and v spill: float32 65 to 68 registers up to widths of 64 and 23 to
// 27 at W above, 16 bits 16 to 19 up to widths of 64; nothing else does.  4096 tokens, 16 heads, W 64, every pair visible: bfloat16 forward
// 614 us (v_sad_u16 alone 264), gradients of q 1755 and of k and v 1889; float16 633, 1673 and 1883; float32 1399, 2521 and 2867.
#pragma once
#include "common.h"
#include "masked.h"
#include "softcap.h"
#include "codes.h"
#include <math.h>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short short2v __attribute__((ext_vector_type(2)));

constexpr int kOwn = 32;        // owner rows of a wave
constexpr int kPad = 36;        // floats in a row of the scratch: 9 chunks of 16 bytes, odd, so rows spread over the banks
constexpr int kPitch(int TB) { return 8 * TB + 8; }  // 16-bit values in a row of transposed values: an odd number of chunks
template <int TB> constexpr int kTile = 8 * TB;  // stream rows of a tile: TB for each of the eight lanes j
constexpr int kScratch = kOwn * kPad * 4;
constexpr int kClasses = 1024;  // tiles whose visibility is worked out at a time
constexpr float kMax = 3.402823466e38f;

template <typename ST> constexpr bool k16 = sizeof(ST) == 2;
// What the weights' exponents are counted in: 16-bit rows take 2^x, so that everything but the distance's factor is multiplied by
// log2(e) once per row instead of once per pair.
template <typename ST> constexpr float kUnit = k16<ST> ? 1.442695041f : 1.f;

// The products with weights go through bfloat16 matrix instructions for float16 rows as well: float16 has no room for weights below
// 2^-28 (at 2^14 times their value), which large values and gradients make seen.  A float16 value is two bfloat16 numbers, exactly.
template <typename ST> constexpr bool kTwoParts = __is_same(ST, _Float16);

// an odd number of 16-byte chunks for n of them: neighbouring rows start in different banks
__host__ __device__ __forceinline__ int odd_chunks(int n) { return n | 1; }

// transposed values of a tile as 16-bit numbers
__host__ __device__ __forceinline__ int plane_bytes(int Wv, int TB) { return (Wv + 15) / 16 * 16 * kPitch(TB) * 2; }

// LDS of a workgroup in bytes from the front, the same on host and device.  Rows: own/str distances' rows, oraw/raw the same
// rows' ordered integers (16-bit backward), y the stream's values (float32: rows in product order; 16-bit: rows in product order in
// the backward), yt the same transposed (16-bit, where they are multiplied by p), as bfloat16 numbers, for float16 the second parts behind the first.
struct Layout {
	int own, oraw, str, raw, y, yt, scratch, rows, total;
	int so, sr, sy;  // bytes of a row of own/str, oraw/raw, y
};

template <typename ST, int TB>
__host__ __device__ inline Layout masked_layout(int W, int Wv, int waves, bool backward, bool weigh)
{
	Layout l;
	const int per = 16 / (int)sizeof(ST);
	l.so = odd_chunks((W + per - 1) / per) * 16;
	l.sr = (W + 7) / 8 * 16;
	l.sy = odd_chunks(k16<ST> ? (Wv + 31) / 32 * 4 : (Wv + 3) / 4) * 16;
	l.own = 0;
	l.oraw = l.own + waves * kOwn * l.so;
	l.str = l.oraw + (k16<ST> && backward ? waves * kOwn * l.sr : 0);
	l.raw = l.str + kTile<TB> * l.so;
	l.y = l.raw + (k16<ST> && backward ? kTile<TB> * l.sr : 0);
	l.yt = l.y + (!k16<ST> || backward ? kTile<TB> * l.sy : 0);
	l.scratch = l.yt + (k16<ST> && weigh ? plane_bytes(Wv, TB) * (kTwoParts<ST> ? 2 : 1) : 0);
	l.rows = l.scratch + waves * kScratch;  // documents, lse, D, what lies outside of the range (64 each), 64 words for reductions, classes
	l.total = l.rows + (4 * kTile<TB> + 64) * 4 + kClasses;
	return l;
}

template <typename ST> __device__ __forceinline__ float to_f(ST x) { return (float)x; }

// what y's rounding to the type leaves out, 0 where that is infinite
template <typename ST>
__device__ __forceinline__ ST rest_of(float y)
{
	const float d = y - to_f((ST)y);
	return (ST)(__builtin_fabsf(d) <= kMax ? d : 0.f);
}

// 16 bytes' worth of a row's elements, raw; elements past `n` are zero
template <typename ST>
__device__ __forceinline__ uint4 load_raw(const ST* __restrict__ p, int n, bool vec)
{
	constexpr int per = 16 / (int)sizeof(ST);
	if (vec && n >= per) return *reinterpret_cast<const uint4*>(p);
	ST h[per];
#pragma unroll
	for (int e = 0; e < per; e++) h[e] = e < n ? p[e] : (ST)0.f;
	uint4 r;
	__builtin_memcpy(&r, h, 16);
	return r;
}

template <typename ST, int per = 16 / (int)sizeof(ST)>
__device__ __forceinline__ void unpack(const uint4& r, float (&x)[per])
{
	ST h[per];
	__builtin_memcpy(h, &r, 16);
#pragma unroll
	for (int e = 0; e < per; e++) x[e] = to_f(h[e]);
}


// stream row r of a tile <-> its place c in the order of the products
__device__ __forceinline__ int col_of(int r) { return 32 * (r >> 5) + 4 * (r & 7) + ((r >> 3) & 3); }
__device__ __forceinline__ int row_of(int c) { return ((c >> 2) & 7) + 8 * (4 * (c >> 5) + (c & 3)); }

// a wave's own stores to LDS before its loads of them (LDS works a wave's accesses off in order; this keeps the compiler to it)
__device__ __forceinline__ void wave_sync()
{
	__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
	__builtin_amdgcn_wave_barrier();
}

// The same value, but unknown to the compiler: what is computed from it is computed here, instead of once for the whole loop and
// kept in registers that the loop needs.
__device__ __forceinline__ int here(int x)
{
	asm volatile("" : "+v"(x));
	return x;
}

__device__ __forceinline__ int wave_min(int x)
{
#pragma unroll
	for (int m = 32; m; m >>= 1) x = min(x, __shfl_xor(x, m));
	return x;
}
__device__ __forceinline__ int wave_max(int x)
{
#pragma unroll
	for (int m = 32; m; m >>= 1) x = max(x, __shfl_xor(x, m));
	return x;
}
__device__ __forceinline__ float wave_minf(float x)
{
#pragma unroll
	for (int m = 32; m; m >>= 1) x = fminf(x, __shfl_xor(x, m));
	return x;
}
__device__ __forceinline__ float wave_maxf(float x)
{
#pragma unroll
	for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
	return x;
}

// ------------------------------------------------------------------------------------------------------------- distances

// float32 rows, columns [0, 4 * chunks): acc[a][b] += L1 distance of owner i + 8a and stream row j + 8b.  Four terms are summed
// as a tree before they join the sum: a quarter of the roundings there.  TWO: every second four has a sum of its own, which halves
// what is left of them; at widths above 64 they are most of a result's error (1.6 times the error of sums in pairs throughout, with
// two sums 1.2).  The backward of widths up to 64 has no registers for it (1.35 to 1.5 times; its step would take 10 % longer).
template <bool AHEAD, bool TWO, int TB>
__device__ __forceinline__ void distances32(const char* own, const char* str, int chunks, int stride, int i, int j, float (&acc)[4][TB])
{
	const char *po = own + i * stride, *ps = str + j * stride;
	if constexpr (!AHEAD) {
		for (int c = 0; c < chunks; c++, po += 16, ps += 16) {
			f4 o[4];
#pragma unroll
			for (int a = 0; a < 4; a++) o[a] = *reinterpret_cast<const f4*>(po + 8 * a * stride);
#pragma unroll
			for (int b = 0; b < TB; b++) {
				const f4 s = *reinterpret_cast<const f4*>(ps + 8 * b * stride);
#pragma unroll
				for (int a = 0; a < 4; a++) {
					const float d0 = o[a][0] - s[0], d1 = o[a][1] - s[1], d2 = o[a][2] - s[2], d3 = o[a][3] - s[3];
					acc[a][b] += (__builtin_fabsf(d0) + __builtin_fabsf(d1)) + (__builtin_fabsf(d2) + __builtin_fabsf(d3));
				}
			}
		}
		return;
	}
	const auto load = [&](f4(&o)[4], f4(&s)[TB], int c) {
		const int d = 16 * min(c, chunks - 1);
#pragma unroll
		for (int a = 0; a < 4; a++) o[a] = *reinterpret_cast<const f4*>(po + 8 * a * stride + d);
#pragma unroll
		for (int b = 0; b < TB; b++) s[b] = *reinterpret_cast<const f4*>(ps + 8 * b * stride + d);
		__builtin_amdgcn_sched_barrier(0);
	};
	float odd[4][TB];
#pragma unroll
	for (int a = 0; a < 4; a++)
#pragma unroll
		for (int b = 0; b < TB; b++) odd[a][b] = 0.f;
	const auto work = [&](const f4(&o)[4], const f4(&s)[TB], float(&sum)[4][TB]) {
#pragma unroll
		for (int b = 0; b < TB; b++)
#pragma unroll
			for (int a = 0; a < 4; a++) {
				const float d0 = o[a][0] - s[b][0], d1 = o[a][1] - s[b][1], d2 = o[a][2] - s[b][2], d3 = o[a][3] - s[b][3];
				sum[a][b] += (__builtin_fabsf(d0) + __builtin_fabsf(d1)) + (__builtin_fabsf(d2) + __builtin_fabsf(d3));
			}
		__builtin_amdgcn_sched_barrier(0);
	};
	f4 o0[4], s0[TB], o1[4], s1[TB];
	load(o0, s0, 0);
	for (int c = 0; c < chunks; c += 2) {
		load(o1, s1, c + 1);
		work(o0, s0, acc);
		if (c + 1 >= chunks) break;
		load(o0, s0, c + 2);
		if constexpr (TWO) work(o1, s1, odd);
		else work(o1, s1, acc);
	}
	if constexpr (TWO)
#pragma unroll
		for (int a = 0; a < 4; a++)
#pragma unroll
			for (int b = 0; b < TB; b++) acc[a][b] += odd[a][b];
}

// Rows of 16-bit codes, eight to a chunk.  AHEAD: reads one step ahead, 48 registers more (2.5 instead of 2.75 cycles per 64
// pair-elements; the backward, where distances are a seventh of the work, needs the registers elsewhere).
template <bool AHEAD, int TB>
__device__ __forceinline__ void distances16(const char* own, const char* str, int chunks, int stride, int i, int j, unsigned (&acc)[4][TB])
{
	const char *po = own + i * stride, *ps = str + j * stride;
	if constexpr (!AHEAD) {
		for (int c = 0; c < chunks; c++, po += 16, ps += 16) {
			uint4 o[4];
#pragma unroll
			for (int a = 0; a < 4; a++) o[a] = *reinterpret_cast<const uint4*>(po + 8 * a * stride);
#pragma unroll
			for (int b = 0; b < TB; b++) {
				const uint4 s = *reinterpret_cast<const uint4*>(ps + 8 * b * stride);
#pragma unroll
				for (int a = 0; a < 4; a++) {
					unsigned t = acc[a][b];
					t = __builtin_amdgcn_sad_u16(o[a].x, s.x, t);
					t = __builtin_amdgcn_sad_u16(o[a].y, s.y, t);
					t = __builtin_amdgcn_sad_u16(o[a].z, s.z, t);
					t = __builtin_amdgcn_sad_u16(o[a].w, s.w, t);
					acc[a][b] = t;
				}
			}
		}
		return;
	}
	const auto load = [&](uint4(&o)[4], uint4(&s)[TB], int c) {
		const int d = 16 * min(c, chunks - 1);
#pragma unroll
		for (int a = 0; a < 4; a++) o[a] = *reinterpret_cast<const uint4*>(po + 8 * a * stride + d);
#pragma unroll
		for (int b = 0; b < TB; b++) s[b] = *reinterpret_cast<const uint4*>(ps + 8 * b * stride + d);
		__builtin_amdgcn_sched_barrier(0);
	};
	const auto work = [&](const uint4(&o)[4], const uint4(&s)[TB]) {
#pragma unroll
		for (int b = 0; b < TB; b++)
#pragma unroll
			for (int a = 0; a < 4; a++) {
				unsigned t = acc[a][b];
				t = __builtin_amdgcn_sad_u16(o[a].x, s[b].x, t);
				t = __builtin_amdgcn_sad_u16(o[a].y, s[b].y, t);
				t = __builtin_amdgcn_sad_u16(o[a].z, s[b].z, t);
				t = __builtin_amdgcn_sad_u16(o[a].w, s[b].w, t);
				acc[a][b] = t;
			}
		__builtin_amdgcn_sched_barrier(0);
	};
	uint4 o0[4], s0[TB], o1[4], s1[TB];
	load(o0, s0, 0);
	for (int c = 0; c < chunks; c += 2) {
		load(o1, s1, c + 1);
		work(o0, s0);
		if (c + 1 >= chunks) break;
		load(o0, s0, c + 2);
		work(o1, s1);
	}
}

// --------------------------------------------------------------------------------------------------------------- staging

// Whether a float32 is below 2^-104 and not zero: two of these may differ by less than 2^-128 (others are multiples of 2^-128).
__device__ __forceinline__ bool is_tiny(unsigned bits) { return (bits & 0x7fffffffu) - 1 < __builtin_bit_cast(unsigned, 0x1p-104f) - 1; }

// columns [w0, w0 + width) of rows [r0, r0 + n) of x as float32 rows of `stride` bytes; whether a value is tiny
template <typename ST>
__device__ __forceinline__ bool stage32(char* dst, const ST* __restrict__ x, int r0, int n, int L, int64_t pitch, int w0, int width,
                                        int stride, bool vec, int tid, int threads)
{
	const int chunks = (width + 3) >> 2, j = tid & 7;
	bool tiny = false;
	for (int r = tid >> 3; r < n; r += threads >> 3) {
		const ST* row = x + (int64_t)(r0 + r) * pitch + w0;
		for (int c = j; c < chunks; c += 8) {
			f4 y = {0.f, 0.f, 0.f, 0.f};
			if (r0 + r < L) {
				if constexpr (!k16<ST>) {
					if (vec && 4 * c + 4 <= width) y = *reinterpret_cast<const f4*>(row + 4 * c);
					else
#pragma unroll
						for (int e = 0; e < 4; e++) y[e] = 4 * c + e < width ? to_f(row[4 * c + e]) : 0.f;
				} else {
#pragma unroll
					for (int e = 0; e < 4; e++) y[e] = 4 * c + e < width ? to_f(row[4 * c + e]) : 0.f;
				}
			}
			*reinterpret_cast<f4*>(dst + r * stride + 16 * c) = y;
#pragma unroll
			for (int e = 0; e < 4; e++) tiny |= is_tiny(__builtin_bit_cast(unsigned, y[e]));
		}
	}
	return tiny;
}

// the grid of a workgroup's codes
// x -> x * sc + b, and the column's offset, in [0, 1], which is 65535 steps; inv: one step
struct Grid { float sc, b, inv; };

// eight values, the c-th of a row, as codes, those behind the first n as zero; over: plus what lies outside of [0, 1]
template <typename ST>
__device__ __forceinline__ uint4 codes_of(const uint4& bits, int c, int n, const Grid& G, float& over)
{
	const float b = G.b + l1_code_eight(c);
	float v[8];
	unpack<ST>(bits, v);
	unsigned w[4];
#pragma unroll
	for (int e = 0; e < 8; e++) {
		v[e] = __builtin_fmaf(v[e], G.sc, b + l1_code_column(e));
		if (n < 8) v[e] = e < n ? v[e] : 0.f;
		over += __builtin_fabsf(v[e] - __builtin_amdgcn_fmed3f(v[e], 0.f, 1.f));
	}
#pragma unroll
	for (int e = 0; e < 4; e++) w[e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(v[2 * e], v[2 * e + 1]));
	return make_uint4(w[0], w[1], w[2], w[3]);
}

// the bits of eight 16-bit floats as integers in the same order: -0 and 0 are 0, and equal values and no others are equal
__device__ __forceinline__ uint4 ordered8(const uint4& bits)
{
	const auto two = [](unsigned x) {
		const short2v m = __builtin_bit_cast(short2v, x) >> 15;
		return __builtin_bit_cast(unsigned, (__builtin_bit_cast(short2v, x & 0x7fff7fffu) ^ m) - m);
	};
	return make_uint4(two(bits.x), two(bits.y), two(bits.z), two(bits.w));
}

// The owner rows of a wave as codes, and (raw, unless NULL) as ordered integers.
template <typename ST>
__device__ __forceinline__ void stage_own16(char* dst, char* raw, const ST* __restrict__ x, int r0, int L, int64_t pitch, int W, int stride, int rstride,
                                            const Grid& G, bool vec, int lane)
{
	const int chunks = (W + 7) >> 3;
	for (int r = lane >> 3; r < kOwn; r += 8)
		for (int c = lane & 7; c < chunks; c += 8) {
			uint4 bits = make_uint4(0, 0, 0, 0);
			if (r0 + r < L) bits = load_raw(x + (int64_t)(r0 + r) * pitch + 8 * c, W - 8 * c, vec);
			float over = 0.f;
			*reinterpret_cast<uint4*>(dst + r * stride + 16 * c) = codes_of<ST>(bits, c, W - 8 * c, G, over);
			if (raw) *reinterpret_cast<uint4*>(raw + r * rstride + 16 * c) = ordered8(bits);
		}
}

// A tile of the stream on its way from memory to LDS.  fetch() issues the loads, one tile ahead of their use: they are under way
// while the tile before is worked on; place() converts and stores.  What a thread has of a tile beyond KN (rows) and VN
// (values) 16-byte pieces is loaded in place().
template <typename ST, int TB, int KN, int VN>
struct Stream {
	uint4 k[KN], va[VN], vb[VN];
	int d;
	float l, dd;

	static __device__ __forceinline__ uint4 piece(const ST* __restrict__ x, int r, int L, int64_t pitch, int w, int width, bool vec)
	{
		if (r < L && w < width) return load_raw(x + (int64_t)r * pitch + w, width - w, vec);
		return make_uint4(0, 0, 0, 0);
	}

	__device__ __forceinline__ void fetch(const ST* __restrict__ x, int64_t xpitch, int W, bool xvec, const ST* __restrict__ y, int64_t ypitch, int Wv,
	                                      bool yvec, int s0, int L, const int* doc, const float* lse, const float* D, int rpitch, int tid, int threads)
	{
		constexpr int per = 16 / (int)sizeof(ST);
		const int ncg = ((W + per - 1) / per + 7) >> 3, steps = (8 * kTile<TB> + threads - 1) / threads;
#pragma unroll
		for (int u = 0; u < KN; u++) {
			const int ur = u / ncg, r = (tid >> 3) + ur * (threads >> 3), c = (tid & 7) + 8 * (u - ur * ncg);
			k[u] = r < kTile<TB> ? piece(x, s0 + r, L, xpitch, per * c, W, xvec) : make_uint4(0, 0, 0, 0);
		}
		if constexpr (k16<ST>) {
#pragma unroll
			for (int u = 0; u < VN; u++) {
				const int x2 = tid + threads * u, c2 = x2 % (kTile<TB> / 2), ch = x2 / (kTile<TB> / 2);
				va[u] = piece(y, s0 + row_of(2 * c2), L, ypitch, 8 * ch, Wv, yvec);
				vb[u] = piece(y, s0 + row_of(2 * c2 + 1), L, ypitch, 8 * ch, Wv, yvec);
			}
		} else {
			const int nvg = ((Wv + 3) / 4 + 7) >> 3;
#pragma unroll
			for (int u = 0; u < VN; u++) {
				const int ur = u / nvg, r = (tid >> 3) + ur * (threads >> 3), c = (tid & 7) + 8 * (u - ur * nvg);
				va[u] = r < kTile<TB> ? piece(y, s0 + r, L, ypitch, 4 * c, Wv, yvec) : make_uint4(0, 0, 0, 0);
			}
		}
		if (tid < kTile<TB>) {
			const bool in = s0 + tid < L;
			d = doc && in ? doc[s0 + tid] : -1;
			if (lse) {
				l = in ? lse[(int64_t)(s0 + tid) * rpitch] : 0.f;
				dd = in ? D[(int64_t)(s0 + tid) * rpitch] : 0.f;
			}
		}
	}

	// str: distance rows; raw, over, y, yt, slse, sD: see Layout, NULL where not wanted; tiny (float32, or NULL) is set where a value
	// is.  Whether a value was not finite.
	__device__ __forceinline__ bool place(char* str, char* raw, float* over, char* ydst, char* yt, int* docs, float* slse, float* sD, int* tiny, const Layout& Y,
	                                      const Grid& G, const ST* __restrict__ x, int64_t xpitch, int W, bool xvec, const ST* __restrict__ y,
	                                      int64_t ypitch, int Wv, bool yvec, int s0, int L, int tid, int threads)
	{
		constexpr int per = 16 / (int)sizeof(ST);
		const int chunks = (W + per - 1) / per, ncg = (chunks + 7) >> 3, steps = (8 * kTile<TB> + threads - 1) / threads, j = tid & 7;
		bool bad = false;
		float out = 0.f;
		const auto rows = [&](const uint4& bits, int r, int cg) {
			const int c = j + 8 * cg;
			if (r >= kTile<TB>) return;  // eight lanes at a time: a row's sum is still formed by all of its lanes
			if constexpr (!k16<ST>) {
				if (c < chunks) *reinterpret_cast<uint4*>(str + r * Y.so + 16 * c) = bits;
				if (tiny && (is_tiny(bits.x) | is_tiny(bits.y) | is_tiny(bits.z) | is_tiny(bits.w))) *tiny = 1;
			} else {
				if (cg == 0) out = 0.f;
				if (c < chunks) {
					*reinterpret_cast<uint4*>(str + r * Y.so + 16 * c) = codes_of<ST>(bits, c, W - 8 * c, G, out);
					if (raw) *reinterpret_cast<uint4*>(raw + r * Y.sr + 16 * c) = ordered8(bits);
				}
				if (cg == ncg - 1) {
					float o = out;
					o += __shfl_xor(o, 1);
					o += __shfl_xor(o, 2);
					o += __shfl_xor(o, 4);
					if (j == 0) over[r] = o;
				}
			}
		};
#pragma unroll
		for (int u = 0; u < KN; u++)
			if (u < steps * ncg) rows(k[u], (tid >> 3) + (u / ncg) * (threads >> 3), u % ncg);
		for (int u = KN; u < steps * ncg; u++) {
			const int r = (tid >> 3) + (u / ncg) * (threads >> 3), cg = u % ncg;
			rows(piece(x, s0 + r, L, xpitch, per * (j + 8 * cg), W, xvec), r, cg);
		}
		if constexpr (!k16<ST>) {
			const int vchunks = Y.sy >> 4, nvg = ((Wv + 3) / 4 + 7) >> 3;
			const auto values = [&](const uint4& bits, int r, int cg) {
				const int c = j + 8 * cg;
				if (r >= kTile<TB>) return;
				if (c < vchunks) *reinterpret_cast<uint4*>(ydst + col_of(r) * Y.sy + 16 * c) = bits;
				const f4 v = __builtin_bit_cast(f4, bits);
#pragma unroll
				for (int e = 0; e < 4; e++) bad |= !(__builtin_fabsf(v[e]) <= kMax);
			};
#pragma unroll
			for (int u = 0; u < VN; u++)
				if (u < steps * nvg) values(va[u], (tid >> 3) + (u / nvg) * (threads >> 3), u % nvg);
			for (int u = VN; u < steps * nvg; u++) {
				const int r = (tid >> 3) + (u / nvg) * (threads >> 3), cg = u % nvg;
				values(piece(y, s0 + r, L, ypitch, 4 * (j + 8 * cg), Wv, yvec), r, cg);
			}
		} else {
			// two rows next to each other in the order of the products, eight columns: transposed they are eight pairs
			const int all = kTile<TB> / 2 * (ydst ? (Wv + 31) / 32 * 4 : (Wv + 15) / 16 * 2), tcols = (Wv + 15) / 16 * 16;
			const auto pair = [&](const uint4& A, const uint4& B, int x2) {
				const int c2 = x2 % (kTile<TB> / 2), ch = x2 / (kTile<TB> / 2);
				if (ydst) {
					*reinterpret_cast<uint4*>(ydst + 2 * c2 * Y.sy + 16 * ch) = A;
					*reinterpret_cast<uint4*>(ydst + (2 * c2 + 1) * Y.sy + 16 * ch) = B;
				}
				if (yt) {
					const unsigned a[4] = {A.x, A.y, A.z, A.w}, b[4] = {B.x, B.y, B.z, B.w};
					// not finite: all bits of the exponent, and one more at its end carries into the sign's place
					constexpr unsigned em = __is_same(ST, _Float16) ? 0x7c007c00u : 0x7f807f80u, one = __is_same(ST, _Float16) ? 0x04000400u : 0x00800080u;
					unsigned carry = 0;
#pragma unroll
					for (int e = 0; e < 4; e++) carry |= ((a[e] & em) + one) | ((b[e] & em) + one);
					bad |= (carry & 0x80008000u) != 0;
					if (8 * ch < tcols) {
						char* to = yt + 8 * ch * kPitch(TB) * 2 + 4 * c2;
#pragma unroll
						for (int e = 0; e < 4; e++)
#pragma unroll
							for (int h = 0; h < 2; h++) {
								const unsigned two = __builtin_amdgcn_perm(b[e], a[e], h ? 0x07060302u : 0x05040100u);
								char* at = to + (2 * e + h) * kPitch(TB) * 2;
								if constexpr (kTwoParts<ST>) {
									_Float16 v[2];
									__builtin_memcpy(v, &two, 4);
									const __bf16 first[2] = {(__bf16)(float)v[0], (__bf16)(float)v[1]};
									const __bf16 second[2] = {(__bf16)((float)v[0] - (float)first[0]), (__bf16)((float)v[1] - (float)first[1])};
									__builtin_memcpy(at, first, 4);
									__builtin_memcpy(at + plane_bytes(Wv, TB), second, 4);
								} else {
									*reinterpret_cast<unsigned*>(at) = two;
								}
							}
					}
				}
			};
#pragma unroll
			for (int u = 0; u < VN; u++)
				if (tid + threads * u < all) pair(va[u], vb[u], tid + threads * u);
			for (int x2 = tid + threads * VN; x2 < all; x2 += threads) {
				const int c2 = x2 % (kTile<TB> / 2), ch = x2 / (kTile<TB> / 2);
				pair(piece(y, s0 + row_of(2 * c2), L, ypitch, 8 * ch, Wv, yvec), piece(y, s0 + row_of(2 * c2 + 1), L, ypitch, 8 * ch, Wv, yvec), x2);
			}
		}
		if (tid < kTile<TB>) {
			docs[tid] = d;
			if (slse) { slse[tid] = l * kUnit<ST>; sD[tid] = dd; }
		}
		return bad;
	}
};

// ---------------------------------------------------------------------------------------------------------------- products

template <typename ST>
__device__ __forceinline__ f4 mma16(const uint4& a, const uint4& b, f4 c)
{
	if constexpr (sizeof(ST) == 4) return c;
	else if constexpr (__is_same(ST, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
	else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// Weights of half a tile into the wave's scratch, and acc[tb][wb] += sum over its 32 columns c of value[c][16 wb + ..] * p[owner][c].
// 16 bits: a weight is the sum of two bfloat16 numbers, itself rounded and what that leaves out: one alone, half a step off, made
// the results half as inexact again as their own rounding; two leave 2^-18 of it.  Second part times a float16 value's second part,
// 2^-18 of the product at most, is left out.
// far: 0, or what is visible of a tile with values that are not finite, 2 if some of it is hidden: a hidden pair's weight of zero must
// not meet them, which a matrix instruction cannot leave out; 1 if nothing is: a weight's second part, zero, must not meet them.
template <typename ST, int NB, int TB>
__device__ __forceinline__ void weigh(f4 (&acc)[2][NB], char* scr, const char* y, const char* yt, int sy, int Wv, const float (&p)[4][4], int half,
                                      int i, int j, int l16, int g, int far)
{
	constexpr int pitch = kPad * 4;  // bytes of an owner's 32 weights, of 16 bits the second parts behind the first: odd chunks
	const int plane = plane_bytes(Wv, TB);
	wave_sync();
#pragma unroll
	for (int a = 0; a < 4; a++) {
		if constexpr (k16<ST>) {
			__bf16 w[4], rest[4];
#pragma unroll
			for (int e = 0; e < 4; e++) {
				w[e] = (__bf16)p[a][e];
				rest[e] = (__bf16)(p[a][e] - (float)w[e]);
			}
			uint2 packed;
			__builtin_memcpy(&packed, w, 8);
			*reinterpret_cast<uint2*>(scr + (i + 8 * a) * pitch + 8 * j) = packed;
			__builtin_memcpy(&packed, rest, 8);
			*reinterpret_cast<uint2*>(scr + (i + 8 * a) * pitch + 64 + 8 * j) = packed;
		} else {
			const f4 w = {p[a][0], p[a][1], p[a][2], p[a][3]};
			*reinterpret_cast<f4*>(scr + (i + 8 * a) * pitch + 16 * j) = w;
		}
	}
	wave_sync();
	if (far) {
		const auto number = [](const char* at) { return k16<ST> ? to_f(*reinterpret_cast<const __bf16*>(at)) : *reinterpret_cast<const float*>(at); };
		for (int c = 0; c < 32; c++)
#pragma unroll
			for (int tb = 0; tb < 2; tb++) {
				const char* at = scr + (l16 + 16 * tb) * pitch + (int)sizeof(ST) * c;
				const float w = number(at) + (k16<ST> ? number(at + 64) : 0.f);
				if (w != 0.f || far == 1)
#pragma unroll
					for (int wb = 0; wb < NB; wb++)
#pragma unroll
						for (int e = 0; e < 4; e++) {
							const int col = 16 * wb + 4 * g + e;
							if (col >= Wv) continue;
							const char* from = k16<ST> ? yt + col * kPitch(TB) * 2 + 64 * half + 2 * c : y + (32 * half + c) * sy + 4 * col;
							float v = number(from);
							if (kTwoParts<ST> && __builtin_fabsf(v) <= kMax) v += number(from + plane);
							acc[tb][wb][e] += w * v;
						}
			}
		return;
	}
	if constexpr (!k16<ST>) {
		const char* val = y + 32 * half * sy;
#pragma unroll
		for (int kc = 0; kc < 2; kc++) {
			f4 pb[2];
#pragma unroll
			for (int tb = 0; tb < 2; tb++) pb[tb] = *reinterpret_cast<const f4*>(scr + (l16 + 16 * tb) * pitch + 64 * kc + 16 * g);
#pragma unroll
			for (int e = 0; e < 4; e++) {
				const char* row = val + (16 * kc + 4 * g + e) * sy;
#pragma unroll
				for (int wb = 0; wb < NB; wb++) {
					const float av = *reinterpret_cast<const float*>(row + 4 * min(16 * wb + l16, Wv - 1));  // rows behind the width are not written
#pragma unroll
					for (int tb = 0; tb < 2; tb++) acc[tb][wb] = __builtin_amdgcn_mfma_f32_16x16x4f32(av, pb[tb][e], acc[tb][wb], 0, 0, 0);
				}
			}
		}
	} else {
		const int blocks = (Wv + 15) >> 4;
		uint4 pb[2], rest[2];
#pragma unroll
		for (int tb = 0; tb < 2; tb++) {
			pb[tb] = *reinterpret_cast<const uint4*>(scr + (l16 + 16 * tb) * pitch + 16 * g);
			rest[tb] = *reinterpret_cast<const uint4*>(scr + (l16 + 16 * tb) * pitch + 64 + 16 * g);
		}
#pragma unroll
		for (int wb = 0; wb < NB; wb++) {
			if (wb >= blocks) break;
			const char* from = yt + (16 * wb + l16) * kPitch(TB) * 2 + 64 * half + 16 * g;
			const uint4 av = *reinterpret_cast<const uint4*>(from);
#pragma unroll
			for (int tb = 0; tb < 2; tb++) acc[tb][wb] = mma16<__bf16>(av, rest[tb], mma16<__bf16>(av, pb[tb], acc[tb][wb]));
			if constexpr (kTwoParts<ST>) {
				const uint4 second = *reinterpret_cast<const uint4*>(from + plane);
#pragma unroll
				for (int tb = 0; tb < 2; tb++) acc[tb][wb] = mma16<__bf16>(second, pb[tb], acc[tb][wb]);
			}
		}
	}
}

// --------------------------------------------------------------------------------------------------------------- visibility

struct Span { int lo, hi; };  // least and largest of the document numbers >= 0 (lo > hi: there is none), over a group of rows

// What a tile of the stream is to a group of owners: 0 nothing of it is visible, 1 all of it, 2 some of it.
// own_lo..own_hi, s_lo..s_hi: places among the S tokens.  OWNK: the owners are keys, the stream queries.
template <bool OWNK>
__device__ __forceinline__ int place_class(const L1MaskedArgs& A, int prefix, int own_lo, int own_hi, int s_lo, int s_hi, bool whole)
{
	if (!A.causal) return whole ? 1 : 2;
	const int key_lo = OWNK ? own_lo : s_lo, key_hi = OWNK ? own_hi : s_hi;
	const int q_lo = OWNK ? s_lo : own_lo, q_hi = OWNK ? s_hi : own_hi;
	if (key_lo > q_hi && key_lo >= prefix) return 0;
	return whole && (key_hi <= q_lo || key_hi < prefix) ? 1 : 2;
}

// the same with documents, by a whole wave; d: the document of stream row `lane` of the tile, -1 where there is none
template <int TB>
__device__ __forceinline__ int doc_class(int c, int d, Span own, bool own_whole, int lane)
{
	if (!__ballot(d >= 0 && d >= own.lo && d <= own.hi && lane < kTile<TB>)) return 0;
	return !own_whole || own.lo != own.hi || __ballot(d != own.lo && lane < kTile<TB>) ? 2 : c;
}

// where a workgroup's owners lie and what the two sides are
struct Block {
	int b, h, hk, own0, nown;    // batch entry, query head, key head, the workgroup's first owner row, rows it has at most
	int own_rows, str_rows;      // rows of the owners' and of the stream's side
	int own_place0, str_place0;  // place of row 0 of either side
};

// classes of the tiles first + step * t, t < n, for the whole workgroup
template <bool OWNK, int TB>
__device__ __forceinline__ void classify(const L1MaskedArgs& A, const Block& K, const int* doc, int prefix, int own_lo, int own_hi, Span own_docs,
                                         bool own_whole, int first, int step, int n, unsigned char* cls, int tid, int threads)
{
	const auto by_place = [&](int t) {
		const int lo = (first + step * t) * kTile<TB>, hi = min(lo + kTile<TB>, K.str_rows);
		return place_class<OWNK>(A, prefix, own_lo, own_hi, K.str_place0 + lo, K.str_place0 + hi - 1, hi - lo == kTile<TB>);
	};
	if (!doc) {
		for (int t = tid; t < n; t += threads) cls[t] = (unsigned char)by_place(t);
		return;
	}
	// a wave for each tile, eight tiles' loads at a time: their latency is most of this
	const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = threads >> 6;
	for (int t0 = wave; t0 < n; t0 += 8 * waves) {
		int d[8];
#pragma unroll
		for (int u = 0; u < 8; u++) {
			const int row = (first + step * (t0 + u * waves)) * kTile<TB> + lane;
			d[u] = -1;
			if (t0 + u * waves < n && lane < kTile<TB> && row < K.str_rows) d[u] = doc[K.str_place0 + row];
		}
#pragma unroll
		for (int u = 0; u < 8; u++) {
			const int t = t0 + u * waves;
			if (t >= n) break;
			int c = by_place(t);
			if (c) c = doc_class<TB>(c, d[u], own_docs, own_whole, lane);
			if (lane == 0) cls[t] = (unsigned char)c;
		}
	}
}

__device__ __forceinline__ int next_tile(const unsigned char* cls, int t, int n)
{
	while (t < n && !cls[t]) t++;
	return __builtin_amdgcn_readfirstlane(t);  // the same in all lanes
}

// no short cuts: a branch for every pair would cost more than the comparisons
__device__ __forceinline__ bool sees(bool open, int prefix, bool nodocs, int qp, int kp, int qd, int kd)
{
	return (open | (kp <= qp) | (kp < prefix)) & (nodocs | ((qd == kd) & (qd >= 0)));
}

// documents of a wave's own rows, and of the workgroup's (through `shared`); whole: each row belongs to one
__device__ __forceinline__ void owner_docs(const int* doc, const Block& K, int row0, int* shared, int lane, int wave, int waves, Span& mine, bool& mine_whole,
                                           Span& all, bool& all_whole)
{
	int lo = 0x7fffffff, hi = -1, none = 0;
	if (doc && lane < kOwn && row0 + lane < K.own_rows) {
		const int d = doc[K.own_place0 + row0 + lane];
		if (d >= 0) lo = hi = d; else none = 1;
	}
	lo = wave_min(lo); hi = wave_max(hi); none = wave_max(none);
	mine = {__builtin_amdgcn_readfirstlane(lo), __builtin_amdgcn_readfirstlane(hi)};
	mine_whole = !__builtin_amdgcn_readfirstlane(none);
	if (lane == 0) { shared[3 * wave] = lo; shared[3 * wave + 1] = hi; shared[3 * wave + 2] = none; }
	__syncthreads();
	for (int w = 0; w < waves; w++) { lo = min(lo, shared[3 * w]); hi = max(hi, shared[3 * w + 1]); none = max(none, shared[3 * w + 2]); }
	all = {lo, hi};
	all_whole = !none;
}

// The grid over the workgroup's owner rows; false where their values spread too far for it, or are not finite.  Rows that
// belong to no document are left out: they take part in nothing.
template <typename ST>
__device__ __forceinline__ bool owner_grid(const ST* __restrict__ x, const int* doc, const Block& K, int row0, int64_t pitch, int W, bool vec, float* shared,
                                           int lane, int wave, int waves, Grid& G)
{
	float lo = kMax, hi = -kMax;
	bool finite = true;
	const int chunks = (W + 7) >> 3;
	for (int r = lane >> 3; r < kOwn; r += 8) {
		if (row0 + r >= K.own_rows || (doc && doc[K.own_place0 + row0 + r] < 0)) continue;
		for (int c = lane & 7; c < chunks; c += 8) {
			float v[8];
			unpack<ST>(load_raw(x + (int64_t)(row0 + r) * pitch + 8 * c, W - 8 * c, vec), v);
#pragma unroll
			for (int e = 0; e < 8; e++)
				if (8 * c + e < W) {
					finite = finite && __builtin_fabsf(v[e]) <= kMax;
					lo = fminf(lo, v[e]);
					hi = fmaxf(hi, v[e]);
				}
		}
	}
	lo = wave_minf(lo); hi = wave_maxf(hi);
	if (lane == 0) { shared[3 * wave] = lo; shared[3 * wave + 1] = hi; }
	const bool all_finite = !__syncthreads_or(!finite);
	for (int w = 0; w < waves; w++) { lo = fminf(lo, shared[3 * w]); hi = fmaxf(hi, shared[3 * w + 1]); }
	if (lo > hi) lo = hi = 0.f;  // no row takes part
	// a margin of 2^-20 on both sides, or the roundings of x * sc + b would put an owner outside
	const float span = (hi - lo) * (1.f + 0x1p-19f);
	lo -= (hi - lo) * 0x1p-20f;
	G.inv = span * (1.f / kCodeSteps);
	G.sc = span > 0.f ? 1.f / (G.inv * 65535.f) : 0.f;
	G.b = -lo * G.sc;
	// b is rounded by 2^-21 at most up to 8, which the margin covers: values that lie further from zero than that, for their
	// span, or next to nothing apart, or all the same, go without codes
	return all_finite && span <= kCodeRange<ST> && span > 0.f && G.sc <= 1e30f && __builtin_fabsf(G.b) <= 8.f;
}

// A wave's distances of one tile, acc[a][b] >= 0 scaled by 1/sqrt(W), NaN where a value is.  Called by all waves of the
// workgroup; `active`: this wave needs them.  Without a grid 16-bit rows go through LDS as float32, half of the columns at a time.
template <typename ST, bool AHEAD, bool TWO, int TB>
__device__ __forceinline__ void tile_distances(char* own, char* str, const float* over, const Layout& Y, int W, float rw, const Grid& G, bool coded,
                                               bool active, const ST* __restrict__ own_x, int own_r0, int own_rows, int64_t own_pitch,
                                               const ST* __restrict__ str_x, int s0, int str_rows, int64_t str_pitch, int i, int j, int tid, int threads,
                                               float (&x)[4][TB])
{
	if constexpr (!k16<ST>) {
#pragma unroll
		for (int a = 0; a < 4; a++)
#pragma unroll
			for (int b = 0; b < TB; b++) x[a][b] = 0.f;
		if (active) distances32<AHEAD, TWO, TB>(own, str, (W + 3) >> 2, Y.so, i, j, x);
#pragma unroll
		for (int a = 0; a < 4; a++)
#pragma unroll
			for (int b = 0; b < TB; b++) x[a][b] *= rw;
	} else if (coded) {
		if (!active) return;
		unsigned acc[4][TB];
#pragma unroll
		for (int a = 0; a < 4; a++)
#pragma unroll
			for (int b = 0; b < TB; b++) acc[a][b] = 0;
		distances16<AHEAD, TB>(own, str, (W + 7) >> 3, Y.so, i, j, acc);
		const float m = G.inv * rw, span = m * 65535.f;
#pragma unroll
		for (int b = 0; b < TB; b++) {
			const float o = over[j + 8 * b] * span;
#pragma unroll
			for (int a = 0; a < 4; a++) x[a][b] = __builtin_fmaf((float)acc[a][b], m, o);
		}
	} else {
#pragma unroll
		for (int a = 0; a < 4; a++)
#pragma unroll
			for (int b = 0; b < TB; b++) x[a][b] = 0.f;
		const int part = 4 * (((W + 7) >> 3));  // columns that fit a row of codes
		for (int w0 = 0; w0 < W; w0 += part) {
			const int n = min(part, W - w0);
			__syncthreads();
			stage32(own, own_x, own_r0, kOwn, own_rows, own_pitch, w0, n, Y.so, false, tid & 63, 64);
			stage32(str, str_x, s0, kTile<TB>, str_rows, str_pitch, w0, n, Y.so, false, tid, threads);
			__syncthreads();
			if (active) distances32<false, false, TB>(own, str, (n + 3) >> 2, Y.so, i, j, x);
		}
#pragma unroll
		for (int a = 0; a < 4; a++)
#pragma unroll
			for (int b = 0; b < TB; b++) x[a][b] *= rw;
	}
}

// Capped scores in those units of half a tile and, in fac, their derivatives by the score, from the distances over sqrt(W) (in
// those units without a cap).
template <typename ST, bool CAP, int TB>
__device__ __forceinline__ void scores(float (&c)[4][4], float (&fac)[4][4], const float (&x)[4][TB], int half, float cap, float icap)
{
	if constexpr (!CAP) {
#pragma unroll
		for (int bb = 0; bb < 4; bb++)
#pragma unroll
			for (int a = 0; a < 4; a++) {
				c[a][bb] = -x[a][4 * half + bb];
				fac[a][bb] = 1.f;
			}
	} else if constexpr (!k16<ST>) {
#pragma unroll
		for (int bb = 0; bb < 4; bb++)
#pragma unroll
			for (int a = 0; a < 4; a++) {
				const float y = -x[a][4 * half + bb] * icap, e = expf(2.f * y), d = 1.f + e;
				fac[a][bb] = 4.f * e / (d * d);  // 1 - tanh^2, with all of its digits
				c[a][bb] = cap * tanhf(y);
			}
	} else {
		unsigned least = 0x7f800000;  // distances are not negative: their bits are in their order
#pragma unroll
		for (int bb = 0; bb < 4; bb++)
#pragma unroll
			for (int a = 0; a < 4; a++) least = min(least, __builtin_bit_cast(unsigned, x[a][4 * half + bb]));
		if (__any(__builtin_bit_cast(float, least) * icap < kCapSeries)) {
#pragma unroll
			for (int bb = 0; bb < 4; bb++)
#pragma unroll
				for (int a = 0; a < 4; a++) {
					float f;
					const float d = x[a][4 * half + bb], y = d * icap, r = l1_tanh_near(y), t = l1_tanh_far(-y, f);
					fac[a][bb] = y < kCapSeries ? 1.f - y * y * r * r : f;
					c[a][bb] = (y < kCapSeries ? -d * r : cap * t) * kUnit<ST>;
				}
		} else {
#pragma unroll
			for (int bb = 0; bb < 4; bb++)
#pragma unroll
				for (int a = 0; a < 4; a++) {
					c[a][bb] = cap * kUnit<ST> * l1_tanh_far(-x[a][4 * half + bb] * icap, fac[a][bb]);
				}
		}
	}
}

template <typename ST>
__device__ __forceinline__ float weight(float x)
{
	if constexpr (k16<ST>) return __builtin_amdgcn_exp2f(x);
	else return expf(x);
}

// ----------------------------------------------------------------------------------------------------------------- forward

// NB: 16-column blocks of the value width held by a wave.  Grid: x = batch * head (heads next to each other go to different
// XCDs and one head's tiles to one), y = owner tiles, the last first: under causality it has the most to do; z = splits: split
// z takes every gridDim.z-th tile of the stream.  part: NULL, or [splits][B][T][H][Wv up to a multiple of 4] sums to be
// joined, and behind them the weights' sums [splits][B][T][H].
template <typename ST, bool CAP, int NB, int TB, int THREADS>
__global__ void __launch_bounds__(THREADS) masked_fwd(L1MaskedArgs A, const ST* __restrict__ q, const ST* __restrict__ k,
                                                      const ST* __restrict__ v, ST* __restrict__ o, float* __restrict__ lse, float* __restrict__ part)
{
	constexpr int KN = k16<ST> && NB == 8 ? 4 : 2, VN = k16<ST> && NB < 8 ? 1 : 2;
	extern __shared__ __align__(16) char lds[];
	const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = threads >> 6;
	const int i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
	Block K;
	K.b = blockIdx.x / A.H; K.h = blockIdx.x % A.H; K.hk = K.h / (A.H / A.Hk);
	K.nown = waves * kOwn; K.own0 = (gridDim.y - 1 - blockIdx.y) * K.nown;
	K.own_rows = A.T; K.str_rows = A.S; K.own_place0 = A.S - A.T; K.str_place0 = 0;
	const int row0 = K.own0 + wave * kOwn;
	const Layout Y = masked_layout<ST, TB>(A.W, A.Wv, waves, false, true);
	char *own = lds + Y.own + wave * kOwn * Y.so, *str = lds + Y.str, *y = lds + Y.y, *yt = lds + Y.yt, *scr = lds + Y.scratch + wave * kScratch;
	int* docs = reinterpret_cast<int*>(lds + Y.rows);
	float* over = reinterpret_cast<float*>(lds + Y.rows) + 3 * kTile<TB>;
	float* red = over + kTile<TB>;
	unsigned char* cls = reinterpret_cast<unsigned char*>(red + 64);
	const int* doc = A.doc ? A.doc + (int64_t)K.b * A.S : nullptr;
	const int prefix = A.prefix ? A.prefix[K.b] : 0;
	const float slope = A.has_slopes ? fminf(A.slopes[K.h] * kUnit<ST>, kMax) : 0.f;  // finite: a distance of zero is multiplied by it
	const int64_t qpitch = (int64_t)A.H * A.W, kpitch = (int64_t)A.Hk * A.W, vpitch = (int64_t)A.Hk * A.Wv;
	const ST* qh = q + ((int64_t)K.b * A.T * A.H + K.h) * A.W;
	const ST* kh = k + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.W;
	const ST* vh = v + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.Wv;

	Span mine, all;
	bool mine_whole, all_whole;
	owner_docs(doc, K, row0, reinterpret_cast<int*>(red), lane, wave, waves, mine, mine_whole, all, all_whole);
	Grid G = {0.f, 0.f, 0.f};
	bool coded = false;
	if constexpr (k16<ST>) {
		coded = owner_grid(qh, doc, K, row0, qpitch, A.W, A.vec & 1, red + 32, lane, wave, waves, G);
		if (coded) stage_own16(own, (char*)nullptr, qh, row0, A.T, qpitch, A.W, Y.so, 0, G, A.vec & 1, lane);
	} else {
		stage32(own, qh, row0, kOwn, A.T, qpitch, 0, A.W, Y.so, A.vec & 1, lane, 64);
	}
	const int own_lo = K.own_place0 + K.own0, own_hi = K.own_place0 + min(K.own0 + K.nown, A.T) - 1;
	const int my_lo = K.own_place0 + row0, my_hi = K.own_place0 + min(row0 + kOwn, A.T) - 1;
	int od4[4];
#pragma unroll
	for (int a = 0; a < 4; a++) od4[a] = doc && row0 + i + 8 * a < A.T ? doc[my_lo + i + 8 * a] : -1;
	f4 out[2][NB];
	float den[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int tb = 0; tb < 2; tb++)
#pragma unroll
		for (int wb = 0; wb < NB; wb++) out[tb][wb] = (f4)(0.f);
	const int s_end = A.causal ? min(A.S, max(own_hi + 1, prefix)) : A.S;  // nothing behind is visible
	const int tiles = (s_end + kTile<TB> - 1) / kTile<TB>, step = gridDim.z;
	for (int t0 = blockIdx.z; t0 < tiles; t0 += step * kClasses) {
		const int n = min(kClasses, (tiles - t0 + step - 1) / step);
		__syncthreads();
		classify<false, TB>(A, K, doc, prefix, own_lo, own_hi, all, all_whole, t0, step, n, cls, tid, threads);
		__syncthreads();
		Stream<ST, TB, KN, VN> F;
		int next = next_tile(cls, 0, n);
		if (next < n) F.fetch(kh, kpitch, A.W, A.vec & 2, vh, vpitch, A.Wv, A.vec & 4, (t0 + step * next) * kTile<TB>, A.S, doc, nullptr, nullptr, 0, tid, threads);
		while (next < n) {
			const int kind = __builtin_amdgcn_readfirstlane(cls[next]), s0 = (t0 + step * next) * kTile<TB>;
			const int tid = here(threadIdx.x), lane = tid & 63, i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
			__syncthreads();
			bool bad = F.place(str, nullptr, over, k16<ST> ? nullptr : y, yt, docs, nullptr, nullptr, nullptr, Y, G, kh, kpitch, A.W, A.vec & 2, vh, vpitch, A.Wv,
			                   A.vec & 4, s0, A.S, tid, threads);
			next = next_tile(cls, next + 1, n);
			if (next < n) F.fetch(kh, kpitch, A.W, A.vec & 2, vh, vpitch, A.Wv, A.vec & 4, (t0 + step * next) * kTile<TB>, A.S, doc, nullptr, nullptr, 0, tid, threads);
			const int far = __syncthreads_or(bad && (k16<ST> || kind == 2)) ? kind : 0;
			int mykind = row0 < A.T ? kind : 0;
			if (mykind == 2) {
				mykind = place_class<false>(A, prefix, my_lo, my_hi, s0, min(s0 + kTile<TB>, A.S) - 1, s0 + kTile<TB> <= A.S);
				if (mykind && doc) mykind = doc_class<TB>(mykind, docs[lane % kTile<TB>], mine, mine_whole, lane);
			}
			mykind = __builtin_amdgcn_readfirstlane(mykind);  // what the tile is to this wave's own rows
			float x[4][TB];
			tile_distances<ST, true, true, TB>(own, str, over, Y, A.W, CAP ? A.rw : A.rw * kUnit<ST>, G, coded, mykind, qh, row0, A.T, qpitch, kh, s0, A.S, kpitch, i, j, tid, threads, x);
			if (!mykind) continue;
			// float32: a tile's sum on its own, then to the total: the roundings of either are fewer
			f4 tile[2][NB];
			if constexpr (!k16<ST>)
#pragma unroll
				for (int tb = 0; tb < 2; tb++)
#pragma unroll
					for (int wb = 0; wb < NB; wb++) tile[tb][wb] = (f4)(0.f);
#pragma unroll
			for (int half = 0; half < TB / 4; half++) {
				float p[4][4], fac[4][4];
				scores<ST, CAP, TB>(p, fac, x, half, A.cap, A.icap);
				if (slope != 0.f) {
					asm volatile("");  // a branch
#pragma unroll
					for (int bb = 0; bb < 4; bb++) {
						const float s = (float)(s0 + j + 8 * (4 * half + bb) - my_lo - i);
#pragma unroll
						for (int a = 0; a < 4; a++) p[a][bb] = __builtin_fmaf(-slope, __builtin_fabsf(s - 8.f * a), p[a][bb]);
					}
				}
#pragma unroll
				for (int bb = 0; bb < 4; bb++)
#pragma unroll
					for (int a = 0; a < 4; a++) p[a][bb] = weight<ST>(p[a][bb]);
				if (mykind == 2) {
					asm volatile("");  // a branch: the compiler would rather compare in every tile and select
#pragma unroll
					for (int bb = 0; bb < 4; bb++) {
						const int s = s0 + j + 8 * (4 * half + bb), sd = docs[j + 8 * (4 * half + bb)];
#pragma unroll
						for (int a = 0; a < 4; a++)
							p[a][bb] = (s < A.S) & sees(!A.causal, prefix, !doc, my_lo + i + 8 * a, s, od4[a], sd) ? p[a][bb] : 0.f;
					}
				}
#pragma unroll
				for (int bb = 0; bb < 4; bb++)
#pragma unroll
					for (int a = 0; a < 4; a++) den[a] += p[a][bb];
				if constexpr (k16<ST>) weigh<ST, NB, TB>(out, scr, y, yt, Y.sy, A.Wv, p, half, i, j, l16, g, far);
				else weigh<ST, NB, TB>(tile, scr, y, yt, Y.sy, A.Wv, p, half, i, j, l16, g, far);
			}
			if constexpr (!k16<ST>)
#pragma unroll
				for (int tb = 0; tb < 2; tb++)
#pragma unroll
					for (int wb = 0; wb < NB; wb++) out[tb][wb] += tile[tb][wb];
		}
	}
	// a row's sum lies in the eight lanes j; then to the lanes that hold the row's output
#pragma unroll
	for (int a = 0; a < 4; a++) {
		den[a] += __shfl_xor(den[a], 8);
		den[a] += __shfl_xor(den[a], 16);
		den[a] += __shfl_xor(den[a], 32);
	}
	float* sc = reinterpret_cast<float*>(scr);
	wave_sync();
	if (j == 0)
#pragma unroll
		for (int a = 0; a < 4; a++) sc[i + 8 * a] = den[a];
	wave_sync();
	const int64_t rows = (int64_t)A.B * A.T * A.H;
#pragma unroll
	for (int tb = 0; tb < 2; tb++) {
		const int t = row0 + 16 * tb + l16;
		const float d = sc[16 * tb + l16];
		if (t >= A.T) continue;
		const int64_t row = ((int64_t)K.b * A.T + t) * A.H + K.h;
		const int wp = (A.Wv + 3) & ~3;
		float* to = part ? part + (blockIdx.z * rows + row) * wp : nullptr;
		const float r = part ? 1.f : 1.f / (1.f + d);
		if (g == 0) {
			if (part) part[gridDim.z * rows * wp + blockIdx.z * rows + row] = d;
			else if (lse) lse[row] = log1pf(d);
		}
#pragma unroll
		for (int wb = 0; wb < NB; wb++) {
			const int w = 16 * wb + 4 * g;
			if (part) {
				if (w < wp) *reinterpret_cast<f4*>(to + w) = out[tb][wb] * r;
			} else if (k16<ST> && A.vec & 8 && w + 4 <= A.Wv) {
				ST h[4];
#pragma unroll
				for (int e = 0; e < 4; e++) h[e] = (ST)(out[tb][wb][e] * r);
				uint2 packed;
				__builtin_memcpy(&packed, h, 8);
				*reinterpret_cast<uint2*>(o + row * A.Wv + w) = packed;
				if (A.rest) {
#pragma unroll
					for (int e = 0; e < 4; e++) h[e] = rest_of<ST>(out[tb][wb][e] * r);
					__builtin_memcpy(&packed, h, 8);
					*reinterpret_cast<uint2*>((ST*)A.rest + row * A.Wv + w) = packed;
				}
			} else {
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (w + e < A.Wv) {
						o[row * A.Wv + w + e] = (ST)(out[tb][wb][e] * r);
						if (k16<ST> && A.rest) ((ST*)A.rest)[row * A.Wv + w + e] = rest_of<ST>(out[tb][wb][e] * r);
					}
			}
		}
	}
}

template <typename ST>
__global__ void __launch_bounds__(256) masked_fwd_join(const float* __restrict__ part, int splits, int64_t rows, int Wv, ST* __restrict__ o, ST* __restrict__ rest,
                                                       float* __restrict__ lse)
{
	const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
	if (row >= rows) return;
	const int lane = threadIdx.x & 63, wp = (Wv + 3) & ~3;
	float d = 0.f, y0 = 0.f, y1 = 0.f;
	for (int z = 0; z < splits; z++) {
		const float* p = part + (z * rows + row) * wp;
		d += part[splits * rows * wp + z * rows + row];
		if (lane < Wv) y0 += p[lane];
		if (lane + 64 < Wv) y1 += p[lane + 64];
	}
	const float r = 1.f / (1.f + d);
	if (lse && lane == 0) lse[row] = log1pf(d);
	if (lane < Wv) o[row * Wv + lane] = (ST)(y0 * r);
	if (lane + 64 < Wv) o[row * Wv + lane + 64] = (ST)(y1 * r);
	if (k16<ST> && rest) {
		if (lane < Wv) rest[row * Wv + lane] = rest_of<ST>(y0 * r);
		if (lane + 64 < Wv) rest[row * Wv + lane + 64] = rest_of<ST>(y1 * r);
	}
}

// ---------------------------------------------------------------------------------------------------------------- backward

// D[row] = sum_w do * o, row = (b, t, h): what the softmax's gradient takes off each do . v.  Where the values have a part in
// common the two nearly cancel, so the 16-bit o alone would do it too roughly (dq off by 2.8 % instead of 0.17 % rms: 512 tokens,
// values of mean 4 and spread 1, bfloat16): rest is what its rounding left out, or NULL.
template <typename ST>
__global__ void __launch_bounds__(256) masked_bwd_rows(const ST* __restrict__ dout, const ST* __restrict__ o, const ST* __restrict__ rest,
                                                       float* __restrict__ D, int64_t rows, int Wv)
{
	for (int64_t first = (int64_t)blockIdx.x * 32; first < rows; first += (int64_t)gridDim.x * 32) {  // the same steps for all threads
		const int64_t row = first + (threadIdx.x >> 3);
		float s = 0.f;
		if (row < rows)
			for (int w = threadIdx.x & 7; w < Wv; w += 8) s += to_f(dout[row * Wv + w]) * (to_f(o[row * Wv + w]) + (k16<ST> && rest ? to_f(rest[row * Wv + w]) : 0.f));
		s += __shfl_xor(s, 1);
		s += __shfl_xor(s, 2);
		s += __shfl_xor(s, 4);
		if (row < rows && (threadIdx.x & 7) == 0) D[row] = s;
	}
}

// sum of the splits' gradients, in their order
template <typename ST>
__global__ void __launch_bounds__(256) masked_bwd_join(const float* __restrict__ part, int splits, int64_t n, ST* __restrict__ x)
{
	const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
	if (at >= n) return;
	float s = 0.f;
	for (int z = 0; z < splits; z++) s += part[z * n + at];
	x[at] = (ST)s;
}

// Signs of one half tile: sum[u][r] += h * g over its 32 columns c, h = 1, 1/2, 0 for owner >, ==, < stream in column w = lane + 64 u.
// Owner r = 4 i' + a' is row i' + 8 a'; scr: the gradients g [c][r].
// 16 bits: the values as integers in order, own + 1/2: h = clamp(own + 1/2 - str, 0, 1), exact.  float32: h =
// clamp((own - str) * 2^127 + 1/2, 0, 1), exact but for differences below 2^-128; where the workgroup has met tiny values, times
// 2^276 instead (v_ldexp takes longer: 4 % of a step, if it were taken always).
template <typename ST, int WL>
__device__ __forceinline__ void signs(float (&sum)[WL][32], const float (&ov)[WL][32], const float* sc, const char* str, int stride, int half, int lane, int W,
                                      bool tiny)
{
	const auto value = [&](int c, int u) {
		const char* at = str + row_of(32 * half + c) * stride + (int)sizeof(ST) * min(lane + 64 * u, W - 1);
		if constexpr (k16<ST>) return (float)*reinterpret_cast<const short*>(at);
		else return *reinterpret_cast<const float*>(at);
	};
	if (!k16<ST> && tiny) {
		for (int c = 0; c < 32; c++)
#pragma unroll
			for (int u = 0; u < WL; u++) {
				const float s = value(c, u);
#pragma unroll
				for (int r = 0; r < 32; r++)
					sum[u][r] = __builtin_fmaf(__builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(ov[u][r] - s, 276) + 0.5f, 0.f, 1.f), sc[c * kPad + r], sum[u][r]);
			}
		return;
	}
	f4 g[4], gn[4];  // the gradients of 16 owners, and of the next 16
	float s[WL];
#pragma unroll
	for (int r = 0; r < 4; r++) g[r] = *reinterpret_cast<const f4*>(sc + 4 * r);
#pragma unroll
	for (int u = 0; u < WL; u++) s[u] = value(0, u);
	const auto add = [&](const f4(&x)[4], int r0) {
#pragma unroll
		for (int r = 0; r < 16; r++)
#pragma unroll
			for (int u = 0; u < WL; u++) {
				const float df = ov[u][r0 + r] - s[u];
				const float hv = __builtin_amdgcn_fmed3f(k16<ST> ? df : __builtin_fmaf(df, 0x1p127f, 0.5f), 0.f, 1.f);
				sum[u][r0 + r] = __builtin_fmaf(hv, x[r >> 2][r & 3], sum[u][r0 + r]);
			}
	};
	for (int c = 0; c < 32; c++) {
		const int d = min(c + 1, 31);
		float sn[WL];
#pragma unroll
		for (int r = 0; r < 4; r++) gn[r] = *reinterpret_cast<const f4*>(sc + c * kPad + 16 + 4 * r);
#pragma unroll
		for (int u = 0; u < WL; u++) sn[u] = value(d, u);
		__builtin_amdgcn_sched_barrier(0);
		add(g, 0);
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int r = 0; r < 4; r++) g[r] = *reinterpret_cast<const f4*>(sc + d * kPad + 4 * r);
		__builtin_amdgcn_sched_barrier(0);
		add(gn, 16);
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int u = 0; u < WL; u++) s[u] = sn[u];
	}
}

// Gradients of one side.  OWNK false: owners are queries, dx = dq.  OWNK true: owners are keys, dx = dk and dy = dv, summed
// over the query heads that share them.  WL: columns w a lane holds in the sign part (W <= 64 * WL).  With g = the gradient of
// the score: sum g * sign = 2 * sum g * h - sum g.  Grid as in the forward; px, py: NULL, or [splits][rows][W], [splits][rows][Wv].
template <typename ST, bool OWNK, bool CAP, int WL, int NB, int TB, int THREADS>
__global__ void __launch_bounds__(THREADS) masked_bwd(L1MaskedArgs A, const ST* __restrict__ q, const ST* __restrict__ k,
                                                      const ST* __restrict__ v, const ST* __restrict__ dout,
                                                      const float* __restrict__ lse, const float* __restrict__ D,
                                                      ST* __restrict__ dx, ST* __restrict__ dy, float* __restrict__ px, float* __restrict__ py)
{
	extern __shared__ __align__(16) char lds[];
	const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = threads >> 6;
	const int i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
	constexpr int KN = k16<ST> && NB == 8 ? 4 : 2, VN = k16<ST> && NB < 8 ? 1 : 2;
	const int group = A.H / A.Hk, heads = OWNK ? A.Hk : A.H;
	Block K;
	K.b = blockIdx.x / heads;
	K.h = blockIdx.x % heads;
	K.hk = OWNK ? K.h : K.h / group;
	K.nown = waves * kOwn;
	// the workgroups with the most to do under causality come first: late queries, early keys
	K.own0 = (OWNK ? blockIdx.y : gridDim.y - 1 - blockIdx.y) * K.nown;
	K.own_rows = OWNK ? A.S : A.T;
	K.str_rows = OWNK ? A.T : A.S;
	K.own_place0 = OWNK ? 0 : A.S - A.T;
	K.str_place0 = OWNK ? A.S - A.T : 0;
	const int row0 = K.own0 + wave * kOwn;
	const Layout Y = masked_layout<ST, TB>(A.W, A.Wv, waves, true, OWNK);
	char *own = lds + Y.own + wave * kOwn * Y.so, *str = lds + Y.str, *raw = lds + Y.raw, *y = lds + Y.y, *yt = lds + Y.yt;
	char* scr = lds + Y.scratch + wave * kScratch;
	float* sc = reinterpret_cast<float*>(scr);
	int* docs = reinterpret_cast<int*>(lds + Y.rows);
	float *slse = reinterpret_cast<float*>(docs) + kTile<TB>, *sD = slse + kTile<TB>, *over = sD + kTile<TB>, *red = over + kTile<TB>;
	unsigned char* cls = reinterpret_cast<unsigned char*>(red + 64);
	const int* doc = A.doc ? A.doc + (int64_t)K.b * A.S : nullptr;
	const int prefix = A.prefix ? A.prefix[K.b] : 0;
	const int64_t qpitch = (int64_t)A.H * A.W, kpitch = (int64_t)A.Hk * A.W;
	const int64_t opitch = (int64_t)A.H * A.Wv, vpitch = (int64_t)A.Hk * A.Wv;
	const ST* kh = k + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.W;
	const ST* vh = v + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.Wv;
	const ST* own_x = OWNK ? kh : q + ((int64_t)K.b * A.T * A.H + K.h) * A.W;
	const int64_t own_pitch = OWNK ? kpitch : qpitch, str_pitch = OWNK ? qpitch : kpitch;
	const bool own_vec = A.vec & (OWNK ? 2 : 1), str_vec = A.vec & (OWNK ? 1 : 2);

	int* tiny = reinterpret_cast<int*>(over);  // float32 has no other use of this: whether the workgroup has met tiny values
	if (!k16<ST> && tid == 0) *tiny = 0;
	Span mine, all;
	bool mine_whole, all_whole;
	owner_docs(doc, K, row0, reinterpret_cast<int*>(red), lane, wave, waves, mine, mine_whole, all, all_whole);
	Grid G = {0.f, 0.f, 0.f};
	bool coded = false;
	if constexpr (k16<ST>) {
		coded = owner_grid(own_x, doc, K, row0, own_pitch, A.W, own_vec, red + 32, lane, wave, waves, G);
		stage_own16(own, lds + Y.oraw + wave * kOwn * Y.sr, own_x, row0, K.own_rows, own_pitch, A.W, Y.so, Y.sr, G, own_vec, lane);
	} else {
		if (stage32(own, own_x, row0, kOwn, K.own_rows, own_pitch, 0, A.W, Y.so, own_vec, lane, 64)) *tiny = 1;
	}
	const int own_lo = K.own_place0 + K.own0, own_hi = K.own_place0 + min(K.own0 + K.nown, K.own_rows) - 1;
	const int my_lo = K.own_place0 + row0, my_hi = K.own_place0 + min(row0 + kOwn, K.own_rows) - 1;
	float sum[WL][32];
#pragma unroll
	for (int u = 0; u < WL; u++)
#pragma unroll
		for (int r = 0; r < 32; r++) sum[u][r] = 0.f;
	int od4[4];
#pragma unroll
	for (int a = 0; a < 4; a++) od4[a] = doc && row0 + i + 8 * a < K.own_rows ? doc[my_lo + i + 8 * a] : -1;
	float gsum[4] = {0.f, 0.f, 0.f, 0.f};
	constexpr int NY = OWNK ? NB : 1;
	f4 dyv[2][NY];
#pragma unroll
	for (int tb = 0; tb < 2; tb++)
#pragma unroll
		for (int wb = 0; wb < NY; wb++) dyv[tb][wb] = (f4)(0.f);
	constexpr int NX = k16<ST> ? (NB + 1) / 2 : NB;  // 16 bytes of a lane each: 32 columns of 16 bits, 16 of float32
	const int xstep = k16<ST> ? 32 : 16, xlane = k16<ST> ? 8 * g : 4 * g;

	for (int hg = 0; hg < (OWNK ? group : 1); hg++) {
		const int h = OWNK ? K.hk * group + hg : K.h;
		const float slope = A.has_slopes ? fminf(A.slopes[h] * kUnit<ST>, kMax) : 0.f;
		const ST* qh = q + ((int64_t)K.b * A.T * A.H + h) * A.W;
		const ST* oh = dout + ((int64_t)K.b * A.T * A.H + h) * A.Wv;
		const ST* str_x = OWNK ? qh : kh;
		// the owners' rows of the second product (v of the keys, do of the queries), as its right operand
		uint4 xr[2][NX];
#pragma unroll
		for (int ob = 0; ob < 2; ob++) {
			const int r = row0 + 16 * ob + l16;
			const ST* row = OWNK ? vh + (int64_t)r * vpitch : oh + (int64_t)r * opitch;
#pragma unroll
			for (int kc = 0; kc < NX; kc++) {
				const int w = xstep * kc + xlane;
				xr[ob][kc] = make_uint4(0, 0, 0, 0);
				if (r < K.own_rows && w < A.Wv) xr[ob][kc] = load_raw(row + w, A.Wv - w, OWNK ? A.vec & 4 : A.vec & 8);
			}
		}
		float olse[4], oD[4];
#pragma unroll
		for (int a = 0; a < 4; a++) {
			const int t = row0 + i + 8 * a;
			const bool in = !OWNK && t < A.T;
			olse[a] = in ? lse[((int64_t)K.b * A.T + t) * A.H + h] * kUnit<ST> : 0.f;
			oD[a] = in ? D[((int64_t)K.b * A.T + t) * A.H + h] : 0.f;
		}
		int first = 0, last = (K.str_rows + kTile<TB> - 1) / kTile<TB>;
		if (A.causal) {
			if (OWNK) { if (own_lo >= prefix) first = max(0, own_lo - K.str_place0) / kTile<TB>; }
			else last = (min(A.S, max(own_hi + 1, prefix)) + kTile<TB> - 1) / kTile<TB>;
		}
		const int step = gridDim.z;
		for (int t0 = first + blockIdx.z; t0 < last; t0 += step * kClasses) {
			const int n = min(kClasses, (last - t0 + step - 1) / step);
			__syncthreads();
			classify<OWNK, TB>(A, K, doc, prefix, own_lo, own_hi, all, all_whole, t0, step, n, cls, tid, threads);
			__syncthreads();
			Stream<ST, TB, KN, VN> F;
			const ST* str_y = OWNK ? oh : vh;
			const int64_t y_pitch = OWNK ? opitch : vpitch;
			const bool y_vec = A.vec & (OWNK ? 8 : 4);
			const int* str_doc = doc ? doc + K.str_place0 : nullptr;
			const float *lh = OWNK ? lse + (int64_t)K.b * A.T * A.H + h : nullptr, *Dh = OWNK ? D + (int64_t)K.b * A.T * A.H + h : nullptr;
			int next = next_tile(cls, 0, n);
			if (next < n) F.fetch(str_x, str_pitch, A.W, str_vec, str_y, y_pitch, A.Wv, y_vec, (t0 + step * next) * kTile<TB>, K.str_rows, str_doc, lh, Dh, A.H, tid, threads);
			while (next < n) {
				const int kind = __builtin_amdgcn_readfirstlane(cls[next]), s0 = (t0 + step * next) * kTile<TB>;
				const int tid = here(threadIdx.x), lane = tid & 63, i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
				__syncthreads();
				// without a grid the codes come out as nonsense that nobody reads; the ordered integers are wanted all the same
				bool bad = F.place(str, raw, over, y, k16<ST> && OWNK ? yt : nullptr, docs, OWNK ? slse : nullptr, sD, k16<ST> ? nullptr : tiny, Y, G, str_x, str_pitch, A.W, str_vec,
				                   str_y, y_pitch, A.Wv, y_vec, s0, K.str_rows, tid, threads);
				next = next_tile(cls, next + 1, n);
				if (next < n) F.fetch(str_x, str_pitch, A.W, str_vec, str_y, y_pitch, A.Wv, y_vec, (t0 + step * next) * kTile<TB>, K.str_rows, str_doc, lh, Dh, A.H, tid, threads);
				const int far = __syncthreads_or(bad && (k16<ST> || kind == 2)) ? kind : 0;
				const bool exact = !k16<ST> && __builtin_amdgcn_readfirstlane(*tiny);
				int mykind = row0 < K.own_rows ? kind : 0;
				if (mykind == 2) {
					mykind = place_class<OWNK>(A, prefix, my_lo, my_hi, K.str_place0 + s0, K.str_place0 + min(s0 + kTile<TB>, K.str_rows) - 1, s0 + kTile<TB> <= K.str_rows);
					if (mykind && doc) mykind = doc_class<TB>(mykind, docs[lane % kTile<TB>], mine, mine_whole, lane);
				}
				mykind = __builtin_amdgcn_readfirstlane(mykind);  // what the tile is to this wave's own rows
				float x[4][TB];
				tile_distances<ST, true, WL == 2, TB>(own, str, over, Y, A.W, CAP ? A.rw : A.rw * kUnit<ST>, G, coded, mykind, own_x, row0, K.own_rows, own_pitch, str_x, s0, K.str_rows, str_pitch, i, j, tid, threads, x);
				if (!mykind) continue;
#pragma unroll
				for (int half = 0; half < TB / 4; half++) {
					const int lane = here(tid & 63), i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
					float p[4][4], pf[4][4];  // weights, and the derivative of their argument by the distance's sum
					scores<ST, CAP, TB>(p, pf, x, half, A.cap, A.icap);
#pragma unroll
					for (int bb = 0; bb < 4; bb++) {
						const int b = 4 * half + bb, r = j + 8 * b;
						const float sl = OWNK ? slse[r] : 0.f;
#pragma unroll
						for (int a = 0; a < 4; a++) {
							p[a][bb] -= OWNK ? sl : olse[a];
							pf[a][bb] *= A.rw;
						}
					}
					if (slope != 0.f) {
						asm volatile("");  // a branch
#pragma unroll
						for (int bb = 0; bb < 4; bb++) {
							const float s = (float)(K.str_place0 + s0 + j + 8 * (4 * half + bb) - my_lo - i);
#pragma unroll
							for (int a = 0; a < 4; a++) p[a][bb] = __builtin_fmaf(-slope, __builtin_fabsf(s - 8.f * a), p[a][bb]);
						}
					}
#pragma unroll
					for (int bb = 0; bb < 4; bb++)
#pragma unroll
						for (int a = 0; a < 4; a++) p[a][bb] = weight<ST>(p[a][bb]);
					if (mykind == 2) {
						asm volatile("");  // a branch, as in the forward
#pragma unroll
						for (int bb = 0; bb < 4; bb++) {
							const int r = j + 8 * (4 * half + bb), sp = K.str_place0 + s0 + r, sd = docs[r];
#pragma unroll
							for (int a = 0; a < 4; a++) {
								const int place = my_lo + i + 8 * a;
								const bool ok = OWNK ? sees(!A.causal, prefix, !doc, sp, place, sd, od4[a]) : sees(!A.causal, prefix, !doc, place, sp, od4[a], sd);
								p[a][bb] = (s0 + r < K.str_rows) & ok ? p[a][bb] : 0.f;
							}
						}
					}
					if constexpr (OWNK) weigh<ST, NY, TB>(dyv, scr, y, yt, Y.sy, A.Wv, p, half, i, j, l16, g, far);
					// dp of this half's 32 columns
					f4 dp[2][2];
#pragma unroll
					for (int cb = 0; cb < 2; cb++) {
						dp[cb][0] = (f4)(0.f);
						dp[cb][1] = (f4)(0.f);
#pragma unroll
						for (int kc = 0; kc < NX; kc++) {
							const int w = xstep * kc + xlane;
							if (xstep * kc >= A.Wv) break;
							const uint4 ya = *reinterpret_cast<const uint4*>(y + (32 * half + 16 * cb + l16) * Y.sy + w * (int)sizeof(ST));
							if constexpr (k16<ST>) {
#pragma unroll
								for (int ob = 0; ob < 2; ob++) dp[cb][ob] = mma16<ST>(ya, xr[ob][kc], dp[cb][ob]);
							} else {
								const f4 yf = w * 4 < Y.sy ? __builtin_bit_cast(f4, ya) : (f4)(0.f);
#pragma unroll
								for (int e = 0; e < 4; e++)
#pragma unroll
									for (int ob = 0; ob < 2; ob++) dp[cb][ob] = __builtin_amdgcn_mfma_f32_16x16x4f32(yf[e], __builtin_bit_cast(f4, xr[ob][kc])[e], dp[cb][ob], 0, 0, 0);
							}
						}
					}
					wave_sync();
#pragma unroll
					for (int cb = 0; cb < 2; cb++)
#pragma unroll
						for (int ob = 0; ob < 2; ob++) *reinterpret_cast<f4*>(sc + (l16 + 16 * ob) * kPad + 16 * cb + 4 * g) = dp[cb][ob];
					wave_sync();
					f4 d4[4];
#pragma unroll
					for (int a = 0; a < 4; a++) d4[a] = *reinterpret_cast<const f4*>(sc + (i + 8 * a) * kPad + 4 * j);
					wave_sync();
#pragma unroll
					for (int bb = 0; bb < 4; bb++) {
						const int b = 4 * half + bb;
						const float dD = OWNK ? sD[j + 8 * b] : 0.f;
						f4 gr;
#pragma unroll
						for (int a = 0; a < 4; a++) {
							// a hidden pair's dp may come from values that are not finite
							gr[a] = p[a][bb] != 0.f ? p[a][bb] * pf[a][bb] * ((OWNK ? dD : oD[a]) - d4[a][bb]) : 0.f;
							gsum[a] += gr[a];
						}
						*reinterpret_cast<f4*>(sc + (4 * j + bb) * kPad + 4 * i) = gr;
					}
					wave_sync();
					float ov[WL][32];  // the owners' columns: register r = 4 i' + a' is row i' + 8 a'
#pragma unroll
					for (int u = 0; u < WL; u++)
#pragma unroll
						for (int r = 0; r < 32; r++) {
							const int row = (r >> 2) + 8 * (r & 3);
							const int w = min(lane + 64 * u, A.W - 1);  // columns behind the width are worked on and not written
							if constexpr (k16<ST>) ov[u][r] = (float)*reinterpret_cast<const short*>(lds + Y.oraw + (wave * kOwn + row) * Y.sr + 2 * w) + 0.5f;
							else ov[u][r] = *reinterpret_cast<const float*>(own + row * Y.so + 4 * w);
						}
					if constexpr (k16<ST>) {
						signs<ST, WL>(sum, ov, sc, raw, Y.sr, half, lane, A.W, false);
					} else {
						// half a tile's sum on its own, then to the total: the roundings of either are fewer
						float part[WL][32];
#pragma unroll
						for (int u = 0; u < WL; u++)
#pragma unroll
							for (int r = 0; r < 32; r++) part[u][r] = 0.f;
						signs<ST, WL>(part, ov, sc, str, Y.so, half, lane, A.W, exact);
#pragma unroll
						for (int u = 0; u < WL; u++)
#pragma unroll
							for (int r = 0; r < 32; r++) sum[u][r] += part[u][r];
					}
					wave_sync();
				}
			}
		}
	}
#pragma unroll
	for (int a = 0; a < 4; a++) {
		gsum[a] += __shfl_xor(gsum[a], 8);
		gsum[a] += __shfl_xor(gsum[a], 16);
		gsum[a] += __shfl_xor(gsum[a], 32);
	}
	wave_sync();
	if (j == 0)
#pragma unroll
		for (int a = 0; a < 4; a++) sc[4 * i + a] = gsum[a];
	wave_sync();
	const int64_t rows = (int64_t)A.B * K.own_rows * heads;
#pragma unroll
	for (int r = 0; r < 32; r++) {
		const int t = row0 + (r >> 2) + 8 * (r & 3);
		const float gs = sc[r];
		if (t >= K.own_rows) continue;
		const int64_t row = ((int64_t)K.b * K.own_rows + t) * heads + K.h;
#pragma unroll
		for (int u = 0; u < WL; u++)
			if (lane + 64 * u < A.W) {
				const float y1 = 2.f * sum[u][r] - gs;
				if (px) px[(blockIdx.z * rows + row) * A.W + lane + 64 * u] = y1;
				else dx[row * A.W + lane + 64 * u] = (ST)y1;
			}
	}
	if constexpr (OWNK) {
#pragma unroll
		for (int tb = 0; tb < 2; tb++) {
			const int s = row0 + 16 * tb + l16;
			if (s >= A.S) continue;
			const int64_t row = ((int64_t)K.b * A.S + s) * A.Hk + K.hk;
#pragma unroll
			for (int wb = 0; wb < NY; wb++)
#pragma unroll
				for (int e = 0; e < 4; e++) {
					const int w = 16 * wb + 4 * g + e;
					if (w >= A.Wv) continue;
					const float y1 = dyv[tb][wb][e];
					if (py) py[(blockIdx.z * rows + row) * A.Wv + w] = y1;
					else dy[row * A.Wv + w] = (ST)y1;
				}
		}
	}
}

// ------------------------------------------------------------------------------------------------------------------- host

template <typename F>
int launch(F* f, dim3 grid, int waves, int bytes, hipStream_t st, void** args)
{
	L1_HIP_CHECK(hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
	L1_HIP_CHECK(hipLaunchKernel((const void*)f, grid, dim3(64 * waves), args, bytes, st));
	return L1ATTN_OK;
}

template <typename ST>
struct MaskedImpl {
	static constexpr int TF = k16<ST> ? 8 : 4, TBW = 4;  // tiles of the forward and of the backward

	template <bool CAP>
	static int fwd_cap(L1MaskedArgs& A, const L1MaskedPlan& P, const void* q, const void* k, const void* v, void* o, float* lse, float* part, hipStream_t st)
	{
		const dim3 grid((unsigned)(A.B * A.H), (unsigned)l1_cdiv(A.T, kOwn * P.waves), (unsigned)P.splits);
		const int bytes = masked_layout<ST, TF>(A.W, A.Wv, P.waves, false, true).total;
		void* args[] = {&A, &q, &k, &v, &o, &lse, &part};
		if (A.Wv > 64) return launch(masked_fwd<ST, CAP, 8, TF, 256>, grid, P.waves, bytes, st, args);
		return launch(masked_fwd<ST, CAP, 4, TF, 512>, grid, P.waves, bytes, st, args);
	}
	static int fwd(L1MaskedArgs& A, const L1MaskedPlan& P, const void* q, const void* k, const void* v, void* o, float* lse, float* part, hipStream_t st)
	{
		const int rc = A.cap > 0.f ? fwd_cap<true>(A, P, q, k, v, o, lse, part, st) : fwd_cap<false>(A, P, q, k, v, o, lse, part, st);
		if (rc != L1ATTN_OK || !part) return rc;
		const int64_t rows = (int64_t)A.B * A.T * A.H;
		hipLaunchKernelGGL(masked_fwd_join<ST>, dim3((unsigned)l1_cdiv(rows, 4)), dim3(256), 0, st, part, P.splits, rows, A.Wv, (ST*)o, (ST*)A.rest, lse);
		L1_LAUNCH_CHECK();
		return L1ATTN_OK;
	}
	static int rows(const void* dout, const void* o, const void* rest, float* D, int64_t rows, int Wv, hipStream_t st)
	{
		const int64_t blocks = l1_cdiv(rows, 32), most = 1 << 23;  // a grid has 2^32 - 1 threads at most
		hipLaunchKernelGGL(masked_bwd_rows<ST>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, (const ST*)dout, (const ST*)o, (const ST*)rest, D, rows, Wv);
		L1_LAUNCH_CHECK();
		return L1ATTN_OK;
	}
	template <bool OWNK, bool CAP>
	static int side_cap(L1MaskedArgs& A, const L1MaskedPlan& P, const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* D,
	                    void* dx, void* dy, float* px, float* py, hipStream_t st)
	{
		const int64_t heads = (int64_t)A.B * (OWNK ? A.Hk : A.H), n = OWNK ? A.S : A.T;
		const dim3 grid((unsigned)heads, (unsigned)l1_cdiv(n, kOwn * P.waves), (unsigned)P.splits);
		const int bytes = masked_layout<ST, TBW>(A.W, A.Wv, P.waves, true, OWNK).total;
		void* args[] = {&A, &q, &k, &v, &dout, &lse, &D, &dx, &dy, &px, &py};
		if (A.W > 64) return launch(masked_bwd<ST, OWNK, CAP, 2, 8, TBW, 256>, grid, P.waves, bytes, st, args);
		if (A.Wv > 64) return launch(masked_bwd<ST, OWNK, CAP, 1, 8, TBW, 256>, grid, P.waves, bytes, st, args);
		return launch(masked_bwd<ST, OWNK, CAP, 1, 4, TBW, 512>, grid, P.waves, bytes, st, args);
	}
	template <bool OWNK>
	static int side(L1MaskedArgs& A, const L1MaskedPlan& P, const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* D,
	                void* dx, void* dy, float* part, hipStream_t st)
	{
		const int64_t nx = (int64_t)A.B * (OWNK ? (int64_t)A.S * A.Hk : (int64_t)A.T * A.H) * A.W, ny = OWNK ? nx / A.W * A.Wv : 0;
		float *px = P.splits > 1 ? part : nullptr, *py = P.splits > 1 && OWNK ? part + P.splits * nx : nullptr;
		const int rc = A.cap > 0.f ? side_cap<OWNK, true>(A, P, q, k, v, dout, lse, D, dx, dy, px, py, st)
		                           : side_cap<OWNK, false>(A, P, q, k, v, dout, lse, D, dx, dy, px, py, st);
		if (rc != L1ATTN_OK || !px) return rc;
		hipLaunchKernelGGL(masked_bwd_join<ST>, dim3((unsigned)l1_cdiv(nx, 256)), dim3(256), 0, st, px, P.splits, nx, (ST*)dx);
		L1_LAUNCH_CHECK();
		if (OWNK) {
			hipLaunchKernelGGL(masked_bwd_join<ST>, dim3((unsigned)l1_cdiv(ny, 256)), dim3(256), 0, st, py, P.splits, ny, (ST*)dy);
			L1_LAUNCH_CHECK();
		}
		return L1ATTN_OK;
	}
	static int side_q(L1MaskedArgs& A, const L1MaskedPlan& P, const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* D,
	                  void* dq, float* part, hipStream_t st)
	{
		return side<false>(A, P, q, k, v, dout, lse, D, dq, nullptr, part, st);
	}
	static int side_k(L1MaskedArgs& A, const L1MaskedPlan& P, const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* D,
	                  void* dk, void* dv, float* part, hipStream_t st)
	{
		return side<true>(A, P, q, k, v, dout, lse, D, dk, dv, part, st);
	}
	static int lds(int W, int Wv, int waves, bool backward, bool weigh)
	{
		return backward ? masked_layout<ST, TBW>(W, Wv, waves, true, weigh).total : masked_layout<ST, TF>(W, Wv, waves, false, weigh).total;
	}
};

}  // namespace

#define L1_MASKED_TABLE(name, ST)                                                                                                      \
	const L1MaskedTable& name()                                                                                                        \
	{                                                                                                                                  \
		static const L1MaskedTable t = {MaskedImpl<ST>::fwd, MaskedImpl<ST>::rows, MaskedImpl<ST>::side_q, MaskedImpl<ST>::side_k, MaskedImpl<ST>::lds}; \
		return t;                                                                                                                      \
	}
