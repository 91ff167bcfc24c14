// L1 attention of each sequence's last tokens over its pages of the 8-bit cache.
//
//   x[r,s] = c(-1/sqrt(W) * sum_w |q[r,w] - code[s,w] * scale[page of s]|) - slope * (place of r - s),   s <= place of r
//   o[r]   = sum_s exp(x) * v[s] / (1 + sum_s exp(x))
//
// The rows r of a workgroup are the query tokens and query heads that read one key head.  Every logit is <= 0 and the no-op
// logit is 0, so partial sums over pieces of a sequence simply add up: no running maximum, and the pieces join in a fixed
// order.  Every byte of the cache is read once for up to 16 rows.
// Distances.  Up to 4 rows, and float32: float32, two instructions an element and row.  From 5 rows of 16 bits on: sums of
// |difference| of 16-bit codes (v_sad_u16, two elements an instruction) on one grid over the rows' values and over what the
// scales of the workgroup's pages allow (128 times the largest); what that does to a logit: codes.h.  Past the range that is
// allowed there, or where a row or scale is not finite, float32.
// Sums.  For 16-bit rows weight times scale is two bfloat16 numbers, itself rounded and what that leaves out (2^-18 of it at most; one
// number alone made results 1.6 times as inexact as their own rounding), a code is exact in bfloat16, and matrix instructions add
// them in float32.  Not float16 for float16 rows: it would want a power of two over all tokens of a step, where one token's large
// scale takes the digits of the others' weights, also in rows that do not see it.  float32 has its own matrix instruction.
// What bounds it: for few rows latency and the reads (32 sequences of about 2050 tokens, 4 rows, W 64, bfloat16: 34 MB in 18 us, and 4
// for the join), for many the vector ALU (16 of about 20480, 16 rows, W 128, float16: 142 us at 2.4 TB/s; 2048 of a step's 4200
// vector instructions are v_sad_u16, which issue in about 4.2 cycles each; the rest makes codes and bfloat16 of the cache's bytes,
// and weights).  With one token a lane instead of two at 16 rows a row's codes would be read from LDS twice as often.  Widths
// of 64 and 128, the same for keys and values, have loops of their own (FULL); all others run the one for up to 128, which for
// values of 64 columns or fewer loads and multiplies columns twice.
// How the steps are dealt out, and so the order of a sequence's sums and the grid of its codes, goes by the lengths of the whole
// batch: the same call gives the same bits, a sequence in another batch may round differently.
#include "paged.h"
#include "softcap.h"
#include "codes.h"
#include <math.h>
#include <type_traits>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

struct AttendArgs {
	L1Cache C;
	int B, n, H, G, slots, step;
	float cap, icap, rw;
	float slopes[256];
};

// length of entry b's sequence, 0 where it names none
__device__ __forceinline__ int seq_of(const AttendArgs& A, const int32_t* seqs, int b, int& s)
{
	s = seqs ? seqs[b] : b;
	if (s < 0 || s >= A.C.rows || A.C.N < 1) return 0;
	return min(max(A.C.lens[s], 0), A.C.M * A.C.P);
}

// How the tokens of all entries are dealt out to A.slots workgroups of each key head and block of rows.  An entry's tokens are whole steps; each workgroup takes up to `per` of them, of one entry, with per =
// ceil(steps of all entries / (slots - entries)): the sum of ceil(steps / per) is then at most `slots`.  So a batch of uneven
// lengths ends everywhere at about the same time.  Found by a sum and a scan over the entries' lengths in every workgroup
// (256 threads; at most 512 entries).  Whose is `slot`?  `spans`, if not NULL, takes each entry's first slot and how many it has.
struct Share {
	int entry, first, per;  // -1 for nobody; first slot of the entry; tokens of a slot
};
__device__ __forceinline__ Share share_of(const AttendArgs& A, const int32_t* seqs, int slot, int* lds, int2* spans)
{
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	int steps[2];
#pragma unroll
	for (int i = 0; i < 2; i++) {
		int s;
		const int b = 2 * tid + i;
		steps[i] = b < A.B ? (seq_of(A, seqs, b, s) + A.step - 1) / A.step : 0;
	}
	unsigned total = steps[0] + steps[1];
#pragma unroll
	for (int m = 32; m; m >>= 1) total += __shfl_xor(total, m);
	if (lane == 0) lds[wave] = total;
	if (tid == 0) lds[8] = -1;
	__syncthreads();
	total = (unsigned)lds[0] + lds[1] + lds[2] + lds[3];
	const unsigned room = A.slots - A.B;
	const int per = max((int)(total / room + (total % room != 0)), 1);
	const int n0 = (steps[0] + per - 1) / per, n1 = (steps[1] + per - 1) / per;
	int before = n0 + n1;  // a scan over the threads
#pragma unroll
	for (int m = 1; m < 64; m <<= 1) {
		const int y = __shfl_up(before, m);
		before += lane >= m ? y : 0;
	}
	if (lane == 63) lds[4 + wave] = before;
	__syncthreads();
	before -= n0 + n1;
	for (int w = 0; w < wave; w++) before += lds[4 + w];
#pragma unroll
	for (int i = 0; i < 2; i++) {
		const int b = 2 * tid + i, first = i ? before + n0 : before, n = i ? n1 : n0;
		if (slot >= first && slot < first + n) { lds[8] = b; lds[9] = first; }
		if (spans && b < A.B) spans[b] = make_int2(first, n);
	}
	__syncthreads();
	const Share S = {__builtin_amdgcn_readfirstlane(lds[8]), __builtin_amdgcn_readfirstlane(lds[9]), __builtin_amdgcn_readfirstlane(per * A.step)};
	return S;
}

// One 16-byte piece of codes as float32.
__device__ __forceinline__ void codes4(int word, float (&x)[4])
{
	x[0] = (float)(int8_t)word;
	x[1] = (float)(int8_t)(word >> 8);
	x[2] = (float)(int8_t)(word >> 16);
	x[3] = (float)(word >> 24);
}

// exp(a)
template <typename ST> __device__ __forceinline__ float exponential(float a)
{
	if constexpr (sizeof(ST) == 4) return expf(a);
	return __builtin_amdgcn_exp2f(1.442695041f * a);
}

// page * stride bytes behind a pool's base
template <typename T> __device__ __forceinline__ const T* page_at(const T* base, int page, unsigned stride)
{
	return reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + (uint64_t)(uint32_t)page * stride);
}

// RB rows of a workgroup.  Grid: slots * key heads, blocks of rows.  part: [slots][n][H][Wv + 1] (the last: the weights' sum); if
// NULL, a slot is an entry, and the workgroup writes o itself.
// Each of the four waves takes 64 U tokens of its own at a time and waits for no other: a lane holds U tokens against all rows,
// whose values are broadcast LDS reads; the weights pass through the wave's own piece of LDS into the layout of the matrix
// instructions, which add up weight * value.  A step's loads are on their way together: the next step's pages, keys, values.
template <typename ST, int RB, int NC, bool FULL, int MINW>
__global__ void __launch_bounds__(256, MINW) paged_attend(AttendArgs A, const ST* __restrict__ q, const int32_t* __restrict__ seqs,
                                                          const int32_t* __restrict__ counts, ST* __restrict__ o, float* __restrict__ part, int2* __restrict__ spans)
{
	constexpr bool F32 = sizeof(ST) == 4, CODED = !F32 && RB >= 8;
	constexpr bool LATE = RB >= 8;  // values are asked for behind the distances: registers hold the rows' codes read ahead (183 -> 164 us)
	constexpr int U = RB <= 4 ? 1 : 2, VG = NC / 4, KB = RB >= 8 ? 2 : 4;  // KB: pieces of 16 bytes of a key row under way
	constexpr int pitch = 64 * U + (F32 ? 4 : 8);                          // between two rows' weights: an odd number of 16-byte pieces
	using PT = std::conditional_t<F32, float, __bf16>;                      // of the weights
	constexpr int TR = 256 / RB;  // threads of a row before and behind the loop
	constexpr int plane = F32 ? 0 : RB * pitch;  // 16-bit weights: what their rounding leaves out lies behind them
	constexpr int pool = 4 * (RB * pitch + plane) * (int)sizeof(PT), join = 2 * RB * 128 * 4;
	__shared__ __align__(16) float qs[RB * 128];
	__shared__ __align__(16) unsigned qc[CODED ? RB * 64 : 1];
	__shared__ __align__(16) char shared_pool[pool > join ? pool : join];
	__shared__ float red[8], dens[4 * RB];
	const L1Cache& C = A.C;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
	const int slot = blockIdx.x / C.Hk, hk = blockIdx.x % C.Hk, r0 = blockIdx.y * RB, R = A.n * A.G;
	int b = slot, lo = 0, per = 0x40000000;
	if (part) {
		__shared__ int lds[10];
		const Share S = share_of(A, seqs, slot, lds, blockIdx.x + blockIdx.y ? nullptr : spans);
		if (S.entry < 0) return;
		b = S.entry;
		lo = (slot - S.first) * S.per;
		per = S.per;
	}
	int s;
	const int len = seq_of(A, seqs, b, s), hi = min(lo + per, len);
	const int cnt = counts ? min(max(counts[b], 0), A.n) : A.n;
	const int32_t* table = C.table + (int64_t)s * C.M;
	const int psh = C.P == 16 ? 4 : C.P == 32 ? 5 : 6;  // a page's tokens are 16, 32 or 64
	const int pk = FULL ? 16 * NC : C.pk, pv = FULL ? 16 * NC : C.pv;
	int after[U];  // page of the lane's tokens in the step behind the coming one
	const int first = lo + 64 * U * wave;
	auto page_of = [&](int t) { return t < hi ? table[t >> psh] : -1; };
	int page[U];
#pragma unroll
	for (int u = 0; u < U; u++) {
		page[u] = page_of(first + 64 * u + lane);
		after[u] = page_of(first + 64 * u + lane + 256 * U);
	}
	// the rows' values, zero behind the width: the cache's rows are zero there as well
	const int my = tid / TR, my0 = tid % TR, myt = (r0 + my) / A.G;
	const int64_t myrow = r0 + my < R ? ((int64_t)b * A.n + myt) * A.H + hk * A.G + (r0 + my - myt * A.G) : -1;
	float least = 0.f, most = 0.f;
	bool finite = true;
	for (int w = my0; w < pk; w += TR) {
		const float y = myrow >= 0 && w < C.W ? (float)q[myrow * C.W + w] : 0.f;
		qs[my * 128 + w] = y;
		finite &= __builtin_fabsf(y) <= 3.402823466e38f;
		least = fminf(least, y);
		most = fmaxf(most, y);
	}
	// what a row sees, -1 for nothing, and its slope
	int place[RB];
	float slope[RB];
	int rt = r0 / A.G, rx = r0 - rt * A.G;
#pragma unroll
	for (int r = 0; r < RB; r++) {
		place[r] = __builtin_amdgcn_readfirstlane(r0 + r < R && rt < cnt ? len - cnt + rt : -1);
		slope[r] = A.slopes[hk * A.G + rx];
		if (++rx == A.G) { rx = 0; rt++; }
	}
	bool coded = false;
	float sc = 0.f, off = 0.f, m = A.rw;
	if constexpr (CODED) {
		// the grid: over the rows' values and over what the pages' scales allow
		float kmax = 0.f;
		for (int j = (lo >> psh) + tid; j << psh < hi; j += 256) {
			const int pg = table[j];
			if (pg < 0 || pg >= C.N) continue;
			const float y = C.ks[(int64_t)pg * C.Hk + hk];
			finite &= __builtin_fabsf(y) <= 3.402823466e38f;
			kmax = fmaxf(kmax, __builtin_fabsf(y));
		}
		least = fminf(least, -128.f * kmax);
		most = fmaxf(most, 128.f * kmax);  // a negative scale as well, and the code -128: from a pool that the caller filled
#pragma unroll
		for (int k = 32; k; k >>= 1) {
			least = fminf(least, __shfl_xor(least, k));
			most = fmaxf(most, __shfl_xor(most, k));
		}
		if (lane == 0) { red[2 * wave] = least; red[2 * wave + 1] = most; }
		finite = !__syncthreads_or(!finite);
#pragma unroll
		for (int w = 0; w < 4; w++) { least = fminf(least, red[2 * w]); most = fmaxf(most, red[2 * w + 1]); }
		const float span = (most - least) * (1.f + 0x1p-19f);
		coded = finite && span > 1e-30f && span <= kCodeRange<ST>;
		const float step = span * (1.f / kCodeSteps);
		sc = coded ? 1.f / (step * 65535.f) : 0.f;
		off = coded ? -(least - (most - least) * 0x1p-20f) * sc : 0.f;
		if (coded) {
			m = step * A.rw;
			for (int w = my0; w < pk / 2; w += TR) {
				const float b = off + l1_code_eight(w >> 2), b0 = b + l1_code_column(2 * (w & 3)), b1 = b + l1_code_column(2 * (w & 3) + 1);
				qc[my * 64 + w] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(__builtin_fmaf(qs[my * 128 + 2 * w], sc, b0),
				                                                                             __builtin_fmaf(qs[my * 128 + 2 * w + 1], sc, b1)));
			}
		}
	}
	__syncthreads();
	PT* ps = reinterpret_cast<PT*>(shared_pool) + wave * (RB * pitch + plane);
	const int kchunks = FULL ? NC : pk / 16;
	float den[RB];
	f4 acc[VG][4];
#pragma unroll
	for (int r = 0; r < RB; r++) den[r] = 0.f;
#pragma unroll
	for (int wg = 0; wg < VG; wg++)
#pragma unroll
		for (int e = 0; e < 4; e++) acc[wg][e] = (f4)(0.f);
	const int kend = (kchunks + KB - 1) / KB * KB;
	float ks[U], vs[U];
	int pg[U];
	const int8_t* krow[U];
	uint4 kr[U][KB];
	// A step begins at a multiple of 64, so a lane's place in its page is always the same.
	const unsigned kstride = (unsigned)C.Hk * C.P * pk, vstride = (unsigned)C.Hk * C.P * pv;
	const int8_t *kbase = C.k + (int64_t)hk * C.P * pk, *vbase = C.v + (int64_t)hk * C.P * pv;
	const int kin = (lane & (C.P - 1)) * pk;
	// where tokens are: no page, page 0 and scales 0 if nowhere
	auto locate = [&](int at, int& to, const int8_t*& row, float& a, float& c) {
		const bool there = at >= 0 && at < C.N;
		to = there ? at : -1;
		const int p0 = there ? at : 0;
		row = page_at(kbase, p0, kstride) + kin;
		const float x = *page_at(C.ks + hk, p0, 4u * C.Hk), y = *page_at(C.vs + hk, p0, 4u * C.Hk);
		a = there ? x : 0.f;
		c = there ? y : 0.f;
	};
	if (first < hi)  // else the pool may have no page
#pragma unroll
	for (int u = 0; u < U; u++) {
		locate(page[u], pg[u], krow[u], ks[u], vs[u]);
#pragma unroll
		for (int c = 0; c < KB; c++) kr[u][c] = *reinterpret_cast<const uint4*>(krow[u] + 16 * (FULL ? c : min(c, kchunks - 1)));
	}
	for (int t0 = first; t0 < hi; t0 += 256 * U) {
		float nks[U], nvs[U];
		int npg[U];
		const int8_t* nrow[U];
#pragma unroll
		for (int u = 0; u < U; u++) {
			locate(after[u], npg[u], nrow[u], nks[u], nvs[u]);
			after[u] = page_of(t0 + 64 * u + lane + 512 * U);
		}
		// piece c of the key rows: of this step's, then the first ones of the next step's
		auto piece = [&](int u, int c) {
			const int8_t* row = c < kend ? krow[u] : nrow[u];
			c -= c < kend ? 0 : kend;
			return *reinterpret_cast<const uint4*>(row + 16 * (FULL ? c : min(c, kchunks - 1)));
		};
		// the values: for 16 bits eight tokens in a row of every 32, for float32 four of every 16, four columns each
		constexpr int VT = F32 ? 4 : 8;
		unsigned vr[16 * U / VT][VG][VT];
		auto load_values = [&]() {
#pragma unroll
			for (int kc = 0; kc < 16 * U / VT; kc++) {
				const int tok = 4 * VT * kc + VT * g;
				const int vp = max(__shfl(pg[kc * 4 * VT / 64], tok & 63), 0);
				const int8_t* row = page_at(vbase, vp, vstride) + (tok & (C.P - 1)) * pv + (FULL ? 4 * l16 : 0);
#pragma unroll
				for (int wg = 0; wg < VG; wg++)
#pragma unroll
					for (int e = 0; e < VT; e++)
						vr[kc][wg][e] = *reinterpret_cast<const unsigned*>(row + e * pv + (FULL ? 64 * wg : min(64 * wg + 4 * l16, pv - 4)));
			}
		};
		if constexpr (!LATE) load_values();
		float dist[U][RB];
		if (coded) {
			unsigned sum[U][RB];
#pragma unroll
			for (int u = 0; u < U; u++)
#pragma unroll
				for (int r = 0; r < RB; r++) sum[u][r] = 0;
#pragma unroll 1
			for (int c0 = 0; c0 < kchunks; c0 += KB) {
#pragma unroll
				for (int i = 0; i < KB; i++) {
					const int c = c0 + i;
					const float b[2] = {off + l1_code_eight(2 * c), off + l1_code_eight(2 * c + 1)};
					unsigned kc[U][8];
#pragma unroll
					for (int u = 0; u < U; u++) {
						const uint4 raw = kr[u][i];
						kr[u][i] = piece(u, c + KB);
						const int word[4] = {(int)raw.x, (int)raw.y, (int)raw.z, (int)raw.w};
						const float f = ks[u] * sc;
#pragma unroll
						for (int d = 0; d < 4; d++) {
							float x[4];
							codes4(word[d], x);
#pragma unroll
							for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(x[e], f, b[d >> 1] + l1_code_column(4 * (d & 1) + e));
							kc[u][2 * d] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(x[0], x[1]));
							kc[u][2 * d + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(x[2], x[3]));
						}
					}
					if (FULL || c < kchunks)
						{
							// the rows' codes are read four pieces ahead of their use
							const unsigned* from = qc + 8 * c;
							uint4 ring[4];
#pragma unroll
							for (int j = 0; j < 4; j++) ring[j] = *reinterpret_cast<const uint4*>(from + (j >> 1) * 64 + 4 * (j & 1));
#pragma unroll
							for (int j = 0; j < 2 * RB; j++) {
								const int r = j >> 1, h = j & 1;
								const uint4 y = ring[j & 3];
#pragma unroll
								for (int u = 0; u < U; u++) {
									unsigned z = sum[u][r];
									z = __builtin_amdgcn_sad_u16(kc[u][4 * h], y.x, z);
									z = __builtin_amdgcn_sad_u16(kc[u][4 * h + 1], y.y, z);
									z = __builtin_amdgcn_sad_u16(kc[u][4 * h + 2], y.z, z);
									z = __builtin_amdgcn_sad_u16(kc[u][4 * h + 3], y.w, z);
									sum[u][r] = z;
								}
								if (j + 4 < 2 * RB) ring[j & 3] = *reinterpret_cast<const uint4*>(from + ((j + 4) >> 1) * 64 + 4 * (j & 1));
								__builtin_amdgcn_sched_barrier(0);
							}
						}
				}
			}
#pragma unroll
			for (int u = 0; u < U; u++)
#pragma unroll
				for (int r = 0; r < RB; r++) dist[u][r] = (float)sum[u][r];
		} else {
#pragma unroll
			for (int u = 0; u < U; u++)
#pragma unroll
				for (int r = 0; r < RB; r++) dist[u][r] = 0.f;
#pragma unroll 1
			for (int c0 = 0; c0 < kchunks; c0 += KB) {
#pragma unroll
				for (int i = 0; i < KB; i++) {
					const int c = c0 + i;
					uint4 raw[U];
#pragma unroll
					for (int u = 0; u < U; u++) {
						raw[u] = kr[u][i];
						kr[u][i] = piece(u, c + KB);
					}
					if (FULL || c < kchunks) {
						const float* from = qs + 16 * c;
						constexpr int AHEAD = 4 * RB < 4 ? 4 * RB : 4;
						float4 ring[AHEAD];
						float k[U][4];
#pragma unroll
						for (int j = 0; j < AHEAD; j++) ring[j] = *reinterpret_cast<const float4*>(from + j % RB * 128 + 4 * (j / RB));
#pragma unroll
						for (int j = 0; j < 4 * RB; j++) {
							const int d = j / RB, r = j % RB;
							if (r == 0)
#pragma unroll
								for (int u = 0; u < U; u++) codes4((int)(d == 0 ? raw[u].x : d == 1 ? raw[u].y : d == 2 ? raw[u].z : raw[u].w), k[u]);
							const float4 y = ring[j % AHEAD];
#pragma unroll
							for (int u = 0; u < U; u++) {
								const float d0 = __builtin_fmaf(-k[u][0], ks[u], y.x), d1 = __builtin_fmaf(-k[u][1], ks[u], y.y);
								const float d2 = __builtin_fmaf(-k[u][2], ks[u], y.z), d3 = __builtin_fmaf(-k[u][3], ks[u], y.w);
								dist[u][r] += (__builtin_fabsf(d0) + __builtin_fabsf(d1)) + (__builtin_fabsf(d2) + __builtin_fabsf(d3));
							}
							if (j + AHEAD < 4 * RB) ring[j % AHEAD] = *reinterpret_cast<const float4*>(from + (j + AHEAD) % RB * 128 + 4 * ((j + AHEAD) / RB));
							__builtin_amdgcn_sched_barrier(0);
						}
					}
				}
			}
		}
		if constexpr (LATE) load_values();
#pragma unroll
		for (int u = 0; u < U; u++)
#pragma unroll
			for (int r = 0; r < RB; r++) dist[u][r] *= -m;
		if (A.cap > 0.f) {  // see softcap.h
			float near = -3.402823466e38f;
			if constexpr (!F32)
#pragma unroll
				for (int u = 0; u < U; u++)
#pragma unroll
					for (int r = 0; r < RB; r++) near = fmaxf(near, dist[u][r]);
			if (!F32 && __any(near * A.icap > -kCapSeries)) {
#pragma unroll
				for (int u = 0; u < U; u++)
#pragma unroll
					for (int r = 0; r < RB; r++) {
						float d;  // the derivative, of which there is no use
						const float y = dist[u][r] * A.icap;
						dist[u][r] = y > -kCapSeries ? dist[u][r] * l1_tanh_near(y) : A.cap * l1_tanh_far(y, d);
					}
			} else {
#pragma unroll
				for (int u = 0; u < U; u++)
#pragma unroll
					for (int r = 0; r < RB; r++) {
						float d;
						dist[u][r] = A.cap * (F32 ? tanhf(dist[u][r] * A.icap) : l1_tanh_far(dist[u][r] * A.icap, d));
					}
			}
		}
#pragma unroll
		for (int u = 0; u < U; u++) {
			const int t = t0 + 64 * u + lane, sees = pg[u] >= 0 ? t : 0x7fffffff;
#pragma unroll
			for (int r = 0; r < RB; r++) {
				const float w = exponential<ST>(__builtin_fmaf(-slope[r], (float)(place[r] - t), dist[u][r]));
				const float p = sees <= place[r] ? w : 0.f;
				den[r] += p;
				const float both = p != 0.f ? p * vs[u] : 0.f;  // the scale of a hidden token has no influence
				const PT first = (PT)both;
				ps[r * pitch + 64 * u + lane] = first;
				const float rest = both - (float)first;  // an infinite weight has none: infinity less itself is NaN
				if constexpr (!F32) ps[plane + r * pitch + 64 * u + lane] = (PT)(__builtin_fabsf(rest) <= 3.402823466e38f ? rest : 0.f);
			}
		}
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		__builtin_amdgcn_wave_barrier();
#pragma unroll
		for (int wg = 0; wg < VG; wg++) {
#pragma unroll
			for (int kc = 0; kc < 16 * U / VT; kc++) {
				const uint4 pa = *reinterpret_cast<const uint4*>(ps + l16 % RB * pitch + 4 * VT * kc + VT * g);
				const uint4 rest = *reinterpret_cast<const uint4*>(ps + plane + l16 % RB * pitch + 4 * VT * kc + VT * g);
				if constexpr (F32) {
					const float a[4] = {__builtin_bit_cast(float, pa.x), __builtin_bit_cast(float, pa.y), __builtin_bit_cast(float, pa.z), __builtin_bit_cast(float, pa.w)};
#pragma unroll
					for (int d = 0; d < 4; d++) {
						float x[4];
						codes4((int)vr[kc][wg][d], x);
#pragma unroll
						for (int e = 0; e < 4; e++) acc[wg][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[d], x[e], acc[wg][e], 0, 0, 0);
					}
				} else {
#pragma unroll
					for (int e = 0; e < 4; e++) {
						unsigned x[4];
#pragma unroll
						for (int d = 0; d < 4; d++) {
							const unsigned v0 = vr[kc][wg][2 * d], v1 = vr[kc][wg][2 * d + 1];
							// a code's float32 ends in 16 zero bits
							const float a = (float)(int8_t)(v0 >> 8 * e), c = (float)(int8_t)(v1 >> 8 * e);
							x[d] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, c), __builtin_bit_cast(unsigned, a), 0x07060302u);
						}
						const uint4 pb = make_uint4(x[0], x[1], x[2], x[3]);
#pragma unroll
						for (int d = 0; d < 2; d++) acc[wg][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, d ? rest : pa), __builtin_bit_cast(b8, pb), acc[wg][e], 0, 0, 0);
					}
				}
			}
		}
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		__builtin_amdgcn_wave_barrier();
#pragma unroll
		for (int u = 0; u < U; u++) { pg[u] = npg[u]; krow[u] = nrow[u]; ks[u] = nks[u]; vs[u] = nvs[u]; }
	}
	// rows 4 g + i (a row again every RB), columns 64 wg + 4 l16 + e; over the waves through LDS, where the weights lay
#pragma unroll
	for (int r = 0; r < RB; r++) {
#pragma unroll
		for (int k = 32; k; k >>= 1) den[r] += __shfl_xor(den[r], k);
		if (lane == 0) dens[wave * RB + r] = den[r];
	}
	__syncthreads();
	float* sums = reinterpret_cast<float*>(shared_pool);  // [2 waves][RB][128], in two turns
	for (int turn = 0; turn < 2; turn++) {
		if ((wave >> 1) == turn)
#pragma unroll
			for (int wg = 0; wg < VG; wg++)
#pragma unroll
				for (int i = 0; i < 4; i++) {
					if (4 * g + i >= RB) continue;
					float* at = sums + ((wave & 1) * RB + 4 * g + i) * 128 + 64 * wg + 4 * l16;
					f4 y = {acc[wg][0][i], acc[wg][1][i], acc[wg][2][i], acc[wg][3][i]};
					if (turn) y += *reinterpret_cast<const f4*>(at);
					*reinterpret_cast<f4*>(at) = y;
				}
		__syncthreads();
	}
	if (myrow < 0) return;
	const float d = dens[my] + dens[RB + my] + dens[2 * RB + my] + dens[3 * RB + my];
	float* to = part + ((int64_t)(slot - b) * A.n * A.H + myrow) * (C.Wv + 1);  // [slot][n][H]
	if (part && my0 == 0) to[C.Wv] = d;
	for (int w = my0; w < C.Wv; w += TR) {
		const float y = sums[my * 128 + w] + sums[(RB + my) * 128 + w];
		if (part) to[w] = y;
		else o[myrow * C.Wv + w] = (ST)(y / (1.f + d));
	}
}

// The sums of each entry's slots, in their order, two heads of a workgroup.  Grid: n, B, heads.
template <typename ST>
__global__ void __launch_bounds__(256) paged_join(AttendArgs A, const float* __restrict__ part, const int2* __restrict__ spans, ST* __restrict__ o)
{
	const int2 S = spans[blockIdx.y];
	const int Wv = A.C.Wv, w = threadIdx.x & 127, h = 2 * blockIdx.z + (threadIdx.x >> 7);
	if (w >= Wv || h >= A.H) return;
	const float* p = part + (((int64_t)S.x * A.n + blockIdx.x) * A.H + h) * (Wv + 1);
	const int64_t pitch = (int64_t)A.n * A.H * (Wv + 1);
	float d = 1.f, y = 0.f;
#pragma unroll 8
	for (int u = 0; u < S.y; u++, p += pitch) {
		d += p[Wv];
		y += p[w];
	}
	o[(((int64_t)blockIdx.y * A.n + blockIdx.x) * A.H + h) * Wv + w] = (ST)(y / d);
}

// rows of a workgroup
int row_block(int64_t R) { return R <= 1 ? 1 : R <= 2 ? 2 : R <= 4 ? 4 : R <= 8 ? 8 : 16; }

// Workgroups of each key head and block of rows: as many as fill the 256 compute units once (two of 8 or 16 rows, four of fewer
// rows), at least two for each entry.  0: each entry has one, which writes the result itself: 12 us for one sequence of 300
// tokens, 16.6 with a kernel that joins; and where the entries alone are many.  Dealing out the steps of all entries instead of
// an equal number of splits for each: 169 -> 140 us for 16 sequences of 8192 to 32768 tokens.
int slots_for(const L1Cache& C, int64_t B, int rows, int64_t others)
{
	if (B > 512 || (int64_t)C.M * C.P <= 512) return 0;
	const int64_t want = l1_cdiv(rows <= 4 ? 1024 : 512, others), most = B * l1_cdiv((int64_t)C.M * C.P, rows <= 4 ? 256 : 512);
	const int64_t n = want > 2 * B ? want : 2 * B;
	return (int)(n < most + B ? n : most + B);
}

template <typename ST>
int attend(const AttendArgs& A, const void* q, const int32_t* seqs, const int32_t* counts, void* o, int2* ws, hipStream_t st)
{
	const int rb = row_block((int64_t)A.n * A.G);
	const dim3 grid((unsigned)((A.slots ? A.slots : A.B) * A.C.Hk), (unsigned)l1_cdiv((int64_t)A.n * A.G, rb));
	int2* spans = A.slots ? ws : nullptr;  // of each entry; behind them the sums
	float* part = spans ? reinterpret_cast<float*>(ws + A.B) : nullptr;
	const int full = A.C.pk == A.C.pv ? A.C.pk : 0;  // rows of 64 or 128 bytes: addresses and loops are known to the compiler
#define L1_ATTEND(RB, MINW)                                                                                                                          \
	if (full == 64) hipLaunchKernelGGL((paged_attend<ST, RB, 4, true, MINW>), grid, dim3(256), 0, st, A, (const ST*)q, seqs, counts, (ST*)o, part, spans);  \
	else if (full == 128) hipLaunchKernelGGL((paged_attend<ST, RB, 8, true, 2>), grid, dim3(256), 0, st, A, (const ST*)q, seqs, counts, (ST*)o, part, spans); \
	else hipLaunchKernelGGL((paged_attend<ST, RB, 8, false, 2>), grid, dim3(256), 0, st, A, (const ST*)q, seqs, counts, (ST*)o, part, spans)
	if (rb == 1) { L1_ATTEND(1, 4); }
	else if (rb == 2) { L1_ATTEND(2, 4); }
	else if (rb == 4) { L1_ATTEND(4, 4); }
	else if (rb == 8) { L1_ATTEND(8, 2); }
	else { L1_ATTEND(16, 2); }
#undef L1_ATTEND
	L1_LAUNCH_CHECK();
	if (part) {
		hipLaunchKernelGGL(paged_join<ST>, dim3((unsigned)A.n, (unsigned)A.B, (unsigned)((A.H + 1) / 2)), dim3(256), 0, st, A, part, spans, (ST*)o);
		L1_LAUNCH_CHECK();
	}
	return L1ATTN_OK;
}

// 0, an error, or 1 for a call with nothing to do
int check_attend(const l1attn_cache* cache, const l1attn_attend_desc* d, AttendArgs* A)
{
	const int rc = l1_cache_args(cache, &A->C);
	if (rc != L1ATTN_OK) return rc;
	if (!d || d->B < 0 || d->n < 0 || d->H < 1 || d->H % A->C.Hk || d->dtype < 0 || d->dtype > 2) return L1ATTN_ERR_ARG;
	if (!(d->softcap >= 0.f) || !(d->softcap <= 3e38f)) return L1ATTN_ERR_ARG;
	if (d->H > 256 || d->B > 65535 || d->n > 65536 || d->B * A->C.Hk > 65535 || d->B * d->n * d->H > 0x7fffffff) return L1ATTN_ERR_RANGE;
	if (d->slopes)
		for (int64_t h = 0; h < d->H; h++)
			if (!(d->slopes[h] >= 0.f) || !(d->slopes[h] <= 3e38f)) return L1ATTN_ERR_ARG;
	A->B = (int)d->B; A->n = (int)d->n; A->H = (int)d->H; A->G = (int)(d->H / A->C.Hk);
	if (l1_cdiv(d->n * A->G, 8) > 65535) return L1ATTN_ERR_RANGE;
	A->cap = d->softcap; A->icap = l1_icap(d->softcap);
	A->rw = (float)(1.0 / sqrt((double)A->C.W));
	for (int h = 0; h < 256; h++) A->slopes[h] = d->slopes && h < d->H ? d->slopes[h] : 0.f;
	if (d->B == 0 || d->n == 0) return 1;
	const int rb = row_block(d->n * A->G);
	A->step = rb <= 4 ? 256 : 512;
	A->slots = slots_for(A->C, d->B, rb, A->C.Hk * l1_cdiv(d->n * A->G, rb));
	return L1ATTN_OK;
}

}  // namespace

extern "C" {

size_t l1attn_cache_attend_workspace_bytes(const l1attn_cache* cache, const l1attn_attend_desc* desc)
{
	AttendArgs A;
	if (check_attend(cache, desc, &A) || !A.slots) return 0;
	return A.B * sizeof(int2) + (size_t)A.slots * A.n * A.H * (A.C.Wv + 1) * sizeof(float);
}

int l1attn_cache_attend(const l1attn_cache* cache, const l1attn_attend_desc* desc, const void* q, const int32_t* seqs, const int32_t* counts,
                        void* o, void* workspace, size_t workspace_bytes, void* stream)
{
	AttendArgs A;
	const int rc = check_attend(cache, desc, &A);
	if (rc) return rc == 1 ? L1ATTN_OK : rc;
	if (!q || !o) return L1ATTN_ERR_ARG;
	const size_t need = l1attn_cache_attend_workspace_bytes(cache, desc);
	if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 8)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	if (desc->dtype == 0) return attend<float>(A, q, seqs, counts, o, (int2*)workspace, st);
	if (desc->dtype == 1) return attend<_Float16>(A, q, seqs, counts, o, (int2*)workspace, st);
	return attend<__bf16>(A, q, seqs, counts, o, (int2*)workspace, st);
}

}  // extern "C"
