// L1 attention of each sequence's last tokens over its pages of the 8-bit cache.
//
//   x[r,s] = c(-1/sqrt(W) * sum_w |q[r,w] - code[s,w] * scale[page of s]|) - slope * (place of r - s),   s <= place of r
//   o[r]   = sum_s exp(x) * v[s] / (1 + sum_s exp(x))
//
// The rows r of a workgroup are the query tokens and query heads that read one key head.  Every logit is <= 0 and the no-op
// logit is 0, so partial sums over pieces of a sequence simply add up: no running maximum, and the pieces join in a fixed
// order.  A workgroup takes 256 tokens at a time: a lane holds one token's key row and forms the distances of all rows
// (the rows' values are broadcast LDS reads); then a lane holds 16 value columns of every 16th token and adds p * v.
// The bytes of the cache are read once and are what bounds it for few rows; with many rows it is the vector ALU.
#include "paged.h"
#include <math.h>

namespace {

constexpr int kTok = 256;  // tokens of a step, one for each thread

struct AttendArgs {
	L1Cache C;
	int B, n, H, G, splits;
	float cap, icap, rw;
	int has_slopes;
	float slopes[256];
};

// the tokens [lo, hi) of a split: whole steps, spread evenly; the same in the join
__device__ __forceinline__ int split_tokens(int len, int splits)
{
	const int per = (len + splits - 1) / splits;
	return (per + kTok - 1) / kTok * kTok;
}

template <typename ST> __device__ __forceinline__ float value(ST x) { return (float)x; }

// length of entry b's sequence, 0 where it names none
__device__ __forceinline__ int seq_of(const AttendArgs& A, const int32_t* seqs, int b, int& s)
{
	s = seqs ? seqs[b] : b;
	if (s < 0 || s >= A.C.rows) return 0;
	return min(max(A.C.lens[s], 0), A.C.M * A.C.P);
}

// RB: rows of a workgroup.  Grid: splits, batch * key heads, blocks of rows.
// part: [splits][B][n][H][Wv + 1] (the last: the weights' sum), or NULL with one split, which writes o itself.
template <typename ST, int RB>
__global__ void __launch_bounds__(256) paged_attend(AttendArgs A, const ST* __restrict__ q, const int32_t* __restrict__ seqs,
                                                    const int32_t* __restrict__ counts, ST* __restrict__ o, float* __restrict__ part)
{
	constexpr int RP = RB < 4 ? RB : RB + 4;  // floats between two tokens' weights
	__shared__ __align__(16) float qs[RB * 128];
	__shared__ __align__(16) float ps[kTok * RP];
	__shared__ float vscale[kTok];
	__shared__ int vpage[kTok];
	const L1Cache& C = A.C;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	const int b = blockIdx.y / C.Hk, hk = blockIdx.y % C.Hk, r0 = blockIdx.z * RB, R = A.n * A.G;
	int s;
	const int len = seq_of(A, seqs, b, s);
	const int cnt = counts ? min(max(counts[b], 0), A.n) : A.n;
	const int per = split_tokens(len, A.splits), lo = blockIdx.x * per, hi = min(lo + per, len);
	if (lo >= hi && part) return;  // the join knows which splits there are
	// the rows' values, zero behind the width: the cache's rows are zero there as well
	for (int x = tid; x < RB * C.pk; x += 256) {
		const int r = r0 + x / C.pk, w = x % C.pk;
		const int t = r / A.G, h = hk * A.G + r % A.G;
		qs[(x / C.pk) * 128 + w] = r < R && w < C.W ? value(q[(((int64_t)b * A.n + t) * A.H + h) * C.W + w]) : 0.f;
	}
	float slope[RB];
	int place[RB];
#pragma unroll
	for (int r = 0; r < RB; r++) {
		const int t = (r0 + r) / A.G;
		slope[r] = A.has_slopes && r0 + r < R ? A.slopes[hk * A.G + (r0 + r) % A.G] : 0.f;
		place[r] = r0 + r < R && t < cnt ? len - cnt + t : -1;  // sees nothing
	}
	const int vchunks = C.pv / 16;           // lanes of a value row
	const int vtok = 64 / vchunks;           // tokens that a wave reads at once
	const int vc = lane % vchunks, vt = lane / vchunks;
	const bool vlane = vt < vtok;
	float acc[RB][16], den[RB];
#pragma unroll
	for (int r = 0; r < RB; r++) {
		den[r] = 0.f;
#pragma unroll
		for (int e = 0; e < 16; e++) acc[r][e] = 0.f;
	}
	const int32_t* table = C.table + (int64_t)s * C.M;
	for (int t0 = lo; t0 < hi; t0 += kTok) {
		__syncthreads();
		const int t = t0 + tid;
		const int page = t < hi ? table[t / C.P] : -1;
		const bool there = page >= 0 && page < C.N;
		const int64_t at = there ? ((int64_t)page * C.Hk + hk) : 0;
		float dist[RB];
#pragma unroll
		for (int r = 0; r < RB; r++) dist[r] = 0.f;
		const float ks = there ? C.ks[at] : 0.f;
		vscale[tid] = there ? C.vs[at] : 0.f;
		vpage[tid] = there ? page : -1;
		if (there) {
			const int8_t* row = C.k + (at * C.P + t % C.P) * C.pk;
			for (int w = 0; w < C.pk; w += 16) {
				const uint4 raw = *reinterpret_cast<const uint4*>(row + w);
				const int word[4] = {(int)raw.x, (int)raw.y, (int)raw.z, (int)raw.w};
#pragma unroll
				for (int d = 0; d < 4; d++) {
					const float k0 = (float)(int8_t)word[d], k1 = (float)(int8_t)(word[d] >> 8), k2 = (float)(int8_t)(word[d] >> 16), k3 = (float)(word[d] >> 24);
#pragma unroll
					for (int r = 0; r < RB; r++) {
						const float4 qv = *reinterpret_cast<const float4*>(qs + r * 128 + w + 4 * d);
						dist[r] += __builtin_fabsf(__builtin_fmaf(-k0, ks, qv.x));
						dist[r] += __builtin_fabsf(__builtin_fmaf(-k1, ks, qv.y));
						dist[r] += __builtin_fabsf(__builtin_fmaf(-k2, ks, qv.z));
						dist[r] += __builtin_fabsf(__builtin_fmaf(-k3, ks, qv.w));
					}
				}
			}
		}
#pragma unroll
		for (int r = 0; r < RB; r++) {
			float c = -dist[r] * A.rw;
			if (A.cap > 0.f) c = A.cap * tanhf(c * A.icap);
			const float p = there && t <= place[r] ? expf(c - slope[r] * (float)(place[r] - t)) : 0.f;
			den[r] += p;
			ps[tid * RP + r] = p;
		}
		__syncthreads();
		// values: wave `wave` takes every fourth group of vtok tokens
		if (vlane)
			for (int u = wave * vtok + vt; u < min(kTok, hi - t0); u += 4 * vtok) {
				const int pg = vpage[u];
				if (pg < 0) continue;
				const float vs = vscale[u];
				const int8_t* row = C.v + (((int64_t)pg * C.Hk + hk) * C.P + (t0 + u) % C.P) * C.pv + 16 * vc;
				const uint4 raw = *reinterpret_cast<const uint4*>(row);
				const int word[4] = {(int)raw.x, (int)raw.y, (int)raw.z, (int)raw.w};
				float x[16];
#pragma unroll
				for (int d = 0; d < 4; d++) {
					x[4 * d] = (float)(int8_t)word[d];
					x[4 * d + 1] = (float)(int8_t)(word[d] >> 8);
					x[4 * d + 2] = (float)(int8_t)(word[d] >> 16);
					x[4 * d + 3] = (float)(word[d] >> 24);
				}
#pragma unroll
				for (int r = 0; r < RB; r++) {
					const float p = ps[u * RP + r];
					const float pv = p != 0.f ? p * vs : 0.f;  // the scale of a hidden token has no influence
#pragma unroll
					for (int e = 0; e < 16; e++) acc[r][e] = __builtin_fmaf(pv, x[e], acc[r][e]);
				}
			}
	}
	// sums over the lanes and waves, in a fixed order, row by row through LDS
	__syncthreads();
	__shared__ float red[4 * 128 + 4];  // a row's columns of each wave, and the sums of its weights
	for (int r = 0; r < RB; r++) {
#pragma unroll
		for (int m = 32; m; m >>= 1) den[r] += __shfl_xor(den[r], m);
	}
#pragma unroll
	for (int r = 0; r < RB; r++) {
		// each wave's own columns: over its tokens vt
		float sum[16];
#pragma unroll
		for (int e = 0; e < 16; e++) sum[e] = acc[r][e];
		__syncthreads();
		for (int step = vtok; step > 1;) {
			const int half = (step + 1) / 2;
#pragma unroll
			for (int e = 0; e < 16; e++) {
				const float y = __shfl(sum[e], min(lane + half * vchunks, 63));
				if (vt + half < step) sum[e] += y;
			}
			step = half;
		}
		if (vlane && vt == 0)
#pragma unroll
			for (int e = 0; e < 16; e++) red[wave * 128 + 16 * vc + e] = sum[e];
		if (lane == 0) red[512 + wave] = den[r];
		__syncthreads();
		const int row = r0 + r;
		if (row < R) {
			const int64_t out = ((int64_t)b * A.n + row / A.G) * A.H + hk * A.G + row % A.G;
			const float d = red[512] + red[513] + red[514] + red[515];
			for (int w = tid; w < C.Wv; w += 256) {
				const float y = red[w] + red[128 + w] + red[256 + w] + red[384 + w];
				if (part) part[((int64_t)blockIdx.x * A.B * A.n * A.H + out) * (C.Wv + 1) + w] = y;
				else o[out * C.Wv + w] = (ST)(y / (1.f + d));
			}
			if (part && tid == 0) part[((int64_t)blockIdx.x * A.B * A.n * A.H + out) * (C.Wv + 1) + C.Wv] = d;
		}
	}
}

// the splits of each row, in their order
template <typename ST>
__global__ void __launch_bounds__(128) paged_join(AttendArgs A, const float* __restrict__ part, const int32_t* __restrict__ seqs, ST* __restrict__ o)
{
	const int64_t row = blockIdx.x, rows = (int64_t)A.B * A.n * A.H;
	const int b = (int)(row / ((int64_t)A.n * A.H));
	int s;
	const int len = seq_of(A, seqs, b, s);
	const int per = split_tokens(len, A.splits), m = len ? (len + per - 1) / per : 0, Wv = A.C.Wv;
	float d = 1.f, y = 0.f;
	for (int u = 0; u < m; u++) {
		const float* p = part + ((int64_t)u * rows + row) * (Wv + 1);
		d += p[Wv];
		if ((int)threadIdx.x < Wv) y += p[threadIdx.x];
	}
	if ((int)threadIdx.x < Wv) o[row * Wv + threadIdx.x] = (ST)(y / d);
}

// workgroups that a call is split into over the tokens: about four for each of the 256 compute units in all
int splits_for(const L1Cache& C, int64_t groups)
{
	const int64_t most = l1_cdiv((int64_t)C.M * C.P, kTok), want = l1_cdiv(1024, groups);
	return (int)(want < 1 ? 1 : want > most ? (most < 1 ? 1 : most) : want);
}

int row_block(int64_t R) { return R <= 1 ? 1 : R <= 2 ? 2 : R <= 4 ? 4 : 8; }

template <typename ST, int RB>
int attend(const AttendArgs& A, const void* q, const int32_t* seqs, const int32_t* counts, void* o, float* part, hipStream_t st)
{
	const dim3 grid((unsigned)A.splits, (unsigned)(A.B * A.C.Hk), (unsigned)l1_cdiv((int64_t)A.n * A.G, RB));
	hipLaunchKernelGGL((paged_attend<ST, RB>), grid, dim3(256), 0, st, A, (const ST*)q, seqs, counts, (ST*)o, A.splits > 1 ? part : nullptr);
	L1_LAUNCH_CHECK();
	if (A.splits > 1) {
		hipLaunchKernelGGL(paged_join<ST>, dim3((unsigned)(A.B * A.n * A.H)), dim3(128), 0, st, A, part, seqs, (ST*)o);
		L1_LAUNCH_CHECK();
	}
	return L1ATTN_OK;
}

template <typename ST>
int attend_rows(const AttendArgs& A, const void* q, const int32_t* seqs, const int32_t* counts, void* o, float* part, hipStream_t st)
{
	switch (row_block((int64_t)A.n * A.G)) {
	case 1: return attend<ST, 1>(A, q, seqs, counts, o, part, st);
	case 2: return attend<ST, 2>(A, q, seqs, counts, o, part, st);
	case 4: return attend<ST, 4>(A, q, seqs, counts, o, part, st);
	default: return attend<ST, 8>(A, q, seqs, counts, o, part, st);
	}
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
	A->cap = d->softcap; A->icap = d->softcap > 0.f ? 1.f / d->softcap : 0.f;
	A->rw = (float)(1.0 / sqrt((double)A->C.W));
	A->has_slopes = d->slopes != nullptr;
	for (int h = 0; h < 256; h++) A->slopes[h] = d->slopes && h < d->H ? d->slopes[h] : 0.f;
	if (d->B == 0 || d->n == 0) return 1;
	const int64_t groups = d->B * A->C.Hk * l1_cdiv(d->n * A->G, row_block(d->n * A->G));
	A->splits = splits_for(A->C, groups);
	return L1ATTN_OK;
}

}  // namespace

extern "C" {

size_t l1attn_cache_attend_workspace_bytes(const l1attn_cache* cache, const l1attn_attend_desc* desc)
{
	AttendArgs A;
	if (check_attend(cache, desc, &A) || A.splits == 1) return 0;
	return (size_t)A.splits * A.B * A.n * A.H * (A.C.Wv + 1) * sizeof(float);
}

int l1attn_cache_attend(const l1attn_cache* cache, const l1attn_attend_desc* desc, const void* q, const int32_t* seqs, const int32_t* counts,
                        void* o, void* workspace, size_t workspace_bytes, void* stream)
{
	AttendArgs A;
	const int rc = check_attend(cache, desc, &A);
	if (rc) return rc == 1 ? L1ATTN_OK : rc;
	if (!q || !o) return L1ATTN_ERR_ARG;
	const size_t need = l1attn_cache_attend_workspace_bytes(cache, desc);
	if (need && (!workspace || workspace_bytes < need)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	if (desc->dtype == 0) return attend_rows<float>(A, q, seqs, counts, o, (float*)workspace, st);
	if (desc->dtype == 1) return attend_rows<_Float16>(A, q, seqs, counts, o, (float*)workspace, st);
	return attend_rows<__bf16>(A, q, seqs, counts, o, (float*)workspace, st);
}

}  // extern "C"
