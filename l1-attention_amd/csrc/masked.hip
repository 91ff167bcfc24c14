// Entry points of the masked L1 attention: checks, how a launch is cut, workspaces.  The kernels: masked_kernels.h.
#include "common.h"
#include "masked.h"
#include "softcap.h"
#include <math.h>

namespace {

__global__ void __launch_bounds__(256) masked_zero(uint16_t* __restrict__ x, int64_t n)
{
	for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) x[at] = 0;
}

unsigned zero_blocks(int64_t n) { return (unsigned)(n < 256 << 16 ? l1_cdiv(n, 256) : 1 << 16); }

bool fits(int64_t x, int64_t most) { return x >= 0 && x <= most; }

// waves of a workgroup: as many as share what they stage, see plan_of
int most_waves(const l1attn_masked_desc* d) { return d->dtype == 0 && d->W <= 64 && d->Wv <= 64 ? 8 : 4; }

// 0, an error, or 1 for a call with nothing to do
int check_desc(const l1attn_masked_desc* d)
{
	if (!d) return L1ATTN_ERR_ARG;
	if (d->B < 0 || d->T < 0 || d->S < d->T || d->H < 1 || d->Hk < 1 || d->H % d->Hk || d->W < 1 || d->Wv < 1) return L1ATTN_ERR_ARG;
	if (d->dtype < 0 || d->dtype > 2 || (d->causal != 0 && d->causal != 1)) return L1ATTN_ERR_ARG;
	if (!(d->softcap >= 0.f) || !(d->softcap <= 3e38f)) return L1ATTN_ERR_ARG;
	// 65535 rows of the grid at two waves of 32 rows; batch * heads is the grid's other side, which has 2^32 - 1 threads at most
	if (d->W > 128 || d->Wv > 128 || d->H > L1_MASKED_HEADS || !fits(d->S, 64 * 65535) || !fits(d->B, 1 << 22) ||
	    !fits(d->B * d->H, 0xffffffffll / (64 * most_waves(d))))
		return L1ATTN_ERR_RANGE;
	if (d->slopes)
		for (int64_t h = 0; h < d->H; h++)
			if (!(d->slopes[h] >= 0.f) || !(d->slopes[h] <= 3e38f)) return L1ATTN_ERR_ARG;
	return d->B == 0 || d->T == 0 ? 1 : L1ATTN_OK;
}

L1MaskedArgs args_of(const l1attn_masked_desc* d, const void* q, const void* k, const void* v, const void* o)
{
	L1MaskedArgs A;
	A.B = (int)d->B; A.T = (int)d->T; A.S = (int)d->S; A.H = (int)d->H; A.Hk = (int)d->Hk; A.W = (int)d->W; A.Wv = (int)d->Wv;
	A.causal = d->causal; A.cap = d->softcap; A.icap = l1_icap(d->softcap);
	A.rw = (float)(1.0 / sqrt((double)d->W));
	A.doc = d->doc; A.prefix = d->causal ? d->prefix : nullptr; A.has_slopes = d->slopes != nullptr;
	A.rest = d->dtype == 0 ? nullptr : d->o_rest;
	for (int h = 0; h < L1_MASKED_HEADS; h++) A.slopes[h] = d->slopes && h < d->H ? d->slopes[h] : 0.f;
	const int per = d->dtype == 0 ? 4 : 8;
	A.vec = (d->W % per == 0 && !((uintptr_t)q & 15) ? 1 : 0) | (d->W % per == 0 && !((uintptr_t)k & 15) ? 2 : 0) |
	        (d->Wv % per == 0 && !((uintptr_t)v & 15) ? 4 : 0) | (d->Wv % per == 0 && !((uintptr_t)o & 15) ? 8 : 0);
	return A;
}

const L1MaskedTable& table_of(int dtype) { return dtype == 0 ? l1_masked_f32() : dtype == 1 ? l1_masked_f16() : l1_masked_bf16(); }

// Waves of a workgroup share what they stage; a compute unit has 160 KB of LDS, and 256 of them want work.  16-bit rows: four
// waves, of which two workgroups fit a compute unit and work while the other one waits (eight in one: 263 instead of 218 us for
// the forward of B1 T4096 H16 W64 with documents); float32: eight where they leave no unit idle, since one workgroup fits either way.
// Then as many splits of the other side's tiles as make 1024 workgroups, which also evens out what masks leave to do (the two
// backward kernels of the same shape: 1.90 ms with 512, 1.28 with 1024, 1.21 with 2048, where shorter ones lose more than that:
// the forward of B2 T1024 S2048 H16/4 W64 takes 168, 156 and 171 us), none of them with fewer than two tiles of 64.
L1MaskedPlan plan_of(const L1MaskedTable& t, int64_t owners, int64_t stream, int64_t heads, const l1attn_masked_desc* d, bool backward, bool weigh)
{
	L1MaskedPlan p;
	const int W = (int)d->W, Wv = (int)d->Wv;
	p.waves = most_waves(d);
	while (p.waves > 2 && (t.lds(W, Wv, p.waves, backward, weigh) > 160 * 1024 || heads * l1_cdiv(owners, 32 * p.waves) < 256)) p.waves >>= 1;
	int64_t s = l1_cdiv(1024, heads * l1_cdiv(owners, 32 * p.waves));
	if (s > l1_cdiv(stream, 64) / 2) s = l1_cdiv(stream, 64) / 2;
	p.splits = (int)(s < 1 ? 1 : s > 16 ? 16 : s);
	return p;
}

L1MaskedPlan plan_fwd(const l1attn_masked_desc* d)
{
	return plan_of(table_of(d->dtype), d->T, d->S, d->B * d->H, d, false, true);
}
L1MaskedPlan plan_q(const l1attn_masked_desc* d)
{
	return plan_of(table_of(d->dtype), d->T, d->S, d->B * d->H, d, true, false);
}
L1MaskedPlan plan_k(const l1attn_masked_desc* d)
{
	return plan_of(table_of(d->dtype), d->S, d->T, d->B * d->Hk, d, true, true);
}

}  // namespace

extern "C" {

size_t l1attn_masked_fwd_workspace_bytes(const l1attn_masked_desc* desc)
{
	if (check_desc(desc)) return 0;
	const L1MaskedPlan p = plan_fwd(desc);
	return p.splits > 1 ? (size_t)p.splits * desc->B * desc->T * desc->H * ((desc->Wv + 3) / 4 * 4 + 1) * sizeof(float) : 0;
}

int l1attn_masked_fwd(const l1attn_masked_desc* desc, const void* q, const void* k, const void* v, void* o, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream)
{
	const int rc = check_desc(desc);
	if (rc) return rc == 1 ? L1ATTN_OK : rc;
	if (!q || !k || !v || !o) return L1ATTN_ERR_ARG;
	const size_t need = l1attn_masked_fwd_workspace_bytes(desc);
	if (need && (!workspace || workspace_bytes < need)) return L1ATTN_ERR_WORKSPACE;
	L1MaskedArgs A = args_of(desc, q, k, v, o);
	if ((uintptr_t)A.rest & 15) A.vec &= ~8;
	return table_of(desc->dtype).fwd(A, plan_fwd(desc), q, k, v, o, lse, need ? (float*)workspace : nullptr, (hipStream_t)stream);
}

// D of each query row, and the larger of the two sides' splits (one side after the other uses them)
size_t l1attn_masked_bwd_workspace_bytes(const l1attn_masked_desc* desc)
{
	if (check_desc(desc)) return 0;
	const size_t rows = l1_align_up((size_t)(desc->B * desc->T * desc->H) * sizeof(float), 256);
	const L1MaskedPlan a = plan_q(desc), b = plan_k(desc);
	const size_t nq = a.splits > 1 ? (size_t)a.splits * desc->B * desc->T * desc->H * desc->W * sizeof(float) : 0;
	const size_t nk = b.splits > 1 ? (size_t)b.splits * desc->B * desc->S * desc->Hk * (desc->W + desc->Wv) * sizeof(float) : 0;
	return rows + (nq > nk ? nq : nk);
}

int l1attn_masked_bwd(const l1attn_masked_desc* desc, const void* q, const void* k, const void* v, const void* o, const float* lse,
                      const void* d_o, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream)
{
	const int rc = check_desc(desc);
	if (rc < 0) return rc;
	if (desc->B * desc->S == 0) return L1ATTN_OK;
	if (!k || !v || !dk || !dv) return L1ATTN_ERR_ARG;
	if (rc == 0 && (!q || !o || !lse || !d_o || !dq)) return L1ATTN_ERR_ARG;
	if (workspace_bytes < l1attn_masked_bwd_workspace_bytes(desc) || (rc == 0 && !workspace)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	if (rc == 1) {  // keys that no query reads
		const int64_t half = desc->dtype == 0 ? 2 : 1, nk = desc->B * desc->S * desc->Hk * desc->W * half, nv = nk / desc->W * desc->Wv;
		hipLaunchKernelGGL(masked_zero, dim3(zero_blocks(nk)), dim3(256), 0, st, (uint16_t*)dk, nk);
		L1_LAUNCH_CHECK();
		hipLaunchKernelGGL(masked_zero, dim3(zero_blocks(nv)), dim3(256), 0, st, (uint16_t*)dv, nv);
		L1_LAUNCH_CHECK();
		return L1ATTN_OK;
	}
	L1MaskedArgs A = args_of(desc, q, k, v, d_o);
	const L1MaskedTable& t = table_of(desc->dtype);
	const int64_t rows = desc->B * desc->T * desc->H;
	float* D = (float*)workspace;
	float* part = (float*)((char*)workspace + l1_align_up((size_t)rows * sizeof(float), 256));
	int e = t.rows(d_o, o, A.rest, D, rows, A.Wv, st);
	if (e == L1ATTN_OK) e = t.side_q(A, plan_q(desc), q, k, v, d_o, lse, D, dq, part, st);
	if (e == L1ATTN_OK) e = t.side_k(A, plan_k(desc), q, k, v, d_o, lse, D, dk, dv, part, st);
	return e;
}

}  // extern "C"
