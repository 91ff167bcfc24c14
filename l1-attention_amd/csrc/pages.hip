// Pages of the 8-bit cache: what sequences hold them, and what tokens they hold.  Integer work on small arrays, bound by
// launches and latency, except for the copies of compact().
//
// A page belongs to `refs` sequences; free pages lie on a stack (free_pages[0, n_free), the top is taken first).  Everything
// that decides where something goes is done by one workgroup or by prefix sums, in the order of the call's rows and of the page
// numbers, so that the same calls give the same tables; the only atomics count references, where the order has no effect.
// Numbers that the device holds (tables, lists of the call) are checked before they are used as an index.
#include "paged.h"

namespace {

constexpr int kRows = 1024;   // rows of a call: one workgroup looks at all of them
constexpr int kChunk = 4096;  // pages that a workgroup of the scans looks at
constexpr int kOne = 4;       // chunks that one workgroup looks at by itself

// inclusive sum over the workgroup's threads (`total`: of all of them); tmp: one int for each wave
__device__ __forceinline__ int block_scan(int x, int* tmp, int& total)
{
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
	for (int m = 1; m < 64; m <<= 1) {
		const int y = __shfl_up(x, m);
		if (lane >= m) x += y;
	}
	__syncthreads();
	if (lane == 63) tmp[wave] = x;
	__syncthreads();
	int before = 0;
	total = 0;
	for (int w = 0; w < waves; w++) {
		if (w < wave) before += tmp[w];
		total += tmp[w];
	}
	return x + before;
}

// Whether x is among ids[0, b).  Sixteen of them a step, the same ones for all threads: one after the other, each read's latency
// counts.
__device__ __forceinline__ bool named_before(const int* ids, int b, int x)
{
	bool found = false;
	for (int c = 0; c < b && !found; c += 16) {
#pragma unroll
		for (int u = 0; u < 16; u += 4) {
			const int4 y = *reinterpret_cast<const int4*>(ids + c + u);
			found |= (c + u < b && y.x == x) | (c + u + 1 < b && y.y == x) | (c + u + 2 < b && y.z == x) | (c + u + 3 < b && y.w == x);
		}
	}
	return found;
}

// The row that entry b of a call names, or -1: out of range, or named before.  ids: one int for each row, filled here.
__device__ __forceinline__ int named_once(const int32_t* seqs, int b, int B, int rows, int* ids)
{
	const int s = b < B ? (seqs ? seqs[b] : b) : -1;
	ids[b] = s;
	__syncthreads();
	return b < B && s >= 0 && s < rows && !(seqs && named_before(ids, b, s)) ? s : -1;
}

// What an append() takes, by one workgroup, a thread for each of its rows: where each row's tokens go and which pages they get.
// A chain of dependent reads and scans: 5.5 us for 64 rows.
// plan[b] = {sequence or -1, first place, tokens, the page to copy from or -1}; take[b][j]: the page that holds the j-th page
// of the row's new tokens.
__global__ void __launch_bounds__(kRows) cache_take(L1Cache C, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, int B, int n,
                                                    int J, uint8_t* __restrict__ served, int4* __restrict__ plan, int32_t* __restrict__ take)
{
	__shared__ __align__(16) int ids[kRows], first[kRows], held[kRows], fresh_page[kRows];
	__shared__ int tmp[16];
	const int b = threadIdx.x;
	const int s = named_once(seqs, b, B, C.rows, ids);
	const int top = min(max(*C.n_free, 0), C.N);
	int start = 0, cnt = 0, last = -1, fresh = 0;
	bool fits = false, share = false;
	if (s >= 0) {
		start = C.lens[s];
		cnt = counts ? min(max(counts[b], 0), n) : n;
		fits = start >= 0 && (int64_t)start + cnt <= (int64_t)C.M * C.P;
		if (fits && cnt > 0) {
			if (start % C.P) {
				last = C.table[(int64_t)s * C.M + start / C.P];
				if (last < 0 || last >= C.N) fits = false;
				else share = C.refs[last] > 1;
			}
			fresh = (start + cnt + C.P - 1) / C.P - (start + C.P - 1) / C.P;
		}
	}
	int need = fits ? fresh + share : 0, total;
	const int upto = block_scan(need, tmp, total);
	const bool ok = fits && (need == 0 || upto <= top);  // once the pool is empty, no later row that needs a page is served
	if (!ok) { need = 0; cnt = 0; share = false; }
	block_scan(need, tmp, total);
	if (b < B) {
		served[b] = ok;
		plan[b] = make_int4(ok ? s : -1, start, cnt, share ? last : -1);
	}
	first[b] = upto - need;                          // the row's first page below the top of the stack
	fresh_page[b] = start % C.P == 0 || share;       // whether the page of its first token is a new one
	held[b] = cnt > 0 ? (start + cnt + C.P - 1) / C.P - start / C.P : 0;
	ids[b] = last;
	__syncthreads();
	for (int64_t x = b; x < (int64_t)B * J; x += blockDim.x) {
		const int r = (int)(x / J), j = (int)(x % J);
		int page = -1;
		if (j < held[r]) {
			if (j == 0 && !fresh_page[r]) page = ids[r];
			else {
				page = C.free[top - 1 - (first[r] + j - (fresh_page[r] ? 0 : 1))];
				if (page >= 0 && page < C.N) C.refs[page] = 1;
				else page = -1;
			}
		}
		take[x] = page;
	}
	if (ok) C.lens[s] = start + cnt;
	if (!__syncthreads_or(share)) {
		if (b == 0) *C.n_free = top - total;
		return;
	}
	// the shared pages that were written to lose a holder; those that lose the last one are free again, in ascending order
	const bool freed = share && atomicSub(&C.refs[last], 1) == 1;
	held[b] = freed ? last : -1;
	__syncthreads();
	int gone;
	block_scan(freed, tmp, gone);
	if (freed) {
		int at = top - total;
		for (int c = 0; c < B; c++) at += held[c] >= 0 && held[c] < last;
		C.free[at] = last;
	}
	if (b == 0) *C.n_free = top - total + gone;
}

// Which forks are possible, by one workgroup: child b gets the length of its parent as it was before the call.
__global__ void __launch_bounds__(kRows) cache_fork(L1Cache C, const int32_t* __restrict__ parents, const int32_t* __restrict__ children, int B,
                                                    uint8_t* __restrict__ served, int32_t* __restrict__ held)
{
	__shared__ __align__(16) int ids[kRows];
	const int b = threadIdx.x;
	const int child = named_once(children, b, B, C.rows, ids);
	const int parent = b < B ? parents[b] : -1;
	const bool ok = child >= 0 && parent >= 0 && parent < C.rows && parent != child && C.lens[child] == 0;
	const int len = ok ? min(max(C.lens[parent], 0), C.M * C.P) : 0;
	__syncthreads();
	if (ok) C.lens[child] = len;
	if (b < B) {
		served[b] = ok;
		held[b] = (len + C.P - 1) / C.P;
	}
}

__global__ void __launch_bounds__(256) cache_fork_rows(L1Cache C, const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
                                                       const uint8_t* __restrict__ served, const int32_t* __restrict__ held)
{
	const int b = blockIdx.x;
	if (!served[b]) return;
	const int32_t* from = C.table + (int64_t)parents[b] * C.M;
	int32_t* to = C.table + (int64_t)children[b] * C.M;
	for (int j = blockIdx.y * 256 + threadIdx.x; j < held[b]; j += 256 * gridDim.y) {
		const int page = from[j];
		if (page < 0 || page >= C.N) continue;
		to[j] = page;
		atomicAdd(&C.refs[page], 1);
	}
}

// A row gives back the pages behind its kept length; a page that loses its last holder is marked (refs -1) for the scan.
__global__ void __launch_bounds__(256) cache_drop(L1Cache C, const int32_t* __restrict__ seqs, const int32_t* __restrict__ keep, int B)
{
	__shared__ int dup;
	const int b = blockIdx.x, s = seqs ? seqs[b] : b;
	if (threadIdx.x == 0) dup = 0;
	__syncthreads();
	if (seqs)
		for (int c = threadIdx.x; c < b; c += 256)
			if (seqs[c] == s) dup = 1;
	__syncthreads();
	if (dup || s < 0 || s >= C.rows) return;
	const int len = min(max(C.lens[s], 0), C.M * C.P);
	const int kept = keep ? min(max(keep[b], 0), len) : 0;
	int32_t* row = C.table + (int64_t)s * C.M;
	for (int j = (kept + C.P - 1) / C.P + threadIdx.x; j < (len + C.P - 1) / C.P; j += 256) {
		const int page = row[j];
		if (page < 0 || page >= C.N) continue;
		row[j] = -1;
		if (atomicSub(&C.refs[page], 1) == 1) C.refs[page] = -1;
	}
	__syncthreads();
	if (threadIdx.x == 0) C.lens[s] = kept;
}

// pages of each chunk for which refs is -1 (FREED) or positive (the pages in use)
template <bool FREED>
__global__ void __launch_bounds__(kRows) cache_count(L1Cache C, int32_t* __restrict__ counts)
{
	__shared__ int tmp[16];
	int n = 0, total;
	for (int u = 0; u < kChunk / kRows; u++) {
		const int p = blockIdx.x * kChunk + threadIdx.x * (kChunk / kRows) + u;
		if (p < C.N) n += FREED ? C.refs[p] == -1 : C.refs[p] > 0;
	}
	block_scan(n, tmp, total);
	if (threadIdx.x == 0) counts[blockIdx.x] = total;
}

// sum of counts[0, upto), by the whole workgroup
__device__ __forceinline__ int sum_before(const int32_t* counts, int upto, int* tmp)
{
	int n = 0, total;
	for (int c = threadIdx.x; c < upto; c += blockDim.x) n += counts[c];
	block_scan(n, tmp, total);
	return total;
}

// the marked pages onto the stack, in ascending order
__global__ void __launch_bounds__(kRows) cache_push(L1Cache C, const int32_t* __restrict__ counts, const int32_t* __restrict__ top_before, int32_t* __restrict__ top_after)
{
	__shared__ int tmp[16];
	const int before = sum_before(counts, blockIdx.x, tmp);
	int flag[kChunk / kRows], n = 0, total;
	const int p0 = blockIdx.x * kChunk + threadIdx.x * (kChunk / kRows);
#pragma unroll
	for (int u = 0; u < kChunk / kRows; u++) {
		flag[u] = p0 + u < C.N && C.refs[p0 + u] == -1;
		n += flag[u];
	}
	const int top = min(max(*top_before, 0), C.N);
	int at = top + before + block_scan(n, tmp, total) - n;
#pragma unroll
	for (int u = 0; u < kChunk / kRows; u++)
		if (flag[u]) {
			C.refs[p0 + u] = 0;
			if (at < C.N) C.free[at] = p0 + u;
			at++;
		}
	if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *top_after = min(top + before + total, C.N);
}

// The same by one workgroup, chunk after chunk, instead of three launches, for pools of up to kOne chunks.
__global__ void __launch_bounds__(kRows) cache_push_one(L1Cache C, int chunks)
{
	__shared__ int tmp[16];
	int top = min(max(*C.n_free, 0), C.N);
	for (int chunk = 0; chunk < chunks; chunk++) {
		const int p0 = chunk * kChunk + threadIdx.x * (kChunk / kRows);
		int flag[kChunk / kRows], n = 0, total;
#pragma unroll
		for (int u = 0; u < kChunk / kRows; u++) {
			flag[u] = p0 + u < C.N && C.refs[p0 + u] == -1;
			n += flag[u];
		}
		int at = top + block_scan(n, tmp, total) - n;
#pragma unroll
		for (int u = 0; u < kChunk / kRows; u++)
			if (flag[u]) {
				C.refs[p0 + u] = 0;
				if (at < C.N) C.free[at] = p0 + u;
				at++;
			}
		top = min(top + total, C.N);
	}
	__syncthreads();
	if (threadIdx.x == 0) *C.n_free = top;
}

__global__ void cache_copy_int(int32_t* to, const int32_t* from) { *to = *from; }

// compact(), first part: the pages in use in ascending order (live), the holes before n_live, and the free stack that is left.
__global__ void __launch_bounds__(kRows) cache_order(L1Cache C, const int32_t* __restrict__ counts, int chunks, int32_t* __restrict__ live,
                                                     int32_t* __restrict__ holes, int32_t* __restrict__ map, int32_t* __restrict__ sums, int32_t* __restrict__ how_many)
{
	__shared__ int tmp[16];
	const int before = sum_before(counts, blockIdx.x, tmp), n_live = sum_before(counts, chunks, tmp);
	int flag[kChunk / kRows], n = 0, total;
	const int p0 = blockIdx.x * kChunk + threadIdx.x * (kChunk / kRows);
#pragma unroll
	for (int u = 0; u < kChunk / kRows; u++) {
		flag[u] = p0 + u < C.N && C.refs[p0 + u] > 0;
		n += flag[u];
	}
	int rank = before + block_scan(n, tmp, total) - n;  // pages in use before p0
#pragma unroll
	for (int u = 0; u < kChunk / kRows; u++) {
		const int p = p0 + u;
		if (p >= C.N) break;
		if (p == n_live) sums[1] = n_live - rank;  // as many holes before n_live as pages in use behind it
		map[p] = p;
		if (flag[u]) live[rank++] = p;
		else if (p < n_live) holes[p - rank] = p;
		if (p >= n_live) C.free[C.N - 1 - p] = p;  // the lowest free page on top
	}
	if (blockIdx.x == 0 && threadIdx.x == 0) {
		sums[0] = n_live;
		*how_many = n_live;
		if (n_live == C.N) sums[1] = 0;
		*C.n_free = C.N - n_live;
	}
}

// second part: page r of those behind n_live moves into the r-th hole; bound by the copy (54 us for 205 MB read and written, 43 at a
// large copy's rate)
__global__ void __launch_bounds__(256) cache_move(L1Cache C, const int32_t* __restrict__ live, const int32_t* __restrict__ holes,
                                                  int32_t* __restrict__ map, const int32_t* __restrict__ sums)
{
	const int n_live = sums[0], n = sums[1];
	const int64_t kb = (int64_t)C.Hk * C.P * C.pk / 16, vb = (int64_t)C.Hk * C.P * C.pv / 16;
	for (int r = blockIdx.x; r < n; r += gridDim.x) {
		const int to = holes[r], from = live[n_live - n + r];
		const uint4 *k0 = reinterpret_cast<const uint4*>(C.k) + from * kb, *v0 = reinterpret_cast<const uint4*>(C.v) + from * vb;
		uint4 *k1 = reinterpret_cast<uint4*>(C.k) + to * kb, *v1 = reinterpret_cast<uint4*>(C.v) + to * vb;
		for (int64_t x = threadIdx.x; x < kb; x += 256) k1[x] = k0[x];
		for (int64_t x = threadIdx.x; x < vb; x += 256) v1[x] = v0[x];
		for (int h = threadIdx.x; h < C.Hk; h += 256) {
			C.ks[(int64_t)to * C.Hk + h] = C.ks[(int64_t)from * C.Hk + h];
			C.vs[(int64_t)to * C.Hk + h] = C.vs[(int64_t)from * C.Hk + h];
		}
		if (threadIdx.x == 0) {
			C.refs[to] = C.refs[from];
			C.refs[from] = 0;
			map[from] = to;
		}
	}
}

// third part: the tables
__global__ void __launch_bounds__(256) cache_rename(L1Cache C, const int32_t* __restrict__ map)
{
	for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < (int64_t)C.rows * C.M; x += (int64_t)gridDim.x * 256) {
		const int page = C.table[x];
		if (page >= 0 && page < C.N) C.table[x] = map[page];
	}
}

// ------------------------------------------------------------------------------------------------------------ new tokens

template <typename ST> __device__ __forceinline__ float value(ST x) { return (float)x; }

// Tokens into pages: a workgroup for each page of each row and head, keys (z 0) and values (z 1).  A value is read once, into
// registers, from where it goes into the scale and, behind the workgroup's barrier, into its code: the loads of a workgroup wait for
// the chain plan, page, and its stores for all of them (29 us for 8 rows of up to 2000 tokens, 8 heads, W 128, bfloat16: 48 MB
// read, 24 MB written, 15.5 us at a large copy's rate; 4.9 us for one token of 64 rows).  The page's scale becomes the larger of
// what it was (if it held tokens) and the new tokens' largest magnitude times 1/127 (in float32); if it grew, or the page is a
// copy of a shared one, the codes that were there are written again.  A value that is not finite does not count for the
// scale: infinities are coded as +-127, NaN as 0.  G: elements a thread holds side by side.
template <typename ST, int G>
__global__ void __launch_bounds__(256) cache_write(L1Cache C, const ST* __restrict__ kx, const ST* __restrict__ vx, int n, int J,
                                                   const int4* __restrict__ plan, const int32_t* __restrict__ take)
{
	constexpr int U = 64 * 128 / 256 / G;  // groups of a thread in the largest page
	__shared__ float wave_top[4];
	const int r = blockIdx.x / J, j = blockIdx.x % J, h = blockIdx.y, isv = blockIdx.z, tid = threadIdx.x;
	const int4 pl = plan[r];
	const int page = take[blockIdx.x];
	if (pl.x < 0 || page < 0) return;
	const int start = pl.y, end = pl.y + pl.z, base = (start / C.P + j) * C.P;
	const int W = isv ? C.Wv : C.W, pitch = isv ? C.pv : C.pk;
	const int64_t bytes = (int64_t)C.P * pitch;
	const ST* x = isv ? vx : kx;
	int8_t* pages = isv ? C.v : C.k;
	float* scales = isv ? C.vs : C.ks;
	const bool copy = j == 0 && pl.w >= 0;
	const int src = copy ? pl.w : page;
	const int8_t* from = pages + ((int64_t)src * C.Hk + h) * bytes;
	int8_t* to = pages + ((int64_t)page * C.Hk + h) * bytes;
	if (h == 0 && !isv && tid == 0) C.table[(int64_t)pl.x * C.M + start / C.P + j] = page;

	const int groups = pitch / G, all = C.P * groups;
	float val[U][G];
	float top = 0.f;
#pragma unroll
	for (int u = 0; u < U; u++) {
		const int at = tid + 256 * u;
		if (at >= all) break;
		const int t = at / groups, w = (at % groups) * G, place = base + t;
		if (place < start || place >= end) continue;
		const ST* row = x + (((int64_t)r * n + place - start) * C.Hk + h) * W;
		ST in[G];
		if (w < W) {
			if constexpr (G > 1) __builtin_memcpy(in, __builtin_assume_aligned(row + w, 16), sizeof(in));
			else in[0] = row[w];
		}
#pragma unroll
		for (int e = 0; e < G; e++) {
			val[u][e] = w < W ? value(in[e]) : 0.f;
			const float m = __builtin_fabsf(val[u][e]);
			top = m <= 3.402823466e38f ? fmaxf(top, m) : top;
		}
	}
#pragma unroll
	for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
	if ((tid & 63) == 0) wave_top[tid >> 6] = top;
	const float held = base < start ? scales[(int64_t)src * C.Hk + h] : 0.f;
	__syncthreads();
	top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
	const float now = fmaxf(__builtin_fabsf(held), top * (1.f / 127.f));  // a scale of a pool that the caller filled may be negative
	const float ratio = now > 0.f ? held / now : 0.f, div = now > 0.f ? now : 1.f;
	const bool again = base < start && (copy || ratio != 1.f);
#pragma unroll
	for (int u = 0; u < U; u++) {
		const int at = tid + 256 * u;
		if (at >= all) break;
		const int t = at / groups, w = (at % groups) * G, place = base + t;
		if (place >= end || (place < start && !again)) continue;
		int8_t code[G];
		if (place < start) {
			__builtin_memcpy(code, from + t * pitch + w, G);
#pragma unroll
			for (int e = 0; e < G; e++) code[e] = (int8_t)fminf(rintf((float)code[e] * ratio), 127.f);  // -128 has no opposite
		} else {
#pragma unroll
			for (int e = 0; e < G; e++) {
				const float y = val[u][e];
				code[e] = y == y ? (int8_t)fminf(fmaxf(rintf(y / div), -127.f), 127.f) : (int8_t)0;
			}
		}
		__builtin_memcpy(to + t * pitch + w, code, G);
	}
	if (tid == 0) scales[(int64_t)page * C.Hk + h] = now;
}

template <typename ST>
int write_tokens(const L1Cache& C, const void* k, const void* v, int B, int n, int J, const int4* plan, const int32_t* take, hipStream_t st)
{
	// eight elements side by side, whole vectors, where both widths are whole eights and the inputs start on 16 bytes
	const dim3 grid((unsigned)(B * J), (unsigned)C.Hk, 2);
	if (C.W % 8 == 0 && C.Wv % 8 == 0 && !(((uintptr_t)k | (uintptr_t)v) & 15))
		hipLaunchKernelGGL((cache_write<ST, 8>), grid, dim3(256), 0, st, C, (const ST*)k, (const ST*)v, n, J, plan, take);
	else hipLaunchKernelGGL((cache_write<ST, 1>), grid, dim3(256), 0, st, C, (const ST*)k, (const ST*)v, n, J, plan, take);
	L1_LAUNCH_CHECK();
	return L1ATTN_OK;
}

int pages_of(int64_t n, int P) { return (int)((n + P - 1) / P) + 1; }

}  // namespace

extern "C" {

size_t l1attn_cache_append_workspace_bytes(const l1attn_cache* cache, int64_t B, int64_t n)
{
	L1Cache C;
	if (l1_cache_args(cache, &C) || B < 0 || B > kRows || n < 0 || n > (1 << 28)) return 0;
	return (size_t)B * (sizeof(int4) + (size_t)pages_of(n, C.P) * sizeof(int32_t));
}

int l1attn_cache_append(const l1attn_cache* cache, int dtype, const void* k, const void* v, const int32_t* seqs, const int32_t* counts,
                        int64_t B, int64_t n, uint8_t* served, void* workspace, size_t workspace_bytes, void* stream)
{
	L1Cache C;
	const int rc = l1_cache_args(cache, &C);
	if (rc != L1ATTN_OK) return rc;
	if (B < 0 || n < 0 || dtype < 0 || dtype > 2) return L1ATTN_ERR_ARG;
	if (B > kRows || n > (1 << 28)) return L1ATTN_ERR_RANGE;
	if (B == 0) return L1ATTN_OK;
	if (!served || (n && (!k || !v))) return L1ATTN_ERR_ARG;
	const int J = pages_of(n, C.P);
	if ((int64_t)B * J > 0xffffff) return L1ATTN_ERR_RANGE;  // 2^32 - 1 threads of the second launch: refused before the first one
	if (!workspace || workspace_bytes < l1attn_cache_append_workspace_bytes(cache, B, n)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	int4* plan = (int4*)workspace;
	int32_t* take = (int32_t*)(plan + B);
	hipLaunchKernelGGL(cache_take, dim3(1), dim3((unsigned)l1_align_up((size_t)B, 64)), 0, st, C, seqs, counts, (int)B, (int)n, J, served, plan, take);
	L1_LAUNCH_CHECK();
	if (n == 0) return L1ATTN_OK;
	if (dtype == 0) return write_tokens<float>(C, k, v, (int)B, (int)n, J, plan, take, st);
	if (dtype == 1) return write_tokens<_Float16>(C, k, v, (int)B, (int)n, J, plan, take, st);
	return write_tokens<__bf16>(C, k, v, (int)B, (int)n, J, plan, take, st);
}

int l1attn_cache_fork(const l1attn_cache* cache, const int32_t* parents, const int32_t* children, int64_t B, uint8_t* served,
                      void* workspace, size_t workspace_bytes, void* stream)
{
	L1Cache C;
	const int rc = l1_cache_args(cache, &C);
	if (rc != L1ATTN_OK) return rc;
	if (B < 0) return L1ATTN_ERR_ARG;
	if (B > kRows) return L1ATTN_ERR_RANGE;
	if (B == 0) return L1ATTN_OK;
	if (!parents || !children || !served) return L1ATTN_ERR_ARG;
	if (!workspace || workspace_bytes < (size_t)B * sizeof(int32_t)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	hipLaunchKernelGGL(cache_fork, dim3(1), dim3((unsigned)l1_align_up((size_t)B, 64)), 0, st, C, parents, children, (int)B, served, (int32_t*)workspace);
	L1_LAUNCH_CHECK();
	hipLaunchKernelGGL(cache_fork_rows, dim3((unsigned)B, (unsigned)min((int64_t)64, l1_cdiv(C.M + 1, 1024))), dim3(256), 0, st, C, parents, children, served, (const int32_t*)workspace);
	L1_LAUNCH_CHECK();
	return L1ATTN_OK;
}

size_t l1attn_cache_free_workspace_bytes(const l1attn_cache* cache)
{
	L1Cache C;
	return l1_cache_args(cache, &C) ? 0 : (size_t)(l1_cdiv(C.N, kChunk) + 2) * sizeof(int32_t);
}

int l1attn_cache_free(const l1attn_cache* cache, const int32_t* seqs, const int32_t* keep, int64_t B, void* workspace,
                      size_t workspace_bytes, void* stream)
{
	L1Cache C;
	const int rc = l1_cache_args(cache, &C);
	if (rc != L1ATTN_OK) return rc;
	if (B < 0) return L1ATTN_ERR_ARG;
	if (B > kRows) return L1ATTN_ERR_RANGE;
	if (B == 0 || C.N == 0) return L1ATTN_OK;
	if (!workspace || workspace_bytes < l1attn_cache_free_workspace_bytes(cache)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	const unsigned chunks = (unsigned)l1_cdiv(C.N, kChunk);
	int32_t* counts = (int32_t*)workspace;
	hipLaunchKernelGGL(cache_drop, dim3((unsigned)B), dim3(256), 0, st, C, seqs, keep, (int)B);
	L1_LAUNCH_CHECK();
	if (chunks <= kOne) {
		hipLaunchKernelGGL(cache_push_one, dim3(1), dim3(kRows), 0, st, C, (int)chunks);
		L1_LAUNCH_CHECK();
		return L1ATTN_OK;
	}
	hipLaunchKernelGGL(cache_count<true>, dim3(chunks), dim3(kRows), 0, st, C, counts);
	L1_LAUNCH_CHECK();
	hipLaunchKernelGGL(cache_push, dim3(chunks), dim3(kRows), 0, st, C, counts, C.n_free, counts + chunks);
	L1_LAUNCH_CHECK();
	hipLaunchKernelGGL(cache_copy_int, dim3(1), dim3(1), 0, st, C.n_free, counts + chunks);
	L1_LAUNCH_CHECK();
	return L1ATTN_OK;
}

size_t l1attn_cache_compact_workspace_bytes(const l1attn_cache* cache)
{
	L1Cache C;
	return l1_cache_args(cache, &C) ? 0 : ((size_t)C.N * 3 + (size_t)l1_cdiv(C.N, kChunk) + 4) * sizeof(int32_t);
}

int l1attn_cache_compact(const l1attn_cache* cache, int32_t* live, void* workspace, size_t workspace_bytes, void* stream)
{
	L1Cache C;
	const int rc = l1_cache_args(cache, &C);
	if (rc != L1ATTN_OK) return rc;
	if (!live) return L1ATTN_ERR_ARG;
	if (!workspace || workspace_bytes < l1attn_cache_compact_workspace_bytes(cache)) return L1ATTN_ERR_WORKSPACE;
	hipStream_t st = (hipStream_t)stream;
	const unsigned chunks = (unsigned)l1_cdiv(C.N, kChunk);
	int32_t* sums = (int32_t*)workspace;
	int32_t* order = sums + 4;
	int32_t* holes = order + C.N;
	int32_t* map = holes + C.N;
	int32_t* counts = map + C.N;
	if (C.N == 0) return L1ATTN_ERR_ARG;
	hipLaunchKernelGGL(cache_count<false>, dim3(chunks), dim3(kRows), 0, st, C, counts);
	L1_LAUNCH_CHECK();
	hipLaunchKernelGGL(cache_order, dim3(chunks), dim3(kRows), 0, st, C, counts, (int)chunks, order, holes, map, sums, live);
	L1_LAUNCH_CHECK();
	hipLaunchKernelGGL(cache_move, dim3(2048), dim3(256), 0, st, C, order, holes, map, sums);
	L1_LAUNCH_CHECK();
	if ((int64_t)C.rows * C.M) {
		const int64_t blocks = l1_cdiv((int64_t)C.rows * C.M, 256), most = 1 << 23;  // a grid has 2^32 - 1 threads at most
		hipLaunchKernelGGL(cache_rename, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, C, map);
		L1_LAUNCH_CHECK();
	}
	return L1ATTN_OK;
}

}  // extern "C"
