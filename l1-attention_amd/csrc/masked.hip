// Masked L1 attention for gfx950, forward and backward, float32 / float16 / bfloat16, grouped key heads:
//
//   a[t,s] = -1/sqrt(W) * sum_w |q[t,w] - k[s,w]|         c = cap * tanh(a / cap)      (cap > 0, else c = a)
//   x[t,s] = c - slope[h] * |i - s|                        i = S - T + t, the query's place among the S tokens
//   p[t,s] = exp(x) / (1 + sum_s exp(x))                   over the visible s; the 1 is the no-op logit
//   o[t]   = sum_s p[t,s] * v[s]
//   visible: (not causal or s <= i or s < prefix[b]) and (no documents or doc[b,s] == doc[b,i] >= 0)
//
// Every logit is <= 0 (slopes are not negative) and the no-op logit is 0, so a row needs no running maximum: exp(x) <= 1,
// the denominator is >= 1, and a row that sees nothing comes out as zero by itself.
//
// One wavefront owns 32 rows ("owners": queries in the forward and in the gradient of q, keys in that of k and v) and walks
// the other side ("stream") in tiles of 64, which the waves of a workgroup share through LDS.  Three parts of a tile use
// three maps of its 32 x 64 pairs onto the lanes, joined by a wave-private LDS scratch of 32 x 32 values at a time:
//   scores   lane (i,j) = (lane & 7, lane >> 3) holds owners i + 8a (a < 4) and stream rows j + 8b (b < 8): 12 LDS reads of
//            16 bytes feed 32 pairs; the L1 distance is no contraction, so this is vector-ALU work
//   products p*v, do*v: matrix instructions; column order of a tile: c = 32*(b/4) + 4*j + b%4, so that a lane's four values
//            of one half of the tile are neighbours
//   signs    lane = column w; the 32 owners' sums live in registers, the score gradients come as broadcast LDS reads
#include "common.h"
#include "masked.h"
#include <math.h>

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kOwn = 32;        // owner rows of a wave
constexpr int kTile = 64;       // stream rows of a tile
constexpr int kPad = 36;        // floats in a row of the scratch: 9 chunks of 16 bytes, odd, so rows spread over the banks
constexpr int kClasses = 1024;  // tiles whose visibility is worked out at a time

// floats in an LDS row of n: whole 16-byte chunks, an odd number of them (neighbouring rows start in different banks)
__host__ __device__ __forceinline__ int row_floats(int n) { return (((n + 3) / 4) | 1) * 4; }

template <typename ST> __device__ __forceinline__ float to_f(ST x) { return (float)x; }

// up to four elements of a row from memory; elements past `n` are zero.  vec: the row starts on 16 bytes (float32) or 8
template <typename ST>
__device__ __forceinline__ f4 load4(const ST* __restrict__ p, int n, bool vec)
{
	f4 r = {0.f, 0.f, 0.f, 0.f};
	if (vec && n >= 4) {
		if constexpr (sizeof(ST) == 4) {
			r = *reinterpret_cast<const f4*>(p);
		} else {
			const uint2 raw = *reinterpret_cast<const uint2*>(p);
			ST h[4];
			__builtin_memcpy(h, &raw, 8);
#pragma unroll
			for (int e = 0; e < 4; e++) r[e] = to_f(h[e]);
		}
	} else {
#pragma unroll
		for (int e = 0; e < 4; e++)
			if (e < n) r[e] = to_f(p[e]);
	}
	return r;
}

// stream row r of a tile <-> its place c in the order of the products
__device__ __forceinline__ int col_of(int r) { return 32 * (r >> 5) + 4 * (r & 7) + ((r >> 3) & 3); }
__device__ __forceinline__ int row_of(int c) { return ((c >> 2) & 7) + 8 * (4 * (c >> 5) + (c & 3)); }

// rows [r0, r0 + n) of x [L, heads, width] (x points at the head) into LDS rows of `stride` floats; whether a value read was not finite
template <typename ST, bool PERMUTE>
__device__ __forceinline__ bool stage(float* __restrict__ dst, const ST* __restrict__ x, int r0, int n, int L, int64_t pitch,
                                      int width, int stride, bool vec, int tid, int threads)
{
	const int chunks = (width + 3) >> 2, j = tid & 7;
	bool bad = false;
	for (int r = tid >> 3; r < n; r += threads >> 3) {
		const bool in = r0 + r < L;
		const ST* row = x + (int64_t)(r0 + r) * pitch;
		float* to = dst + (PERMUTE ? col_of(r) : r) * stride;
		for (int c = j; c < chunks; c += 8) {
			f4 x = {0.f, 0.f, 0.f, 0.f};
			if (in) x = load4(row + 4 * c, width - 4 * c, vec);
			*reinterpret_cast<f4*>(to + 4 * c) = x;
#pragma unroll
			for (int e = 0; e < 4; e++) bad |= !(__builtin_fabsf(x[e]) <= 3.402823466e38f);
		}
	}
	return bad;
}

// a wave's own stores to LDS before its loads of them (LDS works a wave's accesses off in order; this keeps the compiler to it)
__device__ __forceinline__ void wave_sync()
{
	__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
	__builtin_amdgcn_wave_barrier();
}

// L1 distances of a wave's 32 x 64 pairs, acc[a][b] of owner i + 8a and stream row j + 8b
__device__ __forceinline__ void distances(const float* __restrict__ own, const float* __restrict__ str, int chunks, int stride,
                                          int i, int j, float (&acc)[4][8])
{
#pragma unroll
	for (int a = 0; a < 4; a++)
#pragma unroll
		for (int b = 0; b < 8; b++) acc[a][b] = 0.f;
	for (int c = 0; c < chunks; c++) {
		f4 o[4];
#pragma unroll
		for (int a = 0; a < 4; a++) o[a] = *reinterpret_cast<const f4*>(own + (i + 8 * a) * stride + 4 * c);
#pragma unroll
		for (int b = 0; b < 8; b++) {
			const f4 s = *reinterpret_cast<const f4*>(str + (j + 8 * b) * stride + 4 * c);
#pragma unroll
			for (int a = 0; a < 4; a++)
#pragma unroll
				for (int e = 0; e < 4; e++) acc[a][b] += __builtin_fabsf(o[a][e] - s[e]);
		}
	}
}

struct Span { int lo, hi; };  // least and largest of the document numbers >= 0 (lo > hi: there is none), over a group of rows

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

// What a tile of the stream is to a workgroup's owners: 0 nothing of it is visible, 1 all of it, 2 some of it.
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

// classes of the tiles [t0, t0 + n) into cls; every thread of the workgroup takes part
template <bool OWNK>
__device__ __forceinline__ void classify(const L1MaskedArgs& A, const int* doc, int prefix, int own_lo, int own_hi, Span own_docs,
                                         bool own_whole, int L, int place0, int t0, int n, unsigned char* cls, int tid, int threads)
{
	if (!doc) {
		for (int t = tid; t < n; t += threads) {
			const int lo = (t0 + t) * kTile, hi = min(lo + kTile, L);
			cls[t] = (unsigned char)place_class<OWNK>(A, prefix, own_lo, own_hi, place0 + lo, place0 + hi - 1, hi - lo == kTile);
		}
		return;
	}
	const int lane = tid & 63;
	for (int t = tid >> 6; t < n; t += threads >> 6) {
		const int lo = (t0 + t) * kTile, hi = min(lo + kTile, L);
		int c = place_class<OWNK>(A, prefix, own_lo, own_hi, place0 + lo, place0 + hi - 1, hi - lo == kTile);
		if (c) {
			const int d = lo + lane < hi ? doc[place0 + lo + lane] : -1;
			if (!__ballot(d >= 0 && d >= own_docs.lo && d <= own_docs.hi)) c = 0;
			else if (!own_whole || own_docs.lo != own_docs.hi || __ballot(d != own_docs.lo)) c = 2;
		}
		if (lane == 0) cls[t] = (unsigned char)c;
	}
}

// What is common to the kernels: where a workgroup's owners lie and what they may see.
struct Block {
	int b, h, hk, own0, nown;    // batch entry, query head, key head, the workgroup's first owner row, rows it has at most
	int own_rows, str_rows;      // rows of the owners' and of the stream's side
	int own_place0, str_place0;  // place of row 0 of either side
};

template <bool OWNK>
__device__ __forceinline__ Span owner_docs(const int* doc, const Block& K, int* shared, int tid, int threads, bool& whole)
{
	// `whole`: every owner row belongs to a document
	int lo = 0x7fffffff, hi = -1, none = 0;
	if (doc)
		for (int r = tid; r < K.nown && K.own0 + r < K.own_rows; r += threads) {
			const int d = doc[K.own_place0 + K.own0 + r];
			if (d >= 0) { lo = min(lo, d); hi = max(hi, d); } else none = 1;
		}
	lo = wave_min(lo); hi = wave_max(hi); none = wave_max(none);
	if ((tid & 63) == 0) { shared[3 * (tid >> 6)] = lo; shared[3 * (tid >> 6) + 1] = hi; shared[3 * (tid >> 6) + 2] = none; }
	__syncthreads();
	for (int w = 0; w < threads >> 6; w++) { lo = min(lo, shared[3 * w]); hi = max(hi, shared[3 * w + 1]); none = max(none, shared[3 * w + 2]); }
	whole = !none;
	return {lo, hi};
}

// one visible pair
__device__ __forceinline__ bool sees(const L1MaskedArgs& A, int prefix, bool docs, int qp, int kp, int qd, int kd)
{
	bool ok = !A.causal || kp <= qp || kp < prefix;
	if (docs) ok = ok && qd == kd && qd >= 0;
	return ok;
}

// LDS of a workgroup, in floats from the front (the same on the host)
struct Layout { int own, str, y, scratch, rows, total; };

__host__ __device__ inline Layout masked_layout(int W, int Wv, int waves)
{
	Layout l;
	l.own = 0;
	l.str = l.own + waves * kOwn * row_floats(W);
	l.y = l.str + kTile * row_floats(W);
	l.scratch = l.y + kTile * row_floats(Wv);
	l.rows = l.scratch + waves * kOwn * kPad;  // per-row data of the stream: documents, lse, D (64 each), 24 words for reductions, classes
	l.total = l.rows + 3 * kTile + 32 + kClasses / 4;
	return l;
}

// acc[tb][wb] += sum over 32 columns c of val[c][16 wb + ..] * p[owner][c]: p in the wave's scratch, the values' columns on
// rows of the result.  With `bad` (values that are not finite in a tile of which some is hidden) a hidden pair's weight of
// zero must not meet them, which a matrix instruction cannot leave out.
template <int NB>
__device__ __forceinline__ void weigh(f4 (&acc)[2][NB], const float* scr, const float* val, int sv, int l16, int g, bool bad)
{
	if (bad) {
		for (int c = 0; c < 32; c++)
#pragma unroll
			for (int tb = 0; tb < 2; tb++) {
				const float p = scr[(l16 + 16 * tb) * kPad + c];
				if (p != 0.f)
#pragma unroll
					for (int wb = 0; wb < NB; wb++)
#pragma unroll
						for (int e = 0; e < 4; e++)
							if (16 * wb + 4 * g + e < sv) acc[tb][wb][e] += p * val[c * sv + 16 * wb + 4 * g + e];
			}
		return;
	}
#pragma unroll
	for (int kc = 0; kc < 2; kc++) {
		f4 pb[2];
#pragma unroll
		for (int tb = 0; tb < 2; tb++) pb[tb] = *reinterpret_cast<const f4*>(scr + (l16 + 16 * tb) * kPad + 16 * kc + 4 * g);
#pragma unroll
		for (int e = 0; e < 4; e++) {
			const float* row = val + (16 * kc + 4 * g + e) * sv + l16;
#pragma unroll
			for (int wb = 0; wb < NB; wb++) {
				const float av = 16 * wb + l16 < sv ? row[16 * wb] : 0.f;
#pragma unroll
				for (int tb = 0; tb < 2; tb++) acc[tb][wb] = __builtin_amdgcn_mfma_f32_16x16x4f32(av, pb[tb][e], acc[tb][wb], 0, 0, 0);
			}
		}
	}
}

// ---------------------------------------------------------------------------------------------------------------- forward

// NB: 16-column blocks of the value width held per wave.  Grid: x = batch * head (heads next to each other go to different
// XCDs and one head's tiles to one), y = owner tiles, the last first: under causality it has the most to do.
template <typename ST, int NB, int THREADS>
__global__ void __launch_bounds__(THREADS) masked_fwd(L1MaskedArgs A, const ST* __restrict__ q, const ST* __restrict__ k,
                                                      const ST* __restrict__ v, ST* __restrict__ o, float* __restrict__ lse)
{
	extern __shared__ float lds[];
	const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
	const int i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
	Block K;
	K.b = blockIdx.x / A.H; K.h = blockIdx.x % A.H; K.hk = K.h / (A.H / A.Hk);
	K.nown = waves * kOwn; K.own0 = (gridDim.y - 1 - blockIdx.y) * K.nown;
	K.own_rows = A.T; K.str_rows = A.S; K.own_place0 = A.S - A.T; K.str_place0 = 0;
	const Layout Y = masked_layout(A.W, A.Wv, waves);
	const int sw = row_floats(A.W), sv = row_floats(A.Wv), chunks = (A.W + 3) >> 2;
	float* own = lds + Y.own + wave * kOwn * sw;
	float* str = lds + Y.str;
	float* val = lds + Y.y;
	float* scr = lds + Y.scratch + wave * kOwn * kPad;
	int* docs = reinterpret_cast<int*>(lds + Y.rows);
	unsigned char* cls = reinterpret_cast<unsigned char*>(lds + Y.rows + 3 * kTile + 32);
	const int* doc = A.doc ? A.doc + (int64_t)K.b * A.S : nullptr;
	const int prefix = A.prefix ? A.prefix[K.b] : 0;
	const float slope = A.has_slopes ? A.slopes[K.h] : 0.f;
	const int64_t qpitch = (int64_t)A.H * A.W, kpitch = (int64_t)A.Hk * A.W, vpitch = (int64_t)A.Hk * A.Wv;
	const ST* qh = q + ((int64_t)K.b * A.T * A.H + K.h) * A.W;
	const ST* kh = k + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.W;
	const ST* vh = v + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.Wv;

	stage<ST, false>(own, qh, K.own0 + wave * kOwn, kOwn, A.T, qpitch, A.W, sw, A.vec & 1, lane, 64);
	// value columns behind the width are multiplied too: they have to be finite
	for (int x = tid; x < kTile * (sv - A.Wv); x += threads) val[(x / (sv - A.Wv)) * sv + A.Wv + x % (sv - A.Wv)] = 0.f;
	bool whole;
	const Span od = owner_docs<false>(doc, K, reinterpret_cast<int*>(lds + Y.rows + 3 * kTile), tid, threads, whole);
	const int own_lo = K.own_place0 + K.own0, own_hi = K.own_place0 + min(K.own0 + K.nown, A.T) - 1;
	int place[4], od4[4];
#pragma unroll
	for (int a = 0; a < 4; a++) {
		const int t = K.own0 + wave * kOwn + i + 8 * a;
		place[a] = K.own_place0 + t;
		od4[a] = doc && t < A.T ? doc[place[a]] : -1;
	}
	f4 out[2][NB];
	float den[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int tb = 0; tb < 2; tb++)
#pragma unroll
		for (int wb = 0; wb < NB; wb++) out[tb][wb] = (f4)(0.f);
	const int s_end = A.causal ? min(A.S, max(own_hi + 1, prefix)) : A.S;  // nothing behind is visible
	const int tiles = (s_end + kTile - 1) / kTile;
	for (int t0 = 0; t0 < tiles; t0 += kClasses) {
		__syncthreads();
		classify<false>(A, doc, prefix, own_lo, own_hi, od, whole, A.S, 0, t0, min(kClasses, tiles - t0), cls, tid, threads);
		__syncthreads();
		for (int t = 0; t < min(kClasses, tiles - t0); t++) {
			const int kind = cls[t];
			if (!kind) continue;
			const int s0 = (t0 + t) * kTile;
			__syncthreads();
			stage<ST, false>(str, kh, s0, kTile, A.S, kpitch, A.W, sw, A.vec & 2, tid, threads);
			bool bad = stage<ST, true>(val, vh, s0, kTile, A.S, vpitch, A.Wv, sv, A.vec & 4, tid, threads);
			if (tid < kTile) docs[tid] = doc && s0 + tid < A.S ? doc[s0 + tid] : -1;
			bad = __syncthreads_or(bad && kind == 2);
			float x[4][8];
			distances(own, str, chunks, sw, i, j, x);
#pragma unroll
			for (int b = 0; b < 8; b++) {
				const int s = s0 + j + 8 * b;
				const int sd = docs[j + 8 * b];
#pragma unroll
				for (int a = 0; a < 4; a++) {
					float c = -x[a][b] * A.rw;
					if (A.cap > 0.f) c = A.cap * tanhf(c * A.icap);
					float p = expf(c - slope * (float)abs(place[a] - s));
					if (kind == 2 && !(s < A.S && sees(A, prefix, doc, place[a], s, od4[a], sd))) p = 0.f;
					den[a] += p;
					x[a][b] = p;
				}
			}
#pragma unroll
			for (int half = 0; half < 2; half++) {
				wave_sync();
#pragma unroll
				for (int a = 0; a < 4; a++) {
					const f4 w = {x[a][4 * half], x[a][4 * half + 1], x[a][4 * half + 2], x[a][4 * half + 3]};
					*reinterpret_cast<f4*>(scr + (i + 8 * a) * kPad + 4 * j) = w;
				}
				wave_sync();
				weigh<NB>(out, scr, val + 32 * half * sv, sv, l16, g, bad);
			}
		}
	}
	// a row's sum lies in the eight lanes j; then to the lanes that hold the row's output
#pragma unroll
	for (int a = 0; a < 4; a++) {
		den[a] += __shfl_xor(den[a], 8);
		den[a] += __shfl_xor(den[a], 16);
		den[a] += __shfl_xor(den[a], 32);
	}
	wave_sync();
	if (j == 0)
#pragma unroll
		for (int a = 0; a < 4; a++) scr[i + 8 * a] = den[a];
	wave_sync();
#pragma unroll
	for (int tb = 0; tb < 2; tb++) {
		const int t = K.own0 + wave * kOwn + 16 * tb + l16;
		const float d = scr[16 * tb + l16];
		const float r = 1.f / (1.f + d);
		if (t >= A.T) continue;
		const int64_t row = ((int64_t)K.b * A.T + t) * A.H + K.h;
		if (lse && g == 0) lse[row] = log1pf(d);
#pragma unroll
		for (int wb = 0; wb < NB; wb++)
#pragma unroll
			for (int e = 0; e < 4; e++) {
				const int w = 16 * wb + 4 * g + e;
				if (w < A.Wv) o[row * A.Wv + w] = (ST)(out[tb][wb][e] * r);
			}
	}
}

// --------------------------------------------------------------------------------------------------------------- backward

// D[row] = sum_w do * o, row = (b, t, h): what the softmax's gradient subtracts
template <typename ST>
__global__ void __launch_bounds__(256) masked_bwd_rows(const ST* __restrict__ dout, const ST* __restrict__ o, float* __restrict__ D,
                                                       int64_t rows, int Wv)
{
	const int64_t row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
	float s = 0.f;
	if (row < rows)
		for (int w = threadIdx.x & 7; w < Wv; w += 8) s += to_f(dout[row * Wv + w]) * to_f(o[row * Wv + w]);
	s += __shfl_xor(s, 1);
	s += __shfl_xor(s, 2);
	s += __shfl_xor(s, 4);
	if (row < rows && (threadIdx.x & 7) == 0) D[row] = s;
}

// Gradients of one side.  OWNK false: owners are queries, dx = dq.  OWNK true: owners are keys, dx = dk and dy = dv, summed
// over the query heads that share them.  WL: columns w a lane holds in the sign part (W <= 64 * WL).
// sign: h = clamp((own - str) * 2^127 + 1/2, 0, 1) is 1, 1/2, 0 for own >, ==, < str (differences below 2^-128 count in
// part), and sum g * sign = 2 * sum g * h - sum g.
template <typename ST, bool OWNK, int WL, int NB, int THREADS>
__global__ void __launch_bounds__(THREADS) masked_bwd(L1MaskedArgs A, const ST* __restrict__ q, const ST* __restrict__ k,
                                                      const ST* __restrict__ v, const ST* __restrict__ dout,
                                                      const float* __restrict__ lse, const float* __restrict__ D,
                                                      ST* __restrict__ dx, ST* __restrict__ dy)
{
	extern __shared__ float lds[];
	const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
	const int i = lane & 7, j = lane >> 3, l16 = lane & 15, g = lane >> 4;
	const int group = A.H / A.Hk;
	Block K;
	const int heads = OWNK ? A.Hk : A.H;
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
	const Layout Y = masked_layout(A.W, A.Wv, waves);
	const int sw = row_floats(A.W), sv = row_floats(A.Wv), chunks = (A.W + 3) >> 2;
	float* own = lds + Y.own + wave * kOwn * sw;
	float* str = lds + Y.str;
	float* val = lds + Y.y;
	float* scr = lds + Y.scratch + wave * kOwn * kPad;
	int* docs = reinterpret_cast<int*>(lds + Y.rows);
	float* slse = lds + Y.rows + kTile;
	float* sD = lds + Y.rows + 2 * kTile;
	unsigned char* cls = reinterpret_cast<unsigned char*>(lds + Y.rows + 3 * kTile + 32);
	const int* doc = A.doc ? A.doc + (int64_t)K.b * A.S : nullptr;
	const int prefix = A.prefix ? A.prefix[K.b] : 0;
	const int64_t qpitch = (int64_t)A.H * A.W, kpitch = (int64_t)A.Hk * A.W;
	const int64_t opitch = (int64_t)A.H * A.Wv, vpitch = (int64_t)A.Hk * A.Wv;
	const ST* kh = k + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.W;
	const ST* vh = v + ((int64_t)K.b * A.S * A.Hk + K.hk) * A.Wv;
	const int own_row0 = K.own0 + wave * kOwn;

	if (OWNK) stage<ST, false>(own, kh, own_row0, kOwn, A.S, kpitch, A.W, sw, A.vec & 2, lane, 64);
	else stage<ST, false>(own, q + ((int64_t)K.b * A.T * A.H + K.h) * A.W, own_row0, kOwn, A.T, qpitch, A.W, sw, A.vec & 1, lane, 64);
	for (int x = tid; x < kTile * (sv - A.Wv); x += threads) val[(x / (sv - A.Wv)) * sv + A.Wv + x % (sv - A.Wv)] = 0.f;
	bool whole;
	const Span od = owner_docs<OWNK>(doc, K, reinterpret_cast<int*>(lds + Y.rows + 3 * kTile), tid, threads, whole);
	const int own_lo = K.own_place0 + K.own0, own_hi = K.own_place0 + min(K.own0 + K.nown, K.own_rows) - 1;
	// the owners' columns in the sign part: register r = 4i' + a' is owner i' + 8a'
	float ov[WL][32], sum[WL][32];
#pragma unroll
	for (int u = 0; u < WL; u++)
#pragma unroll
		for (int r = 0; r < 32; r++) {
			const int w = lane + 64 * u;
			ov[u][r] = w < A.W ? own[((r >> 2) + 8 * (r & 3)) * sw + w] : 0.f;
			sum[u][r] = 0.f;
		}
	int place[4], od4[4];
#pragma unroll
	for (int a = 0; a < 4; a++) {
		place[a] = K.own_place0 + own_row0 + i + 8 * a;
		od4[a] = doc && own_row0 + i + 8 * a < K.own_rows ? doc[place[a]] : -1;
	}
	float gsum[4] = {0.f, 0.f, 0.f, 0.f};
	f4 dyv[2][OWNK ? NB : 1];
#pragma unroll
	for (int tb = 0; tb < 2; tb++)
#pragma unroll
		for (int wb = 0; wb < (OWNK ? NB : 1); wb++) dyv[tb][wb] = (f4)(0.f);

	for (int hg = 0; hg < (OWNK ? group : 1); hg++) {
		const int h = OWNK ? K.hk * group + hg : K.h;
		const float slope = A.has_slopes ? A.slopes[h] : 0.f;
		const ST* qh = q + ((int64_t)K.b * A.T * A.H + h) * A.W;
		const ST* oh = dout + ((int64_t)K.b * A.T * A.H + h) * A.Wv;
		// the owners' rows of the second product (v of the keys, do of the queries), as its right operand
		f4 xr[2][NB];
#pragma unroll
		for (int ob = 0; ob < 2; ob++) {
			const int r = own_row0 + 16 * ob + l16;
			const ST* row = OWNK ? vh + (int64_t)r * vpitch : oh + (int64_t)r * opitch;
#pragma unroll
			for (int kc = 0; kc < NB; kc++) {
				const int w = 16 * kc + 4 * g;
				xr[ob][kc] = r < K.own_rows && w < A.Wv ? load4(row + w, A.Wv - w, OWNK ? A.vec & 4 : A.vec & 8) : (f4)(0.f);
			}
		}
		float olse[4], oD[4];
#pragma unroll
		for (int a = 0; a < 4; a++) {
			const int t = own_row0 + i + 8 * a;
			const bool in = !OWNK && t < A.T;
			olse[a] = in ? lse[((int64_t)K.b * A.T + t) * A.H + h] : 0.f;
			oD[a] = in ? D[((int64_t)K.b * A.T + t) * A.H + h] : 0.f;
		}
		int first = 0, last = (K.str_rows + kTile - 1) / kTile;
		if (A.causal) {
			if (OWNK) { if (own_lo >= prefix) first = max(0, own_lo - K.str_place0) / kTile; }
			else last = (min(A.S, max(own_hi + 1, prefix)) + kTile - 1) / kTile;
		}
		for (int t0 = first; t0 < last; t0 += kClasses) {
			const int n = min(kClasses, last - t0);
			__syncthreads();
			classify<OWNK>(A, doc, prefix, own_lo, own_hi, od, whole, K.str_rows, K.str_place0, t0, n, cls, tid, threads);
			__syncthreads();
			for (int t = 0; t < n; t++) {
				const int kind = cls[t];
				if (!kind) continue;
				const int s0 = (t0 + t) * kTile;
				__syncthreads();
				bool bad;
				if (OWNK) {
					stage<ST, false>(str, qh, s0, kTile, A.T, qpitch, A.W, sw, A.vec & 1, tid, threads);
					bad = stage<ST, true>(val, oh, s0, kTile, A.T, opitch, A.Wv, sv, A.vec & 8, tid, threads);
				} else {
					stage<ST, false>(str, kh, s0, kTile, A.S, kpitch, A.W, sw, A.vec & 2, tid, threads);
					bad = stage<ST, true>(val, vh, s0, kTile, A.S, vpitch, A.Wv, sv, A.vec & 4, tid, threads);
				}
				if (tid < kTile) {
					const bool in = s0 + tid < K.str_rows;
					docs[tid] = doc && in ? doc[K.str_place0 + s0 + tid] : -1;
					if (OWNK) {
						slse[tid] = in ? lse[((int64_t)K.b * A.T + s0 + tid) * A.H + h] : 0.f;
						sD[tid] = in ? D[((int64_t)K.b * A.T + s0 + tid) * A.H + h] : 0.f;
					}
				}
				bad = __syncthreads_or(bad && kind == 2);
				float x[4][8], f[4][8];
				distances(own, str, chunks, sw, i, j, x);
#pragma unroll
				for (int b = 0; b < 8; b++) {
					const int r = j + 8 * b, sp = K.str_place0 + s0 + r, sd = docs[r];
					const float sl = OWNK ? slse[r] : 0.f;
#pragma unroll
					for (int a = 0; a < 4; a++) {
						float c = -x[a][b] * A.rw, fac = -A.rw;
						if (A.cap > 0.f) {
							const float th = tanhf(c * A.icap);
							c = A.cap * th;
							fac *= 1.f - th * th;
						}
						float p = expf(c - slope * (float)abs(place[a] - sp) - (OWNK ? sl : olse[a]));
						if (kind == 2 && !(s0 + r < K.str_rows && (OWNK ? sees(A, prefix, doc, sp, place[a], sd, od4[a])
						                                              : sees(A, prefix, doc, place[a], sp, od4[a], sd)))) p = 0.f;
						x[a][b] = p;
						f[a][b] = fac;
					}
				}
#pragma unroll
				for (int half = 0; half < 2; half++) {
					if (OWNK) {  // dv += p * do
						wave_sync();
#pragma unroll
						for (int a = 0; a < 4; a++) {
							const f4 w = {x[a][4 * half], x[a][4 * half + 1], x[a][4 * half + 2], x[a][4 * half + 3]};
							*reinterpret_cast<f4*>(scr + (i + 8 * a) * kPad + 4 * j) = w;
						}
						wave_sync();
						weigh<OWNK ? NB : 1>(dyv, scr, val + 32 * half * sv, sv, l16, g, bad);
					}
					// dp of this half's 32 columns
					f4 dp[2][2];
#pragma unroll
					for (int cb = 0; cb < 2; cb++) {
						dp[cb][0] = (f4)(0.f);
						dp[cb][1] = (f4)(0.f);
#pragma unroll
						for (int kc = 0; kc < NB; kc++) {
							const int w = 16 * kc + 4 * g;
							const f4 ya = w < sv ? *reinterpret_cast<const f4*>(val + (32 * half + 16 * cb + l16) * sv + w) : (f4)(0.f);
#pragma unroll
							for (int e = 0; e < 4; e++)
#pragma unroll
								for (int ob = 0; ob < 2; ob++) dp[cb][ob] = __builtin_amdgcn_mfma_f32_16x16x4f32(ya[e], xr[ob][kc][e], dp[cb][ob], 0, 0, 0);
						}
					}
					wave_sync();
#pragma unroll
					for (int cb = 0; cb < 2; cb++)
#pragma unroll
						for (int ob = 0; ob < 2; ob++) *reinterpret_cast<f4*>(scr + (l16 + 16 * ob) * kPad + 16 * cb + 4 * g) = dp[cb][ob];
					wave_sync();
					f4 d4[4];
#pragma unroll
					for (int a = 0; a < 4; a++) d4[a] = *reinterpret_cast<const f4*>(scr + (i + 8 * a) * kPad + 4 * j);
					wave_sync();
#pragma unroll
					for (int bb = 0; bb < 4; bb++) {
						const int b = 4 * half + bb;
						const float dD = OWNK ? sD[j + 8 * b] : 0.f;
						f4 gr;
#pragma unroll
						for (int a = 0; a < 4; a++) {
							const float p = x[a][b];
							// a hidden pair's dp may come from values that are not finite
							gr[a] = p != 0.f ? p * (d4[a][bb] - (OWNK ? dD : oD[a])) * f[a][b] : 0.f;
							gsum[a] += gr[a];
						}
						*reinterpret_cast<f4*>(scr + (4 * j + bb) * kPad + 4 * i) = gr;
					}
					wave_sync();
					// signs: 32 stream rows against the 32 owners, a lane holds its columns of all of them
#pragma unroll 2
					for (int c = 0; c < 32; c++) {
						const float* row = str + row_of(32 * half + c) * sw;
						float sval[WL];
#pragma unroll
						for (int u = 0; u < WL; u++) sval[u] = lane + 64 * u < sw ? row[lane + 64 * u] : 0.f;
#pragma unroll
						for (int r4 = 0; r4 < 8; r4++) {
							const f4 gr = *reinterpret_cast<const f4*>(scr + c * kPad + 4 * r4);
#pragma unroll
							for (int e = 0; e < 4; e++)
#pragma unroll
								for (int u = 0; u < WL; u++) {
									const float hv = __builtin_amdgcn_fmed3f(__builtin_fmaf(ov[u][4 * r4 + e] - sval[u], 0x1p127f, 0.5f), 0.f, 1.f);
									sum[u][4 * r4 + e] = __builtin_fmaf(hv, gr[e], sum[u][4 * r4 + e]);
								}
						}
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
		for (int a = 0; a < 4; a++) scr[4 * i + a] = gsum[a];
	wave_sync();
#pragma unroll
	for (int r = 0; r < 32; r++) {
		const int t = own_row0 + (r >> 2) + 8 * (r & 3);
		const float gs = scr[r];
		if (t >= K.own_rows) continue;
		const int64_t row = ((int64_t)K.b * K.own_rows + t) * heads + K.h;
#pragma unroll
		for (int u = 0; u < WL; u++)
			if (lane + 64 * u < A.W) dx[row * A.W + lane + 64 * u] = (ST)(2.f * sum[u][r] - gs);
	}
	if (OWNK) {
#pragma unroll
		for (int tb = 0; tb < 2; tb++) {
			const int s = own_row0 + 16 * tb + l16;
			if (s >= A.S) continue;
			const int64_t row = ((int64_t)K.b * A.S + s) * A.Hk + K.hk;
#pragma unroll
			for (int wb = 0; wb < (OWNK ? NB : 1); wb++)
#pragma unroll
				for (int e = 0; e < 4; e++) {
					const int w = 16 * wb + 4 * g + e;
					if (w < A.Wv) dy[row * A.Wv + w] = (ST)dyv[tb][wb][e];
				}
		}
	}
}

__global__ void __launch_bounds__(256) masked_zero(uint16_t* __restrict__ x, int64_t n)
{
	const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
	if (at < n) x[at] = 0;
}

// ------------------------------------------------------------------------------------------------------------------- host

bool fits(int64_t x, int64_t most) { return x >= 0 && x <= most; }

// 0, an error, or 1 for a call with nothing to do
int check_desc(const l1attn_masked_desc* d)
{
	if (!d) return L1ATTN_ERR_ARG;
	if (d->B < 0 || d->T < 0 || d->S < d->T || d->H < 1 || d->Hk < 1 || d->H % d->Hk || d->W < 1 || d->Wv < 1) return L1ATTN_ERR_ARG;
	if (d->dtype < 0 || d->dtype > 2 || (d->causal != 0 && d->causal != 1)) return L1ATTN_ERR_ARG;
	if (!(d->softcap >= 0.f) || !(d->softcap <= 3e38f)) return L1ATTN_ERR_ARG;
	if (!d->causal && d->prefix) return L1ATTN_ERR_ARG;
	if (d->W > 128 || d->Wv > 128 || d->H > L1_MASKED_HEADS || !fits(d->S, 1 << 30) || !fits(d->B * d->H, 0x7fffffff)) return L1ATTN_ERR_RANGE;
	if (l1_cdiv(d->S, kOwn) > 65535 * (int64_t)2) return L1ATTN_ERR_RANGE;  // rows of the grid, two waves a workgroup at least
	if (d->slopes)
		for (int64_t h = 0; h < d->H; h++)
			if (!(d->slopes[h] >= 0.f) || !(d->slopes[h] <= 3e38f)) return L1ATTN_ERR_ARG;
	return d->B == 0 || d->T == 0 ? 1 : L1ATTN_OK;
}

L1MaskedArgs args_of(const l1attn_masked_desc* d, const void* q, const void* k, const void* v, const void* dout)
{
	L1MaskedArgs A;
	A.B = (int)d->B; A.T = (int)d->T; A.S = (int)d->S; A.H = (int)d->H; A.Hk = (int)d->Hk; A.W = (int)d->W; A.Wv = (int)d->Wv;
	A.causal = d->causal; A.cap = d->softcap; A.icap = d->softcap > 0.f ? 1.f / d->softcap : 0.f;
	A.rw = (float)(1.0 / sqrt((double)d->W));
	A.doc = d->doc; A.prefix = d->prefix; A.has_slopes = d->slopes != nullptr;
	for (int h = 0; h < L1_MASKED_HEADS; h++) A.slopes[h] = d->slopes && h < d->H ? d->slopes[h] : 0.f;
	const uintptr_t m = d->dtype == 0 ? 15 : 7;
	A.vec = (d->W % 4 == 0 && !((uintptr_t)q & m) ? 1 : 0) | (d->W % 4 == 0 && !((uintptr_t)k & m) ? 2 : 0) |
	        (d->Wv % 4 == 0 && !((uintptr_t)v & m) ? 4 : 0) | (d->Wv % 4 == 0 && !((uintptr_t)dout & m) ? 8 : 0);
	return A;
}

// waves of a workgroup: as many as share a tile of the stream without leaving compute units idle (256 of them)
int waves_for(int64_t owners, int64_t heads, int most)
{
	int w = most;
	while (w > 2 && heads * l1_cdiv(owners, kOwn * w) < 256) w >>= 1;
	return w;
}

template <typename F>
int launch(F* f, dim3 grid, int waves, const L1MaskedArgs& A, hipStream_t st, void** args)
{
	const int bytes = masked_layout(A.W, A.Wv, waves).total * 4;
	L1_HIP_CHECK(hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
	L1_HIP_CHECK(hipLaunchKernel((const void*)f, grid, dim3(64 * waves), args, bytes, st));
	return L1ATTN_OK;
}

template <typename ST>
int run_fwd(const l1attn_masked_desc* d, const void* q, const void* k, const void* v, void* o, float* lse, hipStream_t st)
{
	L1MaskedArgs A = args_of(d, q, k, v, nullptr);
	const bool wide = A.W > 64 || A.Wv > 64;
	const int waves = waves_for(A.T, (int64_t)A.B * A.H, wide ? 4 : 8);
	const dim3 grid((unsigned)(A.B * A.H), (unsigned)l1_cdiv(A.T, kOwn * waves));
	if (grid.y > 65535) return L1ATTN_ERR_RANGE;
	void* args[] = {&A, &q, &k, &v, &o, &lse};
	if (wide) return launch(masked_fwd<ST, 8, 256>, grid, waves, A, st, args);
	if (A.Wv > 32) return launch(masked_fwd<ST, 4, 512>, grid, waves, A, st, args);
	return launch(masked_fwd<ST, 2, 512>, grid, waves, A, st, args);
}

template <typename ST, bool OWNK>
int run_side(L1MaskedArgs A, const void* q, const void* k, const void* v, const void* dout, const float* lse, const float* D,
             void* dx, void* dy, hipStream_t st)
{
	const bool wide = A.W > 64 || A.Wv > 64;
	const int64_t heads = (int64_t)A.B * (OWNK ? A.Hk : A.H), rows = OWNK ? A.S : A.T;
	const int waves = waves_for(rows, heads, wide ? 4 : 8);
	const dim3 grid((unsigned)heads, (unsigned)l1_cdiv(rows, kOwn * waves));
	if (grid.y > 65535) return L1ATTN_ERR_RANGE;
	void* args[] = {&A, &q, &k, &v, &dout, &lse, &D, &dx, &dy};
	if (A.W > 64) return launch(masked_bwd<ST, OWNK, 2, 8, 256>, grid, waves, A, st, args);
	if (A.Wv > 64) return launch(masked_bwd<ST, OWNK, 1, 8, 256>, grid, waves, A, st, args);
	return launch(masked_bwd<ST, OWNK, 1, 4, 512>, grid, waves, A, st, args);
}

template <typename ST>
int run_bwd(const l1attn_masked_desc* d, const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
            void* dq, void* dk, void* dv, float* D, hipStream_t st)
{
	const L1MaskedArgs A = args_of(d, q, k, v, dout);
	const int64_t rows = d->B * d->T * d->H;
	hipLaunchKernelGGL(masked_bwd_rows<ST>, dim3((unsigned)l1_cdiv(rows, 32)), dim3(256), 0, st, (const ST*)dout, (const ST*)o, D, rows, A.Wv);
	L1_LAUNCH_CHECK();
	const int rc = run_side<ST, false>(A, q, k, v, dout, lse, D, dq, nullptr, st);
	return rc != L1ATTN_OK ? rc : run_side<ST, true>(A, q, k, v, dout, lse, D, dk, dv, st);
}

}  // namespace

extern "C" {

int l1attn_masked_fwd(const l1attn_masked_desc* desc, const void* q, const void* k, const void* v, void* o, float* lse, void* stream)
{
	const int rc = check_desc(desc);
	if (rc) return rc == 1 ? L1ATTN_OK : rc;
	if (!q || !k || !v || !o) return L1ATTN_ERR_ARG;
	hipStream_t st = (hipStream_t)stream;
	if (desc->dtype == 0) return run_fwd<float>(desc, q, k, v, o, lse, st);
	if (desc->dtype == 1) return run_fwd<_Float16>(desc, q, k, v, o, lse, st);
	return run_fwd<__bf16>(desc, q, k, v, o, lse, st);
}

size_t l1attn_masked_bwd_workspace_bytes(const l1attn_masked_desc* desc)
{
	return check_desc(desc) ? 0 : (size_t)(desc->B * desc->T * desc->H) * sizeof(float);
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
		hipLaunchKernelGGL(masked_zero, dim3((unsigned)l1_cdiv(nk, 256)), dim3(256), 0, st, (uint16_t*)dk, nk);
		L1_LAUNCH_CHECK();
		hipLaunchKernelGGL(masked_zero, dim3((unsigned)l1_cdiv(nv, 256)), dim3(256), 0, st, (uint16_t*)dv, nv);
		L1_LAUNCH_CHECK();
		return L1ATTN_OK;
	}
	float* D = (float*)workspace;
	if (desc->dtype == 0) return run_bwd<float>(desc, q, k, v, o, lse, d_o, dq, dk, dv, D, st);
	if (desc->dtype == 1) return run_bwd<_Float16>(desc, q, k, v, o, lse, d_o, dq, dk, dv, D, st);
	return run_bwd<__bf16>(desc, q, k, v, o, lse, d_o, dq, dk, dv, D, st);
}

}  // extern "C"
