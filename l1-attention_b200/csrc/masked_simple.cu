// Masked L1 attention (mask.cuh), float32 arithmetic for every storage type and widths up to 256.
//
// Forward: a CTA owns 64 query rows of one head; keys and values stream in tiles of 64 (32), all operands as floats in shared memory.  256
// threads, a 4 x 4 (4 x 2) tile of scores each (rows 4 ty + i, keys tx + 16 j); the 16 lanes of a half-warp own their four rows, so the running maximum
// and sum (one pass over the keys) and the weights never leave the half-warp.  Bound: FP32 instructions -- two per term of the distance, one per term
// of a product -- of which the loads of scores and weights take a quarter of the issue slots: 21 terms per clock and SM ([4,2048,8,128], no mask: 2.75 ms).
// Backward: two kernels without atomics.  One owns 64 query rows and makes dq, the other 64 key rows of one query head and makes its share of dk and dv;
// both recompute the weights from the log-normalisers and stream the other side in
// tiles of 32.  sign(0) = 0.
#include "mask.cuh"

namespace l1b {

namespace {

constexpr int OWN = 64, STREAM = 32, THREADS = 256;

// floats of a row of `w` values: whole float4s, an odd number of them so that 8 rows at one column lie in different banks
__host__ __device__ inline int pitch(int w)
{
	const int p = (w + 3) / 4;
	return 4 * (p % 2 ? p : p + 1);
}

// rows [first, first + rows) of one head as floats, zeros past n and past the width (to `cols` columns); true when a value is not finite
template <typename T>
__device__ bool load_rows(float *dst, int pitch_, int cols, const Strided &x, int b, int head, int first, int rows, int n, int width)
{
	constexpr int AT_ONCE = 4; // rows of a warp whose reads do not wait for one another
	const T *src = static_cast<const T *>(x.p) + b * x.batch + head * x.head;
	const int lane = threadIdx.x % 32;
	bool odd = false;
	if (sizeof(T) == 4 && width % 4 == 0 && reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && (x.batch | x.tok | x.head) % 4 == 0) { // 16 bytes a lane
		for (int r0 = threadIdx.x / 32; r0 < rows; r0 += AT_ONCE * (THREADS / 32))
			for (int c = 4 * lane; c < cols; c += 128) {
				float4 f[AT_ONCE];
#pragma unroll
				for (int i = 0; i < AT_ONCE; i++) {
					const int r = r0 + i * (THREADS / 32);
					f[i] = r < rows && first + r < n && c < width ? *reinterpret_cast<const float4 *>(src + (first + r) * x.tok + c) : make_float4(0.f, 0.f, 0.f, 0.f);
				}
#pragma unroll
				for (int i = 0; i < AT_ONCE; i++)
					if (const int r = r0 + i * (THREADS / 32); r < rows) {
						odd |= !(fabsf(f[i].x) + fabsf(f[i].y) + fabsf(f[i].z) + fabsf(f[i].w) < INFINITY);
						*reinterpret_cast<float4 *>(dst + r * pitch_ + c) = f[i];
					}
			}
		return odd;
	}
	for (int r0 = threadIdx.x / 32; r0 < rows; r0 += AT_ONCE * (THREADS / 32))
		for (int c = lane; c < cols; c += 32) {
			float f[AT_ONCE];
#pragma unroll
			for (int i = 0; i < AT_ONCE; i++) {
				const int r = r0 + i * (THREADS / 32);
				f[i] = r < rows && first + r < n && c < width ? to_float(src[(first + r) * x.tok + c]) : 0.f;
			}
#pragma unroll
			for (int i = 0; i < AT_ONCE; i++)
				if (const int r = r0 + i * (THREADS / 32); r < rows) {
					odd |= !(fabsf(f[i]) < INFINITY);
					dst[r * pitch_ + c] = f[i];
				}
		}
	return odd;
}

__device__ __forceinline__ float half_warp_max(float x)
{
#pragma unroll
	for (int o = 8; o; o >>= 1)
		x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
	return x;
}
__device__ __forceinline__ float half_warp_sum(float x)
{
#pragma unroll
	for (int o = 8; o; o >>= 1)
		x += __shfl_xor_sync(0xffffffffu, x, o);
	return x;
}

// sum_w |a[row i] - b[key j]| of this thread's 4 x J pairs (columns past the width are zeros)
template <int J> __device__ __forceinline__ void distances(const float *A, const float *B, int ap, int cols, int ty, int tx, float (&d)[4][J])
{
#pragma unroll
	for (int i = 0; i < 4; i++)
#pragma unroll
		for (int j = 0; j < J; j++)
			d[i][j] = 0.f;
	for (int w = 0; w < cols; w += 4) {
		float4 x[4], y[J];
#pragma unroll
		for (int i = 0; i < 4; i++)
			x[i] = *reinterpret_cast<const float4 *>(A + (4 * ty + i) * ap + w);
#pragma unroll
		for (int j = 0; j < J; j++)
			y[j] = *reinterpret_cast<const float4 *>(B + (tx + 16 * j) * ap + w);
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int j = 0; j < J; j++)
				d[i][j] += (fabsf(x[i].x - y[j].x) + fabsf(x[i].y - y[j].y)) + (fabsf(x[i].z - y[j].z) + fabsf(x[i].w - y[j].w));
	}
}
template <int J> __device__ __forceinline__ void products(const float *A, const float *B, int ap, int cols, int ty, int tx, float (&d)[4][J])
{
#pragma unroll
	for (int i = 0; i < 4; i++)
#pragma unroll
		for (int j = 0; j < J; j++)
			d[i][j] = 0.f;
	for (int w = 0; w < cols; w += 4) {
		float4 x[4], y[J];
#pragma unroll
		for (int i = 0; i < 4; i++)
			x[i] = *reinterpret_cast<const float4 *>(A + (4 * ty + i) * ap + w);
#pragma unroll
		for (int j = 0; j < J; j++)
			y[j] = *reinterpret_cast<const float4 *>(B + (tx + 16 * j) * ap + w);
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int j = 0; j < J; j++)
				d[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, d[i][j]))));
	}
}

template <typename T, int NV, int KEYS> __global__ void __launch_bounds__(THREADS) masked_fwd_simple_kernel(MaskedArgs a, T *vo, T *rest, float *lse, int tiles)
{
	extern __shared__ float4 smem4[];
	const int wp = pitch(a.width), vp = 64 * NV, tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
	float *Q = reinterpret_cast<float *>(smem4), *K = Q + OWN * wp, *V = K + KEYS * wp, *P = V + KEYS * vp;
	constexpr int PP = KEYS + 4;
	const int bh = blockIdx.x % (a.bs * a.heads), tile = tiles - 1 - int(blockIdx.x / (a.bs * a.heads)); // the longest rows of a causal mask first, of all heads
	const int head = bh % a.heads, b = bh / a.heads, kv = head / (a.heads / a.kv_heads);
	const MaskView mask(a, b);
	const int t0 = tile * OWN, t1 = min(a.n, t0 + OWN);
	const float slope = a.slopes ? a.slopes[head] : 0.f, inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
	load_rows<T>(Q, wp, wp, a.q, b, head, t0, OWN, a.n, a.width);
	float m[4], l[4], acc[4][4 * NV];
	int doc_t[4];
#pragma unroll
	for (int i = 0; i < 4; i++) {
		m[i] = start_max(a.mode);
		l[i] = start_sum(a.mode);
		doc_t[i] = mask.doc && t0 + 4 * ty + i < a.n ? mask.doc[t0 + 4 * ty + i] : 0;
#pragma unroll
		for (int c = 0; c < 4 * NV; c++)
			acc[i][c] = 0.f;
	}
	for (int s0 = 0; s0 < a.n; s0 += KEYS) {
		const int s1 = min(a.n, s0 + KEYS);
		if (!mask.any(t0, t1, s0, s1))
			continue;
		__syncthreads();
		load_rows<T>(K, wp, wp, a.k, b, kv, s0, KEYS, a.n, a.width);
		const bool odd = __syncthreads_or(load_rows<T>(V, vp, vp, a.v, b, kv, s0, KEYS, a.n, a.v_width));
		constexpr int J = KEYS / 16;
		const bool whole = s1 == s0 + KEYS && t1 == t0 + OWN && mask.all(t0, t1, s0, s1);
		float x[4][J];
		distances<J>(Q, K, wp, a.width, ty, tx, x);
#pragma unroll
		for (int i = 0; i < 4; i++) {
			const int t = t0 + 4 * ty + i;
			float top = m[i];
#pragma unroll
			for (int j = 0; j < J; j++) {
				const int s = s0 + tx + 16 * j;
				float y = -a.scale * x[i][j];
				if (a.cap > 0.f)
					y = a.cap * tanhf(y * inv_cap);
				y -= slope * fabsf(float(t - s));
				x[i][j] = whole || mask.sees(t, s, doc_t[i], mask.doc && s < a.n ? mask.doc[s] : 0) ? y : -INFINITY;
				top = fmaxf(top, x[i][j]);
			}
			top = half_warp_max(top);
			const float ref = top == -INFINITY ? 0.f : top, keep = expf(m[i] - ref);
			float sum = 0.f;
#pragma unroll
			for (int j = 0; j < J; j++) {
				const float p = expf(x[i][j] - ref);
				sum += p;
				P[(4 * ty + i) * PP + tx + 16 * j] = p;
			}
			l[i] = l[i] * keep + half_warp_sum(sum);
			m[i] = top;
#pragma unroll
			for (int c = 0; c < 4 * NV; c++)
				acc[i][c] *= keep;
		}
		__syncwarp();
		auto add = [&](const float (&p)[4], int s, bool skip) {
#pragma unroll
			for (int u = 0; u < NV; u++) {
				const float4 v = *reinterpret_cast<const float4 *>(V + s * vp + 64 * u + 4 * tx);
#pragma unroll
				for (int i = 0; i < 4; i++) {
					if (skip && p[i] == 0.f)
						continue;
					acc[i][4 * u] = fmaf(p[i], v.x, acc[i][4 * u]);
					acc[i][4 * u + 1] = fmaf(p[i], v.y, acc[i][4 * u + 1]);
					acc[i][4 * u + 2] = fmaf(p[i], v.z, acc[i][4 * u + 2]);
					acc[i][4 * u + 3] = fmaf(p[i], v.w, acc[i][4 * u + 3]);
				}
			}
		};
		if (odd) // a value that is not finite: what has no weight must not be multiplied
			for (int s = 0; s < s1 - s0; s++) {
				float p[4];
#pragma unroll
				for (int i = 0; i < 4; i++)
					p[i] = P[(4 * ty + i) * PP + s];
				add(p, s, true);
			}
		else // four keys at a time (past the last one: weights and values of zero)
			for (int s = 0; s < s1 - s0; s += 4) {
				float4 p[4];
#pragma unroll
				for (int i = 0; i < 4; i++)
					p[i] = *reinterpret_cast<const float4 *>(P + (4 * ty + i) * PP + s);
				add({p[0].x, p[1].x, p[2].x, p[3].x}, s, false);
				add({p[0].y, p[1].y, p[2].y, p[3].y}, s + 1, false);
				add({p[0].z, p[1].z, p[2].z, p[3].z}, s + 2, false);
				add({p[0].w, p[1].w, p[2].w, p[3].w}, s + 3, false);
			}
	}
#pragma unroll
	for (int i = 0; i < 4; i++) {
		const int t = t0 + 4 * ty + i;
		if (t >= a.n)
			continue;
		const long long row = ((long long)b * a.n + t) * a.heads + head;
		float ls;
		const float f = finish_row(a.mode, m[i], l[i], &ls);
		if (tx == 0 && lse)
			lse[row] = ls;
#pragma unroll
		for (int c = 0; c < 4 * NV; c++) {
			const int w = 64 * (c / 4) + 4 * tx + c % 4;
			if (w < a.v_width) {
				const float y = f == 0.f ? 0.f : acc[i][c] * f;
				vo[row * a.v_width + w] = from_float<T>(y);
				if (rest)
					rest[row * a.v_width + w] = rest_of<T>(y);
			}
		}
	}
}

// sum += sign(a - b) e, minus = -e: two compares and two predicated additions (left to the compiler, selections: 21.4 instead of 19.4 ms for
// [4,2048,8,128] without a mask)
__device__ __forceinline__ void add_by_sign(float &sum, float a, float b, float e, float minus)
{
	asm("{\n\t.reg .pred p, q;\n\t"
	    "setp.gt.f32 p, %1, %2;\n\t"
	    "setp.lt.f32 q, %1, %2;\n\t"
	    "@p add.f32 %0, %0, %3;\n\t"
	    "@q add.f32 %0, %0, %4;\n\t}"
	    : "+f"(sum)
	    : "f"(a), "f"(b), "f"(e), "f"(minus));
}

// OWN_KEYS: a CTA owns 64 keys of one query head and makes its share of their dk and dv; else 64 queries, dq.  A thread owns the columns tx + 16 c of
// four own rows, c < NW (NV), its own values in registers: a streamed row costs a 4-byte load a column and one 16-byte load of the four rows' e.
// OUT: T, or float for the shares of shared heads.
template <typename T, typename OUT, bool OWN_KEYS, int NW, int NV>
__global__ void __launch_bounds__(THREADS, NW >= 6 ? 1 : 0) masked_bwd_simple_kernel(MaskedArgs a, const T *dvo, const float *lse, const float *delta, OUT *dx, OUT *dv, int tiles)
{
	extern __shared__ float4 smem4[];
	const int wp = pitch(a.width), vp = pitch(a.v_width), tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
	constexpr int GP = OWN + 4;
	// (columns past a row's pitch read the next row, the last ones' G: what they come to is not stored)
	float *A = reinterpret_cast<float *>(smem4), *B = A + OWN * wp, *C = B + OWN * vp, *D = C + STREAM * wp, *G = D + STREAM * vp, *P = G + STREAM * GP;
	const int bh = blockIdx.x % (a.bs * a.heads), rank = blockIdx.x / (a.bs * a.heads), tile = OWN_KEYS ? rank : tiles - 1 - rank; // what a causal mask leaves most work first
	const int head = bh % a.heads, b = bh / a.heads, kv = head / (a.heads / a.kv_heads);
	const MaskView mask(a, b);
	const int o0 = tile * OWN, o1 = min(a.n, o0 + OWN);
	const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f, slope = a.slopes ? a.slopes[head] : 0.f;
	const Strided go = {dvo, (long long)a.n * a.heads * a.v_width, (long long)a.heads * a.v_width, a.v_width};
	load_rows<T>(A, wp, wp, OWN_KEYS ? a.k : a.q, b, OWN_KEYS ? kv : head, o0, OWN, a.n, a.width);
	load_rows<T>(B, vp, vp, OWN_KEYS ? a.v : go, b, OWN_KEYS ? kv : head, o0, OWN, a.n, a.v_width);
	__syncthreads();
	float own[4][NW], acc[4][NW], accv[4][OWN_KEYS ? NV : 1];
#pragma unroll
	for (int i = 0; i < 4; i++) {
#pragma unroll
		for (int c = 0; c < NW; c++) {
			own[i][c] = A[(4 * ty + i) * wp + tx + 16 * c];
			acc[i][c] = 0.f;
		}
#pragma unroll
		for (int c = 0; c < (OWN_KEYS ? NV : 1); c++)
			accv[i][c] = 0.f;
	}
	for (int r0 = 0; r0 < a.n; r0 += STREAM) {
		const int r1 = min(a.n, r0 + STREAM);
		if (OWN_KEYS ? !mask.any(r0, r1, o0, o1) : !mask.any(o0, o1, r0, r1))
			continue;
		__syncthreads();
		load_rows<T>(C, wp, wp, OWN_KEYS ? a.q : a.k, b, OWN_KEYS ? head : kv, r0, STREAM, a.n, a.width);
		const bool odd = __syncthreads_or(load_rows<T>(D, vp, vp, OWN_KEYS ? go : a.v, b, OWN_KEYS ? head : kv, r0, STREAM, a.n, a.v_width));
		constexpr int J = STREAM / 16;
		const bool whole = r1 == r0 + STREAM && o1 == o0 + OWN && (OWN_KEYS ? mask.all(r0, r1, o0, o1) : mask.all(o0, o1, r0, r1));
		float x[4][J], dp[4][J];
		distances<J>(A, C, wp, a.width, ty, tx, x);
		products<J>(B, D, vp, a.v_width, ty, tx, dp);
#pragma unroll
		for (int j = 0; j < J; j++) {
			float e[4], p[4];
#pragma unroll
			for (int i = 0; i < 4; i++) {
				const int o = o0 + 4 * ty + i, r = r0 + tx + 16 * j, t = OWN_KEYS ? r : o, s = OWN_KEYS ? o : r;
				p[i] = e[i] = 0.f;
				if (whole || (t < a.n && s < a.n && mask.sees(t, s, mask.doc ? mask.doc[t] : 0, mask.doc ? mask.doc[s] : 0))) {
					const long long row = ((long long)b * a.n + t) * a.heads + head;
					float y = -a.scale * x[i][j], slant = 1.f;
					if (a.cap > 0.f) {
						const float th = tanhf(y * inv_cap);
						slant = 1.f - th * th;
						y = a.cap * th;
					}
					p[i] = weight_of(y - slope * fabsf(float(t - s)), lse[row]);
					if (p[i] != 0.f)
						e[i] = -a.scale * slant * p[i] * (dp[i][j] - delta[row]);
				}
			}
			*reinterpret_cast<float4 *>(G + (tx + 16 * j) * GP + 4 * ty) = make_float4(e[0], e[1], e[2], e[3]);
			if (OWN_KEYS)
				*reinterpret_cast<float4 *>(P + (tx + 16 * j) * GP + 4 * ty) = make_float4(p[0], p[1], p[2], p[3]);
		}
		__syncwarp(); // (a half-warp's rows are its own)
		for (int r = 0; r < r1 - r0; r++) {
			const float4 e4 = *reinterpret_cast<const float4 *>(G + r * GP + 4 * ty);
			const float e[4] = {e4.x, e4.y, e4.z, e4.w}, minus[4] = {-e4.x, -e4.y, -e4.z, -e4.w};
#pragma unroll
			for (int c = 0; c < NW; c++) {
				const float y = C[r * wp + tx + 16 * c];
#pragma unroll
				for (int i = 0; i < 4; i++)
					add_by_sign(acc[i][c], own[i][c], y, e[i], minus[i]);
			}
			if (OWN_KEYS) {
				const float4 p4 = *reinterpret_cast<const float4 *>(P + r * GP + 4 * ty);
				const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
				for (int c = 0; c < NV; c++) {
					const float y = D[r * vp + tx + 16 * c];
#pragma unroll
					for (int i = 0; i < 4; i++)
						if (!odd || p[i] != 0.f)
							accv[i][c % (OWN_KEYS ? NV : 1)] = fmaf(p[i], y, accv[i][c % (OWN_KEYS ? NV : 1)]);
				}
			}
		}
	}
#pragma unroll
	for (int i = 0; i < 4; i++) {
		const int o = o0 + 4 * ty + i;
		if (o >= a.n)
			continue;
		const long long row = ((long long)b * a.n + o) * a.heads + head;
#pragma unroll
		for (int c = 0; c < NW; c++)
			if (tx + 16 * c < a.width)
				dx[row * a.width + tx + 16 * c] = from_float<OUT>(acc[i][c]);
		if (OWN_KEYS)
#pragma unroll
			for (int c = 0; c < NV; c++)
				if (tx + 16 * c < a.v_width)
					dv[row * a.v_width + tx + 16 * c] = from_float<OUT>(accv[i][c % (OWN_KEYS ? NV : 1)]);
	}
}

int grid_of(long long n, unsigned *out)
{
	if (n > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	*out = unsigned(n);
	return L1ATTN_OK;
}

inline int fwd_bytes(int width, int nv, int keys) { return 4 * ((OWN + keys) * pitch(width) + keys * 64 * nv + OWN * (keys + 4)); }

template <typename T, int NV, int KEYS> int fwd_tiles(const MaskedArgs &a, void *vo, void *rest, float *lse, cudaStream_t st)
{
	const int tiles = (a.n + OWN - 1) / OWN, bytes = fwd_bytes(a.width, NV, KEYS);
	unsigned grid = 0;
	if (int rc = grid_of((long long)tiles * a.heads * a.bs, &grid))
		return rc;
	L1B_SHARED_MEMORY((masked_fwd_simple_kernel<T, NV, KEYS>), bytes);
	masked_fwd_simple_kernel<T, NV, KEYS><<<grid, THREADS, bytes, st>>>(a, static_cast<T *>(vo), static_cast<T *>(rest), lse, tiles);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

// Tiles of 32 keys where two CTAs of them fit an SM and two of 64 keys do not, else of 64.  64 against 32: [2,2048,8,64], causal, 402 / 474 us,
// [3,501,6,65] with values of 40 94 / 117, [1,1000,8,200] 378 / 440 (one CTA either way); but [2,2048,8,128] 865 / 725.
template <typename T, int NV> int fwd(const MaskedArgs &a, void *vo, void *rest, float *lse, cudaStream_t st)
{
	return fwd_bytes(a.width, NV, 64) > 113 * 1024 && fwd_bytes(a.width, NV, 32) <= 113 * 1024 ? fwd_tiles<T, NV, 32>(a, vo, rest, lse, st) : fwd_tiles<T, NV, 64>(a, vo, rest, lse, st);
}

template <typename T, typename OUT, bool OWN_KEYS, int NW, int NV>
int bwd_one(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, OUT *dx, OUT *dv, cudaStream_t st)
{
	const int tiles = (a.n + OWN - 1) / OWN;
	const int bytes = 4 * ((OWN + STREAM) * (pitch(a.width) + pitch(a.v_width)) + (OWN_KEYS ? 2 : 1) * STREAM * (OWN + 4)); // (G alone takes in what is read past C and D)
	unsigned grid = 0;
	if (int rc = grid_of((long long)tiles * a.heads * a.bs, &grid))
		return rc;
	L1B_SHARED_MEMORY((masked_bwd_simple_kernel<T, OUT, OWN_KEYS, NW, NV>), bytes);
	masked_bwd_simple_kernel<T, OUT, OWN_KEYS, NW, NV><<<grid, THREADS, bytes, st>>>(a, static_cast<const T *>(dvo), lse, delta, dx, dv, tiles);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

template <typename T, int NW, int NV>
int bwd(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, cudaStream_t st)
{
	if (int rc = bwd_one<T, T, false, NW, NV>(a, dvo, lse, delta, static_cast<T *>(dq), static_cast<T *>(nullptr), st))
		return rc;
	if (a.heads != a.kv_heads)
		return bwd_one<T, float, true, NW, NV>(a, dvo, lse, delta, shares, shares + (long long)a.bs * a.n * a.heads * a.width, st);
	return bwd_one<T, T, true, NW, NV>(a, dvo, lse, delta, static_cast<T *>(dk), static_cast<T *>(dv), st);
}

template <typename T> int fwd_type(const MaskedArgs &a, void *vo, void *rest, float *lse, cudaStream_t st)
{
	if constexpr (sizeof(T) == 2) // (smaller ones of 16 bits are done on the tensor cores)
		return fwd<T, 4>(a, vo, rest, lse, st);
	else
	return a.v_width <= 64 ? fwd<T, 1>(a, vo, rest, lse, st) : a.v_width <= 128 ? fwd<T, 2>(a, vo, rest, lse, st) : fwd<T, 4>(a, vo, rest, lse, st);
}
// columns a thread, for the width and for the values: 32, 64, 96, 128, 256 columns in all
template <typename T, int NW>
int bwd_values(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, cudaStream_t st)
{
	return a.v_width <= 64 ? bwd<T, NW, 4>(a, dvo, lse, delta, dq, dk, dv, shares, st) : a.v_width <= 128 ? bwd<T, NW, 8>(a, dvo, lse, delta, dq, dk, dv, shares, st) :
														       bwd<T, NW, 16>(a, dvo, lse, delta, dq, dk, dv, shares, st);
}
template <typename T>
int bwd_type(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, cudaStream_t st)
{
	if constexpr (sizeof(T) == 2) // (smaller ones of 16 bits are done on the tensor cores)
		return bwd<T, 16, 16>(a, dvo, lse, delta, dq, dk, dv, shares, st);
	else
	return a.width <= 32 ? bwd_values<T, 2>(a, dvo, lse, delta, dq, dk, dv, shares, st) : a.width <= 64 ? bwd_values<T, 4>(a, dvo, lse, delta, dq, dk, dv, shares, st) :
	       a.width <= 96 ? bwd_values<T, 6>(a, dvo, lse, delta, dq, dk, dv, shares, st) : a.width <= 128 ? bwd_values<T, 8>(a, dvo, lse, delta, dq, dk, dv, shares, st) :
														bwd_values<T, 16>(a, dvo, lse, delta, dq, dk, dv, shares, st);
}

} // namespace

int masked_simple_fwd_launch(const MaskedArgs &a, void *vo, void *rest, float *lse, int dtype, cudaStream_t st)
{
	return dtype == L1ATTN_F32 ? fwd_type<float>(a, vo, rest, lse, st) : dtype == L1ATTN_F16 ? fwd_type<__half>(a, vo, rest, lse, st) :
											     fwd_type<__nv_bfloat16>(a, vo, rest, lse, st);
}

int masked_simple_bwd_launch(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, int dtype,
			     cudaStream_t st)
{
	return dtype == L1ATTN_F32 ? bwd_type<float>(a, dvo, lse, delta, dq, dk, dv, shares, st) :
	       dtype == L1ATTN_F16 ? bwd_type<__half>(a, dvo, lse, delta, dq, dk, dv, shares, st) :
				     bwd_type<__nv_bfloat16>(a, dvo, lse, delta, dq, dk, dv, shares, st);
}

} // namespace l1b
