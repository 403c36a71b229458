// Attention of new tokens to a paged cache in 8 bits: the kernel of float32 arithmetic for every type and width, and the one that joins splits.
//
// A CTA takes 16 rows -- consecutive (token, query head of the group) pairs of one sequence, which all read the same keys -- and one range of
// split_keys keys; codes become floats in shared memory, 64 keys at a time.  Running softmax as in masked_simple.cu.
#include "cache.cuh"

namespace l1b {

namespace {

constexpr int ROWS = 16, KEYS = 64, THREADS = 256;

__host__ __device__ inline int pitch(int w)
{
	const int p = (w + 3) / 4;
	return 4 * (p % 2 ? p : p + 1);
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

template <typename T, int NV> __global__ void __launch_bounds__(THREADS) attend_simple_kernel(AttendArgs a)
{
	extern __shared__ float4 smem4[];
	const CacheArgs &c = a.c;
	const int wp = pitch(c.width), vp = 64 * NV, tid = threadIdx.x, tx = tid % 16, ty = tid / 16, kv = blockIdx.y;
	constexpr int PP = KEYS + 4;
	float *Q = reinterpret_cast<float *>(smem4), *K = Q + ROWS * wp, *V = K + KEYS * wp, *P = V + KEYS * vp;
	int *there = reinterpret_cast<int *>(P + ROWS * PP); // keys whose page is in range
	const int seq = cache_find_warp(c, blockIdx.x, a.group, a.tile_rows, 1);
	const SeqView sv = cache_seq(c, seq);
	const long long first = (blockIdx.x - cache_first_unit(c, seq, a.group, a.tile_rows, 1)) * ROWS, all = (long long)sv.count * a.group;
	const long long ends = min(first + ROWS, all + (long long)sv.lost * a.group);
	if (first < 0 || first >= ends)
		return;
	if (!a.part) // rows without a place (else attend_merge_kernel's)
		for (long long lr = max(first, all); lr < ends; lr++)
			for (int w = tid; w < c.v_width; w += THREADS)
				static_cast<T *>(a.vo)[((sv.row + lr / a.group) * a.heads + kv * a.group + lr % a.group) * c.v_width + w] = from_float<T>(0.f);
	if (first >= all)
		return;
	const long long last = min(first + ROWS, all) - 1;
	const int t_lo = sv.start + int(first / a.group), t_hi = sv.start + int(last / a.group);
	int lo = a.window ? max(0, t_lo - a.window + 1) : 0, hi = t_hi + 1;
	lo = max(lo, int(min((long long)blockIdx.z * a.split_keys, (long long)hi)));
	if (blockIdx.z + 1 < a.splits) // (the last split takes whatever is left)
		hi = int(min((long long)hi, (long long)(blockIdx.z + 1) * a.split_keys));
	const bool mine = first + ty <= last;
	const int row = sv.row + int(mine ? (first + ty) / a.group : 0), head = kv * a.group + int((first + ty) % a.group), t = sv.start + row - sv.row;
	const float slope = a.slopes ? a.slopes[head] : 0.f, inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
	for (int i = tid; i < ROWS * wp; i += THREADS) {
		const int r = i / wp, w = i % wp;
		const long long lr = first + r;
		Q[i] = lr <= last && w < c.width ? to_float(static_cast<const T *>(a.q)[(sv.row + lr / a.group) * a.q_row + (kv * a.group + lr % a.group) * a.q_head + w]) : 0.f;
	}
	float m = -INFINITY, l = 0.f, acc[4 * NV];
#pragma unroll
	for (int i = 0; i < 4 * NV; i++)
		acc[i] = 0.f;
	for (int s0 = lo / KEYS * KEYS; s0 < hi; s0 += KEYS) {
		__syncthreads();
		for (int s = tid / 32; s < KEYS; s += THREADS / 32) {
			const int pos = s0 + s, id = pos >= lo && pos < hi ? cache_page(c, seq, pos / c.page) : -1; // (pages before a window may have gone)
			const long long at = (long long)max(id, 0) * c.kv_heads + kv, r = at * c.page + pos % c.page;
			if (tid % 32 == 0)
				there[s] = id >= 0;
			for (int w = tid % 32; w < wp; w += 32)
				K[s * wp + w] = id >= 0 && w < c.width ? c.k_codes[r * c.width + w] * c.k_scale[at] : 0.f;
			for (int w = tid % 32; w < vp; w += 32)
				V[s * vp + w] = id >= 0 && w < c.v_width ? c.v_codes[r * c.v_width + w] * c.v_scale[at] : 0.f;
		}
		__syncthreads();
		float x[4], top = m;
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const float *q = Q + ty * wp, *k = K + (tx + 16 * j) * wp;
			float d = 0.f;
			for (int w = 0; w < c.width; w += 4) {
				const float4 y = *reinterpret_cast<const float4 *>(q + w), z = *reinterpret_cast<const float4 *>(k + w);
				d += (fabsf(y.x - z.x) + fabsf(y.y - z.y)) + (fabsf(y.z - z.z) + fabsf(y.w - z.w));
			}
			const int s = s0 + tx + 16 * j;
			float y = -a.scale * d;
			if (a.cap > 0.f)
				y = a.cap * tanhf(y * inv_cap);
			y -= slope * float(t - s);
			x[j] = mine && there[tx + 16 * j] && s >= lo && s < hi && s <= t && (a.window == 0 || t - s < a.window) ? y : -INFINITY;
			top = fmaxf(top, x[j]);
		}
		top = half_warp_max(top);
		const float ref = top == -INFINITY ? 0.f : top, keep = expf(m - ref);
		float sum = 0.f;
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const float p = expf(x[j] - ref);
			sum += p;
			P[ty * PP + tx + 16 * j] = p;
		}
		l = l * keep + half_warp_sum(sum);
		m = top;
#pragma unroll
		for (int i = 0; i < 4 * NV; i++)
			acc[i] *= keep;
		__syncwarp();
		for (int s = 0; s < KEYS; s++) {
			const float p = P[ty * PP + s];
#pragma unroll
			for (int u = 0; u < NV; u++) {
				const float4 v = *reinterpret_cast<const float4 *>(V + s * vp + 64 * u + 4 * tx);
				acc[4 * u] = fmaf(p, v.x, acc[4 * u]);
				acc[4 * u + 1] = fmaf(p, v.y, acc[4 * u + 1]);
				acc[4 * u + 2] = fmaf(p, v.z, acc[4 * u + 2]);
				acc[4 * u + 3] = fmaf(p, v.w, acc[4 * u + 3]);
			}
		}
	}
	if (!mine)
		return;
	const long long at = (long long)row * a.heads + head;
	if (a.part) {
		float *out = a.part + ((long long)blockIdx.z * c.rows * a.heads + at) * (c.v_width + 2);
		if (tx == 0) {
			out[0] = m;
			out[1] = l;
		}
#pragma unroll
		for (int i = 0; i < 4 * NV; i++)
			if (const int w = 64 * (i / 4) + 4 * tx + i % 4; w < c.v_width)
				out[2 + w] = acc[i];
		return;
	}
	const float f = finish_softmax(a.mode, m, l);
#pragma unroll
	for (int i = 0; i < 4 * NV; i++)
		if (const int w = 64 * (i / 4) + 4 * tx + i % 4; w < c.v_width)
			static_cast<T *>(a.vo)[at * c.v_width + w] = from_float<T>(acc[i] * f);
}

// A warp per (row, head): joins the parts of the splits that reach the row's keys.
template <typename T> __global__ void __launch_bounds__(128) attend_merge_kernel(AttendArgs a)
{
	const CacheArgs &c = a.c;
	const long long unit = blockIdx.x * 4ll + threadIdx.x / 32;
	const int lane = threadIdx.x % 32;
	const long long row = unit / a.heads;
	if (row >= c.rows)
		return;
	const int seq = cache_find_row(c, row);
	const SeqView sv = cache_seq(c, seq);
	if (row < sv.row || row - sv.row >= (long long)sv.count + sv.lost)
		return;
	if (row - sv.row >= sv.count) { // a row without a place
		for (int w = lane; w < c.v_width; w += 32)
			static_cast<T *>(a.vo)[unit * c.v_width + w] = from_float<T>(0.f);
		return;
	}
	const int t = sv.start + int(row - sv.row);
	const int parts = min(a.splits, t / a.split_keys + 1);
	const float *part = a.part + unit * (c.v_width + 2);
	const long long step = (long long)c.rows * a.heads * (c.v_width + 2);
	float m = -INFINITY, l = 0.f;
	for (int i = lane; i < parts; i += 32)
		m = fmaxf(m, part[i * step]);
#pragma unroll
	for (int o = 16; o; o >>= 1)
		m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
	const float ref = m == -INFINITY ? 0.f : m;
	for (int i = lane; i < parts; i += 32)
		l += part[i * step + 1] * expf(part[i * step] - ref);
#pragma unroll
	for (int o = 16; o; o >>= 1)
		l += __shfl_xor_sync(0xffffffffu, l, o);
	const float f = finish_softmax(a.mode, m, l);
	for (int w = lane; w < c.v_width; w += 32) {
		float sum = 0.f;
		for (int i = 0; i < parts; i++) {
			const float e = expf(part[i * step] - ref);
			sum += e == 0.f ? 0.f : e * part[i * step + 2 + w];
		}
		static_cast<T *>(a.vo)[unit * c.v_width + w] = from_float<T>(sum * f);
	}
}

template <typename T, int NV> int simple(const AttendArgs &a, cudaStream_t st)
{
	const int wp = pitch(a.c.width), bytes = 4 * (ROWS * wp + KEYS * wp + KEYS * 64 * NV + ROWS * (KEYS + 4) + KEYS);
	const long long tiles = (long long)a.c.rows * a.group / ROWS + a.c.n_seqs;
	if (tiles > 0x7fffffffll || a.c.kv_heads > 65535 || a.splits > 65535)
		return L1ATTN_ERR_SHAPE;
	L1B_SHARED_MEMORY((attend_simple_kernel<T, NV>), bytes);
	attend_simple_kernel<T, NV><<<dim3(unsigned(tiles), a.c.kv_heads, a.splits), THREADS, bytes, st>>>(a);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

template <typename T> int simple_type(const AttendArgs &a, cudaStream_t st)
{
	return a.c.v_width <= 64 ? simple<T, 1>(a, st) : a.c.v_width <= 128 ? simple<T, 2>(a, st) : simple<T, 4>(a, st);
}

} // namespace

int attend_simple_launch(const AttendArgs &a, int dtype, cudaStream_t st)
{
	return dtype == L1ATTN_F32 ? simple_type<float>(a, st) : dtype == L1ATTN_F16 ? simple_type<__half>(a, st) : simple_type<__nv_bfloat16>(a, st);
}

int attend_merge_launch(const AttendArgs &a, int dtype, cudaStream_t st)
{
	const long long blocks = ((long long)a.c.rows * a.heads + 3) / 4;
	if (blocks > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	if (dtype == L1ATTN_F32)
		attend_merge_kernel<float><<<unsigned(blocks), 128, 0, st>>>(a);
	else if (dtype == L1ATTN_F16)
		attend_merge_kernel<__half><<<unsigned(blocks), 128, 0, st>>>(a);
	else
		attend_merge_kernel<__nv_bfloat16><<<unsigned(blocks), 128, 0, st>>>(a);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

} // namespace l1b
