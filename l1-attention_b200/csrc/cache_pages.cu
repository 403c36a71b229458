// Pages of the 8-bit cache: quantising new tokens into them, reading sequences back, copying pages.
//
// All three are bound by memory: append reads a token's row twice (the second time from L1 or L2) and writes a quarter to a half of it,
// gather reads codes and writes values, copies read and write.
#include "cache.cuh"

namespace l1b {

namespace {

constexpr int THREADS = 128;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// x / s to the nearest whole number, ties to even, of the exact quotient: an estimate, put right by its residual, which one FMA gives
// exactly where it decides (it is a multiple of the smaller last bit and at most about s).  NaN is stored as 0, values beyond as +-127.
__device__ __forceinline__ int quantise(float x, float s, float inv)
{
	if (!finite(x) || s == 0.f)
		return x > 0.f && s > 0.f ? 127 : x < 0.f && s > 0.f ? -127 : 0;
	float q = rintf(inv < INFINITY ? x * inv : x / s);
	const float r = fmaf(-q, s, x), r2 = fabsf(r + r);
	if (r2 > s || (r2 == s && (int(q) & 1)))
		q += copysignf(1.f, r);
	return int(fminf(fmaxf(q, -127.f), 127.f));
}

// A CTA per (page that new tokens touch, head, keys or values): it alone reads and writes that page's rows and scale of that head.
template <typename T>
__global__ void __launch_bounds__(THREADS) append_kernel(CacheArgs c, const T *k, const T *v, long long k_row, long long k_head, long long v_row, long long v_head)
{
	const int seq = cache_find_warp(c, blockIdx.x, 1, c.page, 2), head = blockIdx.y, tid = threadIdx.x;
	const SeqView sv = cache_seq(c, seq);
	const long long unit = blockIdx.x - cache_first_unit(c, seq, 1, c.page, 2), slot = sv.start / c.page + unit;
	if (unit < 0 || sv.count == 0 || slot * c.page >= (long long)sv.start + sv.count)
		return;
	const int id = cache_page(c, seq, int(slot));
	if (id < 0)
		return;
	const bool values = blockIdx.z;
	const int w = values ? c.v_width : c.width, first = int(slot) * c.page;
	const int a = max(sv.start - first, 0), b = int(min((long long)sv.start + sv.count - first, (long long)c.page)); // new rows of the page
	const T *src = (values ? v : k) + (values ? v_head : k_head) * head + (long long)(sv.row + first - sv.start) * (values ? v_row : k_row);
	const long long src_row = values ? v_row : k_row, at = (long long)id * c.kv_heads + head;
	int8_t *codes = (values ? c.v_codes : c.k_codes) + at * c.page * w;
	float *scale = (values ? c.v_scale : c.k_scale) + at;

	float most = 0.f;
	for (int i = tid; i < (b - a) * w; i += THREADS) {
		const float x = fabsf(to_float(src[(a + i / w) * src_row + i % w]));
		most = finite(x) ? fmaxf(most, x) : most;
	}
	__shared__ float part[THREADS / 32];
#pragma unroll
	for (int o = 16; o; o >>= 1)
		most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
	if (tid % 32 == 0)
		part[tid / 32] = most;
	const float old = a > 0 ? *scale : 0.f;
	__syncthreads();
#pragma unroll
	for (int i = 0; i < THREADS / 32; i++)
		most = fmaxf(most, part[i]);
	const float now = fmaxf(most / 127.f, old), inv = 1.f / now;
	if (a > 0 && now > old) // the rows that were there follow the new scale
		for (int i = tid; i < a * w; i += THREADS)
			codes[i] = int8_t(rint(double(codes[i]) * double(old) / double(now)));
	for (int i = tid; i < (b - a) * w; i += THREADS)
		codes[a * w + i] = int8_t(quantise(to_float(src[(a + i / w) * src_row + i % w]), now, inv));
	if (tid == 0)
		*scale = now;
}

// A warp per (row, head): keys and values of the row
template <typename T> __global__ void __launch_bounds__(THREADS) gather_kernel(CacheArgs c, T *k, T *v)
{
	const long long unit = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
	const int lane = threadIdx.x % 32, head = int(unit % c.kv_heads);
	const long long row = unit / c.kv_heads;
	if (row >= c.rows)
		return;
	const int seq = cache_find_row(c, row);
	const SeqView sv = cache_seq(c, seq);
	if (row < sv.row || row - sv.row >= sv.count)
		return;
	const int pos = sv.start + int(row - sv.row), id = cache_page(c, seq, pos / c.page);
	const long long at = (long long)max(id, 0) * c.kv_heads + head;
	const float ks = id < 0 ? 0.f : c.k_scale[at], vs = id < 0 ? 0.f : c.v_scale[at];
	const int8_t *kc = c.k_codes + (at * c.page + pos % c.page) * c.width, *vc = c.v_codes + (at * c.page + pos % c.page) * c.v_width;
	for (int w = lane; w < c.width; w += 32)
		k[unit * c.width + w] = from_float<T>(id < 0 ? 0.f : kc[w] * ks);
	for (int w = lane; w < c.v_width; w += 32)
		v[unit * c.v_width + w] = from_float<T>(id < 0 ? 0.f : vc[w] * vs);
}

struct CopyArgs {
	uint4 *codes[2];
	float *scale[2];
	long long vecs[2]; // 16-byte vectors of a page
	int n_pages, kv_heads, n;
	const int32_t *src, *dst;
	int *status;
};

// grid: (pairs, pieces of a page, layers x {keys, values})
__global__ void __launch_bounds__(256) copy_pages_kernel(CopyArgs c)
{
	const int kind = blockIdx.z & 1;
	const long long layer = blockIdx.z >> 1;
	const int from = c.src[blockIdx.x], to = c.dst[blockIdx.x];
	if (from < 0 || from >= c.n_pages || to < 0 || to >= c.n_pages) {
		if (c.status && threadIdx.x == 0)
			*reinterpret_cast<volatile int *>(c.status) = L1ATTN_ERR_INDEX;
		return;
	}
	const uint4 *a = c.codes[kind] + (layer * c.n_pages + from) * c.vecs[kind];
	uint4 *b = c.codes[kind] + (layer * c.n_pages + to) * c.vecs[kind];
	for (long long i = blockIdx.y * 256ll + threadIdx.x; i < c.vecs[kind]; i += gridDim.y * 256ll)
		b[i] = a[i];
	if (blockIdx.y == 0)
		for (int i = threadIdx.x; i < c.kv_heads; i += 256)
			c.scale[kind][(layer * c.n_pages + to) * c.kv_heads + i] = c.scale[kind][(layer * c.n_pages + from) * c.kv_heads + i];
}

} // namespace

int append_launch(const CacheArgs &c, const void *k, const void *v, const long long *strides, int dtype, cudaStream_t st)
{
	const long long units = (long long)c.rows / c.page + 2ll * c.n_seqs;
	if (units > 0x7fffffffll || c.kv_heads > 65535)
		return L1ATTN_ERR_SHAPE;
	const dim3 grid(unsigned(units), c.kv_heads, 2);
	if (dtype == L1ATTN_F32)
		append_kernel<<<grid, THREADS, 0, st>>>(c, static_cast<const float *>(k), static_cast<const float *>(v), strides[0], strides[1], strides[2], strides[3]);
	else if (dtype == L1ATTN_F16)
		append_kernel<<<grid, THREADS, 0, st>>>(c, static_cast<const __half *>(k), static_cast<const __half *>(v), strides[0], strides[1], strides[2], strides[3]);
	else
		append_kernel<<<grid, THREADS, 0, st>>>(c, static_cast<const __nv_bfloat16 *>(k), static_cast<const __nv_bfloat16 *>(v), strides[0], strides[1], strides[2],
							strides[3]);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

int gather_launch(const CacheArgs &c, void *k, void *v, int dtype, cudaStream_t st)
{
	const long long units = ((long long)c.rows * c.kv_heads + THREADS / 32 - 1) / (THREADS / 32);
	if (units > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	if (dtype == L1ATTN_F32)
		gather_kernel<<<unsigned(units), THREADS, 0, st>>>(c, static_cast<float *>(k), static_cast<float *>(v));
	else if (dtype == L1ATTN_F16)
		gather_kernel<<<unsigned(units), THREADS, 0, st>>>(c, static_cast<__half *>(k), static_cast<__half *>(v));
	else
		gather_kernel<<<unsigned(units), THREADS, 0, st>>>(c, static_cast<__nv_bfloat16 *>(k), static_cast<__nv_bfloat16 *>(v));
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

int copy_pages_launch(const CacheArgs &c, int layers, const int32_t *src, const int32_t *dst, int n, cudaStream_t st)
{
	CopyArgs a = {{reinterpret_cast<uint4 *>(c.k_codes), reinterpret_cast<uint4 *>(c.v_codes)},
		      {c.k_scale, c.v_scale},
		      {(long long)c.kv_heads * c.page * c.width / 16, (long long)c.kv_heads * c.page * c.v_width / 16},
		      c.n_pages, c.kv_heads, n, src, dst, c.status};
	if (layers > 32767)
		return L1ATTN_ERR_SHAPE;
	const long long most = a.vecs[0] > a.vecs[1] ? a.vecs[0] : a.vecs[1];
	long long pieces = (most + 1023) / 1024; // four vectors a thread
	pieces = pieces < 1 ? 1 : pieces > 65535 ? 65535 : pieces;
	copy_pages_kernel<<<dim3(n, unsigned(pieces), 2 * layers), 256, 0, st>>>(a);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

} // namespace l1b
