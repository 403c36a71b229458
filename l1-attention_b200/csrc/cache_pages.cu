// Pages of the 8-bit cache: quantising new tokens into them, reading sequences back, copying pages.
//
// All three are bound by memory, or by the chain of reads that leads to it (offsets, start, page, scale: about 4 us).  8 heads of 128 and 128: 16 prompts of up to
// 1501 tokens appended and read back 52 us (floor 27), 64 single tokens and their sequences of about 130 read back 22 us (12); 4096 pages of 131 KB
// copied 195 us (85 % of the rate of a copy).
#include <type_traits>
#include "cache.cuh"

namespace l1b {

namespace {

constexpr int THREADS = 128;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// x / s to the nearest whole number, ties to even, of the exact quotient: an estimate, put right by its residual, which one FMA gives
// exactly where it decides (it is a multiple of the smaller last bit and at most about s).  NaN is stored as 0, values beyond as +-127.
__device__ __noinline__ int quantise_any(float x, float s, float inv)
{
	if (!finite(x) || s == 0.f)
		return x > 0.f && s > 0.f ? 127 : x < 0.f && s > 0.f ? -127 : 0;
	float q = rintf(inv < INFINITY ? x * inv : x / s);
	const float r = fmaf(-q, s, x), r2 = fabsf(r + r);
	if (r2 > s || (r2 == s && (int(q) & 1)))
		q += copysignf(1.f, r);
	return int(fminf(fmaxf(q, -127.f), 127.f));
}
// The same in the low byte, for sure where *near stays true: 1.5 * 2^23 leaves the whole number in the low bits of the sum, and the residual says that it is
// the nearest (almost always).  half: s / 2, or 0 where that is not exact.
__device__ __forceinline__ uint32_t quantise_near(float x, float s, float inv, float half, bool *near)
{
	const float t = fmaf(x, inv, 12582912.f), r = fmaf(12582912.f - t, s, x);
	*near = *near && fabsf(r) < half;
	return __float_as_uint(t);
}

template <typename T> struct Vector { // 16 bytes of tokens
	static constexpr int N = 16 / sizeof(T);
};
// bits of a value without its sign: ordered as the values are, infinities and NaN behind all others
template <typename T> struct Bits;
template <> struct Bits<float> {
	static constexpr uint32_t ALL = 0x7fffffffu, INF = 0x7f800000u;
};
template <> struct Bits<__half> {
	static constexpr uint32_t ALL = 0x7fff7fffu, INF = 0x7c00u;
};
template <> struct Bits<__nv_bfloat16> {
	static constexpr uint32_t ALL = 0x7fff7fffu, INF = 0x7f80u;
};

// A CTA per (page that new tokens touch, head, keys or values): it alone reads and writes that page's rows and scale of that head.
// HELD: 16-byte vectors of its new rows that a thread keeps between the scale and the codes (0: element by element, the rows are read twice).
template <typename T, int HELD>
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
	const long long src_row = values ? v_row : k_row, at = (long long)id * c.kv_heads + head;
	const T *src = (values ? v : k) + (values ? v_head : k_head) * head + (long long)(sv.row + first - sv.start + a) * src_row; // the first new row
	int8_t *const codes = (values ? c.v_codes : c.k_codes) + at * c.page * w;
	float *const scale = (values ? c.v_scale : c.k_scale) + at;
	const float old = a > 0 ? *scale : 0.f;

	constexpr int N = Vector<T>::N;
	const int per_row = w / N, vectors = (b - a) * per_row;
	uint4 held[HELD ? HELD : 1];
	float most = 0.f;
	if (HELD) {
#pragma unroll
		for (int j = 0; j < HELD; j++) {
			const int i = tid + j * THREADS;
			if (i >= vectors)
				break;
			held[j] = *reinterpret_cast<const uint4 *>(src + (i / per_row) * src_row + i % per_row * N);
		}
		uint32_t top = 0; // the largest bits, two of a word where values are of 16
#pragma unroll
		for (int j = 0; j < HELD; j++) {
			if (tid + j * THREADS >= vectors)
				break;
			for (uint32_t word : {held[j].x, held[j].y, held[j].z, held[j].w})
				top = N == 8 ? __vmaxu2(top, word & Bits<T>::ALL) : max(top, word & Bits<T>::ALL);
		}
		if (N == 8)
			top = max(top >> 16, top & 0xffffu);
		if (top < Bits<T>::INF)
			most = to_float(*reinterpret_cast<const T *>(&top));
		else // what is not finite does not count
#pragma unroll
			for (int j = 0; j < HELD; j++) {
				if (tid + j * THREADS >= vectors)
					break;
#pragma unroll
				for (int e = 0; e < N; e++) {
					const float x = fabsf(to_float(reinterpret_cast<const T *>(&held[j])[e]));
					most = finite(x) ? fmaxf(most, x) : most;
				}
			}
	} else
		for (int i = tid; i < (b - a) * w; i += THREADS) {
			const float x = fabsf(to_float(src[(i / w) * src_row + i % w]));
			most = finite(x) ? fmaxf(most, x) : most;
		}
	__shared__ float part[THREADS / 32];
#pragma unroll
	for (int o = 16; o; o >>= 1)
		most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
	if (tid % 32 == 0)
		part[tid / 32] = most;
	__syncthreads(); // (the scale has been read by all)
#pragma unroll
	for (int i = 0; i < THREADS / 32; i++)
		most = fmaxf(most, part[i]);
	const float now = fmaxf(most / 127.f, old), inv = 1.f / now, half = now >= 0x1p-125f ? 0.5f * now : 0.f;
	if (a > 0 && now > old) // the rows that were there follow the new scale
		for (int i = tid; i < a * w; i += THREADS)
			codes[i] = int8_t(rint(double(codes[i]) * double(old) / double(now)));
	if (HELD) {
#pragma unroll
		for (int j = 0; j < HELD; j++) {
			const int i = tid + j * THREADS;
			if (i >= vectors)
				break;
			uint32_t out[N / 4], q[N];
			bool near = true;
#pragma unroll
			for (int e = 0; e < N; e++)
				q[e] = quantise_near(to_float(reinterpret_cast<const T *>(&held[j])[e]), now, inv, half, &near);
			if (!near)
#pragma unroll
				for (int e = 0; e < N; e++)
					q[e] = uint32_t(quantise_any(to_float(reinterpret_cast<const T *>(&held[j])[e]), now, inv));
#pragma unroll
			for (int i = 0; i < N / 4; i++)
				out[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
			int8_t *const to = codes + (long long)a * w + i * N;
			if constexpr (N == 8)
				*reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[1]);
			else
				*reinterpret_cast<uint32_t *>(to) = out[0];
		}
	} else
		for (int i = tid; i < (b - a) * w; i += THREADS)
			codes[a * w + i] = int8_t(quantise_any(to_float(src[(i / w) * src_row + i % w]), now, inv));
	if (tid == 0)
		*scale = now;
}

// A warp per row: its keys and values, 16 bytes of them at a time where widths allow it (VEC), else one by one.
template <typename T, bool VEC> __global__ void __launch_bounds__(THREADS) gather_kernel(CacheArgs c, T *k, T *v)
{
	const long long row = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
	const int lane = threadIdx.x % 32;
	if (row >= c.rows)
		return;
	const int seq = cache_find_warp(c, row, 1, 1, 0);
	const SeqView sv = cache_seq(c, seq);
	const bool placed = row >= sv.row && row - sv.row < sv.count; // (else zeros, for all that offsets out of order leave to nobody, but behind the last sequence)
	if (!placed && !(row >= sv.row && row - sv.row < (long long)sv.count + sv.lost) && (row < cache_row(c, 0) || row >= cache_row(c, c.n_seqs)))
		return;
	const int pos = placed ? sv.start + int(row - sv.row) : 0, id = placed ? cache_page(c, seq, pos / c.page) : -1;
	const long long at = (long long)max(id, 0) * c.kv_heads;
	for (int values = 0; values < 2; values++) {
		const int w = values ? c.v_width : c.width;
		const int8_t *const codes = (values ? c.v_codes : c.k_codes) + (at * c.page + pos % c.page) * w;
		const float *const scale = (values ? c.v_scale : c.k_scale) + at;
		T *const out = (values ? v : k) + row * c.kv_heads * w;
		const long long head = (long long)c.page * w;
		if (VEC) {
			constexpr int N = Vector<T>::N, AT_ONCE = 4; // vectors of a lane whose reads do not wait for one another
			const unsigned per_head = w / N, all = c.kv_heads * per_head;
			const unsigned over = 0xffffffffu / per_head + 1; // i / per_head = the high half of i * over: exact for i < 2^32 / per_head; 1: itself
			for (unsigned i0 = lane; i0 < all; i0 += 32 * AT_ONCE) {
				uint32_t x[AT_ONCE][N / 4];
				float s[AT_ONCE];
#pragma unroll
				for (int j = 0; j < AT_ONCE; j++) {
					const unsigned i = min(i0 + 32 * j, all - 1), h = per_head == 1 ? i : __umulhi(i, over);
					const int8_t *const from = codes + h * head + (i - h * per_head) * N;
					if constexpr (N == 8) {
						const uint2 y = *reinterpret_cast<const uint2 *>(from);
						x[j][0] = y.x, x[j][N / 4 - 1] = y.y;
					} else
						x[j][0] = *reinterpret_cast<const uint32_t *>(from);
					s[j] = scale[h];
				}
#pragma unroll
				for (int j = 0; j < AT_ONCE; j++) {
					uint4 y;
#pragma unroll
					for (int e = 0; e < N; e++) // (a page out of range: zeros, whatever has been read)
						reinterpret_cast<T *>(&y)[e] = from_float<T>(id < 0 ? 0.f : float(int8_t(x[j][e / 4] >> 8 * (e % 4))) * s[j]);
					if (i0 + 32 * j < all)
						reinterpret_cast<uint4 *>(out)[i0 + 32 * j] = y;
				}
			}
		} else
			for (int i = lane; i < c.kv_heads * w; i += 32)
				out[i] = from_float<T>(id < 0 ? 0.f : codes[i / w * head + i % w] * scale[i / w]);
	}
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
	for (long long i = blockIdx.y * 1024ll + threadIdx.x; i < c.vecs[kind]; i += gridDim.y * 1024ll) { // four vectors of a thread at once
		uint4 x[4];
#pragma unroll
		for (int j = 0; j < 4; j++)
			if (i + 256 * j < c.vecs[kind])
				x[j] = a[i + 256 * j];
#pragma unroll
		for (int j = 0; j < 4; j++)
			if (i + 256 * j < c.vecs[kind])
				b[i + 256 * j] = x[j];
	}
	if (blockIdx.y == 0)
		for (int i = threadIdx.x; i < c.kv_heads; i += 256)
			c.scale[kind][(layer * c.n_pages + to) * c.kv_heads + i] = c.scale[kind][(layer * c.n_pages + from) * c.kv_heads + i];
}

} // namespace

namespace {
template <typename T> int append_type(const CacheArgs &c, const void *k_, const void *v_, const long long *st4, dim3 grid, cudaStream_t st)
{
	const T *k = static_cast<const T *>(k_), *v = static_cast<const T *>(v_);
	constexpr int N = Vector<T>::N;
	bool vec = aligned(k, 16) && aligned(v, 16) && c.width % N == 0 && c.v_width % N == 0;
	for (int i = 0; i < 4; i++)
		vec = vec && st4[i] % N == 0;
	// vectors of a page's rows, at most, by thread
	const int wide = c.width > c.v_width ? c.width : c.v_width, most = (c.page * (wide / N) + THREADS - 1) / THREADS;
	if (vec && most <= 8)
		append_kernel<T, 8><<<grid, THREADS, 0, st>>>(c, k, v, st4[0], st4[1], st4[2], st4[3]);
	else if (vec && most <= 16)
		append_kernel<T, 16><<<grid, THREADS, 0, st>>>(c, k, v, st4[0], st4[1], st4[2], st4[3]);
	else
		append_kernel<T, 0><<<grid, THREADS, 0, st>>>(c, k, v, st4[0], st4[1], st4[2], st4[3]);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}
} // namespace

int append_launch(const CacheArgs &c, const void *k, const void *v, const long long *strides, int dtype, cudaStream_t st)
{
	const long long units = (long long)c.rows / c.page + 2ll * c.n_seqs;
	if (units > 0x7fffffffll || c.kv_heads > 65535)
		return L1ATTN_ERR_SHAPE;
	const dim3 grid(unsigned(units), c.kv_heads, 2);
	if (dtype == L1ATTN_F32)
		return append_type<float>(c, k, v, strides, grid, st);
	return dtype == L1ATTN_F16 ? append_type<__half>(c, k, v, strides, grid, st) : append_type<__nv_bfloat16>(c, k, v, strides, grid, st);
}

int gather_launch(const CacheArgs &c, void *k, void *v, int dtype, cudaStream_t st)
{
	const long long blocks = ((long long)c.rows + THREADS / 32 - 1) / (THREADS / 32);
	if (blocks > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	const int n = dtype == L1ATTN_F32 ? 4 : 8;
	const bool vec = c.width % n == 0 && c.v_width % n == 0 && aligned(k, 16) && aligned(v, 16);
	auto launch = [&](auto *k_, auto *v_) {
		if (vec)
			gather_kernel<std::remove_pointer_t<decltype(k_)>, true><<<unsigned(blocks), THREADS, 0, st>>>(c, k_, v_);
		else
			gather_kernel<std::remove_pointer_t<decltype(k_)>, false><<<unsigned(blocks), THREADS, 0, st>>>(c, k_, v_);
	};
	if (dtype == L1ATTN_F32)
		launch(static_cast<float *>(k), static_cast<float *>(v));
	else if (dtype == L1ATTN_F16)
		launch(static_cast<__half *>(k), static_cast<__half *>(v));
	else
		launch(static_cast<__nv_bfloat16 *>(k), static_cast<__nv_bfloat16 *>(v));
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
