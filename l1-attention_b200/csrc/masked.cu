// Masked L1 attention: entry points, argument checks, and the two small kernels around the main ones.
#include <cmath>
#include "mask.cuh"

namespace l1b {

namespace {

// Range of documents of every tile of 64 tokens, a warp each: lets the main kernels pass over tiles that share no document.
__global__ void doc_ranges_kernel(const int32_t *doc, DocRange *out, int n, long long tiles)
{
	const long long tile = blockIdx.x * (long long)(blockDim.x / 32) + threadIdx.x / 32;
	if (tile >= tiles)
		return;
	const int per = (n + DOC_TILE - 1) / DOC_TILE;
	const long long b = tile / per;
	const int t0 = int(tile % per) * DOC_TILE, lane = threadIdx.x % 32;
	int lo = INT32_MAX, hi = -1, others = 0;
#pragma unroll
	for (int i = 0; i < DOC_TILE; i += 32) {
		const int t = t0 + i + lane;
		if (t >= n)
			continue;
		const int d = doc[b * n + t];
		if (d < 0) {
			others = 1;
			continue;
		}
		lo = min(lo, d);
		hi = max(hi, d);
	}
	lo = __reduce_min_sync(0xffffffffu, lo);
	hi = __reduce_max_sync(0xffffffffu, hi);
	others = __reduce_max_sync(0xffffffffu, others);
	if (lane == 0)
		out[tile] = {lo, hi, others, 0};
}

// delta[row] = <dvo[row], vo[row]> = sum_s p <v_s, dvo>, a warp per row; the exp form has no normaliser to differentiate.  rest: what rounding left of vo, or
// null (without it a row's score gradients are off by what half a step of vo makes, all alike, which shows in dq)
template <typename T> __global__ void delta_kernel(const T *dvo, const T *vo, const T *rest, float *delta, long long rows, int width, int zero)
{
	const long long row = blockIdx.x * (long long)(blockDim.x / 32) + threadIdx.x / 32;
	if (row >= rows)
		return;
	float sum = 0.f;
	if (!zero)
		for (int w = threadIdx.x % 32; w < width; w += 32)
			sum = fmaf(to_float(dvo[row * width + w]), to_float(vo[row * width + w]) + (rest ? to_float(rest[row * width + w]) : 0.f), sum);
#pragma unroll
	for (int o = 16; o; o >>= 1)
		sum += __shfl_xor_sync(0xffffffffu, sum, o);
	if (threadIdx.x % 32 == 0)
		delta[row] = sum;
}

// dk and dv of shared heads: the query heads' shares, in order
template <typename T> __global__ void __launch_bounds__(256) sum_shares_kernel(const float *part, T *out, long long values, int group, int width)
{
	const long long i = blockIdx.x * 256ll + threadIdx.x; // [bs][n][kv_heads][width]
	if (i >= values)
		return;
	const float *from = part + i / width * group * width + i % width;
	float sum = 0.f;
	for (int g = 0; g < group; g++)
		sum += from[(long long)g * width];
	out[i] = from_float<T>(sum);
}

template <typename T> int sum_shares(const MaskedArgs &a, const float *shares, void *dk, void *dv, cudaStream_t st)
{
	const long long rows = (long long)a.bs * a.n * a.kv_heads;
	for (int i = 0; i < 2; i++) {
		const int width = i ? a.v_width : a.width;
		const long long blocks = (rows * width + 255) / 256;
		if (blocks > 0x7fffffffll)
			return L1ATTN_ERR_SHAPE;
		sum_shares_kernel<<<unsigned(blocks), 256, 0, st>>>(shares + (i ? (long long)a.bs * a.n * a.heads * a.width : 0), static_cast<T *>(i ? dv : dk), rows * width,
								     a.heads / a.kv_heads, width);
		L1B_LAUNCH_CHECK();
	}
	return L1ATTN_OK;
}

size_t pad256(size_t x) { return (x + 255) / 256 * 256; }
size_t ranges_bytes(int bs, int n) { return pad256(size_t(bs) * ((n + DOC_TILE - 1) / DOC_TILE) * sizeof(DocRange)); }

int check(const void *q, const void *k, const void *v, const int64_t *strides, const void *const *others, int n_others, int bs, int n_tok, int n_heads,
	  int n_kv_heads, int width, int v_width, const l1attn_mask *mask, int dtype, void *work, MaskedArgs *a)
{
	if (bs < 0 || n_tok < 0 || n_heads < 0 || n_kv_heads < 0 || width < 1 || v_width < 1 || !mask || !strides)
		return L1ATTN_ERR_ARG;
	if (dtype != L1ATTN_F32 && dtype != L1ATTN_F16 && dtype != L1ATTN_BF16)
		return L1ATTN_ERR_ARG;
	if (mask->mode < 0 || mask->mode > 2 || mask->window < 0 || !cap_fits(mask->softcap))
		return L1ATTN_ERR_ARG;
	if (width > 256 || v_width > 256 || n_tok > 1 << 30) // (ends of tiles stay within int)
		return L1ATTN_ERR_SHAPE;
	if (n_heads == 0 && n_kv_heads > 0)
		return L1ATTN_ERR_ARG;
	if (bs == 0 || n_tok == 0 || n_heads == 0)
		return 1; // nothing to do
	if (n_kv_heads == 0 || n_heads % n_kv_heads)
		return L1ATTN_ERR_ARG;
	const size_t es = dtype == L1ATTN_F32 ? 4 : 2;
	if (!q || !k || !v || (mask->doc && !work))
		return L1ATTN_ERR_ARG;
	if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(work, 16) || !aligned(mask->slopes, 4) || !aligned(mask->doc, 4) ||
	    !aligned(mask->prefix, 4))
		return L1ATTN_ERR_ALIGN;
	for (int i = 0; i < n_others; i++) {
		if (!others[i])
			return L1ATTN_ERR_ARG;
		if (!aligned(others[i], es))
			return L1ATTN_ERR_ALIGN;
	}
	for (int i = 0; i < 9; i++)
		if (strides[i] < 0)
			return L1ATTN_ERR_ARG;
	*a = {{q, strides[0], strides[1], strides[2]}, {k, strides[3], strides[4], strides[5]}, {v, strides[6], strides[7], strides[8]},
	      bs, n_tok, n_heads, n_kv_heads, width, v_width, mask->causal != 0, mask->window, mask->mode, mask->softcap, float(1.0 / std::sqrt(double(width))),
	      mask->slopes, mask->doc, mask->prefix, mask->doc ? static_cast<const DocRange *>(work) : nullptr};
	return L1ATTN_OK;
}

int launch_ranges(const MaskedArgs &a, void *work, cudaStream_t st)
{
	if (!a.doc)
		return L1ATTN_OK;
	const long long tiles = (long long)a.bs * ((a.n + DOC_TILE - 1) / DOC_TILE);
	if (tiles / 8 >= 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	doc_ranges_kernel<<<unsigned((tiles + 7) / 8), 256, 0, st>>>(a.doc, static_cast<DocRange *>(work), a.n, tiles);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

template <typename T> void launch_delta(const MaskedArgs &a, const void *dvo, const void *vo, const void *rest, float *delta, long long rows, cudaStream_t st)
{
	delta_kernel<T><<<unsigned((rows + 7) / 8), 256, 0, st>>>(static_cast<const T *>(dvo), static_cast<const T *>(vo), static_cast<const T *>(rest), delta, rows, a.v_width,
								  a.mode == L1ATTN_SV_EXP);
}

} // namespace
} // namespace l1b

using namespace l1b;

namespace {
// the backward's work: document ranges | delta | query heads' shares of dk and dv | gradients of the distances
struct BackwardWork {
	size_t delta, shares, e, bytes;
	bool keeps_e;
	BackwardWork(int bs, int n, int heads, int kv_heads, int width, int v_width, int dtype)
	{
		const size_t rows = size_t(bs) * n * heads;
		const bool mma = masked_mma_fits(width, v_width, dtype);
		const long long units = mma ? masked_units_at_once(bs, n, heads) : 0;
		delta = ranges_bytes(bs, n);
		shares = delta + pad256(rows * sizeof(float));
		e = shares + (heads != kv_heads ? pad256(rows * (width + v_width) * sizeof(float)) : 0);
		keeps_e = units > 0;
		bytes = e + size_t(units) * masked_unit_floats(n) * sizeof(float);
	}
};
} // namespace

extern "C" size_t l1attn_masked_work_bytes(int bs, int n_tok, int n_heads, int n_kv_heads, int width, int v_width, int dtype, int backward)
{
	if (bs < 1 || n_tok < 1 || n_heads < 1 || n_kv_heads < 1 || width < 1 || v_width < 1)
		return 256;
	return backward ? BackwardWork(bs, n_tok, n_heads, n_kv_heads, width, v_width, dtype).bytes : ranges_bytes(bs, n_tok);
}

extern "C" int l1attn_masked_fwd(const void *q, const void *k, const void *v, const int64_t *strides, void *vo, void *rest, float *lse, void *work, int bs, int n_tok,
				 int n_heads, int n_kv_heads, int width, int v_width, const l1attn_mask *mask, int dtype, void *stream)
{
	MaskedArgs a;
	const void *others[] = {vo};
	int rc = check(q, k, v, strides, others, 1, bs, n_tok, n_heads, n_kv_heads, width, v_width, mask, dtype, work, &a);
	if (rc)
		return rc > 0 ? L1ATTN_OK : rc;
	if (!aligned(lse, 4) || !aligned(rest, dtype == L1ATTN_F32 ? 4 : 2))
		return L1ATTN_ERR_ALIGN;
	if (dtype == L1ATTN_F32)
		rest = nullptr;
	const cudaStream_t st = static_cast<cudaStream_t>(stream);
	if ((rc = launch_ranges(a, work, st)))
		return rc;
	return masked_mma_fits(width, v_width, dtype) ? masked_mma_fwd_launch(a, vo, rest, lse, dtype, st) : masked_simple_fwd_launch(a, vo, rest, lse, dtype, st);
}

extern "C" int l1attn_masked_bwd(const void *q, const void *k, const void *v, const int64_t *strides, const void *vo, const void *rest, const void *dvo, const float *lse, void *dq,
				 void *dk, void *dv, void *work, int bs, int n_tok, int n_heads, int n_kv_heads, int width, int v_width, const l1attn_mask *mask,
				 int dtype, void *stream)
{
	MaskedArgs a;
	const void *others[] = {vo, dvo, dq, dk, dv};
	int rc = check(q, k, v, strides, others, 5, bs, n_tok, n_heads, n_kv_heads, width, v_width, mask, dtype, work, &a);
	if (rc)
		return rc > 0 ? L1ATTN_OK : rc;
	if (!lse || !work)
		return L1ATTN_ERR_ARG;
	if (!aligned(lse, 4) || !aligned(rest, dtype == L1ATTN_F32 ? 4 : 2))
		return L1ATTN_ERR_ALIGN;
	const cudaStream_t st = static_cast<cudaStream_t>(stream);
	const long long rows = (long long)bs * n_tok * n_heads;
	if (rows / 8 >= 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	const BackwardWork layout(bs, n_tok, n_heads, n_kv_heads, width, v_width, dtype);
	unsigned char *const base = static_cast<unsigned char *>(work);
	float *const delta = reinterpret_cast<float *>(base + layout.delta), *const shares = reinterpret_cast<float *>(base + layout.shares);
	float *const e = layout.keeps_e ? reinterpret_cast<float *>(base + layout.e) : nullptr;
	if ((rc = launch_ranges(a, work, st)))
		return rc;
	if (dtype == L1ATTN_F32)
		launch_delta<float>(a, dvo, vo, nullptr, delta, rows, st);
	else if (dtype == L1ATTN_F16)
		launch_delta<__half>(a, dvo, vo, rest, delta, rows, st);
	else
		launch_delta<__nv_bfloat16>(a, dvo, vo, rest, delta, rows, st);
	L1B_LAUNCH_CHECK();
	rc = masked_mma_fits(width, v_width, dtype) ? masked_mma_bwd_launch(a, dvo, lse, delta, dq, dk, dv, shares, e, dtype, st) :
						      masked_simple_bwd_launch(a, dvo, lse, delta, dq, dk, dv, shares, dtype, st);
	if (rc || n_heads == n_kv_heads)
		return rc;
	return dtype == L1ATTN_F32 ? sum_shares<float>(a, shares, dk, dv, st) : dtype == L1ATTN_F16 ? sum_shares<__half>(a, shares, dk, dv, st) :
												     sum_shares<__nv_bfloat16>(a, shares, dk, dv, st);
}
