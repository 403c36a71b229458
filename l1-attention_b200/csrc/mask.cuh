// Masks, caps and biases of L1 scores, shared by the kernels of masked attention and of attention to a cache.
//
//   x = -(1/sqrt(width)) sum_w |q - k|;   x = cap tanh(x / cap) where cap > 0;   x -= slope[head] |t - s|
//   query t sees key s when their documents are the same and not negative (where documents are given) and
//     s < prefix, or (s <= t where causal) and (|t - s| < window where window > 0)
//
// A row that sees nothing, or only keys at infinite distance, gets weights, output and gradients of zero.  A key whose weight is zero
// contributes nothing, whatever its value row holds.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include "common.cuh"

namespace l1b {

constexpr int DOC_TILE = 64; // tokens that share an entry of the document ranges

struct DocRange { // of a tile of DOC_TILE tokens: lowest and highest document among its tokens of a document, and whether others are there
	int lo, hi, others, pad;
};

// strides in elements of [bs][n_tok][heads][width]; the width is contiguous
struct Strided {
	const void *p;
	long long batch, tok, head;
};

struct MaskedArgs {
	Strided q, k, v;
	int bs, n, heads, kv_heads, width, v_width;
	int causal, window, mode;
	float cap, scale; // scale: 1/sqrt(width)
	const float *slopes;
	const int32_t *doc, *prefix;
	const DocRange *ranges;
};

// (a cap whose reciprocal is no float32 would give NaN, or no cap at all)
inline bool cap_fits(float cap) { return cap == 0.f || (cap >= 1e-30f && cap <= 1e30f); }

// What one batch item's masks say.
struct MaskView {
	int n, causal, window, prefix;
	const int32_t *doc;
	const DocRange *ranges;

	__device__ MaskView(const MaskedArgs &a, int b)
	    : n(a.n), causal(a.causal), window(a.window), prefix(a.prefix ? a.prefix[b] : 0), doc(a.doc ? a.doc + (long long)b * a.n : nullptr),
	      ranges(a.ranges ? a.ranges + (long long)b * ((a.n + DOC_TILE - 1) / DOC_TILE) : nullptr)
	{
	}
	// positions alone; 0 <= t, s < n
	__device__ __forceinline__ bool reach(int t, int s) const
	{
		const int d = t - s;
		return s < prefix || ((!causal || d >= 0) && (window == 0 || (d < window && -d < window)));
	}
	__device__ __forceinline__ bool sees(int t, int s, int doc_t, int doc_s) const
	{
		return t < n && s < n && reach(t, s) && (!doc || (doc_t == doc_s && doc_s >= 0));
	}
	// Whether any of the queries [t0, t1) may see any of the keys [s0, s1); both ranges non-empty, within one tile of DOC_TILE and within n.
	__device__ __forceinline__ bool any(int t0, int t1, int s0, int s1) const
	{
		bool near = !causal || s0 < t1;
		if (window) // the nearest pair: distance 0 where the ranges meet
			near = near && s1 - 1 > t0 - window && s0 < (long long)t1 - 1 + window;
		if (!near && s0 >= prefix)
			return false;
		if (!doc)
			return true;
		const DocRange a = ranges[t0 / DOC_TILE], b = ranges[s0 / DOC_TILE];
		return a.lo <= b.hi && b.lo <= a.hi;
	}
	// Whether all of them see all.
	__device__ __forceinline__ bool all(int t0, int t1, int s0, int s1) const
	{
		if (s1 > prefix) {
			if (causal && s1 - 1 > t0)
				return false;
			if (window && (t1 - 1 - s0 >= window || s1 - 1 - t0 >= window))
				return false;
		}
		if (!doc)
			return true;
		const DocRange a = ranges[t0 / DOC_TILE], b = ranges[s0 / DOC_TILE];
		return !a.others && !b.others && a.lo == a.hi && b.lo == b.hi && a.lo == b.lo;
	}
};

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

// what rounding to T leaves of a value (0 where that is not finite)
template <typename T> __device__ __forceinline__ T rest_of(float x)
{
	const float rest = x - to_float(from_float<T>(x));
	return from_float<T>(fabsf(rest) < INFINITY ? rest : 0.f);
}

// weight of a score under a row's log-normaliser; a row without any weight has -inf there
__device__ __forceinline__ float weight_of(float x, float lse) { return lse == -INFINITY ? 0.f : expf(x - lse); }

// status of a tile's rows when it begins: the +1 form starts with one key of score 0, the exp form with a fixed reference of 0
__device__ __forceinline__ float start_max(int mode) { return mode == L1ATTN_SV_SOFTMAX ? -INFINITY : 0.f; }
__device__ __forceinline__ float start_sum(int mode) { return mode == L1ATTN_SV_SOFTMAX_PLUS_ONE ? 1.f : 0.f; }
// factor of the accumulated values at the end, and the row's log-normaliser (all weights are exp(x - lse))
__device__ __forceinline__ float finish_row(int mode, float m, float l, float *lse)
{
	if (mode == L1ATTN_SV_EXP) {
		*lse = 0.f;
		return expf(m);
	}
	*lse = l == 0.f ? -INFINITY : m + logf(l);
	return l == 0.f ? 0.f : 1.f / l;
}

// The same for rows that begin with nothing (m = -inf, l = 0) in every mode, so that m is the largest score of a key: the +1 form's key of score 0 joins here.
__device__ __forceinline__ float finish_row_of_keys(int mode, float m, float l, float *lse)
{
	if (mode != L1ATTN_SV_SOFTMAX_PLUS_ONE)
		return finish_row(mode, m, l, lse);
	const float top = fmaxf(m, 0.f), keep = expf(m - top), sum = l * keep + expf(-top);
	*lse = top + logf(sum);
	return keep / sum;
}

// 16-bit types, widths up to 128: distances and products on the tensor cores
bool masked_mma_fits(int width, int v_width, int dtype);
int masked_mma_fwd_launch(const MaskedArgs &a, void *vo, void *rest, float *lse, int dtype, cudaStream_t st);
// shares: [bs][n][heads][width + v_width] floats where heads are shared; e: masked_units_at_once() * masked_unit_floats() floats, or null
long long masked_unit_floats(int n);
long long masked_units_at_once(int bs, int n, int heads);
int masked_mma_bwd_launch(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, float *e, int dtype,
			  cudaStream_t st);
int masked_simple_fwd_launch(const MaskedArgs &a, void *vo, void *rest, float *lse, int dtype, cudaStream_t st);
int masked_simple_bwd_launch(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, int dtype,
			     cudaStream_t st);

} // namespace l1b
