// The 8-bit cache: entry points, argument checks, and how attention to it is split over its long axis.
#include <cmath>
#include "cache.cuh"

using namespace l1b;

namespace {

int check(const l1attn_cache *c, int rows, int dtype, bool tokens, CacheArgs *out)
{
	if (!c || rows < 0 || c->n_pages < 1 || c->n_kv_heads < 1 || c->width < 1 || c->v_width < 1)
		return L1ATTN_ERR_ARG;
	if (dtype != L1ATTN_F32 && dtype != L1ATTN_F16 && dtype != L1ATTN_BF16)
		return L1ATTN_ERR_ARG;
	if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
		return L1ATTN_ERR_ARG;
	if (c->width > 256 || c->v_width > 256 || c->n_kv_heads > 65535)
		return L1ATTN_ERR_SHAPE;
	if (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale)
		return L1ATTN_ERR_ARG;
	if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->status, 4))
		return L1ATTN_ERR_ALIGN;
	if (tokens) {
		if (c->n_seqs < 0 || c->max_pages < 0)
			return L1ATTN_ERR_ARG;
		if ((long long)c->max_pages * c->page > 1 << 30) // (positions and tile ends stay within int)
			return L1ATTN_ERR_SHAPE;
		if (rows == 0 || c->n_seqs == 0)
			return 1; // nothing to do
		if (!c->table || !c->start || !c->cu)
			return L1ATTN_ERR_ARG;
		if (!aligned(c->table, 4) || !aligned(c->start, 4) || !aligned(c->cu, 4))
			return L1ATTN_ERR_ALIGN;
	}
	*out = {c->k_codes, c->v_codes, c->k_scale, c->v_scale, c->n_pages, c->page, c->n_kv_heads, c->width, c->v_width,
		c->table, c->start, c->cu, c->n_seqs, c->max_pages, rows, c->status};
	return L1ATTN_OK;
}

// How a call is divided, and the bytes of work that takes.
int plan(AttendArgs *a, int rows, int heads, int max_len, int dtype, size_t *bytes)
{
	a->heads = heads;
	a->group = heads / a->c.kv_heads;
	if ((long long)rows * heads > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	const size_t part = (a->c.v_width + 2) * sizeof(float);
	if (attend_mma_fits(a->c.width, a->c.v_width, dtype)) { // one wave of CTAs that share the chunks; a unit's costs count as some (cache_attend_mma.cu)
		// eight rows cost half of sixteen; sequences of one token have as many rows as a group has heads
		a->tile_rows = (long long)rows * a->group / a->c.n_seqs <= 8 ? 8 : 16;
		int sms = 0;
		if (int rc = multiprocessors(&sms))
			return rc;
		a->ctas = attend_mma_ctas(a->tile_rows, sms);
		// fewest chunks of a CTA, 6 against 16 and 44: 4 sequences of 1000 tokens 22.8 / 26.4 / 40.6 us, 16 of up to 300 23.5 / 26.8 / 44.4; 3 is no better
		a->least = 6;
		a->splits = 1;
		*bytes = (2ull * a->ctas * a->tile_rows * part + 255) / 256 * 256 + a->ctas * sizeof(AttendSplit);
		return L1ATTN_OK;
	}
	// splits of the keys: eight CTAs a multiprocessor (several waves of them even out unequal lengths), at least 256 keys each
	int sms = 0;
	if (int rc = multiprocessors(&sms))
		return rc;
	a->tile_rows = 16;
	const long long tiles = (long long)rows * a->group / a->tile_rows + a->c.n_seqs, len = max_len < 1 ? 1 : max_len;
	long long want = (8 * sms + tiles * a->c.kv_heads - 1) / (tiles * a->c.kv_heads), most = (len + 255) / 256;
	want = want < most ? want : most;
	a->split_keys = int(((len + want - 1) / want + 63) / 64 * 64);
	a->splits = int((len + a->split_keys - 1) / a->split_keys);
	*bytes = a->splits > 1 ? size_t(a->splits) * rows * heads * part : 0;
	return L1ATTN_OK;
}

} // namespace

extern "C" int l1attn_cache_append(const l1attn_cache *cache, const void *k, const void *v, const int64_t *strides, int rows, int dtype, void *stream)
{
	CacheArgs c;
	if (int rc = check(cache, rows, dtype, true, &c))
		return rc > 0 ? L1ATTN_OK : rc;
	if (!k || !v || !strides)
		return L1ATTN_ERR_ARG;
	const size_t es = dtype == L1ATTN_F32 ? 4 : 2;
	if (!aligned(k, es) || !aligned(v, es))
		return L1ATTN_ERR_ALIGN;
	long long st[4];
	for (int i = 0; i < 4; i++)
		if ((st[i] = strides[i]) < 0)
			return L1ATTN_ERR_ARG;
	return append_launch(c, k, v, st, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int l1attn_cache_gather(const l1attn_cache *cache, void *k, void *v, int rows, int dtype, void *stream)
{
	CacheArgs c;
	if (int rc = check(cache, rows, dtype, true, &c))
		return rc > 0 ? L1ATTN_OK : rc;
	if (!k || !v)
		return L1ATTN_ERR_ARG;
	const size_t es = dtype == L1ATTN_F32 ? 4 : 2;
	if (!aligned(k, es) || !aligned(v, es))
		return L1ATTN_ERR_ALIGN;
	return gather_launch(c, k, v, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int l1attn_cache_copy_pages(const l1attn_cache *cache, int layers, const int32_t *src, const int32_t *dst, int n, void *stream)
{
	CacheArgs c;
	if (int rc = check(cache, 0, L1ATTN_F32, false, &c))
		return rc;
	if (layers < 0 || n < 0)
		return L1ATTN_ERR_ARG;
	if (layers == 0 || n == 0)
		return L1ATTN_OK;
	if (!src || !dst)
		return L1ATTN_ERR_ARG;
	if (!aligned(src, 4) || !aligned(dst, 4))
		return L1ATTN_ERR_ALIGN;
	return copy_pages_launch(c, layers, src, dst, n, static_cast<cudaStream_t>(stream));
}

extern "C" size_t l1attn_cache_attend_bytes(const l1attn_cache *cache, int rows, int n_heads, int max_len, int dtype)
{
	AttendArgs a;
	if (check(cache, rows, dtype, true, &a.c) || n_heads < 1 || n_heads % a.c.kv_heads)
		return 0;
	size_t bytes = 0;
	return plan(&a, rows, n_heads, max_len, dtype, &bytes) ? 0 : bytes;
}

extern "C" int l1attn_cache_attend(const l1attn_cache *cache, const void *q, const int64_t *strides, void *vo, void *work, int rows, int n_heads, int max_len,
				   const l1attn_mask *mask, int dtype, void *stream)
{
	AttendArgs a;
	const int rc = check(cache, rows, dtype, true, &a.c);
	if (rc < 0)
		return rc;
	if (!mask || !strides || n_heads < 1 || n_heads % cache->n_kv_heads || mask->mode < 0 || mask->mode > 2 || mask->window < 0 || !cap_fits(mask->softcap) ||
	    !mask->causal || mask->doc || mask->prefix || strides[0] < 0 || strides[1] < 0)
		return L1ATTN_ERR_ARG;
	if (rc > 0)
		return L1ATTN_OK;
	if (!q || !vo)
		return L1ATTN_ERR_ARG;
	const size_t es = dtype == L1ATTN_F32 ? 4 : 2;
	if (!aligned(q, es) || !aligned(vo, es) || !aligned(work, 16) || !aligned(mask->slopes, 4))
		return L1ATTN_ERR_ALIGN;
	a.q = q;
	a.vo = vo;
	a.q_row = strides[0];
	a.q_head = strides[1];
	a.window = mask->window;
	a.mode = mask->mode;
	a.cap = mask->softcap;
	a.scale = float(1.0 / std::sqrt(double(a.c.width)));
	a.slopes = mask->slopes;
	size_t bytes = 0;
	if (const int e = plan(&a, rows, n_heads, max_len, dtype, &bytes))
		return e;
	if (bytes && !work)
		return L1ATTN_ERR_ARG;
	a.part = bytes ? static_cast<float *>(work) : nullptr;
	const cudaStream_t st = static_cast<cudaStream_t>(stream);
	if (attend_mma_fits(a.c.width, a.c.v_width, dtype)) {
		a.splits_of = reinterpret_cast<AttendSplit *>(static_cast<unsigned char *>(work) + bytes - a.ctas * sizeof(AttendSplit));
		return attend_mma_launch(a, dtype, st);
	}
	if (const int e = attend_simple_launch(a, dtype, st))
		return e;
	return a.splits > 1 ? attend_merge_launch(a, dtype, st) : L1ATTN_OK;
}

extern "C" int l1attn_test_cache_unit(const l1attn_cache *cache, int rows, long long unit, int num, int den, int extra, int slot, int32_t *out)
{
	CacheArgs c;
	if (int rc = check(cache, rows, L1ATTN_F32, true, &c))
		return rc;
	const int seq = cache_find(c, unit, num, den, extra);
	const SeqView v = cache_seq(c, seq);
	const long long mine = unit - cache_first_unit(c, seq, num, den, extra);
	const int32_t got[] = {seq, v.row, v.count, v.start, int32_t(mine), slot >= 0 && slot < c.max_pages ? cache_page(c, seq, slot) : -2};
	for (int i = 0; i < 6; i++)
		out[i] = got[i];
	return L1ATTN_OK;
}
