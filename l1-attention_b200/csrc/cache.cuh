// A paged cache of keys and values in 8 bits (see l1attn_cache in l1attn_b200.h), as the kernels see it.
//
// Pages, starts and row offsets come from device memory that nobody has checked: a page id, a position or an offset out of range sets
// the status word and what it names is left out, never dereferenced.
#pragma once
#include "mask.cuh"

namespace l1b {

struct CacheArgs {
	int8_t *k_codes, *v_codes;
	float *k_scale, *v_scale;
	int n_pages, page, kv_heads, width, v_width;
	const int32_t *table, *start, *cu;
	int n_seqs, max_pages, rows; // rows: of the token tensors
	int *status;
};

#define L1B_BOTH __host__ __device__ __forceinline__

L1B_BOTH void cache_fault(const CacheArgs &c)
{
	if (c.status)
		*reinterpret_cast<volatile int *>(c.status) = L1ATTN_ERR_INDEX;
}

// One sequence's part of a call: rows [row, row + count) of the token tensors are its positions [start, start + count); the `lost` rows behind them are its
// too, but have no place (the offsets or the start are out of range, or the table ends): what is read at them is zeros.
struct SeqView {
	int row, count, start, lost;
};

L1B_BOTH int cache_row(const CacheArgs &c, int seq)
{
	const int r = c.cu[seq];
	return r < 0 ? 0 : r > c.rows ? c.rows : r;
}

L1B_BOTH SeqView cache_seq(const CacheArgs &c, int seq)
{
	const int a = c.cu[seq], b = c.cu[seq + 1], s = c.start[seq];
	SeqView v = {cache_row(c, seq), 0, s, 0};
	if (a < 0 || b < a || b > c.rows || s < 0) {
		cache_fault(c);
		// (an end that is out of order: up to where the next one ends, so that rows of sequences in order stay theirs)
		const int own = (b < a || b > c.rows ? seq + 2 <= c.n_seqs ? cache_row(c, seq + 2) : c.rows : b) - v.row;
		v.lost = own > 0 ? own : 0;
		v.start = 0;
		return v;
	}
	v.count = b - a;
	const long long room = (long long)c.max_pages * c.page - s;
	if (v.count > room) {
		cache_fault(c);
		v.count = room > 0 ? int(room) : 0;
		v.lost = b - a - v.count;
	}
	return v;
}

// page that holds position pos of a sequence (pos / page < max_pages), or -1
L1B_BOTH int cache_page(const CacheArgs &c, int seq, int slot)
{
	const int id = c.table[(long long)seq * c.max_pages + slot];
	if (id < 0 || id >= c.n_pages) {
		cache_fault(c);
		return -1;
	}
	return id;
}

// Work units of a call lie behind one another: sequence i's begin at cu[i] * num / den + i * extra, which leaves room for at least
// ceil(count * num / den) + extra - 1 of them.  The sequence that unit u belongs to (its own units are u - first; there may be fewer).
L1B_BOTH long long cache_first_unit(const CacheArgs &c, int seq, int num, int den, int extra)
{
	return (long long)cache_row(c, seq) * num / den + (long long)seq * extra;
}
L1B_BOTH int cache_find(const CacheArgs &c, long long u, int num, int den, int extra)
{
	int lo = 0, hi = c.n_seqs - 1;
	while (lo < hi) {
		const int mid = (lo + hi + 1) / 2;
		if (cache_first_unit(c, mid, num, den, extra) <= u)
			lo = mid;
		else
			hi = mid - 1;
	}
	return lo;
}

#ifdef __CUDACC__
// cache_find by a whole warp: a lane per sequence, so that the reads do not wait for one another (a CTA's first steps are many such waits).  Where there are
// more than FIND_AT_ONCE, a lane per 32nd of them first: every warp of a call does this, and reading all offsets each time grows with their number's square.
// (append of single tokens, 8 heads of 128 and 128: 128 sequences 14.6 us with 64 at once, 16.7 with 128; 256 22.9, 37.0 with 256; 4096 340 us, 4418 with all.)
constexpr int FIND_AT_ONCE = 64;
__device__ __forceinline__ int cache_find_warp(const CacheArgs &c, long long u, int num, int den, int extra)
{
	const int lane = threadIdx.x % 32;
	int lo = 0, n = c.n_seqs; // it is one of [lo, lo + n)
	while (n > FIND_AT_ONCE) {
		const int step = (n + 31) / 32, at = lane * step;
		const int before = __popc(__ballot_sync(0xffffffffu, at < n && cache_first_unit(c, lo + min(at, n - 1), num, den, extra) <= u));
		const int skip = max(before - 1, 0) * step;
		lo += skip;
		n = min(step, n - skip);
	}
	int before = 0;
	for (int i = lane; i < (n + 31) / 32 * 32; i += 32)
		before += __popc(__ballot_sync(0xffffffffu, i < n && cache_first_unit(c, lo + min(i, n - 1), num, den, extra) <= u));
	return lo + max(before - 1, 0);
}
#endif

// the sequence whose rows [cu[i], cu[i + 1]) hold `row`, if any does: the last one that begins at or before it
L1B_BOTH int cache_find_row(const CacheArgs &c, long long row) { return cache_find(c, row, 1, 1, 0); }

struct AttendSplit;

struct AttendArgs {
	CacheArgs c;
	const void *q;
	void *vo;
	long long q_row, q_head; // element strides of q
	int heads, group;        // group: query heads that share a head of keys and values
	int window, mode;
	float cap, scale;
	const float *slopes;
	float *part; // [splits][rows][heads][v_width + 2], or null: one split
	int splits, split_keys;
	int tile_rows; // rows -- (token, head of the group) pairs of one sequence -- of a CTA: 8 or 16
	// attend_mma: CTAs that share the work equally, the least share in chunks, and what they leave for each other (work: part, then a record a CTA)
	int ctas, least;
	AttendSplit *splits_of;
};

// A unit -- a tile of rows and a head of keys and values -- that begins in a CTA's share and ends in a later one's (last); kv < 0: none
struct AttendSplit {
	int kv, rows, last, pad;
	long long pair; // first (token, head of the group) pair: token row * group + head of the group
};

// joins the splits' running maxima, sums and accumulated values (a part: m, l, values)
int attend_merge_launch(const AttendArgs &a, int dtype, cudaStream_t st);
int append_launch(const CacheArgs &c, const void *k, const void *v, const long long *strides, int dtype, cudaStream_t st);
int gather_launch(const CacheArgs &c, void *k, void *v, int dtype, cudaStream_t st);
int copy_pages_launch(const CacheArgs &c, int layers, const int32_t *src, const int32_t *dst, int n, cudaStream_t st);
// 16-bit types, widths up to 128: on the tensor cores
bool attend_mma_fits(int width, int v_width, int dtype);
int attend_mma_ctas(int tile_rows, int sms);
int attend_mma_launch(const AttendArgs &a, int dtype, cudaStream_t st);
int attend_simple_launch(const AttendArgs &a, int dtype, cudaStream_t st);

// (m, l) of a row that has seen all its keys -> factor of its values; a row without weights gets 0.  The +1 form has one more key of
// score 0, the exp form no normaliser.
__device__ __forceinline__ float finish_softmax(int mode, float m, float l)
{
	if (mode == L1ATTN_SV_EXP)
		return l == 0.f ? 0.f : expf(m);
	if (mode == L1ATTN_SV_SOFTMAX_PLUS_ONE) {
		if (l == 0.f)
			return 0.f;
		const float top = fmaxf(m, 0.f);
		return expf(m - top) / (l * expf(m - top) + expf(-top));
	}
	return l == 0.f ? 0.f : 1.f / l;
}

} // namespace l1b
