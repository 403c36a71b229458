// Masked L1 attention (mask.cuh) of 16-bit rows up to 128 wide: distances and products on the tensor cores (mma.cuh).
//
// Forward: a CTA of four warps owns 64 query rows of one head, a warp 16 of them, in registers; keys and values stream in tiles of 64 through
// two stages of asynchronous copies.  Running softmax in registers (a row's scores lie in one quad); weights are rounded to the inputs' type for the value
// product (11 or 8 bits, as the values have; the normaliser sums them unrounded), everything else is float32.  Rows whose result is not
// finite are done again, exactly, by a warp each: an infinite or NaN operand spoils its neighbours in a product.
// Bound: instruction issue of few warps.  mma.sync does not overlap float32 instructions (mma alone 8 clocks per scheduler, 13.2 with four
// additions, 9.7 with four minima), so the softmax costs what it takes; forming the next step's distances beside it brought [2,2048,8,128] from
// 343 to 293 us, the short copy loop a tenth.  Now 54 terms per clock and SM ([4,2048,8,128], no mask: 1.10 ms) where float32 instructions reach 48 at best.
#include "mma.cuh"

namespace l1b {

namespace {

constexpr int MB = 1, WARPS = 4, ROWS = 16 * MB * WARPS, KEYS = 64, THREADS = 32 * WARPS; // MB: blocks of 16 rows a warp
constexpr float LOG2E = 1.4426950408889634f, LAG = 8.f;

// One query row, by the definition: a warp, 32 keys at a time.  Rare, so simple.
template <typename T> __device__ __noinline__ void exact_row(const MaskedArgs &a, const MaskView &mask, int b, int head, int t, T *vo, float *lse)
{
	const int lane = threadIdx.x % 32, kv = head / (a.heads / a.kv_heads);
	const T *q = static_cast<const T *>(a.q.p) + b * a.q.batch + t * a.q.tok + head * a.q.head;
	const T *k = static_cast<const T *>(a.k.p) + b * a.k.batch + kv * a.k.head, *v = static_cast<const T *>(a.v.p) + b * a.v.batch + kv * a.v.head;
	float m = start_max(a.mode), l = start_sum(a.mode), acc[4] = {0.f, 0.f, 0.f, 0.f};
	const int doc_t = mask.doc ? mask.doc[t] : 0;
	for (int s0 = 0; s0 < a.n; s0 += 32) {
		const int s = s0 + lane;
		const bool seen = s < a.n && mask.sees(t, s, doc_t, mask.doc && s < a.n ? mask.doc[s] : 0);
		if (!__any_sync(0xffffffffu, seen))
			continue;
		float x = -INFINITY;
		if (seen) {
			float d = 0.f;
			for (int w = 0; w < a.width; w++)
				d += fabsf(to_float(q[w]) - to_float(k[(long long)s * a.k.tok + w]));
			x = -a.scale * d;
			if (a.cap > 0.f)
				x = a.cap * tanhf(x / a.cap);
			if (a.slopes)
				x -= a.slopes[head] * fabsf(float(t - s));
		}
		float top = fmaxf(m, x);
#pragma unroll
		for (int o = 16; o; o >>= 1)
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
		const float ref = top == -INFINITY ? 0.f : top, keep = expf(m - ref), p = expf(x - ref);
		float sum = p;
#pragma unroll
		for (int o = 16; o; o >>= 1)
			sum += __shfl_xor_sync(0xffffffffu, sum, o);
		l = l * keep + sum;
		m = top;
#pragma unroll
		for (int i = 0; i < 4; i++)
			acc[i] *= keep;
		for (int j = 0; j < 32; j++) {
			const float pj = __shfl_sync(0xffffffffu, p, j);
			if (pj == 0.f)
				continue;
#pragma unroll
			for (int i = 0; i < 4; i++)
				if (lane + 32 * i < a.v_width)
					acc[i] = fmaf(pj, to_float(v[(long long)(s0 + j) * a.v.tok + lane + 32 * i]), acc[i]);
		}
	}
	const long long row = ((long long)b * a.n + t) * a.heads + head;
	float ls;
	const float f = finish_row(a.mode, m, l, &ls);
	if (lse && lane == 0)
		lse[row] = ls;
#pragma unroll
	for (int i = 0; i < 4; i++)
		if (lane + 32 * i < a.v_width)
			vo[row * a.v_width + lane + 32 * i] = from_float<T>(f == 0.f ? 0.f : acc[i] * f);
}

// W: 32-column groups of the width; V: 16-column groups of the value rows (4 or 8).  CTAs of an SM, two against three (168 registers): [1,4096,8,64]
// with values of 128 339 / 447 us, [2,2048,8,128] 293 / 472, widths of 32 200 / 235; but [1,8192,8,64] 1230 / 1157 and [4,2048,8,128] with values of 64
// (no mask) 1179 / 1005.
template <typename T, int W, int V>
__global__ void __launch_bounds__(THREADS, V == 4 && W > 1 ? 3 : 2) masked_fwd_mma_kernel(MaskedArgs a, T *vo, float *lse, int tiles, int vec)
{
	extern __shared__ uint4 smem16[];
	__shared__ float key_sums[KEYS];
	using H = Half2<T>;
	constexpr int KP = 4 * W, VP = 2 * V; // 16-byte pieces of a row
	const uint32_t base = shared_address(smem16), stage_bytes = KEYS * (KP + VP) * 16;
	const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, j = lane % 4;
	const int bh = blockIdx.x % (a.bs * a.heads), tile = tiles - 1 - int(blockIdx.x / (a.bs * a.heads)); // the longest rows of a causal mask first
	const int head = bh % a.heads, b = bh / a.heads, kv = head / (a.heads / a.kv_heads);
	const MaskView mask(a, b);
	const int t0 = tile * ROWS, t1 = min(a.n, t0 + ROWS), ta = t0 + 16 * MB * warp + g; // this lane's rows: ta + 8 r
	const float slope = a.slopes ? a.slopes[head] : 0.f, inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;

	// the warp's query rows, in registers for good, and their sums
	load_tile16<T, false, KP, ROWS, THREADS>(base, a.q, b, head, t0, a.n, a.width, nullptr, vec & 1, tid);
	cp_async_commit();
	cp_async_wait<0>();
	__syncthreads();
	uint32_t q[MB][2 * W][4]; // [16 rows][16 columns][row g, row g + 8, and again]
	float qs[2 * MB];
#pragma unroll
	for (int i = 0; i < MB; i++) {
		float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
		for (int u = 0; u < W; u++) {
			const int r = 16 * (MB * warp + i) + g;
			const uint4 x = load_shared16(smem16, tile_offset<false>(KP, r, 4 * u + j)), y = load_shared16(smem16, tile_offset<false>(KP, r + 8, 4 * u + j));
			q[i][2 * u][0] = x.x, q[i][2 * u][1] = y.x, q[i][2 * u][2] = x.y, q[i][2 * u][3] = y.y;
			q[i][2 * u + 1][0] = x.z, q[i][2 * u + 1][1] = y.z, q[i][2 * u + 1][2] = x.w, q[i][2 * u + 1][3] = y.w;
		}
#pragma unroll
		for (int u = 0; u < 2 * W; u++)
			H::mma(sum, q[i][u][0], q[i][u][1], q[i][u][2], q[i][u][3], H::ONES, H::ONES);
		qs[2 * i] = sum[0];
		qs[2 * i + 1] = sum[2];
	}
	__syncthreads();

	// tiles of keys that the rows may see
	const int prefix_tiles = (min(mask.prefix, a.n) + KEYS - 1) / KEYS;
	const int lo = mask.window ? max(t0 - mask.window + 1, 0) / KEYS : 0;
	const int end = max(mask.causal ? (t1 + KEYS - 1) / KEYS : (a.n + KEYS - 1) / KEYS, prefix_tiles);
	auto next = [&](int it) {
		for (;; it++) {
			if (it >= prefix_tiles && it < lo)
				it = lo;
			if (it >= end || mask.any(t0, t1, it * KEYS, min(a.n, it * KEYS + KEYS)))
				return it;
		}
	};
	auto fetch = [&](int it, int stage) {
		const uint32_t at = base + stage * stage_bytes;
		const int32_t *doc = mask.doc && mask.ranges[it * KEYS / DOC_TILE].others ? mask.doc : nullptr;
		load_tile16<T, false, KP, KEYS, THREADS>(at, a.k, b, kv, it * KEYS, a.n, a.width, doc, vec & 2, tid);
		load_tile16<T, true, VP, KEYS, THREADS>(at + KEYS * KP * 16, a.v, b, kv, it * KEYS, a.n, a.v_width, doc, vec & 4, tid);
	};

	float m[2 * MB], l[2 * MB], ref[2 * MB]; // per row: the reference of its exponentials (times log2 e; ref: 0 while it is infinite), this lane's share of its sum
	float o[MB][2 * V][4];
#pragma unroll
	for (int r = 0; r < 2 * MB; r++) {
		m[r] = start_max(a.mode);
		l[r] = ref[r] = 0.f;
	}
#pragma unroll
	for (int i = 0; i < MB * 2 * V * 4; i++)
		o[i / (8 * V)][i / 4 % (2 * V)][i % 4] = 0.f;

	// sums of min(q, k) for 16 keys and 16 rows a block: 256 terms a product (mma.cuh)
	auto distances = [&](const unsigned char *kt, int kb, float(&y)[MB][2][4]) {
#pragma unroll
		for (int i = 0; i < MB * 8; i++)
			y[i / 8][i / 4 % 2][i % 4] = 0.f;
#pragma unroll
		for (int n = 0; n < 8; n++) {
			const uint32_t one = g == n ? H::ONES : 0u;
#pragma unroll
			for (int u = 0; u < W; u++)
#pragma unroll
				for (int h = 0; h < 2; h++) { // (two tiles at once: their sums do not wait for each other)
					const uint4 k = load_shared16(kt, tile_offset<false>(KP, 16 * kb + 8 * h + n, 4 * u + j));
#pragma unroll
					for (int i = 0; i < MB; i++)
						H::mma(y[i][h], H::min(q[i][2 * u][0], k.x), H::min(q[i][2 * u][1], k.x), H::min(q[i][2 * u][2], k.y), H::min(q[i][2 * u][3], k.y), one, one);
#pragma unroll
					for (int i = 0; i < MB; i++)
						H::mma(y[i][h], H::min(q[i][2 * u + 1][0], k.z), H::min(q[i][2 * u + 1][1], k.z), H::min(q[i][2 * u + 1][2], k.w),
						       H::min(q[i][2 * u + 1][3], k.w), one, one);
				}
		}
	};
	// weights of 16 keys, and their products with the values
	auto values = [&](uint32_t vt, int kb, const float(&x)[MB][2][4]) {
		uint32_t p[MB][4];
#pragma unroll
		for (int i = 0; i < MB; i++)
#pragma unroll
			for (int h = 0; h < 2; h++) {
				float e[4];
#pragma unroll
				for (int c = 0; c < 4; c++) {
					e[c] = exp2_fast(x[i][h][c] - ref[2 * i + c / 2]);
					l[2 * i + c / 2] += e[c];
				}
				p[i][2 * h] = H::pack(e[0], e[1]);
				p[i][2 * h + 1] = H::pack(e[2], e[3]);
			}
#pragma unroll
		for (int vb = 0; vb < V; vb++) {
			uint32_t y[4];
			ldmatrix4_trans(y, vt + tile_offset<true>(VP, 16 * kb + lane % 16, 2 * vb + lane / 16));
#pragma unroll
			for (int i = 0; i < MB; i++) {
				H::mma(o[i][2 * vb], p[i][0], p[i][1], p[i][2], p[i][3], y[0], y[1]);
				H::mma(o[i][2 * vb + 1], p[i][0], p[i][1], p[i][2], p[i][3], y[2], y[3]);
			}
		}
	};
	// sums -> scores times log2 e, masked; and the rows' references
	auto scores = [&](float(&x)[MB][2][4], int s0, bool whole, bool special) {
		const float unit = special ? a.scale : LOG2E * a.scale; // straight to the exponent where the score is the distance alone
#pragma unroll
		for (int h = 0; h < 2; h++) {
			const float2 ks = *reinterpret_cast<const float2 *>(&key_sums[s0 % KEYS + 8 * h + 2 * j]);
#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int c = 0; c < 4; c++)
					x[i][h][c] = unit * (fmaf(2.f, x[i][h][c], -qs[2 * i + c / 2]) - (c & 1 ? ks.y : ks.x));
		}
		if (special) {
#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int c = 0; c < 8; c++) {
					const int s = s0 + 8 * (c / 4) + 2 * j + (c & 1), t = ta + 16 * i + 8 * (c / 2 % 2);
					float y = x[i][c / 4][c % 4];
					if (a.cap > 0.f)
						y = a.cap * tanhf(y * inv_cap);
					if (a.slopes)
						y -= slope * fabsf(float(t - s));
					if (!whole && !(t < a.n && s < a.n && mask.sees(t, s, mask.doc ? mask.doc[t] : 0, mask.doc ? mask.doc[s] : 0)))
						y = -INFINITY;
					x[i][c / 4][c % 4] = y * LOG2E;
				}
		}
		// The reference of the exponentials need not be the maximum: it follows once a score is beyond it by more than LAG.
		float top[2 * MB];
		bool grew = false;
#pragma unroll
		for (int r = 0; r < 2 * MB; r++) {
			const float(&y)[2][4] = x[r / 2];
			const int c = 2 * (r % 2);
			top[r] = fmaxf(fmaxf(y[0][c], y[0][c + 1]), fmaxf(y[1][c], y[1][c + 1]));
			grew |= top[r] > m[r] + LAG;
		}
		if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
			for (int r = 0; r < 2 * MB; r++) {
				top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
				top[r] = fmaxf(fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2)), m[r]);
				const float keep = top[r] == -INFINITY ? 1.f : exp2_fast(m[r] - top[r]);
				m[r] = top[r];
				ref[r] = top[r] == -INFINITY ? 0.f : top[r];
				l[r] *= keep;
#pragma unroll
				for (int v = 0; v < 2 * V; v++) {
					o[r / 2][v][2 * (r % 2)] *= keep;
					o[r / 2][v][2 * (r % 2) + 1] *= keep;
				}
			}
		}
	};
	auto sum_keys = [&](const unsigned char *kt) { // 16 at a time
		for (int r = 16 * warp; r < KEYS; r += 16 * WARPS) {
			float ks[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
			for (int u = 0; u < W; u++) {
				const uint4 x = load_shared16(kt, tile_offset<false>(KP, r + g, 4 * u + j)), y = load_shared16(kt, tile_offset<false>(KP, r + g + 8, 4 * u + j));
				H::mma(ks, x.x, y.x, x.y, y.y, H::ONES, H::ONES);
				H::mma(ks, x.z, y.z, x.w, y.w, H::ONES, H::ONES);
			}
			if (j == 0) {
				key_sums[r + g] = ks[0];
				key_sums[r + g + 8] = ks[2];
			}
		}
	};

	// The distances to one step's keys are formed beside the weights and value products of the step before (no branch between them): a
	// warp alone then keeps the tensor cores busy.
	int it = next(0), following = end, stage = 0;
	float x[MB][2][4], y[MB][2][4];
	bool whole = false, special = false;
	const unsigned char *kt = nullptr;
	uint32_t vt = 0;
	auto enter = [&](int tile_of_keys) { // flags and places of a tile
		kt = reinterpret_cast<const unsigned char *>(smem16) + stage * stage_bytes;
		whole = tile_of_keys * KEYS + KEYS <= a.n && t1 == t0 + ROWS && mask.all(t0, t1, tile_of_keys * KEYS, tile_of_keys * KEYS + KEYS);
		special = !whole || a.cap > 0.f || a.slopes;
	};
	if (it < end) {
		fetch(it, 0);
		cp_async_commit();
		following = next(it + 1);
		cp_async_wait<0>();
		__syncthreads();
		enter(it);
		sum_keys(kt);
		distances(kt, 0, x);
		__syncthreads();
		if (following < end)
			fetch(following, 1);
		cp_async_commit();
		scores(x, it * KEYS, whole, special);
	}
	while (it < end) {
		vt = base + stage * stage_bytes + KEYS * KP * 16;
#pragma unroll 1
		for (int kb = 0; kb < KEYS / 16 - 1; kb++) {
			distances(kt, kb + 1, y);
			values(vt, kb, x);
			scores(y, it * KEYS + 16 * kb + 16, whole, special);
#pragma unroll
			for (int i = 0; i < MB * 8; i++)
				x[i / 8][i / 4 % 2][i % 4] = y[i / 8][i / 4 % 2][i % 4];
		}
		if (following >= end) {
			values(vt, KEYS / 16 - 1, x);
			break;
		}
		it = following;
		following = next(it + 1);
		stage ^= 1;
		cp_async_wait<0>();
		__syncthreads(); // the next tile is there
		enter(it);
		sum_keys(kt);
		distances(kt, 0, y);
		values(vt, KEYS / 16 - 1, x);
		__syncthreads(); // its keys' sums are there; everyone is done with the tile before
		if (following < end)
			fetch(following, stage ^ 1);
		cp_async_commit();
		scores(y, it * KEYS, whole, special);
#pragma unroll
		for (int i = 0; i < MB * 8; i++)
			x[i / 8][i / 4 % 2][i % 4] = y[i / 8][i / 4 % 2][i % 4];
	}

	// finish: the lanes' shares of the sums, the +1 form's key of score 0, and what is not finite
	unsigned again = 0; // rows to do again
#pragma unroll
	for (int r = 0; r < 2 * MB; r++) {
		l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
		l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
		if (a.mode == L1ATTN_SV_SOFTMAX_PLUS_ONE)
			l[r] += exp2_fast(-m[r]);
		float ls;
		const float f = finish_row(a.mode, m[r] / LOG2E, l[r], &ls);
		bool odd = !(fabsf(l[r]) < INFINITY) || !(fabsf(f) < INFINITY);
		const int t = ta + 8 * r;
		const long long row = ((long long)b * a.n + t) * a.heads + head;
		if (t < a.n && j == 0 && lse)
			lse[row] = ls;
#pragma unroll
		for (int i = 0; i < 2 * V; i++) {
			const int w = 8 * i + 2 * j;
			const float y0 = f == 0.f ? 0.f : o[r / 2][i][2 * (r % 2)] * f, y1 = f == 0.f ? 0.f : o[r / 2][i][2 * (r % 2) + 1] * f;
			odd |= !(fabsf(y0) < INFINITY) || !(fabsf(y1) < INFINITY);
			if (t < a.n && w < a.v_width) {
				if (vec & 8)
					*reinterpret_cast<uint32_t *>(vo + row * a.v_width + w) = H::pack(y0, y1);
				else {
					vo[row * a.v_width + w] = from_float<T>(y0);
					if (w + 1 < a.v_width)
						vo[row * a.v_width + w + 1] = from_float<T>(y1);
				}
			}
		}
		const unsigned lanes = __ballot_sync(0xffffffffu, odd);
#pragma unroll
		for (int i = 0; i < 8; i++)
			again |= (lanes >> (4 * i) & 15u) ? 1u << (8 * r + i) : 0u;
	}
	if (again == 0)
		return;
	__syncwarp();
	for (int r = 0; r < 16 * MB; r++) {
		const int t = t0 + 16 * MB * warp + r;
		if (t < a.n && (again >> r & 1u))
			exact_row<T>(a, mask, b, head, t, vo, lse);
	}
}

template <typename T, int W, int V> int fwd(const MaskedArgs &a, void *vo, float *lse, int vec, cudaStream_t st)
{
	constexpr int bytes = 2 * KEYS * (4 * W + 2 * V) * 16;
	static_assert(bytes >= ROWS * 4 * W * 16 && MB * 16 <= 32, "the query rows pass through the stages");
	const int tiles = (a.n + ROWS - 1) / ROWS;
	const long long grid = (long long)tiles * a.heads * a.bs;
	if (grid > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	L1B_SHARED_MEMORY((masked_fwd_mma_kernel<T, W, V>), bytes);
	masked_fwd_mma_kernel<T, W, V><<<unsigned(grid), THREADS, bytes, st>>>(a, static_cast<T *>(vo), lse, tiles, vec);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

// rows of 16-byte vectors: what asynchronous copies need
bool vectors(const Strided &x) { return aligned(x.p, 16) && x.batch % 8 == 0 && x.tok % 8 == 0 && x.head % 8 == 0; }

template <typename T> int fwd_type(const MaskedArgs &a, void *vo, float *lse, cudaStream_t st)
{
	const int vec = vectors(a.q) | vectors(a.k) << 1 | vectors(a.v) << 2 | (aligned(vo, 4) && a.v_width % 2 == 0) << 3, w = (a.width + 31) / 32;
	if (a.v_width <= 64)
		return w == 1 ? fwd<T, 1, 4>(a, vo, lse, vec, st) : w == 2 ? fwd<T, 2, 4>(a, vo, lse, vec, st) : w == 3 ? fwd<T, 3, 4>(a, vo, lse, vec, st) : fwd<T, 4, 4>(a, vo, lse, vec, st);
	return w == 1 ? fwd<T, 1, 8>(a, vo, lse, vec, st) : w == 2 ? fwd<T, 2, 8>(a, vo, lse, vec, st) : w == 3 ? fwd<T, 3, 8>(a, vo, lse, vec, st) : fwd<T, 4, 8>(a, vo, lse, vec, st);
}

} // namespace

bool masked_mma_fits(const MaskedArgs &a, int dtype) { return dtype != L1ATTN_F32 && a.width <= 128 && a.v_width <= 128; }

int masked_mma_fwd_launch(const MaskedArgs &a, void *vo, float *lse, int dtype, cudaStream_t st)
{
	return dtype == L1ATTN_F16 ? fwd_type<__half>(a, vo, lse, st) : fwd_type<__nv_bfloat16>(a, vo, lse, st);
}

} // namespace l1b
