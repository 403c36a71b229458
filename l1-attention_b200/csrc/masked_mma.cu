// Masked L1 attention (mask.cuh) of 16-bit rows up to 128 wide: distances and products on the tensor cores (mma.cuh).
//
// Forward: a CTA of four warps owns 64 query rows of one head, a warp 16 of them, in registers; keys and values stream in tiles of 64 through
// two stages of asynchronous copies.  Running softmax in registers (a row's scores lie in one quad); weights are rounded to the inputs' type for the value
// product, and what that leaves takes a second one (22 bits, or 16; the normaliser sums them unrounded), everything else is float32.  Rows whose result is not
// finite are done again, exactly, by a warp each: an infinite or NaN operand spoils its neighbours in a product.
// Bound: instruction issue of few warps.  mma.sync does not overlap float32 instructions (mma alone 8 clocks per scheduler, 13.2 with four
// additions, 9.7 with four minima), so the softmax costs what it takes; forming the next step's distances beside it brought [2,2048,8,128] from
// 343 to 293 us, the short copy loop a tenth; the weights' rests cost a tenth of it again: with
// them, and with what rounding leaves of vo kept for delta (masked.cu), dq is as exact as a float32 form's that rounds at the end in bfloat16 (1.38 of its
// error without).  Now 48 terms per clock and SM at widths of 64 ([4,2048,8,64], no mask: 615 us), 49 at 128 (1.20 ms).
#include "mma.cuh"

namespace l1b {

namespace {

constexpr int MB = 1, WARPS = 4, ROWS = 16 * MB * WARPS, KEYS = 64, STREAM = 32, THREADS = 32 * WARPS; // MB: blocks of 16 rows a warp
constexpr float LOG2E = 1.4426950408889634f, LAG = 8.f;
// float16 weights are formed times 2^LIFT, so that those of long flat rows are not lost below 2^-24 of the largest: at most 2^(LAG + LIFT)
template <typename T> constexpr float LIFT = Half2<T>::ONES == Half2<__half>::ONES ? 6.f : 0.f;

// One query row, by the definition: a warp, 32 keys at a time.  Rare, so simple.
template <typename T> __device__ __noinline__ void exact_row(const MaskedArgs &a, const MaskView &mask, int b, int head, int t, T *vo, T *rest, float *lse)
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
		if (lane + 32 * i < a.v_width) {
			const float y = f == 0.f ? 0.f : acc[i] * f;
			vo[row * a.v_width + lane + 32 * i] = from_float<T>(y);
			if (rest)
				rest[row * a.v_width + lane + 32 * i] = rest_of<T>(y);
		}
}

// W: 32-column groups of the width; V: 16-column groups of the value rows (4 or 8).  CTAs of an SM, two against three (168 registers), bfloat16: [1,4096,8,64]
// with values of 128 374 / 509 us, [2,2048,8,128] 327 / 457, widths of 32 227 / 257; but without a mask [4,2048,8,64] 695 / 615, widths of 128 and 96 with values of
// 64 1168 / 1055 and 863 / 837 (causal [1,8192,8,64] 1264 either way).
template <typename T, int W, int V>
__global__ void __launch_bounds__(THREADS, V == 4 && W > 1 ? 3 : 2) masked_fwd_mma_kernel(MaskedArgs a, T *vo, T *rest, float *lse, int tiles, int vec)
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
	const float slope = a.slopes ? a.slopes[head] : 0.f;

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

	float m[2 * MB], l[2 * MB], ref[2 * MB]; // per row: the largest score (times log2 e; it may lag), this lane's share of the sum, what exponents are taken relative to
	float o[MB][2 * V][4];
#pragma unroll
	for (int r = 0; r < 2 * MB; r++) {
		m[r] = -INFINITY; // (in every mode: weights are rounded relative to the row's largest)
		ref[r] = l[r] = 0.f;
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
		uint32_t p[MB][4], low[MB][4];
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
#pragma unroll
				for (int c = 0; c < 2; c++) {
					const uint32_t high = p[i][2 * h + c] = H::pack(e[2 * c], e[2 * c + 1]);
					const float2 f = H::unpack(high);
					low[i][2 * h + c] = H::pack(e[2 * c] - f.x, e[2 * c + 1] - f.y);
				}
			}
#pragma unroll
		for (int vb = 0; vb < V; vb++) {
			uint32_t y[4];
			ldmatrix4_trans(y, vt + tile_offset<true>(VP, 16 * kb + lane % 16, 2 * vb + lane / 16));
#pragma unroll
			for (int i = 0; i < MB; i++) {
				H::mma(o[i][2 * vb], p[i][0], p[i][1], p[i][2], p[i][3], y[0], y[1]);
				H::mma(o[i][2 * vb + 1], p[i][0], p[i][1], p[i][2], p[i][3], y[2], y[3]);
				H::mma(o[i][2 * vb], low[i][0], low[i][1], low[i][2], low[i][3], y[0], y[1]);
				H::mma(o[i][2 * vb + 1], low[i][0], low[i][1], low[i][2], low[i][3], y[2], y[3]);
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
			if (a.cap > 0.f)
				cap_scores<MB * 8, false>(&x[0][0][0], nullptr, a.cap);
#pragma unroll
			for (int i = 0; i < MB; i++)
#pragma unroll
				for (int c = 0; c < 8; c++) {
					const int s = s0 + 8 * (c / 4) + 2 * j + (c & 1), t = ta + 16 * i + 8 * (c / 2 % 2);
					float y = x[i][c / 4][c % 4];
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
				ref[r] = top[r] == -INFINITY ? 0.f : top[r] - LIFT<T>;
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
		l[r] *= exp2f(-LIFT<T>);
		float ls;
		const float f = finish_row_of_keys(a.mode, m[r] / LOG2E, l[r], &ls);
		bool odd = !(fabsf(l[r]) < INFINITY) || !(fabsf(f) < INFINITY);
		const int t = ta + 8 * r;
		const long long row = ((long long)b * a.n + t) * a.heads + head;
		if (t < a.n && j == 0 && lse)
			lse[row] = ls;
#pragma unroll
		for (int i = 0; i < 2 * V; i++) {
			const int w = 8 * i + 2 * j;
			const float y0 = f == 0.f ? 0.f : o[r / 2][i][2 * (r % 2)] * exp2f(-LIFT<T>) * f, y1 = f == 0.f ? 0.f : o[r / 2][i][2 * (r % 2) + 1] * exp2f(-LIFT<T>) * f;
			odd |= !(fabsf(y0) < INFINITY) || !(fabsf(y1) < INFINITY);
			if (t < a.n && w < a.v_width) {
				const long long at = row * a.v_width + w;
				if (vec & 8)
					*reinterpret_cast<uint32_t *>(vo + at) = H::pack(y0, y1);
				else {
					vo[at] = from_float<T>(y0);
					if (w + 1 < a.v_width)
						vo[at + 1] = from_float<T>(y1);
				}
				if (rest) {
					rest[at] = rest_of<T>(y0);
					if (w + 1 < a.v_width)
						rest[at + 1] = rest_of<T>(y1);
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
			exact_row<T>(a, mask, b, head, t, vo, rest, lse);
	}
}

// One row of dq, or of one query head's share of dk and dv, by the definition: a warp, 32 rows of the other side at a time.  Rare, so simple.
template <typename T, bool OWN_KEYS, typename OUT>
__device__ __noinline__ void exact_gradient_row(const MaskedArgs &a, const MaskView &mask, int b, int head, int o, const T *dvo, const float *lse, const float *delta, OUT *dx, OUT *dv)
{
	const int lane = threadIdx.x % 32, kv = head / (a.heads / a.kv_heads);
	const Strided go = {dvo, (long long)a.n * a.heads * a.v_width, (long long)a.heads * a.v_width, a.v_width};
	auto row_of = [&](const Strided &x, int h, int r) { return static_cast<const T *>(x.p) + b * x.batch + h * x.head + r * x.tok; };
	float acc[4] = {0.f, 0.f, 0.f, 0.f}, accv[4] = {0.f, 0.f, 0.f, 0.f};
	for (int r0 = 0; r0 < a.n; r0 += 32) {
		const int r = r0 + lane, t = OWN_KEYS ? r : o, s = OWN_KEYS ? o : r;
		const bool seen = r < a.n && mask.sees(t, s, mask.doc ? mask.doc[t] : 0, mask.doc ? mask.doc[s] : 0);
		if (!__any_sync(0xffffffffu, seen))
			continue;
		float p = 0.f, e = 0.f;
		if (seen) {
			const T *q = row_of(a.q, head, t), *k = row_of(a.k, kv, s), *v = row_of(a.v, kv, s), *g = row_of(go, head, t);
			float x = 0.f, dp = 0.f, slant = 1.f;
			for (int w = 0; w < a.width; w++)
				x += fabsf(to_float(q[w]) - to_float(k[w]));
			for (int w = 0; w < a.v_width; w++)
				dp = fmaf(to_float(v[w]), to_float(g[w]), dp);
			x *= -a.scale;
			if (a.cap > 0.f) {
				const float th = tanhf(x / a.cap);
				slant = 1.f - th * th;
				x = a.cap * th;
			}
			if (a.slopes)
				x -= a.slopes[head] * fabsf(float(t - s));
			const long long row = ((long long)b * a.n + t) * a.heads + head;
			p = weight_of(x, lse[row]);
			e = p == 0.f ? 0.f : -a.scale * slant * p * (dp - delta[row]);
		}
		for (int l = 0; l < 32; l++) {
			const float pl = __shfl_sync(0xffffffffu, p, l), el = __shfl_sync(0xffffffffu, e, l);
			if (pl == 0.f)
				continue;
			const T *mine = OWN_KEYS ? row_of(a.k, kv, o) : row_of(a.q, head, o), *other = OWN_KEYS ? row_of(a.q, head, r0 + l) : row_of(a.k, kv, r0 + l);
#pragma unroll
			for (int c = 0; c < 4; c++) {
				const int w = lane + 32 * c;
				if (w < a.width)
					acc[c] += sign_apply(to_float(mine[w]) - to_float(other[w]), el);
				if (OWN_KEYS && w < a.v_width)
					accv[c] = fmaf(pl, to_float(row_of(go, head, r0 + l)[w]), accv[c]);
			}
		}
	}
	const long long row = ((long long)b * a.n + o) * a.heads + head;
#pragma unroll
	for (int c = 0; c < 4; c++) {
		const int w = lane + 32 * c;
		if (w < a.width)
			dx[row * a.width + w] = from_float<OUT>(acc[c]);
		if (OWN_KEYS && w < a.v_width)
			dv[row * a.v_width + w] = from_float<OUT>(accv[c]);
	}
}

// What a backward kernel of some units -- query heads of batch items, [first, first + units) in order -- leaves beside the gradients.
struct BackwardParts {
	int first, units;
	float *e;               // gradients of the distances, [unit][t][pitch s], for the queries' kernel; or null
	long long unit_floats;
	int pitch;
	float *dk, *dv;         // [bs][n][heads][width]: each query head's share of shared heads' gradients; or null
};

// Own rows for the signs: every value twice in a word, as it is or as its code, [row][g][column block][w = g, g + 8] in pieces of 16 bytes that lie so that
// the eight g of one piece are in different banks.  Returns whether codes do not hold a value.
template <int W> __device__ __forceinline__ int own_word(int row, int g, int word) // word: column block * 2 + half
{
	const int piece = word / 4;
	return (row * 8 + g) * 4 * W + (W == 4 ? piece ^ (g / 2) : W == 2 ? piece ^ (g / 4) : piece) * 4 + word % 4;
}
template <typename T, int W> __device__ __forceinline__ uint32_t own_table(unsigned char *table, const unsigned char *rows, int tid)
{
	uint32_t off = 0;
	for (int i = tid; i < ROWS * 32 * W; i += THREADS) {
		const int r = i / (32 * W), w = i % (32 * W);
		const uint32_t twice = reinterpret_cast<const uint16_t *>(rows)[i] * 0x10001u;
		reinterpret_cast<uint32_t *>(table)[own_word<W>(r, w % 8, w / 16 * 2 + w / 8 % 2)] = Half2<T>::ONES == Half2<__half>::ONES ? twice : codes_of_bf16(twice, &off);
	}
	return off;
}

// 1 - codes of a streamed tile, in the same places
template <int W, int KP> __device__ __forceinline__ void encode_tile(unsigned char *to, const unsigned char *from, uint32_t *off, int tid)
{
#pragma unroll
	for (int i = tid; i < STREAM * 4 * W; i += THREADS) {
		const uint32_t at = tile_offset<true>(KP, i / (4 * W), i % (4 * W));
		uint4 v = *reinterpret_cast<const uint4 *>(from + at);
		v.x = __vsub2(0x10001u, codes_of_bf16(v.x, off));
		v.y = __vsub2(0x10001u, codes_of_bf16(v.y, off));
		v.z = __vsub2(0x10001u, codes_of_bf16(v.z, off));
		v.w = __vsub2(0x10001u, codes_of_bf16(v.w, off));
		*reinterpret_cast<uint4 *>(to + at) = v;
	}
}

// acc[column block][own rows 0-7, 8-15] += signs(own - streamed) e of 16 own rows and 16 streamed ones (rows `first` of the tile at xs); the products' rows
// are columns w, their columns own rows.  coded: both sides are codes, and signs one too large; else streamed values, and own ones of `plain` for bfloat16.
// TWICE: what rounding left of e (el) takes a product of its own, with the same signs; not for codes.
template <typename T, int W, bool TWICE>
__device__ __forceinline__ void add_signed(float (&acc)[2 * W][2][4], const uint32_t (&eb)[2][2], const uint32_t (&el)[2][2], bool coded, uint32_t xs, int first, const unsigned char *table,
					   const uint16_t *plain, int warp, int lane)
{
	using H = Half2<T>;
	constexpr int KP = W == 3 ? 16 : 4 * W, WB = 2 * W;
	constexpr bool CODES = H::ONES == Half2<__nv_bfloat16>::ONES;
	const int g = lane / 4;
	uint32_t x[WB][4]; // streamed rows, [w = g, g + 8][streamed pairs]
#pragma unroll
	for (int wb = 0; wb < WB; wb++)
		ldmatrix4_trans(x[wb], xs + tile_offset<true>(KP, first + lane % 8 + lane / 16 * 8, 2 * wb + lane / 8 % 2));
	const uint32_t *twice = reinterpret_cast<const uint32_t *>(table);
	if (coded) {
#pragma unroll 1
		for (int r = 0; r < 8; r++)
#pragma unroll
			for (int half = 0; half < 2; half++) {
				const uint32_t b0 = g == r ? eb[half][0] : 0u, b1 = g == r ? eb[half][1] : 0u;
#pragma unroll
				for (int wb = 0; wb < WB; wb += 2) {
					const uint4 w = *reinterpret_cast<const uint4 *>(twice + own_word<W>(16 * warp + r + 8 * half, g, 2 * wb));
					Half2<__half>::mma(acc[wb][half], signs_of_codes(w.x, x[wb][0]), signs_of_codes(w.y, x[wb][1]), signs_of_codes(w.x, x[wb][2]),
							   signs_of_codes(w.y, x[wb][3]), b0, b1);
					Half2<__half>::mma(acc[wb + 1][half], signs_of_codes(w.z, x[wb + 1][0]), signs_of_codes(w.w, x[wb + 1][1]),
							   signs_of_codes(w.z, x[wb + 1][2]), signs_of_codes(w.w, x[wb + 1][3]), b0, b1);
				}
			}
		return;
	}
#pragma unroll 1
	for (int r = 0; r < 8; r++)
#pragma unroll
		for (int half = 0; half < 2; half++) {
			const uint32_t b0 = g == r ? eb[half][0] : 0u, b1 = g == r ? eb[half][1] : 0u;
			const uint32_t l0 = TWICE && g == r ? el[half][0] : 0u, l1 = TWICE && g == r ? el[half][1] : 0u;
			const uint16_t *row = plain + (16 * warp + r + 8 * half) * 32 * W + g;
#pragma unroll
			for (int wb = 0; wb < WB; wb += 2) {
				uint4 w;
				if (CODES)
					w = make_uint4(row[16 * wb] * 0x10001u, row[16 * wb + 8] * 0x10001u, row[16 * wb + 16] * 0x10001u, row[16 * wb + 24] * 0x10001u);
				else
					w = *reinterpret_cast<const uint4 *>(twice + own_word<W>(16 * warp + r + 8 * half, g, 2 * wb));
				const uint32_t s0[4] = {H::sign(w.x, x[wb][0]), H::sign(w.y, x[wb][1]), H::sign(w.x, x[wb][2]), H::sign(w.y, x[wb][3])};
				const uint32_t s1[4] = {H::sign(w.z, x[wb + 1][0]), H::sign(w.w, x[wb + 1][1]), H::sign(w.z, x[wb + 1][2]), H::sign(w.w, x[wb + 1][3])};
				Half2<__half>::mma(acc[wb][half], s0[0], s0[1], s0[2], s0[3], b0, b1);
				Half2<__half>::mma(acc[wb + 1][half], s1[0], s1[1], s1[2], s1[3], b0, b1);
				if (TWICE) {
					Half2<__half>::mma(acc[wb][half], s0[0], s0[1], s0[2], s0[3], l0, l1);
					Half2<__half>::mma(acc[wb + 1][half], s1[0], s1[1], s1[2], s1[3], l0, l1);
				}
			}
		}
}

// e is rounded to float16 times a power of two per own row (`unit`; rows g, g + 8 of this lane's quad), which puts the row's largest so far near 2^11: 25
// binades below it keep 11 bits.  Called when an e is beyond a row's limit (2^15 by the present unit); what was added up follows.
template <int W> __device__ __forceinline__ void follow_largest(const float (&e)[2][4], float (&unit)[2], float (&limit)[2], float (&e_sum)[4], float (&acc)[2 * W][2][4], int j)
{
	float keep[2];
#pragma unroll
	for (int r = 0; r < 2; r++) {
		float most = fmaxf(fmaxf(fabsf(e[0][2 * r]), fabsf(e[0][2 * r + 1])), fmaxf(fabsf(e[1][2 * r]), fabsf(e[1][2 * r + 1])));
		most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
		most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
		keep[r] = 1.f;
		if (most > limit[r]) {
			// (exponents cut so that both powers are normal; what is not finite stays so, in its row)
			const int top = min(max(int(__float_as_uint(most) >> 23), 13), 242);
			const float now = __uint_as_float(uint32_t(254 + 11 - top) << 23);
			keep[r] = limit[r] == 0.f ? 1.f : now / unit[r];
			unit[r] = now;
			limit[r] = __uint_as_float(uint32_t(top + 4) << 23);
		}
	}
	e_sum[0] *= keep[0];
	e_sum[2] *= keep[1];
	// the products' columns are own rows: 2 j and 2 j + 1, and the same + 8
	const float k0 = __shfl_sync(0xffffffffu, keep[0], 8 * j), k1 = __shfl_sync(0xffffffffu, keep[0], 8 * j + 4);
	const float k2 = __shfl_sync(0xffffffffu, keep[1], 8 * j), k3 = __shfl_sync(0xffffffffu, keep[1], 8 * j + 4);
#pragma unroll
	for (int wb = 0; wb < 2 * W; wb++) {
		acc[wb][0][0] *= k0, acc[wb][0][1] *= k1, acc[wb][0][2] *= k0, acc[wb][0][3] *= k1;
		acc[wb][1][0] *= k2, acc[wb][1][1] *= k3, acc[wb][1][2] *= k2, acc[wb][1][3] *= k3;
	}
}

// The same for weights on their way to dv in float16, relative to their own row's (key's) largest so far: without a normaliser, or for a key that nobody
// weighs much, they are as small as exp(score).
template <int N> __device__ __forceinline__ void follow_largest_weight(const float (&p)[2][4], float (&unit)[2], float (&limit)[2], float (&acc)[N][4])
{
#pragma unroll
	for (int r = 0; r < 2; r++) {
		float most = fmaxf(fmaxf(p[0][2 * r], p[0][2 * r + 1]), fmaxf(p[1][2 * r], p[1][2 * r + 1]));
		most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
		most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
		float keep = 1.f;
		if (most > limit[r]) {
			const int top = min(max(int(__float_as_uint(most) >> 23), 13), 242);
			const float now = __uint_as_float(uint32_t(254 + 11 - top) << 23);
			keep = limit[r] == 0.f ? 1.f : now / unit[r];
			unit[r] = now;
			limit[r] = __uint_as_float(uint32_t(top + 4) << 23);
		}
#pragma unroll
		for (int i = 0; i < N; i++) {
			acc[i][2 * r] *= keep;
			acc[i][2 * r + 1] *= keep;
		}
	}
}

// Signs were 2^-24 (and one too large where e_sum counts them), e times unit: a warp's 16 rows of the gradient, to `part` or `dx`.  Returns the rows whose
// values are not finite, by this lane.
template <typename T, int W>
__device__ __forceinline__ unsigned store_signed(const float (&acc)[2 * W][2][4], const float (&unit)[2], const float (&e_sum)[4], const MaskedArgs &a, int b, int head,
						 int first, int lane, float *part, T *dx)
{
	const int g = lane / 4, j = lane % 4;
	const float u0 = 0x1p24f / unit[0], u1 = 0x1p24f / unit[1], s0 = e_sum[0] * 0x1p-24f, s1 = e_sum[2] * 0x1p-24f;
	unsigned again = 0;
#pragma unroll
	for (int i = 0; i < 4; i++) { // rows 2 j, 2 j + 1, the same + 8
		const int in_warp = 2 * j + (i & 1) + 8 * (i / 2), o = first + in_warp, from = 8 * j + 4 * (i & 1);
		const float f = __shfl_sync(0xffffffffu, i < 2 ? u0 : u1, from), less = __shfl_sync(0xffffffffu, i < 2 ? s0 : s1, from);
		bool odd = false;
#pragma unroll
		for (int wb = 0; wb < 2 * W; wb++)
#pragma unroll
			for (int h = 0; h < 2; h++) {
				const int w = 16 * wb + 8 * h + g;
				const float y = (acc[wb][i / 2][2 * h + (i & 1)] - less) * f;
				odd |= !(fabsf(y) < INFINITY);
				if (o < a.n && w < a.width) {
					const long long at = (((long long)b * a.n + o) * a.heads + head) * a.width + w;
					if (part)
						part[at] = y;
					else
						dx[at] = from_float<T>(y);
				}
			}
		again |= odd ? 1u << in_warp : 0u;
	}
	return again;
}

// Backward: a CTA owns 64 rows of one query head -- its keys (dk, dv: its share of them, where heads are shared), or its queries (dq) -- and streams the
// other side 32 rows at a time.  The keys' kernel leaves the gradients of the distances for the queries' (masked_dq_mma_kernel), whose own form here, with
// the weights formed again, serves where they would take too much memory.  16 x 16 at a time:
//   scores            rows own, columns streamed, as in the forward
//   dP                own values (or dvo) times streamed dvo (values)
//   e = -scale p (dP - delta) slant, the gradient of the distance; rounded to float16 relative to its row's largest so far (a power of two that follows);
//                     next to float16 outputs what that leaves takes a second product (dk and dq 1.4 and 1.55 times as far from 64 bits without; 8 and 9 % of the time)
//   gradient          sum over the streamed rows of sign(own - streamed) e: for each own row a product with A = the signs [w][streamed], exact, and
//                     B = e in the column of that row: 16 own rows fill two 16 x 8 tiles per 16 columns.  Signs take two instructions for two values
//                     (a subtraction, which mma.sync does not overlap, and a minimum), or one for bfloat16 as codes of 15 bits; a tile with values
//                     that these do not hold takes the two
//   dv                p^T dvo, weights rounded to the type (float16: relative to their row's largest so far, as e) and what that leaves in a second product
//                     (without it dv is 1.4 times as far from 64 bits as when rounded once; 1.5 % of the time)
// No atomics, and the same sums in the same order every time.
// Bound: the tensor pipe and the instructions that feed it, of 8 warps an SM (registers: two CTAs).  [2,2048,8,128], causal, two heads of keys, bfloat16:
// 1.30 ms; [1,8192,8,64], float16: 6.08 ms; [4,2048,8,128], no mask, bfloat16: 4.49 ms (in float32 arithmetic, masked_simple.cu: 15.6).
template <typename T, bool OWN_KEYS, int W, int V>
__global__ void __launch_bounds__(THREADS, 2) masked_bwd_mma_kernel(MaskedArgs a, const T *dvo, const float *lse, const float *delta, T *dx, T *dv, BackwardParts parts, int tiles, int vec)
{
	extern __shared__ uint4 smem16[];
	__shared__ float sums[STREAM], stats[2][2][STREAM]; // [stage][log-normaliser, delta] of streamed queries
	using H = Half2<T>;
	constexpr int KP = W == 3 ? 16 : 4 * W, VP = 2 * V, WB = 2 * W; // 16-byte pieces of a row; 16-column blocks
	constexpr bool CODES = H::ONES == Half2<__nv_bfloat16>::ONES, TWICE = !CODES;
	constexpr uint32_t OWN_Y = ROWS * 64 * W * 2, STAGES = OWN_Y + ROWS * VP * 16, STAGE = STREAM * (KP + VP) * 16, OWN_X = STAGES + 2 * STAGE, CODED = OWN_X + ROWS * 64 * W;
	unsigned char *const smem = reinterpret_cast<unsigned char *>(smem16);
	const uint32_t base = shared_address(smem16);
	const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, j = lane % 4;
	const int unit_bh = blockIdx.x % parts.units, rank = blockIdx.x / parts.units, bh = parts.first + unit_bh; // (a unit: a query head of a batch item)
	const int tile = OWN_KEYS ? rank : tiles - 1 - rank; // what a causal mask leaves most work first
	const int head = bh % a.heads, b = bh / a.heads, kv = head / (a.heads / a.kv_heads);
	const MaskView mask(a, b);
	const int o0 = tile * ROWS, o1 = min(a.n, o0 + ROWS), oa = o0 + 16 * warp + g; // this lane's rows: oa, oa + 8
	const Strided go = {dvo, (long long)a.n * a.heads * a.v_width, (long long)a.heads * a.v_width, a.v_width};

	// own rows stay in shared memory: as they are for the scores (registers that held them were missing beside the sums), as a table for the signs
	const int32_t *own_doc = mask.doc && mask.ranges[o0 / DOC_TILE].others ? mask.doc : nullptr;
	load_tile16<T, false, 4 * W, ROWS, THREADS>(base + OWN_X, OWN_KEYS ? a.k : a.q, b, OWN_KEYS ? kv : head, o0, a.n, a.width, own_doc, vec & (OWN_KEYS ? 2 : 1), tid);
	load_tile16<T, true, VP, ROWS, THREADS>(base + OWN_Y, OWN_KEYS ? a.v : go, b, OWN_KEYS ? kv : head, o0, a.n, a.v_width, own_doc, vec & (OWN_KEYS ? 4 : 8), tid);
	cp_async_commit();
	cp_async_wait<0>();
	__syncthreads();
	const unsigned char *const own_rows = smem + OWN_X;
	float own_sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int u = 0; u < W; u++) {
		const uint4 x = load_shared16(own_rows, tile_offset<false>(4 * W, 16 * warp + g, 4 * u + j)), y = load_shared16(own_rows, tile_offset<false>(4 * W, 16 * warp + g + 8, 4 * u + j));
		H::mma(own_sum, x.x, y.x, x.y, y.y, H::ONES, H::ONES);
		H::mma(own_sum, x.z, y.z, x.w, y.w, H::ONES, H::ONES);
	}
	uint32_t own_off = own_table<T, W>(smem, own_rows, tid);

	float acc[WB][2][4], accv[OWN_KEYS ? 2 * V : 1][4]; // [column block][own rows 0-7, 8-15]: rows of the product are columns w, its columns own rows
#pragma unroll
	for (int i = 0; i < WB * 8; i++)
		acc[i / 8][i / 4 % 2][i % 4] = 0.f;
#pragma unroll
	for (int i = 0; i < (OWN_KEYS ? 2 * V : 1) * 4; i++)
		accv[i / 4][i % 4] = 0.f;
	float e_sum[4] = {0.f, 0.f, 0.f, 0.f}; // CODES: of the rounded e, by own row: signs there are one too large
	float unit[2] = {1.f, 1.f}, limit[2] = {0.f, 0.f}; // per row: a power of two times e is rounded to float16; e may come this far
	float p_unit[2] = {1.f, 1.f}, p_limit[2] = {0.f, 0.f}; // the same for weights, in float16

	// tiles of the other side
	const int first_tile = [&] {
		if (OWN_KEYS)
			return mask.causal && o0 >= mask.prefix ? o0 / STREAM : 0;
		return 0;
	}();
	const int prefix_tiles = OWN_KEYS ? 0 : (min(mask.prefix, a.n) + STREAM - 1) / STREAM;
	const int lo = !OWN_KEYS && mask.window ? max(o0 - mask.window + 1, 0) / STREAM : 0;
	const int all_tiles = (a.n + STREAM - 1) / STREAM;
	const int end = OWN_KEYS ? (mask.causal && mask.window && o0 >= mask.prefix ? int(min((long long)all_tiles, ((long long)o1 + mask.window + STREAM - 1) / STREAM)) : all_tiles) :
				   max(mask.causal ? (o1 + STREAM - 1) / STREAM : all_tiles, prefix_tiles);
	auto next = [&](int i) {
		for (;; i++) {
			if (i >= prefix_tiles && i < lo)
				i = lo;
			if (i >= end)
				return end;
			const int r0 = i * STREAM, r1 = min(a.n, r0 + STREAM);
			if (OWN_KEYS ? mask.any(r0, r1, o0, o1) : mask.any(o0, o1, r0, r1))
				return i;
		}
	};
	auto fetch = [&](int i, int stage) {
		const int other = OWN_KEYS ? head : kv;
		const int32_t *doc = mask.doc && mask.ranges[i * STREAM / DOC_TILE].others ? mask.doc : nullptr;
		const uint32_t at = base + STAGES + stage * STAGE;
		load_tile16<T, true, 4 * W, STREAM, THREADS, KP>(at, OWN_KEYS ? a.q : a.k, b, other, i * STREAM, a.n, a.width, doc, vec & (OWN_KEYS ? 1 : 2), tid);
		load_tile16<T, true, VP, STREAM, THREADS>(at + STREAM * KP * 16, OWN_KEYS ? go : a.v, b, other, i * STREAM, a.n, a.v_width, doc, vec & (OWN_KEYS ? 8 : 4), tid);
		if (OWN_KEYS && tid < 2 * STREAM) {
			const int t = i * STREAM + tid % STREAM;
			const float *from = (tid < STREAM ? lse : delta) + ((long long)b * a.n + min(t, a.n - 1)) * a.heads + head;
			asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(shared_address(&stats[stage][tid / STREAM][tid % STREAM])), "l"(from) : "memory");
		}
	};
	// a row's log-normaliser as the exponent takes it: a row without weights gets +inf, so that its weights are zero
	auto exponent = [&](float x) { return x == -INFINITY ? INFINITY : x * LOG2E; };
	float row_lse[2] = {0.f, 0.f}, row_delta[2] = {0.f, 0.f};
	if (!OWN_KEYS)
#pragma unroll
		for (int r = 0; r < 2; r++) {
			const long long row = ((long long)b * a.n + oa + 8 * r) * a.heads + head;
			row_lse[r] = oa + 8 * r < a.n ? exponent(lse[row]) : INFINITY;
			row_delta[r] = oa + 8 * r < a.n ? delta[row] : 0.f;
		}
	own_off = __syncthreads_or(own_off != 0);

	const float slope = a.slopes ? a.slopes[head] : 0.f;
	int it = next(first_tile), stage = 0;
	if (it < end)
		fetch(it, 0);
	cp_async_commit();
	while (it < end) {
		const int following = next(it + 1), r0 = it * STREAM, r1 = min(a.n, r0 + STREAM);
		cp_async_wait<0>();
		__syncthreads(); // the tile is there; everyone is done with the other stage
		if (following < end)
			fetch(following, stage ^ 1);
		cp_async_commit();
		const unsigned char *xt = smem + STAGES + stage * STAGE;
		const uint32_t xs = base + STAGES + stage * STAGE, ys = xs + STREAM * KP * 16;
		for (int r = 16 * warp; r < STREAM; r += 16 * WARPS) { // sums of the streamed rows
			float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
			for (int u = 0; u < W; u++) {
				const uint4 x = load_shared16(xt, tile_offset<true>(KP, r + g, 4 * u + j)), y = load_shared16(xt, tile_offset<true>(KP, r + g + 8, 4 * u + j));
				H::mma(s, x.x, y.x, x.y, y.y, H::ONES, H::ONES);
				H::mma(s, x.z, y.z, x.w, y.w, H::ONES, H::ONES);
			}
			if (j == 0) {
				sums[r + g] = s[0];
				sums[r + g + 8] = s[2];
			}
		}
		uint32_t off = own_off;
		if (CODES)
			encode_tile<W, KP>(smem + CODED, xt, &off, tid);
		off = __syncthreads_or(off != 0);
		const bool whole = r1 == r0 + STREAM && o1 == o0 + ROWS && (OWN_KEYS ? mask.all(r0, r1, o0, o1) : mask.all(o0, o1, r0, r1));
#pragma unroll 1
		for (int kb = 0; kb < STREAM / 16; kb++) {
			float x[2][4] = {}, dp[2][4] = {};
			uint32_t x_own[WB][4];
#pragma unroll
			for (int u = 0; u < W; u++) {
				const uint4 v = load_shared16(own_rows, tile_offset<false>(4 * W, 16 * warp + g, 4 * u + j)), w = load_shared16(own_rows, tile_offset<false>(4 * W, 16 * warp + g + 8, 4 * u + j));
				x_own[2 * u][0] = v.x, x_own[2 * u][1] = w.x, x_own[2 * u][2] = v.y, x_own[2 * u][3] = w.y;
				x_own[2 * u + 1][0] = v.z, x_own[2 * u + 1][1] = w.z, x_own[2 * u + 1][2] = v.w, x_own[2 * u + 1][3] = w.w;
			}
#pragma unroll
			for (int n = 0; n < 8; n++) {
				const uint32_t one = g == n ? H::ONES : 0u;
#pragma unroll
				for (int u = 0; u < W; u++)
#pragma unroll
					for (int h = 0; h < 2; h++) {
						const uint4 k = load_shared16(xt, tile_offset<true>(KP, 16 * kb + 8 * h + n, 4 * u + j));
						H::mma(x[h], H::min(x_own[2 * u][0], k.x), H::min(x_own[2 * u][1], k.x), H::min(x_own[2 * u][2], k.y), H::min(x_own[2 * u][3], k.y), one, one);
						H::mma(x[h], H::min(x_own[2 * u + 1][0], k.z), H::min(x_own[2 * u + 1][1], k.z), H::min(x_own[2 * u + 1][2], k.w),
						       H::min(x_own[2 * u + 1][3], k.w), one, one);
					}
			}
#pragma unroll
			for (int vb = 0; vb < V; vb++) {
				uint32_t y[4], z[4];
				ldmatrix4(y, base + OWN_Y + tile_offset<true>(VP, 16 * warp + lane % 16, 2 * vb + lane / 16));
				ldmatrix4(z, ys + tile_offset<true>(VP, 16 * kb + lane % 8 + lane / 16 * 8, 2 * vb + lane / 8 % 2));
				H::mma(dp[0], y[0], y[1], y[2], y[3], z[0], z[1]);
				H::mma(dp[1], y[0], y[1], y[2], y[3], z[2], z[3]);
			}
			// weights and gradients of the distances
			float slant[2][4];
			float2 lse_c[2], delta_c[2];
#pragma unroll
			for (int h = 0; h < 2; h++) {
				const int c0 = 16 * kb + 8 * h + 2 * j;
				const float2 s = *reinterpret_cast<const float2 *>(&sums[c0]);
				if (OWN_KEYS) {
					const float2 l = *reinterpret_cast<const float2 *>(&stats[stage][0][c0]);
					lse_c[h] = make_float2(exponent(l.x), exponent(l.y));
					delta_c[h] = *reinterpret_cast<const float2 *>(&stats[stage][1][c0]);
				} else
					lse_c[h] = delta_c[h] = make_float2(0.f, 0.f);
#pragma unroll
				for (int c = 0; c < 4; c++) {
					x[h][c] = a.scale * (fmaf(2.f, x[h][c], -own_sum[c & 2]) - (c & 1 ? s.y : s.x));
					slant[h][c] = -a.scale;
				}
			}
			if (a.cap > 0.f)
				cap_scores<8, true>(&x[0][0], &slant[0][0], a.cap);
			if (!whole || a.slopes) {
#pragma unroll
				for (int h = 0; h < 2; h++)
#pragma unroll
					for (int c = 0; c < 4; c++) {
						const int r = r0 + 16 * kb + 8 * h + 2 * j + (c & 1), o = oa + 8 * (c / 2), t = OWN_KEYS ? r : o, s = OWN_KEYS ? o : r;
						float y = x[h][c];
						if (a.slopes)
							y -= slope * fabsf(float(t - s));
						if (!whole && !(t < a.n && s < a.n && mask.sees(t, s, mask.doc ? mask.doc[t] : 0, mask.doc ? mask.doc[s] : 0)))
							y = -INFINITY;
						x[h][c] = y;
					}
			}
			float e[2][4];
			bool grew = false;
#pragma unroll
			for (int h = 0; h < 2; h++)
#pragma unroll
				for (int c = 0; c < 4; c++) {
					const float ls = OWN_KEYS ? (c & 1 ? lse_c[h].y : lse_c[h].x) : row_lse[c / 2], de = OWN_KEYS ? (c & 1 ? delta_c[h].y : delta_c[h].x) : row_delta[c / 2];
					const float p = exp2_fast(fmaf(x[h][c], LOG2E, -ls));
					e[h][c] = p == 0.f ? 0.f : p * slant[h][c] * (dp[h][c] - de);
					x[h][c] = p;
					grew |= fabsf(e[h][c]) > limit[c / 2] || (OWN_KEYS && !CODES && p > p_limit[c / 2]);
				}
			if (__any_sync(0xffffffffu, grew)) {
				follow_largest<W>(e, unit, limit, e_sum, acc, j);
				if constexpr (OWN_KEYS && !CODES)
					follow_largest_weight(x, p_unit, p_limit, accv);
			}
			uint32_t eb[2][2], el[2][2] = {}; // [own row g, g + 8][streamed 0-7, 8-15]; el: what rounding left
#pragma unroll
			for (int i = 0; i < 4; i++) {
				const float e0 = e[i % 2][i / 2 * 2] * unit[i / 2], e1 = e[i % 2][i / 2 * 2 + 1] * unit[i / 2];
				eb[i / 2][i % 2] = Half2<__half>::pack(e0, e1);
				if (TWICE) {
					const float2 f = Half2<__half>::unpack(eb[i / 2][i % 2]);
					el[i / 2][i % 2] = Half2<__half>::pack(e0 - f.x, e1 - f.y);
				}
			}
			if (OWN_KEYS && parts.e) { // for the queries' kernel: [unit][t][s]
				float *const to = parts.e + unit_bh * parts.unit_floats + (long long)(r0 + 16 * kb + 2 * j) * parts.pitch + oa;
#pragma unroll
				for (int h = 0; h < 2; h++)
#pragma unroll
					for (int c = 0; c < 4; c++)
						to[(8 * h + (c & 1)) * parts.pitch + 8 * (c / 2)] = e[h][c];
			}
			if (OWN_KEYS) {
				uint32_t p[4], low[4]; // low: what rounding left
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const float p0 = x[i / 2][i % 2 * 2] * p_unit[i % 2], p1 = x[i / 2][i % 2 * 2 + 1] * p_unit[i % 2];
					p[i] = H::pack(p0, p1);
					const float2 f = H::unpack(p[i]);
					low[i] = H::pack(p0 - f.x, p1 - f.y);
				}
#pragma unroll
				for (int vb = 0; vb < V; vb++) {
					uint32_t y[4];
					ldmatrix4_trans(y, ys + tile_offset<true>(VP, 16 * kb + lane % 16, 2 * vb + lane / 16));
					float(&a0)[4] = accv[(2 * vb) % (OWN_KEYS ? 2 * V : 1)], (&a1)[4] = accv[(2 * vb + 1) % (OWN_KEYS ? 2 * V : 1)];
					H::mma(a0, p[0], p[1], p[2], p[3], y[0], y[1]);
					H::mma(a1, p[0], p[1], p[2], p[3], y[2], y[3]);
					H::mma(a0, low[0], low[1], low[2], low[3], y[0], y[1]);
					H::mma(a1, low[0], low[1], low[2], low[3], y[2], y[3]);
				}
			}
			const bool coded = CODES && !off;
			if (coded) // (one product: e as A, ones as B)
				Half2<__half>::mma(e_sum, eb[0][0], eb[1][0], eb[0][1], eb[1][1], Half2<__half>::ONES, Half2<__half>::ONES);
			add_signed<T, W, TWICE>(acc, eb, el, coded, coded ? base + CODED : xs, 16 * kb, smem, reinterpret_cast<const uint16_t *>(smem + OWN_X), warp, lane);
		}
		it = following;
		stage ^= 1;
	}

	unsigned again = store_signed<T, W>(acc, unit, e_sum, a, b, head, o0 + 16 * warp, lane, OWN_KEYS ? parts.dk : nullptr, dx);
	if (OWN_KEYS) {
#pragma unroll
		for (int r = 0; r < 2; r++) {
			const int o = oa + 8 * r;
			bool odd = false;
#pragma unroll
			for (int i = 0; i < 2 * V; i++)
#pragma unroll
				for (int c = 0; c < 2; c++) {
					const int w = 8 * i + 2 * j + c;
					const float y = accv[i % (OWN_KEYS ? 2 * V : 1)][2 * r + c] * (1.f / p_unit[r]);
					odd |= !(fabsf(y) < INFINITY);
					if (o < a.n && w < a.v_width) {
						const long long at = (((long long)b * a.n + o) * a.heads + head) * a.v_width + w;
						if (parts.dv)
							parts.dv[at] = y;
						else
							dv[at] = from_float<T>(y);
					}
				}
			again |= odd ? 1u << (g + 8 * r) : 0u;
		}
	}
	again = __reduce_or_sync(0xffffffffu, again);
	for (int r = 0; r < 16; r++)
		if (again >> r & 1u && o0 + 16 * warp + r < a.n) {
			if (OWN_KEYS && parts.dk)
				exact_gradient_row<T, OWN_KEYS>(a, mask, b, head, o0 + 16 * warp + r, dvo, lse, delta, parts.dk, parts.dv);
			else
				exact_gradient_row<T, OWN_KEYS>(a, mask, b, head, o0 + 16 * warp + r, dvo, lse, delta, dx, dv);
		}
}

// The queries' gradients from stored gradients of the distances (parts.e, by the keys' kernel): signs alone.  64 query rows a CTA, keys in tiles of 32.
template <typename T, int W>
__global__ void __launch_bounds__(THREADS, 3) masked_dq_mma_kernel(MaskedArgs a, const T *dvo, const float *lse, const float *delta, T *dq, BackwardParts parts, int tiles, int vec)
{
	extern __shared__ uint4 smem16[];
	constexpr int KP = W == 3 ? 16 : 4 * W, WB = 2 * W;
	constexpr bool CODES = Half2<T>::ONES == Half2<__nv_bfloat16>::ONES, TWICE = !CODES;
	constexpr uint32_t STAGES = ROWS * 128 * W, STAGE = STREAM * KP * 16, OWN_X = STAGES + 2 * STAGE, CODED = OWN_X + ROWS * 64 * W, FROM = CODES ? OWN_X : STAGES;
	unsigned char *const smem = reinterpret_cast<unsigned char *>(smem16);
	const uint32_t base = shared_address(smem16);
	const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, j = lane % 4;
	const int unit_bh = blockIdx.x % parts.units, bh = parts.first + unit_bh, tile = tiles - 1 - int(blockIdx.x / parts.units);
	const int head = bh % a.heads, b = bh / a.heads, kv = head / (a.heads / a.kv_heads);
	const MaskView mask(a, b);
	const int o0 = tile * ROWS, o1 = min(a.n, o0 + ROWS), oa = o0 + 16 * warp + g;
	load_tile16<T, false, 4 * W, ROWS, THREADS>(base + FROM, a.q, b, head, o0, a.n, a.width, mask.doc && mask.ranges[o0 / DOC_TILE].others ? mask.doc : nullptr, vec & 1, tid);
	cp_async_commit();
	cp_async_wait<0>();
	__syncthreads();
	uint32_t own_off = own_table<T, W>(smem, smem + FROM, tid);
	float acc[WB][2][4];
#pragma unroll
	for (int i = 0; i < WB * 8; i++)
		acc[i / 8][i / 4 % 2][i % 4] = 0.f;
	float e_sum[4] = {0.f, 0.f, 0.f, 0.f}, unit[2] = {1.f, 1.f}, limit[2] = {0.f, 0.f};
	const int all_tiles = (a.n + STREAM - 1) / STREAM, prefix_tiles = (min(mask.prefix, a.n) + STREAM - 1) / STREAM;
	const int lo = mask.window ? max(o0 - mask.window + 1, 0) / STREAM : 0, end = max(mask.causal ? (o1 + STREAM - 1) / STREAM : all_tiles, prefix_tiles);
	auto next = [&](int i) {
		for (;; i++) {
			if (i >= prefix_tiles && i < lo)
				i = lo;
			if (i >= end || mask.any(o0, o1, i * STREAM, min(a.n, i * STREAM + STREAM)))
				return i;
		}
	};
	auto fetch = [&](int i, int stage) {
		load_tile16<T, true, 4 * W, STREAM, THREADS, KP>(base + STAGES + stage * STAGE, a.k, b, kv, i * STREAM, a.n, a.width,
								 mask.doc && mask.ranges[i * STREAM / DOC_TILE].others ? mask.doc : nullptr, vec & 2, tid);
	};
	own_off = __syncthreads_or(own_off != 0);
	int it = next(0), stage = 0;
	if (it < end)
		fetch(it, 0);
	cp_async_commit();
	while (it < end) {
		const int following = next(it + 1), r0 = it * STREAM;
		// what the keys' kernel has gone over: blocks of 32 queries and 64 keys that may see each other
		const int t32 = (o0 + 16 * warp) / 32 * 32, s64 = r0 / 64 * 64;
		const bool there = t32 < a.n && mask.any(t32, min(a.n, t32 + 32), s64, min(a.n, s64 + 64));
		const float *const from = parts.e + unit_bh * parts.unit_floats + (long long)oa * parts.pitch + r0 + 2 * j;
		float2 e_all[2][4]; // [step][streamed 0-7, 8-15][own row g, g + 8]
#pragma unroll
		for (int i = 0; i < 8; i++)
			e_all[i / 4][i % 4] = there ? *reinterpret_cast<const float2 *>(from + (i % 2) * 8 * (long long)parts.pitch + 16 * (i / 4) + 8 * (i / 2 % 2)) : make_float2(0.f, 0.f);
		cp_async_wait<0>();
		__syncthreads(); // the tile is there; everyone is done with the other stage, and with the codes
		if (following < end)
			fetch(following, stage ^ 1);
		cp_async_commit();
		uint32_t off = own_off;
		if (CODES)
			encode_tile<W, KP>(smem + CODED, smem + STAGES + stage * STAGE, &off, tid);
		off = CODES ? __syncthreads_or(off != 0) : 0;
		if (there)
#pragma unroll
			for (int kb = 0; kb < STREAM / 16; kb++) {
				float e[2][4];
				bool grew = false;
#pragma unroll
				for (int i = 0; i < 4; i++) {
					e[i / 2][2 * (i % 2)] = e_all[kb][i].x;
					e[i / 2][2 * (i % 2) + 1] = e_all[kb][i].y;
					grew |= fabsf(e_all[kb][i].x) > limit[i % 2] || fabsf(e_all[kb][i].y) > limit[i % 2];
				}
				if (__any_sync(0xffffffffu, grew))
					follow_largest<W>(e, unit, limit, e_sum, acc, j);
				uint32_t eb[2][2], el[2][2] = {};
#pragma unroll
				for (int i = 0; i < 4; i++) {
					const float e0 = e[i % 2][i / 2 * 2] * unit[i / 2], e1 = e[i % 2][i / 2 * 2 + 1] * unit[i / 2];
					eb[i / 2][i % 2] = Half2<__half>::pack(e0, e1);
					if (TWICE) {
						const float2 f = Half2<__half>::unpack(eb[i / 2][i % 2]);
						el[i / 2][i % 2] = Half2<__half>::pack(e0 - f.x, e1 - f.y);
					}
				}
				const bool coded = CODES && !off;
				if (coded)
					Half2<__half>::mma(e_sum, eb[0][0], eb[1][0], eb[0][1], eb[1][1], Half2<__half>::ONES, Half2<__half>::ONES);
				add_signed<T, W, TWICE>(acc, eb, el, coded, coded ? base + CODED : base + STAGES + stage * STAGE, 16 * kb, smem, reinterpret_cast<const uint16_t *>(smem + OWN_X), warp, lane);
			}
		it = following;
		stage ^= 1;
	}
	const unsigned again = __reduce_or_sync(0xffffffffu, store_signed<T, W>(acc, unit, e_sum, a, b, head, o0 + 16 * warp, lane, nullptr, dq));
	for (int r = 0; r < 16; r++)
		if (again >> r & 1u && o0 + 16 * warp + r < a.n)
			exact_gradient_row<T, false>(a, mask, b, head, o0 + 16 * warp + r, dvo, lse, delta, dq, dq);
}

template <typename T, int W, int V>
int bwd(const MaskedArgs &a, const void *dvo_, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, float *e, int vec, cudaStream_t st)
{
	constexpr int KP = W == 3 ? 16 : 4 * W, VP = 2 * V;
	constexpr bool CODES = Half2<T>::ONES == Half2<__nv_bfloat16>::ONES;
	constexpr int bytes = ROWS * 128 * W + ROWS * VP * 16 + 2 * STREAM * (KP + VP) * 16 + ROWS * 64 * W + (CODES ? STREAM * KP * 16 : 0);
	constexpr int dq_bytes = ROWS * 128 * W + 2 * STREAM * KP * 16 + (CODES ? ROWS * 64 * W + STREAM * KP * 16 : 0);
	static_assert(2 * STREAM * KP >= ROWS * 4 * W, "own rows pass through the stages");
	const T *dvo = static_cast<const T *>(dvo_);
	const int tiles = (a.n + ROWS - 1) / ROWS, group = a.heads / a.kv_heads;
	const long long all = (long long)a.bs * a.heads;
	if (all * tiles > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	BackwardParts parts = {0, int(all), e, masked_unit_floats(a.n), int((a.n + 63ll) / 64 * 64), nullptr, nullptr};
	if (group > 1) {
		parts.dk = shares;
		parts.dv = shares + (long long)a.bs * a.n * a.heads * a.width;
	}
	const long long step = e ? masked_units_at_once(a.bs, a.n, a.heads) : all;
	for (long long first = 0; first < all; first += step) {
		parts.first = int(first);
		parts.units = int(all - first < step ? all - first : step);
		const unsigned grid = unsigned(parts.units) * unsigned(tiles);
		L1B_SHARED_MEMORY((masked_bwd_mma_kernel<T, true, W, V>), bytes);
		masked_bwd_mma_kernel<T, true, W, V><<<grid, THREADS, bytes, st>>>(a, dvo, lse, delta, static_cast<T *>(dk), static_cast<T *>(dv), parts, tiles, vec);
		L1B_LAUNCH_CHECK();
		if (e) {
			L1B_SHARED_MEMORY((masked_dq_mma_kernel<T, W>), dq_bytes);
			masked_dq_mma_kernel<T, W><<<grid, THREADS, dq_bytes, st>>>(a, dvo, lse, delta, static_cast<T *>(dq), parts, tiles, vec);
		} else {
			L1B_SHARED_MEMORY((masked_bwd_mma_kernel<T, false, W, V>), bytes);
			masked_bwd_mma_kernel<T, false, W, V><<<grid, THREADS, bytes, st>>>(a, dvo, lse, delta, static_cast<T *>(dq), nullptr, parts, tiles, vec);
		}
		L1B_LAUNCH_CHECK();
	}
	return L1ATTN_OK;
}

template <typename T, int W, int V> int fwd(const MaskedArgs &a, void *vo, void *rest, float *lse, int vec, cudaStream_t st)
{
	constexpr int bytes = 2 * KEYS * (4 * W + 2 * V) * 16;
	static_assert(bytes >= ROWS * 4 * W * 16 && MB * 16 <= 32, "the query rows pass through the stages");
	const int tiles = (a.n + ROWS - 1) / ROWS;
	const long long grid = (long long)tiles * a.heads * a.bs;
	if (grid > 0x7fffffffll)
		return L1ATTN_ERR_SHAPE;
	L1B_SHARED_MEMORY((masked_fwd_mma_kernel<T, W, V>), bytes);
	masked_fwd_mma_kernel<T, W, V><<<unsigned(grid), THREADS, bytes, st>>>(a, static_cast<T *>(vo), static_cast<T *>(rest), lse, tiles, vec);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

// rows of 16-byte vectors: what asynchronous copies need
bool vectors(const Strided &x) { return aligned(x.p, 16) && x.batch % 8 == 0 && x.tok % 8 == 0 && x.head % 8 == 0; }

template <typename T> int fwd_type(const MaskedArgs &a, void *vo, void *rest, float *lse, cudaStream_t st)
{
	const int vec = vectors(a.q) | vectors(a.k) << 1 | vectors(a.v) << 2 | (aligned(vo, 4) && a.v_width % 2 == 0) << 3, w = (a.width + 31) / 32;
	if (a.v_width <= 64)
		return w == 1 ? fwd<T, 1, 4>(a, vo, rest, lse, vec, st) : w == 2 ? fwd<T, 2, 4>(a, vo, rest, lse, vec, st) : w == 3 ? fwd<T, 3, 4>(a, vo, rest, lse, vec, st) : fwd<T, 4, 4>(a, vo, rest, lse, vec, st);
	return w == 1 ? fwd<T, 1, 8>(a, vo, rest, lse, vec, st) : w == 2 ? fwd<T, 2, 8>(a, vo, rest, lse, vec, st) : w == 3 ? fwd<T, 3, 8>(a, vo, rest, lse, vec, st) : fwd<T, 4, 8>(a, vo, rest, lse, vec, st);
}

template <typename T>
int bwd_type(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, float *e, cudaStream_t st)
{
	const int vec = vectors(a.q) | vectors(a.k) << 1 | vectors(a.v) << 2 | (aligned(dvo, 16) && a.v_width % 8 == 0) << 3, w = (a.width + 31) / 32;
	if (a.v_width <= 64)
		return w == 1 ? bwd<T, 1, 4>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st) : w == 2 ? bwd<T, 2, 4>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st) :
		       w == 3 ? bwd<T, 3, 4>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st) : bwd<T, 4, 4>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st);
	return w == 1 ? bwd<T, 1, 8>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st) : w == 2 ? bwd<T, 2, 8>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st) :
	       w == 3 ? bwd<T, 3, 8>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st) : bwd<T, 4, 8>(a, dvo, lse, delta, dq, dk, dv, shares, e, vec, st);
}

} // namespace

bool masked_mma_fits(int width, int v_width, int dtype) { return dtype != L1ATTN_F32 && width <= 128 && v_width <= 128; }

int masked_mma_fwd_launch(const MaskedArgs &a, void *vo, void *rest, float *lse, int dtype, cudaStream_t st)
{
	return dtype == L1ATTN_F16 ? fwd_type<__half>(a, vo, rest, lse, st) : fwd_type<__nv_bfloat16>(a, vo, rest, lse, st);
}


// Floats that hold a unit's e (rows and columns to whole tiles), and units whose e are alive at once: up to a gigabyte of them; none when one unit is
// larger (more than 16384 tokens): the queries' kernel then forms the weights again.
long long masked_unit_floats(int n)
{
	const long long side = (n + 63ll) / 64 * 64;
	return side * side;
}
long long masked_units_at_once(int bs, int n, int heads)
{
	const long long all = (long long)bs * heads, fit = (1ll << 28) / masked_unit_floats(n);
	return fit < all ? fit : all;
}

int masked_mma_bwd_launch(const MaskedArgs &a, const void *dvo, const float *lse, const float *delta, void *dq, void *dk, void *dv, float *shares, float *e, int dtype,
			  cudaStream_t st)
{
	return dtype == L1ATTN_F16 ? bwd_type<__half>(a, dvo, lse, delta, dq, dk, dv, shares, e, st) : bwd_type<__nv_bfloat16>(a, dvo, lse, delta, dq, dk, dv, shares, e, st);
}

} // namespace l1b
