// Attention of new tokens of 16 bits to a paged cache in 8 bits (cache.cuh), widths up to 128: distances and products on the tensor cores.
//
// For a page of scale s:  sum |q - s c| = s (sum q' + sum c - 2 sum min(q', c)) + sum |q - s q'|,  q' = q / s as float16, clipped to +-128.
// Codes are exact as float16, so is the minimum; q' carries 11 bits, at worst 1/32 of a code's step (and what is clipped off is added in float32).
// The minima go through mma.m16n8k16 as in mma.cuh with the sides swapped: A's rows are 16 keys, unpacked once into registers, and the
// query rows -- (token, head of the group) pairs that all read these keys -- are streamed from shared memory, one column each.  Nothing is wasted on
// few query rows.  A second product with B = -1/2 takes off half the sum of the codes, one per page gives the sum of q'.  Weights go to float16 (11 bits;
// for float16 outputs what that leaves, in a second product) times the page's value scale, by movmatrix into the columns of the value product, whose A's rows are 16 channels, unpacked from the codes.
//
// A warp streams chunks of 16 or 32 keys on its own (asynchronous copies into its own stages, no barrier in the loop); the four warps of a CTA
// take runs of its chunks and join at the end.  The chunks of all units -- a tile of query rows and a head of keys and values -- lie behind one
// another, and every CTA of one wave takes an equal share, whatever the lengths (known on the device alone): a unit may end in a later CTA's share, and
// is joined by join_splits_kernel.
// Bound: instruction issue, 55 % of the slots with 12 warps an SM (168 registers); what every chunk costs (copies, unpacking, weights) is half of it, a query
// row a tenth or so.  Widths of 128: 37 sequences of 16384 tokens, one query head 266 us (72 % of the rate of a copy), four 415 (46 %); 64 ragged
// ones of up to 8192, one 138 us, four 203, eight 297.
#include "cache.cuh"
#include "mma.cuh"

namespace l1b {

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr float LOG2E = 1.4426950408889634f, LAG = 8.f;
// Chunks that a unit costs beside its own (query rows, lookups, the join).  5 / 8 / 11 / 15, ragged sequences, four query heads a group: 64 of up to 8192 tokens
// 222 / 207 / 203 / 206 us, 256 of 2048 256 / 249 / 231 / 238, 1024 of 500 411 / 401 / 395 / 393; pieces of 256 tokens on 3001, which share units less, 217 / 219 / 223 / 226.
constexpr int ENTRY = 11;
using H = Half2<__half>;

__device__ __forceinline__ uint32_t permute(uint32_t a, uint32_t b, uint32_t how)
{
	uint32_t d;
	asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(how));
	return d;
}
// two bytes (code ^ 0x80) at places `how` as codes in float16: 0x6400 | u is 1024 + u
__device__ __forceinline__ uint32_t half_codes(uint32_t u, uint32_t how) { return H::sub(permute(u, 0x64646464u, how), 0x64806480u); }
constexpr uint32_t LOW = 0x4140, HIGH = 0x4342;

__device__ __forceinline__ float warp_max(float x)
{
#pragma unroll
	for (int s = 16; s; s >>= 1)
		x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
	return x;
}

template <typename T> __device__ __forceinline__ T half_of(uint32_t x, int which)
{
	const uint16_t bits = uint16_t(x >> 16 * which);
	return *reinterpret_cast<const T *>(&bits);
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
	uint32_t y;
	asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
	return y;
}

// Rows of codes in a stage.  Keys: 16-byte pieces, of odd rows four places off where rows are 128 bytes.  Values: 32-byte groups (eight words, one a lane g)
// so that the rows 2 j of the four j lie in different banks.
template <int WG> __device__ __forceinline__ uint32_t key_place(int row, int piece) { return row * 64 * WG + (WG == 2 ? piece ^ (row & 1) * 4 : piece) * 16; }
template <int VG> __device__ __forceinline__ uint32_t value_place(int row, int group)
{
	return VG == 4 ? row * 128 + (group ^ (row / 2 & 3)) * 32 : row / 2 * 128 + (((row & 1) * 2 + group) ^ (row / 2 & 3)) * 32;
}

// WG: 64-column groups of the width (1, 2); VG: 32-channel groups of the values (2, 4); TILES: of eight query rows; NG: groups of 16 keys a chunk (1 where pages
// are of 16 tokens, so that a chunk has one scale)
template <typename T, int WG, int VG, int TILES, int NG> struct Layout {
	static constexpr int CHUNK = 16 * NG, KEY_BYTES = CHUNK * 64 * WG, STAGE = CHUNK * (64 * WG + 32 * VG), STAGES = 2;
	static constexpr int Q_TABLE = 8 * TILES * 64 * WG * 2, WARP = Q_TABLE + STAGES * STAGE + 64 * TILES; // q' | stages | clipped rests, lowest unit
	static constexpr int Q_ROWS = 8 * TILES * 64 * WG * 2, JOIN = WARPS * 8 * TILES * (32 * VG + 2) * 4;
	static constexpr int BYTES = Q_ROWS + (WARPS * WARP > JOIN ? WARPS * WARP : JOIN);
};

struct Weight { // of a sequence: tiles of rows, chunks of each (from chunk `first` on), chunks in all
	int tiles, first, chunks;
	long long all;
};

template <typename T, int WG, int VG, int TILES, int NG> __global__ void __launch_bounds__(THREADS, TILES == 1 ? 3 : 2) attend_mma_kernel(AttendArgs a, int vec)
{
	extern __shared__ uint4 smem16[];
	using L = Layout<T, WG, VG, TILES, NG>;
	constexpr int CHUNK = L::CHUNK, ROWS = 8 * TILES, W = 64 * WG;
	constexpr bool TWICE = H::ONES == Half2<T>::ONES; // float16 outputs are finer than weights of 11 bits: the rest of a weight takes a product of its own
	const CacheArgs &c = a.c;
	unsigned char *const smem = reinterpret_cast<unsigned char *>(smem16);
	const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, j = lane % 4;

	// all sequences' chunks, and this CTA's share of them
	auto weigh = [&](int i, SeqView *view) {
		Weight w = {0, 0, 0, 0};
		if (i >= c.n_seqs)
			return w;
		*view = cache_seq(c, i);
		w.tiles = (view->count * a.group + a.tile_rows - 1) / a.tile_rows; // (the caller has seen that rows * group fits)
		w.first = a.window ? max(0, view->start - a.window + 1) / CHUNK : 0;
		w.chunks = (view->start + view->count + CHUNK - 1) / CHUNK - w.first;
		w.all = (long long)w.tiles * (w.chunks + ENTRY) * c.kv_heads;
		return w;
	};
	SeqView sv;
	long long total = 0;
	for (int i = lane; i < (c.n_seqs + 31) / 32 * 32; i += 32)
		total += weigh(i, &sv).all;
#pragma unroll
	for (int d = 16; d; d >>= 1)
		total += __shfl_xor_sync(0xffffffffu, total, d);
	const long long share = max((total + a.ctas - 1) / a.ctas, (long long)a.least), to = min(total, (blockIdx.x + 1) * share);
	long long at = blockIdx.x * share, before = 0; // before: chunks of the sequences before seq
	if (a.splits_of && tid == 0)
		a.splits_of[blockIdx.x].kv = -1;
	for (int i = blockIdx.x; i < c.n_seqs; i += gridDim.x) { // queries without a place: zeros, a sequence a CTA
		const SeqView v = cache_seq(c, i);
		const long long size = (long long)a.heads * c.v_width, begin = (v.row + v.count) * size, end = begin + v.lost * size;
		for (long long w = begin + tid; w < end; w += THREADS)
			static_cast<T *>(a.vo)[w] = from_float<T>(0.f);
	}
	if (at >= to)
		return;
	int seq = 0;
	for (int i = lane; i - lane < c.n_seqs; i += 32) { // 32 sequences at a time
		const long long all = weigh(i, &sv).all;
		long long sum = all;
#pragma unroll
		for (int d = 1; d < 32; d <<= 1) {
			const long long x = __shfl_up_sync(0xffffffffu, sum, d);
			sum += lane >= d ? x : 0;
		}
		const unsigned here = __ballot_sync(0xffffffffu, before + sum > at);
		if (here) {
			const int l = __ffs(here) - 1;
			before += __shfl_sync(0xffffffffu, sum - all, l);
			seq = i - lane + l;
			break;
		}
		before += __shfl_sync(0xffffffffu, sum, 31);
	}
	while (at < to) { // unit by unit
		Weight weight = weigh(seq, &sv);
		while (at - before >= weight.all) { // (some may have nothing)
			before += weight.all;
			if (++seq >= c.n_seqs)
				return;
			weight = weigh(seq, &sv);
		}
		const unsigned place = unsigned(weight.chunks + ENTRY), unit = unsigned((at - before) / place), skip = unsigned((at - before) % place);
		const unsigned take = unsigned(min((long long)(place - skip), to - at));
		const int from = max(int(skip) - ENTRY, 0), upto = max(int(skip + take) - ENTRY, 0), kv = unit / weight.tiles; // chunks of the unit
		const int first = int(unit % weight.tiles) * a.tile_rows, rows = min(a.tile_rows, sv.count * a.group - first);
		const unsigned group = a.group;
		const int t_lo = sv.start + int(unsigned(first) / group), t_hi = sv.start + int(unsigned(first + rows - 1) / group);
		const int lo = max((weight.first + from) * CHUNK, a.window ? max(0, t_lo - a.window + 1) : 0), hi = int(min((long long)t_hi + 1, (long long)(weight.first + upto) * CHUNK));
		const bool begins = skip == 0, ends = skip + take == place;
		__syncthreads(); // (shared memory is free)

		// the query rows, zeros past the width and past the last row
		T *const q_rows = reinterpret_cast<T *>(smem);
		for (int i = tid; i < ROWS * W; i += THREADS) {
			const int r = i / W, w = i % W;
			const unsigned lr = first + r;
			q_rows[i] = r < rows && w < c.width ? static_cast<const T *>(a.q)[(long long)(sv.row + lr / group) * a.q_row + (kv * a.group + lr % group) * a.q_head + w] : from_float<T>(0.f);
		}
		unsigned char *const mine = smem + L::Q_ROWS + warp * L::WARP;
		__half2 *const q_table = reinterpret_cast<__half2 *>(mine);
		float *const rest = reinterpret_cast<float *>(mine + L::Q_TABLE + L::STAGES * L::STAGE);
		const uint32_t stages = shared_address(mine) + L::Q_TABLE;
		if (lane < 16 * TILES)
			rest[lane % (16 * TILES)] = 0.f;
		for (int i = lane; i < ROWS * W / 2; i += 32)
			q_table[i] = __floats2half2_rn(0.f, 0.f); // (rows past the last stay zeros)
		__syncthreads();

		// this lane's columns: query rows 8 tile + 2 j, + 1
		int t_of[TILES][2];
		float slope[TILES][2], m[TILES][2], ref[TILES][2], l[TILES][2], o[TILES][2 * VG][4];
#pragma unroll
		for (int i = 0; i < 2 * TILES; i++) {
			const unsigned lr = first + 8 * (i / 2) + 2 * j + (i & 1);
			t_of[i / 2][i & 1] = 8 * (i / 2) + 2 * j + (i & 1) < rows ? sv.start + int(lr / group) : t_hi; // (columns past the last row: whatever they come to is not written)
			slope[i / 2][i & 1] = a.slopes ? a.slopes[kv * a.group + lr % group] : 0.f;
			m[i / 2][i & 1] = -INFINITY;
			ref[i / 2][i & 1] = l[i / 2][i & 1] = 0.f;
		}
#pragma unroll
		for (int i = 0; i < TILES * 2 * VG * 4; i++)
			o[i / (8 * VG)][i / 4 % (2 * VG)][i % 4] = 0.f;
		float q_max = 0.f; // the largest |q| of the rows, infinite with a NaN: whether anything is clipped
		for (int i = lane; i < ROWS * W; i += 32) {
			const float x = fabsf(to_float(q_rows[i]));
			q_max = fmaxf(q_max, x == x ? x : INFINITY);
		}
		q_max = warp_max(q_max);

		// The range's chunks are dealt out to the warps in runs (a run has each page's q' formed once); this warp's number k begins at position
		// (chunk0 + k) CHUNK.  Pages are looked up for 32 chunks at a time, one a lane, two such sets.
		const int in_range = hi > lo ? (hi + CHUNK - 1) / CHUNK - lo / CHUNK : 0;
		const int chunk0 = lo / CHUNK + in_range * warp / WARPS, chunks = lo / CHUNK + in_range * (warp + 1) / WARPS - chunk0;
		int page_id[2] = {-1, -1};
		float page_k[2] = {0.f, 0.f}, page_v[2] = {0.f, 0.f};
		auto look_up = [&](int block) {
			const int k = block * 32 + lane, pos = (chunk0 + k) * CHUNK;
			int id = -1;
			float ks = 0.f, vs = 0.f;
			if (k < chunks) {
				id = cache_page(c, seq, pos / c.page);
				if (id >= 0) {
					ks = c.k_scale[(long long)id * c.kv_heads + kv];
					vs = c.v_scale[(long long)id * c.kv_heads + kv];
				}
			}
			const bool odd = block & 1; // (no index: the sets stay in registers)
			page_id[0] = odd ? page_id[0] : id, page_id[1] = odd ? id : page_id[1];
			page_k[0] = odd ? page_k[0] : ks, page_k[1] = odd ? ks : page_k[1];
			page_v[0] = odd ? page_v[0] : vs, page_v[1] = odd ? vs : page_v[1];
		};
		// this lane's pieces of a chunk: rows lane / pieces + i K_ROWS; where they go differs by whole rows, for values also in the bit that i's parity flips
		constexpr int K_ROWS = 8 / WG, V_ROWS = 16 / VG;
		const int k_row = lane / (4 * WG), k_piece = lane % (4 * WG), v_row = lane / (2 * VG), v_piece = lane % (2 * VG);
		const int k_bytes = min(max(c.width - 16 * k_piece, 0), 16), v_bytes = min(max(c.v_width - 16 * v_piece, 0), 16);
		const int k_from = k_row * c.width + 16 * k_piece, v_from = v_row * c.v_width + 16 * v_piece;
		const uint32_t k_at = key_place<WG>(k_row, k_piece);
		const uint32_t v_at[2] = {L::KEY_BYTES + value_place<VG>(v_row, v_piece / 2) + v_piece % 2 * 16,
					  L::KEY_BYTES + value_place<VG>(v_row + V_ROWS, v_piece / 2) + v_piece % 2 * 16 - V_ROWS * 32 * VG};
		auto of_chunk = [&](auto &set, int k) { return __shfl_sync(0xffffffffu, k & 32 ? set[1] : set[0], k & 31); };
		auto fetch = [&](int k) {
			if (k < chunks) {
				const int pos = (chunk0 + k) * CHUNK, id = of_chunk(page_id, k);
				const uint32_t at = stages + k % L::STAGES * L::STAGE;
				const long long row = ((long long)max(id, 0) * c.kv_heads + kv) * c.page + pos % c.page;
				const int8_t *from_k = c.k_codes + row * c.width, *from_v = c.v_codes + row * c.v_width;
				if (vec) { // a lane copies one column of pieces
					const int kb = id < 0 ? 0 : k_bytes, vb = id < 0 ? 0 : v_bytes;
					from_k += kb ? k_from : 0;
					from_v += vb ? v_from : 0;
					const int k_step = kb ? K_ROWS * c.width : 0, v_step = vb ? V_ROWS * c.v_width : 0;
#pragma unroll
					for (int i = 0; i < CHUNK / K_ROWS; i++, from_k += k_step)
						copy_async16(at + k_at + i * K_ROWS * 64 * WG, from_k, kb);
#pragma unroll
					for (int i = 0; i < CHUNK / V_ROWS; i++, from_v += v_step)
						copy_async16(at + v_at[i & 1] + i * V_ROWS * 32 * VG, from_v, vb);
				} else { // rows that are no 16-byte vectors
					unsigned char *const to = mine + L::Q_TABLE + k % L::STAGES * L::STAGE;
					for (int i = lane; i < CHUNK * W; i += 32) {
						const int r = i / W, w = i % W;
						to[key_place<WG>(r, w / 16) + w % 16] = id >= 0 && w < c.width ? from_k[r * c.width + w] : 0;
					}
					for (int i = lane; i < CHUNK * 32 * VG; i += 32) {
						const int r = i / (32 * VG), w = i % (32 * VG);
						to[L::KEY_BYTES + value_place<VG>(r, w / 32) + w % 32] = id >= 0 && w < c.v_width ? from_v[r * c.v_width + w] : 0;
					}
				}
			}
			cp_async_commit();
		};
		look_up(0);
		look_up(1);
#pragma unroll
		for (int k = 0; k < L::STAGES - 1; k++)
			fetch(k);

		int page_before = -2;
		// k_unit: 2 scale s (log2 e); q_part: of the score.  v_unit: power of two that the page's value scale is taken relative to: 2^4 to 2^7 times it, so that weights far
		// below the largest keep bits (at most 2^15 then).  It follows smaller scales too, since any page may hold a row's weight, but never more than 2^58 times above
		// its lowest: 2^30 keys of 2^22, codes and all, then stay within 2^110.
		int *const lowest = reinterpret_cast<int *>(rest + ROWS);
		float k_unit = 0.f, v_unit = 0.f, q_part[TILES][2];
		for (int k = 0; k < chunks; k++) {
			if (k && k % 32 == 0)
				look_up(k / 32 + 1);
			__syncwarp(); // (everyone is done with the stage that is filled next)
			fetch(k + L::STAGES - 1);
			const int id = of_chunk(page_id, k), s0 = (chunk0 + k) * CHUNK;
			const float ks = of_chunk(page_k, k), vs = of_chunk(page_v, k);
			if (id != page_before) { // q' of this page
				page_before = id;
				// (below 1e-37 every code stands for nothing beside any q)
				const bool none = !(ks >= 1e-37f);
				const float inv = none ? 0.f : 1.f / ks, s = none ? 0.f : ks;
				const bool clips = none || !(q_max * inv <= 128.f);
				if (!clips) {
					for (int i = lane; i < rows * (W / 4); i += 32) {
						const uint2 x = reinterpret_cast<const uint2 *>(q_rows)[i];
						uint2 y;
						y.x = H::pack(to_float(half_of<T>(x.x, 0)) * inv, to_float(half_of<T>(x.x, 1)) * inv);
						y.y = H::pack(to_float(half_of<T>(x.y, 0)) * inv, to_float(half_of<T>(x.y, 1)) * inv);
						reinterpret_cast<uint2 *>(q_table)[i] = y;
					}
				} else {
					for (int r = 0; r < rows; r++) {
						float off = 0.f;
						for (int i = lane; i < W / 2; i += 32) {
							float x[2], y[2];
#pragma unroll
							for (int e = 0; e < 2; e++) {
								x[e] = to_float(q_rows[r * W + 2 * i + e]);
								y[e] = fminf(fmaxf(x[e] * inv, -128.f), 128.f);
								off += fabsf(x[e] * inv) <= 128.f && !none ? 0.f : fabsf(x[e] - s * y[e]);
							}
							q_table[r * (W / 2) + i] = __floats2half2_rn(y[0], y[1]);
						}
#pragma unroll
						for (int d = 16; d; d >>= 1)
							off += __shfl_xor_sync(0xffffffffu, off, d);
						if (lane == 0)
							rest[r] = off;
					}
				}
				__syncwarp();
				const bool straight = a.cap == 0.f && !a.slopes; // to the exponent without a stop
				k_unit = 2.f * a.scale * s * (straight ? LOG2E : 1.f);
#pragma unroll
				for (int i = 0; i < TILES; i++) {
					float sum[4] = {0.f, 0.f, 0.f, 0.f}; // sums of q' of the rows, by columns
#pragma unroll
					for (int u = 0; u < 2 * WG; u++) {
						const uint4 x = *reinterpret_cast<const uint4 *>(mine + ((8 * i + g) * W + 16 * WG * j + 8 * u) * 2);
						H::mma(sum, H::ONES, H::ONES, H::ONES, H::ONES, x.x, x.y);
						H::mma(sum, H::ONES, H::ONES, H::ONES, H::ONES, x.z, x.w);
					}
#pragma unroll
					for (int b = 0; b < 2; b++)
						q_part[i][b] = -0.5f * k_unit * sum[b] - a.scale * (straight ? LOG2E : 1.f) * (clips ? rest[8 * i + 2 * j + b] : 0.f);
				}
				if (__float_as_uint(vs * v_unit) - 0x41800000u > 0x01800000u && vs > 0.f) { // not from 16 to 128; what has been added up follows
					const int was = __float_as_uint(v_unit) >> 23; // exponents; 0: no scale yet
					int to = 260 - min(max(int(__float_as_uint(vs) >> 23), 7), 253), low = to;
					if (was) {
						low = *lowest;
						to = min(to, low + 58);
						low = min(low, to);
					}
					__syncwarp();
					*lowest = low;
					v_unit = __uint_as_float(uint32_t(to) << 23);
					const float keep = !was ? 1.f : to - was < -126 ? 0.f : __uint_as_float(uint32_t(127 + to - was) << 23);
#pragma unroll
					for (int i = 0; i < TILES * 2 * VG * 4; i++)
						o[i / (8 * VG)][i / 4 % (2 * VG)][i % 4] *= keep;
				}
			}
			const float v_rel = vs * v_unit;
			cp_async_wait<L::STAGES - 1>();
			__syncwarp(); // the chunk is there, all lanes' copies of it
			const unsigned char *const stage = mine + L::Q_TABLE + k % L::STAGES * L::STAGE;

			// keys as codes in float16: A's rows are keys g, g + 8 of a group
			uint32_t kf[NG][4 * WG][4];
			float x[NG][TILES][4];
#pragma unroll
			for (int n = 0; n < NG; n++) {
#pragma unroll
				for (int i = 0; i < WG; i++) {
					const uint4 y = *reinterpret_cast<const uint4 *>(stage + key_place<WG>(16 * n + g, j + 4 * i)), z = *reinterpret_cast<const uint4 *>(stage + key_place<WG>(16 * n + g + 8, j + 4 * i));
					const uint32_t yw[4] = {y.x, y.y, y.z, y.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
					for (int w = 0; w < 4; w++) {
						const uint32_t yu = yw[w] ^ 0x80808080u, zu = zw[w] ^ 0x80808080u;
						kf[n][4 * i + w][0] = half_codes(yu, LOW);
						kf[n][4 * i + w][1] = half_codes(zu, LOW);
						kf[n][4 * i + w][2] = half_codes(yu, HIGH);
						kf[n][4 * i + w][3] = half_codes(zu, HIGH);
					}
				}
				float half_sum[4] = {0.f, 0.f, 0.f, 0.f}; // minus half the sums of the codes
#pragma unroll
				for (int w = 0; w < 4 * WG; w++)
					H::mma(half_sum, kf[n][w][0], kf[n][w][1], kf[n][w][2], kf[n][w][3], 0xb800b800u, 0xb800b800u);
#pragma unroll
				for (int i = 0; i < TILES * 4; i++)
					x[n][i / 4][i % 4] = half_sum[i % 4];
			}
#pragma unroll
			for (int i = 0; i < TILES; i++)
#pragma unroll 1
				for (int r = 0; r < min(rows - 8 * i, 8); r++) {
					const uint32_t one = g == r ? H::ONES : 0u;
					const unsigned char *const from = mine + (8 * i + r) * W * 2 + 32 * j;
#pragma unroll
					for (int p = 0; p < WG; p++) {
						const uint4 y = *reinterpret_cast<const uint4 *>(from + 128 * p), z = *reinterpret_cast<const uint4 *>(from + 128 * p + 16);
						const uint32_t q[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
						for (int w = 0; w < 4; w++)
#pragma unroll
							for (int n = 0; n < NG; n++) {
								const uint32_t(&f)[4] = kf[n][4 * p + w];
								H::mma(x[n][i], H::min(f[0], q[2 * w]), H::min(f[1], q[2 * w]), H::min(f[2], q[2 * w + 1]), H::min(f[3], q[2 * w + 1]), one, one);
							}
					}
				}

			// scores times log2 e; this lane's keys are s0 + 16 n + g, + 8
			const bool whole = id >= 0 && s0 >= lo && s0 + CHUNK <= hi && s0 + CHUNK - 1 <= t_lo && (a.window == 0 || t_hi - s0 < a.window);
			bool grew = false;
#pragma unroll
			for (int n = 0; n < NG; n++)
#pragma unroll
				for (int i = 0; i < TILES; i++)
#pragma unroll
					for (int e = 0; e < 4; e++)
						x[n][i][e] = fmaf(k_unit, x[n][i][e], q_part[i][e & 1]);
			if (!whole || a.cap > 0.f || a.slopes) {
				if (a.cap > 0.f)
					cap_scores<NG * TILES * 4, false>(&x[0][0][0], nullptr, a.cap);
#pragma unroll
				for (int n = 0; n < NG; n++)
#pragma unroll
					for (int i = 0; i < TILES; i++)
#pragma unroll
						for (int e = 0; e < 4; e++) {
							const int s = s0 + 16 * n + g + 8 * (e / 2), t = t_of[i][e & 1];
							float y = x[n][i][e];
							if (a.cap > 0.f || a.slopes)
								y = (y - slope[i][e & 1] * float(t - s)) * LOG2E;
							if (id < 0 || s < lo || s >= hi || s > t || (a.window && t - s >= a.window))
								y = -INFINITY;
							x[n][i][e] = y;
						}
			}
#pragma unroll
			for (int i = 0; i < 2 * TILES; i++)
#pragma unroll
				for (int n = 0; n < NG; n++)
					grew |= fmaxf(x[n][i / 2][i & 1], x[n][i / 2][2 + (i & 1)]) > m[i / 2][i & 1] + LAG;
			// The reference of the exponentials need not be the maximum: it follows once a score is beyond it by more than LAG.
			if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
				for (int i = 0; i < TILES; i++)
#pragma unroll
					for (int b = 0; b < 2; b++) {
						float top = m[i][b];
#pragma unroll
						for (int n = 0; n < NG; n++)
							top = fmaxf(top, fmaxf(x[n][i][b], x[n][i][2 + b]));
#pragma unroll
						for (int d = 4; d < 32; d <<= 1)
							top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
						const float keep = top == -INFINITY ? 1.f : exp2_fast(m[i][b] - top);
						m[i][b] = top;
						ref[i][b] = top == -INFINITY ? 0.f : top;
						l[i][b] *= keep;
#pragma unroll
						for (int v = 0; v < 2 * VG; v++) {
							o[i][v][b] *= keep;
							o[i][v][2 + b] *= keep;
						}
					}
			}
			// weights, and their products with the values: A's rows are channels 32 i + 4 g + 2 h, + 1
#pragma unroll
			for (int n = 0; n < NG; n++) {
				uint32_t p[TILES][2], low[TILES][2];
#pragma unroll
				for (int i = 0; i < TILES; i++) {
					float e[4];
#pragma unroll
					for (int d = 0; d < 4; d++) {
						e[d] = exp2_fast(x[n][i][d] - ref[i][d & 1]);
						l[i][d & 1] += e[d];
						e[d] *= v_rel;
					}
#pragma unroll
					for (int d = 0; d < 2; d++) {
						const uint32_t high = H::pack(e[2 * d], e[2 * d + 1]);
						p[i][d] = transpose8x8(high);
						if (TWICE)
							low[i][d] = transpose8x8(H::pack(e[2 * d] - to_float(half_of<__half>(high, 0)), e[2 * d + 1] - to_float(half_of<__half>(high, 1))));
					}
				}
#pragma unroll
				for (int v = 0; v < VG; v++) {
					uint32_t w[4];
#pragma unroll
					for (int d = 0; d < 4; d++) // keys 2 j, 2 j + 1, the same + 8
						w[d] = *reinterpret_cast<const uint32_t *>(stage + L::KEY_BYTES + value_place<VG>(16 * n + 2 * j + (d & 1) + 8 * (d / 2), v) + 4 * g) ^ 0x80808080u;
					const uint32_t b01 = permute(w[0], w[1], 0x5140), b23 = permute(w[0], w[1], 0x7362), d01 = permute(w[2], w[3], 0x5140), d23 = permute(w[2], w[3], 0x7362);
					const uint32_t f[2][4] = {{half_codes(b01, LOW), half_codes(b01, HIGH), half_codes(d01, LOW), half_codes(d01, HIGH)},
								  {half_codes(b23, LOW), half_codes(b23, HIGH), half_codes(d23, LOW), half_codes(d23, HIGH)}};
#pragma unroll
					for (int i = 0; i < TILES; i++)
#pragma unroll
						for (int h = 0; h < 2; h++)
						{
							H::mma(o[i][2 * v + h], f[h][0], f[h][1], f[h][2], f[h][3], p[i][0], p[i][1]);
							if (TWICE)
								H::mma(o[i][2 * v + h], f[h][0], f[h][1], f[h][2], f[h][3], low[i][0], low[i][1]);
						}
				}
			}
		}

		// join the warps: [warp][row] {m, l, values}
		cp_async_wait<0>();
		__syncthreads();
		float *const join = reinterpret_cast<float *>(smem + L::Q_ROWS);
		constexpr int PITCH = 32 * VG + 2;
		const float back = v_unit == 0.f ? 0.f : 1.f / v_unit;
#pragma unroll
		for (int i = 0; i < TILES; i++)
#pragma unroll
			for (int b = 0; b < 2; b++) {
#pragma unroll
				for (int d = 4; d < 32; d <<= 1)
					l[i][b] += __shfl_xor_sync(0xffffffffu, l[i][b], d);
				float *const to = join + (warp * ROWS + 8 * i + 2 * j + b) * PITCH;
				if (g == 0) {
					to[0] = m[i][b] / LOG2E;
					to[1] = l[i][b];
				}
#pragma unroll
				for (int v = 0; v < 2 * VG; v++) {
					const int ch = v / 2 * 32 + 4 * g + v % 2 * 2;
					to[2 + ch] = o[i][v][b] * back;
					to[2 + ch + 1] = o[i][v][2 + b] * back;
				}
			}
		__syncthreads();
		for (int i = tid; i < rows * c.v_width; i += THREADS) {
			const int r = i / c.v_width, w = i % c.v_width;
			float top = -INFINITY, sum = 0.f, value = 0.f;
#pragma unroll
			for (int k = 0; k < WARPS; k++)
				top = fmaxf(top, join[(k * ROWS + r) * PITCH]);
			const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
			for (int k = 0; k < WARPS; k++) {
				const float *const part = join + (k * ROWS + r) * PITCH, e = expf(part[0] - base);
				sum = fmaf(part[1], e, sum);
				value = fmaf(part[2 + w], e, value);
			}
			if (begins && ends) {
				const unsigned lr = first + r;
				const float f = finish_softmax(a.mode, top, sum);
				static_cast<T *>(a.vo)[((long long)(sv.row + lr / group) * a.heads + kv * a.group + lr % group) * c.v_width + w] = from_float<T>(f == 0.f ? 0.f : value * f);
			} else {
				float *const out = a.part + ((2ll * blockIdx.x + begins) * a.tile_rows + r) * (c.v_width + 2);
				if (w == 0) {
					out[0] = top;
					out[1] = sum;
				}
				out[2 + w] = value;
			}
		}
		if (begins && !ends && tid == 0)
			a.splits_of[blockIdx.x] = {kv, rows, int((at + place - 1) / share), 0, sv.row * (long long)a.group + first};
		at += take;
	}
}

// Joins the parts of the units that end in a later CTA's share than they begin in: one block per (CTA they begin in, row of the tile)
template <typename T> __global__ void __launch_bounds__(128) join_splits_kernel(AttendArgs a)
{
	const AttendSplit s = a.splits_of[blockIdx.x];
	const int r = blockIdx.y, w = threadIdx.x, width = a.c.v_width;
	if (s.kv < 0 || r >= s.rows)
		return;
	const long long step = 2ll * a.tile_rows * (width + 2); // from a CTA's part to the next one's; the first is that of a unit's beginning
	const float *const begin = a.part + ((2ll * blockIdx.x + 1) * a.tile_rows + r) * (width + 2), *const rest = begin - a.tile_rows * (long long)(width + 2);
	const int more = s.last - int(blockIdx.x);
	float top = begin[0];
#pragma unroll 8
	for (int i = 1; i <= more; i++)
		top = fmaxf(top, rest[i * step]);
	const float base = top == -INFINITY ? 0.f : top, e0 = expf(begin[0] - base);
	float sum = begin[1] * e0, value = w < width ? begin[2 + w] * e0 : 0.f;
#pragma unroll 8
	for (int i = 1; i <= more; i++) {
		const float *const part = rest + i * step;
		const float e = expf(part[0] - base);
		sum = fmaf(part[1], e, sum);
		value = fmaf(w < width ? part[2 + w] : 0.f, e, value);
	}
	const long long pair = s.pair + r;
	const float f = finish_softmax(a.mode, top, sum);
	if (w < width)
		static_cast<T *>(a.vo)[(pair / a.group * a.heads + s.kv * a.group + pair % a.group) * width + w] = from_float<T>(f == 0.f ? 0.f : value * f);
}

template <typename T, int WG, int VG, int TILES, int NG> int launch(const AttendArgs &a, cudaStream_t st)
{
	using L = Layout<T, WG, VG, TILES, NG>;
	static_assert(L::BYTES <= (TILES == 1 ? 75 : 112) * 1024, "three or two CTAs share an SM");
	const int vec = a.c.width % 16 == 0 && a.c.v_width % 16 == 0;
	L1B_SHARED_MEMORY((attend_mma_kernel<T, WG, VG, TILES, NG>), L::BYTES);
	attend_mma_kernel<T, WG, VG, TILES, NG><<<a.ctas, THREADS, L::BYTES, st>>>(a, vec);
	L1B_LAUNCH_CHECK();
	join_splits_kernel<T><<<dim3(a.ctas, a.tile_rows), 128, 0, st>>>(a);
	L1B_LAUNCH_CHECK();
	return L1ATTN_OK;
}

template <typename T, int WG, int VG> int launch_rows(const AttendArgs &a, cudaStream_t st)
{
	if (a.c.page == 16)
		return a.tile_rows == 8 ? launch<T, WG, VG, 1, 1>(a, st) : launch<T, WG, VG, 2, 1>(a, st);
	return a.tile_rows == 8 ? launch<T, WG, VG, 1, 2>(a, st) : launch<T, WG, VG, 2, 2>(a, st);
}
template <typename T> int launch_type(const AttendArgs &a, cudaStream_t st)
{
	if (a.c.width <= 64)
		return a.c.v_width <= 64 ? launch_rows<T, 1, 2>(a, st) : launch_rows<T, 1, 4>(a, st);
	return a.c.v_width <= 64 ? launch_rows<T, 2, 2>(a, st) : launch_rows<T, 2, 4>(a, st);
}

} // namespace

// a wave: what the kernels' registers and shared memory let an SM hold
int attend_mma_ctas(int tile_rows, int sms) { return (tile_rows == 8 ? 3 : 2) * sms; }

bool attend_mma_fits(int width, int v_width, int dtype) { return dtype != L1ATTN_F32 && width <= 128 && v_width <= 128; }

int attend_mma_launch(const AttendArgs &a, int dtype, cudaStream_t st)
{
	return dtype == L1ATTN_F16 ? launch_type<__half>(a, st) : launch_type<__nv_bfloat16>(a, st);
}

} // namespace l1b
