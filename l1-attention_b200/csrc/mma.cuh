// Pieces of the kernels that sum L1 distances of 16-bit rows on the tensor cores.
//
//   sum_w |q_w - k_w| = sum_w q_w + sum_w k_w - 2 sum_w min(q_w, k_w)
//
// The minimum of two 16-bit values is exact, two at a time in one instruction; the sum over w is a product with ones: mma.m16n8k16, float32 accumulators.  What the three sums
// are off by goes with |q| + |k|, not with the distance: for a channel that q and k share at 1e3, 1e4, 1e5, 1e6 a score (128 wide) was off by 3e-5, 7e-4, 6e-3, 0.1 at most
// (next to a step of the channel itself of 4, 64, 512, 4096 in bfloat16).
// A's 16 rows are 16 (query, key) pairs; which of
// the eight columns gets their sums is chosen by B, ones in that column and zeros elsewhere, so that eight such products fill a 16 x 8
// tile of scores in the layout that the value product reads.  256 terms per mma, which issues every 8 clocks per scheduler: 128 terms per clock and
// SM at most, where float32 subtraction and addition of |.| reach 64.  Measured for the loop alone: 90 terms per clock and SM with 16 warps, 86 with 8.
//
// The order of w is free as long as both sides and all lanes agree per row: lane j of a quad holds the 16-byte pieces j, j + 4, j + 8, ... of a row,
// so that shared memory is read 16 bytes at a time and keys need no swizzle.
#pragma once
#include "mask.cuh"

namespace l1b {

template <typename T> struct Half2; // two 16-bit values in a register
template <> struct Half2<__half> {
	static constexpr uint32_t ONES = 0x3c003c00u;
	static __device__ __forceinline__ uint32_t min(uint32_t a, uint32_t b)
	{
		uint32_t d;
		asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
		return d;
	}
	static __device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
	static __device__ __forceinline__ uint32_t pack(float lo, float hi)
	{
		uint32_t d;
		asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
		return d;
	}
	static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b)
	{
		uint32_t d;
		asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
		return d;
	}
	// sign(a - b) of both halves as the smallest float16, 2^-24, with its sign, or zero: differences do not vanish, subnormal results included
	static __device__ __forceinline__ uint32_t sign(uint32_t a, uint32_t b)
	{
		uint32_t d;
		asm("min.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(sub(a, b)), "r"(0x00010001u));
		return d;
	}
	static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
	{
		asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
			     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
			     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
	}
};
template <> struct Half2<__nv_bfloat16> {
	static constexpr uint32_t ONES = 0x3f803f80u;
	static __device__ __forceinline__ uint32_t min(uint32_t a, uint32_t b)
	{
		uint32_t d;
		asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
		return d;
	}
	static __device__ __forceinline__ float2 unpack(uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }
	static __device__ __forceinline__ uint32_t pack(float lo, float hi)
	{
		uint32_t d;
		asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
		return d;
	}
	static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b)
	{
		uint32_t d;
		asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
		return d;
	}
	// (the smallest bfloat16's bits, read as a float16)
	static __device__ __forceinline__ uint32_t sign(uint32_t a, uint32_t b)
	{
		uint32_t d;
		asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(sub(a, b)), "r"(0x00010001u));
		return d;
	}
	static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
	{
		asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
			     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
			     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
	}
};

__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// (a plain load, which the compiler may move among the products)
__device__ __forceinline__ uint4 load_shared16(const void *base, uint32_t offset) { return *reinterpret_cast<const uint4 *>(static_cast<const unsigned char *>(base) + offset); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t a)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t a)
{
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
		     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
		     : "r"(a));
}
// bytes 0 .. 16 of a 16-byte copy; the rest is zeros
__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src, int bytes)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x)
{
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}
// x = cap tanh(x / cap) of N scores, which are not above 0 but for a rounding; slant, where given, is multiplied by the slope, 1 - tanh^2.
// (t - 1) / (t + 1) with t = e^2u, u = -|x / cap|, cancels where u is small: its error is absolute, 2^-23.  Times the cap that stays below 2^-17, a tenth of
// what sums of 128 distances may be off by, for caps to SHORT_CAP.  Beyond, small u take Lambert's continued fraction, u (105 + 10 u^2) / (105 + 45 u^2 + u^4), whose
// next term is below 2^-24 to 1/2: a relative 2^-21 everywhere, so that a cap far above the scores leaves them as they are.
// ([2,2048,8,128], causal, bfloat16, forward and gradients: cap of 30 366 and 1280 us, of 100 376 and 1288, none 328 and 1264.)
constexpr float SHORT_CAP = 64.f;
template <int N, bool SLANT> __device__ __forceinline__ void cap_scores(float *x, float *slant, float cap)
{
	const float inv_cap = __fdividef(1.f, cap); // (here: a register held for it beside the sums was one too many)
	auto set = [&](int i, float above, float below) {
		const float th = __fdividef(above, below);
		if (SLANT)
			slant[i] *= 1.f - th * th;
		x[i] = -cap * th;
	};
	auto u_of = [&](int i) { return fabsf(x[i] * inv_cap); };
	if (cap <= SHORT_CAP) {
#pragma unroll
		for (int i = 0; i < N; i++) {
			const float t = exp2_fast(-2.885390082f * u_of(i));
			set(i, 1.f - t, 1.f + t);
		}
	} else {
#pragma unroll
		for (int i = 0; i < N; i++) {
			const float u = u_of(i), z = u * u, t = exp2_fast(-2.885390082f * u);
			const bool small = u < 0.5f;
			set(i, small ? u * fmaf(10.f, z, 105.f) : 1.f - t, small ? fmaf(z, z + 45.f, 105.f) : 1.f + t);
		}
	}
}

// bfloat16 values as codes of 15 bits in their order: signs of differences then take one instruction for two (signs_of_codes).  A code is the value's
// magnitude, less CODE_BASE and not below 0, with its sign: exact from 2^-63 to 2^64, and for zero.
constexpr int CODE_BASE = 8063, CODE_MOST = 16383;
// two codes; *off: not zero once a value is not zero and outside
__device__ __forceinline__ uint32_t codes_of_bf16(uint32_t x, uint32_t *off)
{
	const uint32_t size = x & 0x7fff7fffu, above = __viaddmax_s16x2(size, uint32_t(-CODE_BASE & 0xffff) * 0x10001u, 0u);
	const uint32_t m = __vmins2(above, CODE_MOST * 0x10001u), minus = (x >> 15 & 0x10001u) * 0xffffu;
	*off |= (m ^ above) | (__vminu2(m, 0x10001u) ^ __vminu2(size, 0x10001u)); // cut at the top; at the bottom without being zero
	return __vsub2(m ^ minus, minus);
}
// sign(a - b) + 1 as float16: 0, 2^-24 or 2^-23; takes 1 - b
__device__ __forceinline__ uint32_t signs_of_codes(uint32_t a, uint32_t one_less_b) { return __viaddmin_s16x2_relu(a, one_less_b, 0x00020002u); }

// Where 16-byte piece c of row r lies in a tile of rows of `pieces` pieces (4, 8 or 16 where SWIZZLED).  SWIZZLED: for ldmatrix, eight rows at one piece
// in eight different places of the banks.
template <bool SWIZZLED> __device__ __forceinline__ uint32_t tile_offset(int pieces, int r, int c)
{
	return uint32_t(r * pieces + (SWIZZLED ? (pieces < 8 ? c ^ (r / 2 & 3) : c ^ (r & 7)) : c)) * 16;
}

// Rows [first, first + ROWS) of one head into shared memory, asynchronously where rows are 16-byte vectors (`vec`); zeros past n and past the width, and
// for rows of no document (`doc`: the batch item's documents, or null), whose contents are nobody's business.  A tile that is whole goes by the short
// loop: a copy and an addition a piece (the general one took a tenth of the forward).
template <typename T, bool SWIZZLED, int PIECES, int ROWS, int THREADS, int PITCH = PIECES>
__device__ __forceinline__ void load_tile16(uint32_t dst, const Strided &x, int b, int head, int first, int n, int width, const int32_t *doc, bool vec, int tid)
{
	constexpr int STEP = THREADS / PIECES; // rows a pass
	const T *src = static_cast<const T *>(x.p) + b * x.batch + head * x.head + first * x.tok;
	
	if (vec && first + ROWS <= n && !doc) {
		const int r0 = tid / PIECES, c = tid % PIECES, bytes = min(max(2 * width - 16 * c, 0), 16);
		const T *from = src + (bytes ? r0 * x.tok + 8 * c : 0);
		const long long step = bytes ? STEP * x.tok : 0;
		const uint32_t at = dst + tile_offset<SWIZZLED>(PITCH, r0, c);
		if (THREADS % PIECES == 0 || r0 < STEP) {
#pragma unroll
			for (int i = 0; i < (ROWS + STEP - 1) / STEP; i++) {
				if (ROWS % STEP == 0 || r0 + i * STEP < ROWS) // (rows of a thread lie at one place of the swizzle where they are multiples of eight apart)
					copy_async16(!SWIZZLED || STEP % 8 == 0 ? at + i * STEP * PITCH * 16 : dst + tile_offset<SWIZZLED>(PITCH, r0 + i * STEP, c), from, bytes);
				from += step;
			}
		}
		return;
	}
#pragma unroll 1
	for (int i = tid; i < ROWS * PIECES; i += THREADS) {
		const int r = i / PIECES, c = i % PIECES;
		const bool there = first + r < n && (!doc || doc[first + r] >= 0);
		const int left = there ? min(max(2 * width - 16 * c, 0), 16) : 0;
		const uint32_t at = dst + tile_offset<SWIZZLED>(PITCH, r, c);
		const T *from = src + (left ? r * x.tok + 8 * c : 0);
		if (vec) {
			copy_async16(at, left ? from : static_cast<const T *>(x.p), left);
			continue;
		}
		uint32_t v[4];
#pragma unroll
		for (int j = 0; j < 4; j++) {
			const uint32_t lo = 4 * j < left ? reinterpret_cast<const uint16_t *>(from)[2 * j] : 0;
			const uint32_t hi = 4 * j + 2 < left ? reinterpret_cast<const uint16_t *>(from)[2 * j + 1] : 0;
			v[j] = lo | hi << 16;
		}
		asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
	}
}

} // namespace l1b
