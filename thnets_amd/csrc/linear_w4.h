/* What the kernels of 4-bit Linear layers (linear_w4.hip, linear_w4_tile.hip) share: the arguments of a call and how
 * packed codes and rows of x become operands of the matrix core (not installed). */
#ifndef LINEAR_W4_H
#define LINEAR_W4_H

#include "thhip_internal.h"

#define W4_KSTEP 128	/* k of a packed step: four matrix instructions of 32 */
#define W4_X_I8 3	/* kind of x beside THHIP_F32, _F16, _BF16 */

struct w4_args {
	const void *x;
	const float *xscale;
	const unsigned char *codes;
	const void *scales;
	const unsigned char *zeros;
	const float *bias;
	void *y;
	long ldx, ldy;
	int B, nIn, nOut, steps, blocks, groups, group;
	int xgroups;		/* scales of a row of 8-bit x: 1, or one a group */
	int act, dtype;
	float thr, val;
	int shift;		/* log2(group), 31 where the row is one group */
	/* the group that matrix instruction j of a packed step belongs to (the last one past K's end) */
	__host__ __device__ int group_of(int step, int j) const
	{
		const int g = (int)(((long)step * W4_KSTEP + 32 * j) >> shift);
		return g < groups ? g : groups - 1;
	}
};

/* What differs with the kind of x: the matrix core's operand of eight k, its accumulator, and how a
 * word of eight codes and eight elements of x become operands.  PARTS: operands an x vector makes.  zero(z): a zero
 * point as weights() takes it; ZIN: weights() are n - z, else n.  UNIT: what a code of 1 is multiplied as.  Elements of bf16
 * and fp32 x may be as large as the sums they go into: with 2^-11 the 128 products of a step, at most 15 x 2^-11 each, stay
 * below fp32's largest number, as the result does that is kept in the same unit until it is written.  (The price: bits of y are lost
 * where it, or the sum of a group, is below 2^-115 instead of 2^-126.) */
template <int X> struct W4X;

#define W4_UNIT 0x1p-11f	/* of bf16 operands */

template <> struct W4X<THHIP_F16> {
	typedef _Float16 E;
	typedef E E8 __attribute__((ext_vector_type(8)));
	typedef halfx8 V;
	typedef floatx4 A;
	static constexpr int PARTS = 1;
	static constexpr float UNIT = 1.0f;
	static constexpr bool ZIN = true;
	static __device__ __forceinline__ unsigned zero(int z) { return __builtin_bit_cast(unsigned short, (_Float16)-z) * 0x10001u; }
	static __device__ __forceinline__ V weights(unsigned w, unsigned z)
	{
		typedef _Float16 h2 __attribute__((ext_vector_type(2)));
		const unsigned lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
		const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true);
		const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true);
		const h2 m = __builtin_bit_cast(h2, z), e = a + m, f = b + m, g = c + m, h = d + m;
		return (V){e[0], e[1], f[0], f[1], g[0], g[1], h[0], h[1]};
	}
	static __device__ __forceinline__ A mma(V a, V b, A c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
	static __device__ __forceinline__ void operand(const E8 x, V *out) { out[0] = x; }
};

template <> struct W4X<THHIP_BF16> {
	typedef __bf16 E;
	typedef E E8 __attribute__((ext_vector_type(8)));
	typedef bf16x8 V;
	typedef floatx4 A;
	static constexpr int PARTS = 1;
	static constexpr float UNIT = W4_UNIT;
	static constexpr bool ZIN = false;
	static __device__ __forceinline__ unsigned zero(int z) { return __float_as_uint((float)-z); }
	static __device__ __forceinline__ V ones() { return (V)(__bf16)W4_UNIT; }
	static __device__ __forceinline__ V weights(unsigned w, unsigned)
	{
		typedef __bf16 b2 __attribute__((ext_vector_type(2)));
		const unsigned lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
		const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f * W4_UNIT, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f * W4_UNIT, true);
		const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f * W4_UNIT, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f * W4_UNIT, true);
		return (V){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
	}
	static __device__ __forceinline__ A mma(V a, V b, A c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
	static __device__ __forceinline__ void operand(const E8 x, V *out) { out[0] = x; }
};

/* fp32: x = a + b + c, each the top sixteen bits of what is left (so eight bits of x; exact).  An
 * infinity leaves NaN behind: it makes every output of its row NaN. */
template <> struct W4X<THHIP_F32> {
	typedef float E;
	typedef E E8 __attribute__((ext_vector_type(8)));
	typedef bf16x8 V;
	typedef floatx4 A;
	static constexpr int PARTS = 3;
	static constexpr float UNIT = W4_UNIT;
	static constexpr bool ZIN = false;
	static __device__ __forceinline__ unsigned zero(int z) { return __float_as_uint((float)-z); }
	static __device__ __forceinline__ V ones() { return W4X<THHIP_BF16>::ones(); }
	static __device__ __forceinline__ V weights(unsigned w, unsigned z) { return W4X<THHIP_BF16>::weights(w, z); }
	static __device__ __forceinline__ A mma(V a, V b, A c) { return W4X<THHIP_BF16>::mma(a, b, c); }
	static __device__ __forceinline__ void operand(const E8 x, V *out)
	{
		typedef unsigned U __attribute__((ext_vector_type(4)));
		U p[3];
#pragma unroll
		for (int e = 0; e < 8; e += 2) {
			float u = x[e], v = x[e + 1];
#pragma unroll
			for (int i = 0; i < 3; i++) {
				const unsigned ub = __float_as_uint(u), vb = __float_as_uint(v);
				p[i][e / 2] = (ub >> 16) | (vb & 0xffff0000u);
				u -= __uint_as_float(ub & 0xffff0000u);
				v -= __uint_as_float(vb & 0xffff0000u);
			}
		}
#pragma unroll
		for (int i = 0; i < 3; i++)
			out[i] = __builtin_bit_cast(V, p[i]);
	}
};

template <> struct W4X<W4_X_I8> {
	typedef signed char E;
	typedef E E8 __attribute__((ext_vector_type(8)));
	typedef long V;
	typedef intx4 A;
	static constexpr int PARTS = 1;
	static constexpr float UNIT = 1.0f;
	static constexpr bool ZIN = true;
	static __device__ __forceinline__ unsigned zero(int z) { return __builtin_amdgcn_perm(z, z, 0); }
	/* (128 + n - z in every byte, which none borrows from another, without the 128) */
	static __device__ __forceinline__ V weights(unsigned w, unsigned z)
	{
		const unsigned lo = ((w & 0x0f0f0f0fu) | 0x80808080u) - z, hi = ((w >> 4 & 0x0f0f0f0fu) | 0x80808080u) - z;
		return (V)((unsigned long)(lo ^ 0x80808080u) | (unsigned long)(hi ^ 0x80808080u) << 32);
	}
	static __device__ __forceinline__ A mma(V a, V b, A c) { return __builtin_amdgcn_mfma_i32_16x16x32_i8(a, b, c, 0, 0, 0); }
	static __device__ __forceinline__ void operand(const E8 x, V *out) { out[0] = __builtin_bit_cast(V, x); }
};

/* bf16 operands n - z: by sign and magnitude, twice the work of n alone.  Worth it where that replaces the sums of x (the
 * tile kernel: 4096 x 8192 -> 8192 545 -> 525 us, with zero points 590 -> 510, groups of 32 880 -> 704), not where reading the
 * codes is all (one row, 8192 -> 32768 24.3 us with n, 28.3 with n - z). */
struct W4Signed : W4X<THHIP_BF16> {
	static constexpr bool ZIN = true;
	static __device__ __forceinline__ unsigned zero(int z) { return __builtin_amdgcn_perm(z, z, 0); }
	/* four bytes 128 + n - z to sign and magnitude, which e4m3 reads as (n - z) * 2^-9 */
	static __device__ __forceinline__ unsigned signed_bytes(unsigned n, unsigned z)
	{
		const unsigned u = ((n | 0x80808080u) - z) ^ 0x80808080u, s = u & 0x80808080u, one = s >> 7;
		return (u ^ (s - one)) + one;
	}
	static __device__ __forceinline__ V weights(unsigned w, unsigned z)
	{
		typedef __bf16 b2 __attribute__((ext_vector_type(2)));
		const unsigned lo = signed_bytes(w & 0x0f0f0f0fu, z), hi = signed_bytes(w >> 4 & 0x0f0f0f0fu, z);
		const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f * W4_UNIT, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f * W4_UNIT, true);
		const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f * W4_UNIT, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f * W4_UNIT, true);
		return (V){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
	}
};

/* N vectors of eight elements of x that may begin anywhere and end behind their row: vector i lies in row row(i), which
 * begins at element row * ldx, from k on.  fetch loads them without a branch, so that all are on their way together (with
 * one round each, the compiler waited for one before the next), and takes a row's last eight where it ends
 * before; fix moves those to their places, with zeros past the end.  FAR: rows may be further from x than 32 bits
 * reach, or have fewer than eight elements, which are put together one by one. */
template <int X, bool FAR, int N, typename ROW>
__device__ __forceinline__ void w4_fetch_x(typename W4X<X>::E8 (&v)[N], const void *x, long ldx, int nIn, int k, ROW row)
{
	typedef typename W4X<X>::E E;
	typedef typename W4X<X>::E8 E8;
	typedef E8 U __attribute__((aligned(sizeof(E))));
	if constexpr (!FAR) {
		const unsigned at = (unsigned)(k < nIn - 8 ? k : nIn - 8);
#pragma unroll
		for (int i = 0; i < N; i++)
			v[i] = *(const U *)((const char *)x + (unsigned)(((unsigned)row(i) * (unsigned)ldx + at) * (unsigned)sizeof(E)));
	} else if (nIn >= 8) {
		const int at = k < nIn - 8 ? k : nIn - 8;
#pragma unroll
		for (int i = 0; i < N; i++)
			v[i] = *(const U *)((const E *)x + row(i) * ldx + at);
	} else {
#pragma unroll
		for (int i = 0; i < N; i++)
#pragma unroll
			for (int e = 0; e < 8; e++)
				v[i][e] = ((const E *)x + row(i) * ldx)[e < nIn ? e : nIn - 1];
	}
}

template <int X, int N>
__device__ __forceinline__ void w4_fix_x(typename W4X<X>::E8 (&v)[N], int nIn, int k)
{
	typedef typename W4X<X>::E E;
	typedef typename W4X<X>::E8 E8;
	constexpr int ND = sizeof(E8) / 4;
	typedef unsigned D __attribute__((ext_vector_type(ND)));
	if (k >= nIn) {
#pragma unroll
		for (int i = 0; i < N; i++)
			v[i] = (E8)(E)0;
	} else if (k + 8 > nIn) {
		/* the row's last eight, by elements further back than wanted (rows of fewer: from 0) */
		const int by = nIn >= 8 ? k - (nIn - 8) : 0, words = by * (int)sizeof(E) / 4, bits = by * (int)sizeof(E) % 4 * 8;
#pragma unroll
		for (int i = 0; i < N; i++) {
			D d = __builtin_bit_cast(D, v[i]);
#pragma unroll
			for (int b = 1; b < ND; b *= 2)
#pragma unroll
				for (int j = 0; j < ND; j++)
					d[j] = words & b ? (j + b < ND ? d[j + b] : 0u) : d[j];
			if constexpr (sizeof(E) < 4)
#pragma unroll
				for (int j = 0; j < ND; j++)
					d[j] = __builtin_amdgcn_alignbit(j + 1 < ND ? d[j + 1] : 0u, d[j], bits);
			v[i] = __builtin_bit_cast(E8, d);
			if (nIn < 8)
#pragma unroll
				for (int e = 0; e < 8; e++)
					v[i][e] = e < nIn ? v[i][e] : (E)0;
		}
	}
}

/* The batch as seen from row b0 on, n rows */
__host__ __device__ static inline w4_args w4_rows(w4_args a, int b0, int n, size_t esx, size_t esy)
{
	a.x = (const char *)a.x + (long)b0 * a.ldx * esx;
	a.y = (char *)a.y + (long)b0 * a.ldy * esy;
	a.xscale = a.xscale ? a.xscale + (long)b0 * a.xgroups : 0;
	a.B = n;
	return a;
}

/* A result, in the type of x or, where x is 8-bit, in the one the call names */
template <int X>
__device__ __forceinline__ void w4_put(void *p, long i, float v, int dtype)
{
	if constexpr (X != W4_X_I8)
		ThhipElem<X>::st(p, i, v);
	else if (dtype == THHIP_F32)
		ThhipElem<THHIP_F32>::st(p, i, v);
	else if (dtype == THHIP_F16)
		ThhipElem<THHIP_F16>::st(p, i, v);
	else
		ThhipElem<THHIP_BF16>::st(p, i, v);
}

/* linear_w4_tile.hip: batches for which the matrix cores set the time */
void w4_tile(const w4_args &a, int xkind);

#endif
