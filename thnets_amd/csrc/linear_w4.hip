/*
 * Linear layers whose weights have 4 bits.
 *
 *   y[b][o] = act(bias[o] + sum_g s[o][g] * sum_{k in g} (n[o][k] - z[o][g]) * x[b][k])
 *
 * n: codes 0 .. 15; a group of `group` consecutive k of a row shares a scale s and a zero
 * point z (8 where the layer has none).  x is fp32 / fp16 / bf16, or signed 8-bit codes q with
 * fp32 scales, x[b][k] = sx[b][g'] * q[b][k].  The reference's Linear (modules/Linear.c:72-113)
 * knows fp32 weights only; its 8-bit path (lowp_basic.c:299-321) one range for the whole matrix.
 *
 * Arithmetic.  Inside a group the matrix cores sum (n - z) * x, whole numbers that every type holds, in
 * fp32 (int32 for 8-bit x, where the sum is exact).  A finished group adds s times that to the fp32
 * result, so a weight is never rounded and the scale is applied once a group.  z is taken from the codes where
 * an instruction does it for two or four of them (fp16 and 8-bit x: 4096 x 8192 -> 8192 with zero points 610 -> 532 us).
 * bf16 has none: for few rows of x the sums are of n x and, by a matrix of ones, of x, and a group adds
 * s * (sum n x - z * sum x); larger batches make n - z of the bytes by sign and magnitude.  fp32 x is cut into three
 * bf16 parts of eight bits each that add up to it exactly.
 *
 * A code becomes a half value without an integer conversion: the byte 0000nnnn read as an e4m3
 * number is n * 2^-9 for all sixteen codes (eight denormals, eight of the first binade), and
 * v_cvt_scalef32_pk_{f16,bf16}_fp8 widens two of them with a factor of 2^9 (bf16: of 2^-2, as its sums
 * are kept in units of 2^-11; W4_UNIT).  For 8-bit x z is taken
 * from four bytes 128 + n in one subtraction, in which none borrows from another, and a flipped top bit takes the
 * 128 away.
 *
 * Weights are packed by thhip_w4_pack into one buffer:
 *   codes   [16-row block][step of 128 k][lane][4 words], word j of lane l: row l % 16,
 *           k = 32 j + 8 (l / 16) + 0 .. 7, low nibbles of the four bytes first, then the high
 *           ones: 1 KiB that a wavefront loads with one instruction and multiplies as it lies
 *   scales  [16-row block][group][16 rows], fp32 / fp16 / bf16
 *   zeros   [16-row block][group][16 rows], bytes (only where the layer has zero points)
 * Rows past nOut and k past nIn are padded with 0.
 */
#include <stdint.h>
#include <stdio.h>
#include "linear_w4.h"

struct w4_layout {
	int blocks, steps, groups;
	size_t scales, zeros, bytes;	/* offsets of the sections, and the whole */
};

static size_t round16(size_t n)
{
	return (n + 15) & ~(size_t)15;
}

static struct w4_layout w4_layout_of(int nOut, int nIn, int group, int dtype, int zeros)
{
	struct w4_layout l;
	l.blocks = (int)(((long)nOut + 15) / 16);
	l.steps = (int)(((long)nIn + W4_KSTEP - 1) / W4_KSTEP);
	l.groups = group ? (int)(((long)nIn + group - 1) / group) : 1;
	l.scales = (size_t)l.blocks * l.steps * 1024;
	l.zeros = l.scales + round16((size_t)l.blocks * l.groups * 16 * thhip_esize(dtype));
	l.bytes = l.zeros + (zeros ? (size_t)l.blocks * l.groups * 16 : 0);
	return l;
}

static const char *w4_bad(int nOut, int nIn, int group, int dtype)
{
	if (nOut < 1 || nIn < 1 || nOut > 1 << 30 || nIn > 1 << 30)
		return "a layer has 1 to 2^30 inputs and outputs";
	if (group != 0 && group != 32 && group != 64 && group != 128 && group != 256)
		return "a group has 32, 64, 128 or 256 weights, or is the row (0)";
	if (dtype != THHIP_F32 && dtype != THHIP_F16 && dtype != THHIP_BF16)
		return "the type is fp32, fp16 or bf16";
	return 0;
}

extern "C" size_t thhip_w4_packed_bytes(int nOut, int nIn, int group, int dtype, int zeros)
{
	return w4_bad(nOut, nIn, group, dtype) ? 0 : w4_layout_of(nOut, nIn, group, dtype, zeros).bytes;
}

/* ---- laying out and making weights ----
 *
 * Once a layer, bound by memory: a thread makes one word of eight codes from four bytes (8192 -> 32768: 268 MB in 103 us, 2.6
 * TB/s; code by code it was 477). */

__global__ __launch_bounds__(256) void w4_pack_codes_kernel(const unsigned char *codes, unsigned *out, int nOut, int nIn,
	int steps, size_t words)
{
	typedef unsigned U __attribute__((aligned(1)));
	const size_t row_bytes = ((size_t)nIn + 1) / 2;
	for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (size_t)gridDim.x * 256) {
		const int j = i & 3, lane = (i >> 2) & 63;
		const size_t step = i >> 8;
		const long row = (long)(step / steps) * 16 + (lane & 15);
		const long k0 = (long)(step % steps) * W4_KSTEP + 32 * j + 8 * (lane >> 4);
		/* eight codes of the row: four of its bytes, or what is left of them and zeros */
		unsigned u = 0, w = 0;
		if (row < nOut && k0 < nIn) {
			const unsigned char *from = codes + row * row_bytes + k0 / 2;
			if (k0 + 8 <= nIn)
				u = *(const U *)from;
			else
				for (int e = 0; e < nIn - k0; e++)
					u |= (unsigned)(from[e / 2] >> (4 * (e & 1)) & 15) << (4 * e);
		}
#pragma unroll
		for (int e = 0; e < 8; e++)
			w |= (u >> (4 * e) & 15) << (8 * (e & 3) + 4 * (e >> 2));
		out[i] = w;
	}
}

/* scales or zeros: [nOut][groups] -> [16-row block][group][16 rows], esize bytes each */
__global__ __launch_bounds__(256) void w4_pack_groups_kernel(const unsigned char *in, unsigned char *out, int nOut, int groups,
	int esize, size_t n)
{
	for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
		const size_t g = (i >> 4) % groups;
		const long row = (long)((i >> 4) / groups) * 16 + (long)(i & 15);
		for (int b = 0; b < esize; b++)
			out[i * esize + b] = row < nOut ? in[(row * groups + g) * esize + b] : 0;
	}
}

static unsigned w4_grid(size_t n)
{
	const size_t g = (n + 255) / 256;
	return (unsigned)(g < 65536 ? g : 65536);
}

extern "C" int thhip_w4_pack(const unsigned char *codes, const void *scales, const unsigned char *zeros, void *packed,
	int nOut, int nIn, int group, int dtype)
{
	const char *bad = w4_bad(nOut, nIn, group, dtype);
	if (!bad && (!codes || !scales || !packed))
		bad = "codes, scales and the packed buffer are needed";
	if (!bad && (uintptr_t)packed % 16)
		bad = "the packed buffer is not aligned to 16 bytes";
	if (bad) {
		fprintf(stderr, "thhip_w4_pack: %d -> %d, group %d, dtype %d: %s\n", nIn, nOut, group, dtype, bad);
		return -1;
	}
	const struct w4_layout l = w4_layout_of(nOut, nIn, group, dtype, zeros != 0);
	ThhipLaunchScope scope(THHIP_FAM_OTHER, (double)nOut * nIn / 2 + (double)l.bytes);
	const size_t words = l.scales / 4, ns = (size_t)l.blocks * l.groups * 16;
	w4_pack_codes_kernel<<<dim3(w4_grid(words)), dim3(256), 0, thhip_stream()>>>(codes, (unsigned *)packed, nOut, nIn, l.steps, words);
	w4_pack_groups_kernel<<<dim3(w4_grid(ns)), dim3(256), 0, thhip_stream()>>>((const unsigned char *)scales,
		(unsigned char *)packed + l.scales, nOut, l.groups, thhip_esize(dtype), ns);
	if (zeros)
		w4_pack_groups_kernel<<<dim3(w4_grid(ns)), dim3(256), 0, thhip_stream()>>>(zeros, (unsigned char *)packed + l.zeros,
			nOut, l.groups, 1, ns);
	return 0;
}

/* rint(v / s).  v times the reciprocal of s is off by at most 2^-23 of it, 2^-19 for quotients up to 15 (larger ones are cut
 * off): next to the middle between two whole numbers the quotient itself is taken, in 64 bits. */
__device__ __forceinline__ float w4_nearest(float v, float s, float inv)
{
	const float q = v * inv, n = rintf(q);
	return fabsf(q - n) > 0.5f - 0x1p-18f ? (float)rint((double)v / (double)s) : n;
}

/* One wavefront a (row, group): the group's extremes, its scale rounded to the type it is kept in,
 * and the codes nearest to w / scale (+ zero).  Two weights of a byte belong to one lane. */
template <int WDT, int DT>
__global__ __launch_bounds__(256) void w4_quantize_kernel(const void *w, long ldw, unsigned char *codes, void *scales,
	unsigned char *zeros, int nOut, int nIn, int group, int groups)
{
	const int lane = threadIdx.x & 63;
	const size_t n = (size_t)nOut * groups;
	for (size_t i = (size_t)blockIdx.x * 4 + threadIdx.x / 64; i < n; i += (size_t)gridDim.x * 4) {
		const long row = (long)(i / groups);
		const int g = (int)(i % groups);
		const int k0 = g * group, k1 = group && k0 + group < nIn ? k0 + group : nIn;
		float lo = 0, hi = 0;
		for (int k = k0 + lane; k < k1; k += 64) {
			const float v = ThhipElem<WDT>::ld(w, row * ldw + k);
			lo = fminf(lo, v);
			hi = fmaxf(hi, v);
		}
#pragma unroll
		for (int off = 32; off > 0; off >>= 1) {
			lo = fminf(lo, __shfl_xor(lo, off, 64));
			hi = fmaxf(hi, __shfl_xor(hi, off, 64));
		}
		/* (a scale that the type does not hold becomes its largest: the outermost weights are cut off) */
		const float most = DT == THHIP_F16 ? 65504.0f : 3e38f;
		typename ThhipElem<DT>::T sr = (typename ThhipElem<DT>::T)fminf(zeros ? hi / 15.0f - lo / 15.0f : fmaxf(hi, -lo) / 7.0f, most);
		const float s = (float)sr, inv = s > 0 && 1.0f / s < INFINITY ? 1.0f / s : 0.0f;
		const float z = zeros ? fminf(w4_nearest(-lo, s, inv), 15.0f) : 8.0f;
		if (lane == 0) {
			ThhipElem<DT>::st(scales, (long)i, s);
			if (zeros)
				zeros[i] = (unsigned char)(int)z;
		}
		for (int k = k0 + 2 * lane; k < k1; k += 128) {
			unsigned b = 0;
			for (int e = 0; e < 2 && k + e < k1; e++) {
				const float v = ThhipElem<WDT>::ld(w, row * ldw + k + e);
				b |= (unsigned)(int)fminf(fmaxf(w4_nearest(v, s, inv) + z, 0.0f), 15.0f) << (4 * e);
			}
			codes[row * (((long)nIn + 1) / 2) + k / 2] = (unsigned char)b;
		}
	}
}

extern "C" int thhip_quantize_w4(const void *w, long ldw, int wtype, unsigned char *codes, void *scales, unsigned char *zeros,
	int nOut, int nIn, int group, int dtype)
{
	const char *bad = w4_bad(nOut, nIn, group, dtype);
	if (!bad && wtype != THHIP_F32 && wtype != THHIP_F16 && wtype != THHIP_BF16)
		bad = "the weights are fp32, fp16 or bf16";
	if (!bad && (!w || !codes || !scales))
		bad = "weights, codes and scales are needed";
	if (!bad && ldw < nIn)
		bad = "the row stride is smaller than the row";
	if (bad) {
		fprintf(stderr, "thhip_quantize_w4: %d -> %d, group %d, types %d %d: %s\n", nIn, nOut, group, wtype, dtype, bad);
		return -1;
	}
	const int groups = group ? (int)(((long)nIn + group - 1) / group) : 1;
	const unsigned grid = w4_grid(((size_t)nOut * groups + 3) / 4 * 256);
	ThhipLaunchScope scope(THHIP_FAM_OTHER, (double)nOut * nIn * (thhip_esize(wtype) + 0.5));
#define W4_QUANTIZE(WDT) THHIP_DISPATCH_FLOAT(dtype, (w4_quantize_kernel<WDT, DT><<<dim3(grid), dim3(256), 0, thhip_stream()>>>( \
	w, ldw, codes, scales, zeros, nOut, nIn, group, groups)))
	if (wtype == THHIP_F32)
		W4_QUANTIZE(THHIP_F32);
	else if (wtype == THHIP_F16)
		W4_QUANTIZE(THHIP_F16);
	else
		W4_QUANTIZE(THHIP_BF16);
#undef W4_QUANTIZE
	return 0;
}

/* ---- the product ---- */

static int g_w4_shape = -1;

extern "C" void thhip_w4_set_shape(int shape)
{
	g_w4_shape = shape >= 0 && shape <= 5 ? shape : -1;
}

/* ---- few columns: bound by reading the weights once ----
 *
 * A workgroup of W wavefronts computes RB blocks of 16 rows for all columns and all of K.  K is walked in
 * chunks of W steps, wavefront w multiplying step w of every chunk, so that the workgroup reads W KiB of
 * contiguous codes of a row block at a time.  Codes, scales and zeros go straight to registers, D chunks
 * ahead; x goes through LDS, where all wavefronts of the workgroup put a chunk of it down together, one
 * chunk ahead (two buffers, one barrier a chunk): taken to pieces there once, fp32 x is 3 B columns of
 * bf16 from then on, and the matrix core sees columns only.  Columns past the last read a piece of zeros.
 * A 16-byte piece u of a column c's chunk lies in place u ^ c % 16, which puts the 16 columns of an operand on
 * different banks.
 * Of a 16 x 16 tile a lane holds row lane % 16, whose scale and zero point it needs, of columns 4 (lane / 16) + 0 .. 3.  The wavefronts' sums are
 * added through LDS, in their order, and an fp32 row's three columns with them.
 * GM: matrix instructions a group spans within a step (1: groups of 32 or 64, 4: larger).
 *
 * Bound by memory where the layer is large: 1 x 8192 -> 32768 bf16 23.7 us (138 MB, 5.8 TB/s, some of it from the last-level cache; a large copy moves 5.1),
 * 1 x 25088 -> 4096 fp32 13.0 us (53 MB, 4.1 TB/s: 256 workgroups, one a CU, whose start and end do not overlap), 1 x
 * 4096 -> 16384 with 8-bit x 9.0 us (35 MB, 3.9 TB/s).  By the vector unit (codes to operands) and the L2's x from about
 * 32 columns on: 128 x 4096 -> 4096 fp16 11.9 us (360 TFLOP/s). */

/* The workgroup's LDS traffic so far is done, for everybody (loads from memory may still be on their way) */
__device__ __forceinline__ void w4_lds_barrier(void)
{
	asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* What a wavefront fetches ahead of a step: the codes of its row blocks and what their groups need.  (The number of
 * loads does not depend on the call, so that the compiler can count how many may be outstanding when it needs one.) */
template <int X, int RB, int GM, bool ZP> struct W4Step {
	/* 8-bit x: the scale of a type that only the call knows, in the word it lies in */
	typedef typename ThhipElem<X == W4_X_I8 ? THHIP_F32 : X>::T T;
	uintx4 codes[RB];
	T s[RB][4 / GM];
	unsigned char z[RB][4 / GM];
	__device__ __forceinline__ void fetch(const w4_args &a, int rb0, int step, int lane)
	{
		if (step >= a.steps)
			step = a.steps - 1;	/* (loaded, not used) */
#pragma unroll
		for (int r = 0; r < RB; r++) {
			const int rb = rb0 + r < a.blocks ? rb0 + r : a.blocks - 1;
			codes[r] = *(const uintx4 *)(a.codes + ((size_t)rb * a.steps + step) * 1024 + lane * 16);
#pragma unroll
			for (int j = 0; j < 4 / GM; j++) {
				const size_t at = ((size_t)rb * a.groups + a.group_of(step, j * GM)) * 16 + (lane & 15);
				if constexpr (X != W4_X_I8)
					s[r][j] = ((const T *)a.scales)[at];
				else
					s[r][j] = *(const float *)((const char *)a.scales + (a.dtype == THHIP_F32 ? at * 4 : at * 2 & ~(size_t)3));
				if constexpr (ZP)
					z[r][j] = a.zeros[at];
			}
		}
	}
	__device__ __forceinline__ float scale(const w4_args &a, int r, int j, int lane) const
	{
		if constexpr (X != W4_X_I8)
			return (float)s[r][j];
		else {
			const unsigned u = __float_as_uint(s[r][j]), h = u >> (16 * (lane & 1)) & 0xffff;
			const float f16 = (float)__builtin_bit_cast(_Float16, (unsigned short)h);
			return a.dtype == THHIP_F32 ? s[r][j] : a.dtype == THHIP_F16 ? f16 : __uint_as_float(h << 16);
		}
	}
};

template <int X, int RB, int NB, int XV, int GM, bool ZP, int W, int D, bool FAR>
__global__ __launch_bounds__(W * 64) void w4_skinny_kernel(const w4_args all, int slices)
{
	typedef W4X<X> K;
	typedef typename K::V V;
	typedef typename K::A A;
	typedef W4Step<X, RB, GM, ZP> Step;
	constexpr int ES = sizeof(V) / 8;		/* bytes of an operand's element */
	constexpr int T = W * 64, ROWV = W * 16;	/* threads; vectors of eight in a row's chunk */
	constexpr int CK = W * W4_KSTEP;		/* k of a chunk */
	constexpr int STRIDE = CK * ES;
	extern __shared__ __align__(16) unsigned char lds[];
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	const int col = lane & 15, quarter = lane >> 4;
	/* the slices of the batch that need the same codes are neighbours on one XCD (workgroups b, b + 8, ...) */
	const int turn = blockIdx.x >> 3, rb0 = ((turn / slices) * 8 + (blockIdx.x & 7)) * RB;
	if (rb0 >= all.blocks)
		return;
	constexpr int ROWS = NB * 16 / K::PARTS;
	const int b0 = turn % slices * ROWS;
	const w4_args a = w4_rows(all, b0, all.B - b0 < ROWS ? all.B - b0 : ROWS, sizeof(typename K::E),
		X == W4_X_I8 ? (all.dtype == THHIP_F32 ? 4 : 2) : sizeof(typename K::E));
	const int cols = a.B * K::PARTS, buf = cols * STRIDE;
	const int chunks = (a.steps + W - 1) / W;

	/* x of a chunk on its way to LDS: vector tid + i * T of the workgroup's, in the order of the rows */
	typename K::E8 xr[XV];
	auto x_row = [&](int i) { return (tid + i * T) / ROWV; };
	auto load_x = [&](int c) {
		w4_fetch_x<X, FAR>(xr, a.x, a.ldx, a.nIn, c * CK + tid % ROWV * 8, [&](int i) { return (long)(x_row(i) < a.B ? x_row(i) : a.B - 1); });
	};
	auto store_x = [&](int c) {
		if ((c + 1) * CK > a.nIn)
			w4_fix_x<X>(xr, a.nIn, c * CK + tid % ROWV * 8);
#pragma unroll
		for (int i = 0; i < XV; i++)
			if (x_row(i) < a.B) {
				V o[K::PARTS];
				K::operand(xr[i], o);
#pragma unroll
				for (int p = 0; p < K::PARTS; p++)
					*(V *)(lds + (c & 1) * buf + (x_row(i) * K::PARTS + p) * STRIDE +
						(tid % ROWV * 8 * ES ^ ((x_row(i) * K::PARTS + p) & 15) * 16)) = o[p];
			}
	};
	/* 8-bit x: its rows' scales for a chunk go the same way, [buffer][part of a step][row] behind the zeros */
	constexpr int SLOTS = W * 4 / GM, XS = X == W4_X_I8 ? (ROWS * SLOTS + T - 1) / T : 0;
	float *lxs = (float *)(lds + 2 * buf + W4_KSTEP * ES);
	float xs[XS + 1];
	auto load_xs = [&](int c) {
#pragma unroll
		for (int i = 0; i < XS; i++) {
			const int slot = (tid + i * T) / ROWS % SLOTS, row = (tid + i * T) % ROWS;
			const int step = c * W + slot / (4 / GM), g = a.group_of(step < a.steps ? step : a.steps - 1, slot % (4 / GM) * GM);
			xs[i] = a.xscale[(long)(row < a.B ? row : 0) * a.xgroups + (a.xgroups > 1 ? g : 0)];
		}
	};
	auto store_xs = [&](int c) {
#pragma unroll
		for (int i = 0; i < XS; i++)
			if (XS * T == ROWS * SLOTS || tid + i * T < ROWS * SLOTS)
				lxs[(c & 1) * (ROWS * SLOTS) + tid + i * T] = a.xgroups > 1 ? xs[i] : 1.0f;
	};
	/* where a lane's operands lie: in either buffer, or among the zeros; of matrix instruction j at ^ j * 32 * ES */
	int at[2][NB];
#pragma unroll
	for (int n = 0; n < NB; n++)
#pragma unroll
		for (int b = 0; b < 2; b++)
			at[b][n] = n * 16 + col < cols ? b * buf + (n * 16 + col) * STRIDE + ((wave * W4_KSTEP + quarter * 8) * ES ^ col * 16) :
				2 * buf + quarter * 8 * ES;

	floatx4 acc[RB][NB];
#pragma unroll
	for (int r = 0; r < RB; r++)
#pragma unroll
		for (int n = 0; n < NB; n++)
			acc[r][n] = (floatx4)0.0f;

	Step st[D];
	/* (in the order in which the loop asks for them, so that its waits fit the first time round too) */
	load_x(0);
	load_xs(0);
#pragma unroll
	for (int d = 0; d < D - 1; d++)
		st[d].fetch(a, rb0, d * W + wave, lane);
	if (tid < 32 * ES)
		((unsigned *)(lds + 2 * buf))[tid] = 0;
	store_x(0);
	store_xs(0);
	load_x(1);
	load_xs(1);
	st[D - 1].fetch(a, rb0, (D - 1) * W + wave, lane);
	w4_lds_barrier();

	constexpr int U = D % 2 ? 2 * D : D;	/* chunks after which buffers and stages are the first again */
	for (int c0 = 0; c0 < chunks; c0 += U) {
#pragma unroll
		for (int u = 0; u < U; u++) {
			const int c = c0 + u;
			if (c >= chunks)
				break;
			store_x(c + 1);		/* (behind K's end: zeros, which nobody reads) */
			store_xs(c + 1);
			load_x(c + 2);
			load_xs(c + 2);
			const int step = c * W + wave;
			Step &now = st[u % D];
			if (step < a.steps) {
				A p[RB][NB], sx[NB];
#pragma unroll
				for (int j = 0; j < 4; j++) {
					V w[RB];
#pragma unroll
					for (int r = 0; r < RB; r++)
						w[r] = K::weights(now.codes[r][j], K::zero(ZP ? now.z[r][j / GM] : 8));
#pragma unroll
					for (int n = 0; n < NB; n++) {
						const V x = *(const V *)(lds + (at[u & 1][n] ^ j * 32 * ES));
						if constexpr (!K::ZIN)
							sx[n] = K::mma(x, K::ones(), j % GM ? sx[n] : (A)0);
#pragma unroll
						for (int r = 0; r < RB; r++)
							p[r][n] = K::mma(x, w[r], j % GM ? p[r][n] : (A)0);
					}
					if ((j + 1) % GM)
						continue;
					floatx4 xn[NB];
					if constexpr (X == W4_X_I8)
#pragma unroll
						for (int n = 0; n < NB; n++)
							xn[n] = *(const floatx4 *)(lxs + (u & 1) * (ROWS * SLOTS) + (wave * (4 / GM) + j / GM) * ROWS + n * 16 + 4 * quarter);
#pragma unroll
					for (int r = 0; r < RB; r++) {
						const float s = now.scale(a, r, j / GM, lane);
						const float z = ZP ? (float)now.z[r][j / GM] : 8.0f;
#pragma unroll
						for (int n = 0; n < NB; n++)
#pragma unroll
							for (int i = 0; i < 4; i++) {
								if constexpr (X == W4_X_I8)
									acc[r][n][i] += s * xn[n][i] * (float)p[r][n][i];
								else if constexpr (K::ZIN)
									acc[r][n][i] += s * p[r][n][i];
								else
									acc[r][n][i] += s * (p[r][n][i] - z * sx[n][i]);
							}
					}
					/* (now, not at the end of the step, for which the registers do not last) */
					if constexpr (GM == 1)
#pragma unroll
						for (int r = 0; r < RB; r++)
#pragma unroll
							for (int n = 0; n < NB; n++)
								asm("" : "+v"(acc[r][n]));
				}
			}
			now.fetch(a, rb0, step + D * W, lane);
			w4_lds_barrier();
		}
	}

	floatx4 *red = (floatx4 *)lds;	/* [W][RB][NB][64 lanes] */
#pragma unroll
	for (int r = 0; r < RB; r++)
#pragma unroll
		for (int n = 0; n < NB; n++)
			red[((wave * RB + r) * NB + n) * 64 + lane] = acc[r][n];
	__syncthreads();
	for (int t = tid; t < RB * 16 * a.B; t += T) {
		const int row = t % (RB * 16), b = t / (RB * 16), o = rb0 * 16 + row;
		if (o >= a.nOut)
			continue;
		float y = 0;
#pragma unroll
		for (int w = 0; w < W; w++)
#pragma unroll
			for (int p = 0; p < K::PARTS; p++) {
				const int c = b * K::PARTS + p;
				y += ((const float *)&red[((w * RB + row / 16) * NB + c / 16) * 64 + (c % 16 / 4) * 16 + row % 16])[c % 4];
			}
		if (X == W4_X_I8 && a.xgroups == 1)
			y *= a.xscale[b];
		y *= 1.0f / K::UNIT;
		y += a.bias ? a.bias[o] : 0.0f;
		if (a.act)
			y = y > a.thr ? y : a.val;
		w4_put<X>(a.y, b * a.ldy + o, y, a.dtype);
	}
}

template <int X, int RB, int NB, int XV, int GM, bool ZP, int W, int D, bool FAR>
static void w4_skinny_launch(const w4_args &all)
{
	typedef W4X<X> K;
	constexpr int ES = sizeof(typename K::V) / 8, ROWS = NB * 16 / K::PARTS;
	const int rows = all.B < ROWS ? all.B : ROWS;
	size_t lds = 2 * (size_t)rows * K::PARTS * (W * W4_KSTEP * ES) + W4_KSTEP * ES;
	if (X == W4_X_I8)
		lds += 2 * (size_t)ROWS * (W * 4 / GM) * 4;
	const size_t red = (size_t)W * RB * NB * 1024;
	lds = lds > red ? lds : red;
	static bool raised;
	if (!raised) {
		hipcheck(hipFuncSetAttribute((const void *)w4_skinny_kernel<X, RB, NB, XV, GM, ZP, W, D, FAR>,
			hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
		raised = true;
	}
	/* a launch has fewer than 2^32 threads: slices of the batch at a time */
	const unsigned groups = ((all.blocks + RB - 1) / RB + 7) / 8 * 8;
	const long most = 0xffffffffl / (W * 64) / groups * ROWS;
	for (long b0 = 0; b0 < all.B; b0 += most) {
		const w4_args a = w4_rows(all, (int)b0, (int)(all.B - b0 < most ? all.B - b0 : most), sizeof(typename K::E), thhip_esize(all.dtype));
		const unsigned slices = (a.B + ROWS - 1) / ROWS;
		w4_skinny_kernel<X, RB, NB, XV, GM, ZP, W, D, FAR><<<dim3(groups * slices), dim3(W * 64), lds, thhip_stream()>>>(a, slices);
	}
}

/* ---- which kernel and shape ----
 *
 * Up to 16 columns: 16 rows a workgroup and 16 wavefronts, of which a CU holds one (two of the forms that need no more than
 * 64 registers: up to four rows of half types and 8-bit x); from 1024 row blocks on 32 rows and eight wavefronts, two
 * workgroups a CU (1 x 8192 -> 16384 bf16: 13.0 us; the other 19 us.  12288 outputs, by the first form: 12.0).
 * More columns: the shape that takes the least time by the estimate below.  A launch runs in rounds of as many
 * workgroups as the GPU holds; the time of a round was measured at K = 512, 2048 and 8192 and is a start and a
 * slope.  Few rows at a time win in small layers and short K, 64 rows in larger ones (4096 -> 4096 fp16, us, in the
 * order of the table: 128 columns 37 / 24 / 27 / 17.4 / 12.8, tiles 50), tiles from about 512 columns on (768 columns: 81
 * with 64 rows, 56 with tiles).  Of three times 78 layers drawn at random (16 to 1300 rows, 512 to 9216 inputs, 256 to 10240 outputs) the
 * choice took 0.8 to 1.7 % more than the best shape, 27 % at most. */
enum { W4_16x16, W4_32x16, W4_16x32, W4_32x32, W4_64x32, W4_TILES };

static int w4_shape(const w4_args &a, int parts)
{
	static const float round_us[4][5][2] = {	/* start, and us for 1024 k */
		{{4.0f, 0.42f}, {4.9f, 0.57f}, {3.9f, 0.93f}, {4.4f, 1.22f}, {5.5f, 1.75f}},
		{{4.6f, 0.55f}, {5.6f, 0.87f}, {4.2f, 1.25f}, {4.8f, 1.65f}, {5.9f, 2.6f}},	/* groups of 32 and 64 */
		{{3.9f, 0.42f}, {4.9f, 0.54f}, {3.3f, 0.73f}, {4.3f, 1.0f}, {6.3f, 1.6f}},	/* 8-bit x */
		{{4.5f, 0.65f}, {6.0f, 1.2f}, {4.4f, 1.35f}, {5.6f, 2.2f}, {8.0f, 3.8f}},	/* ... in groups of 32 and 64 */
	};
	static const float tile_us[3][3][2] = {
		{{13.0f, 10.0f}, {13.0f, 10.7f}, {14.0f, 13.7f}},	/* groups of 128 and more, 64, 32 */
		{{8.0f, 17.0f}, {8.0f, 19.5f}, {8.0f, 22.0f}},		/* fp32 x, 128 rows */
		{{14.0f, 20.0f}, {15.0f, 21.0f}, {15.0f, 25.0f}},	/* fp32 x, 256 rows */
	};
	static const int rows[5] = {1, 2, 1, 2, 4}, cols[5] = {1, 1, 2, 2, 2};	/* blocks of 16 */
	const float (*us)[2] = round_us[(a.xscale ? 2 : 0) + (a.group == 32 || a.group == 64)];
	const float k = (float)a.nIn / 1024;
	/* tiles: 128 rows x 128 columns, two on a CU (one alone takes two thirds of the time of two); fp32 x 64 rows of x, one on a
	 * CU, of 256 rows where there are more than 256 */
	const long wide = ((long)a.B + (parts > 1 ? 63 : 127)) / (parts > 1 ? 64 : 128), tiles = wide * ((a.blocks + 7) / 8);
	const float *tile = tile_us[parts == 1 ? 0 : tiles <= 256 ? 1 : 2][a.group == 32 ? 2 : a.group == 64];
	const float rounds = tiles <= 256 ? 1.0f : parts > 1 ? (float)((wide * ((a.blocks + 15) / 16) + 255) / 256) : 1.45f * (float)((tiles + 511) / 512);
	float best = (tile[0] + tile[1] * k) * rounds;
	int shape = W4_TILES;
	for (int i = 0; i < 5; i++) {
		const int slice = cols[i] * 16 / parts;
		const long n = (long)((a.blocks + rows[i] - 1) / rows[i]) * (((long)a.B + slice - 1) / slice);
		const float t = (float)((n + 255) / 256) * (us[i][0] + us[i][1] * k);
		if (t < best) {
			best = t;
			shape = i;
		}
	}
	return shape;
}

template <int X, int GM, bool ZP>
static void w4_skinny(const w4_args &a, int shape, bool far)
{
	constexpr int P = W4X<X>::PARTS;
	/* vectors a thread moves a chunk for 16 and 32 columns: four rows each */
	constexpr int X1 = (16 / P + 3) / 4, X2 = (32 / P + 3) / 4;
	if (far)
		w4_skinny_launch<X, 1, 2, X2, GM, ZP, 8, 2, true>(a);
	else if (a.B <= 16 / P && a.blocks >= 1024) {
		if (a.B <= 4)
			w4_skinny_launch<X, 2, 1, 1, GM, ZP, 8, 2, false>(a);
		else
			w4_skinny_launch<X, 2, 1, X1, GM, ZP, 8, 2, false>(a);
	} else if (a.B <= 4)
		w4_skinny_launch<X, 1, 1, 1, GM, ZP, 16, 2, false>(a);
	else if (a.B <= 16 / P || shape == W4_16x16)
		w4_skinny_launch<X, 1, 1, X1, GM, ZP, 16, 2, false>(a);
	else if (shape == W4_32x16)
		w4_skinny_launch<X, 2, 1, X1, GM, ZP, 16, 2, false>(a);
	else if (shape == W4_16x32)
		w4_skinny_launch<X, 1, 2, X2, GM, ZP, 8, 2, false>(a);
	else if (shape == W4_32x32)
		w4_skinny_launch<X, 2, 2, X2, GM, ZP, 8, 2, false>(a);
	else
		w4_skinny_launch<X, 4, 2, X2, GM, ZP, 8, 2, false>(a);
}

template <int X>
static void w4_choose(const w4_args &a)
{
	const bool few = a.B <= 16 / W4X<X>::PARTS, small = a.group == 32 || a.group == 64;
	/* rows that 32 bits do not reach in a workgroup's columns, or of less than a vector */
	const bool far = a.nIn < 8 || a.ldx >= (1l << 31) / (128 * (long)sizeof(typename W4X<X>::E));
	const int shape = g_w4_shape >= 0 ? g_w4_shape : few ? W4_16x16 : w4_shape(a, W4X<X>::PARTS);
	if (shape == W4_TILES && !far)
		w4_tile(a, X);
	else if (a.zeros)
		small ? w4_skinny<X, 1, true>(a, shape, far) : w4_skinny<X, 4, true>(a, shape, far);
	else
		small ? w4_skinny<X, 1, false>(a, shape, far) : w4_skinny<X, 4, false>(a, shape, far);
}

#define W4_OUTPUTS (1 << 24)	/* of a launch, at most */

static int w4_run(const char *who, w4_args &a, const void *packed, int group, int zeros, int xkind, int xgroup, int dtype)
{
	const char *bad = w4_bad(a.nOut, a.nIn, group, dtype);
	const size_t es = dtype == THHIP_F32 ? 4 : 2, esx = xkind == W4_X_I8 ? 1 : es;
	if (!bad && a.B < 0)
		bad = "a batch has at least no rows";
	if (!bad && (a.ldx < a.nIn || a.ldy < a.nOut))
		bad = "a row stride is smaller than the row";
	if (!bad && a.B && (!a.x || !packed || !a.y || (xkind == W4_X_I8 && !a.xscale)))
		bad = "x, the weights and y are needed";
	if (!bad && ((uintptr_t)a.x % esx || (uintptr_t)a.y % es || (uintptr_t)packed % 16 || (uintptr_t)a.bias % 4 || (uintptr_t)a.xscale % 4))
		bad = "a pointer is not aligned to its element (packed weights: 16 bytes)";
	if (!bad && xkind == W4_X_I8 && xgroup != 0 && xgroup != group)
		bad = "the scales of x are one a row (0) or one a group of the weights";
	if (bad) {
		fprintf(stderr, "%s: B=%d %d -> %d, group %d, dtype %d: %s\n", who, a.B, a.nIn, a.nOut, group, dtype, bad);
		return -1;
	}
	if (!a.B)
		return 0;
	const struct w4_layout l = w4_layout_of(a.nOut, a.nIn, group, dtype, zeros);
	const int nOut = a.nOut;
	const float *bias = a.bias;
	void *y = a.y;
	a.steps = l.steps;
	a.groups = l.groups;
	a.group = group;
	a.xgroups = xgroup ? l.groups : 1;
	a.dtype = dtype;
	a.shift = 31;
	for (int i = 5; i <= 8; i++)
		if (group == 1 << i)
			a.shift = i;
	ThhipLaunchScope scope(THHIP_FAM_GEMV, (double)a.nOut * a.nIn / 2 + (double)a.nOut * l.groups * (es + (zeros ? 1 : 0)) +
		(double)a.B * a.nIn * esx + (double)a.B * a.nOut * es);
	for (int o0 = 0; o0 < nOut; o0 += W4_OUTPUTS) {	/* (a grid of them has fewer than 2^32 threads) */
		const size_t rb = o0 / 16;
		a.nOut = nOut - o0 < W4_OUTPUTS ? nOut - o0 : W4_OUTPUTS;
		a.blocks = (a.nOut + 15) / 16;
		a.codes = (const unsigned char *)packed + rb * l.steps * 1024;
		a.scales = (const char *)packed + l.scales + rb * l.groups * 16 * es;
		a.zeros = zeros ? (const unsigned char *)packed + l.zeros + rb * l.groups * 16 : 0;
		a.bias = bias ? bias + o0 : 0;
		a.y = (char *)y + o0 * es;
		if (xkind == W4_X_I8)
			w4_choose<W4_X_I8>(a);
		else
			THHIP_DISPATCH_FLOAT(dtype, (w4_choose<DT>(a)));
	}
	return 0;
}

extern "C" int thhip_linear_w4(const void *x, long ldx, const void *wpacked, const float *bias, void *y, long ldy,
	int B, int nIn, int nOut, int group, int zeros, int act, float thr, float val, int dtype)
{
	w4_args a = {};
	a.x = x; a.ldx = ldx; a.bias = bias; a.y = y; a.ldy = ldy;
	a.B = B; a.nIn = nIn; a.nOut = nOut; a.act = act; a.thr = thr; a.val = val;
	return w4_run("thhip_linear_w4", a, wpacked, group, zeros, dtype, 0, dtype);
}

extern "C" int thhip_linear_w4_i8(const signed char *x, long ldx, const float *xscale, int xgroup, const void *wpacked,
	const float *bias, void *y, long ldy, int B, int nIn, int nOut, int group, int zeros, int act, float thr, float val,
	int dtype)
{
	w4_args a = {};
	a.x = x; a.ldx = ldx; a.xscale = xscale; a.bias = bias; a.y = y; a.ldy = ldy;
	a.B = B; a.nIn = nIn; a.nOut = nOut; a.act = act; a.thr = thr; a.val = val;
	return w4_run("thhip_linear_w4_i8", a, wpacked, group, zeros, W4_X_I8, xgroup, dtype);
}
