/*
 * Root-mean-square norm of rows with a residual's addition, and rows of signed
 * 8-bit codes with scales.
 *
 *   h = x + res                       (fp32; sum = h rounded to the type of x)
 *   y = h * w / sqrt(mean(h * h) + eps)
 *   scale = max|y| / 127,  q = rint(y / scale)          over a row or a group
 *
 * The reference has neither (its norm is nn_SpatialBatchNormalization_updateOutput,
 * modules/SpatialBatchNormalization.c:57-116, its 8-bit codes are unsigned with one
 * range for a tensor, lowp_basic.c:15-35): they belong to networks of Linear layers,
 * beside thhip_linear_w4 and thhip_linear_w4_i8.
 *
 * Bound by memory: every element is read once, kept in registers while the row's
 * sum of squares (and largest |h w|) goes through the wavefronts, and written once.
 * h stays in fp32 between the addition and the norm, so the norm is that of the
 * unrounded sum, and y is rounded once.  Codes do not depend on the root, only on
 * h w and its maximum; where the fp32 quotient is next to the middle between two
 * codes it is taken again in 64 bits, so that the value goes to the nearer one: without
 * that one value in 30000 of fp16 rows did not.
 *
 * Time alone on the GPU, us (a large copy moves 5.1 TB/s): norm of 16384 rows of 8192 bf16 with a residual 181 (1074 MB,
 * 5.9 TB/s), of 333 rows of 5003 fp32 5.4 (13 MB, 2.5 TB/s: half of it is the way of one row through the GPU, 2.4 us);
 * with codes 8192 rows of 4096 bf16 47 (235 MB, 5.0 TB/s); codes alone 700 rows of 9216 fp16 7.5 (19 MB, 2.6 TB/s).
 */
#include <stdint.h>
#include <stdio.h>
#include "thhip_internal.h"

enum { ROWS_NORM, ROWS_NORM_I8, ROWS_QUANT };

struct rows_args {
	const void *x, *res;
	const float *w;
	void *sum, *y;
	signed char *q;
	float *scale;
	long ldx, ldr, lds, ldy, ldq;
	long rows;
	int cols, group, ngroups, ragged;
	float eps;
};

/* N consecutive elements of a row (16 bytes), which need no more than the element's alignment here.
 * fetch() loads without a branch, so that all of a thread's loads are on their way together: a vector that the
 * row's end cuts or that lies behind it is read from the row's last N elements (cols >= N), and widen() puts
 * it right afterwards, elements past the end being 0.  With a branch round each load the compiler waited for one before
 * the next (8192 rows of 4096 bf16 with codes 56 us, without 47; codes of 700 rows of 9216 fp16 11.1 and 7.7). */
template <int DT> struct RowVec {
	static constexpr int N = DT == THHIP_F32 ? 4 : 8;
	typedef typename ThhipElem<DT>::T T;
	typedef T V __attribute__((ext_vector_type(N)));
	typedef V U __attribute__((aligned(sizeof(T))));
	static __device__ __forceinline__ V fetch(const void *p, long base, int col, int cols)
	{
		return *(const U *)((const T *)p + base + (col < cols - N ? col : cols - N));
	}
	/* ragged: the row has vectors that fetch() moved */
	static __device__ __forceinline__ void widen(const V v, int col, int cols, int ragged, float *out)
	{
#pragma unroll
		for (int i = 0; i < N; i++)
			out[i] = (float)v[i];
		if (ragged) {
			const int by = col > cols - N ? col - (cols - N) : 0;
#pragma unroll
			for (int b = 1; b < N; b *= 2)
#pragma unroll
				for (int i = 0; i < N; i++)
					out[i] = by & b ? (i + b < N ? out[i + b] : 0.0f) : out[i];
#pragma unroll
			for (int i = 0; i < N; i++)
				out[i] = by >= N ? 0.0f : out[i];
		}
	}
	/* the same for rows of any length */
	static __device__ __forceinline__ void load(const void *p, long base, int col, int cols, float *out)
	{
		if (col + N <= cols)
			widen(*(const U *)((const T *)p + base + col), col, cols, 0, out);
		else
#pragma unroll
			for (int i = 0; i < N; i++)
				out[i] = col + i < cols ? ThhipElem<DT>::ld(p, base + col + i) : 0.0f;
	}
	static __device__ __forceinline__ void store(void *p, long base, int col, int cols, const float *in)
	{
		if (col + N <= cols) {
			V v;
#pragma unroll
			for (int i = 0; i < N; i++)
				v[i] = (T)in[i];
			*(U *)((T *)p + base + col) = v;
		} else {
#pragma unroll
			for (int i = 0; i < N; i++)
				if (col + i < cols)
					ThhipElem<DT>::st(p, base + col + i, in[i]);
		}
	}
};

/* What a row's or group's values become codes by.  top is the largest |h w|, top * rstd the largest |y|: below
 * 2^-116 (where an fp32 scale loses bits) it counts as nothing, codes 0.  Near either end of the range 127 / top passes
 * fp32's largest number or 1 / top is a denormal, and products next to the lower end lose bits: there all codes are taken
 * in 64 bits. */
struct code_step {
	float top, inv;		/* inv: 127 / top, off by at most 1.5 units, or 0 */
	float sure;		/* a quotient this far from its code or further is taken again in 64 bits */
};

__device__ __forceinline__ struct code_step code_step_of(float top, float rstd)
{
	const bool none = top * rstd < 1.2e-35f, end = top < 0x1p-100f || (top > 0x1p125f && top < INFINITY);
	struct code_step c;
	c.top = top;
	c.inv = none || end ? 0.0f : 127.0f * __builtin_amdgcn_rcpf(top);	/* (a NaN stays one) */
	c.sure = none ? 1.0f : end ? -1.0f : 0.5f - 0x1p-14f;
	return c;
}

/* The codes of N values v * w.  Adding 1.5 * 2^23 leaves the nearest whole number in the sum's low bits.  The product v * w
 * and the reciprocal are off by at most 2^-24 and 3 * 2^-24, that is 3e-5 of a code at 127: a quotient that is
 * further than 2^-14 from a middle between two codes has its nearest one. */
template <int N>
__device__ __forceinline__ void store_codes(signed char *p, long base, int col, int cols, const float *v, const float *w,
	const struct code_step c)
{
	typedef unsigned W __attribute__((ext_vector_type(N / 4), aligned(1)));
	const float whole = 12582912.0f;
	unsigned o[N / 4], u[N];
	float off = 0;
#pragma unroll
	for (int i = 0; i < N; i++) {
		const float x = v[i] * w[i], y = fmaf(x, c.inv, whole);
		off = fmaxf(off, fabsf(fmaf(x, c.inv, whole - y)));
		u[i] = __float_as_uint(y);
	}
	if (off > c.sure) {
		/* v * w / step in 64 bits, by the reciprocal and what the product says is left */
		const double step = (double)c.top * (1.0 / 127.0);
		double inv = __builtin_amdgcn_rcp(step);
		inv = fma(fma(-step, inv, 1.0), inv, inv);
		inv = fma(fma(-step, inv, 1.0), inv, inv);
#pragma unroll
		for (int i = 0; i < N; i++) {
			const double x = (double)v[i] * (double)w[i], y = x * inv;
			const int n = (int)rint(fma(fma(-y, step, x), inv, y));
			u[i] = (unsigned)(n > 127 ? 127 : n < -127 ? -127 : n);
		}
	}
#pragma unroll
	for (int i = 0; i < N / 4; i++)
		o[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[4 * i + 3], u[4 * i + 2], 0x0c0c0400),
			__builtin_amdgcn_perm(u[4 * i + 1], u[4 * i], 0x0c0c0400), 0x05040100);
	if (col + N <= cols) {
		W r;
		if constexpr (N == 8)
			r = (W){o[0], o[1]};
		else
			r = (W)o[0];
		*(W *)(p + base + col) = r;
	} else if (col < cols) {
#pragma unroll
		for (int i = 0; i < N; i++)
			if (col + i < cols)
				p[base + col + i] = (signed char)u[i];
	}
}

/* |v| as an unsigned number: orders as |v| does, infinity above every number and a NaN above
 * infinity, so that a NaN reaches the scale of its row or group */
__device__ __forceinline__ unsigned abs_bits(float v)
{
	return __float_as_uint(v) & 0x7fffffffu;
}

/* (at most what 127 times of is a number: of FLT_MAX the nearest to top / 127 is not) */
__device__ __forceinline__ float code_scale(float top)
{
	const float s = top * (1.0f / 127.0f);
	return top < 1.2e-35f ? 0.0f : top < INFINITY ? fminf(fmaf(fmaf(-s, 127.0f, top), 1.0f / 127.0f, s), 0x1.020406p+121f) : s;
}

/* v of the lane that differs in bits `by` of its number (by = 1, 2), that is mirrored in its half row of 8 lanes (4) or row
 * of 16 (8), or in the other row or half of the wavefront (16, 32): a butterfly over `by` leaves every lane of a
 * group of lanes with the group's sum or maximum.  Moves between registers; through LDS (shuffles) a
 * row of 4096 took 0.1 to 0.3 us longer, of 3. */
template <int BY>
__device__ __forceinline__ unsigned lane_across(unsigned v)
{
	if constexpr (BY == 1)
		return __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, false);	/* quad_perm 1 0 3 2 */
	else if constexpr (BY == 2)
		return __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, false);	/* quad_perm 2 3 0 1 */
	else if constexpr (BY == 4)
		return __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false);	/* row_half_mirror */
	else if constexpr (BY == 8)
		return __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false);	/* row_mirror */
	else {
		/* swaps the odd rows (16) / upper half (32) of the first with the even rows / lower half of the second */
		const auto p = BY == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
		return threadIdx.x & BY ? p[0] : p[1];
	}
}

template <int BY = 32>
__device__ __forceinline__ float lanes_sum(float v)
{
	if constexpr (BY > 1)
		v = lanes_sum<BY / 2>(v);
	return v + __uint_as_float(lane_across<BY>(__float_as_uint(v)));
}

/* over groups of `lanes` lanes (a power of two, uniform) */
template <int BY = 32>
__device__ __forceinline__ unsigned lanes_max(unsigned v, int lanes)
{
	if constexpr (BY > 1)
		v = lanes_max<BY / 2>(v, lanes);
	if (BY < lanes) {
		const unsigned o = lane_across<BY>(v);
		v = o > v ? o : v;
	}
	return v;
}

/* Sum and maximum over the T threads of a row, T = 64 (a wavefront) or the whole workgroup */
template <int T>
__device__ __forceinline__ void row_reduce(float &s, unsigned &m)
{
	s = lanes_sum(s);
	m = lanes_max(m, 64);
	if constexpr (T > 64) {
		constexpr int W = T / 64;
		__shared__ float ps[W];
		__shared__ unsigned pm[W];
		if ((threadIdx.x & 63) == 0) {
			ps[threadIdx.x >> 6] = s;
			pm[threadIdx.x >> 6] = m;
		}
		__syncthreads();
		s = ps[0];
		m = pm[0];
#pragma unroll
		for (int i = 1; i < W; i++) {
			s += ps[i];
			m = pm[i] > m ? pm[i] : m;
		}
	}
}

/* The squares are fp32: where their mean (with eps) is past its largest number, as with a mask of the type's lowest value in the
 * row, or so small that squares have lost bits, the row is taken again times a power of two, eps with it.  (fp16 values
 * are never that large or small.) */
#define NORM_FACTOR(DT, MODE) (DT != THHIP_F16 && MODE != ROWS_QUANT)

__device__ __forceinline__ float norm_factor(float mean)
{
	const float f = mean < 0x1p-96f ? 0x1p96f : mean < INFINITY ? 1.0f : 0x1p-96f;
	return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(f)));
}

/* One vector of a row on its way out: y, or codes and (by the group's first lane) its scale */
template <int DT, int MODE>
__device__ __forceinline__ void row_out(const rows_args &a, long row, int col, const float *h, const float *w, float rstd,
	struct code_step step)
{
	constexpr int N = RowVec<DT>::N;
	if constexpr (MODE == ROWS_NORM) {
		float y[N];
#pragma unroll
		for (int i = 0; i < N; i++)
			y[i] = h[i] * rstd * w[i];
		RowVec<DT>::store(a.y, row * a.ldy, col, a.cols, y);
	} else {
		if (a.group) {
			unsigned m = 0;
#pragma unroll
			for (int i = 0; i < N; i++) {
				const unsigned b = abs_bits(MODE == ROWS_QUANT ? h[i] : h[i] * w[i]);
				m = b > m ? b : m;
			}
			m = lanes_max(m, a.group / N);
			const float top = __uint_as_float(m);
			step = code_step_of(top, rstd);
			if (col < a.cols && col % a.group == 0)
				a.scale[row * a.ngroups + col / a.group] = code_scale(top * rstd);
		}
		store_codes<N>(a.q, row * a.ldq, col, a.cols, h, w, step);
	}
}

/* Rows of at most T * V vectors, T threads a row, each of which keeps its V vectors in registers: a wavefront for rows of
 * up to two vectors a lane (four rows a workgroup, no barrier), 256 threads up to eight, so that several rows share a CU
 * and one's loads run under another's sums, 1024 beyond.  V = 5 and 6 as well as 4 and 8: the registers of unused vectors
 * are rows that do not fit beside (4096 rows of 9216 bf16, V = 8 and 5, us: norm 55 and 49, with codes 70 and 49); 3
 * and 7 changed nothing. */
template <int DT, int MODE, int T, int V>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rows_kernel(const rows_args a)
{
	constexpr int N = RowVec<DT>::N;
	constexpr int RPG = T < 256 ? 256 / T : 1;	/* rows a workgroup */
	const int t = threadIdx.x % T;
	const long row = (long)blockIdx.x * RPG + threadIdx.x / T;
	if (RPG > 1 && row >= a.rows)	/* (whole wavefronts: T = 64) */
		return;
	typedef RowVec<DT> R;
	typedef RowVec<THHIP_F32> R4;
	typename R::V rx[V], rr[V];
	typename R4::V rw[V][N / 4];
#pragma unroll
	for (int v = 0; v < V; v++)
		rx[v] = R::fetch(a.x, row * a.ldx, (v * T + t) * N, a.cols);
	if (a.res)
#pragma unroll
		for (int v = 0; v < V; v++)
			rr[v] = R::fetch(a.res, row * a.ldr, (v * T + t) * N, a.cols);
	if (MODE != ROWS_QUANT && a.w)
#pragma unroll
		for (int v = 0; v < V; v++)
#pragma unroll
			for (int i = 0; i < N / 4; i++)
				rw[v][i] = R4::fetch(a.w, 0, (v * T + t) * N + 4 * i, a.cols);
	float h[V][N], w[V][N];
#pragma unroll
	for (int v = 0; v < V; v++) {
		if (v && v * T * N >= a.cols)	/* (the whole vector lies behind the row) */
			break;
		const int col = (v * T + t) * N;
		R::widen(rx[v], col, a.cols, a.ragged, h[v]);
		if (a.res) {
			float r[N];
			R::widen(rr[v], col, a.cols, a.ragged, r);
#pragma unroll
			for (int i = 0; i < N; i++)
				h[v][i] += r[i];
		}
		if (MODE != ROWS_QUANT && a.w) {
#pragma unroll
			for (int i = 0; i < N / 4; i++)
				R4::widen(rw[v][i], col + 4 * i, a.cols, a.ragged, w[v] + 4 * i);
		} else {
#pragma unroll
			for (int i = 0; i < N; i++)
				w[v][i] = 1.0f;
		}
	}
	float s, rstd = 1, eps = a.eps;
	struct code_step step = {0, 0, 1};
	unsigned m;
	bool summed = false;	/* a.sum is written */
	auto sums = [&]() {
		s = 0;
		m = 0;
#pragma unroll
		for (int v = 0; v < V; v++) {
			if (v && v * T * N >= a.cols)
				break;
#pragma unroll
			for (int i = 0; i < N; i++) {
				if constexpr (MODE != ROWS_QUANT)
					s += h[v][i] * h[v][i];
				if constexpr (MODE != ROWS_NORM) {
					const unsigned b = abs_bits(MODE == ROWS_QUANT ? h[v][i] : h[v][i] * w[v][i]);
					m = b > m ? b : m;
				}
			}
		}
		if (MODE != ROWS_QUANT || !a.group)
			row_reduce<T>(s, m);
	};
	sums();
	if constexpr (NORM_FACTOR(DT, MODE)) {
		const float f = norm_factor(s / (float)a.cols + eps);
		if (f != 1.0f) {	/* (the same for the whole row) */
			summed = a.sum;
#pragma unroll
			for (int v = 0; v < V; v++) {
				if (v && v * T * N >= a.cols)
					break;
				if (a.sum)
					RowVec<DT>::store(a.sum, row * a.lds, (v * T + t) * N, a.cols, h[v]);
#pragma unroll
				for (int i = 0; i < N; i++)
					h[v][i] *= f;
			}
			eps = eps * f * f;
			if (T > 64)
				__syncthreads();	/* row_reduce's LDS is used again */
			sums();
		}
	}
	if constexpr (MODE != ROWS_QUANT)
		rstd = 1.0f / sqrtf(s / (float)a.cols + eps);
	if constexpr (MODE != ROWS_NORM) {
		if (!a.group) {
			step = code_step_of(__uint_as_float(m), rstd);
			if (t == 0)
				a.scale[row] = code_scale(__uint_as_float(m) * rstd);
		}
	}
#pragma unroll
	for (int v = 0; v < V; v++) {
		if (v && v * T * N >= a.cols)
			break;
		const int col = (v * T + t) * N;
		if (a.sum && !summed)
			RowVec<DT>::store(a.sum, row * a.lds, col, a.cols, h[v]);
		row_out<DT, MODE>(a, row, col, h[v], w[v], rstd, step);
	}
}

/* Rows longer than the registers hold, or shorter than a vector: the sum (and maximum) first, then the row again.  A thread
 * reads an element of x and res in the second walk before it writes the same element, so the outputs
 * may be the inputs here too. */
template <int DT, int MODE>
__global__ __launch_bounds__(1024) void rows_long_kernel(const rows_args a)
{
	constexpr int N = RowVec<DT>::N, T = 1024;
	const long row = blockIdx.x;
	const int t = threadIdx.x;
	const int steps = (a.cols - 1) / (T * N) + 1;
	float h[N], w[N], r[N], s = 0, rstd = 1, f = 1, eps = a.eps;
	struct code_step step = {0, 0, 1};
	unsigned m = 0;
	for (int walk = 0; walk < 2; walk++) {
		for (int v = 0; v < steps; v++) {
			const int col = (v * T + t) * N;
			RowVec<DT>::load(a.x, row * a.ldx, col, a.cols, h);
			if (a.res) {
				RowVec<DT>::load(a.res, row * a.ldr, col, a.cols, r);
#pragma unroll
				for (int i = 0; i < N; i++)
					h[i] += r[i];
			}
#pragma unroll
			for (int i = 0; i < N; i++)
				w[i] = MODE != ROWS_QUANT && a.w && col + i < a.cols ? a.w[col + i] : 1.0f;
			if (walk == 1 && a.sum)
				RowVec<DT>::store(a.sum, row * a.lds, col, a.cols, h);
			if constexpr (NORM_FACTOR(DT, MODE))
#pragma unroll
				for (int i = 0; i < N; i++)
					h[i] *= f;
			if (walk == 0) {
#pragma unroll
				for (int i = 0; i < N; i++) {
					s += h[i] * h[i];
					const unsigned b = abs_bits(h[i] * w[i]);
					m = b > m ? b : m;
				}
			} else
				row_out<DT, MODE>(a, row, col, h, w, rstd, step);
		}
		if (walk == 0) {
			row_reduce<T>(s, m);
			if constexpr (NORM_FACTOR(DT, MODE))
				if (f == 1.0f) {
					f = norm_factor(s / (float)a.cols + eps);
					if (f != 1.0f) {	/* (the same for the whole row) */
						eps = eps * f * f;
						s = 0;
						m = 0;
						walk = -1;
						__syncthreads();	/* row_reduce's LDS is used again */
						continue;
					}
				}
			if constexpr (MODE != ROWS_QUANT)
				rstd = 1.0f / sqrtf(s / (float)a.cols + eps);
			if constexpr (MODE != ROWS_NORM) {
				if (!a.group) {
					step = code_step_of(__uint_as_float(m), rstd);
					if (t == 0)
						a.scale[row] = code_scale(__uint_as_float(m) * rstd);
				}
			}
		}
	}
}

template <int DT, int MODE, int T, int V>
static bool rows_try(rows_args &a)
{
	if (a.cols > T * V * RowVec<DT>::N || a.cols < RowVec<DT>::N)
		return false;
	a.ragged = a.cols != T * V * RowVec<DT>::N;
	constexpr int RPG = T < 256 ? 256 / T : 1;
	rows_kernel<DT, MODE, T, V><<<dim3((unsigned)((a.rows + RPG - 1) / RPG)), dim3(T < 256 ? 256 : T), 0, thhip_stream()>>>(a);
	return true;
}

template <int DT, int MODE>
static void rows_launch(rows_args &a)
{
	if (rows_try<DT, MODE, 64, 1>(a) || rows_try<DT, MODE, 64, 2>(a) || rows_try<DT, MODE, 256, 1>(a) ||
	    rows_try<DT, MODE, 256, 2>(a) || rows_try<DT, MODE, 256, 4>(a) || rows_try<DT, MODE, 256, 5>(a) ||
	    rows_try<DT, MODE, 256, 6>(a) || rows_try<DT, MODE, 256, 8>(a) ||
	    rows_try<DT, MODE, 1024, 4>(a))
		return;
	rows_long_kernel<DT, MODE><<<dim3((unsigned)a.rows), dim3(1024), 0, thhip_stream()>>>(a);
}

/* A launch has fewer than 2^32 threads: rows beyond this many go into further launches */
#define ROWS_A_LAUNCH (1l << 21)

/* What is wrong with a call, or NULL; fills in what the kernels derive from the arguments */
static const char *rows_check(rows_args &a, long rows, long cols, int dtype, int mode)
{
	if (dtype != THHIP_F32 && dtype != THHIP_F16 && dtype != THHIP_BF16)
		return "the type of x is fp32, fp16 or bf16";
	if (rows < 0 || cols < 1 || cols > 0x3fffffffl)
		return "rows of 1 to 2^30 - 1 columns";
	const size_t es = thhip_esize(dtype);
	if (rows && (!a.x || (mode == ROWS_NORM ? !a.y : !a.q || !a.scale)))
		return "x and the outputs are needed";
	if (a.ldx < cols || (a.res && a.ldr < cols) || (a.sum && a.lds < cols) || (a.y && a.ldy < cols) || (a.q && a.ldq < cols))
		return "a row stride is smaller than the row";
	if ((uintptr_t)a.x % es || (uintptr_t)a.res % es || (uintptr_t)a.sum % es || (uintptr_t)a.y % es ||
	    (uintptr_t)a.w % 4 || (uintptr_t)a.scale % 4)
		return "a pointer is not aligned to its element";
	if (mode != ROWS_NORM && a.group != 0 && a.group != 32 && a.group != 64 && a.group != 128 && a.group != 256)
		return "a group has 32, 64, 128 or 256 columns, or is the row (0)";
	a.rows = rows;
	a.cols = (int)cols;
	a.ngroups = a.group ? (int)((cols + a.group - 1) / a.group) : 1;
	return 0;
}

static double rows_bytes(const rows_args &a, int dtype)
{
	const double n = (double)a.rows * a.cols, es = thhip_esize(dtype);
	return n * es * (1 + !!a.res + !!a.sum + !!a.y) + (a.w ? 4.0 * a.cols : 0) +
		(a.q ? n + 4.0 * a.rows * a.ngroups : 0);
}

static int rows_run(const char *who, rows_args &a, long rows, long cols, int dtype, int mode)
{
	const char *bad = rows_check(a, rows, cols, dtype, mode);
	if (bad) {
		fprintf(stderr, "%s: %ld x %ld, dtype %d, group %d: %s\n", who, rows, cols, dtype, a.group, bad);
		return -1;
	}
	if (!rows)
		return 0;
	ThhipLaunchScope scope(THHIP_FAM_OTHER, rows_bytes(a, dtype));
	const size_t es = thhip_esize(dtype);
	while (rows > 0) {
		a.rows = rows < ROWS_A_LAUNCH ? rows : ROWS_A_LAUNCH;
		if (mode == ROWS_NORM)
			THHIP_DISPATCH_FLOAT(dtype, (rows_launch<DT, ROWS_NORM>(a)));
		else if (mode == ROWS_NORM_I8)
			THHIP_DISPATCH_FLOAT(dtype, (rows_launch<DT, ROWS_NORM_I8>(a)));
		else
			THHIP_DISPATCH_FLOAT(dtype, (rows_launch<DT, ROWS_QUANT>(a)));
		rows -= a.rows;
		a.x = (const char *)a.x + a.rows * a.ldx * es;
		a.res = a.res ? (const char *)a.res + a.rows * a.ldr * es : 0;
		a.sum = a.sum ? (char *)a.sum + a.rows * a.lds * es : 0;
		a.y = a.y ? (char *)a.y + a.rows * a.ldy * es : 0;
		a.q = a.q ? a.q + a.rows * a.ldq : 0;
		a.scale = a.scale ? a.scale + a.rows * a.ngroups : 0;
	}
	return 0;
}

extern "C" int thhip_rmsnorm(const void *x, long ldx, const void *res, long ldr, const float *weight, float eps,
	void *sum, long lds, void *y, long ldy, long rows, long cols, int dtype)
{
	rows_args a = {};
	a.x = x; a.ldx = ldx; a.res = res; a.ldr = ldr; a.w = weight; a.eps = eps;
	a.sum = sum; a.lds = lds; a.y = y; a.ldy = ldy;
	return rows_run("thhip_rmsnorm", a, rows, cols, dtype, ROWS_NORM);
}

extern "C" int thhip_rmsnorm_i8(const void *x, long ldx, const void *res, long ldr, const float *weight, float eps,
	void *sum, long lds, signed char *q, long ldq, float *qscale, int group, long rows, long cols, int dtype)
{
	rows_args a = {};
	a.x = x; a.ldx = ldx; a.res = res; a.ldr = ldr; a.w = weight; a.eps = eps;
	a.sum = sum; a.lds = lds; a.q = q; a.ldq = ldq; a.scale = qscale; a.group = group;
	return rows_run("thhip_rmsnorm_i8", a, rows, cols, dtype, ROWS_NORM_I8);
}

extern "C" int thhip_quantize_rows(const void *x, long ldx, signed char *q, long ldq, float *qscale, int group,
	long rows, long cols, int dtype)
{
	rows_args a = {};
	a.x = x; a.ldx = ldx; a.q = q; a.ldq = ldq; a.scale = qscale; a.group = group;
	return rows_run("thhip_quantize_rows", a, rows, cols, dtype, ROWS_QUANT);
}

/* y = q * scale.  segs times tx threads (a power of two) walk a row eight columns at a time; a group is a whole
 * number of such vectors.  Few long rows are shared by several workgroups (100 rows of 40000 to fp32 10.6 -> 6.1 us); two
 * vectors a thread for every row took longer where there are many rows (700 of 9216 5.1 -> 6.1).  Bound by memory: 8192 rows of 4096 to bf16 16.7 us (101 MB, 6.0 TB/s), 700 of 9216 to fp16
 * 6.0 us (19 MB, 3.2 TB/s). */
template <int DT>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const signed char *q, long ldq, const float *scale, int group,
	int ngroups, void *y, long ldy, long rows, int cols, int tx, unsigned segs)
{
	typedef unsigned W __attribute__((ext_vector_type(2), aligned(1)));
	const long row = (long)(blockIdx.x / segs) * (256 / tx) + threadIdx.x / tx;
	if (row >= rows)
		return;
	for (long c = ((long)(blockIdx.x % segs) * tx + (threadIdx.x & (tx - 1))) * 8; c < cols; c += (long)segs * tx * 8) {
		const int col = (int)c;
		const float s = scale[row * ngroups + (group ? col / group : 0)];
		float v[8];
		if (col + 8 <= cols) {
			const W w = *(const W *)(q + row * ldq + col);
#pragma unroll
			for (int i = 0; i < 8; i++)
				v[i] = (float)(signed char)(w[i / 4] >> (8 * (i % 4)));
		} else {
#pragma unroll
			for (int i = 0; i < 8; i++)
				v[i] = col + i < cols ? (float)q[row * ldq + col + i] : 0.0f;
		}
#pragma unroll
		for (int i = 0; i < 8; i++)
			v[i] *= s;
#pragma unroll
		for (int i = 0; i < 8; i += RowVec<DT>::N)
			RowVec<DT>::store(y, row * ldy, col + i, cols, v + i);
	}
}

extern "C" int thhip_dequantize_rows(const signed char *q, long ldq, const float *qscale, int group, void *y, long ldy,
	long rows, long cols, int dtype)
{
	rows_args a = {};
	a.x = y; a.ldx = ldy; a.q = (signed char *)q; a.ldq = ldq; a.scale = (float *)qscale; a.group = group;
	const char *bad = rows_check(a, rows, cols, dtype, ROWS_QUANT);
	if (bad) {
		fprintf(stderr, "thhip_dequantize_rows: %ld x %ld, dtype %d, group %d: %s\n", rows, cols, dtype, group, bad);
		return -1;
	}
	if (!rows)
		return 0;
	int tx = 1;
	while (tx < 256 && tx * 8 < cols)
		tx *= 2;
	/* about four workgroups a CU, and at least one vector a thread */
	const long each = (cols - 1) / (tx * 8) + 1, want = 1024 / rows;
	const unsigned segs = tx < 256 || want <= 1 ? 1 : (unsigned)(want < each ? want : each);
	ThhipLaunchScope scope(THHIP_FAM_OTHER, (double)rows * cols * (1 + thhip_esize(dtype)) + 4.0 * rows * a.ngroups);
	for (long r = 0; r < rows; r += ROWS_A_LAUNCH) {
		const long n = rows - r < ROWS_A_LAUNCH ? rows - r : ROWS_A_LAUNCH;
		const unsigned grid = (unsigned)((n + 256 / tx - 1) / (256 / tx)) * segs;
		THHIP_DISPATCH_FLOAT(dtype, (dequantize_rows_kernel<DT><<<dim3(grid), dim3(256), 0, thhip_stream()>>>(q + r * ldq, ldq,
			qscale + r * a.ngroups, group, a.ngroups, (char *)y + r * ldy * thhip_esize(dtype), ldy, n, (int)cols, tx, segs)));
	}
	return 0;
}
