/*
 * 4-bit Linear layers (linear_w4.hip) for larger batches: bound by the matrix cores and by the instructions between
 * theirs, of which a wavefront issues one where it could issue a matrix instruction (codes to operands, a group's sums to
 * the result).  4096 x 8192 -> 8192, us and 10^12 a second: fp16 485 to 505 and 1110, bf16 488 to 518 and 1090 (a library's
 * product of 8192^3: 1150 and 1201), 8-bit x 342 to 350 and 1590 (1779); 2048 rows of fp32 x 696 to 733 and 390 (149).
 * Groups of 64 and 32 take 560 and 680 (bf16), rows that are not whole vectors (4096 x 8190) 578 (fp16).
 *
 * A workgroup of four wavefronts computes 128 rows for BN columns (eight 256 rows: fp32 x), a wavefront 32 rows: each code
 * becomes an operand once (with 64 rows x BN / 2 a wavefront, twice: fp16 550 us).  All operands are n - z, so that no sum
 * of x is needed beside the products.  x goes through LDS a step of 128 k at a time (two buffers); codes go from memory to
 * registers, one step ahead, and become operands there: those of a whole step stay (32 registers) while its columns
 * are walked 16 at a time, so that the sums of one group of 16 columns (of two, the last one's being added to the result
 * while the next are multiplied) are all there is beside the result, which a group's end costs one multiply-add a value.
 * fp32 x is three planes of bf16 in LDS (BN = 64); 8-bit x is multiplied 64 k at a time (32 for groups of 32).
 * LDS rows are 128 k of a column; a 16-byte vector v of row r lies in slot v ^ r % 16 (8-bit x: v ^ r / 2 % 8),
 * which puts the 16 columns of an operand on different banks.  DMA: rows that memory holds in whole, aligned
 * 16-byte vectors are loaded straight into LDS; others go through registers.
 * One barrier a step: what is read of a step's buffers (x, scales, zeros) is read before the barrier at its end, and written
 * again for the step after next behind that barrier.
 * KS: where there are fewer tiles than CUs, eight wavefronts share a tile, four taking every other step of K.
 * Instructions of 32 x 32 outputs in place of 16 x 16 took as long (fp16 490 -> 504 us, 8-bit x 342 -> 384): what they
 * save in issue they need in registers, of which 8-bit x then has too few for a third workgroup.
 */
#include <stdint.h>
#include <type_traits>
#include "linear_w4.h"

template <int X, bool WIDE> struct W4Tile {		/* operands of 32 k, of weights n - z for every kind of x */
	typedef typename std::conditional<W4X<X>::ZIN, W4X<X>, W4Signed>::type K;
	typedef typename W4X<X>::V V;
	typedef typename W4X<X>::A A;
	static constexpr int MK = 32;
	static __device__ __forceinline__ unsigned zero(int z) { return K::zero(z); }
	static __device__ __forceinline__ V weights(const uintx4 &c, int j, unsigned z) { return K::weights(c[j], z); }
	static __device__ __forceinline__ A mma(V a, V b, A c) { return W4X<X>::mma(a, b, c); }
	/* at: the row's address; r: the row in the tile; q: lane / 16 */
	static __device__ __forceinline__ V read(const unsigned char *at, int r, int j, int q)
	{
		if constexpr (X == W4_X_I8)
			return *(const V *)(at + (((2 * j + (q >> 1)) ^ (r >> 1 & 7)) * 16 + (q & 1) * 8));
		else
			return *(const V *)(at + ((4 * j + q) ^ (r & 15)) * 16);
	}
};

template <> struct W4Tile<W4_X_I8, true> {		/* 8-bit operands of 64 k: two of 32 side by side */
	typedef intx4 V;
	typedef intx4 A;
	typedef W4Tile<W4_X_I8, false> H;
	static constexpr int MK = 64;
	static __device__ __forceinline__ unsigned zero(int z) { return H::zero(z); }
	static __device__ __forceinline__ V join(long lo, long hi)
	{
		return (V){(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
	}
	static __device__ __forceinline__ V weights(const uintx4 &c, int j, unsigned z) { return join(H::weights(c, 2 * j, z), H::weights(c, 2 * j + 1, z)); }
	static __device__ __forceinline__ A mma(V a, V b, A c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
	static __device__ __forceinline__ V read(const unsigned char *at, int r, int j, int q)
	{
		return join(H::read(at, r, 2 * j, q), H::read(at, r, 2 * j + 1, q));
	}
};

#define W4_LDS(p) ((__attribute__((address_space(3))) void *)(p))

/* A scale, in the type of x or, where x is 8-bit, in the one the call names */
template <int X>
__device__ __forceinline__ float w4_get(const void *p, long i, int dtype)
{
	if constexpr (X != W4_X_I8)
		return ThhipElem<X>::ld(p, i);
	else {
		const unsigned u = dtype == THHIP_F32 ? ((const unsigned *)p)[i] : (unsigned)((const unsigned short *)p)[i];
		const float h = (float)__builtin_bit_cast(_Float16, (unsigned short)u);
		return dtype == THHIP_F16 ? h : __uint_as_float(dtype == THHIP_F32 ? u : u << 16);
	}
}

/* Wavefronts of a SIMD: with 8-bit x LDS has room for three workgroups (4096 x 8192 -> 8192, us: 387 with two, 352), with
 * fp32 x for one of four or eight */
constexpr int w4_tile_waves(int x, bool dma, int ks, int threads)
{
	return x == W4_X_I8 && dma && ks == 1 ? 3 : x == THHIP_F32 && threads == 256 ? 1 : 2;
}

template <int X, int GM, bool ZP, bool XG, bool DMA, int KS, int TH>
__global__ __launch_bounds__(KS * TH) __attribute__((amdgpu_waves_per_eu(w4_tile_waves(X, DMA, KS, TH), w4_tile_waves(X, DMA, KS, TH)))) void w4_tile_kernel(const w4_args a, int mtiles, int ntiles)
{
	typedef W4X<X> K;
	typedef W4Tile<X, X == W4_X_I8 && GM >= 2> M;
	typedef typename M::V V;
	typedef typename M::A A;
	constexpr int PARTS = K::PARTS, BN = PARTS > 1 ? 64 : 128;
	/* row blocks of a wavefront, and blocks of 16 columns */
	constexpr int BM = TH / 2, R = 2, NB = BN / 16;
	constexpr int ES = sizeof(typename K::V) / 8;
	constexpr int ROW = W4_KSTEP * ES;			/* bytes of a row in LDS */
	constexpr int PLANE = BN * ROW, STAGE = PARTS * PLANE;
	constexpr int NJ = W4_KSTEP / M::MK, GJ = GM * 32 / M::MK;	/* matrix instructions of a step, of a group */
	constexpr int PIECES = BN * 16 / TH;			/* vectors of eight k a thread moves a step */
	constexpr int NG = 4 / GM;				/* groups of a step */
	/* One array: between the loads into LDS and reads of another array the compiler waits for all of the loads.  x; the
	 * BM rows' scales of a step's groups; zeros as zero() makes them; and the scales of x where a row has several */
	constexpr int SCALES = 2 * NG * BM * 4, ZEROS = ZP ? SCALES : 0, XSCALES = XG ? SCALES : 0;
	__shared__ __align__(16) unsigned char all_lds[KS * (2 * STAGE + SCALES + ZEROS + XSCALES)];
	const int part = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;	/* the wavefronts of one take every KS-th step */
	const int tid = threadIdx.x & (TH - 1), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	unsigned char *lds = all_lds + part * (2 * STAGE + SCALES + ZEROS + XSCALES);
	float (*lscale)[NG][BM] = (float (*)[NG][BM])(lds + 2 * STAGE);
	unsigned (*lzero)[NG][BM] = (unsigned (*)[NG][BM])(lds + 2 * STAGE + SCALES);
	float (*lxs)[NG][BN] = (float (*)[NG][BN])(lds + 2 * STAGE + SCALES + ZEROS);
	const int col = lane & 15, quarter = lane >> 4;

	/* the tiles of an XCD (workgroups b, b + 8, ...) are neighbours, in columns of eight row tiles */
	int id = blockIdx.x;
	{
		const int total = mtiles * ntiles, per = total / 8;
		if (id < per * 8)
			id = (id & 7) * per + (id >> 3);
		const int band = 8 * ntiles, m0 = id / band * 8, left = mtiles - m0 < 8 ? mtiles - m0 : 8;
		const int in = id - id / band * band;
		id = (m0 + in % left) * ntiles + in / left;
	}
	const int mt = id / ntiles, nt = id - mt * ntiles;
	const int b0 = nt * BN, nrows = a.B - b0 < BN ? a.B - b0 : BN;
	const int wrow = wave % (BM / 16 / R), rb0 = mt * (BM / 16) + wrow * R, c0 = wave / (BM / 16 / R) * NB * 16;

	const typename K::E *xbase = (const typename K::E *)a.x + (long)b0 * a.ldx;
	const unsigned xend = DMA ? (unsigned)(((nrows - 1) * a.ldx + a.nIn) * (long)sizeof(typename K::E)) : 0;
	const __amdgpu_buffer_rsrc_t xrsrc = __builtin_amdgcn_make_buffer_rsrc((void *)xbase, 0, xend, 0x00020000);
	typename K::E8 xr[DMA ? 1 : PIECES / 2];

	/* x of step t on its way (half: one of the two halves that go through registers one after the other) */
	auto x_issue = [&](int t, int buf, int half) {
		if constexpr (DMA) {
			constexpr int VROW = ROW / 16, RPI = 64 / VROW;	/* vectors of a row; rows a wavefront's load covers */
			const int r0 = wave * RPI + lane / VROW, slot = lane % VROW;
			const int v = ES == 1 ? slot ^ (r0 >> 1 & 7) : slot ^ (r0 & 15);
			const int k = t * ROW + v * 16;		/* (bytes) */
			/* (the whole offset in the vector operand: a scalar one is no part of the bounds check that keeps
			 * rows behind the last from being read) */
#pragma unroll
			for (int i = 0; i < BN / (4 * RPI); i++) {
				__builtin_amdgcn_raw_ptr_buffer_load_lds(xrsrc, W4_LDS(lds + buf * STAGE + (i * 4 + wave) * 1024), 16,
					(k < a.nIn * ES ? (unsigned)(r0 * (int)a.ldx * ES + k) : 0x80000000u) + i * 4 * RPI * (int)a.ldx * ES, 0, 0, 0);
			}
		} else {
			w4_fetch_x<X, false>(xr, xbase, a.ldx, a.nIn, t * W4_KSTEP + (tid & 15) * 8, [&](int i) {
				const int r = (tid + (half * (PIECES / 2) + i) * TH) >> 4;
				return (long)(r < nrows ? r : nrows - 1);
			});
		}
	};
	auto x_land = [&](int t, int buf, int half) {
		if constexpr (!DMA) {
			if ((t + 1) * W4_KSTEP > a.nIn)
				w4_fix_x<X>(xr, a.nIn, t * W4_KSTEP + (tid & 15) * 8);
#pragma unroll
			for (int i = 0; i < PIECES / 2; i++) {
				const int p = tid + (half * (PIECES / 2) + i) * TH, r = p >> 4, v = p & 15;
				typename K::V o[PARTS];
				K::operand(xr[i], o);
				const int to = ES == 1 ? ((v >> 1) ^ (r >> 1 & 7)) * 16 + (v & 1) * 8 : (v ^ (r & 15)) * 16;
#pragma unroll
				for (int q = 0; q < PARTS; q++)
					*(typename K::V *)(lds + buf * STAGE + q * PLANE + r * ROW + to) = o[q];
			}
		}
	};
	/* scales and zeros: thread i fetches row i % BM's, and puts them into LDS at the end of the step */
	float gs[NG], gx[NG];
	unsigned char gz[NG];
	const int gb = mt * (BM / 16) + (tid >> 4 & (BM / 16 - 1)), grb = gb < a.blocks ? gb : a.blocks - 1;
	auto g_issue = [&](int t) {
#pragma unroll
		for (int g = 0; g < NG; g++) {
			const long at = ((long)grb * a.groups + a.group_of(t, g * GM)) * 16 + (tid & 15);
			gs[g] = w4_get<X>(a.scales, at, a.dtype);
			if constexpr (ZP)
				gz[g] = a.zeros[at];
			if constexpr (XG)
				gx[g] = a.xscale[(long)(b0 + ((tid & 127) < nrows ? tid & 127 : 0)) * a.xgroups + a.group_of(t, g * GM)];
		}
	};
	auto g_land = [&](int buf) {
#pragma unroll
		for (int g = 0; g < NG; g++) {
			lscale[buf][g][tid & (BM - 1)] = gs[g];
			if constexpr (ZP)
				lzero[buf][g][tid & (BM - 1)] = M::zero(gz[g]);
			if constexpr (XG)
				lxs[buf][g][tid & 127] = gx[g];
		}
	};
	uintx4 codes[R];
	auto codes_issue = [&](int t) {
#pragma unroll
		for (int r = 0; r < R; r++) {
			const int rb = rb0 + r < a.blocks ? rb0 + r : a.blocks - 1;
			codes[r] = *(const uintx4 *)(a.codes + ((size_t)rb * a.steps + t) * 1024 + lane * 16);
		}
	};
	/* (the loads into LDS are not the compiler's to wait for) */
	auto barrier = [&]() {
		asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
	};

	floatx4 acc[R][NB];
#pragma unroll
	for (int r = 0; r < R; r++)
#pragma unroll
		for (int n = 0; n < NB; n++)
			acc[r][n] = (floatx4)0.0f;

	const int first = part < a.steps ? part : a.steps - 1;
	x_issue(first, 0, 0);
	x_land(first, 0, 0);
	if (!DMA) {
		x_issue(first, 0, 1);
		x_land(first, 0, 1);
	}
	codes_issue(first);
	g_issue(first);
	g_land(0);
	barrier();

	constexpr int NU = NB * NG;		/* units of a step: 16 columns x one group */
	/* a unit's sums are added to the result while the next unit is multiplied (with eight wavefronts of fp32 x the other one of
	 * a SIMD multiplies meanwhile: 2048 x 8192 -> 8192 696 us so, 700 with it) */
	constexpr bool PIPE = DMA || (X == THHIP_F32 && TH == 256);
	const int own = wrow * R * 16 + col;	/* the lane's row of the first row block */
	A p[PIPE ? 2 : 1][R];
	/* the scales that unit u's sums take, from where its step's are */
	struct unit_scales {
		float w[R];
		floatx4 x;
	};
	auto scales_of = [&](int u, int buf) {
		unit_scales s;
#pragma unroll
		for (int r = 0; r < R; r++)
			s.w[r] = lscale[buf][u % NG][own + r * 16];
		if constexpr (XG)
			s.x = *(const floatx4 *)&lxs[buf][u % NG][c0 + u / NG * 16 + 4 * quarter];
		return s;
	};
	/* unit u's finished sums into the result */
	auto flush = [&](int u, const unit_scales &s) {
		const int n = u / NG;
#pragma unroll
		for (int r = 0; r < R; r++) {
#pragma unroll
			for (int i = 0; i < 4; i++)
				acc[r][n][i] += (XG ? s.w[r] * s.x[i] : s.w[r]) * (float)p[PIPE ? u & 1 : 0][r][i];
			/* (here, not at the end of the step, where the compiler would gather all n's sums) */
			asm("" : "+v"(acc[r][n]));
		}
	};
	/* A step's last sums are added at the start of the next, with scales read before the barrier between the two: behind it
	 * another wavefront may already have put the scales of the step after into that buffer. */
	constexpr bool LATE = PIPE && KS == 1 && NG == 1 && PARTS == 1;
	unit_scales late;
	const int rounds = (a.steps + KS - 1) / KS;
	for (int i = 0; i < rounds; i++) {
		const int t = i * KS + part, buf = i & 1, t1 = t + KS < a.steps ? t + KS : a.steps - 1;
		if (KS > 1 && t >= a.steps) {	/* (one step fewer than the others) */
			barrier();
			break;
		}
		const unsigned char *base = lds + buf * STAGE + (c0 + col) * ROW;
		V w[R][NJ], x[2][PARTS][NJ];
		auto x_read = [&](int n) {
#pragma unroll
			for (int q = 0; q < PARTS; q++)
#pragma unroll
				for (int j = 0; j < NJ; j++)
					x[n & 1][q][j] = M::read(base + q * PLANE + n * 16 * ROW, col, j, quarter);
		};
		__builtin_amdgcn_s_setprio(0);
		x_issue(t1, buf ^ 1, 0);
		x_read(0);
#pragma unroll
		for (int g = 0; g < NG; g++)
#pragma unroll
			for (int r = 0; r < R; r++) {
				const unsigned z = ZP ? lzero[buf][g][own + r * 16] : M::zero(8);
#pragma unroll
				for (int j = 0; j < GJ; j++)
					w[r][g * GJ + j] = M::weights(codes[r], g * GJ + j, z);
			}
		if (LATE && i > 0)
			flush(NU - 1, late);
		codes_issue(t1);
		g_issue(t1);
		__builtin_amdgcn_s_setprio(1);
#pragma unroll
		for (int u = 0; u < NU; u++) {
			const int n = u / NG, g = u % NG;
			asm volatile("" ::: "memory");	/* (operands and scales are read again for every unit, not kept) */
			__builtin_amdgcn_sched_barrier(0);
			if (!DMA && u == NU / 2) {
				x_land(t1, buf ^ 1, 0);
				x_issue(t1, buf ^ 1, 1);
			}
			if (g == 0 && n + 1 < NB)
				x_read(n + 1);
#pragma unroll
			for (int r = 0; r < R; r++)
				p[PIPE ? u & 1 : 0][r] = (A)0;
#pragma unroll
			for (int i = 0; i < GJ; i++) {
				const int j = g * GJ + i;
#pragma unroll
				for (int q = 0; q < PARTS; q++)
#pragma unroll
					for (int r = 0; r < R; r++)
						p[PIPE ? u & 1 : 0][r] = M::mma(x[n & 1][q][j], w[r][j], p[PIPE ? u & 1 : 0][r]);
			}
			if (PIPE ? u > 0 : true)
				flush(PIPE ? u - 1 : u, scales_of(PIPE ? u - 1 : u, buf));
			if constexpr (PIPE && (X == THHIP_F16 || X == THHIP_BF16)) {
			/* the order to issue them in: what comes from LDS, then a matrix instruction and the sums' work in turn */
			__builtin_amdgcn_sched_group_barrier(0x100, PARTS * NJ + R, 0);
#pragma unroll
			for (int i = 0; i < R * GJ * PARTS; i++) {
				__builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
				__builtin_amdgcn_sched_group_barrier(0x2, 1, 0);
			}
			}
		}
		if (PIPE && !LATE)
			flush(NU - 1, scales_of(NU - 1, buf));
		if (LATE)
			late = scales_of(NU - 1, buf);
		__builtin_amdgcn_sched_barrier(0);
		x_land(t1, buf ^ 1, DMA ? 0 : 1);
		g_land(buf ^ 1);
		barrier();
	}
	if (LATE)
		flush(NU - 1, late);
	if constexpr (KS > 1) {		/* the parts of K, added in their order */
		floatx4 *sums = (floatx4 *)all_lds;
		barrier();
#pragma unroll
		for (int p = 1; p < KS; p++)
			if (part == p)
#pragma unroll
				for (int r = 0; r < R; r++)
#pragma unroll
					for (int n = 0; n < NB; n++)
						sums[(((p - 1) * R + r) * NB + n) * TH + tid] = acc[r][n];
		barrier();
		if (part)
			return;
#pragma unroll
		for (int p = 1; p < KS; p++)
#pragma unroll
			for (int r = 0; r < R; r++)
#pragma unroll
				for (int n = 0; n < NB; n++)
					acc[r][n] += sums[(((p - 1) * R + r) * NB + n) * TH + tid];
	}

#pragma unroll
	for (int r = 0; r < R; r++) {
		const int o = (rb0 + r) * 16 + col;
		const float bias = a.bias && o < a.nOut ? a.bias[o] : 0.0f;
#pragma unroll
		for (int n = 0; n < NB; n++)
#pragma unroll
			for (int i = 0; i < 4; i++) {
				const int b = b0 + c0 + n * 16 + 4 * quarter + i;
				if (b < a.B && o < a.nOut) {
					float y = acc[r][n][i] * (X == W4_X_I8 && !XG ? a.xscale[b] : 1.0f / K::UNIT) + bias;
					if (a.act)
						y = y > a.thr ? y : a.val;
					w4_put<X>(a.y, b * a.ldy + o, y, a.dtype);
				}
			}
	}
}

/* A launch has at most this many rows of x, so that a grid stays below 2^32 threads */
#define W4_TILE_ROWS (1 << 20)

template <int X, int GM, bool XG>
static void w4_tile_launch(const w4_args &all)
{
	constexpr size_t esx = sizeof(typename W4X<X>::E);
	const size_t esy = thhip_esize(all.dtype);
	constexpr int BN = W4X<X>::PARTS > 1 ? 64 : 128;
	for (long b0 = 0; b0 < all.B; b0 += W4_TILE_ROWS) {	/* (a batch may have up to 2^31 - 1 rows) */
		const w4_args a = w4_rows(all, (int)b0, (int)(all.B - b0 < W4_TILE_ROWS ? all.B - b0 : W4_TILE_ROWS), esx, esy);
		const int ntiles = (a.B + BN - 1) / BN;
		const bool few = (long)((a.blocks + 7) / 8) * ntiles <= 256;	/* tiles of 128 rows: at most one a CU */
		/* rows in whole vectors, and a tile of them within the reach of a buffer descriptor */
		const bool dma = X != THHIP_F32 && (uintptr_t)a.x % 16 == 0 && a.ldx * esx % 16 == 0 && a.nIn * esx % 16 == 0 &&
			a.ldx * esx * BN < (1u << 31);
#define W4_TILE(ZP, DMA, KS, TH) do { \
	const int mtiles = (a.blocks + TH / 32 - 1) / (TH / 32); \
	w4_tile_kernel<X, GM, ZP, XG, DMA, KS, TH><<<dim3((unsigned)mtiles * ntiles), dim3(KS * TH), 0, thhip_stream()>>>(a, mtiles, ntiles); \
} while (0)
#define W4_TILE_ZP(DMA, KS, TH) do { if (a.zeros) W4_TILE(true, DMA, KS, TH); else W4_TILE(false, DMA, KS, TH); } while (0)
		if constexpr (X == THHIP_F32) {
			/* eight wavefronts and 256 rows, so that two share a SIMD (LDS holds one workgroup's x): 2048 x 8192 -> 8192
			 * 1092 -> 733 us, but 512 x 4096 -> 4096, where half the CUs then have nothing to do, 76 -> 92 */
			if (few)
				W4_TILE_ZP(false, 1, 256);
			else
				W4_TILE_ZP(false, 1, 512);
		} else {
			/* K in two halves where there are fewer tiles than CUs (1024 x 4096 -> 4096, us, without and with: 8-bit x 73 ->
			 * 57, fp16 groups of 64 65 -> 54, bf16 groups of 64 68 -> 56) */
			if (dma && few)
				W4_TILE_ZP(true, 2, 256);
			else if (dma)
				W4_TILE_ZP(true, 1, 256);
			else
				W4_TILE_ZP(false, 1, 256);
		}
#undef W4_TILE_ZP
#undef W4_TILE
	}
}

template <int X, bool XG>
static void w4_tile_groups(const w4_args &a)
{
	if (a.group == 32)
		w4_tile_launch<X, 1, XG>(a);
	else if (a.group == 64)
		w4_tile_launch<X, 2, XG>(a);
	else
		w4_tile_launch<X, 4, XG>(a);
}

void w4_tile(const w4_args &a, int xkind)
{
	if (xkind == W4_X_I8 && a.xgroups > 1)
		w4_tile_groups<W4_X_I8, true>(a);
	else if (xkind == W4_X_I8)
		w4_tile_groups<W4_X_I8, false>(a);
	else if (xkind == THHIP_F32)
		w4_tile_groups<THHIP_F32, false>(a);
	else if (xkind == THHIP_F16)
		w4_tile_groups<THHIP_F16, false>(a);
	else
		w4_tile_groups<THHIP_BF16, false>(a);
}
