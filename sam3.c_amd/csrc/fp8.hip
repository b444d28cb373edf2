/*
 * fp8.hip - linear layers in 8-bit floating point (e4m3) with scales for
 * blocks of 128: the quantizers and the products.
 *
 *   C[m,n] = sum_b sa[b,m] * sw[n/128,b] * sum_{k in b} a[m,k] * w[n,k]
 *
 * The inner sum of a block is two v_mfma_f32_32x32x64_f8f6f4 (or one
 * 16x16x128; f16 MFMAs for f32 outputs) from zero; its result times the scales is added to the f32
 * accumulators by the VALU. The product is formed transposed, with the
 * weights as the MFMA's first operand: a lane then holds one row of A
 * (lane & 31), so the scale of a tile is one value per lane (sw is uniform
 * over a tile's 32 weight rows), and 4 neighbouring columns of C per
 * register group, stored together. Both operands are read with the same
 * (lane, byte) -> k map, whatever it is, so the MFMA's k order is free.
 */
#include "gemm_common.h"
#include "lds_dma.h"

namespace s3k {

typedef int f8_i8 __attribute__((ext_vector_type(8)));
typedef int f8_i4 __attribute__((ext_vector_type(4)));

constexpr int F8_BLK = 128;

__device__ __forceinline__ f8_i8 f8_join(const uint4 &a, const uint4 &b)
{
	return (f8_i8){(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

/*
 * c + the product over 64 (32x32) or 128 (16x16) e4m3 values of k.
 *
 * The 8-bit MFMAs add groups of 8 products (8 consecutive bytes of a lane)
 * on a grid of 2^-13 of the group's largest, cutting off what lies below
 * (measured: 2^2 beside 2^16 is lost in a group, 2^3 is kept), and the
 * groups' sums in f32. That is about 1.4e-5 of a result of normal values
 * and 7e-5 of widely spread ones: far below the rounding of a 16-bit
 * output (2^-8, 2^-11), so outputs of 16 bits take it. For f32 outputs
 * (EXACT) the values are widened to f16, which holds every e4m3 value
 * exactly, and the f16 MFMA keeps their products: half the rate.
 */
typedef _Float16 f8_h2 __attribute__((ext_vector_type(2)));

/* 8 e4m3 bytes as 8 f16 (v_cvt_scalef32_pk_f16_fp8, scale 1) */
__device__ __forceinline__ s3k_f16x8 f8_widen(int lo, int hi)
{
	const f8_h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
	const f8_h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
	const f8_h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
	const f8_h2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
	return (s3k_f16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <bool EXACT>
__device__ __forceinline__ s3k_f32x16 f8_mfma32(const f8_i8 &a, const f8_i8 &b, s3k_f32x16 c)
{
	if constexpr (EXACT) {
#pragma unroll
		for (int i = 0; i < 8; i += 2)
			c = __builtin_amdgcn_mfma_f32_32x32x16_f16(f8_widen(a[i], a[i + 1]), f8_widen(b[i], b[i + 1]),
								   c, 0, 0, 0);
		return c;
	} else {
		return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
	}
}
template <bool EXACT>
__device__ __forceinline__ s3k_f32x4 f8_mfma16(const f8_i8 &a, const f8_i8 &b, s3k_f32x4 c)
{
	if constexpr (EXACT) {
#pragma unroll
		for (int i = 0; i < 8; i += 2)
			c = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_widen(a[i], a[i + 1]), f8_widen(b[i], b[i + 1]),
								   c, 0, 0, 0);
		return c;
	} else {
		return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
	}
}

/* The least e >= -126 with amax <= 448 * 2^e = 1.75 * 2^(e + 8), amax
 * finite: from its exponent, one more if its mantissa is past 1.75. */
__device__ __forceinline__ int f8_exp_of(float amax)
{
	const uint32_t u = __float_as_uint(amax);
	const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
	return e < -126 ? -126 : e;
}

/* 2^e, -126 <= e <= 126, is pow2f(e). Four values times `down` as e4m3
 * bytes (v_cvt_pk_fp8_f32, to nearest even; |x * down| <= 448). Infinities
 * and NaN are made NaN first: what the conversion does past 448 is then
 * never asked. */
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float down)
{
	auto one = [&](float x) {
		return __builtin_fabsf(x) <= 3.402823466e38f ? x * down : __builtin_nanf("");
	};
	int w = __builtin_amdgcn_cvt_pk_fp8_f32(one(a), one(b), 0, false);
	w = __builtin_amdgcn_cvt_pk_fp8_f32(one(c), one(d), w, true);
	return (uint32_t)w;
}

/* N values of kind at p + i, those at and past `left` zero. VEC: p + i is
 * aligned to 16 bytes and none is past the end. */
template <int KIND, int N, bool VEC>
__device__ __forceinline__ void f8_load(float (&x)[N], const void *p, long long i, int left)
{
	if constexpr (VEC && KIND == S3K_F32) {
#pragma unroll
		for (int j = 0; j < N / 4; ++j) {
			const float4 t = *(const float4 *)((const float *)p + i + 4 * j);
			x[4 * j] = t.x, x[4 * j + 1] = t.y, x[4 * j + 2] = t.z, x[4 * j + 3] = t.w;
		}
	} else if constexpr (VEC) {
#pragma unroll
		for (int j = 0; j < N / 8; ++j) {
			const uint4 t = *(const uint4 *)((const uint16_t *)p + i + 8 * j);
			const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
			for (int e = 0; e < 8; ++e) {
				const uint32_t u = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
				x[8 * j + e] = KIND == S3K_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
			}
		}
	} else {
#pragma unroll
		for (int j = 0; j < N; ++j)
			x[j] = j < left ? load_as_f32(p, i + j, KIND) : 0.0f;
	}
}

/* ------------------------------------------------------------------ */
/* Quantizers                                                           */
/* ------------------------------------------------------------------ */
/*
 * Rows: 16 lanes take a group of 128 values, 8 each; the largest finite
 * magnitude is a butterfly over the 16 lanes. Reads and writes are whole
 * lines; HBM bounds it.
 */
template <int KIND, bool VEC>
__global__ void __launch_bounds__(256) f8_quant_rows(const void *x, long long ldx, int rows, int K,
						      int KB, uint8_t *q, float *scale)
{
	const long long g = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
	const int li = threadIdx.x & 15;
	if (g >= (long long)rows * KB)
		return;
	const int m = (int)(g / KB), kb = (int)(g - (long long)m * KB);
	const int k0 = kb * F8_BLK + li * 8, left = K - k0;
	float v[8];
	if (VEC && left >= 8)
		f8_load<KIND, 8, VEC>(v, x, m * ldx + k0, 8);
	else
		f8_load<KIND, 8, false>(v, x, m * ldx + k0, left);
	float amax = 0.0f;
#pragma unroll
	for (int e = 0; e < 8; ++e)
		amax = fmaxf(amax, finite_abs(v[e]));
#pragma unroll
	for (int off = 8; off > 0; off >>= 1)
		amax = fmaxf(amax, __shfl_xor(amax, off));
	const int e = f8_exp_of(amax);
	const float down = pow2f(-e);
	const uint32_t lo = f8_pack4(v[0], v[1], v[2], v[3], down), hi = f8_pack4(v[4], v[5], v[6], v[7], down);
	*(uint2 *)(q + g * F8_BLK + li * 8) = make_uint2(lo, hi);
	if (li == 0)
		scale[(long long)kb * rows + m] = pow2f(e);
}

/* Weights: a workgroup per 128 x 128 block, read twice (the second time
 * from cache): once per weight, so its speed does not count. */
__global__ void __launch_bounds__(256) f8_quant_blocks(const void *w, int kind, long long ldw, int N,
							int K, int KB, uint8_t *q, float *scale)
{
	__shared__ float part[4];
	const int nb = (int)(blockIdx.x / (unsigned)KB), kb = (int)(blockIdx.x % (unsigned)KB);
	const int n0 = nb * F8_BLK, k0 = kb * F8_BLK + (threadIdx.x & 31) * 4;
	float amax = 0.0f;
	for (int r = threadIdx.x >> 5; r < F8_BLK && n0 + r < N; r += 8)
		for (int e = 0; e < 4; ++e)
			if (k0 + e < K)
				amax = fmaxf(amax, finite_abs(load_as_f32(w, (n0 + r) * ldw + k0 + e, kind)));
	amax = wave_max_f32(amax);
	if ((threadIdx.x & 63) == 0)
		part[threadIdx.x >> 6] = amax;
	__syncthreads();
	amax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
	const int e = f8_exp_of(amax);
	const float down = pow2f(-e);
	for (int r = threadIdx.x >> 5; r < F8_BLK && n0 + r < N; r += 8) {
		float v[4];
		for (int i = 0; i < 4; ++i)
			v[i] = k0 + i < K ? load_as_f32(w, (n0 + r) * ldw + k0 + i, kind) : 0.0f;
		*(uint32_t *)(q + (n0 + r) * ((long long)KB * F8_BLK) + k0) = f8_pack4(v[0], v[1], v[2], v[3], down);
	}
	if (threadIdx.x == 0)
		scale[(long long)nb * KB + kb] = pow2f(e);
}

/* ------------------------------------------------------------------ */
/* Products                                                             */
/* ------------------------------------------------------------------ */
struct F8Args {
	const uint8_t *a, *w;
	const float *sa, *sw;
	void *c;
	const void *bias;
	int M, N, KB;
	int nmt, nnt;           /* tiles along M and N                       */
	int vec;                /* 4 columns of C (and bias) stored together */
	/* fused quantization: x in place of a, sa */
	const void *x;
	long long ldx;
	int K, xvec;
};

/* n..n+3 of row m, already f32: bias, GELU, one rounding, stored. */
template <int CK>
__device__ __forceinline__ void f8_store4(const F8Args &p, int m, int n, float4 v, int flags)
{
	float x[4] = {v.x, v.y, v.z, v.w};
	if (m >= p.M)
		return;
#pragma unroll
	for (int e = 0; e < 4; ++e) {
		if ((flags & S3K_EPI_BIAS) && n + e < p.N)
			x[e] += load_as_f32(p.bias, n + e, CK);
		if (flags & S3K_EPI_GELU)
			x[e] = gelu_tanh(x[e]);
	}
	const long long at = (long long)m * p.N + n;
	if (p.vec && n + 3 < p.N) {
		if constexpr (CK == S3K_F32)
			*(float4 *)((float *)p.c + at) = make_float4(x[0], x[1], x[2], x[3]);
		else if constexpr (CK == S3K_BF16)
			*(uint2 *)((uint16_t *)p.c + at) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
		else
			*(uint2 *)((uint16_t *)p.c + at) = make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]));
		return;
	}
#pragma unroll
	for (int e = 0; e < 4; ++e)
		if (n + e < p.N)
			store_from_f32(p.c, at + e, CK, x[e]);
}

/*
 * Tiles of BM rows of A by BN rows of W, WM x WN waves, each BM/WM by
 * BN/WN in 32x32 MFMA tiles. A stage holds one block of 128 k of both
 * operands (rows of 8 16-byte chunks, swizzled) and the rows' scales;
 * direct-to-LDS loads fill one of two stages while the other is used.
 */
template <int CK, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) f8_tile(F8Args p, int flags)
{
	constexpr int NW = WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
	constexpr int WB = BN * F8_BLK, AB = BM * F8_BLK, SB = BM * 4, STAGE = WB + AB + SB;
	constexpr int WI = BN / 8, AI = BM / 8; /* 1 KiB loads per stage */
	static_assert((WI + AI) % NW == 0 && BN / WN <= F8_BLK && BM % 64 == 0 && BM / 64 <= NW, "tile");
	__shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
	const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int wm = wave % WM, wn = wave / WM;
	const unsigned lds0 = lds_addr_of(smem);

	const int nt = (int)(blockIdx.x % (unsigned)p.nnt), mt = (int)(blockIdx.x / (unsigned)p.nnt);
	const int n0 = nt * BN, m0 = mt * BM;
	const unsigned Kp = (unsigned)p.KB * F8_BLK;
	const int wrows = min(BN, p.N - n0), arows = min(BM, p.M - m0);
	const s3k_i32x4 rw = buf_rsrc(p.w + (long long)n0 * Kp, (unsigned)wrows * Kp);
	const s3k_i32x4 ra = buf_rsrc(p.a + (long long)m0 * Kp, (unsigned)arows * Kp);

	/* load j = wave + t * NW: rows 8 j .. 8 j + 7 of W, then of A; rows
	 * past the end lie past the buffer and read as zeros */
	constexpr int PER = (WI + AI) / NW;
	unsigned off[PER];
#pragma unroll
	for (int t = 0; t < PER; ++t) {
		const int j = wave + t * NW;
		const int row = (j < WI ? j : j - WI) * 8 + (lane >> 3);
		off[t] = (unsigned)row * Kp + (unsigned)(((lane & 7) ^ lds_swz<8>(row)) * 16);
	}
	auto issue = [&](int kb, unsigned slot) {
#pragma unroll
		for (int t = 0; t < PER; ++t) {
			const int j = wave + t * NW;
			dma16s(lds0 + slot + j * 1024, j < WI ? rw : ra, off[t], (unsigned)kb * F8_BLK);
		}
		if (wave < BM / 64) {
			const s3k_i32x4 rs = buf_rsrc(p.sa + (long long)kb * p.M + m0, (unsigned)arows * 4);
			dma4s(lds0 + slot + WB + AB + wave * 256, rs, (unsigned)(wave * 256 + lane * 4));
		}
	};

	s3k_f32x16 acc[NT][MT];
#pragma unroll
	for (int i = 0; i < NT; ++i)
#pragma unroll
		for (int j = 0; j < MT; ++j)
#pragma unroll
			for (int r = 0; r < 16; ++r)
				acc[i][j][r] = 0.0f;

	/* operand rows of this lane: chunk 2 c + h of row base + l32 */
	auto frag = [&](unsigned at, int row, int s) {
		const int z = lds_swz<8>(row);
		const unsigned b = at + (unsigned)row * F8_BLK;
		return f8_join(lds_rd16(b, (unsigned)(((4 * s + h) ^ z) << 4)),
			       lds_rd16(b, (unsigned)(((4 * s + 2 + h) ^ z) << 4)));
	};
	const float *swp = p.sw + (long long)((n0 + wn * (BN / WN)) / F8_BLK) * p.KB;

	if (p.KB)
		issue(0, 0);
	for (int kb = 0; kb < p.KB; ++kb) {
		const unsigned slot = (unsigned)(kb & 1) * STAGE;
		wait_vm<0>();
		__syncthreads();
		if (kb + 1 < p.KB)
			issue(kb + 1, STAGE - slot);
		const unsigned wat = lds0 + slot, aat = wat + WB;
		const float sw = n0 + wn * (BN / WN) < p.N ? swp[kb] : 0.0f;
		f8_i8 fa[MT][2];
		float s[MT];
#pragma unroll
		for (int j = 0; j < MT; ++j) {
			const int row = wm * (BM / WM) + 32 * j + l32;
			fa[j][0] = frag(aat, row, 0);
			fa[j][1] = frag(aat, row, 1);
			s[j] = *(const float *)(smem + slot + WB + AB + row * 4) * sw;
		}
#pragma unroll
		for (int i = 0; i < NT; ++i) {
			const int row = wn * (BN / WN) + 32 * i + l32;
			const f8_i8 f0 = frag(wat, row, 0), f1 = frag(wat, row, 1);
#pragma unroll
			for (int j = 0; j < MT; ++j) {
				s3k_f32x16 z;
#pragma unroll
				for (int r = 0; r < 16; ++r)
					z[r] = 0.0f;
				z = f8_mfma32<CK == S3K_F32>(f0, fa[j][0], z);
				z = f8_mfma32<CK == S3K_F32>(f1, fa[j][1], z);
#pragma unroll
				for (int r = 0; r < 16; ++r)
					acc[i][j][r] = fmaf(z[r], s[j], acc[i][j][r]);
			}
		}
	}
#pragma unroll
	for (int j = 0; j < MT; ++j)
#pragma unroll
		for (int i = 0; i < NT; ++i)
#pragma unroll
			for (int g = 0; g < 4; ++g)
				f8_store4<CK>(p, m0 + wm * (BM / WM) + 32 * j + l32,
					      n0 + wn * (BN / WN) + 32 * i + 8 * g + 4 * h,
					      make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1],
							  acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]),
					      flags);
}

/*
 * Few rows (M <= 16 MT): a workgroup takes 16 weight rows and all rows of
 * x; its 8 waves share out the blocks of k (wave w takes w, w + 8, ...)
 * and add up in LDS. x is quantized in registers on the way: a lane holds
 * 32 values of row lane & 15, the group's other three quarters are in
 * lanes 16, 32 and 48 apart. The weights are read once, straight into
 * registers; they bound it, or the launch.
 */
template <int XK, int CK, int MT>
__global__ void __launch_bounds__(512) f8_rows(F8Args p, int flags)
{
	__shared__ float red[8][MT][256];
	const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int n0 = (int)blockIdx.x * 16;
	const long long Kp = (long long)p.KB * F8_BLK;
	const bool live = n0 + l16 < p.N;
	const uint8_t *wr = p.w + (long long)(n0 + l16) * Kp + 32 * g;
	const float *swp = p.sw + (long long)(n0 / F8_BLK) * p.KB;

	s3k_f32x4 acc[MT];
#pragma unroll
	for (int j = 0; j < MT; ++j)
		acc[j] = (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f};

	for (int kb = wave; kb < p.KB; kb += 8) {
		uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
		if (live) {
			w0 = *(const uint4 *)(wr + (long long)kb * F8_BLK);
			w1 = *(const uint4 *)(wr + (long long)kb * F8_BLK + 16);
		}
		const f8_i8 fw = f8_join(w0, w1);
		const float sw = swp[kb];
		const int k0 = kb * F8_BLK + 32 * g;
#pragma unroll
		for (int j = 0; j < MT; ++j) {
			const int m = 16 * j + l16;
			float v[32];
			if (m < p.M) {
				if (p.xvec && k0 + 32 <= p.K)
					f8_load<XK, 32, true>(v, p.x, m * p.ldx + k0, 32);
				else
					f8_load<XK, 32, false>(v, p.x, m * p.ldx + k0, p.K - k0);
			} else {
#pragma unroll
				for (int e = 0; e < 32; ++e)
					v[e] = 0.0f;
			}
			float amax = 0.0f;
#pragma unroll
			for (int e = 0; e < 32; ++e)
				amax = fmaxf(amax, finite_abs(v[e]));
			amax = fmaxf(amax, __shfl_xor(amax, 16));
			amax = fmaxf(amax, __shfl_xor(amax, 32));
			const int e = f8_exp_of(amax);
			const float down = pow2f(-e);
			f8_i8 fx;
#pragma unroll
			for (int i = 0; i < 8; ++i)
				fx[i] = (int)f8_pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], down);
			const s3k_f32x4 z = f8_mfma16<CK == S3K_F32>(fw, fx, (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f});
			const float s = pow2f(e) * sw;
#pragma unroll
			for (int r = 0; r < 4; ++r)
				acc[j][r] = fmaf(z[r], s, acc[j][r]);
		}
	}
#pragma unroll
	for (int j = 0; j < MT; ++j)
		*(s3k_f32x4 *)&red[wave][j][lane * 4] = acc[j];
	__syncthreads();
	/* thread t < 64 MT: lane t % 64 of tile t / 64, its four columns */
	const int t = threadIdx.x;
	if (t < 64 * MT) {
		float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
		for (int w = 0; w < 8; ++w) {
			const float4 u = *(const float4 *)&red[w][t >> 6][(t & 63) * 4];
			v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
		}
		f8_store4<CK>(p, 16 * (t >> 6) + (t & 15), n0 + 4 * ((t & 63) >> 4), v, flags);
	}
}

} /* namespace s3k */

using namespace s3k;

namespace {

template <int CK>
int f8_tile_go(F8Args &a, int flags, hipStream_t st)
{
	constexpr int BM = 64, BN = 64;
	a.nmt = (a.M + BM - 1) / BM, a.nnt = (a.N + BN - 1) / BN;
	const long long blocks = (long long)a.nmt * a.nnt;
	if (blocks > 0x7FFFFFFFll)
		return (int)hipErrorInvalidValue;
	hipLaunchKernelGGL((f8_tile<CK, BM, BN, 2, 2>), dim3((unsigned)blocks), dim3(256), 0, st, a, flags);
	return (int)hipGetLastError();
}

template <int XK, int CK>
int f8_rows_go(const F8Args &a, int flags, hipStream_t st)
{
	const unsigned blocks = (unsigned)((a.N + 15) / 16);
	if (a.M <= 16)
		hipLaunchKernelGGL((f8_rows<XK, CK, 1>), dim3(blocks), dim3(512), 0, st, a, flags);
	else
		hipLaunchKernelGGL((f8_rows<XK, CK, 2>), dim3(blocks), dim3(512), 0, st, a, flags);
	return (int)hipGetLastError();
}

template <int XK>
int f8_rows_ck(const F8Args &a, int ck, int flags, hipStream_t st)
{
	switch (ck) {
	case S3K_F32: return f8_rows_go<XK, S3K_F32>(a, flags, st);
	case S3K_F16: return f8_rows_go<XK, S3K_F16>(a, flags, st);
	case S3K_BF16: return f8_rows_go<XK, S3K_BF16>(a, flags, st);
	}
	return (int)hipErrorInvalidValue;
}

bool vec16(const void *p, long long ld, int kind)
{
	return (uintptr_t)p % 16 == 0 && ld % (kind == S3K_F32 ? 4 : 8) == 0;
}

F8Args f8_args(const void *w, const float *sw, void *c, int ck, int M, int N, int K, const void *bias)
{
	F8Args a = {};
	a.w = (const uint8_t *)w, a.sw = sw, a.c = c, a.bias = bias;
	a.M = M, a.N = N, a.K = K, a.KB = (K + F8_BLK - 1) / F8_BLK;
	a.vec = N % 4 == 0 && (uintptr_t)c % (ck == S3K_F32 ? 16 : 8) == 0;
	return a;
}

} /* namespace */

extern "C" int s3k_fp8_quantize(int kind, const void *x, long long ldx, int rows, int K, void *q,
				float *scale, void *stream)
{
	const int KB = (K + F8_BLK - 1) / F8_BLK;
	const long long blocks = ((long long)rows * KB + 15) / 16;
	if (blocks == 0)
		return (int)hipSuccess;
	if (blocks > 0x7FFFFFFFll)
		return (int)hipErrorInvalidValue;
	hipStream_t st = (hipStream_t)stream;
	const bool vec = vec16(x, ldx, kind);
#define F8_Q(KIND)                                                                                   \
	if (vec)                                                                                     \
		hipLaunchKernelGGL((f8_quant_rows<KIND, true>), dim3((unsigned)blocks), dim3(256), 0, st, \
				   x, ldx, rows, K, KB, (uint8_t *)q, scale);                        \
	else                                                                                         \
		hipLaunchKernelGGL((f8_quant_rows<KIND, false>), dim3((unsigned)blocks), dim3(256), 0, \
				   st, x, ldx, rows, K, KB, (uint8_t *)q, scale)
	switch (kind) {
	case S3K_F32: F8_Q(S3K_F32); break;
	case S3K_F16: F8_Q(S3K_F16); break;
	case S3K_BF16: F8_Q(S3K_BF16); break;
	default: return (int)hipErrorInvalidValue;
	}
#undef F8_Q
	return (int)hipGetLastError();
}

extern "C" int s3k_fp8_quantize_weight(int kind, const void *w, long long ldw, int N, int K, void *q,
				       float *scale, void *stream)
{
	const int KB = (K + F8_BLK - 1) / F8_BLK, NB = (N + F8_BLK - 1) / F8_BLK;
	const long long blocks = (long long)KB * NB;
	if (blocks == 0)
		return (int)hipSuccess;
	if (blocks > 0x7FFFFFFFll)
		return (int)hipErrorInvalidValue;
	hipLaunchKernelGGL(f8_quant_blocks, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, w,
			   kind, ldw, N, K, KB, (uint8_t *)q, scale);
	return (int)hipGetLastError();
}

extern "C" int s3k_fp8_matmul(const void *q, const float *sa, const void *w, const float *sw, int ck,
			      void *c, int M, int N, int K, const void *bias, int flags, void *stream)
{
	if (M == 0 || N == 0)
		return (int)hipSuccess;
	F8Args a = f8_args(w, sw, c, ck, M, N, K, bias);
	a.a = (const uint8_t *)q, a.sa = sa;
	switch (ck) {
	case S3K_F32: return f8_tile_go<S3K_F32>(a, flags, (hipStream_t)stream);
	case S3K_F16: return f8_tile_go<S3K_F16>(a, flags, (hipStream_t)stream);
	case S3K_BF16: return f8_tile_go<S3K_BF16>(a, flags, (hipStream_t)stream);
	}
	return (int)hipErrorInvalidValue;
}

extern "C" int s3k_fp8_rows(int xk, const void *x, long long ldx, const void *w, const float *sw, int ck,
			    void *c, int M, int N, int K, const void *bias, int flags, void *stream)
{
	if (M == 0 || N == 0)
		return (int)hipSuccess;
	if (M > S3K_FP8_ROWS_MAX)
		return (int)hipErrorInvalidValue;
	F8Args a = f8_args(w, sw, c, ck, M, N, K, bias);
	a.x = x, a.ldx = ldx, a.xvec = vec16(x, ldx, xk);
	switch (xk) {
	case S3K_F32: return f8_rows_ck<S3K_F32>(a, ck, flags, (hipStream_t)stream);
	case S3K_F16: return f8_rows_ck<S3K_F16>(a, ck, flags, (hipStream_t)stream);
	case S3K_BF16: return f8_rows_ck<S3K_BF16>(a, ck, flags, (hipStream_t)stream);
	}
	return (int)hipErrorInvalidValue;
}
