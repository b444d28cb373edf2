/*
 * fp8.hip - linear layers in 8-bit floating point (e4m3) with scales for
 * blocks of 128: the quantizers and the products.
 *
 *   C[m,n] = sum_b sa[b,m] * sw[n/128,b] * sum_{k in b} a[m,k] * w[n,k]
 *
 * The inner sum of a block is one v_mfma_f32_16x16x128_f8f6f4 (four f16
 * MFMAs for f32 outputs) from zero; its result times the scales is added
 * to the f32 accumulators by the VALU. The product is formed transposed, with the
 * weights as the MFMA's first operand: a lane then holds one row of A
 * (lane & 15), so the scale of a tile is one value per lane (sw is uniform
 * over a tile's 16 weight rows), and 4 neighbouring columns of C per
 * register group, stored together. Both operands are read with the same
 * (lane, byte) -> k map, whatever it is, so the MFMA's k order is free.
 */
#include "gemm_common.h"
#include "lds_dma.h"

namespace s3k {

template <int N>
struct f8_int {
	static constexpr int value = N;
};

typedef int f8_i8 __attribute__((ext_vector_type(8)));
typedef int f8_i4 __attribute__((ext_vector_type(4)));

constexpr int F8_BLK = 128;

__device__ __forceinline__ f8_i8 f8_join(const uint4 &a, const uint4 &b)
{
	return (f8_i8){(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

/*
 * c + the product over 128 e4m3 values of k.
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

/* Four values times `down` = 2^-e as e4m3 bytes (v_cvt_pk_fp8_f32, to
 * nearest even; |x * down| <= 448), infinities and NaN made NaN first: what
 * the conversion does past 448 is never asked. */
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float down)
{
	auto one = [&](float x) {
		return __builtin_fabsf(x) <= 3.402823466e38f ? x * down : __builtin_nanf("");
	};
	int w = __builtin_amdgcn_cvt_pk_fp8_f32(one(a), one(b), 0, false);
	w = __builtin_amdgcn_cvt_pk_fp8_f32(one(c), one(d), w, true);
	return (uint32_t)w;
}

/* Eight values of one row as they lie in memory. */
template <int KIND>
struct F8Raw {
	static constexpr int N = KIND == S3K_F32 ? 2 : 1;
	uint4 v[N];
};

/* Values i..i+7 at p as whole loads: memory takes them at any element's
 * address (1222 x 6503 f16 quantized in 6.7 us, one value at a time 11.2). */
template <int KIND>
__device__ __forceinline__ F8Raw<KIND> f8_whole8(const void *p, long long i)
{
	F8Raw<KIND> r;
#pragma unroll
	for (int j = 0; j < F8Raw<KIND>::N; ++j)
		__builtin_memcpy(&r.v[j], (const char *)p + i * (KIND == S3K_F32 ? 4 : 2) + 16 * j, 16);
	return r;
}

/* Values i..i+7 at p, those at and past `left` zero. */
template <int KIND>
__device__ __forceinline__ F8Raw<KIND> f8_load8(const void *p, long long i, int left)
{
	if (left >= 8)
		return f8_whole8<KIND>(p, i);
	F8Raw<KIND> r;
	uint32_t w[4 * F8Raw<KIND>::N];
#pragma unroll
	for (int j = 0; j < 4 * F8Raw<KIND>::N; ++j) {
		w[j] = 0;
		if constexpr (KIND == S3K_F32) {
			if (j < left)
				w[j] = ((const uint32_t *)p)[i + j];
		} else {
			if (2 * j < left)
				w[j] = ((const uint16_t *)p)[i + 2 * j];
			if (2 * j + 1 < left)
				w[j] |= (uint32_t)((const uint16_t *)p)[i + 2 * j + 1] << 16;
		}
	}
#pragma unroll
	for (int j = 0; j < F8Raw<KIND>::N; ++j)
		r.v[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
	return r;
}

/* Values i..i+7 at p, or zeros. */
template <int KIND>
__device__ __forceinline__ F8Raw<KIND> f8_chunk(const void *p, long long i, bool in)
{
	F8Raw<KIND> r;
#pragma unroll
	for (int j = 0; j < F8Raw<KIND>::N; ++j)
		r.v[j] = make_uint4(0, 0, 0, 0);
	if (in)
		r = f8_whole8<KIND>(p, i);
	return r;
}

/* r without its first s values (0 to 7), zeros behind. */
template <int KIND>
__device__ __forceinline__ void f8_drop(F8Raw<KIND> &r, int s)
{
	constexpr int N = 4 * F8Raw<KIND>::N, PER = 8 / N; /* words, values of one */
	uint32_t w[N];
	__builtin_memcpy(w, r.v, sizeof(w));
#pragma unroll
	for (int n = 4; n >= PER; n >>= 1)
#pragma unroll
		for (int i = 0; i < N; ++i)
			if (s & n)
				w[i] = i + n / PER < N ? w[i + n / PER < N ? i + n / PER : 0] : 0u;
	if (PER == 2 && (s & 1)) {
#pragma unroll
		for (int i = 0; i < N; ++i)
			w[i] = w[i] >> 16 | (i + 1 < N ? w[i + 1 < N ? i + 1 : 0] << 16 : 0u);
	}
	__builtin_memcpy(r.v, w, sizeof(w));
}

typedef unsigned short f8_us2 __attribute__((ext_vector_type(2)));

/* The larger of two keys: magnitudes as the bits of their type without the
 * sign, whose order is that of the values, infinities and NaN above all;
 * 16-bit types keep two keys in a word. */
template <int KIND>
__device__ __forceinline__ uint32_t f8_key_max(uint32_t a, uint32_t b)
{
	if constexpr (KIND == S3K_F32)
		return a > b ? a : b;
	else
		return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(f8_us2, a),
									      __builtin_bit_cast(f8_us2, b)));
}

template <int KIND>
__device__ __forceinline__ uint32_t f8_key(const F8Raw<KIND> &r)
{
	constexpr uint32_t MAG = KIND == S3K_F32 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
	uint32_t k = 0;
#pragma unroll
	for (int j = 0; j < F8Raw<KIND>::N; ++j) {
		k = f8_key_max<KIND>(k, f8_key_max<KIND>(r.v[j].x & MAG, r.v[j].y & MAG));
		k = f8_key_max<KIND>(k, f8_key_max<KIND>(r.v[j].z & MAG, r.v[j].w & MAG));
	}
	return k;
}

/* A key as the magnitude it stands for; infinity and NaN as infinity. */
template <int KIND>
__device__ __forceinline__ float f8_key_value(uint32_t k)
{
	if constexpr (KIND == S3K_F32) {
		return __uint_as_float(k < 0x7F800000u ? k : 0x7F800000u);
	} else {
		k = max(k & 0xFFFFu, k >> 16);
		if constexpr (KIND == S3K_BF16)
			return bf16_to_f32(k < 0x7F80u ? k : 0x7F80u);
		else
			return f16_to_f32(k < 0x7C00u ? k : 0x7C00u);
	}
}

template <int KIND>
__device__ __forceinline__ void f8_floats(const F8Raw<KIND> &r, float (&x)[8])
{
#pragma unroll
	for (int e = 0; e < 8; ++e) {
		if constexpr (KIND == S3K_F32) {
			const uint4 &u = r.v[e / 4];
			x[e] = __uint_as_float(e % 4 == 0 ? u.x : e % 4 == 1 ? u.y : e % 4 == 2 ? u.z : u.w);
		} else {
			const uint32_t u = e / 2 == 0 ? r.v[0].x : e / 2 == 1 ? r.v[0].y : e / 2 == 2 ? r.v[0].z : r.v[0].w;
			const uint32_t b = e & 1 ? u >> 16 : u & 0xFFFFu;
			x[e] = KIND == S3K_BF16 ? bf16_to_f32(b) : f16_to_f32(b);
		}
	}
}

typedef short f8_s2 __attribute__((ext_vector_type(2)));

/* Eight finite values over 2^e = up as e4m3 bytes: v_cvt_scalef32_pk_fp8_*
 * takes two values of the type as it is and the power of two, and rounds
 * to nearest even. */
template <int KIND>
__device__ __forceinline__ uint2 f8_pack8(const F8Raw<KIND> &r, float up)
{
	f8_s2 lo = {0, 0}, hi = {0, 0};
	if constexpr (KIND == S3K_F32) {
		lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, __uint_as_float(r.v[0].x), __uint_as_float(r.v[0].y), up, false);
		lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, __uint_as_float(r.v[0].z), __uint_as_float(r.v[0].w), up, true);
		hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, __uint_as_float(r.v[1].x), __uint_as_float(r.v[1].y), up, false);
		hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, __uint_as_float(r.v[1].z), __uint_as_float(r.v[1].w), up, true);
	} else if constexpr (KIND == S3K_BF16) {
		lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, __builtin_bit_cast(s3k_bf16x2, r.v[0].x), up, false);
		lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, __builtin_bit_cast(s3k_bf16x2, r.v[0].y), up, true);
		hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, __builtin_bit_cast(s3k_bf16x2, r.v[0].z), up, false);
		hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, __builtin_bit_cast(s3k_bf16x2, r.v[0].w), up, true);
	} else {
		lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, __builtin_bit_cast(f8_h2, r.v[0].x), up, false);
		lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(lo, __builtin_bit_cast(f8_h2, r.v[0].y), up, true);
		hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(hi, __builtin_bit_cast(f8_h2, r.v[0].z), up, false);
		hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(hi, __builtin_bit_cast(f8_h2, r.v[0].w), up, true);
	}
	return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

/* The largest magnitude of a group of 128 values of one row, C chunks of 8
 * in each of its lanes (the lanes that differ in the bits of LANES);
 * infinity if it holds one or a NaN. */
template <int KIND, int C, int LANES>
__device__ __forceinline__ float f8_group_max(const F8Raw<KIND> (&r)[C])
{
	uint32_t k = 0;
#pragma unroll
	for (int c = 0; c < C; ++c)
		k = f8_key_max<KIND>(k, f8_key<KIND>(r[c]));
#pragma unroll
	for (int m = 1; m < 64; m <<= 1)
		if (LANES & m)
			k = f8_key_max<KIND>(k, (uint32_t)__shfl_xor((int)k, m));
	return f8_key_value<KIND>(k);
}

/* A group -> e4m3 bytes and the scale. Where some group of the wave holds
 * an infinity or NaN, all of it takes the slow way. */
template <int KIND, int C, int LANES>
__device__ __forceinline__ float f8_group(const F8Raw<KIND> (&r)[C], uint2 (&q)[C])
{
	float amax = f8_group_max<KIND, C, LANES>(r);
	if (!__any(amax > 3.402823466e38f)) {
		const float up = pow2f(f8_exp_of(amax));
#pragma unroll
		for (int c = 0; c < C; ++c)
			q[c] = f8_pack8<KIND>(r[c], up);
		return up;
	}
	amax = 0.0f;
#pragma unroll
	for (int c = 0; c < C; ++c) {
		float x[8];
		f8_floats<KIND>(r[c], x);
#pragma unroll
		for (int e = 0; e < 8; ++e)
			amax = fmaxf(amax, finite_abs(x[e]));
	}
#pragma unroll
	for (int m = 1; m < 64; m <<= 1)
		if (LANES & m)
			amax = fmaxf(amax, __shfl_xor(amax, m));
	const int e = f8_exp_of(amax);
#pragma unroll
	for (int c = 0; c < C; ++c) {
		float x[8];
		f8_floats<KIND>(r[c], x);
		q[c] = make_uint2(f8_pack4(x[0], x[1], x[2], x[3], pow2f(-e)), f8_pack4(x[4], x[5], x[6], x[7], pow2f(-e)));
	}
	return pow2f(e);
}

/* ------------------------------------------------------------------ */
/* Quantizers                                                           */
/* ------------------------------------------------------------------ */
/*
 * Rows: 16 lanes take a group of 128 values, 8 each; the largest finite
 * magnitude is a butterfly over the 16 lanes. Reads and writes are whole
 * lines; HBM bounds it.
 */
template <int KIND>
__global__ void __launch_bounds__(256) f8_quant_rows(const void *x, long long ldx, int rows, int K,
						      int KB, uint8_t *q, float *scale)
{
	const long long g = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
	const int li = threadIdx.x & 15;
	if (g >= (long long)rows * KB)
		return;
	const int m = (int)(g / KB), kb = (int)(g - (long long)m * KB);
	const int k0 = kb * F8_BLK + li * 8;
	const F8Raw<KIND> r[1] = {f8_load8<KIND>(x, m * ldx + k0, K - k0)};
	uint2 o[1];
	const float up = f8_group<KIND, 1, 15>(r, o);
	*(uint2 *)(q + g * F8_BLK + li * 8) = o[0];
	if (li == 0)
		scale[(long long)kb * rows + m] = up;
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
	/* fused quantization: x in place of a, sa */
	const void *x;
	long long ldx;
	int K;
};

/* The bias of columns n..n+3 (zeros without one, and past N). */
template <int CK>
__device__ __forceinline__ float4 f8_bias4(const F8Args &p, int n, int flags)
{
	float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
	if ((flags & S3K_EPI_BIAS) && n + 3 < p.N) {
		if constexpr (CK == S3K_F32) {
			__builtin_memcpy(b, (const float *)p.bias + n, 16);
			return make_float4(b[0], b[1], b[2], b[3]);
		}
		uint2 w;
		__builtin_memcpy(&w, (const uint16_t *)p.bias + n, 8);
		if constexpr (CK == S3K_BF16)
			return make_float4(bf16_to_f32(w.x & 0xFFFFu), bf16_to_f32(w.x >> 16),
					   bf16_to_f32(w.y & 0xFFFFu), bf16_to_f32(w.y >> 16));
		return make_float4(f16_to_f32(w.x & 0xFFFFu), f16_to_f32(w.x >> 16), f16_to_f32(w.y & 0xFFFFu),
				   f16_to_f32(w.y >> 16));
	}
	if (flags & S3K_EPI_BIAS) {
#pragma unroll
		for (int e = 0; e < 4; ++e)
			if (n + e < p.N)
				b[e] = load_as_f32(p.bias, n + e, CK);
	}
	return make_float4(b[0], b[1], b[2], b[3]);
}

/* Four f32 sums: bias, GELU, rounded to 16 bits. */
template <int CK>
__device__ __forceinline__ uint2 f8_pack4c(const s3k_f32x4 &v, const float4 &bias, int flags)
{
	float x[4] = {v[0] + bias.x, v[1] + bias.y, v[2] + bias.z, v[3] + bias.w};
	if (flags & S3K_EPI_GELU) {
#pragma unroll
		for (int e = 0; e < 4; ++e)
			x[e] = gelu_tanh(x[e]);
	}
	if constexpr (CK == S3K_BF16)
		return make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
	else
		return make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]));
}

/* Columns n..n+3 of row m, f32 sums: bias, GELU, one rounding, stored. */
template <int CK>
__device__ __forceinline__ void f8_store4(const F8Args &p, int m, int n, float4 v, float4 bias, int flags)
{
	float x[4] = {v.x + bias.x, v.y + bias.y, v.z + bias.z, v.w + bias.w};
	if (m >= p.M)
		return;
	if (flags & S3K_EPI_GELU) {
#pragma unroll
		for (int e = 0; e < 4; ++e)
			x[e] = gelu_tanh(x[e]);
	}
	const long long at = (long long)m * p.N + n;
	if (n + 3 < p.N) {
		if constexpr (CK == S3K_F32) {
			__builtin_memcpy((float *)p.c + at, x, 16);
		} else {
			const uint2 w = CK == S3K_BF16 ? make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]))
						       : make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]));
			__builtin_memcpy((uint16_t *)p.c + at, &w, 8);
		}
		return;
	}
#pragma unroll
	for (int e = 0; e < 4; ++e)
		if (n + e < p.N)
			store_from_f32(p.c, at + e, CK, x[e]);
}

/*
 * A wave's NT x MT tiles: row m + 16 j, columns n + 16 i + 4 g + 0..3 in
 * acc[i][j] of lane group g. 16-bit outputs are stored 8 columns a lane, at
 * any element's address (20000 x 4001 x 500 106 us, one at a time 156): the
 * groups' pieces of two tiles are exchanged (v_permlane32_swap,
 * v_permlane16_swap) so that groups 0 and 1 hold the first tile and 2 and 3
 * the second, 64 bytes of a row together instead of 32 by halves of 8. The
 * largest tiles' rows of whole 128-byte lines go past the caches (PAST;
 * 20736 x 4096 x 1024 114 us, through them 124); rows that share lines meet
 * there (20736 x 2000 x 1000 62, past them 83).
 */
template <int CK, bool PAST, int NT, int MT>
__device__ __forceinline__ void f8_tile_store(const F8Args &p, const s3k_f32x4 (&acc)[NT][MT], int m, int n,
					      int g, int flags)
{
	if constexpr (CK != S3K_F32 && NT % 2 == 0) {
		if (n + 16 * NT <= p.N) {
#pragma unroll
			for (int i = 0; i < NT; i += 2) {
				const float4 b0 = f8_bias4<CK>(p, n + 16 * i + 4 * g, flags);
				const float4 b1 = f8_bias4<CK>(p, n + 16 * i + 16 + 4 * g, flags);
#pragma unroll
				for (int j = 0; j < MT; ++j) {
					const uint2 t0 = f8_pack4c<CK>(acc[i][j], b0, flags);
					const uint2 t1 = f8_pack4c<CK>(acc[i + 1][j], b1, flags);
					uint32_t w[4];
#pragma unroll
					for (int e = 0; e < 2; ++e) {
						const auto h = __builtin_amdgcn_permlane32_swap(e ? t0.y : t0.x, e ? t1.y : t1.x,
												false, false);
						const auto q = __builtin_amdgcn_permlane16_swap(h[0], h[1], false, false);
						w[e] = q[0], w[2 + e] = q[1];
					}
					const s3k_u32x4 v = {w[0], w[1], w[2], w[3]};
					uint16_t *const at = (uint16_t *)p.c + (long long)(m + 16 * j) * p.N + n + 16 * i + 8 * g;
					if (m + 16 * j < p.M) {
						if constexpr (PAST)
							__builtin_nontemporal_store(v, (s3k_u32x4 *)at);
						else
							__builtin_memcpy(at, &v, 16);
					}
				}
			}
			return;
		}
	}
#pragma unroll
	for (int i = 0; i < NT; ++i) {
		const float4 bias = f8_bias4<CK>(p, n + 16 * i + 4 * g, flags);
#pragma unroll
		for (int j = 0; j < MT; ++j)
			f8_store4<CK>(p, m + 16 * j, n + 16 * i + 4 * g,
				      make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]), bias, flags);
	}
}

/* Chunk c of tile row r lies at c ^ f8_swz(r). A 16-byte LDS read takes 16
 * lanes at a time (0-3, 12-15, 20-27, then the rest of 32, then the same of
 * the upper half); with rows of 128 bytes, row l & 15 and chunk l >> 4 (+ 4)
 * the 16 lanes then meet all 64 banks once. */
__device__ __forceinline__ int f8_swz(int row)
{
	return (row >> 1) & 7;
}

constexpr unsigned F8_STRIP = 8;

/* workgroup -> tile: workgroups go to the 8 XCDs round-robin; each XCD gets
 * a run of the tiles, taken in strips of 8 columns row by row, so that
 * the tiles it works on share rows of A and of W in its L2 */
__device__ __forceinline__ void f8_place(const F8Args &p, unsigned id, int &mt, int &nt)
{
	const unsigned total = (unsigned)p.nmt * (unsigned)p.nnt, x = id & 7u, each = total / 8u, more = total % 8u;
	const unsigned t = x * each + (x < more ? x : more) + (id >> 3);
	const unsigned strip = t / (F8_STRIP * (unsigned)p.nmt), in = t - strip * F8_STRIP * (unsigned)p.nmt;
	const unsigned wide = min(F8_STRIP, (unsigned)p.nnt - strip * F8_STRIP);
	mt = (int)(in / wide);
	nt = (int)(strip * F8_STRIP + in % wide);
}

/*
 * Tiles of BM rows of A by BN rows of W, WM x WN waves, each BM/WM by
 * BN/WN in 16x16 MFMA tiles of a whole block of 128 k. A stage holds one
 * block of both operands (rows of 8 16-byte chunks, swizzled) and the
 * rows' scales; two stages in a ring, filled by direct-to-LDS loads a
 * block ahead, over the end of a tile into the next one where a workgroup
 * takes several (MANY; 20736 x 4096 x 1024 with GELU: 112 us, a workgroup
 * for each tile 117; smaller tiles, more than one on a CU, overlap by
 * themselves, and were 5 % slower with it). KS such groups of waves, each
 * with stages of its own, take every KS-th block and are added up in LDS: for
 * few tiles, whose blocks one after the other would leave most CUs idle.
 */
template <int CK, int BM, int BN, int WM, int WN, int KS, bool PAST>
__global__ void __launch_bounds__(64 * WM * WN * KS, WM * WN * KS == 4 ? 2 : 1) f8_tile(F8Args p, int flags)
{
	constexpr bool MANY = WM * WN > 4; /* tiles of a workgroup */
	constexpr int NST = 2, NW = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
	constexpr int WB = BN * F8_BLK, AB = BM * F8_BLK, SB = NW * 256, STAGE = WB + AB + SB;
	constexpr int WI = BN / 8, AI = BM / 8; /* 1 KiB loads per stage */
	static_assert((WI + AI) % NW == 0 && BN / WN <= F8_BLK && BM * 4 <= SB, "tile");
	static_assert((KS - 1) * BM * BN * 4 <= KS * NST * STAGE, "sums fit the stages");
	__shared__ __attribute__((aligned(1024))) char smem_all[KS * NST * STAGE];
	const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
	const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int ks = all / NW, wave = all % NW;
	const int wm = wave % WM, wn = wave / WM;
	char *const smem = smem_all + ks * NST * STAGE;
	const unsigned lds0 = lds_addr_of(smem);

	/* the tile whose blocks are asked for */
	const unsigned Kp = (unsigned)p.KB * F8_BLK, total = (unsigned)p.nmt * (unsigned)p.nnt;
	int n0, m0;
	s3k_i32x4 rw, ra;
	auto place = [&](unsigned id) {
		f8_place(p, id, m0, n0);
		m0 *= BM, n0 *= BN;
		rw = buf_rsrc(p.w + (long long)n0 * Kp, (unsigned)min(BN, p.N - n0) * Kp);
		ra = buf_rsrc(p.a + (long long)m0 * Kp, (unsigned)min(BM, p.M - m0) * Kp);
	};
	place(blockIdx.x);

	/* load j = wave + t * NW: rows 8 j .. 8 j + 7 of W, then of A; rows
	 * past the end lie past the buffer and read as zeros, and so are
	 * blocks past the last */
	constexpr int PER = (WI + AI) / NW;
	unsigned off[PER];
#pragma unroll
	for (int t = 0; t < PER; ++t) {
		const int j = wave + t * NW;
		const int row = (j < WI ? j : j - WI) * 8 + (lane >> 3);
		off[t] = (unsigned)row * Kp + (unsigned)(((lane & 7) ^ f8_swz(row)) * 16);
	}
	auto issue = [&](int t, int kb, unsigned slot) __attribute__((always_inline)) {
		const bool in = kb < p.KB;
		if (t < PER) {
			const int j = wave + t * NW;
			dma16s(lds0 + slot + j * 1024, j < WI ? rw : ra, in ? off[t] : S3K_OOB, in ? (unsigned)kb * F8_BLK : 0u);
		} else {
			const s3k_i32x4 rs = buf_rsrc(p.sa + (long long)kb * p.M + m0, in ? (unsigned)min(BM, p.M - m0) * 4 : 0u);
			dma4s(lds0 + slot + WB + AB + wave * 256, rs, (unsigned)(wave * 256 + lane * 4));
		}
	};

	/* operand row l16 of tile t: chunks g and g + 4 (the swizzle of rows 16
	 * apart is the same) */
	const unsigned o0 = (unsigned)(l16 * F8_BLK + ((g ^ f8_swz(l16)) << 4));
	const unsigned o1 = (unsigned)(l16 * F8_BLK + (((g + 4) ^ f8_swz(l16)) << 4));
	const unsigned wo = lds0 + wn * (BN / WN) * F8_BLK, ao = lds0 + WB + wm * (BM / WM) * F8_BLK;
#pragma unroll
	for (int t = 0; t <= PER; ++t)
		issue(t, ks, 0);
	unsigned slot = 0;
	wait_vm<0>();
	unsigned tile = blockIdx.x;
	do {
		/* where this tile lies; m0 and n0 move on to the next one at its end */
		const int tm = m0, tn = n0 + wn * (BN / WN);
		const float *swp = p.sw + (long long)(tn / F8_BLK) * p.KB;
		s3k_f32x4 acc[NT][MT];
#pragma unroll
		for (int i = 0; i < NT; ++i)
#pragma unroll
			for (int j = 0; j < MT; ++j)
				acc[i][j] = (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f};
		for (int k0 = 0; k0 < p.KB; k0 += KS) {
			const int kb = k0 + ks;
			int ask = kb + KS;
			if (MANY && k0 + KS >= p.KB && tile + gridDim.x < total) {
				/* the next tile's first block, before this one's is stored */
				place(tile + gridDim.x);
				ask = ks;
			}
			/* block kb has landed here, and everywhere past the barrier; every
			 * wave is past the block before, whose stage is filled again */
			if (k0 > 0)
				wait_vm<0>();
			wg_barrier();
			const float sw = tn < p.N && kb < p.KB ? swp[kb] : 0.0f;
			const unsigned wat = wo + slot, aat = ao + slot;
			f8_i8 fa[MT];
			float s[MT];
#pragma unroll
			for (int j = 0; j < MT; ++j) {
				fa[j] = f8_join(lds_rd16(aat + o0, j * 16 * F8_BLK), lds_rd16(aat + o1, j * 16 * F8_BLK));
				s[j] = *(const float *)(smem + slot + WB + AB + (wm * (BM / WM) + 16 * j + l16) * 4) * sw;
			}
			/* the results of tile row i are added while row i + 1 is formed */
			s3k_f32x4 z[2][MT];
			auto add = [&](int i) {
#pragma unroll
				for (int j = 0; j < MT; ++j)
#pragma unroll
					for (int r = 0; r < 4; ++r)
						acc[i][j][r] = fmaf(z[i & 1][j][r], s[j], acc[i][j][r]);
			};
#pragma unroll
			for (int i = 0; i < NT; ++i) {
				/* the next block's loads a few at a time: asked for at once they
				 * kept the waves waiting at the address unit */
#pragma unroll
				for (int t = i * (PER + 1) / NT; t < (i + 1) * (PER + 1) / NT; ++t)
					issue(t, ask, STAGE - slot);
				const f8_i8 fw = f8_join(lds_rd16(wat + o0, i * 16 * F8_BLK), lds_rd16(wat + o1, i * 16 * F8_BLK));
#pragma unroll
				for (int j = 0; j < MT; ++j)
					z[i & 1][j] = f8_mfma16<CK == S3K_F32>(fw, fa[j], (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f});
				if (i > 0)
					add(i - 1);
			}
			add(NT - 1);
			slot = STAGE - slot;
		}
		/* the next tile's first block, or zeros: before the stores, which a
		 * wait after them would wait for too */
		wait_vm<0>();
		if constexpr (KS > 1) {
			wg_barrier();
			float *const sum = (float *)smem_all + wave * (NT * MT * 256) + lane * 4;
			if (ks > 0) {
				float *const mine = sum + (ks - 1) * (BM * BN);
#pragma unroll
				for (int i = 0; i < NT; ++i)
#pragma unroll
					for (int j = 0; j < MT; ++j)
						*(s3k_f32x4 *)(mine + (i * MT + j) * 256) = acc[i][j];
			}
			__syncthreads();
			if (ks > 0)
				return;
#pragma unroll
			for (int o = 0; o < KS - 1; ++o)
#pragma unroll
				for (int i = 0; i < NT; ++i)
#pragma unroll
					for (int j = 0; j < MT; ++j) {
						const s3k_f32x4 v = *(const s3k_f32x4 *)(sum + o * (BM * BN) + (i * MT + j) * 256);
#pragma unroll
						for (int r = 0; r < 4; ++r)
							acc[i][j][r] += v[r];
					}
		}
		f8_tile_store<CK, PAST, NT, MT>(p, acc, tm + wm * (BM / WM) + l16, tn, g, flags);
		tile += gridDim.x;
	} while (MANY && tile < total);
}

/*
 * Few rows: a workgroup takes 16 weight rows and 16 MT rows of A (with 4
 * weight rows, for more workgroups, 1 x 1024 x 4096 took 3.9 us, with 16 3.5);
 * its NWV waves share out the blocks of k (wave w takes w, w + NWV, ...)
 * and add up in LDS. Every wave has two blocks under way in LDS of its own
 * and meets the others only at the end. The operands come by direct-to-LDS
 * loads, eight lanes to a row's 128 bytes: straight into registers, as the
 * MFMA wants them, neighbouring lanes read different rows and a load takes
 * 64 cycles of address work (17 x 1024 x 4096: 5.9 us). Latency and, with
 * long weights, HBM bound it.
 *
 * XK >= 0 (MT = 1): x of that type is quantized in registers on the way: a
 * lane holds 32 values of row lane & 15, the group's other three quarters
 * are 16, 32 and 48 lanes on. Every workgroup repeats that, which one
 * launch less pays for up to 64 rows. The last values of a K that is no
 * multiple of 8 (TAIL) are read as the row's last 8 (K is at least 8) and
 * moved down; the code for it costs other lengths 0.15 to 0.5 us.
 * XK < 0: quantized rows, 16 MT of them from blockIdx.y on.
 */
template <int XK, int CK, int MT, int NWV, bool TAIL>
__global__ void __launch_bounds__(64 * NWV) f8_rows(F8Args p, int flags)
{
	static_assert(XK < 0 || MT == 1, "quantized on the way: 16 rows a workgroup");
	constexpr int RT = XK < 0 ? 1 + MT : 1, SLOT = RT * 2048; /* row tiles of a block */
	constexpr int RED = NWV * MT * 1024, RING = NWV * 2 * SLOT;
	__shared__ __attribute__((aligned(1024))) char smem[RED > RING ? RED : RING];
	float (*const red)[MT][256] = (float (*)[MT][256])smem;
	const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * MT;
	const unsigned Kp = (unsigned)p.KB * F8_BLK;
	const s3k_i32x4 rw = buf_rsrc(p.w + (long long)n0 * Kp, (unsigned)min(16, p.N - n0) * Kp);
	const s3k_i32x4 ra = buf_rsrc(XK < 0 ? p.a + (long long)m0 * Kp : nullptr,
				      XK < 0 ? (unsigned)min(16 * MT, p.M - m0) * Kp : 0u);
	const float *swp = p.sw + (long long)(n0 / F8_BLK) * p.KB;
	const unsigned mine = lds_addr_of(smem) + wave * 2 * SLOT;

	s3k_f32x4 acc[MT];
#pragma unroll
	for (int j = 0; j < MT; ++j)
		acc[j] = (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f};

	/* rows 8 i + (lane >> 3) of a tile by load i; the swizzles of rows 8
	 * apart differ in bit 2 */
	const unsigned row = (unsigned)lane >> 3;
	const unsigned off0 = row * Kp + ((lane & 7) ^ f8_swz((int)row)) * 16u;
	const unsigned off1 = (row + 8) * Kp + ((lane & 7) ^ f8_swz((int)row + 8)) * 16u;
	const unsigned rd0 = (unsigned)(l16 * F8_BLK + ((g ^ f8_swz(l16)) << 4));
	const unsigned rd1 = (unsigned)(l16 * F8_BLK + (((g + 4) ^ f8_swz(l16)) << 4));

	constexpr int NA = XK < 0 ? MT : 1, NX = XK < 0 ? 1 : 4;
	float sa[2][NA], sw[2];
	F8Raw<XK < 0 ? S3K_BF16 : XK> x[2][NX];
	auto load = [&](auto slot, int kb) __attribute__((always_inline)) {
		constexpr int S = decltype(slot)::value;
		const unsigned at = mine + S * SLOT;
		const unsigned ko = (unsigned)__builtin_amdgcn_readfirstlane(kb * F8_BLK);
		dma16s(at, rw, off0, ko);
		dma16s(at + 1024, rw, off1, ko);
		sw[S] = swp[kb];
		if constexpr (XK < 0) {
#pragma unroll
			for (int j = 0; j < MT; ++j) {
				dma16s(at + 2048 + j * 2048, ra, off0 + 16 * j * Kp, ko);
				dma16s(at + 3072 + j * 2048, ra, off1 + 16 * j * Kp, ko);
				const int m = m0 + 16 * j + l16;
				sa[S][j] = m < p.M ? p.sa[(long long)kb * p.M + m] : 0.0f;
			}
		} else {
			const int k0 = kb * F8_BLK + 16 * g;
#pragma unroll
			for (int c = 0; c < 4; ++c) {
				/* bytes 16 g and 64 + 16 g onward, as the weights' */
				const int k = k0 + 64 * (c >> 1) + 8 * (c & 1);
				x[S][c] = f8_chunk<XK>(p.x, (m0 + l16) * p.ldx + (TAIL ? min(k, p.K - 8) : k), m0 + l16 < p.M && k < p.K);
			}
		}
	};
	auto work = [&](auto slot, int kb) __attribute__((always_inline)) {
		constexpr int S = decltype(slot)::value;
		const unsigned at = mine + S * SLOT;
		const f8_i8 fw = f8_join(lds_rd16(at + rd0, 0), lds_rd16(at + rd1, 0));
#pragma unroll
		for (int j = 0; j < MT; ++j) {
			f8_i8 fx;
			float s;
			if constexpr (XK < 0) {
				fx = f8_join(lds_rd16(at + rd0, 2048 + 2048 * j), lds_rd16(at + rd1, 2048 + 2048 * j));
				s = sa[S][j] * sw[S];
			} else {
				/* an infinity or NaN makes all of its row's results NaN,
				 * whatever the group's other values become */
				if (TAIL && kb == p.KB - 1) {
#pragma unroll
					for (int c = 0; c < 4; ++c) {
						const int k = kb * F8_BLK + 16 * g + 64 * (c >> 1) + 8 * (c & 1);
						f8_drop<XK>(x[S][c], k < p.K ? max(k - (p.K - 8), 0) : 0);
					}
				}
				const float amax = f8_group_max<XK, 4, 48>(x[S]);
				const float up = pow2f(f8_exp_of(amax));
				uint2 q[4];
#pragma unroll
				for (int c = 0; c < 4; ++c)
					q[c] = f8_pack8<XK>(x[S][c], up);
				s = amax <= 3.402823466e38f ? up * sw[S] : __builtin_nanf("");
				fx = (f8_i8){(int)q[0].x, (int)q[0].y, (int)q[1].x, (int)q[1].y,
					     (int)q[2].x, (int)q[2].y, (int)q[3].x, (int)q[3].y};
			}
			const s3k_f32x4 z = f8_mfma16<CK == S3K_F32>(fw, fx, (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
			for (int r = 0; r < 4; ++r)
				acc[j][r] = fmaf(z[r], s, acc[j][r]);
		}
	};
	f8_int<0> even;
	f8_int<1> odd;
	if (wave < p.KB)
		load(even, wave);
	if (wave + NWV < p.KB)
		load(odd, wave + NWV);
	for (int kb = wave; kb < p.KB; kb += 2 * NWV) {
		wait_vm<0>(); /* both blocks: the compiler does not see these loads */
		__builtin_amdgcn_sched_barrier(0);
		work(even, kb);
		if (kb + NWV < p.KB)
			work(odd, kb + NWV);
		if (kb + 2 * NWV < p.KB) {
			asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); /* the slots are read */
			load(even, kb + 2 * NWV);
			if (kb + 3 * NWV < p.KB)
				load(odd, kb + 3 * NWV);
		}
	}
	__syncthreads(); /* the sums go over the ring */
#pragma unroll
	for (int j = 0; j < MT; ++j)
		*(s3k_f32x4 *)&red[wave][j][lane * 4] = acc[j];
	__syncthreads();
	/* thread t < 64 MT: lane t % 64 of tile t / 64, its four columns */
	const int t = threadIdx.x;
	if (t < 64 * MT) {
		float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
		for (int w = 0; w < NWV; ++w) {
			const float4 u = *(const float4 *)&red[w][t >> 6][(t & 63) * 4];
			v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
		}
		const int n = n0 + 4 * ((t & 63) >> 4);
		f8_store4<CK>(p, m0 + 16 * (t >> 6) + (t & 15), n, v, f8_bias4<CK>(p, n, flags), flags);
	}
}

} /* namespace s3k */

using namespace s3k;

namespace {

template <int CK, int BM, int BN, int WM, int WN, int KS>
int f8_tile_run(F8Args &a, int flags, hipStream_t st)
{
	a.nmt = (int)((a.M + BM - 1ll) / BM), a.nnt = (int)((a.N + BN - 1ll) / BN);
	const long long blocks = (long long)a.nmt * a.nnt;
	/* one workgroup a CU for the tiles that leave room for no more; the
	 * others overlap their ends by themselves. 256 is a multiple of the XCDs:
	 * a workgroup's tiles stay on its XCD's run. */
	const long long grid = WM * WN > 4 && a.KB > 0 && blocks > 256 ? 256 : blocks;
	if (blocks > 0x7FFFFFFFll || !s3k_launchable(grid, 64 * WM * WN * KS))
		return (int)hipErrorInvalidValue;
	const dim3 g((unsigned)grid), wg(64 * WM * WN * KS);
	if constexpr (WM * WN > 4) {
		/* rows of whole lines */
		if (a.N % 64 == 0 && (uintptr_t)a.c % 128 == 0) {
			hipLaunchKernelGGL((f8_tile<CK, BM, BN, WM, WN, KS, true>), g, wg, 0, st, a, flags);
			return (int)hipGetLastError();
		}
	}
	hipLaunchKernelGGL((f8_tile<CK, BM, BN, WM, WN, KS, false>), g, wg, 0, st, a, flags);
	return (int)hipGetLastError();
}

template <int XK, int CK, int MT, bool TAIL>
int f8_rows_go(F8Args &a, int flags, hipStream_t st)
{
	const unsigned mb = (unsigned)((a.M + 16 * MT - 1) / (16 * MT)); /* M is small */
	const unsigned nb = (unsigned)((a.N + 15ll) / 16);
	if (!s3k_launchable(nb, 1024))
		return (int)hipErrorInvalidValue;
	/* as many waves as there are blocks of k for, up to 16 (8 with two row
	 * tiles, for their LDS) */
	if constexpr (MT == 1) {
		if (a.KB > 8) {
			hipLaunchKernelGGL((f8_rows<XK, CK, MT, 16, TAIL>), dim3(nb, mb), dim3(1024), 0, st, a, flags);
			return (int)hipGetLastError();
		}
	}
	hipLaunchKernelGGL((f8_rows<XK, CK, MT, 8, TAIL>), dim3(nb, mb), dim3(512), 0, st, a, flags);
	return (int)hipGetLastError();
}

/*
 * The kernel of a product, by an estimate of each one's time from its grid.
 * Measured (bf16, 12 row counts from 24 to 20736 by seven N x K, and
 * 8192^3), the tile kernels take, in us, for a block of k with one workgroup
 * on a CU and with all that fit, and for the rest of a tile; a round is one
 * workgroup in every place. The few-rows kernels are linear in their
 * workgroups. The kernel it takes was at most 4 % behind the quickest, 0.1 %
 * in the mean. Examples, us:
 *
 *     M x N x K            64  64/2  64/4   128  192x256  256  rows 1  2
 *     77 x 1024 x 4096   16.0  11.1   9.7  26.1    40.0  47.9   6.0   4.3
 *     400 x 1024 x 4096  16.5  11.7  10.4  26.5    41.2  48.8  17.4  13.1
 *     1369 x 4096 x 1024 14.4  17.7  25.5  13.7    16.9  19.7  65    71
 *     20736 x 4096 x 1024 163   206   339   118     109   105   942  1031
 *     8192^3              842               570     556   459
 *
 * (64/2: two groups of waves share out the blocks.) The two largest tiles
 * are not built for f32 outputs, whose wider operands spill there.
 */
enum { F8_T64, F8_T64K2, F8_T64K4, F8_T128, F8_T192, F8_T256, F8_ROWS1, F8_ROWS2, F8_KERNELS };

struct F8Cost {
	int bm, bn, ks, fit;    /* tile, groups along k, workgroups a CU     */
	double one, full, rest;
};
const F8Cost f8_costs[F8_ROWS1] = {
	{64, 64, 1, 4, 0.33, 0.84, 1.0},   {64, 64, 2, 2, 0.54, 0.97, 1.2},   {64, 64, 4, 1, 0.88, 1.07, 1.6},
	{128, 128, 1, 2, 0.86, 1.15, 2.1}, {192, 256, 1, 1, 1.42, 1.28, 4.7}, {256, 256, 1, 1, 1.43, 1.35, 8.1},
};

double f8_estimate(int kernel, int M, int N, int KB)
{
	if (kernel >= F8_ROWS1) {
		const int mt = kernel == F8_ROWS1 ? 1 : 2;
		const double wgs = (double)((N + 15ll) / 16) * ((M + 16ll * mt - 1) / (16 * mt));
		return mt == 1 ? 2.4 + 0.004 * KB + wgs * (0.35e-3 * KB + 0.2e-3)
			       : 2.35 + 0.027 * KB + wgs * (0.31e-3 * KB + 2.5e-3);
	}
	const F8Cost &c = f8_costs[kernel];
	const double tiles = (double)((M + c.bm - 1ll) / c.bm) * ((N + c.bn - 1ll) / c.bn), its = (KB + c.ks - 1) / c.ks;
	const double places = 256.0 * c.fit, rounds = (double)(long long)(tiles / places);
	double t = 2.3 + rounds * (its * c.full + c.rest);
	const double left = tiles - rounds * places;
	if (left > 0.0) {
		/* the last round, ceil(left / 256) workgroups on a CU */
		const double on = (double)(long long)((left + 255.0) / 256.0);
		const double per = c.fit > 1 ? c.one + (c.full - c.one) * (on - 1.0) / (c.fit - 1.0) : c.one;
		t += its * per + c.rest;
	}
	return t;
}

template <int CK>
int f8_product(F8Args &a, int flags, hipStream_t st)
{
	int best = F8_T64;
	double least = 1e30;
	for (int k = 0; k < F8_KERNELS; ++k) {
		if ((CK == S3K_F32 && (k == F8_T192 || k == F8_T256)) || (k >= F8_ROWS1 && a.M > 4096))
			continue;
		const double t = f8_estimate(k, a.M, a.N, a.KB);
		if (t < least)
			least = t, best = k;
	}
	switch (best) {
	case F8_T64K2: return f8_tile_run<CK, 64, 64, 2, 2, 2>(a, flags, st);
	case F8_T64K4: return f8_tile_run<CK, 64, 64, 2, 2, 4>(a, flags, st);
	case F8_T128: return f8_tile_run<CK, 128, 128, 2, 2, 1>(a, flags, st);
	case F8_T192:
		if constexpr (CK != S3K_F32)
			return f8_tile_run<CK, 192, 256, 2, 4, 1>(a, flags, st);
		break;
	case F8_T256:
		if constexpr (CK != S3K_F32)
			return f8_tile_run<CK, 256, 256, 4, 2, 1>(a, flags, st);
		break;
	case F8_ROWS1: return f8_rows_go<-1, CK, 1, false>(a, flags, st);
	case F8_ROWS2: return f8_rows_go<-1, CK, 2, false>(a, flags, st);
	}
	return f8_tile_run<CK, 64, 64, 2, 2, 1>(a, flags, st);
}

template <int XK, int CK>
int f8_rows_x(F8Args &a, int flags, hipStream_t st)
{
	return a.K % 8 ? f8_rows_go<XK, CK, 1, true>(a, flags, st) : f8_rows_go<XK, CK, 1, false>(a, flags, st);
}

template <int XK>
int f8_rows_ck(F8Args &a, int ck, int flags, hipStream_t st)
{
	switch (ck) {
	case S3K_F32: return f8_rows_x<XK, S3K_F32>(a, flags, st);
	case S3K_F16: return f8_rows_x<XK, S3K_F16>(a, flags, st);
	case S3K_BF16: return f8_rows_x<XK, S3K_BF16>(a, flags, st);
	}
	return (int)hipErrorInvalidValue;
}

F8Args f8_args(const void *w, const float *sw, void *c, int M, int N, int K, const void *bias)
{
	F8Args a = {};
	a.w = (const uint8_t *)w, a.sw = sw, a.c = c, a.bias = bias;
	a.M = M, a.N = N, a.K = K, a.KB = (K + F8_BLK - 1) / F8_BLK;
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
	if (!s3k_launchable(blocks, 256))
		return (int)hipErrorInvalidValue;
	hipStream_t st = (hipStream_t)stream;
#define F8_Q(KIND)                                                                                  \
	hipLaunchKernelGGL((f8_quant_rows<KIND>), dim3((unsigned)blocks), dim3(256), 0, st, x, ldx, rows, K, \
			   KB, (uint8_t *)q, scale)
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
	const int KB = (K + F8_BLK - 1) / F8_BLK, NB = (int)((N + F8_BLK - 1ll) / F8_BLK);
	const long long blocks = (long long)KB * NB;
	if (blocks == 0)
		return (int)hipSuccess;
	if (!s3k_launchable(blocks, 256))
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
	F8Args a = f8_args(w, sw, c, M, N, K, bias);
	a.a = (const uint8_t *)q, a.sa = sa;
	switch (ck) {
	case S3K_F32: return f8_product<S3K_F32>(a, flags, (hipStream_t)stream);
	case S3K_F16: return f8_product<S3K_F16>(a, flags, (hipStream_t)stream);
	case S3K_BF16: return f8_product<S3K_BF16>(a, flags, (hipStream_t)stream);
	}
	return (int)hipErrorInvalidValue;
}

extern "C" int s3k_fp8_rows_ok(int M, int K)
{
	return M <= S3K_FP8_ROWS_MAX && (K == 0 || K >= 8);
}

extern "C" int s3k_fp8_rows(int xk, const void *x, long long ldx, const void *w, const float *sw, int ck,
			    void *c, int M, int N, int K, const void *bias, int flags, void *stream)
{
	if (M == 0 || N == 0)
		return (int)hipSuccess;
	if (!s3k_fp8_rows_ok(M, K))
		return (int)hipErrorInvalidValue;
	F8Args a = f8_args(w, sw, c, M, N, K, bias);
	a.x = x, a.ldx = ldx;
	switch (xk) {
	case S3K_F32: return f8_rows_ck<S3K_F32>(a, ck, flags, (hipStream_t)stream);
	case S3K_F16: return f8_rows_ck<S3K_F16>(a, ck, flags, (hipStream_t)stream);
	case S3K_BF16: return f8_rows_ck<S3K_BF16>(a, ck, flags, (hipStream_t)stream);
	}
	return (int)hipErrorInvalidValue;
}
