/*
 * rope.hip - RMS norm of each head and rotation of queries and keys by
 * their positions, in one pass.
 *
 * norm_rope_k: y = x / sqrt(mean(x^2) + eps) * w over the D values of a
 * head; then pairs (a, b) of the first rot values are turned by the angle
 * pos * freq[i]: amp * (a cos - b sin, a sin + b cos). Every value is read
 * once and written once, so HBM bounds it.
 *
 * A block takes NR_TOKENS tokens (one where there are few) and first puts
 * their cosines and sines into LDS: all heads of a token share them, so
 * the 64-bit reduction of the angle (a far position times a frequency
 * loses its fraction in 32 bits) is done once per token and pair. Then
 * 256 / L groups of L lanes take a head each; a lane holds V values of
 * either half of the pairs (V = 16 bytes where sizes, strides and
 * addresses allow), so a turn needs no exchange between lanes, and the
 * norm's sum is a butterfly over the L lanes.
 */
#include "s3k.h"
#include "s3k_dev.h"

namespace s3k {

constexpr int NR_TOKENS = 4;
constexpr int NR_MAXD = 512;

struct NrArgs {
	struct s3k_heads q, k;
	const int *pos;
	const double *freq;
	long long pos_b;
	long long T;            /* B * S tokens                              */
	int S, D, rot;
	float amp, eps;
	int norm;
	int tpb;                /* tokens per block                          */
	int rows, rc, nrc;      /* heads of q and k, heads per block, blocks
				 * per group of tokens                       */
	int llog;               /* log2 of the lanes per head                */
};

/* cos and sin of 2 pi t for a 64-bit count of turns: the nearest quarter
 * turn is taken off in 64 bits, the rest (at most pi/4) goes through the
 * Taylor series to x^9 and x^10, whose next terms are below 2e-9. */
__device__ __forceinline__ float2 nr_cos_sin(double turns)
{
	const double f = turns - __builtin_rint(turns);
	const double qd = __builtin_rint(4.0 * f);
	const float x = (float)((f - 0.25 * qd) * 6.283185307179586);
	const float z = x * x;
	float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
	s = fmaf(z, s, 8.3333333e-3f);
	s = fmaf(z, s, -1.6666667e-1f);
	s = fmaf(x * z, s, x);
	float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
	c = fmaf(z, c, -1.3888889e-3f);
	c = fmaf(z, c, 4.1666667e-2f);
	c = fmaf(z, c, -0.5f);
	c = fmaf(z, c, 1.0f);
	const int q = (int)qd & 3;
	const float a = q & 1 ? s : c, b = q & 1 ? c : s;
	return make_float2(q == 1 || q == 2 ? -a : a, q & 2 ? -b : b);
}

/* V values of kind KIND at p (aligned to V elements) */
template <int KIND, int V>
__device__ __forceinline__ void nr_load(float (&x)[V], const void *p, long long i)
{
	if constexpr (KIND == S3K_F32) {
		const float *f = (const float *)p + i;
		if constexpr (V == 4) {
			const float4 t = *(const float4 *)f;
			x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
		} else if constexpr (V == 2) {
			const float2 t = *(const float2 *)f;
			x[0] = t.x, x[1] = t.y;
		} else {
			x[0] = f[0];
		}
	} else {
		const uint16_t *h = (const uint16_t *)p + i;
		uint32_t w[(V + 1) / 2];
		if constexpr (V == 8) {
			const uint4 t = *(const uint4 *)h;
			w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
		} else if constexpr (V == 4) {
			const uint2 t = *(const uint2 *)h;
			w[0] = t.x, w[1] = t.y;
		} else if constexpr (V == 2) {
			w[0] = *(const uint32_t *)h;
		} else {
			w[0] = h[0];
		}
#pragma unroll
		for (int e = 0; e < V; ++e) {
			const uint32_t u = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu;
			x[e] = KIND == S3K_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
		}
	}
}

template <int KIND, int V>
__device__ __forceinline__ void nr_store(const float (&x)[V], void *p, long long i)
{
	if constexpr (KIND == S3K_F32) {
		float *f = (float *)p + i;
		if constexpr (V == 4)
			*(float4 *)f = make_float4(x[0], x[1], x[2], x[3]);
		else if constexpr (V == 2)
			*(float2 *)f = make_float2(x[0], x[1]);
		else
			f[0] = x[0];
	} else {
		uint16_t *h = (uint16_t *)p + i;
		uint32_t w[(V + 1) / 2];
#pragma unroll
		for (int e = 0; e < (V + 1) / 2; ++e) {
			const float hi = 2 * e + 1 < V ? x[2 * e + 1 < V ? 2 * e + 1 : 0] : 0.0f;
			w[e] = KIND == S3K_BF16 ? pack_bf16x2(x[2 * e], hi) : pack_f16x2(x[2 * e], hi);
		}
		if constexpr (V == 8)
			*(uint4 *)h = make_uint4(w[0], w[1], w[2], w[3]);
		else if constexpr (V == 4)
			*(uint2 *)h = make_uint2(w[0], w[1]);
		else if constexpr (V == 2)
			*(uint32_t *)h = w[0];
		else
			h[0] = (uint16_t)w[0];
	}
}

/* NI: items (of 2 V values) a lane holds of one head. */
template <int KIND, int V, int NI, bool HALF>
__global__ void __launch_bounds__(256) norm_rope_k(NrArgs p)
{
	__shared__ float2 cs[NR_TOKENS * NR_MAXD / 2];
	const long long tg = (long long)(blockIdx.x / (unsigned)p.nrc) * p.tpb;
	const int r0 = (int)(blockIdx.x % (unsigned)p.nrc) * p.rc;
	const int rc = min(p.rc, p.rows - r0);
	const int nt = (int)(p.T - tg < p.tpb ? p.T - tg : p.tpb);
	const int half = p.rot / 2;

	for (int i = threadIdx.x; i < nt * half; i += 256) {
		const int t = i / half, e = i - t * half;
		const long long tok = tg + t, b = tok / p.S, s = tok - b * p.S;
		const double ps = p.pos ? (double)p.pos[b * p.pos_b + s] : (double)s;
		float2 c = nr_cos_sin(ps * p.freq[e] * 0.15915494309189535);
		c.x *= p.amp, c.y *= p.amp;
		cs[t * half + e] = c;
	}
	__syncthreads();

	const int L = 1 << p.llog, li = threadIdx.x & (L - 1);
	const int items = p.D / (2 * V), turned = half / V;
	for (int i = threadIdx.x >> p.llog; i < nt * rc; i += 256 >> p.llog) {
		const int t = i / rc, r = r0 + i - t * rc;
		const long long tok = tg + t, b = tok / p.S, s = tok - b * p.S;
		const bool isq = r < p.q.heads;
		const struct s3k_heads &hd = isq ? p.q : p.k;
		const int h = isq ? r : r - p.q.heads;
		const long long in = b * hd.in_b + s * hd.in_s + h * hd.in_h;
		const long long out = b * hd.out_b + s * hd.out_s + h * hd.out_h;

		float x[NI][2][V];
		int at[NI], bt[NI]; /* offsets of the two vectors of an item */
		float sq = 0.0f;
#pragma unroll
		for (int n = 0; n < NI; ++n) {
			const int j = li + n * L;
			const bool rot = j < turned;
			at[n] = HALF && rot ? j * V : 2 * V * j;
			bt[n] = at[n] + (HALF && rot ? half : V);
			if (j < items) {
				nr_load<KIND, V>(x[n][0], hd.in, in + at[n]);
				nr_load<KIND, V>(x[n][1], hd.in, in + bt[n]);
#pragma unroll
				for (int e = 0; e < V; ++e)
					sq = fmaf(x[n][0][e], x[n][0][e], fmaf(x[n][1][e], x[n][1][e], sq));
			}
		}
		if (p.norm) {
			for (int m = 1; m < L; m <<= 1)
				sq += __shfl_xor(sq, m);
			const float rs = 1.0f / __builtin_sqrtf(sq / (float)p.D + p.eps);
#pragma unroll
			for (int n = 0; n < NI; ++n)
				if (li + n * L < items) {
					float w[2][V];
					if (hd.weight) {
						nr_load<KIND, V>(w[0], hd.weight, at[n]);
						nr_load<KIND, V>(w[1], hd.weight, bt[n]);
					}
#pragma unroll
					for (int u = 0; u < 2; ++u)
#pragma unroll
						for (int e = 0; e < V; ++e) {
							x[n][u][e] *= rs;
							if (hd.weight)
								x[n][u][e] *= w[u][e];
						}
				}
		}
#pragma unroll
		for (int n = 0; n < NI; ++n) {
			const int j = li + n * L;
			if (j >= items)
				continue;
			if (j < turned) {
#pragma unroll
				for (int e = 0; e < V; ++e) {
					/* value 2e of the item's 2 V, or value e of its halves */
					const int ua = HALF || V == 1 ? 0 : 2 * e / V, ea = HALF || V == 1 ? e : 2 * e % V;
					const int ub = HALF || V == 1 ? 1 : (2 * e + 1) / V;
					const int eb = HALF || V == 1 ? e : (2 * e + 1) % V;
					const float2 c = cs[t * half + j * V + e];
					const float a = x[n][ua][ea], d = x[n][ub][eb];
					x[n][ua][ea] = fmaf(a, c.x, -(d * c.y));
					x[n][ub][eb] = fmaf(a, c.y, d * c.x);
				}
			}
			nr_store<KIND, V>(x[n][0], hd.out, out + at[n]);
			nr_store<KIND, V>(x[n][1], hd.out, out + bt[n]);
		}
	}
}

} /* namespace s3k */

using namespace s3k;

namespace {

template <int KIND, int V>
int nr_go(const NrArgs &a, int half_layout, int ni, unsigned blocks, hipStream_t st)
{
	if (ni == 1) {
		if (half_layout)
			hipLaunchKernelGGL((norm_rope_k<KIND, V, 1, true>), dim3(blocks), dim3(256), 0, st, a);
		else
			hipLaunchKernelGGL((norm_rope_k<KIND, V, 1, false>), dim3(blocks), dim3(256), 0, st, a);
	} else {
		if (half_layout)
			hipLaunchKernelGGL((norm_rope_k<KIND, V, 4, true>), dim3(blocks), dim3(256), 0, st, a);
		else
			hipLaunchKernelGGL((norm_rope_k<KIND, V, 4, false>), dim3(blocks), dim3(256), 0, st, a);
	}
	return (int)hipGetLastError();
}

template <int KIND>
int nr_kind(const NrArgs &a, int half_layout, int v, int ni, unsigned blocks, hipStream_t st)
{
	switch (v) {
	case 8:
		if constexpr (KIND != S3K_F32)
			return nr_go<KIND, 8>(a, half_layout, ni, blocks, st);
		else
			return (int)hipErrorInvalidValue;
	case 4: return nr_go<KIND, 4>(a, half_layout, ni, blocks, st);
	case 2: return nr_go<KIND, 2>(a, half_layout, ni, blocks, st);
	default: return nr_go<KIND, 1>(a, half_layout, ni, blocks, st);
	}
}

/* Whether every address of t is a multiple of v elements of es bytes. */
bool nr_aligned(const struct s3k_heads &t, int v, int es)
{
	if (!t.heads)
		return true;
	const long long strides = t.in_b | t.in_s | t.in_h | t.out_b | t.out_s | t.out_h;
	const uintptr_t at = (uintptr_t)t.in | (uintptr_t)t.out | (uintptr_t)t.weight;
	return strides % v == 0 && at % (uintptr_t)(v * es) == 0;
}

} /* namespace */

extern "C" int s3k_norm_rope(const struct s3k_norm_rope *d, void *stream)
{
	NrArgs a;
	a.q = d->q, a.k = d->k;
	if (!d->norm)
		a.q.weight = a.k.weight = nullptr;
	a.pos = d->pos, a.pos_b = d->pos_b, a.freq = d->freq;
	a.T = (long long)d->B * d->S;
	a.S = d->S, a.D = d->D, a.rot = d->rot;
	a.amp = d->amp, a.eps = d->eps, a.norm = d->norm;
	a.rows = d->q.heads + d->k.heads;
	if (a.T == 0 || a.rows == 0)
		return (int)hipSuccess;
	const int es = d->kind == S3K_F32 ? 4 : 2;
	int v = 16 / es;
	while (v > 1 && (a.rot / 2 % v || (a.D - a.rot) % (2 * v) || !nr_aligned(a.q, v, es) ||
			 !nr_aligned(a.k, v, es)))
		v /= 2;
	const int items = a.D / (2 * v);
	a.llog = 0;
	while (a.llog < 6 && (1 << a.llog) < items)
		++a.llog;
	const int ni = items > 64 ? 4 : 1;
	/* NR_TOKENS tokens a block once that leaves 4 blocks a CU, else one;
	 * with still fewer the heads are shared out too, one per group of
	 * lanes */
	a.tpb = a.T >= 4096 ? NR_TOKENS : 1;
	a.rc = a.T >= 1024 ? a.rows : 256 >> a.llog;
	if (a.rc > a.rows)
		a.rc = a.rows;
	a.nrc = (a.rows + a.rc - 1) / a.rc;
	const long long blocks = (a.T + a.tpb - 1) / a.tpb * a.nrc;
	if (!s3k_launchable(blocks, 256))
		return (int)hipErrorInvalidValue;
	hipStream_t st = (hipStream_t)stream;
	switch (d->kind) {
	case S3K_F32: return nr_kind<S3K_F32>(a, d->half, v, ni, (unsigned)blocks, st);
	case S3K_F16: return nr_kind<S3K_F16>(a, d->half, v, ni, (unsigned)blocks, st);
	case S3K_BF16: return nr_kind<S3K_BF16>(a, d->half, v, ni, (unsigned)blocks, st);
	}
	return (int)hipErrorInvalidValue;
}
