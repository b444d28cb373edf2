/*
 * xattn.hip - attention of queries to keys and values of another length:
 * strided tensors, lengths per sequence, key heads shared by a group of
 * query heads, keys shared out over workgroups where rows are few.
 *
 *   out[b,s,h] = sum_j softmax_j(scale * q[b,s,h] . k[b,j,h']) v[b,j,h'],
 *   j < k_len[b], h' = h / G, G = H / Hkv
 *
 * The G query heads that share a key head are laid side by side: row
 * r = s * G + g of (b, h') is query s, head h' * G + g, so a tile of rows
 * reads each key and value once for all of them (a decoder's single query
 * has G rows). Softmax runs with a running maximum and sum per row, in
 * base 2, the scale folded into the exponent's multiply.
 *
 * Three kernels:
 *   xa_mfma     f16 / bf16, D a multiple of 8 up to 256, 16-byte aligned;
 *   xa_f32      f32, D a multiple of 4 up to 256, 16-byte aligned;
 *   xa_generic  the rest: one wave per row.
 */
#include "attn_dev.h"
#include "gemm_common.h"
#include "lds_dma.h"

namespace s3k {

struct XaArgs {
	struct s3k_xattn d;
	int G, rows;            /* query heads per key head; Sq * G          */
	int nrb, ns;            /* row blocks per (b, h'); parts of the keys */
	int run;                /* key heads kept on one XCD (xa_place)      */
	int sort;               /* sequences of most keys first (xa_place)   */
	float c;                /* scale * log2(e)                           */
	int ovec;               /* 4 values of an output row stored together */
	float *part;            /* ns > 1: results of the parts              */
};

constexpr int XA_PARTS = 64; /* of a row's keys, at most */
constexpr float XA_NONE = -3.402823466e38f; /* running maximum of no keys */

__device__ __forceinline__ int xa_len(const int *lens, int b, int most)
{
	if (!lens)
		return most;
	const int n = lens[b];
	return n < 0 ? 0 : n > most ? most : n;
}

/* workgroup -> (b * Hkv + h', part, row block): workgroups go to the 8 XCDs
 * round-robin. The row blocks that read the same keys get ids of one
 * residue mod 8 and share an XCD's L2, and so do p.run key heads whose rows
 * lie together in less than 256 bytes: apart, two XCDs each fetched the
 * same lines (16 x 8 heads of 16 f32, 5184 keys: 34 us, together 26). With
 * p.sort the sequences of most keys go first, so that the last workgroups to
 * run are short ones. */
__device__ __forceinline__ void xa_place(const XaArgs &p, unsigned id, int &bh, int &part, int &rb)
{
	const unsigned runs = (unsigned)(p.d.Hkv / p.run), units = (unsigned)(p.d.B * p.ns) * runs;
	const unsigned per = (unsigned)(p.run * p.nrb), whole = units / 8u * 8u * per;
	unsigned u, in;
	if (id < whole) {
		const unsigned sl = id >> 3;
		u = sl / per * 8u + (id & 7u);
		in = sl % per;
	} else {
		u = units / 8u * 8u + (id - whole) / per;
		in = (id - whole) % per;
	}
	const unsigned rest = u / runs;
	const int hk = (int)(u % runs) * p.run + (int)(in / (unsigned)p.nrb);
	rb = (int)(in % (unsigned)p.nrb);
	part = (int)(rest % (unsigned)p.ns);
	int b = (int)(rest / (unsigned)p.ns);
	if (p.sort) {
		/* the sequence with b longer ones: lane i counts those before i */
		const int i = threadIdx.x & 63, n = i < p.d.B ? xa_len(p.d.k_len, i, p.d.Sk) : -1;
		int before = 0;
		for (int j = 0; j < p.d.B; ++j) {
			const int o = __builtin_amdgcn_readlane(n, j);
			before += o > n || (o == n && j < i);
		}
		b = __builtin_ctzll(__ballot(before == b && i < p.d.B));
	}
	bh = b * p.d.Hkv + hk;
}

/* the results of one part: for every (part, b * Hkv + h', row) DP sums,
 * then all rows' maxima and sums of weights */
__device__ __forceinline__ long long xa_prow(const XaArgs &p, int part, int bh, int r)
{
	return ((long long)part * (p.d.B * p.d.Hkv) + bh) * p.rows + r;
}

template <int KIND>
__device__ __forceinline__ void xa_out4(const XaArgs &p, long long at, int d, float4 v)
{
	if (d >= p.d.D)
		return;
	if (p.ovec) {
		if constexpr (KIND == S3K_F32)
			*(float4 *)((float *)p.d.out + at + d) = v;
		else
			*(uint2 *)((uint16_t *)p.d.out + at + d) = make_uint2(at_pack2<KIND>(v.x, v.y), at_pack2<KIND>(v.z, v.w));
		return;
	}
	const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
	for (int e = 0; e < 4; ++e) {
		if (d + e >= p.d.D)
			return;
		if constexpr (KIND == S3K_F32)
			((float *)p.d.out)[at + d + e] = x[e];
		else
			((uint16_t *)p.d.out)[at + d + e] = (uint16_t)at_pack2<KIND>(x[e], 0.0f);
	}
}

__device__ __forceinline__ long long xa_orow(const XaArgs &p, int bh, int r)
{
	const int b = bh / p.d.Hkv, hk = bh - b * p.d.Hkv, s = r / p.G, g = r - s * p.G;
	return b * p.d.o_b + s * p.d.o_s + (long long)(hk * p.G + g) * p.d.o_h;
}

/* ------------------------------------------------------------------ */
/* One wave per row: any D up to 256 and any alignment                   */
/* ------------------------------------------------------------------ */
template <int KIND>
__global__ void __launch_bounds__(256) xa_generic(XaArgs p)
{
	__shared__ float sq[4][256], sp[4][64];
	const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
	const long long row = (long long)blockIdx.x * 4 + w;
	const int bh = (int)(row / p.rows), r = (int)(row % p.rows);
	if (bh >= p.d.B * p.d.Hkv)
		return;
	const int b = bh / p.d.Hkv, hk = bh - b * p.d.Hkv, s = r / p.G, g = r - s * p.G, D = p.d.D;
	if (s >= xa_len(p.d.q_len, b, p.d.Sq))
		return;
	const int n = xa_len(p.d.k_len, b, p.d.Sk);
	const long long qat = b * p.d.q_b + s * p.d.q_s + (long long)(hk * p.G + g) * p.d.q_h;
	const long long kat = b * p.d.k_b + hk * p.d.k_h, vat = b * p.d.v_b + hk * p.d.v_h;
	for (int d = lane; d < D; d += 64)
		sq[w][d] = load_as_f32(p.d.q, qat + d, KIND);
	/* each wave uses its own LDS rows, and LDS works in order for a wave */
	__builtin_amdgcn_wave_barrier();
	float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = XA_NONE, l = 0.0f;
	for (int j0 = 0; j0 < n; j0 += 64) {
		const int j = j0 + lane;
		float sc = -__builtin_inff();
		if (j < n) {
			float acc = 0.0f;
			for (int d = 0; d < D; ++d)
				acc = fmaf(sq[w][d], load_as_f32(p.d.k, kat + j * p.d.k_s + d, KIND), acc);
			sc = acc * p.c;
		}
		const float mt = fmaxf(m, wave_max_f32(sc));
		const float al = __builtin_amdgcn_exp2f(m - mt), pr = __builtin_amdgcn_exp2f(sc - mt);
		m = mt;
		l = l * al + wave_xor_sum(pr);
		__builtin_amdgcn_wave_barrier();
		sp[w][lane] = pr;
		__builtin_amdgcn_wave_barrier();
		const int kn = min(64, n - j0);
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const int d = lane + 64 * i;
			if (d >= D)
				break;
			float acc = o[i] * al;
			for (int e = 0; e < kn; ++e)
				acc = fmaf(sp[w][e], load_as_f32(p.d.v, vat + (j0 + e) * p.d.v_s + d, KIND), acc);
			o[i] = acc;
		}
	}
	/* no key, or no score above -inf: zeros (a NaN sum stays one) */
	const float inv = 1.0f / l;
	const long long at = xa_orow(p, bh, r);
#pragma unroll
	for (int i = 0; i < 4; ++i)
		if (lane + 64 * i < D)
			store_from_f32(p.d.out, at + lane + 64 * i, KIND, l == 0.0f ? 0.0f : o[i] * inv);
}

/* ------------------------------------------------------------------ */
/* 16-bit MFMA                                                           */
/* ------------------------------------------------------------------ */
/*
 * A wave holds 32 rows. Scores are formed transposed, S^T = K Q^T
 * (v_mfma_f32_32x32x16): a lane then has one row (lane & 31) and 16 of 32
 * keys, so maxima and sums are in-lane plus one exchange with lane ^ 32,
 * and the probabilities are, as they lie, the P^T operand of
 * O^T = V^T P^T (its k order is permuted alike for both operands).
 * NWQ waves take different rows of the same keys (many rows), NWK waves
 * different key tiles for the same rows (few rows; each then loads its own
 * tiles and meets the others only when their results are merged through
 * LDS at the end). K and V tiles of KT keys arrive by direct-to-LDS loads,
 * chunks of 16 bytes XOR-swizzled by the key, in a ring of NST stages.
 * Keys past the length and columns past D read as zeros and cost no
 * traffic. A row has DP columns in LDS and in the parts, the products go
 * over DU of them (heads of 65 to 96: 96 of 128; 4 x 16 heads, 2000 x 2000
 * of 80 bf16 137 us over 128, 117 over 96; f32 335 and 282 at 4 x 8 heads,
 * 400 x 4000).
 */
template <int DP>
__device__ __forceinline__ int xa_kswz(int key)
{
	if constexpr (DP == 32)
		return (key >> 2) & 3;
	else if constexpr (DP == 64)
		return (key ^ (key >> 3)) & 7;
	else
		return key & 15;
}
template <int DP>
__device__ __forceinline__ int xa_vswz(int key)
{
	if constexpr (DP == 32)
		return 0;
	else if constexpr (DP == 64)
		return at_vswz(key);
	else
		return (key & 3) << 2;
}

/* The maximum moves, and the accumulators are rescaled, only when a score
 * passes it by more than this (in powers of two): probabilities then reach
 * 2^8, well inside f16, and most tiles pass without a rescale. */
constexpr float XA_SLACK = 8.0f;

template <int N>
struct xa_int {
	static constexpr int value = N;
};

template <int KIND, int DP, int DU, int NWQ, int NWK, int KT, int NST>
__global__ void __launch_bounds__(64 * NWQ * NWK, 8 / (NWQ * NWK)) xa_mfma(XaArgs p)
{
	/* waves that load a tile together: all, or (one wave of rows) each its own */
	constexpr bool PRIV = NWQ == 1;
	constexpr int LW = PRIV ? 1 : NWQ, CH = DP / 8, TB = KT * DP * 2, NMD = DU / 32, NC = DU / 16, NH = KT / 32;
	constexpr int FAM = KIND == S3K_F16 ? FAM_F16 : FAM_BF16;
	constexpr int TI = TB / 1024, PER = TI / LW; /* 1 KiB loads: per tile, per wave */
	static_assert(64 % CH == 0, "a load is whole rows");
	static_assert(NST == 2 || NST == 4, "the ring is unrolled");
	static_assert(TI % LW == 0 && (PRIV || NWK == 1), "loads divide over the waves");
	constexpr int MERGE = (NWK - 1) * NWQ * (NMD * 16 + 2) * 256, STAGE = 2 * TB;
	constexpr int RING = (PRIV ? NWK : 1) * NST * STAGE, LDS = RING > MERGE ? RING : MERGE;
	__shared__ __attribute__((aligned(1024))) char smem[LDS];
	const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int wq = wave % NWQ, wk = wave / NWQ;
	const int lw = PRIV ? 0 : wave; /* place among the waves that load */
	char *const ring = smem + (PRIV ? wk * NST * STAGE : 0);
	const unsigned lds0 = lds_addr_of(ring);

	int bh, part, rb;
	xa_place(p, blockIdx.x, bh, part, rb);
	const int b = bh / p.d.Hkv, hk = bh - b * p.d.Hkv;
	const int qn = xa_len(p.d.q_len, b, p.d.Sq) * p.G, kn = xa_len(p.d.k_len, b, p.d.Sk);
	const int rb0 = rb * 32 * NWQ;
	if (rb0 >= qn)
		return;
	const int r = rb0 + wq * 32 + l32;
	const bool wave_live = rb0 + wq * 32 < qn;

	/* Q^T operand: row r, d 16 c + 8 h onward */
	uint4 qf[NC];
	{
		const int s = r / p.G, g = r - s * p.G;
		const uint16_t *Q = (const uint16_t *)p.d.q + b * p.d.q_b + s * p.d.q_s +
				    (long long)(hk * p.G + g) * p.d.q_h;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			qf[c] = make_uint4(0, 0, 0, 0);
			if (r < qn && 16 * c + 8 * h < p.d.D)
				qf[c] = *(const uint4 *)(Q + 16 * c + 8 * h);
		}
	}

	/* this part's tiles */
	const int tiles = (kn + KT - 1) / KT;
	const int t0 = (int)((long long)tiles * part / p.ns), t1 = (int)((long long)tiles * (part + 1) / p.ns);
	const uint16_t *K0 = (const uint16_t *)p.d.k + b * p.d.k_b + hk * p.d.k_h;
	const uint16_t *V0 = (const uint16_t *)p.d.v + b * p.d.v_b + hk * p.d.v_h;
	/* load t: key row r0 + t RS of the tile, chunk (lane % CH) ^ swizzle.
	 * The row's distance from r0 is a scalar offset, so that loads whose
	 * swizzles agree share one lane offset. */
	constexpr int RS = LW * 64 / CH;
	const int r0 = (lw * 64 + lane) / CH, pos = lane % CH;
	unsigned koff[PER], voff[PER];
#pragma unroll
	for (int t = 0; t < PER; ++t) {
		const int kc = pos ^ xa_kswz<DP>(r0 + t * RS), vc = pos ^ xa_vswz<DP>(r0 + t * RS);
		koff[t] = 8 * kc < p.d.D ? (unsigned)(r0 * (int)p.d.k_s + 8 * kc) * 2u : S3K_OOB;
		voff[t] = 8 * vc < p.d.D ? (unsigned)(r0 * (int)p.d.v_s + 8 * vc) * 2u : S3K_OOB;
	}
	/* a tile (past the keys: zeros): every stage is the same number of loads
	 * to wait for */
	auto issue = [&](int tile, unsigned slot) {
		const int key0 = tile * KT;
		const s3k_i32x4 rk = buf_rsrc(K0 + key0 * p.d.k_s, 0x7FFFFFFFu);
		const s3k_i32x4 rv = buf_rsrc(V0 + key0 * p.d.v_s, 0x7FFFFFFFu);
#pragma unroll
		for (int t = 0; t < PER; ++t) {
			const unsigned at = lds0 + slot + (lw + t * LW) * 1024;
			const bool in = r0 < kn - key0 - t * RS;
			dma16s(at, rk, in ? koff[t] : S3K_OOB, (unsigned)(t * RS * (int)p.d.k_s) * 2u);
			dma16s(at + TB, rv, in ? voff[t] : S3K_OOB, (unsigned)(t * RS * (int)p.d.v_s) * 2u);
		}
	};

	/* LDS offsets within a tile: K row 32 mb + l32, chunk 2 c + h; V^T
	 * rows d = 32 md + (lane & 31), keys 16 cc + 4 h + {0..3} and + 8,
	 * by transposed reads: lane i of the 16-lane group q addresses key
	 * 4 (q >> 1) + i / 4, d 32 md + 16 (q & 1) + 4 (i % 4) */
	const int vg = lane >> 4, vi = lane & 15;

	s3k_f32x16 o[NMD];
#pragma unroll
	for (int md = 0; md < NMD; ++md)
#pragma unroll
		for (int e = 0; e < 16; ++e)
			o[md][e] = 0.0f;
	float m = XA_NONE, l = 0.0f; /* l: of this half of the lanes' keys */

	const int its = (t1 - t0 + NWK - 1) / NWK, tw = t0 + (PRIV ? wk : 0);
#pragma unroll
	for (int t = 0; t < NST - 1; ++t)
		issue(tw + t * NWK, t * STAGE);
	auto step = [&](auto par, int it) __attribute__((always_inline)) {
		constexpr unsigned slot = decltype(par)::value * STAGE, fill = (decltype(par)::value + NST - 1) % NST * STAGE;
		/* the tile has landed (everywhere past the barrier), and the stage
		 * filled now has been read */
		wait_vm<(NST - 2) * 2 * PER>();
		if constexpr (PRIV)
			asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
		else
			__syncthreads();
		issue(tw + (it + NST - 1) * NWK, fill);
		const char *const kt = ring + slot, *const vt = kt + TB;
		const int tile = t0 + it * NWK + wk;
		if (!wave_live || tile >= t1)
			return;
		const int key0 = tile * KT;

		s3k_f32x16 s[NH];
#pragma unroll
		for (int mb = 0; mb < NH; ++mb) {
#pragma unroll
			for (int e = 0; e < 16; ++e)
				s[mb][e] = 0.0f;
			const int row = 32 * mb + l32;
#pragma unroll
			for (int c = 0; c < NC; ++c)
				mfma_chunk<FAM>(s[mb], *(const uint4 *)(kt + row * DP * 2 + (((2 * c + h) ^ xa_kswz<DP>(row)) << 4)),
						qf[c]);
		}
		if (key0 + KT > kn) {
#pragma unroll
			for (int mb = 0; mb < NH; ++mb)
#pragma unroll
				for (int e = 0; e < 16; ++e)
					if (key0 + 32 * mb + 8 * (e >> 2) + 4 * h + (e & 3) >= kn)
						s[mb][e] = -__builtin_inff();
		}
		float mt = s[0][0];
#pragma unroll
		for (int mb = 0; mb < NH; ++mb)
#pragma unroll
			for (int e = 0; e < 16; ++e)
				mt = fmaxf(mt, s[mb][e]);
		mt = at_max_pair(mt) * p.c;
		if (__any(mt > m + XA_SLACK)) {
			const float mn = fmaxf(m, mt), al = __builtin_amdgcn_exp2f(m - mn);
			m = mn;
			l *= al;
#pragma unroll
			for (int md = 0; md < NMD; ++md)
#pragma unroll
				for (int e = 0; e < 16; ++e)
					o[md][e] *= al;
		}
#pragma unroll
		for (int mb = 0; mb < NH; ++mb)
#pragma unroll
			for (int sub = 0; sub < 2; ++sub) {
				float pv[8];
#pragma unroll
				for (int e = 0; e < 8; ++e)
					pv[e] = __builtin_amdgcn_exp2f(fmaf(s[mb][8 * sub + e], p.c, -m));
				const uint4 ph = make_uint4(at_pack2<KIND>(pv[0], pv[1]), at_pack2<KIND>(pv[2], pv[3]),
							    at_pack2<KIND>(pv[4], pv[5]), at_pack2<KIND>(pv[6], pv[7]));
				l = at_sum2<KIND>(ph.x, l), l = at_sum2<KIND>(ph.y, l);
				l = at_sum2<KIND>(ph.z, l), l = at_sum2<KIND>(ph.w, l);
				const int k16 = 32 * mb + 16 * sub;
#pragma unroll
				for (int md = 0; md < NMD; ++md) {
					uint2 v[2];
#pragma unroll
					for (int hl = 0; hl < 2; ++hl) {
						const int key = k16 + 4 * (vg >> 1) + (vi >> 2) + 8 * hl;
						const int d = 32 * md + 16 * (vg & 1) + 4 * (vi & 3);
						v[hl] = at_read_tr(vt, (unsigned)(key * DP * 2 + (((d >> 3) ^ xa_vswz<DP>(key)) << 4) +
										  ((d >> 2) & 1) * 8));
					}
					mfma_chunk<FAM>(o[md], make_uint4(v[0].x, v[0].y, v[1].x, v[1].y), ph);
				}
			}
	};
	for (int it = 0; it < its; it += NST) {
		step(xa_int<0>{}, it);
		if (it + 1 < its)
			step(xa_int<1>{}, it + 1);
		if constexpr (NST == 4) {
			if (it + 2 < its)
				step(xa_int<2>{}, it + 2);
			if (it + 3 < its)
				step(xa_int<3>{}, it + 3);
		}
	}
	wait_vm<0>(); /* the stages asked for past the part, all zeros */
	l = at_sum_pair(l);

	if constexpr (NWK > 1) {
		/* the other waves' results, [value][lane] */
		__syncthreads();
		float *mine = (float *)smem + ((wk - 1) * NWQ + wq) * (NMD * 16 + 2) * 64 + lane;
		if (wk > 0) {
#pragma unroll
			for (int md = 0; md < NMD; ++md)
#pragma unroll
				for (int e = 0; e < 16; ++e)
					mine[(md * 16 + e) * 64] = o[md][e];
			mine[NMD * 16 * 64] = m;
			mine[(NMD * 16 + 1) * 64] = l;
		}
		__syncthreads();
		if (wk > 0)
			return;
#pragma unroll
		for (int w = 0; w < NWK - 1; ++w) {
			const float *other = (const float *)smem + (w * NWQ + wq) * (NMD * 16 + 2) * 64 + lane;
			const float mo = other[NMD * 16 * 64], mn = fmaxf(m, mo);
			const float a0 = __builtin_amdgcn_exp2f(m - mn), a1 = __builtin_amdgcn_exp2f(mo - mn);
			m = mn;
			l = l * a0 + other[(NMD * 16 + 1) * 64] * a1;
#pragma unroll
			for (int md = 0; md < NMD; ++md)
#pragma unroll
				for (int e = 0; e < 16; ++e)
					o[md][e] = o[md][e] * a0 + other[(md * 16 + e) * 64] * a1;
		}
	}
	if (r >= qn)
		return;
	if (p.ns > 1) {
		const long long pr = xa_prow(p, part, bh, r), all = (long long)p.ns * (p.d.B * p.d.Hkv) * p.rows;
#pragma unroll
		for (int md = 0; md < NMD; ++md)
#pragma unroll
			for (int g = 0; g < 4; ++g)
				*(float4 *)(p.part + pr * DP + 32 * md + 8 * g + 4 * h) =
					make_float4(o[md][4 * g], o[md][4 * g + 1], o[md][4 * g + 2], o[md][4 * g + 3]);
		if (h == 0) {
			p.part[all * DP + pr] = m;
			p.part[all * (DP + 1) + pr] = l;
		}
		return;
	}
	/* no key, or no score above -inf: zeros, also where 0 * v is NaN */
	const bool none = l == 0.0f;
	const float inv = 1.0f / l;
	const long long at = xa_orow(p, bh, r);
#pragma unroll
	for (int md = 0; md < NMD; ++md)
#pragma unroll
		for (int g = 0; g < 4; ++g)
			xa_out4<KIND>(p, at, 32 * md + 8 * g + 4 * h,
				      make_float4(none ? 0.0f : o[md][4 * g] * inv, none ? 0.0f : o[md][4 * g + 1] * inv,
						  none ? 0.0f : o[md][4 * g + 2] * inv, none ? 0.0f : o[md][4 * g + 3] * inv));
}

/* ------------------------------------------------------------------ */
/* f32 MFMA                                                              */
/* ------------------------------------------------------------------ */
/*
 * v_mfma_f32_16x16x4_f32 keeps f32 products exact to a rounding. A wave
 * holds RT tiles of 16 rows and takes 16 UN keys at a time, straight from
 * memory into registers, without LDS, the next ones' loads under way (NB =
 * 2, where the registers allow): lane (i = lane & 15, g = lane >> 4)
 * reads 16 bytes of key i at d = 16 j + 4 g (k index g of the product with
 * element e is d = 16 j + 4 g + e for both operands), which gives S^T with
 * row i's scores of keys 4 g + 0..3 in its lane; they are the P^T operand
 * of O^T = V^T P^T as they lie when step e takes keys 4 g + e, whose V
 * values a lane reads VW at a time (d = 16 VW u + VW i + w in tile
 * u VW + w). Waves of a workgroup take different rows (NWQ) or different
 * keys (NWK), merged through LDS.
 */
constexpr int xa_f32_un(int dp)
{
	return dp == 16 ? 4 : dp == 32 ? 2 : 1;
}

template <int DP, int DU, int RT, int NWQ, int NWK>
__global__ void __launch_bounds__(64 * NWQ * NWK, 2) xa_f32(XaArgs p)
{
	constexpr int NT = DU / 16, VW = NT % 4 == 0 ? 4 : NT % 2 == 0 ? 2 : 1, NU = NT / VW;
	constexpr int UN = xa_f32_un(DP), KT = 16 * UN, NB = DP <= 64 ? 2 : 1;
	constexpr int MV = RT * (NT * 4 + 2); /* values a lane merges */
	/* long heads' scores in four sums: in one after the other 256 products
	 * left results of 1440 keys 1.7e-6 off, in four 0.3e-6 (2 % more time) */
	constexpr int NZ = DP >= 64 ? 4 : 1;
	/* results and sums of weights in two where registers allow, for the same
	 * reason (14418 keys in one part: 1.6e-6 off, so 1.2e-6; no more time) */
	constexpr int NO = DP <= 64 ? 2 : 1;
	__shared__ float red[NWK > 1 ? (NWK - 1) * NWQ * MV * 64 : 1];
	const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int wq = wave % NWQ, wk = wave / NWQ;
	int bh, part, rb;
	xa_place(p, blockIdx.x, bh, part, rb);
	const int b = bh / p.d.Hkv, hk = bh - b * p.d.Hkv, D = p.d.D;
	const int qn = xa_len(p.d.q_len, b, p.d.Sq) * p.G, kn = xa_len(p.d.k_len, b, p.d.Sk);
	const int rb0 = rb * 16 * RT * NWQ, rw = rb0 + wq * 16 * RT;
	if (rb0 >= qn)
		return;

	float4 qf[RT][NT];
#pragma unroll
	for (int t = 0; t < RT; ++t) {
		const int r = rw + 16 * t + i, s = r / p.G, hq = hk * p.G + r - s * p.G;
		const float *Q = (const float *)p.d.q + b * p.d.q_b + s * p.d.q_s + hq * p.d.q_h;
#pragma unroll
		for (int j = 0; j < NT; ++j) {
			qf[t][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			if (r < qn && 16 * j + 4 * g < D)
				qf[t][j] = *(const float4 *)(Q + 16 * j + 4 * g);
		}
	}
	const int tiles = (kn + KT - 1) / KT;
	const int t0 = (int)((long long)tiles * part / p.ns), t1 = (int)((long long)tiles * (part + 1) / p.ns);
	const float *K0 = (const float *)p.d.k + b * p.d.k_b + hk * p.d.k_h;
	const float *V0 = (const float *)p.d.v + b * p.d.v_b + hk * p.d.v_h;

	s3k_f32x4 os[NO][RT][NT];
	float m[RT], ls[NO][RT];
#pragma unroll
	for (int t = 0; t < RT; ++t) {
		m[t] = XA_NONE;
#pragma unroll
		for (int a = 0; a < NO; ++a) {
			ls[a][t] = 0.0f;
#pragma unroll
			for (int j = 0; j < NT; ++j)
				os[a][t][j] = (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f};
		}
	}
	float4 kf[NB][UN][NT];
	float vf[NB][UN][4][NU][VW];
	auto load = [&](auto buf, int tile) __attribute__((always_inline)) {
		constexpr int P = decltype(buf)::value;
#pragma unroll
		for (int n = 0; n < UN; ++n) {
			const int key0 = tile * KT + 16 * n, left = kn - key0;
			const float *Kr = K0 + (long long)(key0 + i) * p.d.k_s + 4 * g;
#pragma unroll
			for (int j = 0; j < NT; ++j) {
				kf[P][n][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				if (i < left && 16 * j + 4 * g < D)
					kf[P][n][j] = *(const float4 *)(Kr + 16 * j);
			}
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				const float *Vr = V0 + (long long)(key0 + 4 * g + e) * p.d.v_s;
#pragma unroll
				for (int u = 0; u < NU; ++u) {
					const int d = 16 * VW * u + VW * i;
					float (&x)[VW] = vf[P][n][e][u];
#pragma unroll
					for (int w = 0; w < VW; ++w)
						x[w] = 0.0f;
					/* D is a multiple of 4 and d of VW: all count or none */
					if (4 * g + e < left && d < D) {
						if constexpr (VW == 4) {
							const float4 y = *(const float4 *)(Vr + d);
							x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
						} else if constexpr (VW == 2) {
							const float2 y = *(const float2 *)(Vr + d);
							x[0] = y.x, x[1] = y.y;
						} else {
							x[0] = Vr[d];
						}
					}
				}
			}
		}
	};
	auto work = [&](auto buf, int tile) __attribute__((always_inline)) {
		constexpr int P = decltype(buf)::value;
		const int left = kn - tile * KT;
#pragma unroll
		for (int t = 0; t < RT; ++t) {
			s3k_f32x4 s[UN];
			float mt = -__builtin_inff();
#pragma unroll
			for (int n = 0; n < UN; ++n) {
				s3k_f32x4 z[NZ];
#pragma unroll
				for (int a = 0; a < NZ; ++a)
					z[a] = (s3k_f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
				for (int j = 0; j < NT; ++j) {
					z[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[P][n][j].x, qf[t][j].x, z[0], 0, 0, 0);
					z[1 % NZ] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[P][n][j].y, qf[t][j].y, z[1 % NZ], 0, 0, 0);
					z[2 % NZ] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[P][n][j].z, qf[t][j].z, z[2 % NZ], 0, 0, 0);
					z[3 % NZ] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[P][n][j].w, qf[t][j].w, z[3 % NZ], 0, 0, 0);
				}
				if constexpr (NZ == 4)
					s[n] = (z[0] + z[1]) + (z[2] + z[3]);
				else
					s[n] = z[0];
				if (left < KT) {
#pragma unroll
					for (int e = 0; e < 4; ++e)
						if (16 * n + 4 * g + e >= left)
							s[n][e] = -__builtin_inff();
				}
				mt = fmaxf(mt, fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3])));
			}
			mt *= p.c;
			mt = fmaxf(mt, __shfl_xor(mt, 16));
			mt = at_max_pair(mt);
			if (__any(mt > m[t] + XA_SLACK)) {
				const float mn = fmaxf(m[t], mt), al = __builtin_amdgcn_exp2f(m[t] - mn);
				m[t] = mn;
#pragma unroll
				for (int a = 0; a < NO; ++a) {
					ls[a][t] *= al;
#pragma unroll
					for (int j = 0; j < NT; ++j)
#pragma unroll
						for (int e = 0; e < 4; ++e)
							os[a][t][j][e] *= al;
				}
			}
#pragma unroll
			for (int n = 0; n < UN; ++n)
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					const float pe = __builtin_amdgcn_exp2f(fmaf(s[n][e], p.c, -m[t]));
					ls[e % NO][t] += pe;
#pragma unroll
					for (int u = 0; u < NU; ++u)
#pragma unroll
						for (int w = 0; w < VW; ++w)
							os[e % NO][t][u * VW + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(
								vf[P][n][e][u][w], pe, os[e % NO][t][u * VW + w], 0, 0, 0);
				}
		}
	};
	xa_int<0> b0;
	xa_int<NB - 1> b1;
	const int end = rw < qn ? t1 : 0;
	int tile = t0 + wk;
	if constexpr (NB == 1) {
		for (; tile < end; tile += NWK) {
			load(b0, tile);
			work(b0, tile);
		}
	} else {
		if (tile < end)
			load(b0, tile);
		for (; tile < end; tile += 2 * NWK) {
			if (tile + NWK < end)
				load(b1, tile + NWK);
			work(b0, tile);
			if (tile + NWK >= end)
				break;
			if (tile + 2 * NWK < end)
				load(b0, tile + 2 * NWK);
			work(b1, tile + NWK);
		}
	}
	s3k_f32x4 (&o)[RT][NT] = os[0];
	float (&l)[RT] = ls[0];
#pragma unroll
	for (int t = 0; t < RT; ++t) {
#pragma unroll
		for (int a = 1; a < NO; ++a) {
			l[t] += ls[a][t];
#pragma unroll
			for (int j = 0; j < NT; ++j)
				o[t][j] += os[a][t][j];
		}
		l[t] += __shfl_xor(l[t], 16);
		l[t] = at_sum_pair(l[t]);
	}
	if constexpr (NWK > 1) {
		if (wk > 0) {
			float *mine = red + ((wk - 1) * NWQ + wq) * MV * 64 + lane;
#pragma unroll
			for (int t = 0; t < RT; ++t) {
#pragma unroll
				for (int j = 0; j < NT; ++j)
#pragma unroll
					for (int e = 0; e < 4; ++e)
						mine[(t * (NT * 4 + 2) + j * 4 + e) * 64] = o[t][j][e];
				mine[(t * (NT * 4 + 2) + NT * 4) * 64] = m[t];
				mine[(t * (NT * 4 + 2) + NT * 4 + 1) * 64] = l[t];
			}
		}
		__syncthreads();
		if (wk > 0)
			return;
#pragma unroll
		for (int w = 0; w < NWK - 1; ++w) {
			const float *other = red + (w * NWQ + wq) * MV * 64 + lane;
#pragma unroll
			for (int t = 0; t < RT; ++t) {
				const float mo = other[(t * (NT * 4 + 2) + NT * 4) * 64], mn = fmaxf(m[t], mo);
				const float a0 = __builtin_amdgcn_exp2f(m[t] - mn), a1 = __builtin_amdgcn_exp2f(mo - mn);
				m[t] = mn;
				l[t] = l[t] * a0 + other[(t * (NT * 4 + 2) + NT * 4 + 1) * 64] * a1;
#pragma unroll
				for (int j = 0; j < NT; ++j)
#pragma unroll
					for (int e = 0; e < 4; ++e)
						o[t][j][e] = o[t][j][e] * a0 + other[(t * (NT * 4 + 2) + j * 4 + e) * 64] * a1;
			}
		}
	}
#pragma unroll
	for (int t = 0; t < RT; ++t) {
		const int r = rw + 16 * t + i;
		if (r >= qn)
			continue;
		const bool none = p.ns == 1 && l[t] == 0.0f;
		const float inv = p.ns > 1 ? 1.0f : 1.0f / l[t];
		const long long pr = xa_prow(p, part, bh, r), all = (long long)p.ns * (p.d.B * p.d.Hkv) * p.rows;
		const long long at = xa_orow(p, bh, r);
		/* tile u VW + w, register e: d = 16 VW u + VW (4 g + e) + w. As
		 * runs of 4: VW = 4 by e, 2 by pairs of e, 1 all e */
#pragma unroll
		for (int u = 0; u < NU; ++u)
#pragma unroll
			for (int n = 0; n < VW; ++n) {
				float v[4];
#pragma unroll
				for (int x = 0; x < 4; ++x)
					v[x] = none ? 0.0f : o[t][u * VW + x % VW][n * (4 / VW) + x / VW] * inv;
				const int d = 16 * VW * u + VW * 4 * g + 4 * n;
				const float4 v4 = make_float4(v[0], v[1], v[2], v[3]);
				if (p.ns > 1)
					*(float4 *)(p.part + pr * DP + d) = v4;
				else
					xa_out4<S3K_F32>(p, at, d, v4);
			}
		if (p.ns > 1 && g == 0) {
			p.part[all * DP + pr] = m[t];
			p.part[all * (DP + 1) + pr] = l[t];
		}
	}
}

/* o / l; a row of no key, or no score above -inf: zeros, also where o is NaN
 * (0 times an infinite v) */
__device__ __forceinline__ float4 xa_over(const float4 &o, float l)
{
	const float inv = 1.0f / l;
	return l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

/* The parts of a row joined, many rows: DP / 4 lanes take a row, four
 * values each, part by part. */
template <int KIND, int DP>
__global__ void __launch_bounds__(256) xa_join_many(XaArgs p)
{
	constexpr int L = DP / 4;
	const long long rows = (long long)(p.d.B * p.d.Hkv) * p.rows, row = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
	if (row >= rows)
		return;
	const int bh = (int)(row / p.rows), r = (int)(row - (long long)bh * p.rows), d = threadIdx.x % L * 4;
	if (r >= xa_len(p.d.q_len, bh / p.d.Hkv, p.d.Sq) * p.G)
		return;
	const float *pm = p.part + rows * p.ns * DP, *pl = pm + rows * p.ns;
	float m = XA_NONE;
	for (int s = 0; s < p.ns; ++s)
		m = fmaxf(m, pm[s * rows + row]);
	float l = 0.0f;
	float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
	for (int s = 0; s < p.ns; ++s) {
		const float a = __builtin_amdgcn_exp2f(pm[s * rows + row] - m);
		const float4 v = *(const float4 *)(p.part + (s * rows + row) * DP + d);
		l = fmaf(pl[s * rows + row], a, l);
		o.x = fmaf(v.x, a, o.x), o.y = fmaf(v.y, a, o.y), o.z = fmaf(v.z, a, o.z), o.w = fmaf(v.w, a, o.w);
	}
	xa_out4<KIND>(p, xa_orow(p, bh, r), d, xa_over(o, l));
}

/*
 * The parts of a row joined, few rows: a workgroup per row, DP / 4 lanes with
 * four values each times 16 groups. A group takes every 16th part, all asked
 * for at once (with 4 groups and loads one after the other 2 x 4 heads, 5000
 * keys of 256 took 21.3 us, so 19.3), and the groups are added up in LDS in
 * order.
 */
template <int KIND, int DP>
__global__ void __launch_bounds__(4 * DP) xa_join(XaArgs p)
{
	constexpr int L = DP / 4, NG = 16, NP = XA_PARTS / NG;
	static_assert(XA_PARTS <= 64, "a wave reads all maxima at once");
	__shared__ float4 so[NG][L];
	__shared__ float sl[NG];
	const long long rows = (long long)(p.d.B * p.d.Hkv) * p.rows, row = blockIdx.x;
	const int bh = (int)(row / p.rows), r = (int)(row - (long long)bh * p.rows);
	if (r >= xa_len(p.d.q_len, bh / p.d.Hkv, p.d.Sq) * p.G)
		return;
	const float *pm = p.part + rows * p.ns * DP, *pl = pm + rows * p.ns;
	const int li = threadIdx.x % L, grp = threadIdx.x / L, lane = threadIdx.x & 63;
	float4 v[NP];
	float vm[NP], vl[NP];
#pragma unroll
	for (int i = 0; i < NP; ++i) {
		const int s = grp + NG * i;
		v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), vm[i] = XA_NONE, vl[i] = 0.0f;
		if (s < p.ns) {
			const long long at = s * rows + row;
			v[i] = *(const float4 *)(p.part + at * DP + 4 * li);
			vm[i] = pm[at], vl[i] = pl[at];
		}
	}
	const float m = wave_max_f32(lane < p.ns ? pm[lane * rows + row] : XA_NONE);
	float l = 0.0f;
	float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
	for (int i = 0; i < NP; ++i) {
		const float a = __builtin_amdgcn_exp2f(vm[i] - m);
		l = fmaf(vl[i], a, l);
		o.x = fmaf(v[i].x, a, o.x), o.y = fmaf(v[i].y, a, o.y);
		o.z = fmaf(v[i].z, a, o.z), o.w = fmaf(v[i].w, a, o.w);
	}
	so[grp][li] = o;
	if (li == 0)
		sl[grp] = l;
	__syncthreads();
	if (grp > 0)
		return;
	const int n = p.ns < NG ? p.ns : NG;
	for (int g = 1; g < n; ++g) {
		const float4 u = so[g][li];
		o.x += u.x, o.y += u.y, o.z += u.z, o.w += u.w;
		l += sl[g];
	}
	xa_out4<KIND>(p, xa_orow(p, bh, r), 4 * li, xa_over(o, l));
}

} /* namespace s3k */

using namespace s3k;

namespace {

int xa_dp(int D)
{
	return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256;
}

bool xa_16(const void *p, long long strides, int es)
{
	return (uintptr_t)p % 16 == 0 && strides * es % 16 == 0;
}

/* Waves along the rows and along the keys, and keys per step. */
struct XaShape {
	int dp, rows, nwk, kt, fit; /* fit: workgroups a CU */
};

XaShape xa_shape(const struct s3k_xattn *d, int path)
{
	XaShape s = {xa_dp(d->D), 0, 1, 16, 2};
	const long long rows = (long long)d->Sq * (d->H / d->Hkv);
	if (path == S3K_XATTN_MFMA) {
		if (s.dp < 32)
			s.dp = 32;
		const bool few = rows <= 32;
		s.rows = few ? 32 : 128;
		s.nwk = few ? (s.dp == 256 ? 2 : 4) : 1;
		s.kt = few || s.dp == 256 ? 32 : 64;
		s.fit = few && s.dp >= 128 ? 1 : 2;
	} else if (path == S3K_XATTN_F32) {
		const bool few = rows <= 16;
		s.rows = few ? 16 : s.dp == 256 ? 64 : 128;
		s.nwk = few ? 4 : 1;
		s.kt = 16 * xa_f32_un(s.dp);
	}
	return s;
}

template <int KIND, int DP, int DU>
int xa_go16(const XaArgs &a, const XaShape &s, unsigned blocks, hipStream_t st)
{
	if (s.rows == 32) {
		constexpr int NWK = DP == 256 ? 2 : 4, NST = DP == 32 ? 4 : 2;
		hipLaunchKernelGGL((xa_mfma<KIND, DP, DU, 1, NWK, 32, NST>), dim3(blocks), dim3(64 * NWK), 0, st, a);
	} else {
		constexpr int KT = DP == 256 ? 32 : 64;
		hipLaunchKernelGGL((xa_mfma<KIND, DP, DU, 4, 1, KT, 2>), dim3(blocks), dim3(256), 0, st, a);
	}
	return (int)hipGetLastError();
}

template <int KIND>
int xa_go16(const XaArgs &a, const XaShape &s, unsigned blocks, hipStream_t st)
{
	switch (s.dp) {
	case 32: return xa_go16<KIND, 32, 32>(a, s, blocks, st);
	case 64: return xa_go16<KIND, 64, 64>(a, s, blocks, st);
	case 128:
		return a.d.D <= 96 ? xa_go16<KIND, 128, 96>(a, s, blocks, st) : xa_go16<KIND, 128, 128>(a, s, blocks, st);
	default: return xa_go16<KIND, 256, 256>(a, s, blocks, st);
	}
}

template <int DP, int DU>
int xa_gof(const XaArgs &a, const XaShape &s, unsigned blocks, hipStream_t st)
{
	if (s.rows == 16)
		hipLaunchKernelGGL((xa_f32<DP, DU, 1, 1, 4>), dim3(blocks), dim3(256), 0, st, a);
	else
		hipLaunchKernelGGL((xa_f32<DP, DU, DP == 256 ? 1 : 2, 4, 1>), dim3(blocks), dim3(256), 0, st, a);
	return (int)hipGetLastError();
}

template <int KIND, int DP>
int xa_joined(const XaArgs &a, hipStream_t st)
{
	const long long rows = (long long)a.d.B * a.d.Hkv * a.rows, per = 256 / (DP / 4);
	/* whole calls of 4000 keys, 256 rows of 64 values: 16.6 us by lanes, 11.9
	 * by workgroups; 2048 of 256 46.0 and 45.8; 4096 of 256 51 and 56 */
	if (rows > 2048)
		hipLaunchKernelGGL((xa_join_many<KIND, DP>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, st, a);
	else
		hipLaunchKernelGGL((xa_join<KIND, DP>), dim3((unsigned)rows), dim3(4 * DP), 0, st, a);
	return (int)hipGetLastError();
}

template <int KIND>
int xa_joined(const XaArgs &a, int dp, hipStream_t st)
{
	switch (dp) {
	case 16: return xa_joined<KIND, 16>(a, st);
	case 32: return xa_joined<KIND, 32>(a, st);
	case 64: return xa_joined<KIND, 64>(a, st);
	case 128: return xa_joined<KIND, 128>(a, st);
	default: return xa_joined<KIND, 256>(a, st);
	}
}

} /* namespace */

extern "C" int s3k_xattn_can(const struct s3k_xattn *d, int path)
{
	const int es = d->kind == S3K_F32 ? 4 : 2;
	const long long qs = d->q_b | d->q_s | d->q_h, ks = d->k_b | d->k_s | d->k_h, vs = d->v_b | d->v_s | d->v_h;
	const bool vec = xa_16(d->q, qs, es) && xa_16(d->k, ks, es) && xa_16(d->v, vs, es) && d->D <= 256;
	switch (path) {
	case S3K_XATTN_MFMA:
		/* 32-bit offsets within a tile of at most 64 keys */
		return d->kind != S3K_F32 && d->D % 8 == 0 && vec && d->k_s <= 1 << 23 && d->v_s <= 1 << 23;
	case S3K_XATTN_F32: return d->kind == S3K_F32 && d->D % 4 == 0 && vec;
	case S3K_XATTN_GENERIC: return d->D <= 256;
	}
	return 0;
}

extern "C" int s3k_xattn_path(const struct s3k_xattn *d)
{
	for (int path = S3K_XATTN_MFMA; path <= S3K_XATTN_GENERIC; ++path)
		if (s3k_xattn_can(d, path))
			return path;
	return 0;
}

extern "C" int s3k_xattn_parts(const struct s3k_xattn *d, int path)
{
	if (path == S3K_XATTN_GENERIC || d->Sk == 0)
		return 1;
	const XaShape s = xa_shape(d, path);
	const long long rows = (long long)d->Sq * (d->H / d->Hkv);
	const long long wgs = (rows + s.rows - 1) / s.rows * d->B * d->Hkv;
	/* the places for workgroups filled once. Many rows: each with at least
	 * four steps (400 rows x 1000 keys 14.9 us, with one 18.4); few rows: with
	 * one (2000 keys 8.5 us, with four 10.2), from four on (500 keys 6.9 us
	 * in one part, 8.0 in two), and no more parts than a join reads quickly
	 * (40000 keys 16.4 us in 78, 19.3 in 128) */
	const long long step = (long long)s.kt * s.nwk, few = s.nwk > 1;
	long long parts = 256 * s.fit / (wgs ? wgs : 1);
	const long long most = few ? (d->Sk >= 4 * step ? d->Sk / step : 1) : d->Sk / (4 * step);
	if (parts > most)
		parts = most;
	if (parts > XA_PARTS)
		parts = XA_PARTS;
	return parts < 2 ? 1 : (int)parts;
}

extern "C" size_t s3k_xattn_bytes(const struct s3k_xattn *d, int path, int parts)
{
	if (parts < 2)
		return 0;
	return (size_t)parts * d->B * d->H * d->Sq * (xa_shape(d, path).dp + 2) * 4;
}

extern "C" int s3k_xattn_run(const struct s3k_xattn *d, int path, int parts, void *work, void *stream)
{
	XaArgs a;
	a.d = *d;
	a.G = d->H / d->Hkv;
	const long long rows = (long long)d->Sq * a.G, bh = (long long)d->B * d->Hkv;
	if (rows == 0 || bh == 0)
		return (int)hipSuccess;
	if (rows > 0x3FFFFFFFll)
		return (int)hipErrorInvalidValue;
	a.rows = (int)rows;
	a.ns = parts;
	a.part = (float *)work;
	a.c = d->scale * 1.44269504088896341f;
	a.ovec = d->D % 4 == 0 && (uintptr_t)d->out % (d->kind == S3K_F32 ? 16 : 8) == 0 &&
		 (d->o_b | d->o_s | d->o_h) % 4 == 0;
	hipStream_t st = (hipStream_t)stream;
	if (path == S3K_XATTN_GENERIC) {
		const long long blocks = (rows * bh + 3) / 4;
		if (!s3k_launchable(blocks, 256))
			return (int)hipErrorInvalidValue;
		a.nrb = 0;
		switch (d->kind) {
		case S3K_F32: hipLaunchKernelGGL((xa_generic<S3K_F32>), dim3((unsigned)blocks), dim3(256), 0, st, a); break;
		case S3K_F16: hipLaunchKernelGGL((xa_generic<S3K_F16>), dim3((unsigned)blocks), dim3(256), 0, st, a); break;
		default: hipLaunchKernelGGL((xa_generic<S3K_BF16>), dim3((unsigned)blocks), dim3(256), 0, st, a); break;
		}
		return (int)hipGetLastError();
	}
	const XaShape s = xa_shape(d, path);
	const long long nrb = (rows + s.rows - 1) / s.rows, blocks = nrb * bh * parts;
	if (!s3k_launchable(blocks, 256))
		return (int)hipErrorInvalidValue;
	a.nrb = (int)nrb;
	const int es = d->kind == S3K_F32 ? 4 : 2;
	a.run = 1;
	while (d->Hkv % (2 * a.run) == 0 && 2 * a.run * d->k_h * es <= 256)
		a.run *= 2;
	/* 16 x 8 heads, 533 rows, lengths to 3931 of 64: 94 us, sorted 82 to 88;
	 * two sequences gain nothing, and short ones lose to the counting (60 x 8
	 * heads, 300 rows, to 500: 34.0 and 35.3) */
	a.sort = parts == 1 && d->k_len && d->B > 2 && d->B <= 64 && d->Sk >= 1024 && blocks > 256;
	int rc;
	if (path == S3K_XATTN_MFMA) {
		rc = d->kind == S3K_F16 ? xa_go16<S3K_F16>(a, s, (unsigned)blocks, st)
					: xa_go16<S3K_BF16>(a, s, (unsigned)blocks, st);
	} else {
		switch (s.dp) {
		case 16: rc = xa_gof<16, 16>(a, s, (unsigned)blocks, st); break;
		case 32: rc = xa_gof<32, 32>(a, s, (unsigned)blocks, st); break;
		case 64: rc = xa_gof<64, 64>(a, s, (unsigned)blocks, st); break;
		case 128:
			rc = d->D <= 96 ? xa_gof<128, 96>(a, s, (unsigned)blocks, st) : xa_gof<128, 128>(a, s, (unsigned)blocks, st);
			break;
		default: rc = xa_gof<256, 256>(a, s, (unsigned)blocks, st); break;
		}
	}
	if (rc != (int)hipSuccess || parts < 2)
		return rc;
	switch (d->kind) {
	case S3K_F32: return xa_joined<S3K_F32>(a, s.dp, st);
	case S3K_F16: return xa_joined<S3K_F16>(a, s.dp, st);
	default: return xa_joined<S3K_BF16>(a, s.dp, st);
	}
}
