/*
 * attn_dev.h - device helpers shared by the attention kernels (attn.hip,
 * xattn.hip).
 */
#ifndef SAM3_ATTN_DEV_H
#define SAM3_ATTN_DEV_H

#include "s3k.h"
#include "s3k_dev.h"

namespace s3k {

template <int DT>
__device__ __forceinline__ uint32_t at_pack2(float lo, float hi)
{
	if constexpr (DT == S3K_F16)
		return pack_f16x2(lo, hi);
	else
		return pack_bf16x2(lo, hi);
}

/* f32 sum of the two 16-bit values of w, added to acc (v_dot2 with 1, 1) */
template <int DT>
__device__ __forceinline__ float at_sum2(uint32_t w, float acc)
{
	if constexpr (DT == S3K_F16) {
		typedef _Float16 h2 __attribute__((ext_vector_type(2)));
		const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
		return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), one, acc, false);
	} else {
		const s3k_bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
		return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s3k_bf16x2, w), one, acc, false);
	}
}

/* Chunk swizzle of a direct-to-LDS V tile row: it depends on the key's
 * low four bits only, so the transposed reads of the four 16-key chunks
 * of a tile differ by a constant offset. */
__device__ __forceinline__ int at_vswz(int key)
{
	const int r = key & 15;
	return (r ^ (r >> 3)) & 7;
}

typedef short at_v4i16 __attribute__((ext_vector_type(4)));

/* ds_read_b64_tr_b16: within each group of 16 lanes, lane i receives
 * element i % 4 of the 8 bytes addressed by lanes i / 4, 4 + i / 4,
 * 8 + i / 4 and 12 + i / 4 (measured on gfx950). */
__device__ __forceinline__ uint2 at_read_tr(const char *smem, unsigned off)
{
	const at_v4i16 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
		(__attribute__((address_space(3))) at_v4i16 *)((__attribute__((address_space(3))) char *)
								       smem + off));
	return __builtin_bit_cast(uint2, r);
}

/* x combined with the value of lane ^ 32 (v_permlane32_swap) */
__device__ __forceinline__ float at_max_pair(float x)
{
	const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
	return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float at_sum_pair(float x)
{
	const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
	return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

} /* namespace s3k */

#endif /* SAM3_ATTN_DEV_H */
