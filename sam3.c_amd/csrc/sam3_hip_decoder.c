/*
 * sam3_hip_decoder.c - C11 host side of the operators of a decoder that
 * reads an encoder's states: e4m3 linear layers, norm and rotation of
 * queries and keys, cross attention. Argument checks, work space and the
 * choice of the kernel; errors as in sam3_hip_ops.c (SAM3_EINVAL before
 * any launch, SAM3_EDTYPE for a type without a kernel).
 */
#include "sam3_hip.h"
#include "sam3_hip_internal.h"
#include "s3k.h"

#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdint.h>

static int is_float_dtype(int dt)
{
	return dt == SAM3_DTYPE_F32 || dt == SAM3_DTYPE_F16 || dt == SAM3_DTYPE_BF16;
}

static uintptr_t esize(int dt)
{
	return dt == SAM3_DTYPE_F32 ? 4 : 2;
}

/* Whether work on stream is being captured, or that cannot be told. */
static int captured(void *stream)
{
	hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
	if (hipStreamIsCapturing((hipStream_t)stream, &cs) != hipSuccess) {
		(void)hipGetLastError();
		return 1;
	}
	return cs != hipStreamCaptureStatusNone;
}

#define REFUSE(code, ...)                \
	do {                             \
		s3h_error(__VA_ARGS__);  \
		return code;             \
	} while (0)

/* ------------------------------------------------------------------ */
/* e4m3 linear layers                                                   */
/* ------------------------------------------------------------------ */
#define FP8_MAX_K (1 << 22) /* 256 rows of a tile stay below 2^31 bytes */
#define FP8_MAX_ROWS (1 << 30) /* of either operand: a tile's last row is an int */

/* The result of a launcher: one that finds more workgroups than a launch
 * takes returns hipErrorInvalidValue before any. */
static enum sam3_error launched(int e, const char *what)
{
	if (e == hipErrorInvalidValue)
		REFUSE(SAM3_EINVAL, "%s: more workgroups than one launch takes", what);
	return s3h_hip(e, what);
}

static enum sam3_error fp8_quant_check(const char *what, int dtype, const void *x, long long ld,
				       int rows, int K, const void *q, const void *scale)
{
	if (!is_float_dtype(dtype))
		REFUSE(SAM3_EDTYPE, "%s: dtype %d is not F32, F16 or BF16", what, dtype);
	if (rows < 0 || rows > FP8_MAX_ROWS || K < 0 || K > FP8_MAX_K || ld < K)
		REFUSE(SAM3_EINVAL, "%s: rows=%d K=%d ld=%lld", what, rows, K, ld);
	if (rows == 0 || K == 0)
		return SAM3_OK;
	if (!x || !q || !scale)
		REFUSE(SAM3_EINVAL, "%s: NULL pointer", what);
	if ((uintptr_t)x % esize(dtype) || (uintptr_t)q % 16 || (uintptr_t)scale % 4)
		REFUSE(SAM3_EINVAL, "%s: x must be element-aligned, q 16-byte and scale 4-byte aligned",
		       what);
	return SAM3_OK;
}

enum sam3_error sam3_hip_fp8_quantize(int x_dtype, const void *x, long long ldx, int rows, int K,
				      void *q, float *scale, void *stream)
{
	const enum sam3_error err = fp8_quant_check("fp8_quantize", x_dtype, x, ldx, rows, K, q, scale);
	if (err != SAM3_OK)
		return err;
	return launched(s3k_fp8_quantize(x_dtype, x, ldx, rows, K, q, scale, stream), "fp8_quantize");
}

enum sam3_error sam3_hip_fp8_quantize_weight(int w_dtype, const void *w, long long ldw, int N, int K,
					     void *q, float *scale, void *stream)
{
	const enum sam3_error err =
		fp8_quant_check("fp8_quantize_weight", w_dtype, w, ldw, N, K, q, scale);
	if (err != SAM3_OK)
		return err;
	return launched(s3k_fp8_quantize_weight(w_dtype, w, ldw, N, K, q, scale, stream),
		       "fp8_quantize_weight");
}

/* What both products ask of their weights, output and bias. */
static enum sam3_error fp8_product_check(const char *what, const void *w, const void *w_scale,
					 int c_dtype, const void *c, int M, int N, int K,
					 const void *bias, int flags)
{
	if (!is_float_dtype(c_dtype))
		REFUSE(SAM3_EDTYPE, "%s: output dtype %d is not F32, F16 or BF16", what, c_dtype);
	if (M < 0 || M > FP8_MAX_ROWS || N < 0 || N > FP8_MAX_ROWS || K < 0 || K > FP8_MAX_K)
		REFUSE(SAM3_EINVAL, "%s: M=%d N=%d K=%d", what, M, N, K);
	if (flags & ~(SAM3_HIP_BIAS | SAM3_HIP_GELU))
		REFUSE(SAM3_EINVAL, "%s: unknown flags %d", what, flags);
	if (M == 0 || N == 0)
		return SAM3_OK;
	if (!c || (K > 0 && (!w || !w_scale)) || ((flags & SAM3_HIP_BIAS) && !bias))
		REFUSE(SAM3_EINVAL, "%s: NULL pointer", what);
	if ((uintptr_t)w % 16 || (uintptr_t)w_scale % 4 || (uintptr_t)c % esize(c_dtype) ||
	    ((flags & SAM3_HIP_BIAS) && (uintptr_t)bias % esize(c_dtype)))
		REFUSE(SAM3_EINVAL, "%s: w must be 16-byte, w_scale 4-byte, c and bias element-aligned",
		       what);
	return SAM3_OK;
}

enum sam3_error sam3_hip_matmul_fp8(const void *a, const float *a_scale, const void *w,
				    const float *w_scale, int c_dtype, void *c, int M, int N, int K,
				    const void *bias, int flags, void *stream)
{
	const enum sam3_error err =
		fp8_product_check("matmul_fp8", w, w_scale, c_dtype, c, M, N, K, bias, flags);
	if (err != SAM3_OK)
		return err;
	if (M > 0 && N > 0 && K > 0 && (!a || !a_scale))
		REFUSE(SAM3_EINVAL, "matmul_fp8: NULL pointer");
	if ((uintptr_t)a % 16 || (uintptr_t)a_scale % 4)
		REFUSE(SAM3_EINVAL, "matmul_fp8: a must be 16-byte, a_scale 4-byte aligned");
	return launched(s3k_fp8_matmul(a, a_scale, w, w_scale, c_dtype, c, M, N, K, bias, flags, stream),
		       "matmul_fp8");
}

/* Bytes of the e4m3 rows, and of them with the scales. */
static size_t fp8_rows_bytes(int M, int K, size_t *total)
{
	const size_t kb = ((size_t)K + 127) / 128, q = (size_t)M * kb * 128;
	*total = q + (size_t)M * kb * 4;
	return q;
}

size_t sam3_hip_linear_fp8_work(int M, int N, int K)
{
	size_t total;
	if (M <= 0 || N <= 0 || K <= 0)
		return 0;
	(void)fp8_rows_bytes(M, K, &total);
	return total;
}

enum sam3_error sam3_hip_linear_fp8(int x_dtype, const void *x, long long ldx, const void *w,
				    const float *w_scale, int c_dtype, void *c, int M, int N, int K,
				    const void *bias, int flags, void *work, size_t work_bytes,
				    void *stream)
{
	if (!is_float_dtype(x_dtype))
		REFUSE(SAM3_EDTYPE, "linear_fp8: dtype %d is not F32, F16 or BF16", x_dtype);
	enum sam3_error err =
		fp8_product_check("linear_fp8", w, w_scale, c_dtype, c, M, N, K, bias, flags);
	if (err != SAM3_OK)
		return err;
	if (ldx < K)
		REFUSE(SAM3_EINVAL, "linear_fp8: rows of %d values %lld apart", K, ldx);
	if (M == 0 || N == 0)
		return SAM3_OK;
	if (K > 0 && (!x || (uintptr_t)x % esize(x_dtype)))
		REFUSE(SAM3_EINVAL, "linear_fp8: x is NULL or not element-aligned");
	/* Every workgroup quantizes its 16 rows of x again: with more than 256
	 * blocks of x a launch of its own is quicker (16 x 4096 x 4096 6.7 us,
	 * inside 7.8; 8 x 4096 x 4096 6.4 and 6.3; 64 x 1024 x 512 4.9 and 3.2), and
	 * with many workgroups for more than 16 rows (64 x 8192 x 512 6.7 and 8.0;
	 * 64 x 4096 x 512 6.3 and 5.2). */
	const long long wgs = ((N + 15ll) / 16) * ((M + 15ll) / 16);
	const int inside = (long long)M * ((K + 127) / 128) <= 256 && (M <= 16 || wgs <= 1024);
	if (s3k_fp8_rows_ok(M, K) && (inside || (!work && captured(stream))))
		return launched(s3k_fp8_rows(x_dtype, x, ldx, w, w_scale, c_dtype, c, M, N, K, bias, flags,
					    stream),
			       "linear_fp8");
	size_t need;
	const size_t scales = fp8_rows_bytes(M, K, &need);
	void *own = NULL;
	if (work && (work_bytes < need || (uintptr_t)work % 16))
		REFUSE(SAM3_EINVAL, "linear_fp8: %zu bytes of work space, %zu needed (16-byte aligned)",
		       work_bytes, need);
	if (!work && need) {
		if (captured(stream))
			REFUSE(SAM3_EINVAL, "linear_fp8: a captured call of %d rows of %d values needs %zu "
			       "bytes of work space from the caller", M, K, need);
		err = s3h_scratch_alloc(&own, need, stream);
		if (err != SAM3_OK)
			return err;
		work = own;
	}
	float *scale = (float *)((char *)work + scales);
	err = launched(s3k_fp8_quantize(x_dtype, x, ldx, M, K, work, scale, stream), "linear_fp8 quantize");
	if (err == SAM3_OK)
		err = launched(s3k_fp8_matmul(work, scale, w, w_scale, c_dtype, c, M, N, K, bias, flags,
					     stream),
			      "linear_fp8");
	const enum sam3_error ferr = s3h_scratch_free(own, stream);
	return err != SAM3_OK ? err : ferr;
}

/* ------------------------------------------------------------------ */
/* Norm and rotation of queries and keys                                */
/* ------------------------------------------------------------------ */
/* Strides of [B, S, heads] outputs: none negative, none zero along an
 * axis of more than one. */
static int out_strides_ok(long long b, long long s, long long h, int B, int S, int heads)
{
	return b >= 0 && s >= 0 && h >= 0 && (B < 2 || b) && (S < 2 || s) && (heads < 2 || h);
}

static enum sam3_error heads_check(const struct sam3_hip_norm_rope *p, const struct sam3_hip_heads *t,
				   const char *name)
{
	const uintptr_t es = esize(p->dtype);
	if (t->heads < 0)
		REFUSE(SAM3_EINVAL, "norm_rope: %s has %d heads", name, t->heads);
	if (t->heads == 0 || p->B == 0 || p->S == 0)
		return SAM3_OK;
	if (!t->in || !t->out)
		REFUSE(SAM3_EINVAL, "norm_rope: %s is NULL", name);
	if ((uintptr_t)t->in % es || (uintptr_t)t->out % es || (p->norm && (uintptr_t)t->weight % es))
		REFUSE(SAM3_EINVAL, "norm_rope: %s must be element-aligned", name);
	if (t->in_b < 0 || t->in_s < 0 || t->in_h < 0 ||
	    !out_strides_ok(t->out_b, t->out_s, t->out_h, p->B, p->S, t->heads))
		REFUSE(SAM3_EINVAL, "norm_rope: %s has a negative stride, or outputs in one place", name);
	if (t->in == t->out && ((p->B > 1 && t->in_b != t->out_b) || (p->S > 1 && t->in_s != t->out_s) ||
				(t->heads > 1 && t->in_h != t->out_h)))
		REFUSE(SAM3_EINVAL, "norm_rope: %s in place with other strides", name);
	return SAM3_OK;
}

static struct s3k_heads heads_of(const struct sam3_hip_heads *t)
{
	return (struct s3k_heads){t->in, t->out, t->heads, t->in_b, t->in_s, t->in_h,
				  t->out_b, t->out_s, t->out_h, t->weight};
}

enum sam3_error sam3_hip_norm_rope(const struct sam3_hip_norm_rope *p, void *stream)
{
	if (!p)
		REFUSE(SAM3_EINVAL, "norm_rope: NULL");
	if (!is_float_dtype(p->dtype))
		REFUSE(SAM3_EDTYPE, "norm_rope: dtype %d is not F32, F16 or BF16", p->dtype);
	if (p->B < 0 || p->S < 0 || p->D < 2 || p->D > 512 || p->D % 2 || p->rot < 0 || p->rot > p->D ||
	    p->rot % 2)
		REFUSE(SAM3_EINVAL, "norm_rope: B=%d S=%d D=%d rot=%d (D even, 2 to 512; rot even, to D)",
		       p->B, p->S, p->D, p->rot);
	if (p->layout != SAM3_HIP_ROPE_INTERLEAVED && p->layout != SAM3_HIP_ROPE_HALF)
		REFUSE(SAM3_EINVAL, "norm_rope: layout %d", p->layout);
	if (p->norm && !(p->eps >= 0.0f && p->eps <= 3.402823466e38f))
		REFUSE(SAM3_EINVAL, "norm_rope: eps is negative or not finite");
	enum sam3_error err = heads_check(p, &p->q, "q");
	if (err == SAM3_OK)
		err = heads_check(p, &p->k, "k");
	if (err != SAM3_OK)
		return err;
	if (p->q.heads > (1 << 20) || p->k.heads > (1 << 20))
		REFUSE(SAM3_EINVAL, "norm_rope: more than 2^20 heads");
	if (p->B == 0 || p->S == 0 || p->q.heads + p->k.heads == 0)
		return SAM3_OK;
	if (p->rot > 0 && (!p->freq || (uintptr_t)p->freq % 8))
		REFUSE(SAM3_EINVAL, "norm_rope: freq is NULL or not 8-byte aligned");
	if ((uintptr_t)p->pos % 4 || (p->pos && p->pos_b < 0))
		REFUSE(SAM3_EINVAL, "norm_rope: pos must be 4-byte aligned, its stride not negative");
	const struct s3k_norm_rope d = {p->dtype, p->B, p->S, p->D, p->rot,
					p->layout == SAM3_HIP_ROPE_HALF, heads_of(&p->q),
					heads_of(&p->k), p->pos, p->pos_b, p->freq, p->amp,
					p->norm != 0, p->eps};
	return launched(s3k_norm_rope(&d, stream), "norm_rope");
}

enum sam3_error sam3_hip_rope_frequencies(int rot, double theta, int scaling, double factor,
					  double trained, double fast, double slow, double *freq,
					  float *amp)
{
	if (rot < 0 || rot % 2 || !(theta > 0.0 && theta <= 1e300) || !freq || !amp)
		REFUSE(SAM3_EINVAL, "rope_frequencies: rot=%d theta=%g, or a NULL output", rot, theta);
	if (scaling != SAM3_HIP_ROPE_PLAIN && scaling != SAM3_HIP_ROPE_LINEAR &&
	    scaling != SAM3_HIP_ROPE_PARTS)
		REFUSE(SAM3_EINVAL, "rope_frequencies: scaling %d", scaling);
	if (scaling != SAM3_HIP_ROPE_PLAIN && !(factor >= 1.0 && factor <= 1e18))
		REFUSE(SAM3_EINVAL, "rope_frequencies: factor %g is below 1", factor);
	if (scaling == SAM3_HIP_ROPE_PARTS &&
	    !(trained >= 1.0 && trained <= 1e18 && slow >= 0.0 && fast > slow && fast <= 1e18))
		REFUSE(SAM3_EINVAL, "rope_frequencies: trained=%g fast=%g slow=%g", trained, fast, slow);
	for (int i = 0; i < rot / 2; i++) {
		const double f = pow(theta, -2.0 * i / rot);
		double keep = scaling == SAM3_HIP_ROPE_PLAIN ? 1.0 : 0.0;
		if (scaling == SAM3_HIP_ROPE_PARTS) {
			const double turns = trained * f / 6.283185307179586;
			keep = (turns - slow) / (fast - slow);
			keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
		}
		freq[i] = keep == 1.0 ? f : f * keep + f / factor * (1.0 - keep);
	}
	*amp = scaling == SAM3_HIP_ROPE_PARTS ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
	return SAM3_OK;
}

/* ------------------------------------------------------------------ */
/* Cross attention                                                      */
/* ------------------------------------------------------------------ */
/* Checks p and fills d; *empty: nothing to do. */
static enum sam3_error xattn_check(const struct sam3_hip_cross_attention *p, struct s3k_xattn *d,
				   int *empty)
{
	*empty = 0;
	if (!p)
		REFUSE(SAM3_EINVAL, "cross_attention: NULL");
	if (!is_float_dtype(p->dtype))
		REFUSE(SAM3_EDTYPE, "cross_attention: dtype %d is not F32, F16 or BF16", p->dtype);
	if (p->B < 0 || p->H < 0 || p->Hkv < 0 || p->Sq < 0 || p->Sk < 0 || p->D < 1 || p->D > 256)
		REFUSE(SAM3_EINVAL, "cross_attention: B=%d H=%d Hkv=%d Sq=%d Sk=%d D=%d (D 1 to 256)",
		       p->B, p->H, p->Hkv, p->Sq, p->Sk, p->D);
	if (!(p->scale >= 0.0f && p->scale <= 1e30f))
		REFUSE(SAM3_EINVAL, "cross_attention: scale %g", (double)p->scale);
	if (p->B == 0 || p->H == 0 || p->Sq == 0) {
		*empty = 1;
		return SAM3_OK;
	}
	if (p->Hkv == 0 || p->H % p->Hkv)
		REFUSE(SAM3_EINVAL, "cross_attention: %d heads over %d key heads", p->H, p->Hkv);
	if (!p->q || !p->out || (p->Sk > 0 && (!p->k || !p->v)))
		REFUSE(SAM3_EINVAL, "cross_attention: NULL tensor");
	const uintptr_t es = esize(p->dtype);
	if ((uintptr_t)p->q % es || (uintptr_t)p->k % es || (uintptr_t)p->v % es ||
	    (uintptr_t)p->out % es || (uintptr_t)p->q_len % 4 || (uintptr_t)p->k_len % 4)
		REFUSE(SAM3_EINVAL, "cross_attention: tensors must be element-aligned, lengths 4-byte");
	if ((p->q_b | p->q_s | p->q_h | p->k_b | p->k_s | p->k_h | p->v_b | p->v_s | p->v_h) < 0 ||
	    !out_strides_ok(p->o_b, p->o_s, p->o_h, p->B, p->Sq, p->H))
		REFUSE(SAM3_EINVAL, "cross_attention: negative stride, or outputs in one place");
	if ((long long)p->Sq * (p->H / p->Hkv) > 0x3FFFFFFFll || p->Sk > 0x3FFFFFFF ||
	    (long long)p->B * p->H > 0xFFFFFFll)
		REFUSE(SAM3_EINVAL, "cross_attention: 2^30 keys, or rows of one key head, or 2^24 heads");
	const float scale = p->scale > 0.0f ? p->scale : (float)(1.0 / sqrt((double)p->D));
	*d = (struct s3k_xattn){p->dtype, p->B, p->H, p->Hkv, p->Sq, p->Sk, p->D, scale,
				p->q, p->k, p->v, p->out,
				p->q_b, p->q_s, p->q_h, p->k_b, p->k_s, p->k_h,
				p->v_b, p->v_s, p->v_h, p->o_b, p->o_s, p->o_h, p->q_len, p->k_len};
	return SAM3_OK;
}

size_t sam3_hip_cross_attention_work(const struct sam3_hip_cross_attention *p)
{
	struct s3k_xattn d;
	int empty;
	if (xattn_check(p, &d, &empty) != SAM3_OK || empty)
		return 0;
	const int path = s3k_xattn_path(&d);
	return s3k_xattn_bytes(&d, path, s3k_xattn_parts(&d, path));
}

int sam3_hip_cross_attention_path(const struct sam3_hip_cross_attention *p)
{
	struct s3k_xattn d;
	int empty;
	if (xattn_check(p, &d, &empty) != SAM3_OK || empty)
		return 0;
	return s3k_xattn_path(&d);
}

enum sam3_error sam3_hip_cross_attention_on_path(int path, const struct sam3_hip_cross_attention *p,
						 void *work, size_t work_bytes, void *stream)
{
	struct s3k_xattn d;
	int empty;
	enum sam3_error err = xattn_check(p, &d, &empty);
	if (err != SAM3_OK || empty)
		return err;
	if (path == 0)
		path = s3k_xattn_path(&d);
	else if (!s3k_xattn_can(&d, path))
		REFUSE(SAM3_EINVAL, "cross_attention: kernel %d cannot run this problem", path);
	int parts = s3k_xattn_parts(&d, path);
	const size_t need = s3k_xattn_bytes(&d, path, parts);
	void *own = NULL;
	if (work && (work_bytes < need || (uintptr_t)work % 16))
		REFUSE(SAM3_EINVAL, "cross_attention: %zu bytes of work space, %zu needed (16-byte "
		       "aligned)", work_bytes, need);
	if (!work && need) {
		if (captured(stream) || s3h_scratch_alloc(&own, need, stream) != SAM3_OK) {
			(void)hipGetLastError();
			own = NULL;
			parts = 1;
		}
		work = own;
	}
	err = launched(s3k_xattn_run(&d, path, parts, work, stream), "cross_attention");
	const enum sam3_error ferr = s3h_scratch_free(own, stream);
	return err != SAM3_OK ? err : ferr;
}

enum sam3_error sam3_hip_cross_attention(const struct sam3_hip_cross_attention *p, void *work,
					 size_t work_bytes, void *stream)
{
	return sam3_hip_cross_attention_on_path(0, p, work, work_bytes, stream);
}
