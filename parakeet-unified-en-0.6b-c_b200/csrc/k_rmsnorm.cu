// k_rmsnorm.cu -- residual + root-mean-square norm with an 8-bit output, the
// producer of the 8-bit activations that pkcu_wmatmul_q8 multiplies. No
// counterpart in the reference, whose norms are LayerNorms; it stands beside
// pkcu_residual_layer_norm.
//
//   x'     = x + alpha (y + bias), rounded to the stream's type and stored
//   t      = x' gamma,  r = 1 / sqrt(mean(x'^2) + eps)      (fp32)
//   scale  = max|t| r / Q           Q = 127 (int8) or 448 (e4m3)
//   q      = round(t Q / max|t|)    (r cancels: t r / scale)
//
// The norm is of the stored x', so the fused call equals the residual add
// followed by a call without y. Both statistics come from one pass over the
// row, so a row is read once, kept in registers as fp32, and written once: 13
// bytes of HBM traffic per element in fp32, 7 in 16 bits. That traffic is the
// bound.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

#include "pk_common.cuh"
#include "pk_types.cuh"

namespace pk {

struct RmsArgs {
  const void *x, *y;
  const float *bias, *gamma;
  void *x_out, *q;
  float *scales;
  float alpha, eps;
  long long n_rows, ldq;
  int D;
};

// ── what a row's statistics become ───────────────────────────────────────────

struct RowQ {
  float mul;    // t -> t mul pre is the value that is rounded
  float pre;    // 2^100 for rows whose largest |t| is so small that Q / max|t| would overflow
  float scale;
};
template <bool E4M3>
__device__ __forceinline__ RowQ row_q(float ss, float amax, float eps, int D) {
  constexpr float Q = E4M3 ? 448.0f : 127.0f;
  RowQ o;
  const float r = 1.0f / sqrtf(ss / (float)D + eps);
  o.pre = amax < 0x1p-100f ? 0x1p100f : 1.0f;
  if (amax == 0.0f) {          // a row of zeros: q = 0, scale = 0
    o.mul = 0.0f;
    o.scale = 0.0f;
  } else {
    o.mul = Q / (amax * o.pre);
    o.scale = amax * r / Q;
  }
  // a NaN or an infinity anywhere in the row (or squares past fp32): every
  // entry stands for NaN, carried by the scale
  if (!(ss < INFINITY) || !(amax < INFINITY)) {
    o.mul = 0.0f;
    o.scale = __int_as_float(0x7fffffff);
  }
  return o;
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// t mul rounded to nearest even, as its 8-bit pattern; |t mul| <= Q (1 + 2^-22),
// which rounds to Q at most, so nothing saturates. With mul = 0 (a row of
// zeros, or one that stands for NaN) q is 0 whatever t is.
template <bool E4M3>
__device__ __forceinline__ unsigned char q8(float t, const RowQ &rq) {
  if (rq.mul == 0.0f) return 0;
  const float v = (t * rq.pre) * rq.mul;
  if (E4M3) return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  return (unsigned char)(signed char)__float2int_rn(v);
}

// (ss, amax) over the TPR threads of a row. TPR 32: the row's warp, by
// shuffles; else the whole CTA. red: 2 * 32 floats, used once per row.
template <int TPR>
__device__ __forceinline__ void row_reduce(float &ss, float &amax, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(PK_FULL_MASK, ss, o);
    amax = max_nan(amax, __shfl_xor_sync(PK_FULL_MASK, amax, o));
  }
  if (TPR > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int W = TPR / 32;
    if (lane == 0) {
      red[warp] = ss;
      red[32 + warp] = amax;
    }
    __syncthreads();
    // every warp folds the partials in the same order
    ss = red[0];
    amax = red[32];
#pragma unroll
    for (int w = 1; w < W; w++) {
      ss += red[w];
      amax = max_nan(amax, red[32 + w]);
    }
  }
}

// ── any row length: one CTA per row, two passes (the second from x_out) ───────

template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) rms_q8_long_kernel(RmsArgs a) {
  __shared__ float red[64];
  const long long row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.D;
  const T *y = a.y ? static_cast<const T *>(a.y) + row * a.D : nullptr;
  T *xo = a.x_out ? static_cast<T *>(a.x_out) + row * a.D : nullptr;
  float ss = 0.0f, amax = 0.0f;
  for (int i = threadIdx.x; i < a.D; i += 256) {
    float v = to_f32(x[i]);
    if (y) {
      float t = to_f32(y[i]);
      if (a.bias) t = t + __ldg(a.bias + i);
      v = to_f32(from_f32<T>(fmaf(t, a.alpha, v)));
    }
    if (xo) xo[i] = from_f32<T>(v);
    ss = fmaf(v, v, ss);
    amax = max_nan(amax, fabsf(v * __ldg(a.gamma + i)));
  }
  row_reduce<256>(ss, amax, red);
  const RowQ rq = row_q<E4M3>(ss, amax, a.eps, a.D);
  unsigned char *q = static_cast<unsigned char *>(a.q) + row * a.ldq;
  const T *v = xo ? xo : x;   // each thread re-reads the entries that it wrote itself
  for (int i = threadIdx.x; i < a.D; i += 256) q[i] = q8<E4M3>(to_f32(v[i]) * __ldg(a.gamma + i), rq);
  if (threadIdx.x == 0) a.scales[row] = rq.scale;
}

template <typename T>
int rms_launch(const RmsArgs &a, int e4m3, cudaStream_t s) {
  if (e4m3) rms_q8_long_kernel<T, true><<<(unsigned)a.n_rows, 256, 0, s>>>(a);
  else rms_q8_long_kernel<T, false><<<(unsigned)a.n_rows, 256, 0, s>>>(a);
  return pkcu_launch_status("pkcu_residual_rms_norm_q8");
}

}  // namespace pk

using namespace pk;

extern "C" int pkcu_residual_rms_norm_q8(const void *x, const void *y, const float *bias, float alpha,
                                         const float *gamma, float eps, int dtype, void *x_out, void *q,
                                         int qtype, long long ldq, float *scales, int n_rows, int D,
                                         pkcu_stream_t stream) {
  const char *what = "pkcu_residual_rms_norm_q8";
  if (n_rows < 0 || D <= 0 || D > (1 << 24)) return pkcu_fail(PKCU_ERR_ARG, "%s: %d rows of %d", what, n_rows, D);
  if (dtype_size(dtype) < 2) return pkcu_fail(PKCU_ERR_ARG, "%s: rows of type %d (F32, BF16 or F16)", what, dtype);
  if (qtype != PKCU_DTYPE_I8 && qtype != PKCU_DTYPE_E4M3)
    return pkcu_fail(PKCU_ERR_ARG, "%s: output of type %d (I8 or E4M3)", what, qtype);
  if (ldq < D) return pkcu_fail(PKCU_ERR_ARG, "%s: ldq %lld is less than D = %d", what, ldq, D);
  if (!(eps > 0.0f) || !(eps < INFINITY)) return pkcu_fail(PKCU_ERR_ARG, "%s: eps %g must be positive", what, eps);
  if (n_rows == 0) return PKCU_OK;
  if (!x || !gamma || !q || !scales || (y && !x_out))
    return pkcu_fail(PKCU_ERR_ARG, "%s: NULL argument", what);
  if (!y && bias) return pkcu_fail(PKCU_ERR_ARG, "%s: a bias without y", what);
  const int size = dtype_size(dtype);
  if (misaligned(x, size) || misaligned(y, size) || misaligned(x_out, size) || misaligned(gamma, 4) ||
      misaligned(bias, 4) || misaligned(scales, 4))
    return pkcu_fail(PKCU_ERR_ARG, "%s: a pointer is not aligned to its type", what);
  const RmsArgs a = {x, y, bias, gamma, x_out, q, scales, alpha, eps, n_rows, ldq, D};
  cudaStream_t s = (cudaStream_t)stream;
  const int e4m3 = qtype == PKCU_DTYPE_E4M3;
  if (dtype == PKCU_DTYPE_F32) return rms_launch<float>(a, e4m3, s);
  if (dtype == PKCU_DTYPE_BF16) return rms_launch<__nv_bfloat16>(a, e4m3, s);
  return rms_launch<__half>(a, e4m3, s);
}
