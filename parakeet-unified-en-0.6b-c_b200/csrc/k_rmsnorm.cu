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
// bound in fp32: 12000 x 1024 to int8 in 28.0 us = 5.7 TB/s, 0.87 of the copy
// bandwidth, to e4m3 28.7; 4000 x 4096 0.88. 16-bit rows take 0.8 of the time for 0.54
// of the bytes (12000 x 1024 bf16 22.4 us = 0.59): issue slots are 62 % busy with 35
// instructions per entry, and the warps wait for loads (10.5 of them on the long
// scoreboard per issue), of which gamma's and bias's, fp32 through L1 again for every
// row, are twice the bytes of the row's own. Wide 16-bit rows where they are many come
// through shared memory by bulk copies (2049 x 8192 to int8 without a bias 24.6 us = 0.73,
// 6000 x 8192 0.89; 1024-wide rows 24 to 28 us that way). Measured and not kept: persistent
// CTAs that load the next row into registers before they finish this one (34 to 44 us
// fp32, 25 to 33 bf16), rows kept packed in 16 bits between the two looks at them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

#include "pk_common.cuh"
#include "pk_types.cuh"

namespace pk {

constexpr int RING_MAX = 8;   // rows ahead per group
constexpr int LONG_THREADS = 1024;

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

// q = round(t mul): what every thread of a row needs. mul 0: q is 0 (a row of
// zeros, or one that stands for NaN).
template <bool E4M3>
struct Quant {
  static constexpr float Q = E4M3 ? 448.0f : 127.0f;
};
__device__ __forceinline__ bool row_finite(float ss, float amax) { return ss < INFINITY && amax < INFINITY; }
// Below this largest |t|, Q / max|t| would overflow; t is scaled up first.
constexpr float kTiny = 0x1p-100f, kTinyUp = 0x1p100f;

// The row's scale (one thread): a NaN or an infinity anywhere in the row (or
// squares or an x' gamma past fp32) makes it NaN, so that every entry stands for
// NaN. Not kept: such finite rows once more from memory, with scaled squares and
// products; the path, never taken, cost 1 to 4 % of every row's time (2049 x 8192 bf16
// to e4m3 31.5 us and 32.7, 12000 x 300 fp32 11.2 and 11.6), called, inlined or behind
// the ring's loop.
template <bool E4M3>
__device__ __forceinline__ float row_scale(float ss, float amax, float eps, int D) {
  if (!row_finite(ss, amax)) return __int_as_float(0x7fffffff);
  if (amax == 0.0f) return 0.0f;
  const float r = 1.0f / sqrtf(ss / (float)D + eps), top = amax * r;   // top: of the norm, perhaps past fp32
  return top < INFINITY ? top / Quant<E4M3>::Q : amax * (r / Quant<E4M3>::Q);
}
// Q / max|t| (max|t| times up, what t is multiplied by first), 0 for a row whose q
// is 0; lo (e4m3): what its rounding left.
struct RowMul {
  float hi, lo, up;
};
template <bool E4M3>
__device__ __forceinline__ RowMul row_mul(float ss, float amax) {
  RowMul m;
  m.up = amax < kTiny ? kTinyUp : 1.0f;
  m.hi = amax == 0.0f || !row_finite(ss, amax) ? 0.0f : Quant<E4M3>::Q / (amax * m.up);
  m.lo = E4M3 ? fmaf(-m.hi, amax * m.up, Quant<E4M3>::Q) * (m.hi * (1.0f / Quant<E4M3>::Q)) : 0.0f;
  return m;
}

// N entries x gamma mul rounded to nearest even, as their 8-bit patterns, for
// finite ones; |x gamma mul| <= Q (1 + 2^-22), which rounds to Q at most, so
// nothing saturates. int8: t = x gamma, and t mul + 1.5 2^23 in one fused
// multiply-add rounds to an integer whose two's complement is the sum's low byte.
// e4m3: what the two products and mul itself lost is added before the rounding, so
// that entries next to a border between two values fall on the side of the exact
// ones (half as many of them astray as the plain product leaves).
template <bool E4M3, int N>
__device__ __forceinline__ void q8(const float (&x)[N], const float (&g)[N], RowMul m, unsigned char *o) {
  float v[N];
  if constexpr (E4M3) {   // two entries per operation; c: the correction, negative
    const float2 neg = splat2(-1.0f), hi = splat2(m.hi), nhi = splat2(-m.hi), nlo = splat2(-m.lo);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 x2 = make_float2(x[i], N > 1 ? x[i + (N > 1)] : 0.0f), g2 = make_float2(g[i], N > 1 ? g[i + (N > 1)] : 0.0f);
      float2 t = mul2(x2, g2), lo = fma2(x2, g2, mul2(t, neg));
      if (m.up != 1.0f) {
        t = mul2(t, splat2(m.up));
        lo = mul2(lo, splat2(m.up));
      }
      const float2 p = mul2(t, hi);
      const float2 c = fma2(lo, nhi, fma2(t, nlo, fma2(t, nhi, p)));
      const float2 r = fma2(c, neg, p);
      v[i] = r.x;
      if (N > 1) v[i + (N > 1)] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = x[i] * g[i];
    if (m.up != 1.0f) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] *= m.up;
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = fmaf(v[i], m.hi, 12582912.0f);
  }
  if constexpr (E4M3) {
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) {
      const __nv_fp8x2_storage_t p = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE, __NV_E4M3);
      o[i] = (unsigned char)(p & 0xff);
      o[i + 1] = (unsigned char)(p >> 8);
    }
    if (N & 1) o[N - 1] = __nv_cvt_float_to_fp8(v[N - 1], __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = (unsigned char)(__float_as_uint(v[i]) & 0xff);
  }
}

__device__ __forceinline__ void warp_reduce(float &ss, float &amax) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(PK_FULL_MASK, ss, o);
  // (as bits: none is negative, and NaN is above infinity)
  amax = __uint_as_float(__reduce_max_sync(PK_FULL_MASK, __float_as_uint(amax)));
}

// (ss, amax) over the TPR threads of a row. TPR 32: the row's warp, by
// shuffles; else the whole CTA. red: 64 floats, used once.
template <int TPR>
__device__ __forceinline__ void row_reduce(float &ss, float &amax, float *red) {
  warp_reduce(ss, amax);
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

// ── rows held in registers ────────────────────────────────────────────────────
// TPR threads per row (a warp, eight rows to a CTA; or a whole CTA), each
// holding EPT entries in chunks of VEC (16 bytes of the stream's type, or one
// entry where rows are not 16-byte aligned), chunk c of the row at thread c mod
// TPR, so every access of a warp is contiguous. All of a thread's loads of x
// and y are issued before the first is used.

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T e[VEC];
};

template <typename T, int VEC, bool STREAM>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
  Pack<T, VEC> r;
  if constexpr (VEC == 1) {
    r.e[0] = *p;
  } else {
    const float4 v = STREAM ? __ldcs(reinterpret_cast<const float4 *>(p)) : *reinterpret_cast<const float4 *>(p);
    r = *reinterpret_cast<const Pack<T, VEC> *>(&v);
  }
  return r;
}

// VEC fp32 parameters (gamma, bias)
template <int VEC>
__device__ __forceinline__ void load_param(float (&o)[VEC], const float *p) {
  if constexpr (VEC == 1) {
    o[0] = __ldg(p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(p + i));
      o[i] = v.x;
      o[i + 1] = v.y;
      o[i + 2] = v.z;
      o[i + 3] = v.w;
    }
  }
}

// ── any row length: one CTA per row, two passes (the second from x_out) ───────
template <typename T, bool E4M3, int VEC>
__global__ void __launch_bounds__(LONG_THREADS) rms_q8_long_kernel(RmsArgs a) {
  __shared__ float red[64];
  const long long row = blockIdx.x;
  const int nc = a.D / VEC;
  const T *x = static_cast<const T *>(a.x) + row * a.D;
  const T *y = a.y ? static_cast<const T *>(a.y) + row * a.D : nullptr;
  T *xo = a.x_out ? static_cast<T *>(a.x_out) + row * a.D : nullptr;
  float ss = 0.0f, amax = 0.0f;
#pragma unroll 2
  for (int c = threadIdx.x; c < nc; c += LONG_THREADS) {
    Pack<T, VEC> px = load_pack<T, VEC, false>(x + (long long)c * VEC);
    float p[VEC];
    if (y) {
      const Pack<T, VEC> py = load_pack<T, VEC, true>(y + (long long)c * VEC);
      if (a.bias) load_param<VEC>(p, a.bias + (long long)c * VEC);
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        float add = to_f32(py.e[i]);
        if (a.bias) add = add + p[i];
        px.e[i] = from_f32<T>(fmaf(add, a.alpha, to_f32(px.e[i])));
      }
    }
    if (xo) *reinterpret_cast<Pack<T, VEC> *>(xo + (long long)c * VEC) = px;
    load_param<VEC>(p, a.gamma + (long long)c * VEC);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const float v = to_f32(px.e[i]);
      ss = fmaf(v, v, ss);
      amax = max_nan(amax, fabsf(v * p[i]));
    }
  }
  row_reduce<LONG_THREADS>(ss, amax, red);
  const RowMul mul = row_mul<E4M3>(ss, amax);
  unsigned char *q = static_cast<unsigned char *>(a.q) + row * a.ldq;
  const T *kept = xo ? xo : x;   // each thread re-reads the entries that it wrote itself
#pragma unroll 2
  for (int c = threadIdx.x; c < nc; c += LONG_THREADS) {
    const Pack<T, VEC> px = load_pack<T, VEC, false>(kept + (long long)c * VEC);
    float v[VEC], g[VEC];
    load_param<VEC>(g, a.gamma + (long long)c * VEC);
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = to_f32(px.e[i]);
    Pack<unsigned char, VEC> o = {};
    if (mul.hi != 0.0f) q8<E4M3, VEC>(v, g, mul, o.e);
    *reinterpret_cast<Pack<unsigned char, VEC> *>(q + (long long)c * VEC) = o;
  }
  if (threadIdx.x == 0) a.scales[row] = row_scale<E4M3>(ss, amax, a.eps, a.D);
}

// ── rows held in registers: the kernel ────────────────────────────────────────
template <typename T, bool E4M3, int TPR, int VEC, int EPT>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) rms_q8_kernel(RmsArgs a) {
  constexpr int NV = EPT / VEC, ROWS = TPR == 32 ? 8 : 1;
  __shared__ float red[64];
  const long long row = (long long)blockIdx.x * ROWS + (TPR == 32 ? threadIdx.x / TPR : 0);
  if (TPR == 32 && row >= a.n_rows) return;
  const int t = threadIdx.x % TPR;
  const int nc = a.D / VEC;   // chunks in a row (VEC > 1: D % VEC == 0)
  const T *x = static_cast<const T *>(a.x) + row * a.D;
  float v[EPT];
  {
    Pack<T, VEC> px[NV];
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (t + j * TPR < nc) px[j] = load_pack<T, VEC, false>(x + (t + j * TPR) * VEC);
    if (a.y) {
      const T *y = static_cast<const T *>(a.y) + row * a.D;
      Pack<T, VEC> py[NV];
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (t + j * TPR < nc) py[j] = load_pack<T, VEC, true>(y + (t + j * TPR) * VEC);
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (t + j * TPR < nc) {
          float b[VEC];
          if (a.bias) load_param<VEC>(b, a.bias + (t + j * TPR) * VEC);
#pragma unroll
          for (int i = 0; i < VEC; i++) {
            float add = to_f32(py[j].e[i]);
            if (a.bias) add = add + b[i];
            px[j].e[i] = from_f32<T>(fmaf(add, a.alpha, to_f32(px[j].e[i])));
          }
        }
    }
    if (a.x_out) {
      T *xo = static_cast<T *>(a.x_out) + row * a.D;
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (t + j * TPR < nc) *reinterpret_cast<Pack<T, VEC> *>(xo + (t + j * TPR) * VEC) = px[j];
    }
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j * VEC + i] = t + j * TPR < nc ? to_f32(px[j].e[i]) : 0.0f;
  }
  float ss = 0.0f, amax = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; j++)
    if (t + j * TPR < nc) {
      float g[VEC];
      load_param<VEC>(g, a.gamma + (t + j * TPR) * VEC);
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const float x1 = v[j * VEC + i], n = x1 * g[i];
        ss = fmaf(x1, x1, ss);
        amax = max_nan(amax, fabsf(n));
        if (!E4M3) v[j * VEC + i] = n;
      }
    }
  row_reduce<TPR>(ss, amax, red);
  const RowMul mul = row_mul<E4M3>(ss, amax);
  unsigned char *q = static_cast<unsigned char *>(a.q) + row * a.ldq;
#pragma unroll
  for (int j = 0; j < NV; j++)
    if (t + j * TPR < nc) {
      Pack<unsigned char, VEC> o = {};
      float x1[VEC], g[VEC];   // e4m3: gamma once more; int8: x gamma is at hand
      if (E4M3) load_param<VEC>(g, a.gamma + (t + j * TPR) * VEC);
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        x1[i] = v[j * VEC + i];
        if (!E4M3) g[i] = 1.0f;
      }
      if (mul.hi != 0.0f) q8<E4M3, VEC>(x1, g, mul, o.e);
      *reinterpret_cast<Pack<unsigned char, VEC> *>(q + (t + j * TPR) * VEC) = o;
    }
  if (t == 0) a.scales[row] = row_scale<E4M3>(ss, amax, a.eps, a.D);
}

// ── many rows in 16 bits ──────────────────────────────────────────────────────
// One CTA per SM, of G groups of TPR threads. A group takes rows first, first +
// step, ... through a ring of its own: bulk copies bring x and y of the next rows
// into shared memory while this one is worked on, so bytes under way need no
// registers and no thread waits for the whole of a row's latency; gamma and
// bias stay in registers (bias read again from L1 for every row: 2049 x 8192 to int8
// 31.7 us for 27.6). A slot is free once the row's reduction has passed its
// barrier (every thread holds its entries by then).
template <typename T, bool E4M3, int TPR, int NV, int G>
__global__ void __launch_bounds__(TPR *G, 1) rms_q8_ring_kernel(RmsArgs a, int stages) {
  constexpr int VEC = 16 / (int)sizeof(T), W = TPR / 32;
  extern __shared__ __align__(128) unsigned char ring_smem[];
  __shared__ unsigned long long full[G][RING_MAX];
  __shared__ float red[2][G][2][W];   // the row's partial sums and maxima; alternating
  __shared__ int stop[2][G];          // a wait for this row ran out; alternating as well
  const int g = threadIdx.x / TPR, t = threadIdx.x % TPR, lane = t & 31, warp = t >> 5;
  const int nc = a.D / VEC;
  const unsigned row_bytes = (unsigned)a.D * sizeof(T), slot = a.y ? 2 * row_bytes : row_bytes;
  unsigned char *ring = ring_smem + (size_t)g * stages * slot;
  const long long first = (long long)blockIdx.x * G + g, step = (long long)gridDim.x * G;
  auto load = [&](long long row, int i) {
    mbar_arrive_tx(&full[g][i], slot);
    bulk_g2s(ring + i * slot, static_cast<const T *>(a.x) + row * a.D, row_bytes, &full[g][i]);
    if (a.y) bulk_g2s(ring + i * slot + row_bytes, static_cast<const T *>(a.y) + row * a.D, row_bytes, &full[g][i]);
  };
  if (t == 0) {
    for (int i = 0; i < stages; i++) mbar_init(&full[g][i], 1);
    mbar_init_fence();
    stop[0][g] = stop[1][g] = 0;
    for (int i = 0; i < stages; i++)
      if (first + i * step < a.n_rows) load(first + i * step, i);
  }
  float gm[NV][VEC], bs[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; j++)
    if (t + j * TPR < nc) {
      load_param<VEC>(gm[j], a.gamma + (t + j * TPR) * VEC);
      if (a.bias) load_param<VEC>(bs[j], a.bias + (t + j * TPR) * VEC);
    }
  __syncthreads();
  int at = 0, phase = 0, flip = 0;
  for (long long row = first; row < a.n_rows; row += step) {
    const bool here = mbar_wait(&full[g][at], phase);
    if (!here) {
      if (t == 0) atomicAdd(&g_wait_timeouts, 1u);
      stop[flip][g] = 1;
    }
    const Pack<T, VEC> *sx = reinterpret_cast<const Pack<T, VEC> *>(ring + at * slot);
    const Pack<T, VEC> *sy = reinterpret_cast<const Pack<T, VEC> *>(ring + at * slot + row_bytes);
    Pack<T, VEC> px[NV];   // x'
    float ss = 0.0f, amax = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (t + j * TPR < nc) {
        px[j] = sx[t + j * TPR];
        if (a.y) {
          const Pack<T, VEC> py = sy[t + j * TPR];
#pragma unroll
          for (int i = 0; i < VEC; i++) {
            float add = to_f32(py.e[i]);
            if (a.bias) add = add + bs[j][i];
            px[j].e[i] = from_f32<T>(fmaf(add, a.alpha, to_f32(px[j].e[i])));
          }
        }
        if (a.x_out && here)
          reinterpret_cast<Pack<T, VEC> *>(static_cast<T *>(a.x_out) + row * a.D)[t + j * TPR] = px[j];
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const float x1 = to_f32(px[j].e[i]);
          ss = fmaf(x1, x1, ss);
          amax = max_nan(amax, fabsf(x1 * gm[j][i]));
        }
      }
    warp_reduce(ss, amax);
    if (lane == 0) {
      red[flip][g][0][warp] = ss;
      red[flip][g][1][warp] = amax;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + g), "n"(TPR) : "memory");
    // the whole group reads this row's word and leaves together: a thread that is ahead,
    // and whose wait for the next row runs out, writes the other one
    if (*(volatile int *)&stop[flip][g]) break;
    if (t == 0 && row + stages * step < a.n_rows) load(row + stages * step, at);
    ss = red[flip][g][0][0];
    amax = red[flip][g][1][0];
#pragma unroll
    for (int w = 1; w < W; w++) {
      ss += red[flip][g][0][w];
      amax = max_nan(amax, red[flip][g][1][w]);
    }
    const RowMul mul = row_mul<E4M3>(ss, amax);
    unsigned char *q = static_cast<unsigned char *>(a.q) + row * a.ldq;
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (t + j * TPR < nc) {
        Pack<unsigned char, VEC> o = {};
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = to_f32(px[j].e[i]);
        if (mul.hi != 0.0f) q8<E4M3, VEC>(v, gm[j], mul, o.e);
        *reinterpret_cast<Pack<unsigned char, VEC> *>(q + (t + j * TPR) * VEC) = o;
      }
    if (t == 0) a.scales[row] = row_scale<E4M3>(ss, amax, a.eps, a.D);
    flip ^= 1;
    if (++at == stages) {
      at = 0;
      phase ^= 1;
    }
  }
  // a wait ran out: the copies still in flight land (bounded) before the CTA's
  // shared memory is released
  if (t == 0 && (*(volatile int *)&stop[0][g] | *(volatile int *)&stop[1][g]))
    for (int i = 0; i < stages; i++) {
      mbar_wait(&full[g][i], 0);
      mbar_wait(&full[g][i], 1);
    }
}

template <typename T, bool E4M3, int VEC, int TPR, int EPT>
void rms_launch_as(const RmsArgs &a, cudaStream_t s) {
  const long long grid = TPR == 32 ? (a.n_rows + 7) / 8 : a.n_rows;
  rms_q8_kernel<T, E4M3, TPR, VEC, EPT><<<(unsigned)grid, TPR == 32 ? 256 : TPR, 0, s>>>(a);
}

// Eight entries per thread up to 2048-wide rows: 12000 x 1024 fp32 took 27.8 us
// with 128 threads per row, 28.0 with 128 threads of 16 (D padded to 2048),
// 28.7 with 64 of 16 and 30.7 with a warp of 32 (more registers, fewer rows in
// flight per SM). Wider rows take 16 or 32 per thread: 4000 x 4096 fp32 35.8 us
// with 256 of 16, 36.9 with 512 of 8; 2049 x 8192 fp32 37.9 with 512 of 16, 39.9
// with 256 of 32, but bf16, whose chunks take half the registers, 35.8 and 32.8.
// Many wide 16-bit rows go through the ring: 2049 x 8192 bf16 to int8 31.7 us in
// registers, 27.6 through the ring, to e4m3 36.8 and 31.6; 6000 x 8192 76 and 65; 4000 x
// 5120 42 and 37; 900 x 8192 16.8 and 17.2 (too few rows per group). Up to 4096 wide the
// two are within 10 % of each other, and the registers win below 3000 rows.
constexpr int RING_BYTES = 200 * 1024;
template <typename T, bool E4M3, int TPR, int NV, int G>
void rms_launch_ring(const RmsArgs &a, cudaStream_t s) {
  static int flags[64];
  smem_optin(rms_q8_ring_kernel<T, E4M3, TPR, NV, G>, RING_BYTES, flags);
  const int slot = a.D * (int)sizeof(T) * (a.y ? 2 : 1);
  const int fit = RING_BYTES / (G * slot), stages = fit < RING_MAX ? fit : RING_MAX;
  const long long ctas = (a.n_rows + G - 1) / G;
  const int sms = pkcu_sm_count();
  rms_q8_ring_kernel<T, E4M3, TPR, NV, G><<<(unsigned)(ctas < sms ? ctas : sms), TPR * G, (size_t)stages * G * slot, s>>>(a, stages);
}

template <typename T, bool E4M3, int VEC>
void rms_launch_rows(const RmsArgs &a, cudaStream_t s) {
  if (a.D <= 256) rms_launch_as<T, E4M3, VEC, 32, 8>(a, s);
  else if (a.D <= 512) rms_launch_as<T, E4M3, VEC, 64, 8>(a, s);
  else if (a.D <= 1024) rms_launch_as<T, E4M3, VEC, 128, 8>(a, s);
  else if (a.D <= 2048) rms_launch_as<T, E4M3, VEC, 256, 8>(a, s);
  else if (a.D <= 4096) rms_launch_as<T, E4M3, VEC, 256, 16>(a, s);
  else if constexpr (VEC == 8) {
    if (a.n_rows >= 8LL * pkcu_sm_count()) rms_launch_ring<T, E4M3, 256, 4, 2>(a, s);
    else rms_launch_as<T, E4M3, VEC, 256, 32>(a, s);
  } else rms_launch_as<T, E4M3, VEC, 512, 16>(a, s);
}

template <typename T, bool E4M3>
int rms_launch_q(const RmsArgs &a, cudaStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.x_out | (uintptr_t)a.bias | (uintptr_t)a.gamma;
  const bool vec = a.D % VEC == 0 && (at & 15) == 0 && ((uintptr_t)a.q | (uintptr_t)a.ldq) % VEC == 0;
  if (a.D > 8192 && vec) rms_q8_long_kernel<T, E4M3, VEC><<<(unsigned)a.n_rows, LONG_THREADS, 0, s>>>(a);
  else if (a.D > 8192) rms_q8_long_kernel<T, E4M3, 1><<<(unsigned)a.n_rows, LONG_THREADS, 0, s>>>(a);
  else if (vec) rms_launch_rows<T, E4M3, VEC>(a, s);
  else rms_launch_rows<T, E4M3, 1>(a, s);
  return pkcu_launch_status("pkcu_residual_rms_norm_q8");
}

template <typename T>
int rms_launch(const RmsArgs &a, int e4m3, cudaStream_t s) {
  return e4m3 ? rms_launch_q<T, true>(a, s) : rms_launch_q<T, false>(a, s);
}

}  // namespace pk

using namespace pk;

PK_WAIT_WORD(pk_rms_wait_word)

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
