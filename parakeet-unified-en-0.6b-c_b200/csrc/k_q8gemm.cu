// k_q8gemm.cu -- products of 8-bit activations and 8-bit weights on the tcgen05
// tensor cores, with the bias, the activation and the residual in the epilogue:
//
//   C[m, n] = R[m, n] + r act(s_a[m] s_w[n] sum_k A[m, k] W[k, n] + bias[n])
//
// for int8 (kind::i8, exact 32-bit integer sums) and e4m3 (kind::f8f6f4, fp32
// sums). The library's other products (k_tcgemm.cu) take fp32 activations as
// three bf16 parts: three MMAs at half this rate per product.
//
// Two kernels, chosen by a time model (plan() below).
//
// Few tokens (q8_gemm_kernel) computes C transposed: 128 rows of the K-major
// weight (128 outputs n) are the MMA's M, 16 to 128 activation rows (tokens m) its
// N. A TMEM lane then holds one n and its columns run over m, so a warp's loads
// and stores of one token are 32 consecutive n whatever the pitch or alignment of
// C (rows of 1025 logits included); bias and weight scale are one register per
// thread; one token wastes nothing but columns of a 16-wide tile; and where the
// tiles are few a cluster splits K. Bound by its fixed costs and the weight's
// bytes: 1 x 1024 x 4096 5.7 us, 32 x 640 x 1025 4.7 us, 1 x 8192 x 8192 19 us =
// 3.6 TB/s (set-up, 12 stages in flight per SM, epilogue: the products and a
// kernel's launch alone are 3 us of the first two).
//
// Many tokens (q8_pair_kernel): 256 x 256 tiles of CTA pairs. 12000 x 1024 x 4096
// int8 to bf16 50 us, with Swish 63 to 66, with GELU 71; 12000 x 4096 x 1024 with an
// fp32 residual 55 us; 8192^3 375 to 395 us = 2.8 to 2.9 Pop/s, 0.85 to 0.90 of twice the
// measured bf16 GEMM rate.
//
// Operands. Rows of 128 bytes of K per stage, 128-byte swizzled, by TMA (no
// multicast); K needs no alignment: the tensor maps' extent is K itself, so
// what lies past it reads as zeros.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "pk_common.cuh"
#include "pk_tcgen05.cuh"
#include "pk_types.cuh"

namespace pk {
namespace q8 {

constexpr int BP = 128;    // outputs n per tile: the MMA's M
constexpr int BK = 128;    // bytes (entries) of K per stage
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr int W_TILE = BP * BK;

template <int BQ>
struct Cfg {
  static constexpr int A_TILE = BQ * BK;
  static constexpr int STAGE = W_TILE + A_TILE;
  static constexpr int STAGES = (216 * 1024) / STAGE < 12 ? (216 * 1024) / STAGE : 12;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 512;
  static constexpr int TMEM_COLS = 2 * BQ < 32 ? 32 : 2 * BQ;   // two accumulators
  static constexpr int CW = BQ / 2;                             // columns per epilogue warp
  static constexpr int CH = CW < 32 ? CW : 32;                  // columns per chunk
};

struct Args {
  const float *a_scales, *w_scales, *bias;
  const void *R;
  void *C;
  long long ldc, ldr;
  float rscale;
  int act, dtype;
  int M, N, nkb;
  int r_vec, c_vec;   // rows of R / C 16-byte aligned
};

// ── PTX wrappers ──────────────────────────────────────────────────────────────

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<unsigned long long>(map)) : "memory");
}

// Shared-memory matrix descriptor: K-major rows of 128 bytes, 128-byte swizzle,
// 8-row groups 1024 bytes apart.
__device__ __forceinline__ unsigned long long sdesc_k128(unsigned saddr) {
  unsigned long long d = 0;
  d |= (unsigned long long)((saddr & 0x3FFFFu) >> 4);
  d |= (unsigned long long)1 << 16;
  d |= (unsigned long long)(1024u >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;   // 128-byte swizzle
  return d;
}

// Instruction descriptors, both operands K-major, M x N. kind::i8: signed 32-bit
// D, signed 8-bit A and B; kind::f8f6f4: fp32 D, e4m3 A and B.
__host__ __device__ constexpr unsigned idesc(bool e4m3, int M, int N) {
  return (e4m3 ? 1u << 4 : (2u << 4) | (1u << 7) | (1u << 10)) | ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24);
}

template <bool E4M3>
__device__ __forceinline__ void umma(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned desc,
                                     unsigned accumulate) {
  if constexpr (E4M3)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(desc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(desc), "r"(accumulate)
        : "memory");
}
// One lane polls for its warp (32 would take issue slots and shared-memory cycles
// from the warps at work); the outcome is warp-uniform, as tcgen05.ld needs it.
__device__ __forceinline__ bool mbar_wait_warp(unsigned long long *bar, unsigned parity) {
  int ok = 0;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity);
  return __shfl_sync(PK_FULL_MASK, ok, 0) != 0;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A 32-bit word at the same shared-memory address in CTA `rank` of the cluster.
__device__ __forceinline__ unsigned ld_peer(unsigned saddr, unsigned rank) {
  unsigned a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// ── epilogue ──────────────────────────────────────────────────────────────────

// v / (1 + exp(-v)) on a pair: exp(-v) = 2^-h (1 + l ln 2) with h the rounded
// product v log2 e and -l the rest of the exact one, 2^-h and the reciprocal by
// the hardware's approximations (2 and 1 units in the last place). The power is
// of v held to +-86, so that nothing in it overflows: above, 1 + exp(-v) is 1 and
// the result v, infinity included; below, v counts as -86 in the product too, and
// the result is within 5e-36 of 0. A NaN stays one.
__device__ __forceinline__ float clamp_sym_nan(float v, float most) {   // min(|v|, most) with v's sign
  float r;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
  return r;
}
__device__ __forceinline__ float2 swish_ex2(float2 v) {
  const float2 t = make_float2(clamp_sym_nan(v.x, 86.0f), clamp_sym_nan(v.y, 86.0f));
  v = make_float2(max_nan(v.x, -86.0f), max_nan(v.y, -86.0f));
  const float2 h = mul2(t, splat2(GATE_L2E_HI));
  float2 l = fma2(t, splat2(-GATE_L2E_HI), h);
  l = mul2(fma2(t, splat2(-GATE_L2E_LO), l), splat2(0.693147180559945f));
  float2 e = make_float2(ex2_approx(-h.x), ex2_approx(-h.y));
  e = fma2(e, l, e);
  const float2 d = add2(splat2(1.0f), e);
  return mul2(v, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}

// v (1 + erf(v / sqrt 2)) / 2 on a pair, as max(v, 0) - g with g = |v| erfc(|v| / sqrt
// 2) / 2: the form with erf leaves nothing of the values below v = -5 (1 + erf
// cancels). g = a e^(-a^2 / 2) P(t), a = |v|, t = 1 / (1 + 0.3 a), where P is the
// polynomial of degree 8 whose largest relative distance from erfcx(a / sqrt 2) / 2
// over 0 <= a <= 13.5 is least (0.96 x 2^-24; by reweighted least squares). Within (2
// v^2 + 20) 2^-24 of the value: a^2 / 2 is off by three roundings, the power by 4 x
// 2^-24, t by 3, of which P shows 2.7 times as much at most, P's own steps 4, and the
// products. a counts as 20 at most, where the power is 0: v stays, infinity
// included, and -infinity gives 0. 12000 x 1024 x 4096 bf16 92 us with erff, 132 with
// erfcf, 71 this way.
__device__ __forceinline__ float2 gelu2(float2 v) {
  const float2 a = make_float2(min_nan(fabsf(v.x), 20.0f), min_nan(fabsf(v.y), 20.0f));
  const float2 d = fma2(a, splat2(0.3f), splat2(1.0f));
  const float2 t = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  const float2 s = mul2(mul2(a, a), splat2(-0.72134752044448170f));   // -log2(e) / 2
  float2 p = splat2(0.038334265f);
  p = fma2(p, t, splat2(-0.16895193f));
  p = fma2(p, t, splat2(0.22821721f));
  p = fma2(p, t, splat2(-0.075999506f));
  p = fma2(p, t, splat2(0.142185f));
  p = fma2(p, t, splat2(0.094833f));
  p = fma2(p, t, splat2(0.12188206f));
  p = fma2(p, t, splat2(0.11949307f));
  p = fma2(p, t, splat2(6.8528907e-06f));
  const float2 g = mul2(mul2(a, p), make_float2(ex2_approx(s.x), ex2_approx(s.y)));
  return sub2(make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f)), g);
}

template <int NC>
__device__ __forceinline__ void activate(int act, float (&v)[NC]) {
  switch (act) {
    case PKCU_ACT_RELU:
#pragma unroll
      for (int j = 0; j < NC; j++) v[j] = v[j] < 0.0f ? 0.0f : v[j];
      break;
    case PKCU_ACT_TANH:
#pragma unroll
      for (int j = 0; j < NC; j++) v[j] = tanhf(v[j]);
      break;
    case PKCU_ACT_SWISH:
#pragma unroll
      for (int j = 0; j < NC; j += 2) {
        const float2 s = swish_ex2(make_float2(v[j], v[j + 1]));
        v[j] = s.x;
        v[j + 1] = s.y;
      }
      break;
    case PKCU_ACT_GELU:
#pragma unroll
      for (int j = 0; j < NC; j += 2) {
        const float2 s = gelu2(make_float2(v[j], v[j + 1]));
        v[j] = s.x;
        v[j + 1] = s.y;
      }
      break;
    default: break;
  }
}

template <bool E4M3>
__device__ __forceinline__ float sum_as_float(unsigned acc) {
  return E4M3 ? __uint_as_float(acc) : __int2float_rn((int)acc);
}

// Tokens m .. m + NC - 1 of output n, from their sums; sa: this lane's a_scales
// entry (lane j holds token m + j's). Runs on whole warps; a lane past N only
// lends its scale.
template <bool E4M3, int NC, typename T>
__device__ __forceinline__ void finish(const Args &a, int m, int n, float sw, float bias, float sa,
                                       const unsigned (&acc)[NC]) {
  float v[NC];
#pragma unroll
  for (int j = 0; j < NC; j++)
    v[j] = fmaf(sum_as_float<E4M3>(acc[j]) * sw, __shfl_sync(PK_FULL_MASK, sa, j), bias);
  activate<NC>(a.act, v);
  if (n >= a.N) return;
  const int nm = a.M - m < NC ? a.M - m : NC;
  if (a.R) {
    const T *r = static_cast<const T *>(a.R) + (long long)m * a.ldr + n;
    T x[NC];
#pragma unroll
    for (int j = 0; j < NC; j++, r += a.ldr)
      if (j < nm) x[j] = *r;
#pragma unroll
    for (int j = 0; j < NC; j++)
      if (j < nm) v[j] = fmaf(v[j], a.rscale, to_f32(x[j]));
  } else {
#pragma unroll
    for (int j = 0; j < NC; j++) v[j] *= a.rscale;
  }
  T *c = static_cast<T *>(a.C) + (long long)m * a.ldc + n;
  if (nm == NC) {
#pragma unroll
    for (int j = 0; j < NC; j++, c += a.ldc) *c = from_f32<T>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < NC; j++, c += a.ldc)
      if (j < nm) *c = from_f32<T>(v[j]);
  }
}

// Lane j < NC: the scale of token m + j.
template <int NC>
__device__ __forceinline__ float token_scale(const Args &a, int m) {
  const int lane = threadIdx.x & 31;
  return lane < NC && m + lane < a.M ? __ldg(a.a_scales + m + lane) : 0.0f;
}
template <bool E4M3, int NC>
__device__ __forceinline__ void finish_any(const Args &a, int m, int n, float sw, float bias, float sa,
                                           const unsigned (&acc)[NC]) {
  if (a.dtype == PKCU_DTYPE_F32) finish<E4M3, NC, float>(a, m, n, sw, bias, sa, acc);
  else if (a.dtype == PKCU_DTYPE_BF16) finish<E4M3, NC, __nv_bfloat16>(a, m, n, sw, bias, sa, acc);
  else finish<E4M3, NC, __half>(a, m, n, sw, bias, sa, acc);
}

// Persistent: a CTA takes output tiles blockIdx.x, + gridDim.x, ... Warp 0 issues
// the TMA loads, one thread of warp 1 the MMAs, warps 2..9 drain one of two
// accumulators while the MMAs of the next tile fill the other. SPLIT: a cluster
// of S CTAs shares one tile, each summing a range of K; the partial sums meet
// through distributed shared memory, in rank order.
template <bool E4M3, int BQ, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
q8_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, Args a,
               int split) {
  using C = Cfg<BQ>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned long long *full = reinterpret_cast<unsigned long long *>(smem + C::STAGES * C::STAGE);
  unsigned long long *empty = full + C::STAGES;
  unsigned long long *acc_full = empty + C::STAGES;    // [2]
  unsigned long long *acc_empty = acc_full + 2;        // [2]
  unsigned long long *done = acc_empty + 2;            // the MMA thread's last commit
  unsigned *tmem_slot = reinterpret_cast<unsigned *>(done + 1);
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (a.M + BQ - 1) / BQ;
  const long long n_tiles = (long long)tiles_m * ((a.N + BP - 1) / BP);
  const int rank = SPLIT ? (int)(blockIdx.x % split) : 0;
  const int kb0 = SPLIT ? (int)((long long)a.nkb * rank / split) : 0;
  const int kb1 = SPLIT ? (int)((long long)a.nkb * (rank + 1) / split) : a.nkb;
  const long long tile0 = SPLIT ? blockIdx.x / split : blockIdx.x;
  const long long step = SPLIT ? n_tiles : gridDim.x;

  // the first tile's loads are on their way before anything else is set up
  const int first_kb = kb1 - kb0 < C::STAGES ? kb1 - kb0 : C::STAGES;
  auto load_stage = [&](int s, int kb, int n0, int m0) {
    unsigned char *st = smem + s * C::STAGE;
    mbar_arrive_tx(full + s, C::STAGE);
    tma_load_2d(st, &map_w, kb * BK, n0, full + s);
    tma_load_2d(st + W_TILE, &map_a, kb * BK, m0, full + s);
  };
  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_a);
    for (int s = 0; s < C::STAGES; s++) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, EPI_WARPS);
    }
    mbar_init(done, 1);
    mbar_init_fence();
    s_abort = 0;
    for (int i = 0; i < first_kb; i++)
      load_stage(i, kb0 + i, (int)(tile0 / tiles_m) * BP, (int)(tile0 % tiles_m) * BQ);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      long long it = first_kb;   // stages filled by this CTA, over all its tiles
      bool stop = false;
      for (long long tile = tile0; tile < n_tiles && !stop; tile += step) {
        const int n0 = (int)(tile / tiles_m) * BP, m0 = (int)(tile % tiles_m) * BQ;
        for (int kb = tile == tile0 ? kb0 + first_kb : kb0; kb < kb1; kb++, it++) {
          const int s = (int)(it % C::STAGES);
          if (it >= C::STAGES && !mbar_wait(empty + s, (unsigned)((it / C::STAGES) - 1) & 1)) {
            atomicAdd(&g_wait_timeouts, 1u);
            s_abort = 1;
          }
          if (*(volatile int *)&s_abort) {
            stop = true;
            break;
          }
          load_stage(s, kb, n0, m0);
        }
      }
      if (*(volatile int *)&s_abort) {
        // a wait ran out somewhere: let this CTA's copies still in flight land
        // (bounded) before its shared memory is released
        for (long long j = it > C::STAGES ? it - C::STAGES : 0; j < it; j++)
          mbar_wait(full + j % C::STAGES, (unsigned)(j / C::STAGES) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr unsigned DESC = idesc(E4M3, BP, BQ);
      long long it = 0;
      int gt = 0;   // tiles of this CTA
      for (long long tile = tile0; tile < n_tiles && !*(volatile int *)&s_abort; tile += step, gt++) {
        const int buf = gt & 1;
        if (gt >= 2 && !mbar_wait(acc_empty + buf, ((gt >> 1) - 1) & 1)) {
          atomicAdd(&g_wait_timeouts, 1u);
          s_abort = 1;
          break;
        }
        tc_fence_after();
        const unsigned d = tmem + buf * BQ;
        for (int kb = kb0; kb < kb1; kb++, it++) {
          const int s = (int)(it % C::STAGES);
          if (!mbar_wait(full + s, (unsigned)(it / C::STAGES) & 1)) {
            atomicAdd(&g_wait_timeouts, 1u);
            s_abort = 1;
            break;
          }
          tc_fence_after();
          const unsigned st = smem_u32(smem + s * C::STAGE);
#pragma unroll
          for (int k = 0; k < BK / 32; k++)
            umma<E4M3>(d, sdesc_k128(st + k * 32), sdesc_k128(st + W_TILE + k * 32), DESC, kb > kb0 || k > 0);
          umma_commit(empty + s);   // the stage is free once these MMAs are done
        }
        if (*(volatile int *)&s_abort) break;
        umma_commit(acc_full + buf);
      }
      // every MMA issued here has finished before the TMEM is released
      umma_commit(done);
      mbar_wait(done, 0);
    }
  } else {
    // warp w reads TMEM lanes 32 (w % 4) .. + 31, half of the columns each
    const int q = warp & 3, half = (warp - 2) >> 2;
    const unsigned lane_addr = ((unsigned)(q * 32) << 16) + half * C::CW;
    int gt = 0;
    for (long long tile = tile0; tile < n_tiles; tile += step, gt++) {
      const int n0 = (int)(tile / tiles_m) * BP, m0 = (int)(tile % tiles_m) * BQ;
      const int buf = gt & 1, n = n0 + q * 32 + lane;
      const float sw = n < a.N ? __ldg(a.w_scales + n) : 0.0f;
      const float bias = a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
      float sa = SPLIT ? 0.0f : token_scale<C::CH>(a, m0 + half * C::CW);
      if (!mbar_wait_warp(acc_full + buf, (gt >> 1) & 1)) {
        if (lane == 0) atomicAdd(&g_wait_timeouts, 1u);
        s_abort = 1;
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < C::CW; c += C::CH) {
        unsigned r[C::CH];
        tmem_ld<C::CH>(tmem + lane_addr + buf * BQ + c, r);
        if constexpr (SPLIT) {
          // the ring is free (every stage's MMAs are behind this accumulator):
          // partial sums to [BQ][128] words, column by column
          unsigned *part = reinterpret_cast<unsigned *>(smem);
#pragma unroll
          for (int j = 0; j < C::CH; j++) part[(half * C::CW + c + j) * BP + q * 32 + lane] = r[j];
        } else {
          const int m = m0 + half * C::CW + c;
          const float now = sa;
          if (c + C::CH < C::CW) {
            sa = token_scale<C::CH>(a, m + C::CH);
          } else {   // the sums are in registers: the accumulator may be filled again
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty + buf);
          }
          if (m < a.M) finish_any<E4M3, C::CH>(a, m, n, sw, bias, now, r);
        }
      }
    }
  }
  if constexpr (SPLIT) {
    // columns (tokens) 8 i .. 8 i + 7 go to rank i mod S, a warp of each
    // quadrant of n; sums in rank order
    const int q = warp & 3, half = (warp - 2) >> 2;
    const int n0 = (int)(tile0 / tiles_m) * BP, m0 = (int)(tile0 % tiles_m) * BQ;
    const int n = n0 + q * 32 + lane;
    const float sw = n < a.N ? __ldg(a.w_scales + n) : 0.0f;
    const float bias = a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
    float sa = warp >= 2 ? token_scale<8>(a, m0 + (rank + half * split) * 8) : 0.0f;
    __syncwarp();
    cluster_sync_all();   // every rank's partial sums are in its shared memory
    if (warp >= 2 && !*(volatile int *)&s_abort) {
      const unsigned base = smem_u32(smem);
      for (int g = rank + half * split; g < BQ / 8; g += 2 * split) {
        if (m0 + g * 8 >= a.M) break;
        unsigned r[8];
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = 0;
        for (int p = 0; p < split; p++) {
          unsigned t[8];
#pragma unroll
          for (int j = 0; j < 8; j++) t[j] = ld_peer(base + 4u * ((g * 8 + j) * BP + q * 32 + lane), p);
#pragma unroll
          for (int j = 0; j < 8; j++)
            r[j] = E4M3 ? __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(t[j])) : r[j] + t[j];
        }
        finish_any<E4M3, 8>(a, m0 + g * 8, n, sw, bias, sa, r);
        sa = token_scale<8>(a, m0 + (g + 2 * split) * 8);
      }
    }
    __syncwarp();
    cluster_sync_all();   // no rank leaves while a peer still reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS)
                 : "memory");
  }
}

// ── many tokens: CTA pairs ────────────────────────────────────────────────────
//
// One 256-token x 256-output tile per pair of CTAs (tcgen05 cta_group::2): each
// CTA brings 128 tokens and half of the outputs' weight rows, the pair's MMA reads
// both CTAs' shared memory, and each CTA's TMEM holds its 128 tokens x 256 sums, in
// two accumulators. So a CTA loads 256 bytes per byte of K for 128 x 256 products,
// two thirds of what a tile of its own would (128 x 256 tiles of single CTAs moved
// 9 to 11 TB/s from L2 and no more: 12000 x 1024 x 4096 98 us, pairs 51).
//
// Here a TMEM lane is a token and its columns are outputs: a thread turns 16
// columns at a time into bytes of its row, with the token's scale in a register
// and the outputs' scales and biases from shared memory, into a swizzled box of
// its warp, which leaves as 64-byte pieces of eight rows per store: 14
// instructions per output with Swish, against 26 for one store per output and
// token. (A TMA store of the box measured the same and asks for aligned rows.)

constexpr int CN = 16;      // columns finished at a time
constexpr int BOX_B = 64;   // bytes of a row of a warp's box

// EPI epilogue warps: 16 (four per scheduler) where there is no residual, 8
// where there is one. With 8 a tile's epilogue takes longer than the products
// of K = 1024; the residual's rows, read by 16 warps at once, cost more than
// that gains (12000 x 1024 x 4096 bf16, Swish: 16 warps 62 us, 8 warps 78; 12000
// x 4096 x 1024 fp32 + residual: 63 and 55).
template <int EPI>
struct PairCfg {
  static constexpr int THREADS = 32 * (2 + EPI);
  static constexpr int BN = 256;
  static constexpr int A_TILE = 128 * BK, B_TILE = BN / 2 * BK;
  static constexpr int STAGE = A_TILE + B_TILE;
  static constexpr int OUT = EPI * 32 * BOX_B;   // a 32-row box per epilogue warp
  static constexpr int PAR = BN * 8;                 // scale and bias of the tile's outputs
  static constexpr int REST = OUT + PAR + 256;
  static constexpr int STAGES = (227 * 1024 - REST) / STAGE < 8 ? (227 * 1024 - REST) / STAGE : 8;
  static constexpr int SMEM = STAGES * STAGE + REST;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int CW = BN / (EPI / 4);   // columns per epilogue warp
};

__device__ __forceinline__ unsigned mapa(unsigned saddr, unsigned rank) {
  unsigned a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  return a;
}
// A load into this CTA's shared memory that reports to a barrier of either CTA
// of the pair (bar: a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(unsigned dst, const CUtensorMap *map, int x, int y, unsigned bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
template <bool E4M3>
__device__ __forceinline__ void umma_pair(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned desc,
                                          unsigned accumulate) {
  if constexpr (E4M3)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(desc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(desc), "r"(accumulate)
        : "memory");
}
// The barrier at this address in both CTAs, once the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(unsigned long long *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((unsigned short)3)
      : "memory");
}
// Relaxed: what it announces is that TMEM reads are done, and no memory operation.
// tcgen05.wait::ld has completed them (their registers are written), and
// tcgen05.fence::before_thread_sync ahead of the arrival with
// tcgen05.fence::after_thread_sync behind the waiter's observing it order tcgen05
// operations across threads whatever the semantics of the arrival itself (PTX's
// memory consistency model for tcgen05: the fences make an execution ordering
// instruction, a relaxed mbarrier operation among them, order what stands before
// the one before what stands behind the other). A release would also wait for the
// stores to C in flight, 3000 cycles a tile.
__device__ __forceinline__ void mbar_arrive_cluster(unsigned bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// TMEM columns without waiting; tmem_wait() before the first use.
__device__ __forceinline__ void tmem_ld_async(unsigned taddr, unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// The registers pass through, so that no use moves above the wait.
__device__ __forceinline__ void tmem_wait(unsigned (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// CN entries n .. n + CN - 1 of a row of R as raw 16-byte words (r NULL: none).
template <typename T>
struct RowChunk {
  static constexpr int VEC = 16 / (int)sizeof(T);
  float4 raw[CN / VEC];
  __device__ __forceinline__ void load(const Args &a, const T *r, int n) {
    if (!r) return;
    if (a.r_vec && n + CN <= a.N) {
#pragma unroll
      for (int i = 0; i < CN / VEC; i++) raw[i] = *reinterpret_cast<const float4 *>(r + n + i * VEC);
    } else {
      T *e = reinterpret_cast<T *>(raw);
#pragma unroll
      for (int j = 0; j < CN; j++) e[j] = n + j < a.N ? r[n + j] : from_f32<T>(0.0f);
    }
  }
};

// CN sums of this thread's token with scales and bias. par: for each pair of
// outputs the two scales and the two biases, in shared memory, the same for
// every lane.
template <bool E4M3>
__device__ __forceinline__ void scale_row(const float4 *par, float sa, const unsigned (&acc)[CN], float (&v)[CN]) {
#pragma unroll
  for (int j = 0; j < CN; j += 2) {
    const float4 p = par[j / 2];
    const float2 s = mul2(make_float2(sum_as_float<E4M3>(acc[j]), sum_as_float<E4M3>(acc[j + 1])), splat2(sa));
    const float2 o = fma2(s, make_float2(p.x, p.y), make_float2(p.z, p.w));
    v[j] = o.x;
    v[j + 1] = o.y;
  }
}
template <typename T>
__device__ __forceinline__ void add_residual_row(const Args &a, bool resid, const RowChunk<T> &rc, float (&v)[CN]) {
  if (resid) {
    const T *x = reinterpret_cast<const T *>(rc.raw);
#pragma unroll
    for (int j = 0; j < CN; j++) v[j] = fmaf(v[j], a.rscale, to_f32(x[j]));
  } else if (a.rscale != 1.0f) {
#pragma unroll
    for (int j = 0; j < CN; j++) v[j] *= a.rscale;
  }
}

// CN finished outputs as chunks 16 bytes wide of this lane's row of the box.
// Chunk c of row r lies at c ^ (r / 2 mod 4): eight rows' chunks fill the banks.
template <typename T>
__device__ __forceinline__ void box_row(unsigned char *box, int first, const float (&v)[CN]) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < CN; j += VEC) {
    alignas(16) T o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) o[i] = from_f32<T>(v[j + i]);
    const int chunk = (first + j) / VEC;
    *reinterpret_cast<uint4 *>(box + lane * BOX_B + ((chunk ^ ((lane >> 1) & 3)) << 4)) =
        *reinterpret_cast<const uint4 *>(o);
  }
}

// The box (32 tokens from m0, 64 bytes of outputs from n0) to C: a store of the
// warp covers eight rows, 64 bytes of each.
template <typename T>
__device__ __forceinline__ void box_store(const Args &a, const unsigned char *box, int m0, int n0) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31, chunk = lane & 3;
  const int n = n0 + chunk * VEC;
  T *c = static_cast<T *>(a.C) + (long long)(m0 + (lane >> 2)) * a.ldc + n;
  const bool whole = a.c_vec && n + VEC <= a.N;
#pragma unroll
  for (int i = 0; i < 4; i++, c += 8 * a.ldc) {
    const int row = 8 * i + (lane >> 2);
    const uint4 d = *reinterpret_cast<const uint4 *>(box + row * BOX_B + ((chunk ^ ((row >> 1) & 3)) << 4));
    if (m0 + row < a.M) {
      if (whole) {
        *reinterpret_cast<uint4 *>(c) = d;
      } else {
        const T *e = reinterpret_cast<const T *>(&d);
#pragma unroll
        for (int j = 0; j < VEC; j++)
          if (n + j < a.N) c[j] = e[j];
      }
    }
  }
}

template <bool E4M3, typename T, int EPI>
__global__ void __launch_bounds__(PairCfg<EPI>::THREADS, 1) __cluster_dims__(2, 1, 1)
q8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, Args a) {
  using C = PairCfg<EPI>;
  constexpr int BN = C::BN;
  // the same offsets in both CTAs: an MMA's descriptors serve both
  extern __shared__ __align__(1024) unsigned char pair_smem[];
  unsigned char *smem = pair_smem;
  unsigned char *out = smem + C::STAGES * C::STAGE;
  float *par = reinterpret_cast<float *>(out + C::OUT);   // [BN / 2] x {scale, scale, bias, bias}
  unsigned long long *full = reinterpret_cast<unsigned long long *>(out + C::OUT + C::PAR);   // the leader's is used
  unsigned long long *empty = full + C::STAGES;
  unsigned long long *acc_full = empty + C::STAGES;    // [2]
  unsigned long long *acc_empty = acc_full + 2;        // [2], the leader's is used
  unsigned long long *done = acc_empty + 2;
  unsigned *tmem_slot = reinterpret_cast<unsigned *>(done + 1);
  int &s_abort = *reinterpret_cast<int *>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = blockIdx.x & 1;   // clusters of two consecutive CTAs; rank 0 leads
  const int tiles_m = (a.M + 255) / 256;
  const long long n_tiles = (long long)tiles_m * ((a.N + BN - 1) / BN);
  const long long step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_a);
    for (int s = 0; s < C::STAGES; s++) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, 2 * EPI);
    }
    mbar_init(done, 1);
    mbar_init_fence();
    s_abort = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers and TMEM exist before either signals or fills the other's
  tc_fence_after();
  const unsigned tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      long long it = 0;
      bool stop = false;
      for (long long tile = blockIdx.x >> 1; tile < n_tiles && !stop; tile += step) {
        const int m0 = (int)(tile % tiles_m) * 256 + (int)rank * 128;
        const int n0 = (int)(tile / tiles_m) * BN + (int)rank * (BN / 2);
        for (int kb = 0; kb < a.nkb; kb++, it++) {
          const int s = (int)(it % C::STAGES);
          if (it >= C::STAGES && !mbar_wait(empty + s, (unsigned)((it / C::STAGES) - 1) & 1)) {
            atomicAdd(&g_wait_timeouts, 1u);
            s_abort = 1;
          }
          if (*(volatile int *)&s_abort) {
            stop = true;
            break;
          }
          // the leader's barrier counts the bytes of both CTAs; a peer's bytes that
          // land before its expect-tx leave the phase open all the same
          if (rank == 0) mbar_arrive_tx(full + s, 2 * C::STAGE);
          const unsigned st = smem_u32(smem + s * C::STAGE), bar = mapa(smem_u32(full + s), 0);
          tma_load_2d_pair(st, &map_a, kb * BK, m0, bar);
          tma_load_2d_pair(st + C::A_TILE, &map_w, kb * BK, n0, bar);
        }
      }
      if (rank == 0 && *(volatile int *)&s_abort) {
        for (long long j = it > C::STAGES ? it - C::STAGES : 0; j < it; j++)
          mbar_wait(full + j % C::STAGES, (unsigned)(j / C::STAGES) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr unsigned DESC = idesc(E4M3, 256, BN);
      long long it = 0;
      int gt = 0;
      for (long long tile = blockIdx.x >> 1; tile < n_tiles && !*(volatile int *)&s_abort; tile += step, gt++) {
        const int buf = gt & 1;
        if (gt >= 2 && !mbar_wait(acc_empty + buf, ((gt >> 1) - 1) & 1)) {
          atomicAdd(&g_wait_timeouts, 1u);
          s_abort = 1;
          break;
        }
        tc_fence_after();
        const unsigned d = tmem + buf * BN;
        for (int kb = 0; kb < a.nkb; kb++, it++) {
          const int s = (int)(it % C::STAGES);
          if (!mbar_wait(full + s, (unsigned)(it / C::STAGES) & 1)) {
            atomicAdd(&g_wait_timeouts, 1u);
            s_abort = 1;
            break;
          }
          tc_fence_after();
          const unsigned st = smem_u32(smem + s * C::STAGE);
#pragma unroll
          for (int k = 0; k < BK / 32; k++)
            umma_pair<E4M3>(d, sdesc_k128(st + k * 32), sdesc_k128(st + C::A_TILE + k * 32), DESC, kb > 0 || k > 0);
          umma_commit_pair(empty + s);
        }
        if (*(volatile int *)&s_abort) break;
        umma_commit_pair(acc_full + buf);
      }
      umma_commit_pair(done);
      mbar_wait(done, 0);
    }
  } else {
    // warp w: tokens 32 (w % 4) .. + 31 of this CTA's 128, C::CW of the columns
    const int q = warp & 3, part = (warp - 2) >> 2;
    const unsigned lane_addr = ((unsigned)(q * 32) << 16) + part * C::CW;
    unsigned char *box = out + (warp - 2) * (32 * BOX_B);
    float *my_par = par + part * C::CW * 2;   // shared by the four warps of this part
    constexpr int COLS = BOX_B / (int)sizeof(T);   // outputs per box
    int gt = 0;
    bool ok = true;   // after a wait that ran out a warp only keeps the others' barriers going
    for (long long tile = blockIdx.x >> 1; tile < n_tiles; tile += step, gt++) {
      const int m0 = (int)(tile % tiles_m) * 256 + (int)rank * 128 + q * 32;
      const int n0 = (int)(tile / tiles_m) * BN + part * C::CW;
      const int m = m0 + lane, buf = gt & 1;
      asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");   // the last tile's pairs are read
      for (int i = q * 32 + lane; i < C::CW; i += 128) {
        const int n = n0 + i, at = (i & ~1) * 2 + (i & 1);
        my_par[at] = n < a.N ? __ldg(a.w_scales + n) : 0.0f;
        my_par[at + 2] = a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
      }
      const float sa = m < a.M ? __ldg(a.a_scales + m) : 0.0f;
      const T *r = a.R && m < a.M ? static_cast<const T *>(a.R) + (long long)m * a.ldr : nullptr;
      RowChunk<T> rc;
      rc.load(a, n0 < a.N ? r : nullptr, n0);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
      if (ok && !mbar_wait_warp(acc_full + buf, (gt >> 1) & 1)) {
        if (lane == 0) atomicAdd(&g_wait_timeouts, 1u);
        s_abort = 1;
        ok = false;
      }
      if (!ok) continue;
      tc_fence_after();
      // CN columns at a time; the next ones' TMEM load is in flight while the
      // activation and the store of these go on, and their residual after it
      unsigned acc[CN];
      const unsigned t0 = tmem + lane_addr + buf * BN;
      tmem_ld_async(t0, acc);
      const float4 *p4 = reinterpret_cast<const float4 *>(my_par);
#pragma unroll 1
      for (int c = 0; c < C::CW; c += CN) {
        float v[CN];
        tmem_wait(acc);
        scale_row<E4M3>(p4 + c / 2, sa, acc, v);
        if (c + CN < C::CW) {
          tmem_ld_async(t0 + c + CN, acc);
        } else {   // this warp's last sums are in registers: the accumulator may be filled again
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(acc_empty + buf), 0));
        }
        activate<CN>(a.act, v);
        add_residual_row<T>(a, r != nullptr, rc, v);
        if (c + CN < C::CW) rc.load(a, n0 + c + CN < a.N ? r : nullptr, n0 + c + CN);
        const int first = c & (COLS - 1);   // this chunk's place in its box
        box_row<T>(box, first, v);
        if (first + CN == COLS) {
          __syncwarp();
          if (n0 + c - first < a.N) box_store<T>(a, box, m0, n0 + c - first);
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // The commits' arrivals at the peer's barriers are no operations of the leader's
  // threads, so the cluster's barrier does not order them before the peer's exit: the
  // peer, too, waits for the last one.
  if (rank == 1 && threadIdx.x == 32) mbar_wait(done, 0);
  __syncwarp();
  // no CTA leaves (or frees its TMEM) while the pair's MMAs, loads or signals may reach it
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS)
                 : "memory");
  }
}

// ── weight preparation (once per weight) ─────────────────────────────────────

// W [K, N] bytes -> [N, Kp] bytes, zeros from column K on: 64 x 64 tiles through
// shared memory, reads along N and writes along K, byte by byte.
__global__ void prep_q8_kernel(const unsigned char *__restrict__ W, unsigned char *__restrict__ out, int K, int N,
                               int Kp) {
  __shared__ unsigned char tile[64][65];
  const long long k0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
  for (int i = threadIdx.x; i < 64 * 64; i += blockDim.x) {
    const int kk = i >> 6, nn = i & 63;
    tile[kk][nn] = k0 + kk < K && n0 + nn < N ? W[(k0 + kk) * N + n0 + nn] : 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 64; i += blockDim.x) {
    const int nn = i >> 6, kk = i & 63;
    if (n0 + nn < N && k0 + kk < Kp) out[(n0 + nn) * Kp + k0 + kk] = tile[kk][nn];
  }
}
__global__ void fill_scales_kernel(const float *__restrict__ scales, int n_scales, float *__restrict__ out, int N) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < N) out[i] = scales[n_scales == 1 ? 0 : i];
}

PK_WAIT_WORD(pk_q8_wait_word)

}  // namespace q8
}  // namespace pk

using namespace pk;

// ── host side ─────────────────────────────────────────────────────────────────

struct pkcu_weight_q8 {
  int K, N, Kp, e4m3, device;
  void *planes;        // [N, Kp] bytes
  float *scales;       // [N]
  CUtensorMap map;     // boxes of 128 rows x 128 bytes
};

namespace {

// 2-D tensor map over rows of `cols` bytes (pitch `pitch`), boxes of box_rows x
// 128 bytes, 128-byte swizzle, zeros out of bounds.
int tmap_bytes(CUtensorMap *map, const void *base, long long rows, long long cols, long long pitch, int box_rows) {
  void *f = nullptr;
  int st = pk_tensor_map_encoder(&f);
  if (st) return st;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)q8::BK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f)(
      map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return pkcu_fail(PKCU_ERR_ARG, "8-bit product: tensor map rejected (%d) for %lld x %lld", (int)r, rows, cols);
  return PKCU_OK;
}

template <bool E4M3, int BQ, bool SPLIT>
int *narrow_flags() {
  static int flags[64];
  return flags;
}

template <bool E4M3, int BQ, bool SPLIT>
int launch(const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, int split, cudaStream_t s) {
  using C = q8::Cfg<BQ>;
  smem_optin(q8::q8_gemm_kernel<E4M3, BQ, SPLIT>, C::SMEM, narrow_flags<E4M3, BQ, SPLIT>());
  const long long tiles = (long long)((a.M + BQ - 1) / BQ) * ((a.N + q8::BP - 1) / q8::BP);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(q8::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  if (SPLIT) {
    cfg.gridDim = dim3((unsigned)(tiles * split));
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  } else {
    cfg.gridDim = dim3((unsigned)(tiles < pkcu_sm_count() ? tiles : pkcu_sm_count()));
  }
  cudaLaunchKernelEx(&cfg, q8::q8_gemm_kernel<E4M3, BQ, SPLIT>, W->map, ma, a, split);
  return pkcu_launch_status("pkcu_wmatmul_q8");
}

template <bool E4M3, typename T, int EPI>
int launch_pair(const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, cudaStream_t s) {
  using C = q8::PairCfg<EPI>;
  static int flags[64];
  smem_optin(q8::q8_pair_kernel<E4M3, T, EPI>, C::SMEM, flags);
  const long long tiles = (long long)((a.M + 255) / 256) * ((a.N + C::BN - 1) / C::BN);
  const long long pairs = pkcu_sm_count() / 2;
  const unsigned grid = 2 * (unsigned)(tiles < pairs ? tiles : pairs);
  q8::q8_pair_kernel<E4M3, T, EPI><<<grid, C::THREADS, C::SMEM, s>>>(W->map, ma, a);
  return pkcu_launch_status("pkcu_wmatmul_q8");
}

template <bool E4M3, typename T>
int launch_pair_as(const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, cudaStream_t s) {
  return a.R ? launch_pair<E4M3, T, 8>(W, ma, a, s) : launch_pair<E4M3, T, 16>(W, ma, a, s);
}
template <typename T>
int launch_pair_type(const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, cudaStream_t s) {
  return W->e4m3 ? launch_pair_as<true, T>(W, ma, a, s) : launch_pair_as<false, T>(W, ma, a, s);
}
int launch_pair_any(const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, cudaStream_t s) {
  if (a.dtype == PKCU_DTYPE_F32) return launch_pair_type<float>(W, ma, a, s);
  if (a.dtype == PKCU_DTYPE_BF16) return launch_pair_type<__nv_bfloat16>(W, ma, a, s);
  return launch_pair_type<__half>(W, ma, a, s);
}

template <bool E4M3, bool SPLIT>
int launch_bq(int bq, const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, int split, cudaStream_t s) {
  switch (bq) {
    case 16: return launch<E4M3, 16, SPLIT>(W, ma, a, split, s);
    case 32: return launch<E4M3, 32, SPLIT>(W, ma, a, split, s);
    case 64: return launch<E4M3, 64, SPLIT>(W, ma, a, split, s);
    default: return launch<E4M3, 128, SPLIT>(W, ma, a, split, s);
  }
}

// Clusters of `split` CTAs of the narrow kernel that run at the same time on the
// current device (one CTA per SM; a cluster lies within a GPC, so fewer than
// SMs / split). Asked of the runtime once per device.
int cluster_slots(int split) {
  static int slots[64][4];
  const int dev = pkcu_device(), k = split == 2 ? 1 : split == 4 ? 2 : 3;
  int n = dev < 64 ? __atomic_load_n(&slots[dev][k], __ATOMIC_ACQUIRE) : 0;
  if (n) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pkcu_sm_count() / split * split));
  cfg.blockDim = dim3(q8::THREADS);
  cfg.dynamicSmemBytes = q8::Cfg<16>::SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  smem_optin(q8::q8_gemm_kernel<false, 16, true>, q8::Cfg<16>::SMEM, narrow_flags<false, 16, true>());
  if (cudaOccupancyMaxActiveClusters(&n, q8::q8_gemm_kernel<false, 16, true>, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = pkcu_sm_count() / split / 2 + 1;
  }
  if (dev < 64) __atomic_store_n(&slots[dev][k], n, __ATOMIC_RELEASE);
  return n;
}

constexpr int PAIR = 256;   // the pair kernel's tokens per tile
struct Plan {
  int bq, split;
};
// Tile (tokens: 16 .. 128 of the one-CTA kernel, 256 of the pair kernel) and split
// of K with the least modelled time: a set-up, the first tile's products, then
// per further tile of a CTA the longer of its products and its epilogue, and the
// last epilogue. Measured on a B200: 0.34 us per 128 of K for any tile of one
// CTA or pair, the epilogues below (the pair kernel's stores of one entry at a
// time where rows of C are not 16-byte aligned), about 2 us for a cluster's
// launch and exchange. Over 14 token counts (1 .. 2000) x 4 weights the choice was
// within 5 % of the best tile and split: M = 128, 1024 -> 4096: 16 tokens 9.1 us, 32
// 6.7, 64 7.3, 128 8.6, pair 12.2; M = 375, 4096 -> 1024: 128 tokens alone 17.7, split
// in two 17.1, in four 12.5, pair 23.9.
Plan plan(int M, int N, int nkb, bool c_vec) {
  static const float epi_us[5] = {0.8f, 1.25f, 2.0f, 3.3f, 5.5f};
  const int sms = pkcu_sm_count();
  Plan best = {PAIR, 1};
  float best_us = INFINITY;
  for (int i = 0; i < 5; i++) {
    const int bq = 16 << i;
    const bool pair = bq == PAIR;
    const int bn = pair ? 256 : q8::BP;
    const long long tiles = (((long long)M + bq - 1) / bq) * (((long long)N + bn - 1) / bn);
    const float epi = pair && !c_vec ? 14.0f : epi_us[i];
    for (int split = 1; split <= (pair ? 1 : 8) && split <= nkb; split *= 2) {
      if (split > 1 && (tiles * split > sms || tiles > cluster_slots(split))) break;
      const long long slots = pair ? sms / 2 : sms;
      const float products = (float)((nkb + split - 1) / split) * 0.34f;
      const float more = split > 1 ? 0.0f : (float)((tiles + slots - 1) / slots - 1);
      const float us = 2.7f + products + more * (products > epi ? products : epi) + epi + (split > 1 ? 2.0f + 0.2f * split : 0.0f);
      if (us < best_us) {
        best_us = us;
        best.bq = bq;
        best.split = split;
      }
    }
  }
  return best;
}
}  // namespace

extern "C" void pkcu_weight_q8_destroy(pkcu_weight_q8 *w) {
  if (!w) return;
  if (w->planes) cudaFree(w->planes);
  if (w->scales) cudaFree(w->scales);
  free(w);
}

extern "C" int pkcu_weight_q8_create(const void *data, int dtype, const float *scales, int n_scales, int K, int N,
                                     pkcu_stream_t stream, pkcu_weight_q8 **out) {
  const char *what = "pkcu_weight_q8_create";
  if (!out) return pkcu_fail(PKCU_ERR_ARG, "%s: NULL out", what);
  *out = nullptr;
  if (dtype != PKCU_DTYPE_I8 && dtype != PKCU_DTYPE_E4M3)
    return pkcu_fail(PKCU_ERR_ARG, "%s: type %d (I8 or E4M3)", what, dtype);
  if (K <= 0 || K > 131071 || N <= 0 || N > 0x7fffff00)
    return pkcu_fail(PKCU_ERR_ARG, "%s: K %d must be 1 .. 131071 and N %d positive", what, K, N);
  if (n_scales != 1 && n_scales != N) return pkcu_fail(PKCU_ERR_ARG, "%s: %d scales (1 or N)", what, n_scales);
  if (!data || !scales) return pkcu_fail(PKCU_ERR_ARG, "%s: NULL argument", what);
  if (misaligned(scales, 4)) return pkcu_fail(PKCU_ERR_ARG, "%s: scales are not aligned to their type", what);
  void *mem = nullptr;   // a tensor map is encoded at a 64-byte boundary
  if (posix_memalign(&mem, 64, sizeof(pkcu_weight_q8)) != 0)
    return pkcu_fail(PKCU_ERR_NOMEM, "%s: host allocation", what);
  memset(mem, 0, sizeof(pkcu_weight_q8));
  pkcu_weight_q8 *w = static_cast<pkcu_weight_q8 *>(mem);
  w->K = K;
  w->N = N;
  w->Kp = (K + 15) & ~15;
  w->e4m3 = dtype == PKCU_DTYPE_E4M3;
  w->device = pkcu_device();
  const size_t bytes = (size_t)N * w->Kp;
  int st = PKCU_OK;
  if (cudaMalloc(&w->planes, bytes) != cudaSuccess) {
    w->planes = nullptr;
    st = PKCU_ERR_NOMEM;
  } else if (cudaMalloc((void **)&w->scales, sizeof(float) * (size_t)N) != cudaSuccess) {
    w->scales = nullptr;
    st = PKCU_ERR_NOMEM;
  }
  if (st) {
    cudaGetLastError();
    pkcu_fail(st, "%s: %zu bytes", what, bytes);
  }
  if (!st) st = tmap_bytes(&w->map, w->planes, N, K, w->Kp, q8::BP);
  if (!st) {
    cudaStream_t s = (cudaStream_t)stream;
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((w->Kp + 63) / 64));
    q8::prep_q8_kernel<<<grid, 256, 0, s>>>(static_cast<const unsigned char *>(data),
                                           static_cast<unsigned char *>(w->planes), K, N, w->Kp);
    q8::fill_scales_kernel<<<(unsigned)((N + 255) / 256), 256, 0, s>>>(scales, n_scales, w->scales, N);
    st = pkcu_launch_status(what);
    if (cudaStreamSynchronize(s) != cudaSuccess && !st)
      st = pkcu_fail(PKCU_ERR_CUDA, "%s: %s", what, cudaGetErrorString(cudaGetLastError()));
  }
  if (st) {
    pkcu_weight_q8_destroy(w);
    return st;
  }
  *out = w;
  return PKCU_OK;
}

extern "C" int pkcu_wmatmul_q8(const void *A, long long lda, const float *a_scales, const pkcu_weight_q8 *W,
                               const float *bias, int act, const void *R, long long ldr, float rscale, void *C,
                               long long ldc, int dtype, int M, pkcu_stream_t stream) {
  const char *what = "pkcu_wmatmul_q8";
  if (!W) return pkcu_fail(PKCU_ERR_ARG, "%s: NULL weight", what);
  if (M < 0 || M > 0x7fffff00) return pkcu_fail(PKCU_ERR_ARG, "%s: %d rows", what, M);
  const int size = dtype_size(dtype);
  if (!size) return pkcu_fail(PKCU_ERR_ARG, "%s: output of type %d (F32, BF16 or F16)", what, dtype);
  if (act < PKCU_ACT_RELU || act > PKCU_ACT_GELU) return pkcu_fail(PKCU_ERR_ARG, "%s: activation %d", what, act);
  if (M == 0) return PKCU_OK;
  if (!A || !a_scales || !C) return pkcu_fail(PKCU_ERR_ARG, "%s: NULL argument", what);
  if (!PK_ALIGNED16(A) || lda % 16 || lda < W->K || lda >= 1LL << 40)
    return pkcu_fail(PKCU_ERR_ARG, "%s: A must be 16-byte aligned, its pitch %lld a multiple of 16 and at least K = %d",
                     what, lda, W->K);
  if (ldc < W->N || (R && ldr < W->N))
    return pkcu_fail(PKCU_ERR_ARG, "%s: rows of C or R shorter than N = %d", what, W->N);
  if (misaligned(C, size) || misaligned(R, size) || misaligned(a_scales, 4) || misaligned(bias, 4))
    return pkcu_fail(PKCU_ERR_ARG, "%s: a pointer is not aligned to its type", what);
  if (W->device != pkcu_device())
    return pkcu_fail(PKCU_ERR_ARG, "%s: the weight is on device %d, the current one is %d", what, W->device,
                     pkcu_device());
  q8::Args a = {};
  a.a_scales = a_scales;
  a.w_scales = W->scales;
  a.bias = bias;
  a.R = R;
  a.C = C;
  a.ldc = ldc;
  a.ldr = ldr;
  a.rscale = rscale;
  a.act = act;
  a.dtype = dtype;
  a.M = M;
  a.N = W->N;
  a.nkb = (W->K + q8::BK - 1) / q8::BK;
  a.r_vec = PK_ALIGNED16(R) && ldr * size % 16 == 0;
  a.c_vec = PK_ALIGNED16(C) && ldc * size % 16 == 0;
  const Plan p = plan(M, W->N, a.nkb, a.c_vec != 0);
  CUtensorMap ma;
  const int st = tmap_bytes(&ma, A, M, W->K, lda, p.bq == PAIR ? 128 : p.bq);
  if (st) return st;
  if (p.bq == PAIR) return launch_pair_any(W, ma, a, (cudaStream_t)stream);
  const int bq = p.bq, split = p.split;
  cudaStream_t s = (cudaStream_t)stream;
  if (split > 1)
    return W->e4m3 ? launch_bq<true, true>(bq, W, ma, a, split, s) : launch_bq<false, true>(bq, W, ma, a, split, s);
  return W->e4m3 ? launch_bq<true, false>(bq, W, ma, a, 1, s) : launch_bq<false, false>(bq, W, ma, a, 1, s);
}
