// k_q8gemm.cu -- products of 8-bit activations and 8-bit weights on the tcgen05
// tensor cores, with the bias, the activation and the residual in the epilogue:
//
//   C[m, n] = R[m, n] + r act(s_a[m] s_w[n] sum_k A[m, k] W[k, n] + bias[n])
//
// for int8 (kind::i8, exact 32-bit integer sums) and e4m3 (kind::f8f6f4, fp32
// sums). The library's other products (k_tcgemm.cu) take fp32 activations as
// three bf16 parts: three MMAs at half this rate per product.
//
// Orientation. The kernel computes C transposed: 128 rows of the K-major weight
// (128 outputs n) are the MMA's M, BQ activation rows (tokens m) its N. A TMEM
// lane then holds one n and its columns run over m, so a warp's loads and stores
// of one token are 32 consecutive n whatever the pitch or alignment of C (rows of
// 1025 logits included); bias and weight scale are one register per thread; and
// one token wastes nothing but columns of a 16-wide tile.
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

#include <mutex>

#include "pk_common.cuh"
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
};

// ── PTX wrappers ──────────────────────────────────────────────────────────────

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y,
                                            unsigned long long *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
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
__device__ __forceinline__ void umma_commit(unsigned long long *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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

// NC consecutive TMEM columns of this warp's 32 lanes.
template <int NC>
__device__ __forceinline__ void tmem_ld(unsigned taddr, unsigned (&r)[NC]) {
  static_assert(NC == 8 || NC == 16 || NC == 32, "");
  if constexpr (NC == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
  else if constexpr (NC == 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ── epilogue ──────────────────────────────────────────────────────────────────

// Tokens m .. m + NC - 1 of output n, from their sums; sa: this lane's a_scales
// entry (lane j holds token m + j's). Runs on whole warps; a lane past N only
// lends its scale.
template <bool E4M3, int NC, typename T>
__device__ __forceinline__ void finish(const Args &a, int m, int n, float sw, float bias, float sa,
                                       const unsigned (&acc)[NC]) {
  float v[NC];
#pragma unroll
  for (int j = 0; j < NC; j++) {
    const float s = E4M3 ? __uint_as_float(acc[j]) : __int2float_rn((int)acc[j]);
    v[j] = fmaf(s * sw, __shfl_sync(PK_FULL_MASK, sa, j), bias);
  }
  switch (a.act) {
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
        const float2 s = glu_gate2(make_float2(v[j], v[j + 1]), make_float2(v[j], v[j + 1]), splat2(-0.0f));
        v[j] = s.x;
        v[j + 1] = s.y;
      }
      break;
    case PKCU_ACT_GELU:
#pragma unroll
      for (int j = 0; j < NC; j++) v[j] = 0.5f * v[j] * (1.0f + erff(v[j] * 0.70710678118654752f));
      break;
    default: break;
  }
  if (n >= a.N) return;
  const int nm = a.M - m < NC ? a.M - m : NC;
  if (a.R) {
    const T *r = static_cast<const T *>(a.R) + (long long)m * a.ldr + n;
    T x[NC];
#pragma unroll
    for (int j = 0; j < NC; j++)
      if (j < nm) x[j] = r[(long long)j * a.ldr];
#pragma unroll
    for (int j = 0; j < NC; j++)
      if (j < nm) v[j] = fmaf(v[j], a.rscale, to_f32(x[j]));
  } else if (a.rscale != 1.0f) {
#pragma unroll
    for (int j = 0; j < NC; j++) v[j] *= a.rscale;
  }
  T *c = static_cast<T *>(a.C) + (long long)m * a.ldc + n;
#pragma unroll
  for (int j = 0; j < NC; j++)
    if (j < nm) c[(long long)j * a.ldc] = from_f32<T>(v[j]);
}

template <bool E4M3, int NC>
__device__ __forceinline__ void finish_any(const Args &a, int m, int n, float sw, float bias,
                                           const unsigned (&acc)[NC]) {
  const int lane = threadIdx.x & 31;
  const float sa = lane < NC && m + lane < a.M ? __ldg(a.a_scales + m + lane) : 0.0f;
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

  if (threadIdx.x == 0) {
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
      long long it = 0;   // stages filled by this CTA, over all its tiles
      bool stop = false;
      for (long long tile = tile0; tile < n_tiles && !stop; tile += step) {
        const int n0 = (int)(tile / tiles_m) * BP, m0 = (int)(tile % tiles_m) * BQ;
        for (int kb = kb0; kb < kb1; kb++, it++) {
          const int s = (int)(it % C::STAGES);
          if (it >= C::STAGES && !mbar_wait(empty + s, (unsigned)((it / C::STAGES) - 1) & 1)) {
            atomicAdd(&g_wait_timeouts, 1u);
            s_abort = 1;
          }
          if (*(volatile int *)&s_abort) {
            stop = true;
            break;
          }
          unsigned char *st = smem + s * C::STAGE;
          mbar_arrive_tx(full + s, C::STAGE);
          tma_load_2d(st, &map_w, kb * BK, n0, full + s);
          tma_load_2d(st + W_TILE, &map_a, kb * BK, m0, full + s);
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
      // the outcome is made warp-uniform: tcgen05.ld needs every lane
      if (!__all_sync(PK_FULL_MASK, mbar_wait(acc_full + buf, (gt >> 1) & 1))) {
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
          if (m < a.M) finish_any<E4M3, C::CH>(a, m, n, sw, bias, r);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + buf);
    }
  }
  if constexpr (SPLIT) {
    __syncwarp();
    cluster_sync_all();   // every rank's partial sums are in its shared memory
    if (warp >= 2 && !*(volatile int *)&s_abort) {
      // columns (tokens) 8 i .. 8 i + 7 go to rank i mod S, a warp of each
      // quadrant of n; sums in rank order
      const int q = warp & 3, half = (warp - 2) >> 2;
      const int n0 = (int)(tile0 / tiles_m) * BP, m0 = (int)(tile0 % tiles_m) * BQ;
      const int n = n0 + q * 32 + lane;
      const float sw = n < a.N ? __ldg(a.w_scales + n) : 0.0f;
      const float bias = a.bias && n < a.N ? __ldg(a.bias + n) : 0.0f;
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
        finish_any<E4M3, 8>(a, m0 + g * 8, n, sw, bias, r);
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

// ── weight preparation (once per weight) ─────────────────────────────────────

// W [K, N] bytes -> [N, Kp] bytes, zeros from column K on: 64 x 64 tiles through
// shared memory, reads along N and writes along K in 4-byte words.
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

PK_WAIT_TIMEOUTS_ACCESSOR(pk_q8_wait_timeouts_acc)

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
int launch(const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, int split, cudaStream_t s) {
  using C = q8::Cfg<BQ>;
  static int flags[64];
  smem_optin(q8::q8_gemm_kernel<E4M3, BQ, SPLIT>, C::SMEM, flags);
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

template <bool E4M3, bool SPLIT>
int launch_bq(int bq, const pkcu_weight_q8 *W, const CUtensorMap &ma, const q8::Args &a, int split, cudaStream_t s) {
  switch (bq) {
    case 16: return launch<E4M3, 16, SPLIT>(W, ma, a, split, s);
    case 32: return launch<E4M3, 32, SPLIT>(W, ma, a, split, s);
    case 64: return launch<E4M3, 64, SPLIT>(W, ma, a, split, s);
    case 128: return launch<E4M3, 128, SPLIT>(W, ma, a, split, s);
    default: return launch<E4M3, 256, false>(W, ma, a, split, s);
  }
}

}  // namespace

extern "C" int pk_q8_wait_timeouts(unsigned *count, int reset) { return q8::pk_q8_wait_timeouts_acc(count, reset); }

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
  const int sms = pkcu_sm_count();
  const long long tiles_n = (W->N + q8::BP - 1) / q8::BP;
  int bq = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  while (bq > 64 && tiles_n * ((M + bq - 1) / bq) * 2 < sms) bq >>= 1;
  const long long tiles = tiles_n * ((M + bq - 1) / bq);
  int split = 1;
  if (bq <= 128)
    while (split < 8 && tiles * split * 2 <= sms && split * 2 <= a.nkb) split *= 2;
  CUtensorMap ma;
  const int st = tmap_bytes(&ma, A, M, W->K, lda, bq);
  if (st) return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (split > 1)
    return W->e4m3 ? launch_bq<true, true>(bq, W, ma, a, split, s) : launch_bq<false, true>(bq, W, ma, a, split, s);
  return W->e4m3 ? launch_bq<true, false>(bq, W, ma, a, 1, s) : launch_bq<false, false>(bq, W, ma, a, 1, s);
}
