// k_sample.cu -- one token per row of logits: temperature, top-k, top-p, min-p,
// then the inverse of the cumulative distribution at a given number. No
// counterpart in the reference, whose decode takes the argmax
// (csrc/decoder.c:106-114); it stands beside pkcu_argmax_rows.
//
// Mathematics. Weights w_v = exp((l_v - max) / T), in (0, 1]. Every filter keeps
// a prefix of the order "larger logit first, lower index first among equals":
// top-k its first k, top-p the shortest prefix whose weight reaches p times the
// weight of what top-k left, min-p what is at least min_p. So a row's choice is
// a smallest kept logit tau and how many of the entries equal to it are kept,
// in index order. The token is the first, in index order, at which the kept
// weights' running sum exceeds u times their total.
//
// Exactness. Whether a running sum passes u S or p S is decided between
// neighbours 1e-5 S apart in a large vocabulary, so fp32 weights would draw
// another token than the definition in one row out of a few. Weights are
// computed in fp64 (16 table entries x a degree-5 polynomial: relative error
// below 2e-13) and summed as integers, rounded to 2^-44 of the largest: a sum of
// 2^18 of them fits 64 bits, and it is the same in any order, so the shared
// -memory atomics that gather candidates cannot change a result.
//
// Kernel. A row belongs to a group of threads: a warp (rows up to 2048 entries,
// where there are many), a CTA, or a cluster of CTAs for few long rows. Its logits
// are read once into shared memory and everything after that works from there.
// Top-k and top-p look for their border in a histogram of max - l over linear
// bins (counts are exact; weights in fp32, a hint that exact sums then confirm);
// the entries of the bins up to the border's are listed in index order and the
// rest of the row is not looked at again. Within the border's bin the entries
// are ranked against each other; equal logits beyond a list's length are counted
// by halving the range of keys. For the draw each thread adds up a contiguous
// run of entries, a scan over the threads finds the run that u falls in, and the
// run's warp finds the entry.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

#include "pk_common.cuh"
#include "pk_types.cuh"

namespace pk {
namespace sample {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int MAX_V = 1 << 18;            // sums of weights <= 2^44 fit 62 bits
constexpr int SMEM_LOGITS = 128 * 1024;   // bytes of logits a CTA holds at most
enum { WARP, CTA, CLUSTER };              // what a row's group is

struct Args {
  const void *logits;
  long long ld, n_rows;
  int V, seg;              // seg: entries per CTA of a cluster (or per warp: the row)
  const float *temperature, *top_p, *min_p, *u;
  const int *top_k;
  int *tokens;
  float *logprobs;
};

// Entries as unsigned keys in the order of the values, 0 for what is never
// taken (-infinity, NaN); -0 counts as 0.
__device__ __forceinline__ unsigned key_of(float v) {
  if (!(v > -INFINITY)) return 0;
  const unsigned b = __float_as_uint(__fadd_rn(v, 0.0f));
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// 2^(i / 16)
__constant__ double kPow2[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484,
    1.2968395546510096, 1.3542555469368927, 1.4142135623730951, 1.4768261459394993, 1.5422108254079407,
    1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// exp((v - max) / T) as an integer multiple of 2^-44, rounded; exactly 2^44 for
// v = max. With y = (v - max) 16 log2(e) / T = n + r, |r| <= 1/2: 2^(y / 16) =
// 2^(n div 16) 2^((n mod 16) / 16) e^(r ln 2 / 16), the last by the Taylor series
// of degree 5 (|r ln 2 / 16| < 0.0217: the next term is below 1.5e-13). Sums that
// round to an integer are formed by adding 1.5 2^52.
struct Weight {
  const double *tab;   // kPow2 in shared memory
  double c;            // 16 log2(e) / T
  float max;
  __device__ __forceinline__ u64 operator()(float v) const {
    if (v == max) return 1ull << 44;
    // the maximum of a difference and a limit: also NaN (infinite max, T) becomes the limit
    const double d = (double)v - (double)max;
    const double y = fmax(__dmul_rn(d, c), -16.0 * 60.0);
    constexpr double kShift = 6755399441055744.0;   // 1.5 2^52
    const double t = __dadd_rn(y, kShift);
    const double r = __dadd_rn(y, -__dadd_rn(t, -kShift));
    const int n = __double2loint(t);
    constexpr double L = 0.693147180559945309417 / 16;
    const double z = r * L;
    double p = fma(z, 1.0 / 120, 1.0 / 24);
    p = fma(z, p, 1.0 / 6);
    p = fma(z, p, 0.5);
    p = fma(z, p, 1.0);
    p = fma(z, p, 1.0);
    const double w = __dmul_rn(tab[n & 15], p);
    // times 2^(n div 16 + 44), then to an integer
    const double s = __hiloint2double(__double2hiint(w) + (((n >> 4) + 44) << 20), __double2loint(w));
    return (u64)__double_as_longlong(__dadd_rn(s, 4503599627370496.0)) & 0xfffffffffffffull;   // + 2^52
  }
};

// A row's shared memory, per group (per CTA of a cluster).
template <int MODE>
struct Shared {
  static constexpr int NB = MODE == WARP ? 256 : 1024;    // bins
  static constexpr int CAP = MODE == WARP ? 128 : 1024;   // entries of the list
  static constexpr int RANK = MODE == WARP ? 64 : 512;    // candidates ranked against each other
  static constexpr int NW = MODE == WARP ? 1 : 32;
  u64 part_w[2][NW];        // a warp's part of a reduction or scan; alternating
  unsigned part_n[2][NW], part_lo[2][NW], part_hi[2][NW];
  u64 cta_w[2];             // this CTA's part, read by the cluster; alternating
  unsigned cta_n[2], cta_lo[2], cta_hi[2];
  u64 all_w[RANK];
  float all[RANK];
  float cand[RANK];         // this CTA's candidates, read by the cluster
  union {
    unsigned cnt[NB];
    float mass[NB];
  };
  float list[CAP];          // this CTA's list: values and indices, in index order
  int index[CAP];
  unsigned n_cand;
  int bin;
  unsigned cut_key, cut_take, cut_ties;
};

// Sums and extremes over a row's entries.
struct Sums {
  u64 w;            // weights
  unsigned n;       // entries
  unsigned lo, hi;  // smallest, largest key
};
__device__ __forceinline__ Sums no_sums() { return Sums{0, 0, 0xffffffffu, 0}; }

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(PK_FULL_MASK, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan_u64(u64 v) {   // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(PK_FULL_MASK, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Where entries come from: the row in shared memory, or the list.
template <typename T>
struct FromRow {
  const T *x;
  int n, base;
  __device__ __forceinline__ float value(int i) const { return to_f32(x[i]); }
  __device__ __forceinline__ int index(int i) const { return base + i; }
};
struct FromList {
  const float *x;
  const int *at;
  int n;
  __device__ __forceinline__ float value(int i) const { return x[i]; }
  __device__ __forceinline__ int index(int i) const { return at[i]; }
};

template <typename T, int MODE>
struct Row {
  typedef Shared<MODE> S;
  const Args &a;
  S &s;
  T *x;                 // this group's (CTA's) entries
  int base, n;          // the first one's index in the row, their number
  unsigned rank, size;  // of the cluster
  int tid, nt;          // thread of the group (CTA), threads
  int flip, cflip;
  Weight weight;
  float max, scale;     // bins: (max - l) scale

  // ── the group ──
  __device__ __forceinline__ void lsync() const {   // this group's (CTA's) threads
    if (MODE == WARP) __syncwarp();
    else __syncthreads();
  }
  __device__ __forceinline__ void gsync() const {   // all of the row's threads
    if (MODE == CLUSTER) cg::this_cluster().sync();
    else lsync();
  }
  template <typename P>
  __device__ __forceinline__ P *peer(P *p, unsigned r) const {
    return MODE == CLUSTER ? cg::this_cluster().map_shared_rank(p, r) : p;
  }

  // Totals over the row's threads, to every thread. What is asked for: W weights,
  // N entries, K extreme keys.
  template <bool W, bool N, bool K>
  __device__ __forceinline__ Sums total(Sums v) {
    const int lane = threadIdx.x & 31;
    reduce<W, N, K>(v);
    if (MODE != WARP) {
      const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
      if (lane == 0) {
        if (W) s.part_w[flip][warp] = v.w;
        if (N) s.part_n[flip][warp] = v.n;
        if (K) {
          s.part_lo[flip][warp] = v.lo;
          s.part_hi[flip][warp] = v.hi;
        }
      }
      __syncthreads();   // (two calls later the buffer is free: every thread has passed the next call's barrier)
      v = no_sums();
      if (lane < nw) {
        if (W) v.w = s.part_w[flip][lane];
        if (N) v.n = s.part_n[flip][lane];
        if (K) {
          v.lo = s.part_lo[flip][lane];
          v.hi = s.part_hi[flip][lane];
        }
      }
      reduce<W, N, K>(v);
      flip ^= 1;
    }
    if (MODE == CLUSTER) {
      if (threadIdx.x == 0) {
        if (W) s.cta_w[cflip] = v.w;
        if (N) s.cta_n[cflip] = v.n;
        if (K) {
          s.cta_lo[cflip] = v.lo;
          s.cta_hi[cflip] = v.hi;
        }
      }
      gsync();
      v = no_sums();
      if (lane < (int)size) {
        if (W) v.w = *peer(&s.cta_w[cflip], lane);
        if (N) v.n = *peer(&s.cta_n[cflip], lane);
        if (K) {
          v.lo = *peer(&s.cta_lo[cflip], lane);
          v.hi = *peer(&s.cta_hi[cflip], lane);
        }
      }
      reduce<W, N, K>(v);
      cflip ^= 1;
    }
    return v;
  }
  template <bool W, bool N, bool K>
  __device__ __forceinline__ static void reduce(Sums &v) {
    if (W) v.w = warp_sum_u64(v.w);
    if (N) v.n = __reduce_add_sync(PK_FULL_MASK, v.n);
    if (K) {
      v.lo = __reduce_min_sync(PK_FULL_MASK, v.lo);
      v.hi = __reduce_max_sync(PK_FULL_MASK, v.hi);
    }
  }

  // Sum over the threads before this one (of the whole row, in rank order; LOCAL:
  // of this CTA) and over all of them; most: the largest CTA's sum.
  template <bool LOCAL>
  __device__ __forceinline__ u64 scan(u64 v, u64 &all, u64 &most) {
    const int lane = threadIdx.x & 31;
    const u64 inc = warp_scan_u64(v);
    u64 before = inc - v;
    all = __shfl_sync(PK_FULL_MASK, inc, 31);
    if (MODE != WARP) {
      const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
      if (lane == 0) s.part_w[flip][warp] = all;
      __syncthreads();
      const u64 w = warp_scan_u64(lane < nw ? s.part_w[flip][lane] : 0);
      flip ^= 1;
      if (warp > 0) before += __shfl_sync(PK_FULL_MASK, w, warp - 1);
      all = __shfl_sync(PK_FULL_MASK, w, 31);
    }
    most = all;
    if (MODE == CLUSTER) {
      if (threadIdx.x == 0) s.cta_w[cflip] = all;
      gsync();
      const u64 c = lane < (int)size ? *peer(&s.cta_w[cflip], lane) : 0;
      const u64 cs = warp_scan_u64(c);
      cflip ^= 1;
      if (!LOCAL && rank > 0) before += __shfl_sync(PK_FULL_MASK, cs, rank - 1);
      all = __shfl_sync(PK_FULL_MASK, cs, 31);
      most = c;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(PK_FULL_MASK, most, o);
        most = other > most ? other : most;
      }
      most = __shfl_sync(PK_FULL_MASK, most, 0);
    }
    return before;
  }

  // ── bins ──
  // Linear in max - l, the last bin open-ended (and for an infinite maximum's NaN).
  __device__ __forceinline__ int bin_of(unsigned k) const {
    const float f = (max - value_of(k)) * scale;
    return f < (float)(S::NB - 1) ? (int)f : S::NB - 1;
  }
  __device__ __forceinline__ void clear_bins() {
    lsync();
    for (int b = tid; b < S::NB; b += nt) s.cnt[b] = 0;
    lsync();
  }
  // The first bin at which the bins' running sum reaches target, `before` what the
  // bins before it hold and `inside` what it holds itself (BY_WEIGHT: a hint, in fp32).
  template <bool BY_WEIGHT>
  __device__ int find_bin(u64 target, unsigned &before, unsigned &inside) {
    gsync();   // every CTA's bins are filled
    const int per = (S::NB + nt - 1) / nt, b0 = tid * per;
    float run_w = 0.0f;
    unsigned run_n = 0;
    for (int b = b0; b < b0 + per && b < S::NB; b++)
      for (unsigned r = 0; r < (MODE == CLUSTER ? size : 1); r++) {
        if (BY_WEIGHT) run_w += *peer(&s.mass[b], r);
        else run_n += *peer(&s.cnt[b], r);
      }
    // hints in units of 2^-40 of the largest weight, so that one integer scan serves
    // both (and, being integers, agrees in every CTA of a cluster)
    const u64 mine = BY_WEIGHT ? (u64)(run_w * 0x1p40f) : run_n;
    const u64 goal = BY_WEIGHT ? (target >> 4 ? target >> 4 : 1) : target;
    u64 run;
    {   // the bins are the row's already: scan this CTA's threads only
      const u64 inc = warp_scan_u64(mine);
      run = inc - mine;
      const u64 all = __shfl_sync(PK_FULL_MASK, inc, 31);
      if (MODE != WARP) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
        if (lane == 0) s.part_w[flip][warp] = all;
        if (threadIdx.x == 0) s.bin = S::NB - 1;
        __syncthreads();
        const u64 w = warp_scan_u64(lane < nw ? s.part_w[flip][lane] : 0);
        flip ^= 1;
        if (warp > 0) run += __shfl_sync(PK_FULL_MASK, w, warp - 1);
      } else {
        if (tid == 0) s.bin = S::NB - 1;
        __syncwarp();
      }
    }
    if (run < goal && goal <= run + mine) {
      int b = b0;
      u64 c = 0;
      for (;; b++) {
        float bw = 0.0f;
        unsigned bn = 0;
        for (unsigned r = 0; r < (MODE == CLUSTER ? size : 1); r++) {
          if (BY_WEIGHT) bw += *peer(&s.mass[b], r);
          else bn += *peer(&s.cnt[b], r);
        }
        c = BY_WEIGHT ? (u64)(bw * 0x1p40f) : bn;
        if (run + c >= goal || b == b0 + per - 1 || b == S::NB - 1) break;
        run += c;
      }
      s.bin = b;
      s.cut_take = (unsigned)run;
      s.cut_ties = (unsigned)c;
    }
    lsync();
    before = s.cut_take;
    inside = s.cut_ties;
    return s.bin;
  }

  // The border of a prefix of the order among a source's entries with key > above:
  // the first of them, from the largest, at which the count (BY_WEIGHT: the weight)
  // reaches `target` (1 .. what there is), given the bins of these entries. Leaves
  // s.cut_key, the border's key, s.cut_take, how many of its equals belong to the
  // prefix, s.cut_ties, how many there are.
  template <bool BY_WEIGHT, typename Src>
  __device__ void border(const Src &src, unsigned above, u64 target, int bin, unsigned bin_before, unsigned bin_inside) {
    unsigned hi = 0xffffffffu, lo = above;    // the border's key is in (lo, hi]
    u64 before = bin_before;                  // count or weight of the keys > hi
    unsigned inside = bin_inside;             // entries with keys in (lo, hi]
    bool found = !BY_WEIGHT;                  // counts need no confirmation, only the bin's keys
    for (int tries = 0; tries < (BY_WEIGHT ? 3 : 1); tries++) {
      Sums up = no_sums(), in = no_sums();
      for (int i = tid; i < src.n; i += nt) {
        const unsigned k = key_of(src.value(i));
        if (k <= above) continue;
        const int b = bin_of(k);
        if (b > bin) continue;
        const u64 w = BY_WEIGHT ? weight(value_of(k)) : 0;
        if (b < bin) {
          up.w += w;
        } else {
          in.n++;
          in.lo = min(in.lo, k);
          in.hi = ::max(in.hi, k);
          in.w += w;
        }
      }
      if (BY_WEIGHT) up = total<true, false, false>(up);
      in = total<BY_WEIGHT, BY_WEIGHT, true>(in);
      if (BY_WEIGHT) {
        found = up.w < target && target <= up.w + in.w;
        before = up.w;
        inside = in.n;
      }
      if (found) {
        hi = in.hi;
        lo = in.lo - 1;
        break;
      }
      bin = target <= up.w ? ::max(bin - 1, 0) : min(bin + 1, S::NB - 1);   // a rounding of the hint: one bin off
    }
    if (!found) {   // all of them
      Sums in = no_sums();
      for (int i = tid; i < src.n; i += nt) {
        const unsigned k = key_of(src.value(i));
        if (k <= above) continue;
        in.n++;
        in.hi = ::max(in.hi, k);
      }
      in = total<false, true, true>(in);
      inside = in.n;
      hi = in.hi;
      before = 0;
    }
    // too many to rank: halve the range of keys until few are left, or one key
    while (inside > (unsigned)S::RANK && hi - lo > 1) {
      const unsigned mid = lo + (hi - lo) / 2;
      Sums up = no_sums();   // keys in (mid, hi]
      for (int i = tid; i < src.n; i += nt) {
        const unsigned k = key_of(src.value(i));
        if (k <= mid || k > hi) continue;
        up.n++;
        if (BY_WEIGHT) up.w += weight(value_of(k));
      }
      up = total<BY_WEIGHT, true, false>(up);
      const u64 more = BY_WEIGHT ? up.w : up.n;
      if (before + more >= target) {
        lo = mid;
        inside = up.n;
      } else {
        before += more;
        hi = mid;
        inside -= up.n;
      }
    }
    lsync();   // the caller's and the bin search's words are read
    if (inside > (unsigned)S::RANK) {   // all equal
      if (tid == 0) {
        const u64 each = BY_WEIGHT ? weight(value_of(hi)) : 1;
        s.cut_key = hi;
        s.cut_ties = inside;
        s.cut_take = (unsigned)((target - before + each - 1) / each);
      }
      lsync();
      return;
    }
    // list the candidates, in every CTA the same ones (in any order)
    if (tid == 0) s.n_cand = 0;
    lsync();
    for (int i = tid; i < src.n; i += nt) {
      const unsigned k = key_of(src.value(i));
      if (k > lo && k <= hi) s.cand[atomicAdd(&s.n_cand, 1u)] = value_of(k);
    }
    gsync();
    unsigned n_all = 0;
    for (unsigned r = 0; r < (MODE == CLUSTER ? size : 1); r++) {
      const unsigned m = *peer(&s.n_cand, r);
      const float *c = peer(s.cand, r);
      for (unsigned i = tid; i < m; i += nt) {
        s.all[n_all + i] = c[i];
        if (BY_WEIGHT) s.all_w[n_all + i] = weight(c[i]);
      }
      n_all += m;
    }
    lsync();
    for (unsigned i = tid; i < n_all; i += nt) {
      const float v = s.all[i];
      u64 more = 0;         // count or weight of the larger ones
      unsigned ties = 0;
      for (unsigned j = 0; j < n_all; j++) {
        const float o = s.all[j];
        ties += o == v;
        if (o > v) more += BY_WEIGHT ? s.all_w[j] : 1;
      }
      const u64 each = BY_WEIGHT ? s.all_w[i] : 1, start = before + more;
      if (start < target && target <= start + each * ties) {   // equals write the same
        s.cut_key = key_of(v);
        s.cut_ties = ties;
        s.cut_take = (unsigned)((target - start + each - 1) / each);
      }
    }
    gsync();   // (cluster: the candidates are read)
  }

  // The entries with key >= cut into the list, in index order, where every CTA's fit.
  template <typename Src>
  __device__ bool make_list(const Src &src, unsigned cut, FromList &out) {
    const int per = ((src.n + nt - 1) / nt) | 1;   // odd: no bank conflicts between the threads' runs
    const int i0 = min(tid * per, src.n), i1 = min(i0 + per, src.n);
    unsigned c = 0;
    for (int i = i0; i < i1; i++) c += key_of(src.value(i)) >= cut;
    u64 all, most;
    u64 at = scan<true>(c, all, most);
    if (most > (u64)S::CAP) return false;
    if (c)
      for (int i = i0; i < i1; i++) {
        const float v = src.value(i);
        if (key_of(v) >= cut) {
          s.list[at] = v;
          s.index[at] = src.index(i);
          at++;
        }
      }
    out.x = s.list;
    out.at = s.index;
    // this CTA's own number: the last thread's end
    if (tid == nt - 1) s.n_cand = (unsigned)at;
    lsync();
    out.n = (int)s.n_cand;
    lsync();
    return true;
  }

  // What the filters leave of a source, and the draw from it. Kept are keys > cut
  // and the first `take` of its `ties` equals.
  template <typename Src>
  __device__ void top_p_and_draw(const Src &src, long long row, unsigned cut, unsigned take, unsigned ties, float p,
                                 float mp, double temp);
  template <typename Src>
  __device__ void draw(const Src &src, long long row, unsigned cut, unsigned take, unsigned ties, float mp, double temp);
  __device__ void run(long long row);
};

template <typename T, int MODE>
template <typename Src>
__device__ void Row<T, MODE>::draw(const Src &src, long long row, unsigned cut, unsigned take, unsigned ties, float mp,
                                   double temp) {
  const int lane = threadIdx.x & 31;
  // min-p: a weight at least min_p of the largest, which always stays
  u64 least = 0;
  if (mp > 0.0f) least = (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * 0x1p44);
  const int per = ((src.n + nt - 1) / nt) | 1;
  const int i0 = min(tid * per, src.n), i1 = min(i0 + per, src.n);
  const bool part = take < ties;
  unsigned tie0 = 0;   // equals of the cut before this thread's run
  if (part) {
    unsigned c = 0;
    for (int i = i0; i < i1; i++) c += key_of(src.value(i)) == cut;
    u64 all, most;
    tie0 = (unsigned)scan<false>(c, all, most);
  }
  u64 mine = 0;
  unsigned seen = tie0;
  for (int i = i0; i < i1; i++) {
    const float v = src.value(i);
    const unsigned k = key_of(v);
    if (k < cut || k == 0) continue;
    if (k == cut && part && seen++ >= take) continue;
    const u64 w = weight(v);
    mine += w >= least ? w : 0;
  }
  u64 sum, most;
  const u64 before = scan<false>(mine, sum, most);
  const float uu = __ldg(a.u + row);
  u64 target = uu > 0.0f ? (u64)((double)uu * (double)sum) : 0;   // floor; the running sum has to exceed it
  target = target < sum ? target : sum - 1;
  const unsigned owner = __ballot_sync(PK_FULL_MASK, target >= before && target < before + mine);
  if (!owner) return;
  // this warp has the run: its lanes take the run's entries
  const int o = __ffs(owner) - 1;
  const int j0 = __shfl_sync(PK_FULL_MASK, i0, o), j1 = __shfl_sync(PK_FULL_MASK, i1, o);
  u64 run = __shfl_sync(PK_FULL_MASK, before, o);
  seen = __shfl_sync(PK_FULL_MASK, tie0, o);
  for (int j = j0; j < j1; j += 32) {
    const int i = j + lane;
    const float v = i < j1 ? src.value(i) : -INFINITY;
    const unsigned k = key_of(v);
    bool keep = k > cut || (k == cut && k != 0);
    if (part) {
      const unsigned same = __ballot_sync(PK_FULL_MASK, k == cut);
      if (k == cut) keep = seen + __popc(same & ((1u << lane) - 1)) < take;
      seen += __popc(same);
    }
    u64 w = keep ? weight(v) : 0;
    w = w >= least ? w : 0;
    const u64 inc = warp_scan_u64(w);
    const unsigned past = __ballot_sync(PK_FULL_MASK, run + inc > target);
    if (past) {
      if (lane == __ffs(past) - 1) {
        a.tokens[row] = src.index(i);
        if (a.logprobs) {
          // log(w / S): the exponent itself less log S, S in units of the largest weight
          const double y = v == max ? 0.0 : ((double)v - (double)max) / temp;
          const double over = (double)(sum - (1ull << 44)) * 0x1p-44;
          a.logprobs[row] = (float)(y - (double)log1pf((float)over));
        }
      }
      break;
    }
    run += __shfl_sync(PK_FULL_MASK, inc, 31);
  }
}

template <typename T, int MODE>
template <typename Src>
__device__ void Row<T, MODE>::top_p_and_draw(const Src &src, long long row, unsigned cut, unsigned take, unsigned ties,
                                             float p, float mp, double temp) {
  if (p < 1.0f) {
    clear_bins();
    Sums t = no_sums();
    for (int i = tid; i < src.n; i += nt) {
      const float v = src.value(i);
      const unsigned k = key_of(v);
      if (k <= cut) continue;
      const u64 w = weight(v);
      t.w += w;
      atomicAdd(&s.mass[bin_of(k)], (float)w * 0x1p-44f);
    }
    t = total<true, false, false>(t);
    const u64 each = cut ? weight(value_of(cut)) : 0;
    const u64 sum = t.w + take * each;
    // the least integer that is at least p times the sum (and at least 1)
    u64 target = p > 0.0f ? (u64)ceil((double)p * (double)sum) : 1;
    target = target < 1 ? 1 : target < sum ? target : sum;
    if (target > t.w) {   // inside the equals of the top-k's border
      take = (unsigned)((target - t.w + each - 1) / each);
    } else {
      unsigned before, inside;
      const int bin = find_bin<true>(target, before, inside);
      // from here on only the entries of the bins up to that one count, and where
      // they are few only they are looked at: keys from the bin's lower edge on
      border<true>(src, cut, target, bin, 0, 0);
      cut = s.cut_key;
      take = s.cut_take;
      ties = s.cut_ties;
    }
  }
  draw(src, row, cut, take, ties, mp, temp);
}

template <typename T, int MODE>
__device__ void Row<T, MODE>::run(long long row) {
  const T *in = static_cast<const T *>(a.logits) + row * a.ld + base;
  // the row, once; its largest and smallest values
  Sums v = no_sums();
#pragma unroll 8
  for (int i = tid; i < n; i += nt) {
    const T e = in[i];
    x[i] = e;
    const unsigned k = key_of(to_f32(e));
    if (k) {
      v.lo = min(v.lo, k);
      v.hi = ::max(v.hi, k);
      v.n++;
    }
  }
  v = total<false, true, true>(v);
  const unsigned max_key = v.hi;
  if (v.n == 0) {   // nothing to take
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  lsync();
  FromRow<T> all{x, n, base};
  max = value_of(max_key);
  const float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  if (!(temp > 0.0f)) {   // greedy: the first largest
    Sums f = no_sums();
    for (int i = tid; i < n; i += nt)
      if (key_of(all.value(i)) == max_key) f.lo = min(f.lo, (unsigned)(base + i));
    f = total<false, false, true>(f);
    if (rank == 0 && tid == 0) {
      a.tokens[row] = (int)f.lo;
      if (a.logprobs) a.logprobs[row] = 0.0f;
    }
    return;
  }
  weight.c = 16.0 * 1.44269504088896340736 / (double)temp;
  weight.max = max;
  const int k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float p = a.top_p ? __ldg(a.top_p + row) : 1.0f;
  const float mp = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  // bins over the values' range, at most 64 wide (below it one open bin)
  float range = max - value_of(v.lo);
  range = range < 64.0f ? range : 64.0f;
  scale = (float)(S::NB - 2) / fmaxf(range, 1e-30f);
  if (k > 0 && (unsigned)k < v.n) {
    clear_bins();
    for (int i = tid; i < n; i += nt) {
      const unsigned e = key_of(all.value(i));
      if (e) atomicAdd(&s.cnt[bin_of(e)], 1u);
    }
    unsigned before, inside;
    const int bin = find_bin<false>((u64)k, before, inside);
    border<false>(all, 0, (u64)k, bin, before, inside);
    const unsigned cut = s.cut_key, take = s.cut_take, ties = s.cut_ties;
    lsync();
    FromList few;
    if (make_list(all, cut, few)) top_p_and_draw(few, row, cut, take, ties, p, mp, (double)temp);
    else top_p_and_draw(all, row, cut, take, ties, p, mp, (double)temp);
  } else {
    top_p_and_draw(all, row, 0, 0, 0, p, mp, (double)temp);
  }
}

template <typename T, int MODE>
__global__ void __launch_bounds__(MODE == WARP ? 256 : 1024) sample_kernel(Args a) {
  typedef Shared<MODE> S;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ double tab[16];
  if (threadIdx.x < 16) tab[threadIdx.x] = kPow2[threadIdx.x];
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const size_t group = sizeof(S) + (((size_t)a.seg * sizeof(T) + 15) & ~(size_t)15);
  unsigned char *mem = smem + (MODE == WARP ? warp * group : 0);
  S &s = *reinterpret_cast<S *>(mem);
  Row<T, MODE> r{a, s};
  r.x = reinterpret_cast<T *>(mem + sizeof(S));
  r.weight.tab = tab;
  r.flip = r.cflip = 0;
  r.size = MODE == CLUSTER ? cg::this_cluster().num_blocks() : 1;
  r.rank = MODE == CLUSTER ? cg::this_cluster().block_rank() : 0;
  r.base = (int)r.rank * a.seg;
  r.n = a.V - r.base < a.seg ? a.V - r.base : a.seg;
  if (r.n < 0) r.n = 0;
  r.tid = MODE == WARP ? threadIdx.x & 31 : threadIdx.x;
  r.nt = MODE == WARP ? 32 : blockDim.x;
  const long long step = MODE == WARP ? (long long)gridDim.x * (blockDim.x >> 5) : gridDim.x / r.size;
  for (long long row = MODE == WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x / r.size;
       row < a.n_rows; row += step) {
    r.run(row);
    r.gsync();   // shared memory is free for the next row, the peers' reads are done
  }
}

template <typename T, int MODE>
int launch(Args a, int size, int threads, cudaStream_t s) {
  static int flags[64];
  a.seg = MODE == CLUSTER ? ((a.V + size - 1) / size + 31) & ~31 : a.V;
  const int groups = MODE == WARP ? threads / 32 : 1;
  const size_t bytes = groups * (sizeof(Shared<MODE>) + (((size_t)a.seg * sizeof(T) + 15) & ~(size_t)15));
  smem_optin(sample_kernel<T, MODE>, 200 * 1024, flags);
  const long long most = 1 << 20;
  const long long rows = (a.n_rows + groups - 1) / groups;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((rows < most ? rows : most) * size));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  if (MODE == CLUSTER) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  cudaLaunchKernelEx(&cfg, sample_kernel<T, MODE>, a);
  return pkcu_launch_status("pkcu_sample_rows");
}

template <typename T>
int launch_rows(const Args &a, cudaStream_t s) {
  static const char *e = getenv("SMODE");
  int mode = -1, size = 1, threads = 0;
  if (e) sscanf(e, "%d,%d,%d", &mode, &size, &threads);
  if (mode == 0 || (mode < 0 && a.V <= 2048 && a.n_rows > pkcu_sm_count())) return launch<T, WARP>(a, 1, mode < 0 ? 256 : threads, s);
  if (mode < 0) {
    // CTAs per row: what the logits need, and more while that leaves SMs idle
    while ((((a.V + size - 1) / size + 31) & ~31) * (long long)sizeof(T) > SMEM_LOGITS) size *= 2;
    while (size < 8 && a.n_rows * size * 2 <= pkcu_sm_count() && a.V / size > 4096) size *= 2;
    const int each = (a.V + size - 1) / size;
    threads = each <= 2048 ? 128 : each <= 8192 ? 512 : 1024;
  }
  return size > 1 ? launch<T, CLUSTER>(a, size, threads, s) : launch<T, CTA>(a, 1, threads, s);
}

}  // namespace sample
}  // namespace pk

using namespace pk;

extern "C" int pkcu_sample_rows(const void *logits, int dtype, long long ld, const float *temperature,
                                const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                                int32_t *tokens, float *logprobs, long long n_rows, int V, pkcu_stream_t stream) {
  const char *what = "pkcu_sample_rows";
  if (n_rows < 0 || V <= 0 || V > sample::MAX_V)
    return pkcu_fail(PKCU_ERR_ARG, "%s: %lld rows of %d (1 .. %d)", what, n_rows, V, sample::MAX_V);
  const int size = dtype_size(dtype);
  if (!size) return pkcu_fail(PKCU_ERR_ARG, "%s: logits of type %d (F32, BF16 or F16)", what, dtype);
  if (n_rows == 0) return PKCU_OK;
  if (!logits || !u || !tokens) return pkcu_fail(PKCU_ERR_ARG, "%s: NULL argument", what);
  if (ld < V) return pkcu_fail(PKCU_ERR_ARG, "%s: ld %lld is less than V = %d", what, ld, V);
  if (misaligned(logits, size) || misaligned(temperature, 4) || misaligned(top_k, 4) || misaligned(top_p, 4) ||
      misaligned(min_p, 4) || misaligned(u, 4) || misaligned(tokens, 4) || misaligned(logprobs, 4))
    return pkcu_fail(PKCU_ERR_ARG, "%s: a pointer is not aligned to its type", what);
  const sample::Args a = {logits, ld, n_rows, V, 0, temperature, top_p, min_p, u, top_k, tokens, logprobs};
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == PKCU_DTYPE_F32) return sample::launch_rows<float>(a, s);
  if (dtype == PKCU_DTYPE_BF16) return sample::launch_rows<__nv_bfloat16>(a, s);
  return sample::launch_rows<__half>(a, s);
}
