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
// Kernel. A row belongs to a group of threads: a warp (rows up to 2016 entries,
// where there are many), a CTA, or a cluster of CTAs for few long rows. Its logits
// are read once into shared memory and everything after that works from there.
// Top-k and top-p look for their border in a histogram of max - l over linear
// bins (counts are exact; weights in coarse units, a hint that exact sums then
// confirm); a warp's top-k bounds it by its lanes' largest entries instead. What is
// as large as the border's bin is listed in index order. A list of at most 256 is
// finished by one warp in its registers: it halves the range of keys, counting or
// adding up weights by warp reductions, until the border is found, then draws.
// A longer list, or the row, is looked through again by all threads: the entries of
// the border's bin are ranked against each other (more than fit are first reduced
// by halving the range of keys), and for the draw each thread adds up a contiguous
// run of entries, a scan over the threads finds the run that u falls in, and the
// run's warp finds the entry.
//
// What bounds it, on a B200. Not memory: 12000 x 1025 fp32 logits are 49 MB, 7.5 us
// of reading, and take 30 us without filters (issue slots: 62 instructions per entry,
// of which the fp64 exponential and its conversions are 40), 37 us with top-k (one per
// listed entry, but the list), 74 us with top-p (also the bins' atomics and a second
// look at the row), 73 us with all kinds mixed. 256 x 32000 fp32, 5 us of reading: 28
// us without filters, 32 with top-k, 76 with top-p, whose nuclei of thousands of
// entries are looked through three or four times between barriers. 1 x 131072 bf16, in a
// cluster of eight: 11 us without filters, 17 with top-k, 32 with top-p: one cluster
// barrier after another. Not kept: contiguous runs per thread in every pass with the
// draw's sums taken from top-p's (the same), more loads in flight per thread (more registers).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "pk_common.cuh"
#include "pk_types.cuh"

namespace pk {
namespace sample {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int MAX_V = 1 << 18;            // sums of weights <= 2^44 fit 62 bits
constexpr int SMEM_VALUES = 128 * 1024;     // bytes of values a CTA holds at most
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

// Entries in shared memory are fp32 values, -infinity for what is never taken
// (-infinity, NaN), +0 for zeros of both signs. Keys: finite and +infinite values
// as unsigned numbers in the same order, for halving a range of values.
__device__ __forceinline__ float clean(float v) { return __fadd_rn(fmaxf(v, -INFINITY), 0.0f); }
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned b = __float_as_uint(v);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
  return __uint_as_float(k ^ (~(unsigned)((int)k >> 31) | 0x80000000u));
}

// e^x on |x| <= ln 2 / 32 by the Taylor series of degree 5 (the next term is below
// 1.5e-13), with x = r L, L = ln 2 / 16, as K (((((r + a) r + b) r + c) r + d) r + e),
// K = L^5 / 120, a = 5 / L, b = 20 / L^2, c = 60 / L^3, d = 120 / L^4, e = 120 / L^5:
// one constant per operation, each read from constant memory as an operand (as
// literals they took more instructions than the arithmetic). kPow2: K 2^44 2^(i / 16).
__constant__ double kExp[5] = {115.41560327111708, 10656.609182748713, 737963.386590881, 34068995.78215325, 786418740.2076721};
__constant__ double kPow2[16] = {
    22369.998507118962, 23360.40295392472, 24394.656351723497, 25474.700059431234,
    26602.56138726612, 27780.35740213786, 29010.298901515907, 30294.694563235866,
    31635.955279033526, 33036.59867994085, 34499.25386203834, 36026.66632143434,
    37621.70310773456, 39287.35820567516, 41026.758155021096, 42843.167919278625};
// log(1 + z) on |z| <= 2^(1/32) - 1 by its series up to z^6 (the next term is below 4e-13);
// 1 / (K 2^88) for kPow2's scale and that of the sums; L.
__constant__ double kLog[6] = {-1.0 / 6, 1.0 / 5, -1.0 / 4, 1.0 / 3, 2.541055997063135e-18, 0.04332169878499658};
// Sums that round to an integer: 1.5 2^52 and 2^52.
__constant__ double kRound[2] = {6755399441055744.0, 4503599627370496.0};

// exp((v - max) / T) as an integer multiple of 2^-44, rounded; 2^44 for v = max
// (finite). With y = (v - max) 16 log2(e) / T = n + r, |r| <= 1/2: 2^(y / 16) =
// 2^(n div 16) 2^((n mod 16) / 16) e^(r L). Below `least`, where the weight is under
// 2^-60, the result is 0 whatever the arithmetic gives.
struct Weight {
  const double *tab;   // kPow2 in shared memory
  double c, top;       // 16 log2(e) / T; max
  float max, least;
  __device__ __forceinline__ void set(float m, float temp) {
    max = m;
    top = (double)m;
    c = 16.0 * 1.44269504088896340736 / (double)temp;
    least = __fsub_rn(m, __fmul_rn(41.6f, temp));   // 60 ln 2 = 41.59; rounds to a float no entry lies between
  }
  // For v >= least (else any number).
  __device__ __forceinline__ u64 raw(float v) const {
    const double d = __dadd_rn((double)v, -top);
    const double t = fma(d, c, kRound[0]);
    const double r = fma(d, c, __dadd_rn(kRound[0], -t));
    const int n = __double2loint(t);
    double p = __dadd_rn(r, kExp[0]);
    p = fma(p, r, kExp[1]);
    p = fma(p, r, kExp[2]);
    p = fma(p, r, kExp[3]);
    p = fma(p, r, kExp[4]);
    const double w = __dmul_rn(tab[n & 15], p);
    // times 2^(n div 16), then to an integer: the mantissa after adding 2^52
    const double s = __hiloint2double(__double2hiint(w) + ((n & ~15) << 16), __double2loint(w));
    return (u64)__double_as_longlong(__dadd_rn(s, kRound[1])) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ u64 operator()(float v) const { return v >= least ? raw(v) : 0; }
  // log(sum 2^-44) for a sum of at least 2^44: k L + log(1 + z) with k the nearest
  // integer to 16 log2 of it (or one that is as good: an approximation finds it).
  __device__ __forceinline__ double log_sum(u64 sum) const {
    const double x = (double)sum;
    const int n = -__float2int_rn(16.0f * __log2f((float)x * 0x1p-44f));
    const double w = tab[n & 15];
    const double z = fma(__dmul_rn(x, __hiloint2double(__double2hiint(w) + ((n & ~15) << 16), __double2loint(w))),
                         kLog[4], -1.0);
    double p = fma(kLog[0], z, kLog[1]);
    p = fma(p, z, kLog[2]);
    p = fma(p, z, kLog[3]);
    p = fma(p, z, -0.5);
    p = fma(p, z, 1.0);
    return fma(p, z, __dmul_rn((double)-n, kLog[5]));
  }
  // (v - max) / T
  __device__ __forceinline__ double exponent(float v) const {
    return __dmul_rn(__dmul_rn(__dadd_rn((double)v, -top), c), 0.693147180559945309417 / 16);
  }
};

// A row's shared memory, per group (per CTA of a cluster). A warp's row uses its
// list or its bins and candidates, never both.
template <int MODE>
struct Listed {
  static constexpr int CAP = MODE == WARP ? 256 : 2048;   // entries of the list
  float list[CAP];          // this CTA's: values and indices, in index order
  int index[CAP];
};
template <int MODE>
struct Binned {
  static constexpr int NB = MODE == WARP ? 256 : 1024;    // bins
  static constexpr int RANK = MODE == WARP ? 64 : 512;    // candidates ranked against each other
  u64 all_w[RANK];
  float all[RANK];
  float cand[RANK];         // this CTA's candidates, read by the cluster
  unsigned bins[NB];        // counts, or weights in hint units
};
template <int MODE>
struct Both : Listed<MODE>, Binned<MODE> {};
template <>
struct Both<WARP> {
  union {
    struct {
      float list[Listed<WARP>::CAP];
      int index[Listed<WARP>::CAP];
    };
    struct {
      u64 all_w[Binned<WARP>::RANK];
      float all[Binned<WARP>::RANK], cand[Binned<WARP>::RANK];
      unsigned bins[Binned<WARP>::NB];
    };
  };
};
template <int MODE>
struct alignas(16) Shared : Both<MODE> {
  static constexpr int NB = Binned<MODE>::NB, CAP = Listed<MODE>::CAP, RANK = Binned<MODE>::RANK;
  static constexpr int NW = MODE == WARP ? 1 : 32;
  u64 part_w[2][NW], part_w2[2][NW];   // a warp's part of a reduction or scan; alternating
  unsigned part_n[2][NW], part_lo[2][NW], part_hi[2][NW];
  u64 cta_w[2], cta_w2[2];             // this CTA's part, read by the cluster; alternating
  unsigned cta_n[2], cta_lo[2], cta_hi[2];
  unsigned n_cand;
  int bin;
  unsigned bin_before, bin_inside;
  float cut;
  unsigned cut_take, cut_ties;
};

// Sums and extremes over a row's entries.
struct Sums {
  u64 w, w2;     // weights
  unsigned n;    // entries
  float lo, hi;  // smallest, largest value
};
__device__ __forceinline__ Sums no_sums() { return Sums{0, 0, 0, INFINITY, -INFINITY}; }

// (three 22-bit parts, whose sums over 32 lanes fit 27 bits; v < 2^66)
__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
  const unsigned a = __reduce_add_sync(PK_FULL_MASK, (unsigned)v & 0x3fffffu);
  const unsigned b = __reduce_add_sync(PK_FULL_MASK, (unsigned)(v >> 22) & 0x3fffffu);
  const unsigned c = __reduce_add_sync(PK_FULL_MASK, (unsigned)(v >> 44));
  return a + ((u64)b << 22) + ((u64)c << 44);
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

// Where entries come from: the row in shared memory, or the list (with indices).
struct Src {
  const float *x;
  const int *at;
  int n, base;   // this CTA's number of entries
  int total;     // a list: the row's
  __device__ __forceinline__ float value(int i) const { return x[i]; }
  __device__ __forceinline__ int index(int i) const { return at ? at[i] : base + i; }
};

template <typename T, int MODE>
struct Row {
  typedef Shared<MODE> S;
  const Args &a;
  S &s;
  float *room, *x;      // this group's (CTA's) entries, in room from where their alignment asks
  int base, n;          // the first one's index in the row, their number
  unsigned rank, size;  // of the cluster
  int tid;              // thread of the group (CTA)
  int flip, cflip;
  Weight weight;
  float scale;          // bins: (max - l) scale
  int hint;             // bins of weights: units of 2^(hint - 44)

  // ── the group ──
  __device__ __forceinline__ int nt() const { return MODE == WARP ? 32 : (int)blockDim.x; }
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

  // Totals over the row's threads, to every thread. What is asked for: W weights
  // (1 or 2 sums), N entries, K extreme values (reduced as keys).
  template <int W, bool N, bool K>
  __device__ __forceinline__ Sums total(Sums v) {
    const int lane = threadIdx.x & 31;
    unsigned lo = K ? key_of(v.lo) : 0, hi = K ? key_of(v.hi) : 0;
    reduce<W, N, K>(v, lo, hi);
    if (MODE != WARP) {
      const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
      if (lane == 0) {
        if (W > 0) s.part_w[flip][warp] = v.w;
        if (W > 1) s.part_w2[flip][warp] = v.w2;
        if (N) s.part_n[flip][warp] = v.n;
        if (K) {
          s.part_lo[flip][warp] = lo;
          s.part_hi[flip][warp] = hi;
        }
      }
      __syncthreads();   // (two calls later the buffer is free: every thread has passed the next call's barrier)
      const bool in = lane < nw;
      if (W > 0) v.w = in ? s.part_w[flip][lane] : 0;
      if (W > 1) v.w2 = in ? s.part_w2[flip][lane] : 0;
      if (N) v.n = in ? s.part_n[flip][lane] : 0;
      if (K) {
        lo = in ? s.part_lo[flip][lane] : 0xffffffffu;
        hi = in ? s.part_hi[flip][lane] : 0;
      }
      reduce<W, N, K>(v, lo, hi);
      flip ^= 1;
    }
    if (MODE == CLUSTER) {
      if (threadIdx.x == 0) {
        if (W > 0) s.cta_w[cflip] = v.w;
        if (W > 1) s.cta_w2[cflip] = v.w2;
        if (N) s.cta_n[cflip] = v.n;
        if (K) {
          s.cta_lo[cflip] = lo;
          s.cta_hi[cflip] = hi;
        }
      }
      gsync();
      const bool in = lane < (int)size;
      if (W > 0) v.w = in ? *peer(&s.cta_w[cflip], lane) : 0;
      if (W > 1) v.w2 = in ? *peer(&s.cta_w2[cflip], lane) : 0;
      if (N) v.n = in ? *peer(&s.cta_n[cflip], lane) : 0;
      if (K) {
        lo = in ? *peer(&s.cta_lo[cflip], lane) : 0xffffffffu;
        hi = in ? *peer(&s.cta_hi[cflip], lane) : 0;
      }
      reduce<W, N, K>(v, lo, hi);
      cflip ^= 1;
    }
    if (K) {
      v.lo = value_of(lo);
      v.hi = value_of(hi);
    }
    return v;
  }
  template <int W, bool N, bool K>
  __device__ __forceinline__ static void reduce(Sums &v, unsigned &lo, unsigned &hi) {
    if (W > 0) v.w = warp_sum_u64(v.w);
    if (W > 1) v.w2 = warp_sum_u64(v.w2);
    if (N) v.n = __reduce_add_sync(PK_FULL_MASK, v.n);
    if (K) {
      lo = __reduce_min_sync(PK_FULL_MASK, lo);
      hi = __reduce_max_sync(PK_FULL_MASK, hi);
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
  // Linear in max - l, rounded, the last one open-ended.
  __device__ __forceinline__ int bin_of(float v) const {
    const float f = __fmul_rn(__fsub_rn(weight.max, v), scale);
    return __float_as_int(__fadd_rn(fminf(f, (float)(S::NB - 1)), 8388608.0f)) - 0x4B000000;
  }
  // A value that every entry of the bins up to `bin` is at least (a few of the next
  // bin's may be too): the bin's lower edge, a tenth of a bin further down. The
  // margin covers the roundings of bin_of (2 x 2^-24 of at most 1023 bins); the
  // edge's own rounding to a float passes no entry, as those are floats as well.
  __device__ __forceinline__ float edge_of(int bin) const {
    return bin >= S::NB - 1 ? -INFINITY : __fsub_rn(weight.max, __fdiv_rn((float)bin + 0.6f, scale));
  }
  // Bins from the maximum down to `lowest`, at least.
  __device__ __forceinline__ void set_scale(float lowest) {
    scale = (float)(S::NB - 2) / fmaxf(__fsub_rn(weight.max, lowest), 1e-30f);
  }
  __device__ __forceinline__ void clear_bins() {
    lsync();
    for (int b = tid; b < S::NB; b += nt()) s.bins[b] = 0;
    lsync();
  }
  // The first bin at which the bins' running sum reaches goal, `before` what the
  // bins before it hold, `inside` what it holds itself, `all` what all hold. It ends
  // with a barrier of this CTA alone: a peer may still read this CTA's bins, so they
  // are not filled again before a barrier of the cluster.
  __device__ int find_bin(u64 goal, unsigned &before, unsigned &inside, u64 &all, bool synced = false) {
    if (!synced) gsync();   // every CTA's bins are filled
    constexpr int MAXPER = MODE == WARP ? S::NB / 32 : 8;   // at least 128 threads in a CTA
    const int per = (S::NB + nt() - 1) / nt(), b0 = tid * per;
    unsigned held[MAXPER];
    u64 mine = 0;
#pragma unroll
    for (int j = 0; j < MAXPER; j++) {
      held[j] = 0;
      if (j < per && b0 + j < S::NB) {
        u64 c = 0;
        for (unsigned r = 0; r < (MODE == CLUSTER ? size : 1); r++) c += *peer(&s.bins[b0 + j], r);
        held[j] = (unsigned)c;   // the row's total fits 32 bits
      }
      mine += held[j];
    }
    const u64 inc = warp_scan_u64(mine);
    u64 run = inc - mine;
    all = __shfl_sync(PK_FULL_MASK, inc, 31);
    if (tid == 0) s.bin = S::NB - 1;
    if (MODE != WARP) {
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
      if (lane == 0) s.part_w[flip][warp] = all;
      __syncthreads();
      const u64 w = warp_scan_u64(lane < nw ? s.part_w[flip][lane] : 0);
      flip ^= 1;
      if (warp > 0) run += __shfl_sync(PK_FULL_MASK, w, warp - 1);
      all = __shfl_sync(PK_FULL_MASK, w, 31);
    } else {
      __syncwarp();
    }
    if (goal > all) goal = all;   // hints: roundings may have lost the last
    if (run < goal && goal <= run + mine) {
      int b = -1;
      u64 at = run;
#pragma unroll
      for (int j = 0; j < MAXPER; j++)
        if (b < 0) {
          if (at + held[j] >= goal) {
            b = b0 + j;
            s.bin_before = (unsigned)at;
            s.bin_inside = held[j];
          }
          at += held[j];
        }
      s.bin = b;
    }
    lsync();
    before = s.bin_before;
    inside = s.bin_inside;
    return s.bin;
  }

  // The border of a prefix of the order among a source's entries > above: the first
  // of them, from the largest, at which the count (BY_WEIGHT: the weight) reaches
  // `target` (1 .. what there is), given the bin that the bins of these entries
  // say. Leaves s.cut, the border's value, s.cut_take, how many of its equals
  // belong to the prefix, s.cut_ties, how many there are. only: the source holds
  // the bins up to that one; false where they do not reach the target (a rounding
  // of the hint).
  template <bool BY_WEIGHT>
  __device__ bool border(const Src &src, float above, u64 target, int bin, unsigned bin_before, unsigned bin_inside,
                         bool only = false) {
    float hi = INFINITY, lo = above;          // the border is in (lo, hi], or [lo, hi] once `found`
    u64 before = bin_before;                  // count or weight of the values > hi
    unsigned inside = bin_inside;             // entries there
    bool found = !BY_WEIGHT;                  // counts need no confirmation, only the bin's values
    for (int tries = 0; tries < (BY_WEIGHT ? 3 : 1); tries++) {
      Sums up = no_sums(), in = no_sums();
      constexpr int G = MODE == WARP ? 4 : 1;   // a warp: independent entries side by side
      for (int i = tid; i < src.n; i += G * nt()) {
        float v[G];
        u64 w[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
          v[g] = i + g * nt() < src.n ? src.value(i + g * nt()) : -INFINITY;
          w[g] = BY_WEIGHT ? weight(v[g]) : 0;
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
          const int b = bin_of(v[g]);
          if (!(v[g] > above) || b > bin) continue;
          if (b < bin) {
            up.w += w[g];
          } else {
            in.n++;
            in.lo = fminf(in.lo, v[g]);
            in.hi = fmaxf(in.hi, v[g]);
            in.w += w[g];
          }
        }
      }
      in.w2 = up.w;
      in = total<BY_WEIGHT ? 2 : 0, BY_WEIGHT, true>(in);
      up.w = in.w2;
      if (BY_WEIGHT) {
        if (only && up.w + in.w < target) return false;
        found = up.w < target && target <= up.w + in.w;
        before = up.w;
        inside = in.n;
      }
      if (found) {
        hi = in.hi;
        lo = in.lo;
        break;
      }
      bin = target <= up.w ? max(bin - 1, 0) : min(bin + 1, S::NB - 1);   // a rounding of the hint: one bin off
    }
    if (!found) {   // all of them
      Sums in = no_sums();
      for (int i = tid; i < src.n; i += nt()) {
        const float v = src.value(i);
        if (!(v > above)) continue;
        in.n++;
        in.lo = fminf(in.lo, v);
        in.hi = fmaxf(in.hi, v);
      }
      in = total<0, true, true>(in);
      inside = in.n;
      lo = in.lo;
      hi = in.hi;
      before = 0;
    }
    // too many to rank: halve the range of values (as keys) until few are left, or one value
    while (inside > (unsigned)S::RANK && lo < hi) {
      const unsigned kl = key_of(lo);
      const float mid = value_of(kl + (key_of(hi) - kl) / 2);   // lo <= mid < hi
      Sums up = no_sums();   // values in (mid, hi]
      for (int i = tid; i < src.n; i += nt()) {
        const float v = src.value(i);
        if (!(v > mid) || v > hi) continue;
        up.n++;
        if (BY_WEIGHT) up.w += weight(v);
      }
      up = total<BY_WEIGHT ? 1 : 0, true, false>(up);
      const u64 more = BY_WEIGHT ? up.w : up.n;
      if (before + more >= target) {
        lo = value_of(key_of(mid) + 1);
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
        const u64 each = BY_WEIGHT ? weight(hi) : 1;
        s.cut = hi;
        s.cut_ties = inside;
        s.cut_take = (unsigned)(BY_WEIGHT ? (target - before + each - 1) / each : target - before);
      }
      lsync();
      return true;
    }
    // list the candidates, in every CTA the same ones (in any order)
    if (tid == 0) s.n_cand = 0;
    lsync();
    for (int i = tid; i < src.n; i += nt()) {
      const float v = src.value(i);
      if (v >= lo && v <= hi) s.cand[atomicAdd(&s.n_cand, 1u)] = v;
    }
    gsync();
    unsigned n_all = 0;
    for (unsigned r = 0; r < (MODE == CLUSTER ? size : 1); r++) {
      const unsigned m = *peer(&s.n_cand, r);
      const float *c = peer(s.cand, r);
      for (unsigned i = tid; i < m; i += nt()) {
        s.all[n_all + i] = c[i];
        if (BY_WEIGHT) s.all_w[n_all + i] = weight(c[i]);
      }
      n_all += m;
    }
    lsync();
    for (unsigned i = tid; i < n_all; i += nt()) {
      const float v = s.all[i];
      u64 more = 0;         // count or weight of the larger ones
      unsigned ties = 0;
#pragma unroll 4
      for (unsigned j = 0; j < n_all; j++) {
        const float o = s.all[j];
        ties += o == v;
        if (o > v) more += BY_WEIGHT ? s.all_w[j] : 1;
      }
      const u64 each = BY_WEIGHT ? s.all_w[i] : 1, start = before + more;
      if (start < target && target <= start + each * ties) {   // equals write the same
        s.cut = v;
        s.cut_ties = ties;
        s.cut_take = ties == 1 ? 1 : (unsigned)(BY_WEIGHT ? (target - start + each - 1) / each : target - start);
      }
    }
    gsync();   // (cluster: the candidates are read)
    return true;
  }

  // The row's entries >= edge (finite) into the list, in index order, where every
  // CTA's fit.
  __device__ bool make_list(const Src &src, float edge, Src &out) {
    const int lane = threadIdx.x & 31;
    edge = fmaxf(edge, -3.402823466e38f);
    if constexpr (MODE == WARP) {
      // a contiguous run per lane, of odd length (no bank conflicts), at most 63: which
      // of its entries belong, as bits; reads past the run's end are masked
      const int per = ((src.n + 31) / 32) | 1, i0 = min(lane * per, src.n), len = min(per, src.n - i0);
      u64 in = 0;
      for (int j = 0; j < per; j += 8) {
        unsigned m = 0;
#pragma unroll
        for (int g = 0; g < 8; g++) m |= src.value(lane * per + j + g) >= edge ? 1u << g : 0;
        in |= (u64)m << j;
      }
      in &= (1ull << len) - 1;
      const unsigned c = __popcll(in);
      unsigned end = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(PK_FULL_MASK, end, o);
        if (lane >= o) end += up;
      }
      out.n = (int)__shfl_sync(PK_FULL_MASK, end, 31);
      if (out.n > S::CAP) return false;
      for (unsigned at = end - c; in; in &= in - 1, at++) {
        const int i = i0 + __ffsll((long long)in) - 1;
        s.list[at] = src.value(i);
        s.index[at] = src.index(i);
      }
      __syncwarp();
    } else {
      // a contiguous segment per warp; eight groups of 32 entries at a time, so that
      // their reads and votes overlap
      constexpr int G = 8;
      const int warp = threadIdx.x >> 5, nw = (int)(blockDim.x >> 5);
      const int per = ((src.n + nw - 1) / nw + 31) & ~31, i0 = min(warp * per, src.n), i1 = min(i0 + per, src.n);
      unsigned c = 0;
#pragma unroll 8
      for (int i = i0 + lane; i < i1; i += 32) c += src.value(i) >= edge;
      c = __reduce_add_sync(PK_FULL_MASK, c);
      u64 all, most;
      const u64 b = scan<true>(lane == 0 ? c : 0, all, most);
      unsigned at = (unsigned)__shfl_sync(PK_FULL_MASK, b, 0);
      if (most > (u64)S::CAP) return false;
      if (threadIdx.x == blockDim.x - 32) s.n_cand = at + c;
      if (c)
        for (int i = i0 + lane; i - lane < i1; i += 32 * G) {
          float v[G];
          unsigned who[G];
#pragma unroll
          for (int g = 0; g < G; g++) v[g] = i + 32 * g < i1 ? src.value(i + 32 * g) : -INFINITY;
#pragma unroll
          for (int g = 0; g < G; g++) who[g] = __ballot_sync(PK_FULL_MASK, v[g] >= edge);
#pragma unroll
          for (int g = 0; g < G; g++) {
            if (!who[g]) continue;
            if (v[g] >= edge) {
              const unsigned o = at + __popc(who[g] & ((1u << lane) - 1));
              s.list[o] = v[g];
              s.index[o] = src.index(i + 32 * g);
            }
            at += __popc(who[g]);
          }
        }
      __syncthreads();
      out.n = (int)s.n_cand;
      out.total = (int)all;
      __syncthreads();
    }
    out.x = s.list;
    out.at = s.index;
    out.base = 0;
    return true;
  }

  __device__ bool small(int n, long long row, int k, float p, u64 all_w, float mp, float uu);

  // log(w / S) of a value: the exponent itself less log S, S in units of the
  // largest weight (which is one of its parts), in fp64 and rounded once. The weights'
  // own rounding leaves 2^-45 per entry in S: 10^-10 of it in a row of 10^4 whose
  // weights nearly all lie below that.
  // (The library's log: 12000 x 1025 top-k 37.7 us, 36.6 this way.)
  __device__ __forceinline__ float log_prob(float v, u64 sum) const {
    return (float)((v == weight.max ? 0.0 : weight.exponent(v)) - weight.log_sum(sum));
  }

  // Kept are values > v and the first `take` of the `ties` equal to it.
  struct Cut {
    float v;
    unsigned take, ties;
  };
  __device__ __forceinline__ Cut read_cut() const { return Cut{s.cut, s.cut_take, s.cut_ties}; }

  // The sum of the weights of the values > cut; BINS: their bins too, in units of
  // which the row's total fits 32 bits.
  template <bool BINS>
  __device__ __forceinline__ u64 weigh(const Src &src, float cut) {
    if (BINS) clear_bins();
    Sums t = no_sums();
    constexpr int G = 4;   // independent chains of fp64 operations; 6 fetches more code than it hides waits
    // at least the limit below which weights are 0, and past the cut
    const float low = weight.least > cut ? weight.least : cut;
    const bool past = low == cut;
    auto group = [&](int i, bool whole) {
      float v[G];
      u64 w[G];
#pragma unroll
      for (int g = 0; g < G; g++) {
        v[g] = whole || i + g * nt() < src.n ? src.value(i + g * nt()) : -INFINITY;
        w[g] = weight.raw(v[g]);
      }
#pragma unroll
      for (int g = 0; g < G; g++)
        if (past ? v[g] > low : v[g] >= low) {
          t.w += w[g];
          if (BINS) atomicAdd(&s.bins[bin_of(v[g])], (unsigned)((w[g] + (1ull << hint >> 1)) >> hint));
        }
    };
    int i = tid;
    for (; i + (G - 1) * nt() < src.n; i += G * nt()) group(i, true);
    if (i < src.n) group(i, false);
    return total<1, false, false>(t).w;
  }
  // The least integer that is at least p times the sum (and at least 1).
  __device__ __forceinline__ static u64 share(float p, u64 sum) {
    const u64 t = p > 0.0f ? (u64)ceil((double)p * (double)sum) : 1;
    return t < 1 ? 1 : t < sum ? t : sum;
  }
  __device__ __forceinline__ int find_weight(u64 target, u64 &binned) {   // binned: what the bins hold
    unsigned before, inside;
    const u64 goal = target >> hint;
    const int bin = find_bin(goal ? goal : 1, before, inside, binned, MODE != WARP);   // weigh's total was a barrier
    binned <<= hint;
    return bin;
  }
  __device__ void draw(const Src &src, long long row, Cut cut, float mp, float uu);
  __device__ void run(long long row);
};

template <typename T, int MODE>
__device__ void Row<T, MODE>::draw(const Src &src, long long row, Cut cut, float mp, float uu) {
  const int lane = threadIdx.x & 31;
  // min-p: a weight at least min_p of the largest, which always stays
  u64 least = 0;
  if (mp > 0.0f) least = (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * 0x1p44);
  // a contiguous run of entries per thread, of odd length: no bank conflicts between the threads
  const int per = ((src.n + nt() - 1) / nt()) | 1;
  const int i0 = min(tid * per, src.n), i1 = min(i0 + per, src.n);
  const bool part = cut.take < cut.ties;
  const float low = cut.ties ? cut.v : -3.402823466e38f;   // kept are values >= low
  unsigned tie0 = 0;   // equals of the cut before this thread's run
  if (part) {
    unsigned c = 0;
    for (int i = i0; i < i1; i++) c += src.value(i) == low;
    u64 all, most;
    tie0 = (unsigned)scan<false>(c, all, most);
  }
  const float low0 = fmaxf(low, weight.least);   // below it weights are 0
  u64 mine = 0;
  unsigned seen = tie0;
  constexpr int G = 4;
  auto group = [&](int i, bool whole) {
    float v[G];
    u64 w[G];
#pragma unroll
    for (int j = 0; j < G; j++) {
      v[j] = whole || i + j < i1 ? src.value(i + j) : -INFINITY;
      w[j] = weight.raw(v[j]);
    }
    if (part || least) {
#pragma unroll
      for (int j = 0; j < G; j++) {
        bool keep = v[j] >= low0 && w[j] >= least;
        if (part && v[j] == low) keep = keep && seen++ < cut.take;
        if (keep) mine += w[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < G; j++)
        if (v[j] >= low0) mine += w[j];
    }
  };
  int i = i0;
  for (; i + G <= i1; i += G) group(i, true);
  if (i < i1) group(i, false);
  u64 sum, most;
  const u64 before = scan<false>(mine, sum, most);
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
    bool keep = v >= low;
    if (part) {
      const unsigned same = __ballot_sync(PK_FULL_MASK, v == low);
      if (v == low) keep = seen + __popc(same & ((1u << lane) - 1)) < cut.take;
      seen += __popc(same);
    }
    u64 w = weight(v);
    w = keep && w >= least ? w : 0;
    const u64 inc = warp_scan_u64(w);
    const unsigned past = __ballot_sync(PK_FULL_MASK, run + inc > target);
    if (past) {
      if (lane == __ffs(past) - 1) {
        a.tokens[row] = src.index(i);
        if (a.logprobs) a.logprobs[row] = log_prob(v, sum);
      }
      break;
    }
    run += __shfl_sync(PK_FULL_MASK, inc, 31);
  }
}

// Filters and draw for at most 256 listed entries, by one warp in its registers:
// entry 32 j + lane is the lane's j-th. n: the list's length (all of the row's lists
// in rank order, for a cluster's first warp). k > 0: the k largest of them; p < 1:
// of these those whose weight reaches p times theirs, or times all_w where k is 0.
// A border is found by halving the range of keys, counts and weights (in two
// 22-bit halves, so that 256 of them fit a 32-bit reduction) summed exactly in
// each step, until one entry is left in the range, or one key. False: the entries
// weigh less than the share asked for, nothing is drawn.
template <typename T, int MODE>
__device__ bool Row<T, MODE>::small(int n, long long row, int k, float p, u64 all_w, float mp,
                                    float uu) {
  constexpr int J = 8;
  const int lane = threadIdx.x & 31;
  unsigned key[J], wl[J], wh[J];   // key 0: dropped
  unsigned lowest = 0xffffffffu;
  // the list (a cluster: rank and place in its list) that entry i is in
  auto place = [&](int i, unsigned &r) {
    r = 0;
    if (MODE == CLUSTER)
      for (; r < size - 1; r++) {
        const int m = (int)*peer(&s.n_cand, r);
        if (i < m) break;
        i -= m;
      }
    return i;
  };
#pragma unroll
  for (int j = 0; j < J; j++) {
    const int i = 32 * j + lane;
    float v = -INFINITY;
    key[j] = wl[j] = wh[j] = 0;
    if (32 * j >= n) continue;
    if (i < n) {
      unsigned r;
      const int at = place(i, r);
      v = *peer(&s.list[at], r);
    }
    const u64 w = i < n ? weight(v) : 0;
    key[j] = i < n ? key_of(v) : 0;
    wl[j] = (unsigned)w & 0x3fffffu;
    wh[j] = (unsigned)(w >> 22);
    lowest = min(lowest, key[j] - 1);
  }
  lowest = __reduce_min_sync(PK_FULL_MASK, lowest);   // below every entry's key
  const unsigned highest = key_of(weight.max);
  auto count = [&](unsigned above) {
    unsigned c = 0;
#pragma unroll
    for (int j = 0; j < J; j++)
      if (32 * j < n) c += key[j] > above;
    return (int)__reduce_add_sync(PK_FULL_MASK, c);
  };
  auto mass = [&](unsigned above) {
    unsigned l = 0, h = 0;
#pragma unroll
    for (int j = 0; j < J; j++)
      if (32 * j < n && key[j] > above) {
        l += wl[j];
        h += wh[j];
      }
    return ((u64)__reduce_add_sync(PK_FULL_MASK, h) << 22) + __reduce_add_sync(PK_FULL_MASK, l);
  };
  // keeps keys > above, and of those equal to it the first `take`
  auto drop = [&](unsigned above, unsigned take) {
    unsigned seen = 0;
#pragma unroll
    for (int j = 0; j < J; j++) {
      bool keep = key[j] > above;
      if (take) {
        const unsigned same = __ballot_sync(PK_FULL_MASK, key[j] == above);
        if (key[j] == above) keep = seen + __popc(same & ((1u << lane) - 1)) < take;
        seen += __popc(same);
      }
      if (!keep) key[j] = wl[j] = wh[j] = 0;
    }
  };
  if (k > 0 && k < n) {
    unsigned lo = lowest, hi = highest;   // count(lo) > k > count(hi)
    for (;;) {
      if (hi - lo == 1) {   // equals at the border
        drop(hi, (unsigned)(k - count(hi)));
        break;
      }
      const unsigned mid = lo + (hi - lo) / 2;
      const int c = count(mid);
      if (c == k) {
        drop(mid, 0);
        lo = mid;
        break;
      }
      if (c > k) lo = mid;
      else hi = mid;
    }
    lowest = lo;
  }
  if (p < 1.0f) {
    const u64 have = mass(0);
    const u64 target = share(p, k > 0 ? have : all_w);
    if (have < target) return false;
    unsigned lo = lowest, hi = highest;   // mass(lo) >= target > mass(hi)
    int clo = count(lo), chi = 0;
    for (;;) {
      if (clo - chi == 1) {   // the border's entry alone
        drop(lo, 0);
        break;
      }
      if (hi - lo == 1) {   // equals at the border
        const u64 each = weight(value_of(hi));
        drop(hi, (unsigned)((target - mass(hi) + each - 1) / each));
        break;
      }
      const unsigned mid = lo + (hi - lo) / 2;
      if (mass(mid) >= target) {
        lo = mid;
        clo = count(mid);
      } else {
        hi = mid;
        chi = count(mid);
      }
    }
  }
  if (mp > 0.0f) {
    const u64 least = (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * 0x1p44);
#pragma unroll
    for (int j = 0; j < J; j++)
      if (((u64)wh[j] << 22) + wl[j] < least) key[j] = wl[j] = wh[j] = 0;
  }
  const u64 sum = mass(0);
  u64 target = uu > 0.0f ? (u64)((double)uu * (double)sum) : 0;
  target = target < sum ? target : sum - 1;
  u64 run = 0;
#pragma unroll
  for (int j = 0; j < J; j++) {
    const u64 part = ((u64)__reduce_add_sync(PK_FULL_MASK, wh[j]) << 22) + __reduce_add_sync(PK_FULL_MASK, wl[j]);
    if (target < run + part) {
      const u64 inc = warp_scan_u64(((u64)wh[j] << 22) + wl[j]);
      const unsigned past = __ballot_sync(PK_FULL_MASK, run + inc > target);
      if (lane == __ffs(past) - 1) {
        unsigned r;
        const int at = place(32 * j + lane, r);
        a.tokens[row] = *peer(&s.index[at], r);
        if (a.logprobs) a.logprobs[row] = log_prob(value_of(key[j]), sum);
      }
      break;
    }
    run += part;
  }
  return true;
}

template <typename T, int MODE>
__device__ void Row<T, MODE>::run(long long row) {
  const T *in = static_cast<const T *>(a.logits) + row * a.ld + base;
  const float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  const int k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float p = a.top_p ? __ldg(a.top_p + row) : 1.0f;
  const float mp = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  const float uu = __ldg(a.u + row);
  // the row, once; its largest value. Its smallest finite one for the bins; a warp
  // that looks for the k largest takes instead the smallest of its lanes' second
  // largest: 190 +- 45 entries are as large whatever the distribution, and mostly
  // only they matter (for the 48 largest, the smallest of the lanes' largest:
  // 130 +- 41).
  Sums v = no_sums();
  float second = -INFINITY;
  auto take = [&](float e) {
    if (MODE == WARP) second = fmaxf(second, fminf(v.hi, e));
    else v.lo = fminf(v.lo, e == -INFINITY ? INFINITY : e);
    v.hi = fmaxf(v.hi, e);
  };
  // 16 bytes at a time from the first 16-byte boundary on, which shared memory has at
  // the same place, what lies before it and behind the last whole piece singly: 256 x
  // 32000 fp32 top-k 37 us by single entries, 32 by pieces, 12000 x 100 42 and 35 (12000
  // x 1025, whose rows are aligned to their type alone, 36 and 36.6)
  constexpr int E = 16 / (int)sizeof(T);
  const int mis = (int)((uintptr_t)in / sizeof(T)) & (E - 1);
  x = room + mis;
  const int lo = min((E - mis) & (E - 1), n), pieces = (n - lo) / E, hi = lo + pieces * E;
  const int edge = tid < lo ? tid : tid + (hi - lo);   // fewer than 2 E: one per thread
  T at_edge = from_f32<T>(0.0f);
  if (edge < n) at_edge = in[edge];
#pragma unroll 4
  for (int c = tid; c < pieces; c += nt()) {
    const uint4 q = *reinterpret_cast<const uint4 *>(in + lo + c * E);
    const T *e = reinterpret_cast<const T *>(&q);
    float f[E];
#pragma unroll
    for (int j = 0; j < E; j++) {
      f[j] = clean(to_f32(e[j]));
      take(f[j]);
    }
#pragma unroll
    for (int j = 0; j < E; j += 4) *reinterpret_cast<float4 *>(x + lo + c * E + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
  }
  if (edge < n) {
    const float e = clean(to_f32(at_edge));
    x[edge] = e;
    take(e);
  }
  if (MODE == WARP) v.lo = k <= 48 ? v.hi : second;
  v = total<0, false, true>(v);
  if (v.hi == -INFINITY) {   // nothing to take
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  lsync();
  const Src all{x, nullptr, n, base, 0};
  if (!(temp > 0.0f)) {   // greedy: the first largest
    unsigned first = 0xffffffffu;
    for (int i = tid; i < n; i += nt())
      if (x[i] == v.hi) first = min(first, (unsigned)(base + i));
    Sums f = no_sums();
    f.lo = first == 0xffffffffu ? INFINITY : (float)first;   // indices below 2^18 are exact
    f = total<0, false, true>(f);
    if (rank == 0 && tid == 0) {
      a.tokens[row] = (int)f.lo;
      if (a.logprobs) a.logprobs[row] = 0.0f;
    }
    return;
  }
  if (v.hi == INFINITY) {   // infinite ones share everything: they are zeros, the rest is masked
    for (int i = tid; i < n; i += nt()) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
    v.hi = 0.0f;
    v.lo = MODE == WARP ? -INFINITY : 0.0f;
    lsync();
  }
  weight.set(v.hi, temp);
  Cut cut = {-INFINITY, 0, 0};
  Src src = all, few;   // what is left to look at; a list
  const bool by_p = p < 1.0f;
  // a warp's few bins reach down 28 T, where a weight is e^-28 of the largest
  const float low = __fsub_rn(v.hi, __fmul_rn(28.0f, temp));
  u64 all_w = 0, target = 0;
  int bin = 0;
  if (MODE == WARP && (k > 0 || by_p)) {
    // mostly a list of at most 256 holds all that the filters leave: with top-k, of
    // what is as large as v.lo; without, of the bins up to the one in which p is reached
    if (k <= 0) {
      set_scale(low);
      all_w = weigh<true>(all, -INFINITY);
      target = share(p, all_w);
      u64 binned;
      bin = find_weight(target, binned);
    }
    if (make_list(all, k > 0 ? v.lo : edge_of(bin), few) && (k <= few.n || v.lo == -INFINITY) &&
        small(few.n, row, k, p, all_w, mp, uu))
      return;
    if (k > 0) {
      v.lo = INFINITY;
      for (int i = tid; i < n; i += nt()) v.lo = fminf(v.lo, x[i] == -INFINITY ? INFINITY : x[i]);
      v = total<0, false, true>(v);
    }
  }
  if (k > 0) {
    set_scale(fmaxf(v.lo, __fsub_rn(v.hi, 64.0f)));
    clear_bins();
#pragma unroll 8
    for (int i = tid; i < n; i += nt()) {
      const float e = x[i];
      if (e > -INFINITY) atomicAdd(&s.bins[bin_of(e)], 1u);
    }
    unsigned before, inside;
    u64 count;
    const int kbin = find_bin((u64)k, before, inside, count);
    if ((u64)k < count) {
      if (MODE != WARP && before + inside <= (unsigned)S::CAP && make_list(all, edge_of(kbin), few)) {
        if (few.total <= 256) {
          gsync();   // every CTA's list is there
          if (rank == 0 && threadIdx.x < 32) small(few.total, row, k, p, 0, mp, uu);
          return;
        }
        src = few;
      }
      border<false>(src, -INFINITY, (u64)k, kbin, before, inside);
      cut = read_cut();
    } else {
      gsync();   // (cluster: the bins are read; border's and make_list's barriers say so where there is a cut)
    }
  }
  if (by_p) {
    bool inside_ties = false;
    if (MODE != WARP || k > 0) {
      set_scale(MODE == WARP ? low : fmaxf(v.lo, __fsub_rn(v.hi, 64.0f)));
      const u64 w = weigh<true>(src, cut.v);
      const u64 each = cut.ties ? weight(cut.v) : 0;
      all_w = w + cut.take * each;
      target = share(p, all_w);
      inside_ties = target > w;   // of the top-k's border
      if (inside_ties) cut.take = (unsigned)((target - w + each - 1) / each);
      else {
        u64 binned;
        bin = find_weight(target, binned);
        // weights below half a unit are missing from the bins: where that is more than
        // 2^-8 of the sum and the border is among weights of a few units, again in finer
        // units, now that the sum is known (1 x 131072 bf16, top-p 0.98: 59 us, 163
        // without, the border's bin being far off; top-p 0.6, where it is not needed, 31
        // us, 41 if it were always done)
        const int coarse = hint, fine = 33 - __clzll((long long)w);   // w < 2^31 fine units
        if (MODE != WARP && fine < coarse && binned + (w >> 8) < w && weight(edge_of(bin)) < (4ull << coarse)) {
          hint = max(fine, 0);
          gsync();   // (cluster: the bins are read)
          weigh<true>(src, cut.v);
          bin = find_weight(target, binned);
          hint = coarse;
        }
      }
    }
    if (!inside_ties) {
      for (int tries = cut.ties ? 2 : 0;; tries++, bin = min(bin + 1, S::NB - 1)) {
        // of a list of the bins up to the border's; a list that proves short of the
        // target (a rounding of the hint) is made again with one bin more
        const bool listed = MODE != WARP && tries < 2 && make_list(all, edge_of(bin), few);
        if (listed && few.total <= 256) {
          if (weigh<false>(few, -INFINITY) < target) continue;   // (a barrier: every CTA's list is there)
          if (rank == 0 && threadIdx.x < 32) small(few.total, row, 0, p, all_w, mp, uu);
          return;
        }
        if (!cut.ties) src = listed ? few : all;
        if (border<true>(src, cut.v, target, bin, 0, 0, listed)) break;
      }
      cut = read_cut();
    }
  }
  draw(src, row, cut, mp, uu);
}

// A group's shared memory: entries from up to 7 places on; a warp reads up to 32 runs
// of odd length, and 8 more.
template <int MODE>
__host__ __device__ constexpr size_t group_bytes(int seg) {
  return sizeof(Shared<MODE>) + (((size_t)((MODE == WARP ? ((seg + 31) / 32 | 1) * 32 + 8 : seg) + 7) * 4 + 15) & ~(size_t)15);
}
constexpr int WARP_MAX = 2016;   // entries of a warp's row: runs of 63

template <typename T, int MODE>
__global__ void __launch_bounds__(MODE == WARP ? 256 : 1024, MODE == WARP ? 4 : 1) sample_kernel(Args a) {
  typedef Shared<MODE> S;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ double tab[16];
  if (threadIdx.x < 16) tab[threadIdx.x] = kPow2[threadIdx.x];
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  const size_t group = group_bytes<MODE>(a.seg);
  unsigned char *mem = smem + (MODE == WARP ? warp * group : 0);
  S &s = *reinterpret_cast<S *>(mem);
  Row<T, MODE> r{a, s};
  r.x = r.room = reinterpret_cast<float *>(mem + sizeof(S));
  r.hint = 44 - 31 + (32 - __clz(a.V));   // V < 2^(32 - clz) weights of 2^44: 31 bits
  r.weight.tab = tab;
  r.flip = r.cflip = 0;
  r.size = MODE == CLUSTER ? cg::this_cluster().num_blocks() : 1;
  r.rank = MODE == CLUSTER ? cg::this_cluster().block_rank() : 0;
  r.base = (int)r.rank * a.seg;
  r.n = a.V - r.base < a.seg ? a.V - r.base : a.seg;
  if (r.n < 0) r.n = 0;
  r.tid = MODE == WARP ? threadIdx.x & 31 : threadIdx.x;
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
  const size_t bytes = groups * group_bytes<MODE>(a.seg);
  smem_optin(sample_kernel<T, MODE>, 200 * 1024, flags);
  const long long rows = (a.n_rows + groups - 1) / groups;
  cudaLaunchConfig_t cfg = {};
  const long long most = 1 << 20;
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

// Group by row length and number of rows, as measured on a B200:
//  a warp per row for short rows where they are many: 3000 x 1025 fp32, mixed
//  settings, 29 us against 50 with a CTA of 128 per row; 1000 rows 24 and 21; 400
//  rows 22 and 12 (a row with a wide nucleus is slow in one warp);
//  a CTA of 128 to 1024: 100 x 1025 11.5 us with 128, 10.8 with 256; 500 x 5000 23
//  with 256, 28 with 512; 100 x 5000 18.5 and 14.8; 256 x 32000 108 with 512, 91 with
//  1024, 94 in clusters of two of 512;
//  a cluster where the row does not fit a CTA's shared memory, or for few long
//  rows: 4 x 32000 bf16, top-p, 46 us in one CTA, 31 in two, 27 in four or eight;
//  1 x 131072 in eight CTAs of 512 32, of 1024 34; 1 x 8000 16 in one, 21 in two.
template <typename T>
int launch_rows(const Args &a, cudaStream_t s) {
  const int sms = pkcu_sm_count();
  if (a.V <= WARP_MAX && a.n_rows > 6LL * sms) return launch<T, WARP>(a, 1, 128, s);
  int size = 1;
  while ((((a.V + size - 1) / size + 31) & ~31) * 4LL > SMEM_VALUES) size *= 2;
  while (size < 8 && a.n_rows * size * 2 <= sms && a.V / size > 8192) size *= 2;
  const int each = (a.V + size - 1) / size;
  if (size > 1) return launch<T, CLUSTER>(a, size, each <= 16384 ? 512 : 1024, s);
  const int threads = each <= 512 ? 128 : each <= 2048 ? 256 : each <= 8192 ? (a.n_rows > 2 * sms ? 256 : 512) : 1024;
  return launch<T, CTA>(a, 1, threads, s);
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
