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
// Kernel. A row belongs to one CTA, or to a cluster of up to 8 for few long
// rows; its logits are read once into shared memory and everything after that
// works from there. Top-k and top-p search their border in a histogram of
// max - l over linear bins (counts exact; weights in fp32 only as a hint that
// exact sums then confirm), narrow to at most a few hundred candidates and rank
// these against each other; equal logits beyond that are counted, not listed.
// One warp then walks to the token inside its own segment.
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

constexpr int MAX_V = 1 << 18;      // sums of weights <= 2^44 fit 62 bits
constexpr int NBINS = 1024;
constexpr int MAX_CAND = 512;       // candidates ranked against each other
constexpr int MAX_WARPS = 32;
constexpr int SMEM_LOGITS = 128 * 1024;   // bytes of logits a CTA holds

struct Args {
  const void *logits;
  long long ld, n_rows;
  int V, seg;              // seg: entries per CTA of a cluster
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

// exp((v - max) / T) as an integer multiple of 2^-44, rounded; exactly 2^44 for
// v = max. With y = (v - max) 16 log2(e) / T = n + r, |r| <= 1/2: 2^(y / 16) =
// 2^(n div 16) 2^((n mod 16) / 16) e^(r ln 2 / 16), the last by the Taylor series
// of degree 5 (|r ln 2 / 16| < 0.0217: the next term is below 1.5e-13). Sums that
// round to an integer are formed by adding 1.5 2^52.
struct Weight {
  const double *tab;   // 2^(i / 16), shared memory
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

// What one pass over a row adds up, over the threads of a group.
struct Sums {
  u64 w;            // weights
  unsigned n;       // entries
  unsigned lo, hi;  // smallest, largest key
};
__device__ __forceinline__ Sums no_sums() { return Sums{0, 0, 0xffffffffu, 0}; }
__device__ __forceinline__ void add(Sums &a, const Sums &b) {
  a.w += b.w;
  a.n += b.n;
  a.lo = min(a.lo, b.lo);
  a.hi = max(a.hi, b.hi);
}

struct Shared {
  double tab[16];
  Sums warp[MAX_WARPS];
  Sums cta[2];              // this CTA's, read by the cluster; alternating
  unsigned cnt[NBINS];
  float mass[NBINS];
  unsigned scan_n[MAX_WARPS];
  float scan_w[MAX_WARPS];
  int bin;
  unsigned n_cand;
  float cand[MAX_CAND];     // this CTA's, read by the cluster
  float all[MAX_CAND];
  u64 all_w[MAX_CAND];
  unsigned cut_key, cut_take, cut_ties;
  unsigned ties[MAX_WARPS]; // entries equal to the cut, per warp
  u64 kept[MAX_WARPS];      // kept weight per warp
  unsigned first;           // argmax
};

template <typename T, bool CLUSTER>
struct Row {
  const Args &a;
  Shared &s;
  T *x;                     // this CTA's entries
  int base, n;              // first entry's index in the row, entries
  int w0, w1;               // this warp's entries
  unsigned rank, size;
  int phase;

  __device__ __forceinline__ void sync() const {
    if (CLUSTER) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename V>
  __device__ __forceinline__ V *peer(V *p, unsigned r) const {
    return CLUSTER ? cg::this_cluster().map_shared_rank(p, r) : p;
  }
  __device__ __forceinline__ unsigned key(int i) const { return key_of(to_f32(x[i])); }

  // The sums of every thread of the row, to every thread.
  __device__ __forceinline__ Sums total(Sums v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Sums b;
      b.w = __shfl_xor_sync(PK_FULL_MASK, v.w, o);
      b.n = __shfl_xor_sync(PK_FULL_MASK, v.n, o);
      b.lo = __shfl_xor_sync(PK_FULL_MASK, v.lo, o);
      b.hi = __shfl_xor_sync(PK_FULL_MASK, v.hi, o);
      add(v, b);
    }
    __syncthreads();   // the last call's entries are read
    if (lane == 0) s.warp[warp] = v;
    __syncthreads();
    if (CLUSTER) {
      if (threadIdx.x == 0) {
        Sums c = s.warp[0];
        for (int i = 1; i < nw; i++) add(c, s.warp[i]);
        s.cta[phase] = c;
      }
      sync();
      v = *peer(&s.cta[phase], 0);
      for (unsigned r = 1; r < size; r++) add(v, *peer(&s.cta[phase], r));
      phase ^= 1;   // a slot is written again only two cluster barriers later
    } else {
      v = s.warp[0];
      for (int i = 1; i < nw; i++) add(v, s.warp[i]);
    }
    return v;
  }

  // Bin of a key: linear in max - l, the last bin open-ended.
  __device__ __forceinline__ static int bin_of(unsigned k, float max, float scale) {
    const float f = (max - value_of(k)) * scale;
    return f < (float)(NBINS - 1) ? (int)f : NBINS - 1;   // NaN (infinite max): the last
  }

  // The border of a prefix of the order among the entries with key > above: the
  // first of them, from the largest, at which the count (BY_WEIGHT: the weight)
  // reaches `target` (1 .. what there is). Leaves s.cut_key, the border's key,
  // s.cut_take, how many of its equals belong to the prefix, s.cut_ties, how many
  // there are. hist: the bins are filled (for these entries).
  template <bool BY_WEIGHT>
  __device__ void border(unsigned above, u64 target, unsigned max_key, float max, float scale, const Weight &weight) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    sync();   // every CTA's bins are filled
    // each thread takes a run of bins; the first run whose running sum reaches the target
    const int per = (NBINS + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * per;
    unsigned tn = 0;
    float tw = 0.0f;
    for (int b = b0; b < b0 + per && b < NBINS; b++)
      for (unsigned r = 0; r < size; r++) {
        if (BY_WEIGHT) tw += *peer(&s.mass[b], r);
        else tn += *peer(&s.cnt[b], r);
      }
    unsigned pn = tn;
    float pw = tw;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned un = __shfl_up_sync(PK_FULL_MASK, pn, o);
      const float uw = __shfl_up_sync(PK_FULL_MASK, pw, o);
      if (lane >= o) {
        pn += un;
        pw += uw;
      }
    }
    if (lane == 31) {
      s.scan_n[warp] = pn;
      s.scan_w[warp] = pw;
    }
    if (threadIdx.x == 0) s.bin = NBINS - 1;
    __syncthreads();
    for (int i = 0; i < warp; i++) {
      pn += s.scan_n[i];
      pw += s.scan_w[i];
    }
    const float ft = (float)target * 0x1p-44f;
    const bool here = BY_WEIGHT ? pw - tw < ft && ft <= pw : (u64)(pn - tn) < target && target <= (u64)pn;
    if (here) {
      unsigned n = pn - tn;
      float w = pw - tw;
      int b = b0;
      for (; b < b0 + per - 1 && b < NBINS - 1; b++) {
        for (unsigned r = 0; r < size; r++) {
          if (BY_WEIGHT) w += *peer(&s.mass[b], r);
          else n += *peer(&s.cnt[b], r);
        }
        if (BY_WEIGHT ? w >= ft : (u64)n >= target) break;
      }
      // rounding may let neighbouring threads both find theirs (or none: the last bin)
      atomicMin(&s.bin, b);
    }
    __syncthreads();
    // the bin's keys, confirmed by exact sums of what lies above it (a rounding of
    // the hint can be one bin off)
    unsigned hi = max_key, lo = above;        // the border's key is in (lo, hi]
    u64 before = 0;                           // count or weight of the keys > hi
    unsigned inside = 0;                      // entries with keys in (lo, hi]
    bool found = false;
    int bin = s.bin;
    for (int tries = 0; tries < 3 && !found; tries++) {
      Sums up = no_sums(), in = no_sums();
      for (int i = w0 + lane; i < w1; i += 32) {
        const unsigned k = key(i);
        if (k <= above) continue;
        const int b = bin_of(k, max, scale);
        if (b < bin) {
          up.n++;
          if (BY_WEIGHT) up.w += weight(value_of(k));
        } else if (b == bin) {
          in.n++;
          in.lo = min(in.lo, k);
          in.hi = ::max(in.hi, k);
          if (BY_WEIGHT) in.w += weight(value_of(k));
        }
      }
      up = total(up);
      in = total(in);
      const u64 u = BY_WEIGHT ? up.w : up.n, t = BY_WEIGHT ? in.w : in.n;
      found = u < target && target <= u + t;
      if (found) {
        hi = in.hi;
        lo = in.lo - 1;
        before = u;
        inside = in.n;
      }
      bin = target <= u ? ::max(bin - 1, 0) : min(bin + 1, NBINS - 1);
    }
    if (!found) {   // all of them
      Sums in = no_sums();
      for (int i = w0 + lane; i < w1; i += 32) in.n += key(i) > above;
      inside = total(in).n;
    }
    const unsigned cap = 2 * blockDim.x < MAX_CAND ? 2 * blockDim.x : MAX_CAND;
    // too many to rank: halve the range of keys until few are left, or one key
    while (inside > cap && hi - lo > 1) {
      const unsigned mid = lo + (hi - lo) / 2;
      Sums up = no_sums();   // keys in (mid, hi]
      Sums in = no_sums();   // keys in (lo, mid]
      for (int i = w0 + lane; i < w1; i += 32) {
        const unsigned k = key(i);
        if (k <= lo || k > hi) continue;
        Sums &z = k > mid ? up : in;
        z.n++;
        if (BY_WEIGHT) z.w += weight(value_of(k));
      }
      up = total(up);
      in = total(in);
      if (before + (BY_WEIGHT ? up.w : up.n) >= target) {
        lo = mid;
        inside = up.n;
      } else {
        before += BY_WEIGHT ? up.w : up.n;
        hi = mid;
        inside = in.n;
      }
    }
    if (inside > cap) {   // all equal
      if (threadIdx.x == 0) {
        const u64 each = BY_WEIGHT ? weight(value_of(hi)) : 1;
        s.cut_key = hi;
        s.cut_ties = inside;
        s.cut_take = (unsigned)((target - before + each - 1) / each);
      }
      __syncthreads();
      return;
    }
    // list the candidates, everywhere the same ones (in any order)
    if (threadIdx.x == 0) s.n_cand = 0;
    __syncthreads();
    for (int i = w0 + lane; i < w1; i += 32) {
      const unsigned k = key(i);
      if (k > lo && k <= hi) s.cand[atomicAdd(&s.n_cand, 1u)] = value_of(k);
    }
    sync();
    unsigned at = 0;
    for (unsigned r = 0; r < size; r++) {
      const unsigned m = *peer(&s.n_cand, r);
      const float *c = peer(s.cand, r);
      for (unsigned i = threadIdx.x; i < m; i += blockDim.x) {
        s.all[at + i] = c[i];
        if (BY_WEIGHT) s.all_w[at + i] = weight(c[i]);
      }
      at += m;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < at; i += blockDim.x) {
      const float v = s.all[i];
      u64 more = 0;         // count or weight of the larger ones
      unsigned ties = 0;
      for (unsigned j = 0; j < at; j++) {
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
    sync();   // (cluster: the lists are read)
  }

  __device__ __forceinline__ void clear_bins() {
    __syncthreads();
    for (int b = threadIdx.x; b < NBINS; b += blockDim.x) {
      s.cnt[b] = 0;
      s.mass[b] = 0.0f;
    }
    __syncthreads();
  }

  __device__ void run(long long row);
};

template <typename T, bool CLUSTER>
__device__ void Row<T, CLUSTER>::run(long long row) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const T *src = static_cast<const T *>(a.logits) + row * a.ld + base;
  // 1. the row, once; its largest and smallest values
  Sums v = no_sums();
#pragma unroll 8
  for (int i = w0 + lane; i < w1; i += 32) {
    const T e = src[i];
    x[i] = e;
    const unsigned k = key_of(to_f32(e));
    if (k) {
      v.n++;
      v.lo = min(v.lo, k);
      v.hi = ::max(v.hi, k);
    }
  }
  v = total(v);
  const unsigned n_valid = v.n, max_key = v.hi;
  if (n_valid == 0) {   // nothing to take
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  const float max = value_of(max_key);
  const float temp = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  if (!(temp > 0.0f)) {   // greedy: the first largest
    Sums f = no_sums();
    for (int i = w0 + lane; i < w1; i += 32)
      if (key(i) == max_key) f.lo = min(f.lo, (unsigned)(base + i));
    f = total(f);
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = (int)f.lo;
      if (a.logprobs) a.logprobs[row] = 0.0f;
    }
    return;
  }
  Weight weight;
  weight.tab = s.tab;
  weight.c = 16.0 * 1.44269504088896340736 / (double)temp;
  weight.max = max;
  const int k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float p = a.top_p ? __ldg(a.top_p + row) : 1.0f;
  const float mp = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  // bins over the values' range, at most 64 wide (below it one open bin)
  float range = max - value_of(v.lo);
  range = range < 64.0f ? range : 64.0f;
  const float scale = (float)(NBINS - 2) / ::fmaxf(range, 1e-30f);

  // 2. the cut: kept are keys > cut and the first `take` of its `ties` equals
  unsigned cut = 0, take = 0, ties = 0;
  if (k > 0 && (unsigned)k < n_valid) {
    clear_bins();
    for (int i = w0 + lane; i < w1; i += 32) {
      const unsigned e = key(i);
      if (e) atomicAdd(&s.cnt[bin_of(e, max, scale)], 1u);
    }
    border<false>(0, (u64)k, max_key, max, scale, weight);
    cut = s.cut_key;
    take = s.cut_take;
    ties = s.cut_ties;
  }
  if (p < 1.0f) {
    clear_bins();
    Sums t = no_sums();
    for (int i = w0 + lane; i < w1; i += 32) {
      const unsigned e = key(i);
      if (e <= cut) continue;
      const u64 w = weight(value_of(e));
      t.w += w;
      atomicAdd(&s.mass[bin_of(e, max, scale)], (float)w * 0x1p-44f);
    }
    t = total(t);
    const u64 each = cut ? weight(value_of(cut)) : 0;
    const u64 sum = t.w + take * each;
    // the least integer that is at least p times the sum (and at least 1)
    u64 target = p > 0.0f ? (u64)ceil((double)p * (double)sum) : 1;
    target = target < 1 ? 1 : target < sum ? target : sum;
    if (target > t.w) {   // inside the equals of the top-k's border
      take = (unsigned)((target - t.w + each - 1) / each);
    } else {
      border<true>(cut, target, max_key, max, scale, weight);
      cut = s.cut_key;
      take = s.cut_take;
      ties = s.cut_ties;
    }
  }
  // min-p: a weight at least min_p of the largest, which always stays
  u64 least = 0;
  if (mp > 0.0f) least = (u64)ceil((double)(mp < 1.0f ? mp : 1.0f) * 0x1p44);

  // 3. equals of the cut before each warp, where not all are kept
  unsigned tie_rank = 0;
  const bool part = take < ties;
  if (part) {
    unsigned c = 0;
    for (int i = w0 + lane; i < w1; i += 32) c += key(i) == cut;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(PK_FULL_MASK, c, o);
    if (lane == 0) s.ties[warp] = c;
    sync();
    for (unsigned r = 0; r < rank; r++)
      for (int i = 0; i < nw; i++) tie_rank += *peer(&s.ties[i], r);
    for (int i = 0; i < warp; i++) tie_rank += s.ties[i];
  }
  // kept weight of entry i (0: none) for the warp's entries in order
  unsigned seen = tie_rank;
  auto kept = [&](int i) -> u64 {
    const unsigned e = i < w1 ? key(i) : 0;
    bool keep = e > cut;
    if (part) {
      const unsigned same = __ballot_sync(PK_FULL_MASK, e == cut);
      keep = keep || (e == cut && seen + __popc(same & ((1u << lane) - 1)) < take);
      seen += __popc(same);
    } else {
      keep = keep || (e == cut && e != 0);
    }
    if (!keep) return 0;
    const u64 w = weight(value_of(e));
    return w >= least ? w : 0;
  };

  // 4. the kept weight of every warp, and where u falls
  u64 mine = 0;
  for (int i = w0; i < w1; i += 32) mine += kept(i + lane);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(PK_FULL_MASK, mine, o);
  if (lane == 0) s.kept[warp] = mine;
  sync();
  u64 sum = 0, before = 0;
  for (unsigned r = 0; r < size; r++)
    for (int i = 0; i < nw; i++) {
      const u64 w = *peer(&s.kept[i], r);
      if (r < rank || (r == rank && i < warp)) before += w;
      sum += w;
    }
  const float uu = a.u ? __ldg(a.u + row) : 0.0f;
  u64 target = uu > 0.0f ? (u64)((double)uu * (double)sum) : 0;   // floor; the sum of an entry exceeds it
  target = target < sum ? target : sum - 1;
  if (target >= before && target < before + mine) {   // this warp's
    seen = tie_rank;
    u64 run = before;
    for (int i = w0; i < w1; i += 32) {
      const u64 w = kept(i + lane);
      u64 inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(PK_FULL_MASK, inc, o);
        if (lane >= o) inc += up;
      }
      const u64 all = __shfl_sync(PK_FULL_MASK, inc, 31);
      if (target < run + all) {
        const unsigned past = __ballot_sync(PK_FULL_MASK, run + inc > target);
        if (lane == __ffs(past) - 1) {
          a.tokens[row] = base + i + lane;
          if (a.logprobs) {
            // log(w / S): the exponent itself less log S, S in units of the largest weight
            const float val = to_f32(x[i + lane]);
            const double y = val == max ? 0.0 : ((double)val - (double)max) / (double)temp;
            const double over = (double)(sum - (1ull << 44)) * 0x1p-44;
            a.logprobs[row] = (float)(y - (double)log1pf((float)over));
          }
        }
        break;
      }
      run += all;
    }
  }
}

template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(1024) sample_kernel(Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Shared s;
  Row<T, CLUSTER> r{a, s};
  r.x = reinterpret_cast<T *>(smem);
  r.size = CLUSTER ? cg::this_cluster().num_blocks() : 1;
  r.rank = CLUSTER ? cg::this_cluster().block_rank() : 0;
  r.phase = 0;
  r.base = (int)r.rank * a.seg;
  r.n = a.V - r.base < a.seg ? a.V - r.base : a.seg;
  if (r.n < 0) r.n = 0;
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int per = ((r.n + nw - 1) / nw + 31) & ~31;
  r.w0 = warp * per < r.n ? warp * per : r.n;
  r.w1 = r.w0 + per < r.n ? r.w0 + per : r.n;
  if (threadIdx.x < 16) s.tab[threadIdx.x] = exp2(threadIdx.x / 16.0);
  __syncthreads();
  const long long step = gridDim.x / r.size;
  for (long long row = blockIdx.x / r.size; row < a.n_rows; row += step) {
    r.run(row);
    r.sync();   // shared memory is free for the next row (and the peers' reads are done)
  }
}

template <typename T, bool CLUSTER>
int launch(Args a, int size, int threads, cudaStream_t s) {
  static int flags[64];
  smem_optin(sample_kernel<T, CLUSTER>, SMEM_LOGITS, flags);
  a.seg = ((a.V + size - 1) / size + 31) & ~31;
  const long long most = 1 << 20;
  const long long rows = a.n_rows < most ? a.n_rows : most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * size));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)a.seg * sizeof(T);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  if (CLUSTER) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  cudaLaunchKernelEx(&cfg, sample_kernel<T, CLUSTER>, a);
  return pkcu_launch_status("pkcu_sample_rows");
}

template <typename T>
int launch_rows(const Args &a, cudaStream_t s) {
  // CTAs per row: what the logits need, and more while that leaves SMs idle
  int size = 1;
  while ((((a.V + size - 1) / size + 31) & ~31) * (long long)sizeof(T) > SMEM_LOGITS) size *= 2;
  while (size < 8 && a.n_rows * size * 2 <= pkcu_sm_count() && a.V / size > 4096) size *= 2;
  const int each = (a.V + size - 1) / size;
  const int threads = each <= 2048 ? 128 : each <= 8192 ? 512 : 1024;
  return size > 1 ? launch<T, true>(a, size, threads, s) : launch<T, false>(a, 1, threads, s);
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
