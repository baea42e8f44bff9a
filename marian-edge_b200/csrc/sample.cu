// sample.cu -- the next token of each row from its logits and one given
// random number: temperature, top-k, top-p, min-p (mc_sample).
//
// With the tokens ordered by logit (largest first, ties by id), weights
// w = exp((logit - max) / T):
//   A = the first k,  B = the shortest prefix of A with sum w >= p sum_A w,
//   C = those of B with w >= min_p,
//   token = the first id, ascending, whose running sum over C exceeds u sum_C w.
//
// One cluster of CTAs per row: each keeps a slice of the logits in shared
// memory, so they are read from HBM once, and every later pass runs there.
// The row is not sorted.  One histogram of counts, linear in the logits, says
// above which bin all that can matter lies (the k-th logit, top_p's border by
// the bins' smallest weights, min_p's floor); those tokens, seldom more than a
// few hundred, go to one CTA, of which one warp (or all, for more than 256)
// orders them and finds the three cuts and the draw exactly, while the other
// CTAs are done.  Without cuts, the draw is the place of u times the sum of
// all weights, in the part of the row that holds it.
//
// Rows with more candidates than the list takes go the general way: each cut
// is the border of a prefix of the order, "above a key, and so many ties of
// it"; a histogram of exact weights or counts finds the bin that it lies in,
// whose tokens are sorted, and the draw is from all tokens before it.
//
// Measured at 1,024 x 32,000 f32, mixed settings, for other layouts: every
// border by histograms of keys 587 us; three passes over L2 by one CTA per row
// 225 us (L2 gives 17 bytes a cycle and SM there); one pass over HBM with a
// sample's threshold 321 us, of which the few rows that the sample misjudges
// are two thirds; slices of 16,384 or 4,096 logits 200 and 270 us.
//
// Weights are fixed-point integers, 40 fraction bits (a 64-bit sum holds
// 2^24 of them): sums do not depend on their order, so neither atomics nor
// the split over CTAs can change a token, and at a relative 2^-41 per weight
// the chance that a token differs from the real-number definition is about
// 1e-9 a row.  (In f32 the sums' errors, 1e-7 of the whole, move each of
// 32,000 borders by that much: a token in a few hundred would differ.)
#include <cooperative_groups.h>

#include <cstring>

#include "decode_ops.cuh"

namespace mc {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kFull = 0xFFFFFFFFu;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;                  // of the general way's histograms
constexpr int kBinBits = 10;
static_assert(kBins == 1 << kBinBits, "a bin is the leading bits of a key's place");
constexpr int kThreadBits = 8;
static_assert(kThreads == 1 << kThreadBits, "a thread is the leading bits of an id's place");
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 393216;  // as the lexical shortlist's masks (kernels.cuh)

struct SampleParams {
  const void* logits;
  long long row_stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t* top_k;
  const uint32_t* candidates;
  long long candidates_stride;
  int32_t* tokens;
  float* probs;
  int rows, vocab, segment;  // segment: ids of one warp
  uint32_t* status;
};

// Order-preserving bit pattern of a float (no NaN, no -0).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr uint32_t kKeyNone = 0x007FFFFFu;  // key_of(-inf): a token that cannot be drawn
constexpr int kCoarse = 512;                // bins of the histogram of counts
constexpr int kList = 2048;                 // candidates that one CTA takes
constexpr int kAhead = 2;                   // the largest logit's bin, about
constexpr int kWarpList = 256;              // candidates that one warp takes
constexpr int kCrowd = 64;                  // tokens of one bin beyond which comparing all pairs costs more than a sort
// Weights vanish 42 halvings below the top: (top - v) / T above 42 ln 2.
constexpr float kReach = 29.2f;

template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float none() { return -INFINITY; }
};
template <>
struct Logit<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half none() { return __ushort_as_half(0xFC00); }
};
template <>
struct Logit<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 none() { return __ushort_as_bfloat16(0xFF80); }
};

// Exact f32 -> f64 in integer operations (the conversion instruction runs at
// a fraction of the rate).  Subnormals, which come out as about 2^-127, and
// zero differ from their value by less than 2^-126.
__device__ __forceinline__ double widen(float v) {
  const uint32_t b = __float_as_uint(v);
  return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u)), (int)(b << 29));
}

struct Weigher {
  double top, rate;      // the weight's logit of 1; log2(e) / T
  uint32_t top_key;
  const double* powers;  // 2^-(j / 64)
  double per_step, per_logit;

  __device__ __forceinline__ Weigher(float top_, double temperature, const double* powers_)
      : top(widen(top_)), rate(1.4426950408889634074 / temperature), top_key(key_of(top_)), powers(powers_) {
    per_step = rate * -64.0;
    per_logit = 1.0 / temperature;
  }
  // w = exp((v - top) / T) as *rest times the result: with k = 64 rate (top - v)
  // to the nearest whole number (the sum with 1.5 * 2^52), 2^-(k / 64) from the
  // table times exp(z), z = (v - top) / T + k ln 2 / 64, |z| <= 0.0055, by its
  // series to the fourth power (the fifth is below 5e-14).  For |top - v| rate <
  // 1000, without a branch, so that several are in flight; 1 at the top.
  __device__ __forceinline__ double near(float v, double* rest) const {
    const double d = __dsub_rn(widen(v), top), t = __fma_rn(d, per_step, 6755399441055744.0);
    const int k = __double2loint(t);
    const double z = __fma_rn(__dsub_rn(t, 6755399441055744.0), 0.010830424696249145, __dmul_rn(d, per_logit));
    double s = __fma_rn(z, 1.0 / 24, 1.0 / 6);
    s = __fma_rn(s, z, 0.5);
    s = __fma_rn(s, z, 1.0);
    *rest = __fma_rn(s, z, 1.0);
    const double p = powers[k & 63];
    return __hiloint2double(__double2hiint(p) - ((k >> 6) << 20), __double2loint(p));
  }
  __device__ __forceinline__ double near(float v) const {
    double rest;
    const double p = near(v, &rest);
    return __dmul_rn(p, rest);
  }
  __device__ __forceinline__ unsigned long long fixed_near(float v) const {
    double rest;
    const double p = near(v, &rest);
    return last_bits(__fma_rn(p, rest, 4096.0));
  }
  // Any v, top and T: 0 below 2^-42, 1 at the top even where it or rate is infinite.
  __device__ double real(float v, uint32_t key) const {
    if (key == top_key) return 1.0;
    const double y = __dmul_rn(__dsub_rn((double)value_of(top_key), (double)v), rate);
    return y < 42.0 ? exp2(-y) : 0.0;
  }
  // Of 2^12 + w: the 40 fraction bits are at the end of the mantissa.
  static __device__ __forceinline__ unsigned long long last_bits(double w) {
    return (unsigned long long)__double_as_longlong(w) & ((1ull << 51) - 1);
  }
  static __device__ __forceinline__ unsigned long long fixed(double w) { return last_bits(__dadd_rn(w, 4096.0)); }
};

// What the CTAs of a row tell one another; two of each, used in turn, so
// that one cluster barrier per exchange is enough.
struct Exchange {
  unsigned long long value[2][2];
};

struct Shared {
  union {
    unsigned long long hist[2][kBins];  // the general way
    unsigned long long list[kList];     // candidates: key, then ~id
  };
  uint32_t counts[kCoarse];      // tokens of this slice per bin; in a long list's draw, weights per range of ids
  uint32_t starts[kCoarse + 1];  // of the whole row, up to each bin
  uint32_t filled[kCoarse];      // candidates of each bin that have arrived
  uint32_t listed;               // tokens of a border's bin
  double powers[64];
  Exchange out;
  unsigned long long warp_value[kWarps];
  unsigned long long found[3];
};

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_prefix(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

// Sorts list[0, 2^m) in descending order (bitonic).
__device__ void sort_list(unsigned long long* list, int n2, int tid) {
  for (int size = 2; size <= n2; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < n2 / 2; i += kThreads) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const unsigned long long u = list[a], v = list[b];
        if ((u < v) == ((a & size) == 0)) {
          list[a] = v;
          list[b] = u;
        }
      }
      // pairs up to 32 apart stay within one warp's 64 elements
      if (step > 32 || (step == 1 && size >= 64))
        __syncthreads();
      else
        __syncwarp();
    }
  __syncthreads();
}

// Which tokens are still in: those above `key`, and those equal to it with an
// id up to `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool holds(uint32_t k, int id) const { return k > key || (k == key && id <= last); }
};

template <typename T>
struct Row {
  const SampleParams& p;
  Shared& sh;
  T* x;  // this CTA's slice in shared memory
  cg::cluster_group cluster;
  int ranks, rank, base, n, tid, lane, warp, turn, level;

  // A logit as it orders: NaN is never drawn, -0 is 0.
  __device__ __forceinline__ float at(int i) const {
    const float v = Logit<T>::get(x[i]);
    return v == v ? __fadd_rn(v, 0.0f) : -INFINITY;
  }
  // One pass over the slice, each warp over its segment, 16 bytes at a time:
  // f(logit, place).  The slice is padded with tokens that cannot be drawn.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int kVec = 16 / (int)sizeof(T);
    const int begin = min(n, warp * p.segment), end = min(n, begin + p.segment);
    for (int i = begin + lane * kVec; i < end; i += 32 * kVec) {
      const uint4 q = *reinterpret_cast<const uint4*>(x + i);
      T t[kVec];
      memcpy(t, &q, 16);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f(Logit<T>::get(t[j]), i + j);
    }
  }

  // ---- reductions over the row ----
  __device__ __forceinline__ unsigned long long block_sum(unsigned long long v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.warp_value[warp] = v;
    __syncthreads();
    v = sh.warp_value[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v += sh.warp_value[w];
    return v;
  }
  // The largest of two values over the block, in one exchange.
  __device__ __forceinline__ void block_max2(uint32_t& a, uint32_t& b) {
    a = __reduce_max_sync(kFull, a);
    b = __reduce_max_sync(kFull, b);
    __syncthreads();
    if (lane == 0) sh.warp_value[warp] = (unsigned long long)a << 32 | b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const unsigned long long o = sh.warp_value[w];
      a = max(a, (uint32_t)(o >> 32));
      b = max(b, (uint32_t)o);
    }
  }
  // Publishes this CTA's values; afterwards peer(r, i) reads those of CTA r.
  __device__ __forceinline__ void publish(unsigned long long a, unsigned long long b = 0) {
    turn ^= 1;
    if (tid == 0) {
      sh.out.value[turn][0] = a;
      sh.out.value[turn][1] = b;
    }
    cluster.sync();
  }
  __device__ __forceinline__ unsigned long long peer(int r, int i) {
    return cluster.map_shared_rank(&sh, r)->out.value[turn][i];
  }

  // ---- the border of a prefix of the order ----
  // Cuts `cut` to the shortest prefix of the order (of the tokens it holds)
  // whose sum of f reaches target, or `share` of the whole sum where that is
  // not negative; leaves it alone when the whole sum does not reach target.
  // A histogram linear in the logits finds the bin of the border; its tokens
  // are sorted in CTA 0.  Where they are too many, histograms of the keys'
  // leading bits narrow them down to one key, and its ties are counted.
  template <typename F>
  __device__ void border(Cut* cut, F f, unsigned long long target, float top, float range, uint32_t key_min,
                         uint32_t key_max, double share) {
    const Cut in = *cut;
    uint32_t lo = key_min, hi = key_max;
    unsigned long long over = 0, ties = 0;
    const bool linear = range > 0.0f && range < INFINITY;
    const float step = linear ? __fdiv_rn((float)kBins * 0.999f, range) : 0.0f;
    // whole ranges of keys, as rounding keeps the order
    auto bin_of = [&](float v) { return (int)fminf(__fmul_rn(__fsub_rn(top, v), step), (float)(kBins - 1)); };
    auto held = [&](float& v, int i, uint32_t* k) {
      v = v == v ? __fadd_rn(v, 0.0f) : -INFINITY;
      *k = key_of(v);
      return *k >= lo && *k <= hi && in.holds(*k, base + i);
    };
    int first_bin = -1;
    for (bool start = linear;; start = false) {
      unsigned long long* hist = sh.hist[level & 1];
      ++level;
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
      __syncthreads();
      int shift = 0;
      if (!start) {
        const uint32_t span = hi - lo;
        shift = span < kBins ? 0 : 32 - kBinBits - __clz(span);
      }
      each([&](float v, int i) {
        uint32_t k;
        if (!held(v, i, &k) || (!start && first_bin >= 0 && bin_of(v) != first_bin)) return;
        const unsigned long long w = f(v, k);
        if (w) atomicAdd(&hist[start ? bin_of(v) : (int)((hi - k) >> shift)], w);
      });
      cluster.sync();
      constexpr int kPer = kBins / kThreads;
      unsigned long long mine[kPer], sum = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) mine[j] = 0;
      for (int r = 0; r < ranks; ++r) {
        const unsigned long long* other = cluster.map_shared_rank(&sh, r)->hist[(level - 1) & 1];
#pragma unroll
        for (int j = 0; j < kPer; ++j) mine[j] += other[tid * kPer + j];
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum += mine[j];
      const unsigned long long inc = warp_prefix(sum, lane);
      if (lane == 31) sh.warp_value[warp] = inc;
      __syncthreads();
      unsigned long long before = over + inc - sum, total = over;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh.warp_value[w];
        total += sh.warp_value[w];
      }
      if (share >= 0.0) {  // known after the first pass
        target = (unsigned long long)ceil(__dmul_rn(share, (double)total));
        target = target < 1 ? 1 : target > total ? total : target;
        share = -1.0;
      }
      if (total < target) return;  // every CTA of the row sees the same
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (before < target && target <= before + mine[j]) {
          sh.found[0] = tid * kPer + j;
          sh.found[1] = before;
          sh.found[2] = mine[j];
        }
        before += mine[j];
      }
      __syncthreads();
      const int bin = (int)sh.found[0];
      over = sh.found[1];
      ties = sh.found[2];
      __syncthreads();
      if (start) {
        first_bin = bin;
        // the keys of the bin, with a margin that covers the rounding of bin_of
        const float from = __fsub_rn(top, __fdiv_rn((float)bin - 0.01f, step));
        const float to = __fsub_rn(top, __fdiv_rn((float)bin + 1.01f, step));
        if (bin > 0) hi = min(hi, key_of(__fadd_rn(from, 0.0f)));
        if (bin < kBins - 1) lo = max(lo, key_of(__fadd_rn(to, 0.0f)));
        if (sort_border(cut, f, [&](float& v, int i, uint32_t* k) { return held(v, i, k) && bin_of(v) == bin; }, over, target))
          return;
      } else {
        hi -= (uint32_t)bin << shift;
        const uint32_t width = (1u << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
        if (shift == 0) break;
      }
    }
    const unsigned long long w = f(value_of(hi), hi), kept = (target - over + w - 1) / w;
    cut->last = kept * w < ties ? nth_tie(in, hi, kept) : hi == in.key ? in.last : INT32_MAX;
    cut->key = hi;
  }

  // The border among the tokens of one bin, by sorting them in CTA 0; false
  // when they are more than its list takes.
  template <typename F, typename H>
  __device__ bool sort_border(Cut* cut, F f, H in_bin, unsigned long long over, unsigned long long target) {
    if (tid == 0) sh.listed = 0;
    cluster.sync();  // also: every CTA has read the histogram that the list replaces
    Shared* home = cluster.map_shared_rank(&sh, 0);
    each([&](float v, int i) {
      uint32_t k;
      if (!in_bin(v, i, &k) || !f(v, k)) return;
      const uint32_t slot = atomicAdd(&home->listed, 1u);
      if (slot < kList) home->list[slot] = (unsigned long long)k << 32 | (kFull - (uint32_t)(base + i));
    });
    cluster.sync();
    unsigned long long found = 0;
    if (rank == 0 && sh.listed <= kList) {
      const int n = (int)sh.listed;
      int n2 = 64;
      while (n2 < n) n2 <<= 1;
      for (int i = n + tid; i < n2; i += kThreads) sh.list[i] = 0;
      __syncthreads();
      sort_list(sh.list, n2, tid);
      constexpr int kEach = kList / kThreads;
      unsigned long long weight[kEach], sum = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = tid * kEach + j;
        const uint32_t k = i < n ? (uint32_t)(sh.list[i] >> 32) : 0u;
        weight[j] = i < n ? f(value_of(k), k) : 0ull;
        sum += weight[j];
      }
      const unsigned long long inc = warp_prefix(sum, lane);
      __syncthreads();
      if (tid == 0) sh.found[0] = 0;
      if (lane == 31) sh.warp_value[warp] = inc;
      __syncthreads();
      unsigned long long run = over + inc - sum;
      for (int w = 0; w < warp; ++w) run += sh.warp_value[w];
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (run < target && target <= run + weight[j]) sh.found[0] = sh.list[tid * kEach + j];
        run += weight[j];
      }
      __syncthreads();
      found = sh.found[0];
    }
    publish(found);
    found = peer(0, 0);
    if (!found) return false;
    cut->key = (uint32_t)(found >> 32);
    cut->last = (int)(kFull - (uint32_t)found);
    return true;
  }

  // ---- the first id, ascending, at which a running sum exceeds a target ----
  // One warp's part of f over its segment.
  template <typename F>
  __device__ __forceinline__ unsigned long long segment_sum(F f) const {
    unsigned long long s = 0;
    each([&](float v, int i) {
      v = v == v ? __fadd_rn(v, 0.0f) : -INFINITY;
      s += f(v, key_of(v), base + i);
    });
    return warp_sum(s);
  }
  // The id for a target, from the sums of f before and after each warp's
  // segment (one warp's `after` is the next one's `before`); -1 in the CTAs that
  // do not hold it.  The warp that does shares its segment out over the block,
  // until each warp's part is short.
  template <typename F>
  __device__ int locate(F f, unsigned long long before, unsigned long long after, unsigned long long target) {
    __syncthreads();
    if (tid == 0) sh.found[0] = kWarps;
    __syncthreads();
    if (lane == 0 && before <= target && target < after) {
      sh.found[0] = warp;
      sh.found[1] = before;
    }
    __syncthreads();
    const int owner = (int)sh.found[0];
    if (owner == kWarps) return -1;  // the whole block
    before = sh.found[1];
    int lo = owner * p.segment, hi = min(n, lo + p.segment);
    constexpr int kFew = 16;  // loads that one warp has in flight at the end
    while (hi - lo > 32 * kFew) {
      const int part = ((hi - lo) / 32 + kWarps - 1) / kWarps * 32 + 32;
      const int begin = min(hi, lo + warp * part), stop = min(hi, begin + part);
      unsigned long long sum = 0;
#pragma unroll 4
      for (int i = begin + lane; i < stop; i += 32) {
        const float v = at(i);
        sum += f(v, key_of(v), base + i);
      }
      sum = warp_sum(sum);
      __syncthreads();
      if (lane == 0) sh.warp_value[warp] = sum;
      __syncthreads();
      unsigned long long run = before, start = before;
      int mine = 0;  // the first part whose sum passes the target, or the last with any
      bool hit = false;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const unsigned long long s = sh.warp_value[w];
        if (s > 0 && !hit) {
          mine = w;
          start = run;
          hit = target < run + s;
        }
        run += s;
      }
      before = start;
      lo = min(hi, lo + mine * part);
      hi = min(hi, lo + part);
    }
    if (warp == 0) {
      float v[kFew];
#pragma unroll
      for (int k = 0; k < kFew; ++k) v[k] = lo + 32 * k + lane < hi ? at(lo + 32 * k + lane) : -INFINITY;
      int id = -1;
      bool hit = false;
#pragma unroll
      for (int k = 0; k < kFew; ++k) {
        const int i = lo + 32 * k;
        if (hit || i >= hi) continue;
        const unsigned long long w = i + lane < hi ? f(v[k], key_of(v[k]), base + i + lane) : 0ull;
        const unsigned long long inc = before + warp_prefix(w, lane);
        const uint32_t past = __ballot_sync(kFull, w > 0 && inc > target), some = __ballot_sync(kFull, w > 0);
        if (some) id = base + i + 31 - __clz(some);
        if (past) {
          id = base + i + __ffs(past) - 1;
          hit = true;
        }
        before = __shfl_sync(kFull, inc, 31);
      }
      if (lane == 0) sh.found[2] = (unsigned long long)id;
    }
    __syncthreads();
    return (int)sh.found[2];
  }
  // Sums of f before this warp, and of the whole row.
  __device__ __forceinline__ unsigned long long prefix(unsigned long long sum, unsigned long long* total) {
    __syncthreads();
    if (lane == 0) sh.warp_value[warp] = sum;
    __syncthreads();
    unsigned long long before = 0, own = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.warp_value[w];
      own += sh.warp_value[w];
    }
    publish(own);
    *total = 0;
    for (int r = 0; r < ranks; ++r) {
      const unsigned long long o = peer(r, 0);
      if (r < rank) before += o;
      *total += o;
    }
    return before;
  }
  // The id of the count-th tie of key among the tokens of `in`.
  __device__ int nth_tie(const Cut& in, uint32_t key, unsigned long long count) {
    auto one = [&](float, uint32_t k, int id) -> unsigned long long { return k == key && in.holds(k, id); };
    const unsigned long long sum = segment_sum(one);
    unsigned long long total;
    const unsigned long long before = prefix(sum, &total);
    const int id = locate(one, before, before + sum, count - 1);
    publish((unsigned long long)(id + 1));
    unsigned long long best = 0;
    for (int r = 0; r < ranks; ++r) {
      const unsigned long long o = peer(r, 0);
      best = o > best ? o : best;
    }
    return (int)best - 1;
  }
};

// Puts list[0, n) in the row's order.  The candidates arrived bin by bin, so
// each takes its place among its bin's; a crowded bin makes that cost more
// than sorting them all.
template <int THREADS, typename F>
__device__ void order_list(Shared& sh, int n, bool crowded, int tid, F bin_of_key) {
  if (crowded) {
    int n2 = 64;
    while (n2 < n) n2 <<= 1;
    for (int i = n + tid; i < n2; i += THREADS) sh.list[i] = 0;
    __syncthreads();
    sort_list(sh.list, n2, tid);
    return;
  }
  constexpr int kEach = (THREADS == 32 ? kWarpList : kList) / THREADS;
  unsigned long long own[kEach];
  uint32_t place[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = tid + j * THREADS;
    own[j] = 0;
    if (i >= n) continue;
    own[j] = sh.list[i];
    const uint32_t bin = bin_of_key((uint32_t)(own[j] >> 32));
    const uint32_t from = sh.starts[bin], to = sh.starts[bin + 1];
    uint32_t ahead = 0;
    for (uint32_t k = from; k < to; ++k) ahead += sh.list[k] > own[j];
    place[j] = from + ahead;
  }
  if (THREADS == 32) __syncwarp(); else __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (own[j]) sh.list[place[j]] = own[j];
  if (THREADS == 32) __syncwarp(); else __syncthreads();
}

struct Cuts {
  bool by_k, by_p;
  int top_k;
  double top_p, floor_w, u;
  unsigned long long whole;  // weights of the row
};

// The cuts and the draw from the ordered list, by one warp or by the block.
template <typename T, bool WARP>
__device__ void finish_list(Row<T>& r, const Weigher& weigh, const Cuts& q, int listed) {
  Shared& sh = r.sh;
  constexpr int kEach = (WARP ? kWarpList : kList) / (WARP ? 32 : kThreads);
  const int tid = r.tid, lane = r.lane, first = tid * kEach;
  auto total_of = [&](unsigned long long v) { return WARP ? warp_sum(v) : r.block_sum(v); };
  auto count_of = [&](uint32_t v) { return WARP ? __reduce_add_sync(kFull, v) : (uint32_t)r.block_sum(v); };
  // thread i holds the ordered candidates kEach i .. kEach i + kEach - 1
  const int in_a = q.by_k ? min(listed, q.top_k) : listed;
  unsigned long long weight[kEach], sum = 0;
  uint32_t above_floor = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    weight[j] = 0;
    if (first + j < in_a) {
      const uint32_t key = (uint32_t)(sh.list[first + j] >> 32);
      weight[j] = weigh.fixed_near(value_of(key));
      above_floor += weigh.near(value_of(key)) >= q.floor_w;
    }
    sum += weight[j];
  }
  int in_c = in_a;
  if (q.by_p) {
    unsigned long long run = warp_prefix(sum, lane) - sum, all;
    if (WARP) {
      all = __shfl_sync(kFull, run + sum, 31);
    } else {
      __syncthreads();
      if (lane == 31) sh.warp_value[r.warp] = run + sum;
      __syncthreads();
      all = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < r.warp) run += sh.warp_value[i];
        all += sh.warp_value[i];
      }
    }
    const unsigned long long mass_a = q.by_k ? all : q.whole;
    unsigned long long border = (unsigned long long)ceil(__dmul_rn(q.top_p, (double)mass_a));
    border = border < 1 ? 1 : border > mass_a ? mass_a : border;
    // those whose running sum before them is below the border
    uint32_t below = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      below += first + j < in_a && run < border;
      run += weight[j];
    }
    in_c = (int)count_of(below);
  }
  in_c = min(in_c, (int)count_of(above_floor));
  sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (first + j >= in_c) weight[j] = 0;
    sum += weight[j];
  }
  const unsigned long long total = total_of(sum);
  unsigned long long target = (unsigned long long)floor(__dmul_rn(q.u, (double)total));
  if (target >= total) target = total - 1;
  uint32_t drawn = 0;
  unsigned long long drawn_weight = 0;
  if (WARP && in_c <= 96) {
    // The candidate whose running sum by id passes target: all pairs.
    unsigned long long* const weights = sh.list + kWarpList;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (first + j < in_c) weights[first + j] = weight[j];
    __syncwarp();
    unsigned long long run[3] = {0, 0, 0}, own[3];
    uint32_t mark[3];  // smaller ids have larger complements
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      own[j] = lane + 32 * j < in_c ? weights[lane + 32 * j] : 0ull;
      mark[j] = lane + 32 * j < in_c ? (uint32_t)sh.list[lane + 32 * j] : kFull;
    }
#pragma unroll 4
    for (int k = 0; k < in_c; ++k) {
      const uint32_t m = (uint32_t)sh.list[k];
      const unsigned long long w = weights[k];
#pragma unroll
      for (int j = 0; j < 3; ++j) run[j] += m > mark[j] ? w : 0ull;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const uint32_t hit = __ballot_sync(kFull, run[j] <= target && target < run[j] + own[j]);
      if (hit) {
        drawn = kFull - __shfl_sync(kFull, mark[j], __ffs(hit) - 1);
        drawn_weight = __shfl_sync(kFull, own[j], __ffs(hit) - 1);
      }
    }
  } else if (WARP) {
    // The lowest id at which the weights up to it exceed target, by halving.
    uint32_t id[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) id[j] = weight[j] ? kFull - (uint32_t)sh.list[first + j] : kFull;
    uint32_t lo = 0, hi = (uint32_t)r.p.vocab - 1;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      unsigned long long s = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) s += id[j] <= mid ? weight[j] : 0ull;
      if (warp_sum(s) > target)
        hi = mid;
      else
        lo = mid + 1;
    }
    drawn = lo;
#pragma unroll
    for (int j = 0; j < kEach; ++j) drawn_weight += id[j] == drawn ? weight[j] : 0ull;
    drawn_weight = warp_sum(drawn_weight);
  } else {
    // The same, a range of ids per thread at a time, by their weights.
    unsigned long long* ranges = reinterpret_cast<unsigned long long*>(sh.counts);
    static_assert(sizeof(sh.counts) >= kThreads * sizeof(unsigned long long), "a range per thread");
    for (int shift = max(0, 32 - kThreadBits - __clz((uint32_t)r.p.vocab));; shift = max(0, shift - kThreadBits)) {
      __syncthreads();
      ranges[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (weight[j]) {
          const uint32_t id = kFull - (uint32_t)sh.list[first + j], at = (id - drawn) >> shift;
          if (id >= drawn && at < kThreads) atomicAdd(&ranges[at], weight[j]);
        }
      __syncthreads();
      const unsigned long long mine = ranges[tid], inc = warp_prefix(mine, lane);
      if (lane == 31) sh.warp_value[r.warp] = inc;
      __syncthreads();
      unsigned long long start = inc - mine;
#pragma unroll
      for (int i = 0; i < kWarps; ++i)
        if (i < r.warp) start += sh.warp_value[i];
      if (start <= target && target < start + mine) {
        sh.found[0] = tid;
        sh.found[1] = start;
        sh.found[2] = mine;
      }
      __syncthreads();
      drawn += (uint32_t)sh.found[0] << shift;
      target -= sh.found[1];
      drawn_weight = sh.found[2];
      if (shift == 0) break;
    }
  }
  if (tid == 0) {
    const int row = blockIdx.x / r.ranks;
    r.p.tokens[row] = (int32_t)drawn;
    if (r.p.probs) r.p.probs[row] = (float)__ddiv_rn((double)drawn_weight, (double)total);
  }
}

// The bins of a row's logits: bin = round(step (reference - v)) + kAhead or so,
// as the sum of a constant, v times -step and 1.5 * 2^23, whose last bits are
// the rounded whole number.  It never decreases as v falls; what lies above
// the bins is in bin 0, NaN and what lies below them in none (kCoarse or more).
struct Bins {
  float step, origin, lead, halvings;  // lead: the reference's place; halvings: of the weight, per bin
  __device__ __forceinline__ uint32_t of(float v) const {
    return (uint32_t)max((int)(__float_as_uint(__fmaf_rn(v, -step, origin)) - 0x4B400000u), 0);
  }
  __device__ __forceinline__ uint32_t of_key(uint32_t key) const { return of(value_of(key)); }
  // False where a range or reference has no such bins.
  __device__ __forceinline__ bool set(float reference, float range, double rate) {
    if (!(range > 0.0f && range < 1e30f && fabsf(reference) < 1e30f)) return false;
    step = __fdiv_rn((float)(kCoarse - 8), range);
    if (!(__fmul_rn(fabsf(reference), step) < 4194304.0f)) return false;  // the constant would lose the bins
    origin = __fadd_rn(__fmul_rn(reference, step), 12582912.0f + (float)kAhead);
    lead = __fmaf_rn(-reference, step, __fsub_rn(origin, 12582912.0f));
    halvings = __fdiv_rn((float)rate, step);
    return true;
  }
};

// Where the cuts lie in a histogram of counts, two bins per thread (c0, c1):
// starts[] are its prefix sums, *last the first bin by which every cut is met
// (kCoarse when none is): top_k tokens; top_p's share of `whole`, the sum of
// all weights, by the bins' least weights; or, without either, min_p's
// floor_bin.  *crowded: a bin up to it has more than kCrowd tokens.
template <typename T>
__device__ __forceinline__ void find_cuts(Row<T>& r, const Bins& bins, uint32_t c0, uint32_t c1, const Cuts& q, float share,
                                          float whole, float floor_bin, uint32_t* last, bool* crowded) {
  Shared& sh = r.sh;
  const int tid = r.tid, lane = r.lane, bin0 = 2 * tid;
  static_assert(kCoarse == 2 * kThreads, "a thread has two bins");
  // Counts and least weights up to each bin, both in one scan.
  const float w0 = __fmul_rn((float)c0, exp2_approx(__fmul_rn(bins.halvings, __fsub_rn(bins.lead, (float)bin0 + 0.52f))));
  const float w1 = __fmul_rn((float)c1, exp2_approx(__fmul_rn(bins.halvings, __fsub_rn(bins.lead, (float)bin0 + 1.52f))));
  uint32_t count = c0 + c1;
  float mass = __fadd_rn(w0, w1);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(kFull, count, o);
    const float b = __shfl_up_sync(kFull, mass, o);
    if (lane >= o) {
      count += a;
      mass = __fadd_rn(mass, b);
    }
  }
  __syncthreads();
  if (lane == 31) sh.warp_value[r.warp] = (unsigned long long)count << 32 | __float_as_uint(mass);
  if (tid == 0) sh.found[0] = kCoarse;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const unsigned long long o = sh.warp_value[i];
    if (i < r.warp) {
      count += (uint32_t)(o >> 32);
      mass = __fadd_rn(mass, __uint_as_float((uint32_t)o));
    }
  }
  sh.starts[bin0] = count - c0 - c1;
  sh.starts[bin0 + 1] = count - c1;
  if (tid == kThreads - 1) sh.starts[kCoarse] = count;
  const float past_p = __fmul_rn(__fmul_rn(share, whole), 1.0001f);
  const bool p_alone = q.by_p && !q.by_k;
  auto enough = [&](int bin, uint32_t c, float m) {
    return (q.by_k && c >= (uint32_t)q.top_k) || (p_alone && c > 0 && m >= past_p) || (!q.by_p && c > 0 && (float)bin >= floor_bin);
  };
  if (enough(bin0, count - c1, __fsub_rn(mass, w1)))
    atomicMin(&sh.found[0], (unsigned long long)bin0);
  else if (enough(bin0 + 1, count, mass))
    atomicMin(&sh.found[0], (unsigned long long)(bin0 + 1));
  __syncthreads();
  *last = (uint32_t)sh.found[0];
  *crowded = __syncthreads_or((bin0 <= (int)*last && c0 > kCrowd) || (bin0 + 1 <= (int)*last && c1 > kCrowd));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  T* x = reinterpret_cast<T*>(dyn + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31;
  const int slice = p.segment * kWarps, base = min(p.vocab, rank * slice), n = min(slice, p.vocab - base);
  if (tid < 64) sh.powers[tid] = exp2(-(double)tid / 64.0);
  for (int i = tid; i < kCoarse; i += kThreads) sh.counts[i] = sh.filled[i] = 0;
  if (tid == 0) sh.listed = 0;
  pdl_enter();

  // ---- the logits, once ----
  constexpr int kVec = 16 / (int)sizeof(T);
  const T* src = static_cast<const T*>(p.logits) + (long long)row * p.row_stride + base;
  const int vecs = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? n / kVec : 0;
  for (int i = tid; i < vecs; i += kThreads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(x + i * kVec)), "l"(src + i * kVec)
                 : "memory");
#pragma unroll 8
  for (int i = vecs * kVec + tid; i < n; i += kThreads) x[i] = src[i];
  for (int i = n + tid; i < (n + kVec - 1) / kVec * kVec; i += kThreads) x[i] = Logit<T>::none();
  const float temperature = p.temperature ? p.temperature[row] : 1.0f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.0f;
  const float min_p = p.min_p ? p.min_p[row] : 0.0f;
  const double u = fmin(fmax((double)p.uniform[row], 0.0), 1.0);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (p.candidates) {
    const uint32_t* mask = p.candidates + (long long)row * p.candidates_stride;
    for (int i = tid; i < n; i += kThreads)
      if (!(mask[(base + i) >> 5] >> ((base + i) & 31) & 1)) x[i] = Logit<T>::none();
    __syncthreads();
  }
  Row<T> r{p, sh, x, cluster, ranks, rank, base, n, tid, lane, tid >> 5, 0, 0};
  float most = -INFINITY, least = INFINITY;
  bool nan = false;
  r.each([&](float v, int) {
    most = fmaxf(most, v);
    least = fminf(least, v);
    nan |= v != v;
  });
  if (nan) flag_status(p.status, kStatusNonFinite);
  uint32_t key_max = key_of(__fadd_rn(most, 0.0f)), key_low = ~key_of(least);
  r.block_max2(key_max, key_low);
  r.publish(key_max, key_low);
  for (int i = 0; i < ranks; ++i) {
    key_max = max(key_max, (uint32_t)r.peer(i, 0));
    key_low = max(key_low, (uint32_t)r.peer(i, 1));
  }
  const float top = value_of(key_max);
  const bool refused = !(temperature >= 0.0f);
  if (refused || top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      if (refused) flag_status(p.status, kStatusBadIndex);
      p.tokens[row] = -1;
      if (p.probs) p.probs[row] = 0.0f;
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
    return;
  }
  if (temperature == 0.0f) {
    uint32_t id = kFull;
    r.each([&](float v, int i) {
      if (v == top) id = min(id, (uint32_t)(base + i));
    });
    uint32_t inverse = kFull - id, none = 0;
    r.block_max2(inverse, none);
    r.publish(inverse);
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < ranks; ++i) inverse = max(inverse, (uint32_t)r.peer(i, 0));
      p.tokens[row] = (int32_t)(kFull - inverse);
      if (p.probs) p.probs[row] = 1.0f;
    }
    cluster.sync();
    return;
  }
  const Weigher weigh(top, (double)temperature, sh.powers);
  const float reach = __fmul_rn(kReach, temperature), lowest = __fsub_rn(top, reach);  // below it weights vanish
  // near() holds: a temperature of 2^46 times what widen() loses of a subnormal
  // logit or more, and numbers to subtract
  const bool regular = top < INFINITY && temperature >= 8.2718061e-25f;
  const bool by_k = top_k > 0 && top_k < p.vocab, by_p = top_p < 1.0f, by_floor = min_p > 0.0f;
  const double floor_p = by_floor ? fmin((double)min_p, 1.0) : 0.0;
  const float share = fmaxf(top_p, 0.0f);

  // ---- the few that matter, in one CTA ----
  Bins bins;
  if ((by_k || by_p || by_floor) && regular &&
      bins.set(top, fminf(reach, __fsub_rn(top, value_of(~key_low))), weigh.rate)) {
    Cuts q{by_k, by_p, top_k, (double)share, floor_p, u, 0};
    unsigned long long whole = 0;
    if (by_p && !by_k) {
      r.each([&](float v, int) {
        const uint32_t b = bins.of(v);
        const unsigned long long w = weigh.fixed_near(v);
        if (b < kCoarse) {
          atomicAdd(&sh.counts[b], 1u);
          whole += w;
        }
      });
      whole = r.block_sum(whole);
    } else {
      r.each([&](float v, int) {
        const uint32_t b = bins.of(v);
        if (b < kCoarse) atomicAdd(&sh.counts[b], 1u);
      });
    }
    __syncthreads();
    r.publish(whole);
    uint32_t c0 = 0, c1 = 0;
    for (int i = 0; i < ranks; ++i) {
      const uint2 o = reinterpret_cast<const uint2*>(cluster.map_shared_rank(&sh, i)->counts)[tid];
      c0 += o.x;
      c1 += o.y;
      q.whole += r.peer(i, 0);
    }
    const float floor_bin = by_floor ? __fadd_rn(__fdiv_rn(-log2f((float)floor_p), bins.halvings), bins.lead + 3.0f) : 1e30f;
    uint32_t last;
    bool crowded;
    find_cuts(r, bins, c0, c1, q, share, __fmul_rn((float)q.whole, 1.0f / 1099511627776.0f), floor_bin, &last, &crowded);
    const uint32_t listed = last < kCoarse ? sh.starts[last + 1] : kList + 1;
    if (listed <= kList) {
      Shared* home = cluster.map_shared_rank(&sh, 0);
      r.each([&](float v, int i) {
        const uint32_t b = bins.of(v);
        if (b > last) return;
        v = __fadd_rn(v, 0.0f);
        const uint32_t slot = sh.starts[b] + atomicAdd(&home->filled[b], 1u);
        if (slot < kList) home->list[slot] = (unsigned long long)key_of(v) << 32 | (kFull - (uint32_t)(base + i));
      });
      cluster.sync();
      // the list holds every cut: the other CTAs, and for short lists the
      // other warps, are done
      if (rank != 0) return;
      auto bin_of_key = [&](uint32_t key) { return bins.of_key(key); };
      if (listed > kWarpList || crowded) {
        order_list<kThreads>(sh, (int)listed, crowded, tid, bin_of_key);
        finish_list<T, false>(r, weigh, q, (int)listed);
      } else if (tid < 32) {
        order_list<32>(sh, (int)listed, false, tid, bin_of_key);
        finish_list<T, true>(r, weigh, q, (int)listed);
      }
      return;
    }
  }

  // ---- the general way: top-k, then top-p ----
  // (an infinite logit less an infinite reach is no number: only its ties count)
  const uint32_t key_min = top == INFINITY ? key_max : max(kKeyNone + 1, key_of(__fsub_rn(top, reach)));
  auto fixed_weight = [&](float v, uint32_t k) -> unsigned long long {
    if (!regular) return Weigher::fixed(weigh.real(v, k));
    const unsigned long long w = weigh.fixed_near(v);
    return v >= lowest ? w : 0ull;
  };
  Cut cut{kKeyNone, -1};
  if (by_k) r.border(&cut, [](float, uint32_t) { return 1ull; }, top_k, top, reach, key_min, key_max, -1.0);
  if (by_p) r.border(&cut, fixed_weight, 0, top, reach, max(key_min, cut.key), key_max, (double)share);

  // ---- the draw from all ----
  auto weight = [&](float v, uint32_t k, int id) -> unsigned long long {
    if (!cut.holds(k, id)) return 0;
    if (by_floor && !(weigh.real(v, k) >= floor_p)) return 0;
    return fixed_weight(v, k);
  };
  const unsigned long long sum = r.segment_sum(weight);
  unsigned long long total;
  const unsigned long long before = r.prefix(sum, &total);
  // running > u * total  <=>  running > floor(u * total) for whole numbers
  unsigned long long target = (unsigned long long)floor(__dmul_rn(u, (double)total));
  if (target >= total) target = total - 1;
  const int id = r.locate(weight, before, before + sum, target);
  if (id >= 0 && tid == 0) {
    p.tokens[row] = id;
    const float v = r.at(id - base);
    if (p.probs) p.probs[row] = (float)__ddiv_rn((double)weight(v, key_of(v), id), (double)total);
  }
  cluster.sync();
}

// CTAs per row: slices of at most 8,192 logits keep four CTAs on an SM, so
// that the loads of some rows overlap the passes of others; a call with fewer
// rows than SMs spreads each over more.
int cluster_of(int rows, int vocab) {
  int c = 1;
  while (c < kMaxCluster && (vocab > c * 8192 || (rows * c * 2 <= kSms && vocab > c * 2048))) c *= 2;
  return c;
}

template <typename T>
cudaError_t launch_sample(SampleParams p, cudaStream_t s) {
  const int c = cluster_of(p.rows, p.vocab);
  p.segment = ((p.vocab + c * kWarps - 1) / (c * kWarps) + 31) / 32 * 32;
  const size_t fixed = (sizeof(Shared) + 15) / 16 * 16;
  const size_t smem = fixed + (size_t)p.segment * kWarps * sizeof(T);
  static uint64_t done = 0;
  const int most = (kMaxVocab + kMaxCluster * kWarps - 1) / (kMaxCluster * kWarps);
  cudaError_t e = allow_smem(sample_kernel<T>, fixed + (size_t)(most + 31) / 32 * 32 * kWarps * sizeof(T), &done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = c;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
}

}  // namespace
}  // namespace mc

extern "C" mc_status mc_sample(const mc_sample_args* a, void* stream) {
  if (!a) return MC_INVALID_INPUT;
  const int bytes = mc::dtype_bytes(a->dtype);
  if (bytes == 0 || a->rows < 0 || a->rows > (1 << 24) || a->vocab < 1 || a->vocab > mc::kMaxVocab) return MC_INVALID_INPUT;
  if (a->rows == 0) return MC_OK;
  if (!a->logits || reinterpret_cast<uintptr_t>(a->logits) % bytes != 0 || a->row_stride < 0 ||
      a->row_stride >= (int64_t(1) << 40) || !mc::aligned4(a->temperature) || !mc::aligned4(a->top_k) ||
      !mc::aligned4(a->top_p) || !mc::aligned4(a->min_p) || !a->uniform || !mc::aligned4(a->uniform) || !a->tokens ||
      !mc::aligned4(a->tokens) || !mc::aligned4(a->probs) || !mc::aligned4(a->candidates) ||
      (a->candidates && (a->candidates_stride < 0 || a->candidates_stride >= (int64_t(1) << 40))))
    return MC_INVALID_INPUT;
  const mc_status where = mc::on_current_device({a->logits, a->temperature, a->top_k, a->top_p, a->min_p, a->uniform,
                                                 a->candidates, a->tokens, a->probs});
  if (where != MC_OK) return where;
  mc::SampleParams p;
  std::memset(&p, 0, sizeof(p));
  p.logits = a->logits;
  p.row_stride = a->row_stride;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.uniform = a->uniform;
  p.candidates = a->candidates;
  p.candidates_stride = a->candidates_stride;
  p.tokens = a->tokens;
  p.probs = a->probs;
  p.rows = a->rows;
  p.vocab = a->vocab;
  p.status = mc::op_status_word();
  if (!p.status) return MC_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == MC_F32   ? mc::launch_sample<float>(p, s)
                        : a->dtype == MC_F16 ? mc::launch_sample<__half>(p, s)
                                             : mc::launch_sample<__nv_bfloat16>(p, s);
  return mc::launched(e);
}
