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
// above which bin all that can matter lies (the k-th logit, an estimate of
// top_p's border, min_p's floor); those tokens, seldom more than a few hundred, go
// to one CTA, which sorts them and finds the three cuts and the draw exactly.
// A row whose candidates do not fit its list, or whose estimate turns out too
// small, takes the general way: the border of a prefix of the order is "above
// a key, and so many ties of it", and histograms narrow the key's range,
// linear in the logits first and in their bit patterns from then on.
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
constexpr int kBins = 1024;
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
constexpr int kList = 2048;                 // candidates that one CTA sorts
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
  double top, rate;      // the largest logit; log2(e) / T
  uint32_t top_key;
  const double* powers;  // 2^-(j / 64)

  // w = 2^-((top - v) rate) in [0, 1]: 2^-(k / 64) from the table times the
  // exponential series of the rest, |rest| <= ln 2 / 128, to its fourth
  // power (the fifth is below 4e-14).  0 below 2^-42.
  __device__ __forceinline__ double real(float v, uint32_t key) const {
    if (key == top_key) return 1.0;
    const double y = __dmul_rn(__dsub_rn(top, widen(v)), rate);
    if (!(y < 42.0)) return 0.0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double t = __fma_rn(y, 64.0, magic);
    const int k = __double2loint(t);
    const double r = __fma_rn(__dsub_rn(t, magic), 0.015625, -y);  // k / 64 - y
    const double z = __dmul_rn(r, 0.69314718055994530942);
    double s = __fma_rn(z, 1.0 / 24, 1.0 / 6);
    s = __fma_rn(s, z, 0.5);
    s = __fma_rn(s, z, 1.0);
    s = __fma_rn(s, z, 1.0);
    const double p = __dmul_rn(powers[k & 63], s);
    return __hiloint2double(__double2hiint(p) - ((k >> 6) << 20), __double2loint(p));
  }
  static __device__ __forceinline__ unsigned long long fixed(double w) {
    // adding 2^12 leaves the 40 fraction bits at the end of the mantissa
    return (unsigned long long)__double_as_longlong(__dadd_rn(w, 4096.0)) & ((1ull << 51) - 1);
  }
};

// What the CTAs of a row tell one another; two of each, used in turn, so
// that one cluster barrier per exchange is enough.
struct Exchange {
  unsigned long long value[2][3];
};

struct Shared {
  union {
    unsigned long long hist[2][kBins];  // the general way
    unsigned long long list[kList];     // candidates: key, then ~id
  };
  uint32_t counts[kBins];
  uint32_t listed;
  double powers[64];
  Exchange out;
  unsigned long long warp_value[kWarps];
  unsigned long long found[3];
};

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(kFull, v, o);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ unsigned long long warp_prefix(unsigned long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long w = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += w;
  }
  return v;
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
  const T* x;  // this CTA's slice in shared memory
  cg::cluster_group cluster;
  int ranks, rank, base, n, tid, lane, warp, turn, level;

  // A logit as it orders: NaN is never drawn, -0 is 0.
  __device__ __forceinline__ float at(int i) const {
    const float v = Logit<T>::get(x[i]);
    return v == v ? __fadd_rn(v, 0.0f) : -INFINITY;
  }

  // ---- reductions over the row ----
  template <bool MAX>
  __device__ __forceinline__ unsigned long long block(unsigned long long v) {
    v = MAX ? warp_max(v) : warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.warp_value[warp] = v;
    __syncthreads();
    v = sh.warp_value[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const unsigned long long o = sh.warp_value[w];
      v = MAX ? (o > v ? o : v) : v + o;
    }
    return v;
  }
  // Publishes this CTA's values; afterwards peer(r, i) reads those of CTA r.
  __device__ __forceinline__ void publish(unsigned long long a, unsigned long long b, unsigned long long c) {
    turn ^= 1;
    if (tid == 0) {
      sh.out.value[turn][0] = a;
      sh.out.value[turn][1] = b;
      sh.out.value[turn][2] = c;
    }
    cluster.sync();
  }
  __device__ __forceinline__ unsigned long long peer(int r, int i) {
    return cluster.map_shared_rank(&sh, r)->out.value[turn][i];
  }

  // ---- the border of a prefix of the order ----
  // The first key (descending) at which the sum of f over the tokens of `in`
  // reaches target; *above is the sum over larger keys, *ties that over the
  // key itself.  Returns 0 when the whole sum does not reach target.
  template <typename F>
  __device__ uint32_t border(const Cut& in, F f, unsigned long long target, float top, float range, uint32_t key_min,
                             uint32_t key_max, unsigned long long* above, unsigned long long* ties,
                             unsigned long long* whole, double share) {
    uint32_t lo = key_min, hi = key_max;
    unsigned long long over = 0;
    // A first histogram linear in the logits, where they are spread out; its
    // bins are whole ranges of keys, as rounding keeps the order.
    const bool linear = range > 0.0f && range < INFINITY;
    const float step = linear ? __fdiv_rn((float)kBins * 0.999f, range) : 0.0f;
    auto bin_of = [&](float v) {
      return (int)fminf(__fmul_rn(__fsub_rn(top, v), step), (float)(kBins - 1));
    };
    int first_bin = -1;
    for (bool start = linear;; start = false) {
      unsigned long long* hist = sh.hist[level & 1];
      ++level;
      for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
      __syncthreads();
      int shift = 0;
      if (!start) {
        const uint32_t span = hi - lo;
        shift = span < kBins ? 0 : 32 - 10 - __clz(span);
      }
      const int begin = warp * p.segment, end = min(n, begin + p.segment);
      for (int i = begin + lane; i < end; i += 32) {
        const float v = at(i);
        const uint32_t k = key_of(v);
        if (k < lo || k > hi || !in.holds(k, base + i)) continue;
        int bin;
        if (start) {
          bin = bin_of(v);
        } else {
          if (first_bin >= 0 && bin_of(v) != first_bin) continue;
          bin = (int)((hi - k) >> shift);
        }
        const unsigned long long w = f(v, k);
        if (w) atomicAdd(&hist[bin], w);
      }
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
      if (share < 0.0 && total < target) return 0;  // every CTA of the row sees the same
      if (share >= 0.0) {  // the target is a share of the whole, known after the first pass
        target = (unsigned long long)ceil(__dmul_rn(share, (double)total));
        if (target < 1) target = 1;
        if (target > total) target = total;
        *whole = total;
        share = -1.0;
      }
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
      *ties = sh.found[2];
      __syncthreads();
      if (start) {
        first_bin = bin;
        // the keys of the bin, with a margin that covers the rounding of bin_of
        const float from = __fsub_rn(top, __fdiv_rn((float)bin - 0.01f, step));
        const float to = __fsub_rn(top, __fdiv_rn((float)bin + 1.01f, step));
        if (bin > 0) hi = min(hi, key_of(__fadd_rn(from, 0.0f)));
        if (bin < kBins - 1) lo = max(lo, key_of(__fadd_rn(to, 0.0f)));
      } else {
        hi -= (uint32_t)bin << shift;
        const uint32_t width = (1u << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
        if (shift == 0) break;
      }
    }
    *above = over;
    return hi;
  }

  // ---- the first id, ascending, at which a running sum exceeds a target ----
  // One warp's part of f over its segment.
  template <typename F>
  __device__ __forceinline__ unsigned long long segment_sum(F f) {
    unsigned long long s = 0;
    const int begin = warp * p.segment, end = min(n, begin + p.segment);
    for (int i = begin + lane; i < end; i += 32) {
      const float v = at(i);
      s += f(v, key_of(v), base + i);
    }
    return warp_sum(s);
  }
  // The id for a target in [before, before + the warp's sum); -1 elsewhere.
  template <typename F>
  __device__ int locate(F f, unsigned long long before, unsigned long long sum, unsigned long long target) {
    if (target < before || target >= before + sum) return -1;
    const int begin = warp * p.segment, end = min(n, begin + p.segment);
    for (int i = begin; i < end; i += 32) {
      unsigned long long w = 0;
      if (i + lane < end) {
        const float v = at(i + lane);
        w = f(v, key_of(v), base + i + lane);
      }
      const unsigned long long inc = before + warp_prefix(w, lane);
      const uint32_t past = __ballot_sync(kFull, inc > target);
      if (past) return base + i + __ffs(past) - 1;
      before = __shfl_sync(kFull, inc, 31);
    }
    return -1;
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
    publish(own, 0, 0);
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
    const int id = locate(one, before, sum, count - 1);
    const unsigned long long mine = block<true>(id >= 0 ? (unsigned long long)id + 1 : 0ull);
    publish(mine, 0, 0);
    unsigned long long best = 0;
    for (int r = 0; r < ranks; ++r) {
      const unsigned long long o = peer(r, 0);
      best = o > best ? o : best;
    }
    return (int)best - 1;
  }
};

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
  if (tid == 0) sh.listed = 0;
  for (int i = tid; i < kBins; i += kThreads) sh.counts[i] = 0;
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
  const float temperature = p.temperature ? p.temperature[row] : 1.0f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.0f;
  const float min_p = p.min_p ? p.min_p[row] : 0.0f;
  const double u = fmin(fmax((double)p.uniform[row], 0.0), 1.0);
  for (int i = n + tid; i < (n + kVec - 1) / kVec * kVec; i += kThreads) x[i] = Logit<T>::none();
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (p.candidates) {
    const uint32_t* mask = p.candidates + (long long)row * p.candidates_stride;
    for (int i = tid; i < n; i += kThreads)
      if (!(mask[(base + i) >> 5] >> ((base + i) & 31) & 1)) x[i] = Logit<T>::none();
    __syncthreads();
  }
  // One pass over the slice, 16 bytes at a time: f(logit, id).
  const int all_vecs = (n + kVec - 1) / kVec;
  auto each = [&](auto f) {
    for (int i = tid; i < all_vecs; i += kThreads) {
      const uint4 q = *reinterpret_cast<const uint4*>(x + i * kVec);
      T t[kVec];
      memcpy(t, &q, 16);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f(Logit<T>::get(t[j]), i * kVec + j);
    }
  };
  float most = -INFINITY, least = INFINITY;
  bool nan = false;
  each([&](float v, int) {
    most = fmaxf(most, v);
    least = fminf(least, v);
    nan |= v != v;
  });
  if (nan) flag_status(p.status, kStatusNonFinite);

  Row<T> r{p, sh, x, cluster, ranks, rank, base, n, tid, lane, tid >> 5, 0, 0};
  {
    const unsigned long long a = r.template block<true>(key_of(most)), b = r.template block<true>(~key_of(least) & kFull);
    r.publish(a, b, 0);
  }
  unsigned long long top_bits = 0, least_bits = 0;
  for (int i = 0; i < ranks; ++i) {
    const unsigned long long a = r.peer(i, 0), b = r.peer(i, 1);
    top_bits = a > top_bits ? a : top_bits;
    least_bits = b > least_bits ? b : least_bits;
  }
  const float top = __fadd_rn(value_of((uint32_t)top_bits), 0.0f);  // -0 is 0
  const uint32_t key_max = key_of(top);
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
    each([&](float v, int i) {
      if (v == top) id = min(id, (uint32_t)(base + i));
    });
    r.publish(r.template block<true>((unsigned long long)(kFull - id)), 0, 0);
    if (rank == 0 && tid == 0) {
      unsigned long long best = 0;
      for (int i = 0; i < ranks; ++i) {
        const unsigned long long o = r.peer(i, 0);
        best = o > best ? o : best;
      }
      p.tokens[row] = (int32_t)(kFull - (uint32_t)best);
      if (p.probs) p.probs[row] = 1.0f;
    }
    cluster.sync();
    return;
  }
  const Weigher weigh{(double)top, __ddiv_rn(1.4426950408889634074, (double)temperature), key_max, sh.powers};
  const double floor_w = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
  const float low = value_of(~(uint32_t)least_bits);
  const float range = fminf(__fmul_rn(kReach, temperature), __fsub_rn(top, low));
  const bool by_k = top_k > 0 && top_k < p.vocab, by_p = top_p < 1.0f;

  // ---- the few that matter, in one CTA ----
  if ((by_k || by_p || floor_w > 0.0) && range > 0.0f && range < 1e30f && top < INFINITY) {
    // bin = round(step (top - v)) + 1 or so: the sum of a constant, v times
    // -step and 1.5 * 2^23, whose last bits are the rounded whole number; it
    // never decreases as v falls.  NaN and what lies out of reach end above kBins.
    const float step = __fdiv_rn((float)(kBins - 8), range);
    const float origin = __fadd_rn(__fmul_rn(top, step), 12582912.0f + 2.0f);
    const bool binned = __fmul_rn(fabsf(top), step) < 4194304.0f;  // else the constant loses the bins
    if (binned) {
      auto bin_of = [&](float v) { return __float_as_uint(__fmaf_rn(v, -step, origin)) - 0x4B400000u; };
      unsigned long long whole = 0;
      const bool need_whole = by_p && !by_k;
      if (need_whole) {
        each([&](float v, int) {
          const uint32_t b = bin_of(v);
          if (b >= kBins) return;
          atomicAdd(&sh.counts[b], 1u);
          v = __fadd_rn(v, 0.0f);
          whole += Weigher::fixed(weigh.real(v, key_of(v)));
        });
        whole = r.template block<false>(whole);
      } else {
        each([&](float v, int) {
          const uint32_t b = bin_of(v);
          if (b < kBins) atomicAdd(&sh.counts[b], 1u);
        });
      }
      __syncthreads();
      r.publish(whole, 0, 0);
      constexpr int kPer = kBins / kThreads;
      static_assert(kPer == 4, "a thread's bins are one 16-byte load");
      uint32_t c[kPer] = {0, 0, 0, 0};
      whole = 0;
      for (int i = 0; i < ranks; ++i) {
        const uint4 o = reinterpret_cast<const uint4*>(cluster.map_shared_rank(&sh, i)->counts)[tid];
        c[0] += o.x;
        c[1] += o.y;
        c[2] += o.z;
        c[3] += o.w;
        whole += r.peer(i, 0);
      }
      // Counts and estimated weights up to each bin.
      const float bits = __fdiv_rn((float)weigh.rate, step);  // halvings per bin
      float w[kPer];
      uint32_t count = 0;
      float mass = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        w[j] = __fmul_rn((float)c[j], exp2f(__fmul_rn(-bits, (float)(tid * kPer + j - 2))));
        count += c[j];
        mass = __fadd_rn(mass, w[j]);
      }
      // both prefixes of the block in one scan: the count above, the estimate
      // (f32 bits) beside it
      uint32_t count_in = count;
      float mass_in = mass;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(kFull, count_in, o);
        const float b = __shfl_up_sync(kFull, mass_in, o);
        if (lane >= o) {
          count_in += a;
          mass_in = __fadd_rn(mass_in, b);
        }
      }
      if (lane == 31)
        sh.warp_value[tid >> 5] = (unsigned long long)count_in << 32 | __float_as_uint(mass_in);
      if (tid == 0) sh.found[0] = kBins;
      __syncthreads();
      uint32_t before = count_in - count, total = 0;
      float mass_before = __fsub_rn(mass_in, mass), mass_total = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const unsigned long long o = sh.warp_value[i];
        if (i < (tid >> 5)) {
          before += (uint32_t)(o >> 32);
          mass_before = __fadd_rn(mass_before, __uint_as_float((uint32_t)o));
        }
        total += (uint32_t)(o >> 32);
        mass_total = __fadd_rn(mass_total, __uint_as_float((uint32_t)o));
      }
      // The last bin that can matter: the first that satisfies any of the cuts.
      const float want = __fmul_rn(__fadd_rn(fmaxf(top_p, 0.0f), 0.01f), mass_total);
      const float floor_bin = floor_w > 0.0 ? __fadd_rn(__fdiv_rn(-log2f((float)floor_w), bits), 6.0f) : 1e30f;
      uint32_t last = kBins;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int bin = tid * kPer + j;
        before += c[j];
        mass_before = __fadd_rn(mass_before, w[j]);
        const bool enough = (by_k && before >= (uint32_t)top_k) || (need_whole && mass_before >= want) ||
                            (!by_p && (float)bin >= floor_bin);
        if (enough && last == kBins) last = bin;
      }
      atomicMin(reinterpret_cast<unsigned long long*>(&sh.found[0]), (unsigned long long)last);
      __syncthreads();
      last = min((uint32_t)sh.found[0], (uint32_t)kBins - 1);
      // how many tokens lie up to it
      if (tid == (int)last / kPer) {
        uint32_t up_to = before;
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j)
          if (tid * kPer + j > (int)last) up_to -= c[j];
        sh.found[1] = up_to;
      }
      __syncthreads();
      const uint32_t listed = (uint32_t)sh.found[1];
      if (listed <= kList) {
        Shared* home = cluster.map_shared_rank(&sh, 0);
        each([&](float v, int i) {
          if (bin_of(v) > last) return;
          const uint32_t slot = atomicAdd(&home->listed, 1u);
          v = __fadd_rn(v, 0.0f);
          if (slot < kList) home->list[slot] = (unsigned long long)key_of(v) << 32 | (kFull - (uint32_t)(base + i));
        });
        cluster.sync();
        int done = 0;
        if (rank == 0) {
          int n2 = 64;
          while (n2 < (int)listed) n2 <<= 1;
          for (int i = listed + tid; i < n2; i += kThreads) sh.list[i] = 0;
          __syncthreads();
          sort_list(sh.list, n2, tid);
          // thread i holds the sorted candidates kEach i .. kEach i + kEach - 1
          constexpr int kEach = kList / kThreads;
          const int first = tid * kEach;
          unsigned long long weight[kEach], sum = 0;
          uint32_t above_floor = 0;
          const int in_a = by_k ? min((int)listed, top_k) : (int)listed;
#pragma unroll
          for (int j = 0; j < kEach; ++j) {
            weight[j] = 0;
            if (first + j < in_a) {
              const uint32_t k = (uint32_t)(sh.list[first + j] >> 32);
              const double real = weigh.real(value_of(k), k);
              weight[j] = Weigher::fixed(real);
              above_floor += real >= floor_w;
            }
            sum += weight[j];
          }
          const unsigned long long in = warp_prefix(sum, lane);
          __syncthreads();
          if (lane == 31) sh.warp_value[tid >> 5] = in;
          __syncthreads();
          unsigned long long run = in - sum, all = 0;
#pragma unroll
          for (int i = 0; i < kWarps; ++i) {
            if (i < (tid >> 5)) run += sh.warp_value[i];
            all += sh.warp_value[i];
          }
          int in_c = in_a;
          bool covered = true;
          if (by_p) {
            const unsigned long long mass_a = by_k ? all : whole;
            unsigned long long border = (unsigned long long)ceil(__dmul_rn(fmax((double)top_p, 0.0), (double)mass_a));
            border = border < 1 ? 1 : border > mass_a ? mass_a : border;
            covered = all >= border;
            // those whose running sum before them is below the border
            uint32_t below = 0;
            unsigned long long s = run;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
              below += first + j < in_a && s < border;
              s += weight[j];
            }
            in_c = (int)r.template block<false>(below);
          }
          if (covered) {
            done = 1;
            in_c = min(in_c, (int)r.template block<false>(above_floor));
            sum = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
              if (first + j >= in_c) weight[j] = 0;
              sum += weight[j];
            }
            const unsigned long long total_c = r.template block<false>(sum);
            unsigned long long target = (unsigned long long)floor(__dmul_rn(u, (double)total_c));
            if (target >= total_c) target = total_c - 1;
            // The first id at which the running sum passes target: 256 ranges
            // of ids at a time, by their weights.
            uint32_t from = 0;
            int shift = max(0, 32 - 8 - __clz((uint32_t)p.vocab));
            unsigned long long drawn = 0;
            for (;; shift = max(0, shift - 8)) {
              unsigned long long* ranges = reinterpret_cast<unsigned long long*>(sh.counts);  // 256 of them
              ranges[tid] = 0;
              __syncthreads();
#pragma unroll
              for (int j = 0; j < kEach; ++j)
                if (weight[j]) {
                  const uint32_t id = kFull - (uint32_t)sh.list[first + j];
                  const uint32_t at = (id - from) >> shift;
                  if (id >= from && at < 256) atomicAdd(&ranges[at], weight[j]);
                }
              __syncthreads();
              const unsigned long long mine = ranges[tid], inc = warp_prefix(mine, lane);
              if (lane == 31) sh.warp_value[tid >> 5] = inc;
              __syncthreads();
              unsigned long long start = inc - mine;
#pragma unroll
              for (int i = 0; i < kWarps; ++i)
                if (i < (tid >> 5)) start += sh.warp_value[i];
              if (start <= target && target < start + mine) {
                sh.found[0] = tid;
                sh.found[1] = start;
                sh.found[2] = mine;
              }
              __syncthreads();
              from += (uint32_t)sh.found[0] << shift;
              target -= sh.found[1];
              drawn = sh.found[2];
              __syncthreads();
              if (shift == 0) break;
            }
            if (tid == 0) {
              p.tokens[row] = (int32_t)from;
              if (p.probs) p.probs[row] = (float)__ddiv_rn((double)drawn, (double)total_c);
            }
          }
        }
        if (!need_whole) return;  // nothing was estimated: the list holds every cut
        // every CTA learns whether the list reached top_p's border
        r.publish(done, 0, 0);
        done = (int)r.peer(0, 0);
        cluster.sync();
        if (done) return;
      }
    }
  }

  // ---- the general way: top-k, then top-p ----
  const uint32_t key_min = max(kKeyNone + 1, key_of(__fsub_rn(top, __fmul_rn(kReach, temperature))));
  Cut cut{kKeyNone, -1};
  unsigned long long above, ties, whole;
  if (by_k) {
    auto one = [](float, uint32_t) -> unsigned long long { return 1; };
    const uint32_t key = r.border(cut, one, top_k, top, range, key_min, key_max, &above, &ties, &whole, -1.0);
    if (key) {
      const unsigned long long kept = (unsigned long long)top_k - above;
      cut.last = kept < ties ? r.nth_tie(cut, key, kept) : INT32_MAX;
      cut.key = key;
    }
  }
  if (by_p) {
    auto mass = [&](float v, uint32_t k) { return Weigher::fixed(weigh.real(v, k)); };
    const uint32_t key = r.border(cut, mass, 0, top, range, max(key_min, cut.key), key_max, &above, &ties, &whole,
                                  fmax((double)top_p, 0.0));
    unsigned long long target = (unsigned long long)ceil(__dmul_rn(fmax((double)top_p, 0.0), (double)whole));
    target = target < 1 ? 1 : target > whole ? whole : target;
    const unsigned long long w = mass(value_of(key), key);
    const unsigned long long kept = (target - above + w - 1) / w;
    const int last = kept * w < ties ? r.nth_tie(cut, key, kept) : (key == cut.key ? cut.last : INT32_MAX);
    cut.key = key;
    cut.last = last;
  }

  // ---- the draw ----
  auto weight = [&](float v, uint32_t k, int id) -> unsigned long long {
    if (!cut.holds(k, id)) return 0;
    const double w = weigh.real(v, k);
    return w >= floor_w ? Weigher::fixed(w) : 0ull;
  };
  const unsigned long long sum = r.segment_sum(weight);
  unsigned long long total;
  const unsigned long long before = r.prefix(sum, &total);
  // running > u * total  <=>  running > floor(u * total) for whole numbers
  unsigned long long target = (unsigned long long)floor(__dmul_rn(u, (double)total));
  if (target >= total) target = total - 1;
  const int id = r.locate(weight, before, sum, target);
  if (id >= 0 && lane == 0) {
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
  while (c < kMaxCluster && (vocab > c * 8192 || (rows * c * 2 <= 148 && vocab > c * 2048))) c *= 2;
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
  mc_status where = mc::on_current_device(a->logits);
  if (where == MC_OK) where = mc::on_current_device(a->tokens);
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
  return e == cudaSuccess ? MC_OK : MC_CUDA;
}
