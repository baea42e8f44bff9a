// kv4.cu -- a paged key/value cache held in 4 bits: rows quantized into it,
// read back from it, and attention over it.
//
// A row x of head_dim values is held as minimum = f16(min x), scale =
// f16((max x - minimum) / 15) and codes c = round((x - minimum) / scale).  With
// middle = minimum + 8 scale
//   q . k_j      = scale_j (q . (c_j - 8)) + middle_j sum(q)
//   sum_j w_j v_j = sum_j (w_j scale_j) (c_j - 8) + sum_j w_j middle_j:
// both products of an attention run on the codes themselves, and scale and
// minimum enter once per row, not once per value.  Taking the codes about
// their middle matters: about the minimum, rows of mean zero would come out
// as the difference of two sums tens of times their size (measured: f32
// outputs 9e-6 off instead of 2e-7).
#include <cstring>
#include <type_traits>

#include "decode_ops.cuh"

namespace mc {
namespace {

constexpr uint32_t kFull = 0xFFFFFFFFu;

struct Kv4Pool {
  uint8_t* pages;
  const int32_t* table;
  long long n_pages;
  int token_shift;  // log2 page_tokens
  int kv_heads, head_dim, batch, per_seq;
};

// Bytes of one head's part of a page.
__host__ __device__ __forceinline__ int head_block(int tokens, int head_dim) { return tokens * (head_dim + 8); }

// ---- append and read ---------------------------------------------------------------
// A CTA takes up to 32 tokens of a sequence.  A group of L lanes (the power of
// two that holds head_dim / 8 lanes of 8 values) takes a head's key or value
// rows, token after token, page by page, four rows in flight.  Bound by its
// instructions: about 150 for a lane's eight values, of which the codes are 50.
// Measured, 131k rows of 8 heads of 128, bf16, keys and values: quantized in
// 300 us, read back in 125 (4.9 TB/s); with the page looked up for every row
// 446 and 129, with scalar arithmetic and a page lookup per row 690 and 190.
struct Kv4RowsDev {
  void *k, *v;
  const int32_t *start, *count, *first;
  long long rows;
  long long k_rs, k_hs, v_rs, v_hs;
  int max_count;
};

constexpr int kRowThreads = 256;
constexpr int kRowTokens = 32;
constexpr int kRowsInFlight = 4;

// Eight neighbouring values of a row, as they lie in memory.
template <int TYPE>
struct Eight {
  uint32_t w[TYPE == MC_F32 ? 8 : 4];
  __device__ __forceinline__ void load(const char* x) {
#pragma unroll
    for (int i = 0; i < (TYPE == MC_F32 ? 2 : 1); ++i) {
      const uint4 a = __ldcs(reinterpret_cast<const uint4*>(x) + i);
      w[4 * i] = a.x;
      w[4 * i + 1] = a.y;
      w[4 * i + 2] = a.z;
      w[4 * i + 3] = a.w;
    }
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = TYPE == MC_F32   ? make_float2(__uint_as_float(w[(2 * i) % (TYPE == MC_F32 ? 8 : 4)]),
                                                      __uint_as_float(w[(2 * i + 1) % (TYPE == MC_F32 ? 8 : 4)]))
                       : TYPE == MC_F16 ? unpack_f16(w[i])
                                        : unpack_bf16(w[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
};

template <int TYPE>
__device__ __forceinline__ void store_eight(char* x, const float (&f)[8]) {
  if (TYPE == MC_F32) {
    __stcs(reinterpret_cast<float4*>(x), make_float4(f[0], f[1], f[2], f[3]));
    __stcs(reinterpret_cast<float4*>(x) + 1, make_float4(f[4], f[5], f[6], f[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = TYPE == MC_F16 ? pack_f16(f[2 * i], f[2 * i + 1]) : pack_bf16(f[2 * i], f[2 * i + 1]);
    __stcs(reinterpret_cast<uint4*>(x), make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// The smallest and largest of the row's values over L lanes; smallest -inf
// when one of them is not finite (0 x it is NaN then).
template <int TYPE, int L>
__device__ __forceinline__ void row_range(const Eight<TYPE>& x, bool live, float* low, float* high) {
  if (TYPE == MC_F32) {
    float lo = INFINITY, hi = -INFINITY, z = 0.0f;
    if (live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = __uint_as_float(x.w[i % (TYPE == MC_F32 ? 8 : 4)]);
        lo = fminf(lo, f);
        hi = fmaxf(hi, f);
        z = __fmaf_rn(f, 0.0f, z);
      }
      if (z != z) lo = -INFINITY;
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
    }
    *low = lo;
    *high = hi;
  } else {
    // both at once: the 16-bit pair (smallest, -largest), whose minimum is taken
    using T2 = typename std::conditional<TYPE == MC_F16, __half2, __nv_bfloat162>::type;
    auto as2 = [](uint32_t w) { return *reinterpret_cast<T2*>(&w); };
    auto bits = [](T2 v) { return *reinterpret_cast<uint32_t*>(&v); };
    const uint32_t inf = TYPE == MC_F16 ? 0x7C007C00u : 0x7F807F80u;
    uint32_t both = inf;
    if (live) {
      T2 lo = as2(x.w[0]), hi = lo, z = __hmul2(lo, as2(0u));
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        lo = __hmin2(lo, as2(x.w[i]));
        hi = __hmax2(hi, as2(x.w[i]));
        z = __hfma2(as2(x.w[i]), as2(0u), z);
      }
      const uint32_t l = bits(lo), h = bits(hi) ^ 0x80008000u;
      // (low halves, high halves) of both, then their minimum
      both = bits(__hmin2(as2(__byte_perm(l, h, 0x5410)), as2(__byte_perm(l, h, 0x7632))));
      const uint32_t zb = bits(z) & 0x7FFF7FFFu;
      if (zb) both = inf | 0x80008000u;  // a NaN there, as 0 x finite has no bits left: (-inf, -inf)
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) both = bits(__hmin2(as2(both), as2(__shfl_xor_sync(kFull, both, o))));
    const float2 t = TYPE == MC_F16 ? unpack_f16(both) : unpack_bf16(both);
    *low = t.x;
    *high = -t.y;
  }
}

// The codes of eight values: round((x - minimum) / scale) of the real
// quotient.  A single-precision quotient is within 3e-6 of it for codes up to
// 16, so only one that lands within 1e-5 of a half needs the double-precision
// one, whose ties are exact (the scale has 11 significant bits).  Rounding is
// the addition of 1.5 * 2^23; six codes are one exact float.
__device__ __forceinline__ uint32_t codes_of(const float (&f)[8], float minimum, float scale) {
  const float inverse = __frcp_rn(scale);
  const uint64_t minus = pair(-minimum, -minimum), times = pair(inverse, inverse), magic = pair(12582912.0f, 12582912.0f);
  uint64_t c[4];
  float off = 0.0f;  // how far the quotients are from whole numbers, at most
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    unpair(mul2(add2(pair(f[2 * i], f[2 * i + 1]), minus), times), a, b);
    const uint64_t t = pair(fminf(fmaxf(a, 0.0f), 15.0f), fminf(fmaxf(b, 0.0f), 15.0f));
    c[i] = add2(add2(t, magic), pair(-12582912.0f, -12582912.0f));
    unpair(fma2(c[i], pair(-1.0f, -1.0f), t), a, b);
    off = fmaxf(off, fmaxf(fabsf(a), fabsf(b)));
  }
  if (off > 0.49999f) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      float x = f[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) x = i == j ? f[j] : x;
      const float r = (float)fmin(fmax(rint(__ddiv_rn(__dsub_rn((double)x, (double)minimum), (double)scale)), 0.0), 15.0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a, b;
        unpair(c[j], a, b);
        c[j] = pair(i == 2 * j ? r : a, i == 2 * j + 1 ? r : b);
      }
    }
  }
  const uint64_t p256 = pair(256.0f, 256.0f);
  float even, odd, c6, c7;
  unpair(fma2(fma2(c[2], p256, c[1]), p256, c[0]), even, odd);
  unpair(c[3], c6, c7);
  return (uint32_t)__fmaf_rn(odd, 16.0f, even) | (uint32_t)__fmaf_rn(c7, 16.0f, c6) << 24;
}

template <int TYPE, int L, bool READ>
__global__ void __launch_bounds__(kRowThreads, 3) kv4_rows_kernel(const Kv4Pool p, const Kv4RowsDev r, int chunks,
                                                               uint32_t* status) {
  pdl_enter();
  const int b = blockIdx.x / chunks, chunk = blockIdx.x - b * chunks;
  const int count = r.count[b], start = r.start[b], first = r.first[b];
  const long long capacity = (long long)p.per_seq << p.token_shift;
  if (count < 0 || count > r.max_count || start < 0 || (long long)start + count > r.rows || first < 0 ||
      (long long)first + count > capacity) {
    if (chunk == 0 && threadIdx.x == 0) flag_status(status, kStatusBadIndex);
    return;
  }
  const int t0 = chunk * kRowTokens, nt = min(kRowTokens, count - t0);
  if (nt <= 0) return;
  const int d = p.head_dim, lane = threadIdx.x % L, group = threadIdx.x / L, tokens = 1 << p.token_shift;
  constexpr int kGroups = kRowThreads / L, kBytes = TYPE == MC_F32 ? 4 : 2;
  const bool active = lane * 8 < d;
  const long long block_bytes = head_block(tokens, d);
  const int32_t* table = p.table + (long long)b * p.per_seq;
  bool bad = false, bad_page = false;
  for (int pair0 = 0; pair0 < 2 * p.kv_heads; pair0 += kGroups) {
    const int h = (pair0 + group) >> 1, which = group & 1;
    const bool mine = h < p.kv_heads && active;
    const long long rs = (which ? r.v_rs : r.k_rs) * kBytes;
    char* x0 = static_cast<char*>(which ? r.v : r.k) + (start + t0) * rs + (h * (which ? r.v_hs : r.k_hs) + lane * 8) * kBytes;
    // The rows that lie in one page follow one another in it.
    for (int t = 0, run; t < nt; t += run) {
      const int pos = first + t0 + t, in_page = pos & (tokens - 1);
      run = min(tokens - in_page, nt - t);
      const long long page = table[pos >> p.token_shift];
      if (page < 0 || page >= p.n_pages) {
        bad_page = true;
        continue;
      }
      uint8_t* block = p.pages + (page * p.kv_heads + h) * block_bytes;
      uint8_t* codes = block + (which * tokens + in_page) * (d / 2) + lane * 4;
      __half2* pairs = reinterpret_cast<__half2*>(block + tokens * d) + which * tokens + in_page;
      char* from = x0 + t * rs;
      for (int done = 0; done < run; done += kRowsInFlight) {
        Eight<TYPE> x[kRowsInFlight];
        uint32_t word[kRowsInFlight];
        __half2 pair[kRowsInFlight];
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
          if (!mine || done + u >= run) continue;
          if (READ) {
            word[u] = __ldcs(reinterpret_cast<const uint32_t*>(codes + u * (d / 2)));
            pair[u] = pairs[u];
          } else {
            x[u].load(from + u * rs);
          }
        }
#pragma unroll
        for (int u = 0; u < kRowsInFlight; ++u) {
          const bool live = mine && done + u < run;
          float f[8];
          if (READ) {
            if (!live) continue;
            const float scale = __low2float(pair[u]), minimum = __high2float(pair[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __fmaf_rn(scale, (float)((word[u] >> (4 * i)) & 15), minimum);
            store_eight<TYPE>(from + u * rs, f);
          } else {
            float low, high;
            row_range<TYPE, L>(x[u], live, &low, &high);
            if (!live) continue;
            __half min_h = __float2half_rn(low);
            __half scale_h = __float2half_rn(__fmul_rn(__fsub_rn(high, __half2float(min_h)), 1.0f / 15.0f));
            uint32_t w = 0;
            if (__hisinf(min_h) || __hisinf(scale_h) || __hisnan(scale_h)) {
              bad = true;
              min_h = scale_h = __float2half_rn(0.0f);
            } else if (__half2float(scale_h) > 0.0f) {
              x[u].values(f);
              w = codes_of(f, __half2float(min_h), __half2float(scale_h));
            }
            *reinterpret_cast<uint32_t*>(codes + u * (d / 2)) = w;
            if (lane == 0) pairs[u] = __halves2half2(scale_h, min_h);
          }
        }
        codes += kRowsInFlight * (d / 2);
        pairs += kRowsInFlight;
        from += kRowsInFlight * rs;
      }
    }
  }
  if (bad) flag_status(status, kStatusNonFinite);
  if (bad_page) flag_status(status, kStatusBadIndex);
}

// ---- attention ------------------------------------------------------------------------
// One warp per unit (sequence, key/value head, NT tiles of query columns) and
// key range, four warps per CTA.  A warp streams its keys 32 at a time
// through a private ring: each page's part for the head is contiguous, so a
// tile is 1, 2 or 4 bulk copies that complete on the stage's mbarrier.
//
// Both products are m16n8k16 with the codes as the row operand:
//   S^T [16 tokens x 8 queries]    = K codes [16 x 16 channels] . Q^T
//   O^T [16 channels x 8 queries] += V codes^T [16 x 16 tokens] . W^T
// so one query wastes 7 of 8 columns, not 15 of 16 rows.  A nibble c or-ed
// into the low mantissa bits of 1024.0 is the f16 1024 + c, and one packed
// subtraction makes c - 8 of it, exactly: two operands for an AND-OR and a
// subtraction, with no conversion.  Nibbles one place up give 16 (c - 8),
// which q (a sixteenth of it) or the output takes back.
//
// q is scaled by a power of two to below 2^9 (exact for 16-bit types, but for
// elements 2^20 and more below the row's largest; f32 is two f16 parts in the
// columns 0-3 and 4-7 of a tile, 22 bits).  The weights
// meet the values as w = p * scale_v in f16 (f32: two parts, again by
// columns), so the running maximum is taken over x_j + exponent(scale_v_j),
// which keeps w below 2^11 whatever the scales are; the sums of p and of
// p * middle_v are f32.
//
// Bound by the integer pipe where caches are long (64% busy: an AND-OR for two
// operands, a byte permute for four) and by set-up and output where they are
// short.  Measured: 8 x 65,536 keys, 8 heads of 128 with 4 queries each, bf16,
// 186 us (3.1 TB/s of 4-bit rows; 201 us with four stages, whose memory leaves
// three CTAs per SM, 198 with five CTAs' registers); 1,024 single tokens over
// 30 keys on average, 8 heads of 64, f32, 28 us.
struct Kv4AttnParams {
  Kv4Pool pool;
  AttnRows rows;
  AttnSplit split;
  float scale;
  int row_tiles, warps_log2;  // column tiles per (sequence, head); log2 warps per unit
  uint32_t units;
  uint32_t* status;
};

constexpr int kAttnWarps = 4;
constexpr int kAttnStages = 2;
constexpr int kTileKeys = 32;

__host__ __device__ constexpr int stage_bytes(int d) { return kTileKeys * (d + 8); }
// CTAs per SM that the registers are kept to.
constexpr int attn_blocks(int nt) { return nt == 1 ? 4 : 3; }
__host__ __device__ constexpr int attn_smem(int d) {
  return kAttnWarps * kAttnStages * (stage_bytes(d) + 16);
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// c - 8 of the low nibble of each 16-bit half, and 16 (c - 8) of the next.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
  const uint32_t x = (w & 0x000F000Fu) | 0x64006400u;
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6408)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) {
  const uint32_t x = (w & 0x00F000F0u) | 0x64006400u;
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// floor(log2 |v|) of an f16 value that is held in f32, where f16's subnormals
// are normal; -24, the smallest one's, for 0.
__device__ __forceinline__ float half_exponent(float v) {
  return (float)max((int)((__float_as_uint(v) >> 23) & 255) - 127, -24);
}

template <int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(kAttnWarps * 32, attn_blocks(NT)) kv4_attn_kernel(const Kv4AttnParams p) {
  constexpr int kCols = SPLIT ? 4 : 8;  // queries of a column tile
  constexpr int kQ = kCols * NT;
  constexpr int kSteps = D / 16;        // k16 steps of a score, m16 tiles of the output
  constexpr int kStage = stage_bytes(D);
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kAttnStages * kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kAttnWarps * kAttnStages * kStage) + warp * kAttnStages;
  uint32_t* valid =
      reinterpret_cast<uint32_t*>(smem + kAttnWarps * kAttnStages * (kStage + 8)) + warp * kAttnStages;
  if (lane == 0) {
    for (int i = 0; i < kAttnStages; ++i) mbar_init(&bars[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_enter();

  const AttnRows& r = p.rows;
  const int dtype = SPLIT ? (int)MC_F32 : r.dtype;
  const int wpu = 1 << p.warps_log2, sub = warp & (wpu - 1);
  const uint32_t unit = blockIdx.x * (kAttnWarps >> p.warps_log2) + (warp >> p.warps_log2);
  const int split = blockIdx.y;
  bool live = unit < p.units;
  int b = 0, head = 0, tile = 0;
  if (live) {
    const uint32_t bh = share(unit, (uint32_t)p.row_tiles);
    tile = (int)(unit - bh * p.row_tiles);
    b = (int)share(bh, (uint32_t)r.kv_heads);
    head = (int)(bh - (uint32_t)b * r.kv_heads);
  }
  AttnSeq seq = {0, 0, 0, 0, false};
  if (live) seq = attn_seq(r, b, p.status, head == 0 && tile == 0 && split == 0 && sub == 0 && lane == 0);
  const int n_rows = seq.nq * r.group, row0 = tile * kQ;
  live = live && row0 < n_rows;
  // The keys that the unit's last query sees, and this warp's tiles of them.
  const int pos_last = live ? min(seq.nq - 1, (int)share((uint32_t)(row0 + kQ - 1), (uint32_t)r.group)) : 0;
  const int pos_first = live ? (int)share((uint32_t)row0, (uint32_t)r.group) : 0;
  const int keys = live ? max(0, r.causal ? seq.nk - (seq.nq - 1 - pos_last) : seq.nk) : 0;
  const int keys_all = live ? max(0, r.causal ? seq.nk - (seq.nq - 1 - pos_first) : seq.nk) : 0;  // seen by every query
  const int splits_here = !live                 ? 0
                          : p.split.splits == 1 ? 1
                                                : max(1, ((seq.nk + kTileKeys - 1) / kTileKeys + p.split.chunk - 1) / p.split.chunk);
  live = live && split < splits_here;
  const int n_tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int lo = min(n_tiles, split * p.split.chunk), hi = min(n_tiles, lo + p.split.chunk);
  const int per = (hi - lo + wpu - 1) >> p.warps_log2;
  const int begin = live ? min(hi, lo + sub * per) : 0, end = live ? min(hi, begin + per) : 0;

  // ---- q: this lane's channels of column g ----
  const int col = SPLIT ? (g & 3) : g;
  uint32_t qb[NT][kSteps][2];
  float q_fac[NT][2], q_sum[NT][2];  // of the lane's columns 2t, 2t + 1
  int limit[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = row0 + n * kCols + col;
    const bool there = live && row < n_rows;
    const int pos = there ? (int)share((uint32_t)row, (uint32_t)r.group) : 0, h = head * r.group + (there ? row - pos * r.group : 0);
    const char* src = static_cast<const char*>(r.q) +
                      ((long long)(seq.q0 + pos) * r.q_row_stride + (long long)h * r.q_head_stride) *
                          (SPLIT ? 4 : 2);
    // words t * (D / 32) + c of the whole 32-channel blocks, then the tail's four channels
    float f[kSteps * 4];
    constexpr int kWhole = (D / 32) * 8;
#pragma unroll
    for (int i = 0; i < kSteps * 4; i += 2) {
      const int ch = i < kWhole ? t * kWhole + i : (D / 32) * 32 + 4 * t + i - kWhole;
      const float2 v = there ? load2(src, ch, dtype) : make_float2(0.0f, 0.0f);
      f[i] = v.x;
      f[i + 1] = v.y;
    }
    float amax = 0.0f, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps * 4; ++i) {
      amax = fmaxf(amax, fabsf(f[i]));
      sum = __fadd_rn(sum, f[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, o));
      sum = __fadd_rn(sum, __shfl_xor_sync(kFull, sum, o));
    }
    // 2^(8 - exponent(amax)) as a bit pattern, for any finite amax; tiny rows
    // keep a finite factor.
    const int e = min(max((int)((__float_as_uint(amax) >> 23) & 255) - 127, -110), 127);
    const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
    const float down = __uint_as_float((uint32_t)(127 - 8 + e) << 23);
    auto part = [&](float a, float b2, float m) -> uint32_t {
      const float x = __fmul_rn(a, __fmul_rn(up, m)), y = __fmul_rn(b2, __fmul_rn(up, m));
      const uint32_t w = pack_f16(x, y);
      if (!SPLIT || g < 4) return w;
      const float2 hi2 = unpack_f16(w);
      return pack_f16(__fsub_rn(x, hi2.x), __fsub_rn(y, hi2.y));
    };
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      qb[n][2 * c][0] = part(f[8 * c + 0], f[8 * c + 4], 1.0f);
      qb[n][2 * c][1] = part(f[8 * c + 1], f[8 * c + 5], 0.0625f);
      qb[n][2 * c + 1][0] = part(f[8 * c + 2], f[8 * c + 6], 1.0f);
      qb[n][2 * c + 1][1] = part(f[8 * c + 3], f[8 * c + 7], 0.0625f);
    }
    if (D % 32) {
      qb[n][kSteps - 1][0] = part(f[kWhole + 0], f[kWhole + 2], 1.0f);
      qb[n][kSteps - 1][1] = part(f[kWhole + 1], f[kWhole + 3], 0.0625f);
    }
    const float c2 = __fmul_rn(p.scale, kLog2e);
    const float fac = __fmul_rn(down, c2), qs = __fmul_rn(sum, c2);
    const int lim = there ? max(0, r.causal ? seq.nk - (seq.nq - 1 - pos) : seq.nk) : 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int from = (SPLIT ? ((2 * t + j) & 3) : 2 * t + j) * 4;
      q_fac[n][j] = __shfl_sync(kFull, fac, from);
      q_sum[n][j] = __shfl_sync(kFull, qs, from);
      limit[n][j] = __shfl_sync(kFull, lim, from);
    }
  }

  // ---- the ring ----
  const int tokens = 1 << p.pool.token_shift, blocks = kTileKeys >> p.pool.token_shift;
  const uint32_t block_bytes = (uint32_t)head_block(tokens, D);
  const int n_blocks = (keys + tokens - 1) >> p.pool.token_shift;
  const int32_t* table = p.pool.table + (long long)b * p.pool.per_seq;
  int ids = -1, ids_at = -1000;
  auto issue = [&](int tl) {
    const int s = (tl - begin) % kAttnStages, blk = tl * blocks;
    if (ids_at < 0 || blk + blocks > ids_at + 32) {
      ids_at = blk;
      ids = blk + lane < n_blocks ? table[blk + lane] : -1;
    }
    const int id = __shfl_sync(kFull, ids, (blk - ids_at + lane) & 31);
    const bool want = lane < blocks && blk + lane < n_blocks;
    const bool ok = want && id >= 0 && id < p.pool.n_pages;
    const uint32_t mask = __ballot_sync(kFull, ok);
    if (want && !ok) flag_status(p.status, kStatusBadIndex);
    if (lane == 0) {
      valid[s] = mask;
      mbar_arrive_expect_tx(&bars[s], __popc(mask) * block_bytes);
    }
    __syncwarp();
    if (ok)
      bulk_load(ring + s * kStage + lane * block_bytes,
                p.pool.pages + ((long long)id * p.pool.kv_heads + head) * block_bytes, block_bytes, &bars[s]);
  };
  for (int tl = begin; tl < min(end, begin + kAttnStages); ++tl) issue(tl);

  // Row g of a score tile is token (g / 2) + 4 (g % 2): the value product then
  // finds its neighbouring pairs (2t, 2t + 1) in tokens t and t + 4, whose
  // rows lie in different banks.
  const int tok = (g >> 1) + 4 * (g & 1);
  auto block_of = [&](int i) { return (uint32_t)(i >> p.pool.token_shift) * block_bytes; };
  auto slot_of = [&](int i) { return (uint32_t)(i & (tokens - 1)); };

  float top[NT][2], sum_p[NT][2], sum_m[NT][2];
  float acc[NT][kSteps][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      top[n][j] = -INFINITY;
      sum_p[n][j] = sum_m[n][j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][i][j] = 0.0f;
  }

  bool broken = false;
  for (int tl = begin; tl < end; ++tl) {
    const int s = (tl - begin) % kAttnStages;
    if (!mbar_wait(&bars[s], ((tl - begin) / kAttnStages) & 1, p.status)) {
      // Let the copies of the other stages land before the block leaves.
      for (int k = tl + 1; k < min(end, tl + kAttnStages); ++k)
        mbar_wait(&bars[(k - begin) % kAttnStages], ((k - begin) / kAttnStages) & 1, p.status);
      broken = true;
      break;
    }
    const uint8_t* st = ring + s * kStage;
    const int key0 = tl * kTileKeys;
    const uint32_t here = valid[s];
    const bool masked = key0 + kTileKeys > keys_all || here != (1u << blocks) - 1u;

    // ---- scores, tokens 16 m + tok (+ 8) ----
    float x[NT][2][4];
    uint32_t vpair[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[n][m][j] = 0.0f;
      const uint32_t i0 = 16 * m + tok, i1 = i0 + 8;
      const uint8_t* k0 = st + block_of(i0) + slot_of(i0) * (D / 2);
      const uint8_t* k1 = st + block_of(i1) + slot_of(i1) * (D / 2);
      constexpr int kWords = D / 32;
      uint32_t w0[kWords + 1], w1[kWords + 1];
      if (D == 128) {
        const uint4 a = *reinterpret_cast<const uint4*>(k0 + 16 * t), c = *reinterpret_cast<const uint4*>(k1 + 16 * t);
        w0[0] = a.x; w0[1 % (kWords + 1)] = a.y; w0[2 % (kWords + 1)] = a.z; w0[3 % (kWords + 1)] = a.w;
        w1[0] = c.x; w1[1 % (kWords + 1)] = c.y; w1[2 % (kWords + 1)] = c.z; w1[3 % (kWords + 1)] = c.w;
      } else if (D == 64) {
        const uint2 a = *reinterpret_cast<const uint2*>(k0 + 8 * t), c = *reinterpret_cast<const uint2*>(k1 + 8 * t);
        w0[0] = a.x; w0[1 % (kWords + 1)] = a.y;
        w1[0] = c.x; w1[1 % (kWords + 1)] = c.y;
      } else {
#pragma unroll
        for (int c = 0; c < kWords; ++c) {
          w0[c] = *reinterpret_cast<const uint32_t*>(k0 + 4 * (t * kWords + c));
          w1[c] = *reinterpret_cast<const uint32_t*>(k1 + 4 * (t * kWords + c));
        }
      }
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        const uint32_t a0 = low_codes(w0[c]), a1 = low_codes(w1[c]), a2 = high_codes(w0[c]), a3 = high_codes(w1[c]);
        const uint32_t u0 = w0[c] >> 8, u1 = w1[c] >> 8;
        const uint32_t e0 = low_codes(u0), e1 = low_codes(u1), e2 = high_codes(u0), e3 = high_codes(u1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(x[n][m], a0, a1, a2, a3, qb[n][2 * c][0], qb[n][2 * c][1]);
          mma_f16(x[n][m], e0, e1, e2, e3, qb[n][2 * c + 1][0], qb[n][2 * c + 1][1]);
        }
      }
      if (D % 32) {
        uint32_t u0 = *reinterpret_cast<const uint16_t*>(k0 + 16 * kWords + 2 * t);
        uint32_t u1 = *reinterpret_cast<const uint16_t*>(k1 + 16 * kWords + 2 * t);
        u0 |= u0 << 8;
        u1 |= u1 << 8;
        const uint32_t a0 = low_codes(u0), a1 = low_codes(u1), a2 = high_codes(u0), a3 = high_codes(u1);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma_f16(x[n][m], a0, a1, a2, a3, qb[n][kSteps - 1][0], qb[n][kSteps - 1][1]);
      }
      const uint32_t* pr0 = reinterpret_cast<const uint32_t*>(st + block_of(i0) + tokens * D) + slot_of(i0);
      const uint32_t* pr1 = reinterpret_cast<const uint32_t*>(st + block_of(i1) + tokens * D) + slot_of(i1);
      float2 kp0 = unpack_f16(pr0[0]), kp1 = unpack_f16(pr1[0]);
      kp0.y = __fmaf_rn(8.0f, kp0.x, kp0.y);
      kp1.y = __fmaf_rn(8.0f, kp1.x, kp1.y);
      vpair[m][0] = pr0[tokens];
      vpair[m][1] = pr1[tokens];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a = x[n][m][j];
          if (SPLIT) a = __fadd_rn(a, __shfl_xor_sync(kFull, a, 2));
          const float2 kp = j < 2 ? kp0 : kp1;
          // q's own size comes last: a code times it may pass the largest number
          x[n][m][j] = __fmaf_rn(__fmul_rn(a, kp.x), q_fac[n][j & 1], __fmul_rn(kp.y, q_sum[n][j & 1]));
        }
      if (masked) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = half ? i1 : i0;
          const bool held = here >> (i >> p.pool.token_shift) & 1;
          if (!held || key0 + i >= keys) vpair[m][half] = 0;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (!held || key0 + i >= limit[n][j]) x[n][m][2 * half + j] = -INFINITY;
        }
      }
    }

    // ---- the running maximum of x + exponent(scale_v) ----
    float ev[2][2];
    bool grows = false;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        ev[m][half] = half_exponent(unpack_f16(vpair[m][half]).x);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) grows |= __fadd_rn(x[n][m][2 * half + j], ev[m][half]) > top[n][j];
      }
    if (__any_sync(kFull, grows)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float shrink[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v = top[n][j];
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int half = 0; half < 2; ++half) v = fmaxf(v, __fadd_rn(x[n][m][2 * half + j], ev[m][half]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
          shrink[j] = top[n][j] == -INFINITY ? 0.0f : exp2_approx(__fsub_rn(top[n][j], v));
          top[n][j] = v;
          sum_p[n][j] = __fmul_rn(sum_p[n][j], shrink[j]);
          sum_m[n][j] = __fmul_rn(sum_m[n][j], shrink[j]);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[n][i][j] = __fmul_rn(acc[n][i][j], shrink[j & 1]);
      }
    }

    // ---- weights ----
    uint32_t wb[NT][2][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float base[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) base[j] = top[n][j] == -INFINITY ? 0.0f : __fsub_rn(top[n][j], 10.0f);
      float here_p[2] = {0.0f, 0.0f}, here_m[2] = {0.0f, 0.0f};  // small weights are added up before they meet a large sum
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float2 vp = unpack_f16(vpair[m][half]);
          vp.y = __fmaf_rn(8.0f, vp.x, vp.y);
          float w[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float e = exp2_approx(__fsub_rn(x[n][m][2 * half + j], base[j]));
            here_p[j] = __fadd_rn(here_p[j], e);
            here_m[j] = __fmaf_rn(e, vp.y, here_m[j]);
            w[j] = __fmul_rn(e, vp.x);
          }
          uint32_t packed = pack_f16(w[0], w[1]);
          if (SPLIT) {
            const float2 hi2 = unpack_f16(packed);
            const uint32_t rest = pack_f16(__fmul_rn(__fsub_rn(w[0], hi2.x), 2048.0f),
                                           __fmul_rn(__fsub_rn(w[1], hi2.y), 2048.0f));
            packed = t < 2 ? packed : rest;
          }
          wb[n][m][half] = transpose8(packed);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sum_p[n][j] = __fadd_rn(sum_p[n][j], here_p[j]);
        sum_m[n][j] = __fadd_rn(sum_m[n][j], here_m[j]);
      }
    }

    // ---- values: byte i of a lane holds channels 2c (row g) and 2c + 1 (row g + 8) ----
    // The tensor cores' own additions cut off what lies below their sum's last
    // bit, so a sum over many keys drifts: theirs runs over one tile, and tiles
    // are added in f32.  Error of one warp's 262,144 keys, values of mean 0: 9e-5
    // of the output instead of 1.6e-2 (of mean 1: 1.5e-6 instead of 5e-5); no
    // slower (8 x 65,536 keys: 186 us).
    const uint8_t* v[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t i = 16 * m + t + 4 * k;
        v[m][k] = st + block_of(i) + (uint32_t)(tokens + slot_of(i)) * (D / 2);
      }
    auto step = [&](int i, const uint32_t (&w)[2][4], int byte) {
      const uint32_t sel = byte | (byte << 4) | ((4 + byte) << 8) | ((4 + byte) << 12);
      float add[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) add[n][j] = 0.0f;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t ab = __byte_perm(w[m][0], w[m][1], sel), cd = __byte_perm(w[m][2], w[m][3], sel);
        const uint32_t a0 = low_codes(ab), a1 = high_codes(ab), a2 = low_codes(cd), a3 = high_codes(cd);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(add[n], a0, a1, a2, a3, wb[n][m][0], wb[n][m][1]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][i][j] = __fadd_rn(acc[n][i][j], add[n][j]);
    };
    uint32_t w[2][4];
    if (D == 128) {
      uint32_t w2[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint2 both = *reinterpret_cast<const uint2*>(v[m][k] + 8 * g);
          w[m][k] = both.x;
          w2[m][k] = both.y;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        step(i % kSteps, w, i);
        step((4 + i) % kSteps, w2, i);
      }
    } else {
      constexpr int kAt2 = kSteps & 4, kAt1 = kSteps & 6;
      auto load = [&](auto part, int at) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[m][k] = *reinterpret_cast<const decltype(part)*>(v[m][k] + at + (int)sizeof(part) * g);
      };
      if (kSteps & 4) {
        load(uint32_t(), 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) step(i % kSteps, w, i);
      }
      if (kSteps & 2) {
        load(uint16_t(), 8 * kAt2);
#pragma unroll
        for (int i = 0; i < 2; ++i) step((kAt2 + i) % kSteps, w, i);
      }
      if (kSteps & 1) {
        load(uint8_t(), 8 * kAt1);
        step(kAt1 % kSteps, w, 0);
      }
    }
    __syncwarp();
    if (tl + kAttnStages < end) issue(tl + kAttnStages);
  }
  if (broken) live = false;

  // ---- normalize: rows of this warp's keys, and their log2 sum ----
  const bool join = p.warps_log2 > 0;
  if (join) __syncthreads();  // the rings of a unit's warps become their results
  float* own_out = reinterpret_cast<float*>(ring);
  float* own_lse = own_out + kQ * D;
  const long long slot0 = (long long)unit * kQ;
  const bool direct = splits_here <= 1;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float inv[2], zero[2], lse2[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        sum_p[n][j] = __fadd_rn(sum_p[n][j], __shfl_xor_sync(kFull, sum_p[n][j], o));
        sum_m[n][j] = __fadd_rn(sum_m[n][j], __shfl_xor_sync(kFull, sum_m[n][j], o));
      }
      inv[j] = sum_p[n][j] == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum_p[n][j]);
      zero[j] = sum_m[n][j];
      lse2[j] = sum_p[n][j] == 0.0f ? -INFINITY : __fadd_rn(__fsub_rn(top[n][j], 10.0f), log2f(sum_p[n][j]));
    }
    long long at[2];  // where the lane's columns go: their output row, or their slot
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = min(row0 + n * kCols + 2 * t + j, max(n_rows - 1, 0));
      const int pos = (int)share((uint32_t)row, (uint32_t)r.group), h = head * r.group + row - pos * r.group;
      at[j] = direct ? (long long)(seq.q0 + pos) * r.out_row_stride + (long long)h * r.out_head_stride
                     : ((slot0 + n * kCols + 2 * t + j) * p.split.splits + split) * D;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      // the byte that tile i took from this lane's values
      int byte;
      if (D == 128) {
        byte = 8 * g + i;
      } else if (i < (kSteps & 4)) {
        byte = 4 * g + i;
      } else if (i < (kSteps & 6)) {
        byte = 8 * (kSteps & 4) + 2 * g + i - (kSteps & 4);
      } else {
        byte = 8 * (kSteps & 6) + g;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float even = acc[n][i][j], odd = acc[n][i][2 + j];
        if (SPLIT) {
          even = __fmaf_rn(__shfl_xor_sync(kFull, even, 2), 1.0f / 2048.0f, even);
          odd = __fmaf_rn(__shfl_xor_sync(kFull, odd, 2), 1.0f / 2048.0f, odd);
        }
        even = __fmul_rn(__fadd_rn(even, zero[j]), inv[j]);
        odd = __fmul_rn(__fmaf_rn(odd, 0.0625f, zero[j]), inv[j]);
        const int c = 2 * t + j, q = n * kCols + c;
        if (!live || (SPLIT && t >= 2) || row0 + q >= n_rows) continue;
        if (join) {
          *reinterpret_cast<float2*>(own_out + q * D + 2 * byte) = make_float2(even, odd);
        } else if (direct) {
          store2(r.out, at[j] + 2 * byte, dtype, even, odd);
        } else {
          *reinterpret_cast<float2*>(p.split.out + at[j] + 2 * byte) = make_float2(even, odd);
        }
      }
    }
    if (live && g == 0) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = 2 * t + j, q = n * kCols + c;
        if ((SPLIT && t >= 2) || row0 + q >= n_rows) continue;
        if (join) {
          own_lse[q] = lse2[j];
        } else if (direct) {
          const int pos = (int)share((uint32_t)(row0 + q), (uint32_t)r.group), h = head * r.group + (row0 + q) - pos * r.group;
          if (r.lse) r.lse[(long long)(seq.q0 + pos) * r.kv_heads * r.group + h] = __fmul_rn(lse2[j], kLn2);
        } else {
          p.split.lse[(slot0 + q) * p.split.splits + split] = lse2[j];
        }
      }
    }
  }
  if (!join) return;
  __syncthreads();
  // ---- join the unit's warps: each takes every wpu-th query ----
  const int warp0 = warp & ~(wpu - 1);
  for (int q = sub; q < kQ; q += wpu) {
    if (!live || row0 + q >= n_rows) break;
    float l[kAttnWarps], best = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      l[w] = w < wpu ? reinterpret_cast<const float*>(smem + (warp0 + w) * kAttnStages * kStage)[kQ * D + q] : -INFINITY;
      best = fmaxf(best, l[w]);
    }
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      l[w] = join_weight(l[w], best);
      total = __fadd_rn(total, l[w]);
    }
    const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    const int pos = (int)share((uint32_t)(row0 + q), (uint32_t)r.group), h = head * r.group + (row0 + q) - pos * r.group;
    for (int c = 2 * lane; c < D; c += 64) {
      float a = 0.0f, e = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w)
        if (w < wpu && l[w] != 0.0f) {
          const float2 v = *reinterpret_cast<const float2*>(
              reinterpret_cast<const float*>(smem + (warp0 + w) * kAttnStages * kStage) + q * D + c);
          a = __fmaf_rn(l[w], v.x, a);
          e = __fmaf_rn(l[w], v.y, e);
        }
      a = __fmul_rn(a, inv);
      e = __fmul_rn(e, inv);
      if (direct)
        store2(r.out, (long long)(seq.q0 + pos) * r.out_row_stride + (long long)h * r.out_head_stride + c, dtype, a,
               e);
      else
        *reinterpret_cast<float2*>(p.split.out + ((slot0 + q) * p.split.splits + split) * D + c) = make_float2(a, e);
    }
    if (lane == 0) {
      const float lse2 = total == 0.0f ? -INFINITY : __fadd_rn(best, log2f(total));
      if (!direct)
        p.split.lse[(slot0 + q) * p.split.splits + split] = lse2;
      else if (r.lse)
        r.lse[(long long)(seq.q0 + pos) * r.kv_heads * r.group + h] = __fmul_rn(lse2, kLn2);
    }
  }
}

// ---- join of split keys: one warp per query row ----
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnRows r, const AttnSplit s, int tile_keys,
                                                        int unit_rows, int row_tiles, long long slots) {
  pdl_enter();
  const long long slot = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (slot >= slots) return;
  const uint32_t nth = (uint32_t)(slot / unit_rows), unit = s.first + nth, bh = unit / (uint32_t)row_tiles;
  const int q = (int)(slot - (long long)nth * unit_rows) + (int)(unit - bh * row_tiles) * unit_rows;
  const int b = (int)(bh / (uint32_t)r.kv_heads), head = (int)(bh - (uint32_t)b * r.kv_heads);
  const AttnSeq seq = attn_seq(r, b, nullptr, false);
  if (!seq.ok || q >= seq.nq * r.group) return;
  const int parts = ((seq.nk + tile_keys - 1) / tile_keys + s.chunk - 1) / s.chunk;
  if (parts <= 1) return;
  const float* lse = s.lse + slot * s.splits;
  float best = -INFINITY, total = 0.0f;
  for (int i = lane; i < parts; i += 32) best = fmaxf(best, lse[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(kFull, best, o));
  for (int i = lane; i < parts; i += 32) total = __fadd_rn(total, join_weight(lse[i], best));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total = __fadd_rn(total, __shfl_xor_sync(kFull, total, o));
  const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
  const int pos = q / r.group, h = head * r.group + q - pos * r.group, d = r.head_dim;
  float2 sum[kOpMaxHeadDim / 64] = {};
  for (int i = 0; i < parts; ++i) {
    const float w = join_weight(lse[i], best);
    if (w == 0.0f) continue;
    const float* row = s.out + (slot * s.splits + i) * d;
#pragma unroll
    for (int k = 0; k < kOpMaxHeadDim / 64; ++k)
      if (64 * k + 2 * lane < d) {
        const float2 v = *reinterpret_cast<const float2*>(row + 64 * k + 2 * lane);
        sum[k].x = __fmaf_rn(w, v.x, sum[k].x);
        sum[k].y = __fmaf_rn(w, v.y, sum[k].y);
      }
  }
#pragma unroll
  for (int k = 0; k < kOpMaxHeadDim / 64; ++k)
    if (64 * k + 2 * lane < d)
      store2(r.out,
             (long long)(seq.q0 + pos) * r.out_row_stride + (long long)h * r.out_head_stride + 64 * k + 2 * lane,
             r.dtype, __fmul_rn(sum[k].x, inv), __fmul_rn(sum[k].y, inv));
  if (lane == 0 && r.lse)
    r.lse[(long long)(seq.q0 + pos) * r.kv_heads * r.group + h] =
        total == 0.0f ? -INFINITY : __fmul_rn(__fadd_rn(best, log2f(total)), kLn2);
}

// ---- shapes of a launch ----
struct Kv4Plan {
  int nt, row_tiles, warps_log2, splits, chunk;
  long long units;
  uint64_t slots, bytes;
};

bool kv4_shape_ok(int32_t page_tokens, int32_t kv_heads, int32_t head_dim) {
  return (page_tokens == 8 || page_tokens == 16 || page_tokens == 32) && kv_heads >= 1 && kv_heads <= 65536 &&
         head_dim >= 16 && head_dim <= kOpMaxHeadDim && head_dim % 16 == 0;
}

bool kv4_cache_ok(const mc_kv4_cache* c) {
  return c && kv4_shape_ok(c->page_tokens, c->kv_heads, c->head_dim) && c->n_pages >= 0 && c->n_pages <= INT32_MAX &&
         c->batch >= 0 && c->pages_per_seq >= 1 && (int64_t)c->pages_per_seq * c->page_tokens <= INT32_MAX &&
         (int64_t)c->batch * c->kv_heads <= INT32_MAX;
}

// How many columns a unit takes, how many warps share its keys and into how
// many ranges they are cut.  A warp alone per unit needs no join; more are
// used while there are fewer than 16 warps per SM, and each keeps at least
// two tiles (of 32 keys), as a join costs about as much as a tile.
bool kv4_plan(const mc_kv4_cache* c, const mc_kv4_attention_args* a, Kv4Plan* plan) {
  if (!kv4_cache_ok(c) || !a || dtype_bytes(a->dtype) == 0 || a->heads < 1 || a->heads % c->kv_heads != 0 ||
      a->max_q_len < 0 || a->max_kv_len < 0 || a->max_kv_len > kOpMaxKeys)
    return false;
  const int64_t group = a->heads / c->kv_heads, rows = group * a->max_q_len;
  if (rows > INT32_MAX / 2) return false;
  const int cols = a->dtype == MC_F32 ? 4 : 8;
  plan->nt = rows > cols ? 2 : 1;
  plan->row_tiles = (int)((rows + cols * plan->nt - 1) / (cols * plan->nt));
  plan->units = (long long)c->batch * c->kv_heads * plan->row_tiles;
  if (plan->units > INT32_MAX) return false;
  const int tiles = (int)(((int64_t)a->max_kv_len + kTileKeys - 1) / kTileKeys);
  long long want = plan->units > 0 ? (kSms * 16) / plan->units : 1;
  if (want > tiles / 2) want = tiles / 2;
  plan->warps_log2 = want >= 4 ? 2 : want >= 2 ? 1 : 0;
  long long splits = plan->warps_log2 == 2 ? want / kAttnWarps : 1;
  if (splits > 256) splits = 256;
  if (splits < 1) splits = 1;
  plan->chunk = tiles > 0 ? (int)((tiles + splits - 1) / splits) : 1;
  plan->splits = tiles > 0 ? (tiles + plan->chunk - 1) / plan->chunk : 1;
  plan->slots = (uint64_t)plan->units * cols * plan->nt;
  plan->bytes = attn_split_bytes(plan->slots, plan->splits, c->head_dim);
  return true;
}

template <int D, int NT, bool SPLIT>
cudaError_t launch_kv4_attn(const Kv4AttnParams& p, const Kv4Plan& plan, cudaStream_t s) {
  static uint64_t done = 0;
  cudaError_t e = allow_smem(kv4_attn_kernel<D, NT, SPLIT>, attn_smem(D), &done);
  if (e != cudaSuccess) return e;
  const int per_cta = kAttnWarps >> plan.warps_log2;
  return launch_pdl(kv4_attn_kernel<D, NT, SPLIT>, dim3((unsigned)((plan.units + per_cta - 1) / per_cta), plan.splits),
                    dim3(kAttnWarps * 32), attn_smem(D), s, p);
}

template <int D>
cudaError_t launch_kv4_attn_d(const Kv4AttnParams& p, const Kv4Plan& plan, cudaStream_t s) {
  if (p.rows.dtype == MC_F32)
    return plan.nt == 1 ? launch_kv4_attn<D, 1, true>(p, plan, s) : launch_kv4_attn<D, 2, true>(p, plan, s);
  return plan.nt == 1 ? launch_kv4_attn<D, 1, false>(p, plan, s) : launch_kv4_attn<D, 2, false>(p, plan, s);
}

Kv4Pool pool_of(const mc_kv4_cache* c) {
  Kv4Pool p;
  p.pages = static_cast<uint8_t*>(c->pages);
  p.table = c->page_table;
  p.n_pages = c->n_pages;
  p.token_shift = c->page_tokens == 8 ? 3 : c->page_tokens == 16 ? 4 : 5;
  p.kv_heads = c->kv_heads;
  p.head_dim = c->head_dim;
  p.batch = c->batch;
  p.per_seq = c->pages_per_seq;
  return p;
}

template <int TYPE, int L, bool READ>
cudaError_t launch_rows(const Kv4Pool& p, const Kv4RowsDev& r, long long grid, int chunks, uint32_t* status,
                        cudaStream_t s) {
  return launch_pdl(kv4_rows_kernel<TYPE, L, READ>, dim3((unsigned)grid), dim3(kRowThreads), 0, s, p, r, chunks, status);
}
template <int TYPE, bool READ>
cudaError_t launch_rows_l(const Kv4Pool& p, const Kv4RowsDev& r, long long grid, int chunks, uint32_t* status,
                          cudaStream_t s) {
  const int lanes = p.head_dim / 8;
  return lanes <= 2   ? launch_rows<TYPE, 2, READ>(p, r, grid, chunks, status, s)
         : lanes <= 4 ? launch_rows<TYPE, 4, READ>(p, r, grid, chunks, status, s)
         : lanes <= 8 ? launch_rows<TYPE, 8, READ>(p, r, grid, chunks, status, s)
                      : launch_rows<TYPE, 16, READ>(p, r, grid, chunks, status, s);
}

template <bool READ>
mc_status kv4_rows(const mc_kv4_cache* c, const mc_kv4_rows* a, void* stream) {
  const int bytes = a ? dtype_bytes(a->dtype) : 0;
  if (!kv4_cache_ok(c) || !a || bytes == 0 || a->rows < 0 || a->rows > INT32_MAX || a->max_count < 0) return MC_INVALID_INPUT;
  if (c->batch == 0 || a->max_count == 0) return MC_OK;
  const long long chunks = (a->max_count + (long long)kRowTokens - 1) / kRowTokens, grid = chunks * c->batch;
  if (grid > INT32_MAX || (!c->pages && c->n_pages > 0) || !aligned16(c->pages) || !c->page_table || !aligned4(c->page_table) ||
      !a->start || !a->count || !a->first || !aligned4(a->start) || !aligned4(a->count) || !aligned4(a->first) ||
      !strides_ok(a->k, a->rows, a->k_row_stride, a->k_head_stride, bytes) ||
      !strides_ok(a->v, a->rows, a->v_row_stride, a->v_head_stride, bytes))
    return MC_INVALID_INPUT;
  if (READ && (!strides_apart(a->rows, c->kv_heads, c->head_dim, a->k_row_stride, a->k_head_stride) ||
               !strides_apart(a->rows, c->kv_heads, c->head_dim, a->v_row_stride, a->v_head_stride) || (a->k && a->k == a->v)))
    return MC_INVALID_INPUT;
  const mc_status where = on_current_device({c->pages, c->page_table, a->k, a->v, a->start, a->count, a->first});
  if (where != MC_OK) return where;
  uint32_t* status = op_status_word();
  if (!status) return MC_CUDA;
  const Kv4Pool pool = pool_of(c);
  const Kv4RowsDev r = {a->k,           a->v,           a->start,       a->count,        a->first,      a->rows,
                        a->k_row_stride, a->k_head_stride, a->v_row_stride, a->v_head_stride, a->max_count};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == MC_F32   ? launch_rows_l<MC_F32, READ>(pool, r, grid, (int)chunks, status, s)
                        : a->dtype == MC_F16 ? launch_rows_l<MC_F16, READ>(pool, r, grid, (int)chunks, status, s)
                                             : launch_rows_l<MC_BF16, READ>(pool, r, grid, (int)chunks, status, s);
  return launched(e);
}

}  // namespace

cudaError_t launch_attn_join(const AttnRows& r, const AttnSplit& s, int tile_keys, int unit_rows, int row_tiles,
                             cudaStream_t stream) {
  const long long slots = ((long long)r.batch * r.kv_heads * row_tiles - s.first) * unit_rows;
  return launch_pdl(attn_join_kernel, dim3((unsigned)((slots + 3) / 4)), dim3(128), 0, stream, r, s, tile_keys,
                    unit_rows, row_tiles, slots);
}

}  // namespace mc

extern "C" uint64_t mc_kv4_page_bytes(int32_t page_tokens, int32_t kv_heads, int32_t head_dim) {
  if (!mc::kv4_shape_ok(page_tokens, kv_heads, head_dim)) return 0;
  return (uint64_t)kv_heads * mc::head_block(page_tokens, head_dim);
}

extern "C" mc_status mc_kv4_append(const mc_kv4_cache* cache, const mc_kv4_rows* rows, void* stream) {
  return mc::kv4_rows<false>(cache, rows, stream);
}

extern "C" mc_status mc_kv4_read(const mc_kv4_cache* cache, const mc_kv4_rows* rows, void* stream) {
  return mc::kv4_rows<true>(cache, rows, stream);
}

extern "C" uint64_t mc_kv4_attention_workspace(const mc_kv4_cache* cache, const mc_kv4_attention_args* args) {
  mc::Kv4Plan plan;
  return mc::kv4_plan(cache, args, &plan) ? plan.bytes : 0;
}

extern "C" mc_status mc_kv4_attention(const mc_kv4_cache* c, const mc_kv4_attention_args* a, void* stream) {
  mc::Kv4Plan plan;
  if (!mc::kv4_plan(c, a, &plan) || !mc::scale_ok(a->scale) || a->q_rows < 0 || a->q_rows > INT32_MAX)
    return MC_INVALID_INPUT;
  if (plan.units == 0) return MC_OK;
  const int bytes = mc::dtype_bytes(a->dtype);
  if (a->max_kv_len > (int64_t)c->pages_per_seq * c->page_tokens || (!c->pages && c->n_pages > 0) || !mc::aligned16(c->pages) ||
      !c->page_table || !mc::aligned4(c->page_table) || !a->q_start || !a->q_len || !a->kv_len ||
      !mc::aligned4(a->q_start) || !mc::aligned4(a->q_len) || !mc::aligned4(a->kv_len) || !mc::aligned4(a->lse) ||
      !mc::strides_ok(a->q, a->q_rows, a->q_row_stride, a->q_head_stride, bytes) ||
      !mc::strides_ok(a->out, a->q_rows, a->out_row_stride, a->out_head_stride, bytes) ||
      !mc::strides_apart(a->q_rows, a->heads, c->head_dim, a->out_row_stride, a->out_head_stride) ||
      (a->out && a->q == a->out))
    return MC_INVALID_INPUT;
  if (plan.bytes > 0 && (!a->workspace || !mc::aligned16(a->workspace) || a->workspace_bytes < plan.bytes))
    return MC_INVALID_INPUT;
  const mc_status where = mc::on_current_device({c->pages, c->page_table, a->q, a->out, a->lse, a->q_start, a->q_len,
                                                 a->kv_len, plan.bytes > 0 ? a->workspace : nullptr});
  if (where != MC_OK) return where;
  uint32_t* status = mc::op_status_word();
  if (!status) return MC_CUDA;
  mc::Kv4AttnParams p;
  std::memset(&p, 0, sizeof(p));
  p.pool = mc::pool_of(c);
  mc::AttnRows& r = p.rows;
  r.q = a->q;
  r.out = a->out;
  r.lse = a->lse;
  r.q_start = a->q_start;
  r.q_len = a->q_len;
  r.k_len = a->kv_len;
  r.q_rows = a->q_rows;
  r.q_row_stride = a->q_row_stride;
  r.q_head_stride = a->q_head_stride;
  r.out_row_stride = a->out_row_stride;
  r.out_head_stride = a->out_head_stride;
  r.dtype = a->dtype;
  r.batch = c->batch;
  r.kv_heads = c->kv_heads;
  r.group = a->heads / c->kv_heads;
  r.head_dim = c->head_dim;
  r.max_q = a->max_q_len;
  r.max_k = a->max_kv_len;
  r.causal = a->causal != 0;
  p.split.splits = plan.splits;
  p.split.chunk = plan.chunk;
  if (plan.splits > 1) {
    p.split.out = static_cast<float*>(a->workspace);
    p.split.lse = p.split.out + plan.slots * plan.splits * c->head_dim;
  }
  p.scale = a->scale;
  p.row_tiles = plan.row_tiles;
  p.warps_log2 = plan.warps_log2;
  p.units = (uint32_t)plan.units;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorInvalidValue;
  switch (c->head_dim) {
    case 16: e = mc::launch_kv4_attn_d<16>(p, plan, s); break;
    case 32: e = mc::launch_kv4_attn_d<32>(p, plan, s); break;
    case 48: e = mc::launch_kv4_attn_d<48>(p, plan, s); break;
    case 64: e = mc::launch_kv4_attn_d<64>(p, plan, s); break;
    case 80: e = mc::launch_kv4_attn_d<80>(p, plan, s); break;
    case 96: e = mc::launch_kv4_attn_d<96>(p, plan, s); break;
    case 112: e = mc::launch_kv4_attn_d<112>(p, plan, s); break;
    case 128: e = mc::launch_kv4_attn_d<128>(p, plan, s); break;
  }
  if (e == cudaSuccess && plan.splits > 1)
    e = mc::launch_attn_join(r, p.split, mc::kTileKeys, plan.nt * (a->dtype == MC_F32 ? 4 : 8), plan.row_tiles, s);
  return mc::launched(e);
}
