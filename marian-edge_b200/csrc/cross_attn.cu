// cross_attn.cu -- attention of packed queries to the states of an encoder
// whose sequences have another length (mc_cross_attention).
//
// out_i = sum_j w_ij v_j / sum_j w_ij, w_ij = exp(scale q_i . k_j), over the
// keys of the query's sequence that the mask leaves in.  One pass over the
// keys with the running maximum and sum of each row in registers.
#include <cstring>

#include "cross_attn.cuh"

namespace mc {
namespace {

constexpr uint32_t kFull = 0xFFFFFFFFu;

// ---- small tiles: mma.sync ------------------------------------------------------------
// Four warps: WR of them side by side over 16 rows each, the other 4 / WR
// groups over parts of every key tile, so that a unit of 16 rows (a decode
// step's) still has four warps on its keys.  Rows are (position, head of the
// group): shared heads fill the row tile of a single position.
//
// 16-bit types: m16n8k16, weights rounded to the values' type after a shift
// of 2^8 that keeps small f16 weights normal.  f32: m16n8k8 on tf32 halves of
// each operand (11 + 11 bits; high x high + high x low + low x high), within
// 2^-21 of each product.
template <typename T>
struct Tile;
template <>
struct Tile<float> {
  static constexpr int kKeys = 32;
};
template <>
struct Tile<__half> {
  static constexpr int kKeys = 64;
};
template <>
struct Tile<__nv_bfloat16> {
  static constexpr int kKeys = 64;
};

constexpr int kStages = 2;
constexpr float kShift = 8.0f;

template <typename T, int D>
constexpr int pitch() {
  return D + 8;
}
template <typename T, int D>
constexpr int stage_elems() {
  return Tile<T>::kKeys * pitch<T, D>();  // one of K and V
}
template <typename T, int D>
constexpr int cross_smem() {
  return kStages * (2 * stage_elems<T, D>() * (int)sizeof(T) + 16);
}

__device__ __forceinline__ void cp16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = high + low: x rounded to 11 bits, and the rest.  (Cut off instead of
// rounded, the rests are all of one sign, and so are the errors of the 11 bits
// that are left of them: outputs 8e-7 off instead of 5e-7.)
__device__ __forceinline__ uint32_t tf32_high(float x) { return (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u; }
__device__ __forceinline__ uint32_t tf32_low(float x) {
  return __float_as_uint(__fsub_rn(x, __uint_as_float(tf32_high(x))));
}
// d += high x high, rest += the products with a low part.  The tensor cores'
// own additions do not round to nearest, so a sum of many terms drifts: the
// small products have a sum of their own, and neither runs past one tile.
__device__ __forceinline__ void mma_split(float (&d)[4], float (&rest)[4], const uint32_t (&ah)[4],
                                          const uint32_t (&al)[4], float b0, float b1) {
  const uint32_t h0 = tf32_high(b0), h1 = tf32_high(b1);
  mma_tf32(rest, al, h0, h1);
  mma_tf32(rest, ah, tf32_low(b0), tf32_low(b1));
  mma_tf32(d, ah, h0, h1);
}

// CTAs per SM that the registers are kept to, 0: as they come.  Ragged
// sentences in 16 bits are latency, of which five CTAs hide more than four
// (256 sentences, 8 heads of 64: 24.0 us, 25.0 with four, 41 with six, which
// spill); f32 spills at four (14 us instead of 12 for 64 single tokens).
template <typename T, int D>
constexpr int small_blocks() {
  return sizeof(T) == 2 && D <= 64 ? 5 : 0;
}

template <typename T, int D, int WR>
__global__ void __launch_bounds__(128, small_blocks<T, D>()) cross_small_kernel(const CrossParams p) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kType = kF32 ? MC_F32 : std::is_same<T, __half>::value ? MC_F16 : MC_BF16;
  constexpr int kKeys = Tile<T>::kKeys, kGroups = 4 / WR, kOwn = kKeys / kGroups, kNT = kOwn / 8;
  constexpr int kPitch = pitch<T, D>(), kElems = stage_elems<T, D>(), kRows = 16 * WR;
  constexpr int kChunk = 16 / (int)sizeof(T), kRowChunks = D / kChunk;
  constexpr int kOut = D / 8;  // n8 tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  T* ring = reinterpret_cast<T*>(smem);
  uint32_t* live_bits = reinterpret_cast<uint32_t*>(smem + kStages * 2 * kElems * sizeof(T));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wr = warp % WR, kg = warp / WR;
  pdl_enter();

  const AttnRows& r = p.rows;
  const uint32_t unit = blockIdx.x, bh = share(unit, (uint32_t)p.row_tiles);
  const int tile = (int)(unit - bh * p.row_tiles), b = (int)share(bh, (uint32_t)r.kv_heads), head = (int)(bh - (uint32_t)b * r.kv_heads);
  const int split = blockIdx.y;
  const AttnSeq seq = attn_seq(r, b, p.status, head == 0 && tile == 0 && split == 0 && tid == 0);
  const int n_rows = seq.nq * r.group, row0 = tile * kRows;
  if (!seq.ok || row0 >= n_rows) return;
  const int n_tiles = (seq.nk + kKeys - 1) / kKeys;
  const int parts = p.split.splits == 1 ? 1 : max(1, (n_tiles + p.split.chunk - 1) / p.split.chunk);
  if (split >= parts) return;
  const int begin = split * p.split.chunk, end = min(n_tiles, begin + p.split.chunk);

  const T* kbase = static_cast<const T*>(p.k) + (long long)seq.k0 * p.k_rs + (long long)head * p.k_hs;
  const T* vbase = static_cast<const T*>(p.v) + (long long)seq.k0 * p.v_rs + (long long)head * p.v_hs;
  const uint8_t* mask = p.mask ? p.mask + seq.k0 : nullptr;

  auto load_tile = [&](int tl) {
    const int s = tl & (kStages - 1), key0 = tl * kKeys;
    T* ks = ring + s * 2 * kElems;
    T* vs = ks + kElems;
    if (warp < kKeys / 32) {
      const int key = key0 + warp * 32 + lane;
      const uint32_t w = __ballot_sync(kFull, key < seq.nk && (!mask || mask[key]));
      if (lane == 0) live_bits[s * 2 + warp] = w;
    }
#pragma unroll
    for (int c = tid; c < kKeys * kRowChunks; c += 128) {
      const int row = c / kRowChunks, at = (c - row * kRowChunks) * kChunk;
      const int key = key0 + row;
      // A key that is left out is zeros, whatever it holds: a weight of 0
      // times an infinity would be NaN.
      const bool there = key < seq.nk && (!mask || mask[key]);
      const int from = there ? key : 0;
      cp16(ks + row * kPitch + at, kbase + (long long)from * p.k_rs + at, there);
      cp16(vs + row * kPitch + at, vbase + (long long)from * p.v_rs + at, there);
    }
    cp_commit();
  };
  if (begin < end) load_tile(begin);

  // ---- the warp's 16 query rows ----
  const int own = row0 + wr * 16;
  const void* src[2];
  bool there[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = own + g + 8 * h;
    there[h] = row < n_rows;
    const int pos = there[h] ? (int)share((uint32_t)row, (uint32_t)r.group) : 0, qh = head * r.group + (there[h] ? row - pos * r.group : 0);
    src[h] = static_cast<const T*>(r.q) + (long long)(seq.q0 + pos) * r.q_row_stride + (long long)qh * r.q_head_stride;
  }
  const bool busy = own < n_rows;
  uint32_t qa[kF32 ? D / 8 : D / 16][4];
  if (kF32) {
    // step s: k = t is channel 8 s + 2 t, k = t + 4 the one after it
#pragma unroll
    for (int s = 0; s < D / 8; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 v = there[h] ? *reinterpret_cast<const float2*>(static_cast<const float*>(src[h]) + 8 * s + 2 * t)
                                  : make_float2(0.0f, 0.0f);
        qa[s][h] = __float_as_uint(v.x);
        qa[s][2 + h] = __float_as_uint(v.y);
      }
  } else {
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qa[s % (kF32 ? D / 8 : D / 16)][2 * e + h] =
              there[h] ? *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(src[h]) + 16 * s + 8 * e + 2 * t)
                       : 0u;
  }

  const float factor = __fmul_rn(p.scale, kLog2e);
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  float acc[kOut][4];
#pragma unroll
  for (int i = 0; i < kOut; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;

  for (int tl = begin; tl < end; ++tl) {
    if (tl + 1 < end) {
      load_tile(tl + 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    if (busy) {
      const int s = tl & (kStages - 1);
      const T* ks = ring + s * 2 * kElems + kg * kOwn * kPitch;
      const T* vs = ks + kElems;
      const int keys = seq.nk - tl * kKeys - kg * kOwn;  // of this warp's; n-tiles past them are left out
      float x[kNT][4];
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = 0.0f;
      // column n of a score tile: key n (16 bits), or key (n / 2) + 4 (n % 2)
      // (f32), so that a thread's two columns are the rows t and t + 4 of the
      // values, which lie in different banks
      if constexpr (kF32) {
        float rest[kNT][4] = {};
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint32_t ah[4], al[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ah[e] = tf32_high(__uint_as_float(qa[c][e]));
            al[e] = tf32_low(__uint_as_float(qa[c][e]));
          }
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            if (8 * j >= keys) break;
            const float2 kv = *reinterpret_cast<const float2*>(ks + (8 * j + (g >> 1) + 4 * (g & 1)) * kPitch + 8 * c + 2 * t);
            mma_split(x[j], rest[j], ah, al, kv.x, kv.y);
          }
        }
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j][e] = __fadd_rn(x[j][e], rest[j][e]);
      } else {
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int j = 0; j < kNT; j += 2) {
            if (8 * j >= keys) break;
            uint32_t kb[4];
            ldsm4(kb, ks + (8 * j + (lane & 7) + (lane >> 4) * 8) * kPitch + 16 * c + ((lane >> 3) & 1) * 8);
            if constexpr (sizeof(T) == 2) {
              if (std::is_same<T, __half>::value) {
                mma_f16(x[j], qa[c][0], qa[c][1], qa[c][2], qa[c][3], kb[0], kb[1]);
                mma_f16(x[j + 1], qa[c][0], qa[c][1], qa[c][2], qa[c][3], kb[2], kb[3]);
              } else {
                mma_bf16(x[j], qa[c][0], qa[c][1], qa[c][2], qa[c][3], kb[0], kb[1]);
                mma_bf16(x[j + 1], qa[c][0], qa[c][1], qa[c][2], qa[c][3], kb[2], kb[3]);
              }
            }
          }
      }
      // ---- scale, mask, running maximum ----
      uint32_t bits[(kOwn + 31) / 32];
      bool all = true;
#pragma unroll
      for (int w = 0; w < (kOwn + 31) / 32; ++w) {
        const int at = kg * kOwn + 32 * w;
        bits[w] = live_bits[s * 2 + (at >> 5)] >> (at & 31);
        const uint32_t want = kOwn >= 32 ? kFull : (1u << (kOwn & 31)) - 1u;
        all = all && (bits[w] & want) == want;
      }
      float most[2] = {top[0], top[1]};
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = __fmul_rn(x[j][e], factor);
          const int key = 8 * j + (kF32 ? t + 4 * (e & 1) : 2 * t + (e & 1));
          if (!all && !(bits[key >> 5] >> (key & 31) & 1)) x[j][e] = -INFINITY;
          most[e >> 1] = fmaxf(most[e >> 1], x[j][e]);
        }
      float base[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        most[h] = fmaxf(most[h], __shfl_xor_sync(kFull, most[h], 1));
        most[h] = fmaxf(most[h], __shfl_xor_sync(kFull, most[h], 2));
      }
      if (__any_sync(kFull, most[0] > top[0] || most[1] > top[1])) {
        float shrink[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          shrink[h] = top[h] == -INFINITY ? 0.0f : exp2_approx(__fsub_rn(top[h], most[h]));
          top[h] = most[h];
          sum[h] = __fmul_rn(sum[h], shrink[h]);
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][e] = __fmul_rn(acc[i][e], shrink[e >> 1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) base[h] = top[h] == -INFINITY ? 0.0f : __fsub_rn(top[h], kShift);
      float here[2] = {0.0f, 0.0f};  // small weights are added up before they meet a large sum
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = exp2_approx(__fsub_rn(x[j][e], base[e >> 1]));
          here[e >> 1] = __fadd_rn(here[e >> 1], x[j][e]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) sum[h] = __fadd_rn(sum[h], here[h]);
      // ---- values ----
      if constexpr (kF32) {
        // k = t: column 2 t (key t); k = t + 4: column 2 t + 1 (key t + 4)
        uint32_t ah[kNT][4], al[kNT][4];
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = x[j][e == 0 ? 0 : e == 1 ? 2 : e == 2 ? 1 : 3];
            ah[j][e] = tf32_high(w);
            al[j][e] = tf32_low(w);
          }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float sum0[4] = {}, sum1[4] = {}, rest0[4] = {}, rest1[4] = {};
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            if (8 * j >= keys) break;
            const T* v0 = vs + (8 * j + t) * kPitch + 16 * c + 2 * g;
            const float2 a = *reinterpret_cast<const float2*>(v0), e = *reinterpret_cast<const float2*>(v0 + 4 * kPitch);
            mma_split(sum0, rest0, ah[j], al[j], a.x, e.x);
            mma_split(sum1, rest1, ah[j], al[j], a.y, e.y);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[2 * c][e] = __fadd_rn(acc[2 * c][e], __fadd_rn(sum0[e], rest0[e]));
            acc[2 * c + 1][e] = __fadd_rn(acc[2 * c + 1][e], __fadd_rn(sum1[e], rest1[e]));
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kNT; j += 2) {
          if (8 * j >= keys) break;
          uint32_t a[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float lo = x[j + (e >> 1)][2 * (e & 1)], hi = x[j + (e >> 1)][2 * (e & 1) + 1];
            a[e] = std::is_same<T, __half>::value ? pack_f16(lo, hi) : pack_bf16(lo, hi);
          }
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t vb[4];
            ldsm4t(vb, vs + (8 * j + (lane & 15)) * kPitch + 16 * c + (lane >> 4) * 8);
            if (std::is_same<T, __half>::value) {
              mma_f16(acc[2 * c], a[0], a[1], a[2], a[3], vb[0], vb[1]);
              mma_f16(acc[2 * c + 1], a[0], a[1], a[2], a[3], vb[2], vb[3]);
            } else {
              mma_bf16(acc[2 * c], a[0], a[1], a[2], a[3], vb[0], vb[1]);
              mma_bf16(acc[2 * c + 1], a[0], a[1], a[2], a[3], vb[2], vb[3]);
            }
          }
        }
      }
    }
    __syncthreads();
  }

  // ---- normalize ----
  float inv[2], lse2[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] = __fadd_rn(sum[h], __shfl_xor_sync(kFull, sum[h], 1));
    sum[h] = __fadd_rn(sum[h], __shfl_xor_sync(kFull, sum[h], 2));
    inv[h] = sum[h] == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum[h]);
    lse2[h] = sum[h] == 0.0f ? -INFINITY : __fadd_rn(__fsub_rn(top[h], kShift), log2f(sum[h]));
  }
  const long long slot0 = (long long)unit * kRows;
  const bool direct = parts <= 1;
  struct Place {
    long long out, lse;
  };
  auto place_of = [&](int row) {  // of the unit
    if (!direct) return Place{((slot0 + row) * p.split.splits + split) * D, (slot0 + row) * p.split.splits + split};
    const int pos = (int)share((uint32_t)(row0 + row), (uint32_t)r.group), h = head * r.group + (row0 + row) - pos * r.group;
    return Place{(long long)(seq.q0 + pos) * r.out_row_stride + (long long)h * r.out_head_stride,
                 (long long)(seq.q0 + pos) * r.kv_heads * r.group + h};
  };
  auto emit = [&](const Place& to, int ch, float a, float e) {
    if (direct)
      store2(r.out, to.out + ch, kType, a, e);
    else
      *reinterpret_cast<float2*>(p.split.out + to.out + ch) = make_float2(a, e);
  };
  auto emit_lse = [&](const Place& to, float l) {
    if (!direct)
      p.split.lse[to.lse] = l;
    else if (r.lse)
      r.lse[to.lse] = __fmul_rn(l, kLn2);
  };
  float* part = reinterpret_cast<float*>(smem) + (kg * WR + wr) * 16 * (D + 1);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = wr * 16 + g + 8 * h;
    if (row0 + row >= n_rows) continue;
    Place to = {};
    if (kGroups == 1) to = place_of(row);
#pragma unroll
    for (int i = 0; i < kOut; i += (kF32 ? 2 : 1)) {
      if constexpr (kF32) {
        // tiles i, i + 1: channels 8 i + 4 t + {0, 1} of column 2 t, + {2, 3} of column 2 t + 1
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = __fmul_rn(acc[i][2 * h + e], inv[h]), c = __fmul_rn(acc[i + 1][2 * h + e], inv[h]);
          const int ch = 8 * i + 4 * t + 2 * e;
          if (kGroups == 1) {
            emit(to, ch, a, c);
          } else {
            part[(g + 8 * h) * D + ch] = a;
            part[(g + 8 * h) * D + ch + 1] = c;
          }
        }
      } else {
        const float a = __fmul_rn(acc[i][2 * h], inv[h]), c = __fmul_rn(acc[i][2 * h + 1], inv[h]);
        const int ch = 8 * i + 2 * t;
        if (kGroups == 1) {
          emit(to, ch, a, c);
        } else {
          part[(g + 8 * h) * D + ch] = a;
          part[(g + 8 * h) * D + ch + 1] = c;
        }
      }
    }
    if (t == 0) {
      if (kGroups == 1)
        emit_lse(to, lse2[h]);
      else
        part[16 * D + g + 8 * h] = lse2[h];
    }
  }
  if constexpr (kF32) {
    // A value that rounds past the largest number, or an infinity, has no two
    // tf32 halves (its low part is an infinity or a NaN), and shifted weights
    // times values next to the largest may pass it: a row that is not finite
    // is computed again from its f32 numbers, key after key, a pair of
    // channels per lane.  That takes 30 times as long (1,024 x 1,024, 8 heads of
    // 64, every row: 2.0 ms instead of 67 us), and costs the other calls nothing
    // (64 single tokens: 10.3 us).
    uint32_t lost[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool finite = fabsf(sum[h]) < INFINITY;
#pragma unroll
      for (int i = 0; i < kOut; ++i) finite = finite && fabsf(acc[i][2 * h]) < INFINITY && fabsf(acc[i][2 * h + 1]) < INFINITY;
      lost[h] = __ballot_sync(kFull, !finite);
    }
    if (lost[0] | lost[1]) {
      __syncwarp();
#pragma unroll 1
      for (int own_row = 0; own_row < 16; ++own_row) {
        const int row = wr * 16 + own_row;
        if (row0 + row >= n_rows) break;
        if (!((own_row < 8 ? lost[0] : lost[1]) >> (4 * (own_row & 7)) & 15)) continue;
        constexpr int kPairs = (D + 63) / 64;
        const int pos = (int)share((uint32_t)(row0 + row), (uint32_t)r.group), qh = head * r.group + (row0 + row) - pos * r.group;
        const float* q = static_cast<const float*>(r.q) + (long long)(seq.q0 + pos) * r.q_row_stride + (long long)qh * r.q_head_stride;
        float2 qv[kPairs], o[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int ch = 64 * i + 2 * lane;
          qv[i] = ch < D ? *reinterpret_cast<const float2*>(q + ch) : make_float2(0.0f, 0.0f);
          o[i] = make_float2(0.0f, 0.0f);
        }
        // a NaN in the query leaves nothing to compute
        bool nan = false;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) nan = nan || qv[i].x != qv[i].x || qv[i].y != qv[i].y;
        if (__any_sync(kFull, nan)) continue;
        float most = -INFINITY, total = 0.0f;
#pragma unroll 1
        for (int at = 0; at < (end - begin) * kOwn; ++at) {
          const int key = (begin + at / kOwn) * kKeys + kg * kOwn + at % kOwn;
          if (key >= seq.nk || (mask && !mask[key])) continue;
          float2 v[kPairs];
          float x = 0.0f;
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const int ch = 64 * i + 2 * lane;
            v[i] = make_float2(0.0f, 0.0f);
            if (ch < D) {
              const float2 k2 = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(kbase) + (long long)key * p.k_rs + ch);
              v[i] = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(vbase) + (long long)key * p.v_rs + ch);
              x = __fmaf_rn(qv[i].y, k2.y, __fmaf_rn(qv[i].x, k2.x, x));
            }
          }
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) x = __fadd_rn(x, __shfl_xor_sync(kFull, x, d));
          x = __fmul_rn(x, factor);
          if (x > most) {
            const float shrink = most == -INFINITY ? 0.0f : exp2_approx(__fsub_rn(most, x));
            most = x;
            total = __fmul_rn(total, shrink);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) o[i] = make_float2(__fmul_rn(o[i].x, shrink), __fmul_rn(o[i].y, shrink));
          }
          const float w = x == -INFINITY ? 0.0f : exp2_approx(__fsub_rn(x, most));
          total = __fadd_rn(total, w);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) o[i] = make_float2(__fmaf_rn(w, v[i].x, o[i].x), __fmaf_rn(w, v[i].y, o[i].y));
        }
        const float share_of = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
        const float l = total == 0.0f ? -INFINITY : __fadd_rn(most, log2f(total));
        const Place to = kGroups == 1 ? place_of(row) : Place{};
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int ch = 64 * i + 2 * lane;
          if (ch >= D) continue;
          const float a = __fmul_rn(o[i].x, share_of), c = __fmul_rn(o[i].y, share_of);
          if (kGroups == 1) {
            emit(to, ch, a, c);
          } else {
            part[own_row * D + ch] = a;
            part[own_row * D + ch + 1] = c;
          }
        }
        if (lane == 0) {
          if (kGroups == 1)
            emit_lse(to, l);
          else
            part[16 * D + own_row] = l;
        }
      }
    }
  }
  if (kGroups == 1) return;
  __syncthreads();
  // ---- join the key groups: warp w takes every fourth row ----
  for (int row = warp; row < kRows && row0 + row < n_rows; row += 4) {
    const float* of = reinterpret_cast<const float*>(smem) + (row / 16) * 16 * (D + 1);
    constexpr int kStep = WR * 16 * (D + 1);
    float w[kGroups], best = -INFINITY, total = 0.0f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      w[k] = of[k * kStep + 16 * D + row % 16];
      best = fmaxf(best, w[k]);
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      w[k] = w[k] != w[k] ? w[k] : join_weight(w[k], best);
      total = __fadd_rn(total, w[k]);
    }
    const float scale = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    const Place to = place_of(row);
    for (int ch = 2 * lane; ch < D; ch += 64) {
      float a = 0.0f, e = 0.0f;
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
        if (w[k] != 0.0f) {
          a = __fmaf_rn(w[k], of[k * kStep + (row % 16) * D + ch], a);
          e = __fmaf_rn(w[k], of[k * kStep + (row % 16) * D + ch + 1], e);
        }
      emit(to, ch, __fmul_rn(a, scale), __fmul_rn(e, scale));
    }
    if (lane == 0) emit_lse(to, total == 0.0f ? -INFINITY : __fadd_rn(best, log2f(total)));
  }
}

// ---- shapes of a launch ----
struct CrossPlan {
  bool long_tiles;
  int tile_rows, row_tiles, splits, chunk, tile_keys;
  long long units, first;
  uint64_t slots, bytes;
};

bool cross_sizes_ok(const mc_cross_attention_args* a) {
  return a && dtype_bytes(a->dtype) != 0 && a->batch >= 0 && a->kv_heads >= 1 && a->heads >= 1 &&
         a->heads % a->kv_heads == 0 && a->head_dim >= 16 && a->head_dim <= kOpMaxHeadDim && a->head_dim % 16 == 0 &&
         a->max_q_len >= 0 && a->max_k_len >= 0 && a->max_k_len <= kOpMaxKeys && a->heads <= 65536 &&
         (int64_t)(a->heads / a->kv_heads) * a->max_q_len <= INT32_MAX / 2 &&
         (int64_t)a->batch * a->kv_heads <= INT32_MAX &&  // the product below stays within 64 bits
         (int64_t)a->batch * a->kv_heads * ((int64_t)(a->heads / a->kv_heads) * a->max_q_len / 16 + 1) <= INT32_MAX;
}

// Long tiles pay where the sequences' rows fill one of two on average: below,
// the small kernel's 16-row warps waste less.
bool long_fits(const mc_cross_attention_args* a, int64_t positions) {
  return a->dtype != MC_F32 && a->heads / a->kv_heads * positions >= kLongRows / 2 && a->max_k_len >= kLongKeys;
}
bool long_pays(const mc_cross_attention_args* a) {
  const int64_t mean = a->batch > 0 ? a->q_rows / a->batch : 0;
  return !a->key_mask && a->scale > 0.0f && cross_long_strides(a) && long_fits(a, mean < a->max_q_len ? mean : a->max_q_len);
}

// The most keys that one CTA sums.  In 16 bits a row's sum over its keys stays
// in the tensor cores' accumulator, whose additions cut off up to 2^-23 of it,
// once for 16 keys: 2^-13 of the output over 2^14 keys (f16) and 2^-10 over 2^17
// (bf16), a quarter of half a step of the type.  (f16, 262,144 keys of one sign in
// one range: 2e-3 too small.  Sums per tile in registers, as f32 has, cost the
// small tiles 20% at 2 x 1,024 x 2,048 and 5% on ragged sentences.)
int64_t most_keys(int32_t dtype) {
  return dtype == MC_F16 ? 1 << 14 : dtype == MC_BF16 ? 1 << 17 : INT32_MAX;
}

CrossPlan cross_plan(const mc_cross_attention_args* a, bool long_tiles) {
  CrossPlan plan;
  const int64_t rows = (int64_t)(a->heads / a->kv_heads) * a->max_q_len;
  plan.long_tiles = long_tiles;
  plan.tile_keys = long_tiles ? kLongKeys : a->dtype == MC_F32 ? 32 : 64;
  plan.tile_rows = long_tiles ? kLongRows : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  plan.row_tiles = (int)((rows + plan.tile_rows - 1) / plan.tile_rows);
  plan.units = (int64_t)a->batch * a->kv_heads * plan.row_tiles;
  // Ranges of keys for units too few to fill the GPU (one long CTA or three
  // small ones per SM), each of four tiles at least.
  const int tiles = (int)(((int64_t)a->max_k_len + plan.tile_keys - 1) / plan.tile_keys);
  // Long CTAs take one SM each, in waves; the last wave's units are cut too
  // where they are half of one or less (512 units of 64 tiles: four waves of
  // which the last is 68 units, 605 us; three and a half, 570 us).
  plan.first = 0;
  long long cut = plan.units;
  if (long_tiles && plan.units > kSms) {
    cut = plan.units % kSms;
    if (cut > kSms / 2) cut = 0;
    plan.first = plan.units - cut;
  }
  long long splits = cut > 0 ? kSms * (long_tiles ? 1 : 3) / cut : 1;
  if (splits > tiles / 4) splits = tiles / 4;
  const long long needed = (a->max_k_len + most_keys(a->dtype) - 1) / most_keys(a->dtype);
  if (needed > 1) plan.first = 0;  // no unit is whole
  if (splits < needed) splits = needed;
  if (splits > 256) splits = 256;
  if (plan.units > 0 && splits > INT32_MAX / plan.units) splits = INT32_MAX / plan.units;
  if (splits < 1) splits = 1;
  plan.chunk = tiles > 0 ? (int)((tiles + splits - 1) / splits) : 1;
  plan.splits = tiles > 0 ? (tiles + plan.chunk - 1) / plan.chunk : 1;
  if (plan.splits == 1) plan.first = 0;
  plan.slots = (uint64_t)(plan.units - plan.first) * plan.tile_rows;
  plan.bytes = attn_split_bytes(plan.slots, plan.splits, a->head_dim);
  return plan;
}

template <typename T, int D, int WR>
cudaError_t launch_small(const CrossParams& p, const CrossPlan& plan, cudaStream_t s) {
  static uint64_t done = 0;
  constexpr int bytes = cross_smem<T, D>();
  cudaError_t e = allow_smem(cross_small_kernel<T, D, WR>, bytes, &done);
  if (e != cudaSuccess) return e;
  return launch_pdl(cross_small_kernel<T, D, WR>, dim3((unsigned)plan.units, plan.splits), dim3(128), bytes, s, p);
}

template <typename T, int D>
cudaError_t launch_small_w(const CrossParams& p, const CrossPlan& plan, cudaStream_t s) {
  return plan.tile_rows == 16   ? launch_small<T, D, 1>(p, plan, s)
         : plan.tile_rows == 32 ? launch_small<T, D, 2>(p, plan, s)
                                : launch_small<T, D, 4>(p, plan, s);
}

template <int D>
cudaError_t launch_small_t(const CrossParams& p, const CrossPlan& plan, cudaStream_t s) {
  return p.rows.dtype == MC_F32   ? launch_small_w<float, D>(p, plan, s)
         : p.rows.dtype == MC_F16 ? launch_small_w<__half, D>(p, plan, s)
                                  : launch_small_w<__nv_bfloat16, D>(p, plan, s);
}

cudaError_t launch_small_d(const CrossParams& p, const CrossPlan& plan, cudaStream_t s) {
  switch (p.rows.head_dim) {
    case 16: return launch_small_t<16>(p, plan, s);
    case 32: return launch_small_t<32>(p, plan, s);
    case 48: return launch_small_t<48>(p, plan, s);
    case 64: return launch_small_t<64>(p, plan, s);
    case 80: return launch_small_t<80>(p, plan, s);
    case 96: return launch_small_t<96>(p, plan, s);
    case 112: return launch_small_t<112>(p, plan, s);
    case 128: return launch_small_t<128>(p, plan, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_cross(CrossParams p, const CrossPlan& plan, void* workspace, cudaStream_t s) {
  p.split.splits = plan.splits;
  p.split.chunk = plan.chunk;
  p.split.first = (uint32_t)plan.first;
  p.row_tiles = plan.row_tiles;
  if (plan.splits > 1) {
    p.split.out = static_cast<float*>(workspace);
    p.split.lse = p.split.out + plan.slots * plan.splits * p.rows.head_dim;
  }
  const cudaError_t e = plan.long_tiles ? launch_cross_long(p, plan.units, s) : launch_small_d(p, plan, s);
  if (e != cudaSuccess || plan.splits <= 1) return e;
  return launch_attn_join(p.rows, p.split, plan.tile_keys, plan.tile_rows, plan.row_tiles, s);
}

}  // namespace
}  // namespace mc

extern "C" uint64_t mc_cross_attention_workspace(const mc_cross_attention_args* args) {
  if (!mc::cross_sizes_ok(args)) return 0;
  // where both may run, which one goes by the strides, the mask and the rows in use
  const uint64_t small = mc::cross_plan(args, false).bytes;
  const uint64_t wide = mc::long_fits(args, args->max_q_len) ? mc::cross_plan(args, true).bytes : 0;
  return small > wide ? small : wide;
}

extern "C" mc_status mc_cross_attention(const mc_cross_attention_args* a, void* stream) {
  if (!mc::cross_sizes_ok(a) || !mc::scale_ok(a->scale) || a->q_rows < 0 || a->q_rows > INT32_MAX || a->k_rows < 0 ||
      a->k_rows > INT32_MAX)
    return MC_INVALID_INPUT;
  if (a->batch == 0 || a->max_q_len == 0) return MC_OK;
  const int bytes = mc::dtype_bytes(a->dtype);
  if (!a->q_start || !a->q_len || !a->k_start || !a->k_len || !mc::aligned4(a->q_start) || !mc::aligned4(a->q_len) ||
      !mc::aligned4(a->k_start) || !mc::aligned4(a->k_len) || !mc::aligned4(a->lse) ||
      !mc::strides_ok(a->q, a->q_rows, a->q_row_stride, a->q_head_stride, bytes) ||
      !mc::strides_ok(a->k, a->k_rows, a->k_row_stride, a->k_head_stride, bytes) ||
      !mc::strides_ok(a->v, a->k_rows, a->v_row_stride, a->v_head_stride, bytes) ||
      !mc::strides_ok(a->out, a->q_rows, a->out_row_stride, a->out_head_stride, bytes) ||
      !mc::strides_apart(a->q_rows, a->heads, a->head_dim, a->out_row_stride, a->out_head_stride) ||
      (a->out && (a->out == a->q || a->out == a->k || a->out == a->v)))
    return MC_INVALID_INPUT;
  const uint64_t need = mc_cross_attention_workspace(a);
  if (need > 0 && (!a->workspace || !mc::aligned16(a->workspace) || a->workspace_bytes < need)) return MC_INVALID_INPUT;
  const mc_status where = mc::on_current_device({a->q, a->k, a->v, a->out, a->lse, a->q_start, a->q_len, a->k_start, a->k_len,
                                                 a->key_mask, need > 0 ? a->workspace : nullptr});
  if (where != MC_OK) return where;
  uint32_t* status = mc::op_status_word();
  if (!status) return MC_CUDA;
  mc::CrossParams p;
  std::memset(&p, 0, sizeof(p));
  mc::AttnRows& r = p.rows;
  r.q = a->q;
  r.out = a->out;
  r.lse = a->lse;
  r.q_start = a->q_start;
  r.q_len = a->q_len;
  r.k_len = a->k_len;
  r.k_start = a->k_start;
  r.q_rows = a->q_rows;
  r.k_rows = a->k_rows;
  r.q_row_stride = a->q_row_stride;
  r.q_head_stride = a->q_head_stride;
  r.out_row_stride = a->out_row_stride;
  r.out_head_stride = a->out_head_stride;
  r.dtype = a->dtype;
  r.batch = a->batch;
  r.kv_heads = a->kv_heads;
  r.group = a->heads / a->kv_heads;
  r.head_dim = a->head_dim;
  r.max_q = a->max_q_len;
  r.max_k = a->max_k_len;
  p.k = a->k;
  p.v = a->v;
  p.k_rs = a->k_row_stride;
  p.k_hs = a->k_head_stride;
  p.v_rs = a->v_row_stride;
  p.v_hs = a->v_head_stride;
  p.mask = a->key_mask;
  p.scale = a->scale;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorNotSupported;
  if (mc::long_pays(a)) e = mc::launch_cross(p, mc::cross_plan(a, true), a->workspace, s);
  if (e == cudaErrorNotSupported) e = mc::launch_cross(p, mc::cross_plan(a, false), a->workspace, s);
  return mc::launched(e);
}
