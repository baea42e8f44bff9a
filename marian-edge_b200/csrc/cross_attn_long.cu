// cross_attn_long.cu -- mc_cross_attention for long sequences: tcgen05 MMAs
// with accumulators in TMEM, fed by TMA.
//
// One CTA per unit (sequence, key/value head, 256 query rows) and key range.
// Its rows are two tiles of 128, whose steps alternate on the tensor pipe:
// while one tile's weights are computed, the other's products run.
//   S_i [128 x 128 keys]  = Q_i K_j^T   (both K-major in shared memory)
//   O_i [128 x head_dim] += W_i V_j     (W_i from TMEM, V_j as it lies, N-major)
// Warp 0 loads K and V tiles through a ring, warp 1 issues the MMAs, warps
// 4-7 and 8-11 hold one query row per thread of tile 0 and 1: they read S_i,
// keep the row's maximum and sum, and write the weights, rounded to the
// type, over S_i.  O_i is only rescaled when a maximum grows by more than 8
// (in powers of two): the weights stay below 2^8 (f16: 2^15, by weight_shift),
// and their sum is as stale.
//
// What bounds it: with M = N = 128 the tensor pipe, one issuing warp's round
// through its barriers between the products of a step, and the exponentials
// (16 a cycle) share the time.  Measured at 2 x 4,096 x 8,192, 16 heads of 128,
// bf16 (329 us at the measured GEMM rate): MMAs without weights 514 us; a
// quarter of the exponentials by a polynomial on the FMA pipe 4% slower; the
// weights handed over by halves 2% slower; votes after the MMA warp's waits 3%
// slower; K and V in stages of their own, and an arrival for every product,
// 10% slower; a stage peeked at with try_wait, whose suspension takes some
// hundred cycles, 20% slower.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cstring>

#include "cross_attn.cuh"

namespace mc {
namespace {

constexpr uint32_t kFull = 0xFFFFFFFFu;
constexpr int kThreads = 384;
constexpr int kTileBytes = 128 * 128;  // 128 rows of 64 channels
constexpr float kGrowth = 8.0f;
// f16 weights are taken 2^7 larger, so that those down to 2^-21 of a row's
// maximum are normal numbers and only those below 2^-32 are lost: in a long tail
// behind one key they count together.  With the growth they stay below 2^15.
// bf16 has f32's range.
constexpr float weight_shift(bool bf16) { return bf16 ? 0.0f : 7.0f; }

constexpr int chunks_of(int d) { return (d + 63) / 64; }
// Ring stages, each for the V tile of one step and the K tile of the next,
// which the MMAs of a step read together.
constexpr int stages_of(int d) { return d > 64 ? 2 : 4; }
constexpr int long_smem(int d) { return (2 + 2 * stages_of(d)) * chunks_of(d) * kTileBytes + 1024 + 256; }

struct Barriers {
  uint64_t full[4], empty[4];
  uint64_t k0_full, k0_done, q_ready, s_full[2], w_ready[2], o_done[2], v_clean;
  uint32_t tmem, stop;
};

// Bounded wait that also ends when another warp has given up.
__device__ __forceinline__ bool wait_for(Barriers* b, uint64_t* bar, uint32_t phase, uint32_t* status) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if ((i & 63) == 63 && *reinterpret_cast<volatile uint32_t*>(&b->stop)) return false;
  }
  flag_status(status, kStatusWaitTimeout);
  *reinterpret_cast<volatile uint32_t*>(&b->stop) = 1;
  return false;
}

// The same for a whole warp, whose lanes agree on what came out.
__device__ __forceinline__ bool warp_wait(Barriers* b, uint64_t* bar, uint32_t phase, uint32_t* status) {
  return __all_sync(kFull, wait_for(b, bar, phase, status));
}

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// B operand whose N (channels) is contiguous: 64-channel chunks `chunk` bytes
// apart, groups of 8 keys 1,024 bytes apart, 128-byte swizzle.
__device__ __forceinline__ uint64_t sdesc_n_sw128(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)(kTileBytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Instruction descriptor: 16-bit operands of one type, f32 sums, M = 128.
__host__ __device__ constexpr uint32_t idesc_16(int n, bool bf16, bool b_n_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_n_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// True in one lane of a converged warp.  MMAs are issued under it by warps
// that run their control flow whole: their descriptors then stay in uniform
// registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    cross_long_kernel(const CrossParams p, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
  constexpr int kChunks = chunks_of(D), kStages = stages_of(D), kSteps = D / 16;
  constexpr float kShift = weight_shift(BF16);
  constexpr uint32_t kS0 = 0, kO0 = 256;  // TMEM columns: S_i at 128 i, O_i at 256 + 128 i
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* ring = smem + 2 * kChunks * kTileBytes;
  Barriers* bar = reinterpret_cast<Barriers*>(ring + 2 * kStages * kChunks * kTileBytes);
  const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    mbar_init(&bar->k0_full, 1);
    mbar_init(&bar->k0_done, 1);
    mbar_init(&bar->q_ready, 8);
    mbar_init(&bar->v_clean, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->w_ready[i], 4);
      mbar_init(&bar->o_done[i], 1);
    }
    bar->stop = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&bar->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(kFull, bar->tmem, 0);
  pdl_enter();

  const AttnRows& r = p.rows;
  // Whole units first, then the cut ones, range by range.
  const uint32_t cut_block = blockIdx.x < p.split.first ? 0 : blockIdx.x - p.split.first;
  const bool whole = blockIdx.x < p.split.first;
  const uint32_t nth = cut_block / (uint32_t)p.split.splits, unit = whole ? blockIdx.x : p.split.first + nth;
  const uint32_t bh = unit / (uint32_t)p.row_tiles;
  const int tile = (int)(unit - bh * p.row_tiles), b = (int)(bh / (uint32_t)r.kv_heads), head = (int)(bh - (uint32_t)b * r.kv_heads);
  const int split = whole ? 0 : (int)(cut_block - nth * p.split.splits);
  const AttnSeq seq = attn_seq(r, b, p.status, head == 0 && tile == 0 && split == 0 && threadIdx.x == 0);
  const int n_rows = seq.nq * r.group, row0 = tile * kLongRows;
  const int n_tiles = (seq.nk + kLongKeys - 1) / kLongKeys;
  const int chunk = whole ? max(n_tiles, 1) : p.split.chunk, parts = max(1, (n_tiles + chunk - 1) / chunk);
  const bool live = seq.ok && row0 < n_rows && split < parts;
  const int begin = split * chunk, end = live ? min(n_tiles, begin + chunk) : begin;
  const int steps = end - begin;
  const int row_tiles = row0 + 128 < n_rows ? 2 : 1;
  const int spare = steps > 0 ? max(0, end * kLongKeys - seq.nk) : 0;  // keys of the last tile behind the sequence

  if (warp == 0 && steps > 0) {
    // ---- loads: K_0 (where the last stage's K goes later), then V_j with K_{j+1} ----
    constexpr int kPart = kChunks * kTileBytes;  // a stage: V, then K
    auto load = [&](uint8_t* to, const CUtensorMap* map, bool by_head, int step, uint64_t* full) {
      const int row = seq.k0 + (begin + step) * kLongKeys;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) tma_load_3d(to + c * kTileBytes, map, 64 * c, by_head ? head : 0, row, full);
    };
    if (lane == 0) {
      mbar_arrive_expect_tx(&bar->k0_full, kPart);
      load(ring + (2 * kStages - 1) * kPart, &k_map, p.k_hs != 0, 0, &bar->k0_full);
    }
    bool ok = true;
    int j = 0;
    for (; j < steps; ++j) {
      const int st = j % kStages;
      if (j >= kStages) ok = warp_wait(bar, &bar->empty[st], (j / kStages - 1) & 1, p.status);
      if (ok && j == kStages - 1) ok = warp_wait(bar, &bar->k0_done, 0, p.status);
      if (!ok) break;
      if (lane == 0) {
        const bool more = j + 1 < steps;
        mbar_arrive_expect_tx(&bar->full[st], more ? 2 * kPart : kPart);
        load(ring + 2 * st * kPart, &v_map, p.v_hs != 0, j, &bar->full[st]);
        if (more) load(ring + (2 * st + 1) * kPart, &k_map, p.k_hs != 0, j + 1, &bar->full[st]);
      }
      __syncwarp();
    }
    if (ok && spare) {
      // The rows behind the sequence are the next one's, or anything: a
      // weight of 0 times an infinity would be NaN.
      const int st = (steps - 1) % kStages;
      ok = warp_wait(bar, &bar->full[st], ((steps - 1) / kStages) & 1, p.status);
      uint8_t* v = ring + 2 * st * kPart + (128 - spare) * 128;
      for (int i = lane; i < spare * 8; i += 32)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) *reinterpret_cast<uint4*>(v + c * kTileBytes + i * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) arrive(&bar->v_clean);
    }
    if (!ok) {  // let the loads in flight land before the block leaves
      for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&bar->k0_full, 0); ++i) {
      }
      for (int k = max(0, j - kStages); k < min(j, steps); ++k)
        for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&bar->full[k % kStages], (k / kStages) & 1); ++i) {
        }
    }
  } else if (warp == 1 && steps > 0) {
    // ---- MMAs ----
    // One lane issues them all, and the tensor pipe waits for it: every
    // descriptor is a base plus a constant (16-byte units; shared memory
    // addresses need no carry), and the next stage is waited for while the
    // pipe has tile 0's products before it.  An arrival on s_full also says
    // that the tile's product before it is done, as one thread's MMAs are.
    constexpr uint32_t kIdescS = idesc_16(128, BF16, false), kIdescO = idesc_16(D, BF16, true);
    constexpr uint32_t kPart = kChunks * kTileBytes / 16;
    const int n = __shfl_sync(kFull, steps, 0), tiles = __shfl_sync(kFull, row_tiles, 0);
    const bool cut = __shfl_sync(kFull, spare, 0) > 0;
    const uint64_t q_desc = sdesc_k_sw128(smem_u32(q_smem)), k_desc = sdesc_k_sw128(smem_u32(ring)),
                   v_desc = sdesc_n_sw128(smem_u32(ring));
    auto scores = [&](int i, int stage) {
      const uint64_t q = q_desc + i * kPart, k = k_desc + (2 * stage + 1) * kPart;
      const uint32_t d = tmem + kS0 + 128 * i;
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint32_t at = ((s / 4) * kTileBytes + (s % 4) * 32) / 16;
          mma_ss(d, q + at, k + at, kIdescS, s > 0);
        }
        mma_commit(&bar->s_full[i]);
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* b) {
      if (elect_one()) mma_commit(b);
      __syncwarp();
    };
    // A wait that gave up has set `stop`, which ends the others at once: the
    // warp runs on, through MMAs on whatever is there, to the end.
    auto wait = [&](uint64_t* b, int phase) { wait_for(bar, b, phase, p.status); };
    auto stage_ready = [&](int j) {
      wait(&bar->full[j % kStages], (j / kStages) & 1);
      if (j + 1 == n && cut) wait(&bar->v_clean, 0);
    };
    wait(&bar->q_ready, 0);
    wait(&bar->k0_full, 0);
    tc_fence_after();
    for (int i = 0; i < tiles; ++i) scores(i, kStages - 1);
    commit(&bar->k0_done);
    stage_ready(0);
    for (int j = 0; j < n; ++j) {
      const int st = j % kStages;
      const uint64_t v = v_desc + 2 * st * kPart;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= tiles) break;
        const uint32_t d = tmem + kO0 + 128 * i, w = tmem + kS0 + 128 * i;
        wait(&bar->w_ready[i], j & 1);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 8; ++s) mma_ts(d, w + 8 * s, v + s * 128, kIdescO, j > 0 || s > 0);
        }
        __syncwarp();
        if (j + 1 < n) {
          scores(i, st);
          if (i == 0) stage_ready(j + 1);
        } else {
          commit(&bar->o_done[i]);
        }
      }
      commit(&bar->empty[st]);
    }
    // the last arrival lands before the block, and its barriers, are gone
    wait(&bar->empty[(n - 1) % kStages], ((n - 1) / kStages) & 1);
  } else if (warp >= 4 && live) {
    // ---- one query row per thread ----
    const int i = (warp - 4) >> 2, quarter = warp & 3, row_in = quarter * 32 + lane, row = row0 + 128 * i + row_in;
    const bool there = row < n_rows;
    const int pos = there ? row / r.group : 0, h = head * r.group + (there ? row - pos * r.group : 0);
    {
      // the row of Q into its swizzled place: 16-byte chunk c of line l at c ^ (l % 8)
      const uint16_t* src = static_cast<const uint16_t*>(r.q) + (long long)(seq.q0 + pos) * r.q_row_stride + (long long)h * r.q_head_stride;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = there ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(q_smem + (i * kChunks + c / 8) * kTileBytes + row_in * 128 + (((c & 7) ^ (row_in & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) arrive(&bar->q_ready);
    }
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lanes + kS0 + 128 * i, o_addr = tmem + lanes + kO0 + 128 * i;
    const float factor = __fmul_rn(p.scale, kLog2e);
    float top = -INFINITY, sum = 0.0f;
    const bool used = steps > 0 && i < row_tiles;
    bool ok = true;  // no wait gave up; the steps run on if one did, and the row is not written
    for (int j = 0; used && j < steps; ++j) {
      ok = wait_for(bar, &bar->s_full[i], j & 1, p.status) && ok;
      __syncwarp();
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + 32 * c, s[c]);
      tmem_ld_wait();
      if (spare && j + 1 == steps) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (32 * c + k >= 128 - spare) s[c][k] = 0xFF800000u;
      }
      float most[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        most[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
        for (int k = 2; k < 32; k += 2) most[c] = max3(most[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
      }
      const float high = max3(fmaxf(most[0], most[1]), most[2], most[3]);
      // a row goes by its own maximum alone, so that no other row of the warp
      // (a NaN one, a batch's neighbour) has a part in its roundings
      const bool grows = __fmul_rn(__fsub_rn(high, top), factor) > kGrowth;
      if (__any_sync(kFull, grows)) {
        const float shrink = !grows ? 1.0f : top == -INFINITY ? 0.0f : exp2_approx(__fmul_rn(__fsub_rn(top, high), factor));
        if (grows) top = high;
        sum = __fmul_rn(sum, shrink);
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_x16(o_addr + 16 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__fmul_rn(__uint_as_float(o[k]), shrink));
            tmem_st_x16(o_addr + 16 * c, o);
          }
        }
      }
      const float base = top == -INFINITY ? 0.0f : BF16 ? __fmul_rn(-top, factor) : __fmaf_rn(-top, factor, kShift);
      const uint64_t factor2 = pair(factor, factor), base2 = pair(base, base);
      uint64_t add[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint64_t x = fma2(pair(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1])), factor2, base2);
          float a, e;
          unpair(x, a, e);
          a = exp2_approx(a);
          e = exp2_approx(e);
          add[k & 1] = add2(add[k & 1], pair(a, e));
          w[k] = BF16 ? pack_bf16(a, e) : pack_f16(a, e);
        }
        tmem_st_x16(s_addr + 16 * c, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive(&bar->w_ready[i]);
      float a0, a1;
      unpair(add2(add[0], add[1]), a0, a1);
      sum = __fadd_rn(sum, __fadd_rn(a0, a1));
    }
    if (used) ok = wait_for(bar, &bar->o_done[i], 0, p.status) && ok;
    const bool written = i < row_tiles && ok && there;
    // ---- the row, normalized ----
    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    const float lse2 = sum == 0.0f ? -INFINITY : __fadd_rn(BF16 ? __fmul_rn(top, factor) : __fmaf_rn(top, factor, -kShift), log2f(sum));
    const bool direct = parts <= 1;
    const long long slot = ((long long)nth * kLongRows + 128 * i + row_in) * p.split.splits + split;
    __syncwarp();
    tc_fence_after();
    {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        __syncwarp();
        if (used) {
          tmem_ld_x16(o_addr + 16 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0;
        }
        float f[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) f[k] = __fmul_rn(__uint_as_float(o[k]), inv);
        if (direct && written) {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = BF16 ? pack_bf16(f[2 * k], f[2 * k + 1]) : pack_f16(f[2 * k], f[2 * k + 1]);
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(r.out) + (long long)(seq.q0 + pos) * r.out_row_stride +
                                                (long long)h * r.out_head_stride + 16 * c);
          dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
          dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else if (written) {
          float4* dst = reinterpret_cast<float4*>(p.split.out + slot * D + 16 * c);
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[k] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
        }
      }
      if (written) {
        if (!direct)
          p.split.lse[slot] = lse2;
        else if (r.lse)
          r.lse[(long long)(seq.q0 + pos) * r.kv_heads * r.group + h] = __fmul_rn(lse2, kLn2);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(found ? ptr : nullptr);
  }();
  return fn;
}

// {channels, heads, rows} of k or v, boxes of 64 channels of one head and 128
// rows; channels past head_dim and rows past the last come as zeros.  Heads
// that share one row (a stride of 0) are one head there.
bool encode_rows(CUtensorMap* map, const void* base, const AttnRows& r, long long row_stride, long long head_stride) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)r.head_dim, (cuuint64_t)(head_stride ? r.kv_heads : 1), (cuuint64_t)r.k_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)(head_stride ? head_stride : r.head_dim) * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, 1, kLongKeys}, steps[3] = {1, 1, 1};
  return fn(map, r.dtype == MC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16>
cudaError_t launch_long(const CrossParams& p, long long units, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  static uint64_t done = 0;
  cudaError_t e = allow_smem(cross_long_kernel<D, BF16>, long_smem(D), &done);
  if (e != cudaSuccess) return e;
  return launch_pdl(cross_long_kernel<D, BF16>, dim3((unsigned)(p.split.first + (units - p.split.first) * p.split.splits)), dim3(kThreads), long_smem(D), s, p, k, v);
}

template <int D>
cudaError_t launch_long_t(const CrossParams& p, long long units, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  return p.rows.dtype == MC_BF16 ? launch_long<D, true>(p, units, k, v, s) : launch_long<D, false>(p, units, k, v, s);
}

}  // namespace

bool cross_long_strides(const mc_cross_attention_args* a) {
  return a->k_rows > 0 && a->k_row_stride >= a->head_dim && a->v_row_stride >= a->head_dim;
}

cudaError_t launch_cross_long(const CrossParams& p, long long units, cudaStream_t s) {
  CUtensorMap k, v;
  if (!encode_rows(&k, p.k, p.rows, p.k_rs, p.k_hs) || !encode_rows(&v, p.v, p.rows, p.v_rs, p.v_hs))
    return cudaErrorNotSupported;
  switch (p.rows.head_dim) {
    case 16: return launch_long_t<16>(p, units, k, v, s);
    case 32: return launch_long_t<32>(p, units, k, v, s);
    case 48: return launch_long_t<48>(p, units, k, v, s);
    case 64: return launch_long_t<64>(p, units, k, v, s);
    case 80: return launch_long_t<80>(p, units, k, v, s);
    case 96: return launch_long_t<96>(p, units, k, v, s);
    case 112: return launch_long_t<112>(p, units, k, v, s);
    case 128: return launch_long_t<128>(p, units, k, v, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mc
