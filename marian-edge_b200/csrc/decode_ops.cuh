// decode_ops.cuh -- what the decode-step operators (4-bit cache, cross
// attention, sampling) share: typed rows, the split-key partial results and
// the checks of the C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include <initializer_list>

#include "common.cuh"
#include "marian_cuda.h"

namespace mc {

// The operator API's status word on the current device (ops_capi.cu);
// nullptr when there is none to be had.
uint32_t* op_status_word();

constexpr int kSms = 148;
constexpr int kOpMaxHeadDim = 128;
constexpr int kOpMaxKeys = INT32_MAX - 255;  // of a sequence: positions a tile further on still are an int
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ---- typed values -------------------------------------------------------------
__device__ __forceinline__ float2 unpack_f16(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two neighbouring values at element i (even) of a row of the given type.
__device__ __forceinline__ float2 load2(const void* row, long long i, int dtype) {
  if (dtype == MC_F32) return *reinterpret_cast<const float2*>(static_cast<const float*>(row) + i);
  const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(row) + i);
  return dtype == MC_F16 ? unpack_f16(w) : unpack_bf16(w);
}
__device__ __forceinline__ void store2(void* row, long long i, int dtype, float a, float b) {
  if (dtype == MC_F32) {
    *reinterpret_cast<float2*>(static_cast<float*>(row) + i) = make_float2(a, b);
  } else {
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(row) + i) = dtype == MC_F16 ? pack_f16(a, b) : pack_bf16(a, b);
  }
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- pairs of f32 (one instruction, two lanes) ----
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// D (+)= A B for m16n8k16 with f16 or bf16 operands and f32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- attention rows ---------------------------------------------------------------
// The query rows of one sequence and one key/value head, row i = position
// i / group of the sequence, query head kv_head * group + i % group.
struct AttnRows {
  const void* q;
  void* out;
  float* lse;
  const int32_t* q_start;
  const int32_t* q_len;
  const int32_t* k_len;    // keys of each sequence
  const int32_t* k_start;  // first key row of each sequence; nullptr for a cache
  long long q_rows, k_rows;
  long long q_row_stride, q_head_stride, out_row_stride, out_head_stride;
  int dtype, batch, kv_heads, group, head_dim, max_q, max_k, causal;
};

// a / d for the divisors that are mostly 1 (heads of a group, row tiles): a
// division is some twenty instructions, and a short unit has several.
__device__ __forceinline__ uint32_t share(uint32_t a, uint32_t d) { return d == 1 ? a : a / d; }

struct AttnSeq {
  int q0, nq, k0, nk;
  bool ok;
};

// The bounds check of one sequence's lengths: a sequence that fails it is
// reported and left alone.
__device__ __forceinline__ AttnSeq attn_seq(const AttnRows& r, int b, uint32_t* status, bool report) {
  AttnSeq s;
  s.q0 = r.q_start[b];
  s.nq = r.q_len[b];
  s.nk = r.k_len[b];
  s.k0 = r.k_start ? r.k_start[b] : 0;
  s.ok = s.q0 >= 0 && s.nq >= 0 && s.nq <= r.max_q && (long long)s.q0 + s.nq <= r.q_rows && s.nk >= 0 &&
         s.nk <= r.max_k && s.k0 >= 0 && (!r.k_start || (long long)s.k0 + s.nk <= r.k_rows);
  if (!s.ok) {
    if (report) flag_status(status, kStatusBadIndex);
    s.nq = 0;
  }
  return s;
}

// ---- split keys -----------------------------------------------------------------
// When there are too few (sequence, head, row tile) units to fill the GPU,
// the keys of a unit are cut into ranges of `chunk` tiles, one CTA each;
// every range writes its normalized rows and their log2-sum-exp2, and
// attn_join averages them.  A sequence whose keys fit one range writes its
// rows at once, and attn_join leaves it alone.  Units before `first` are
// whole: a launch may cut its last ones only.
struct AttnSplit {
  float* out;  // [(units - first) * rows][splits][head_dim]
  float* lse;  // [(units - first) * rows][splits], base 2
  int splits, chunk;
  uint32_t first;
};

cudaError_t launch_attn_join(const AttnRows& r, const AttnSplit& s, int tile_keys, int unit_rows, int row_tiles,
                             cudaStream_t stream);

inline uint64_t attn_split_bytes(uint64_t slots, int splits, int head_dim) {
  return splits <= 1 ? 0 : slots * (uint64_t)splits * ((uint64_t)head_dim + 1) * sizeof(float);
}

// The weight of a key range in a join: 2^(its log2 sum - the largest one).
__device__ __forceinline__ float join_weight(float l, float top) {
  return l == -INFINITY ? 0.0f : exp2f(__fsub_rn(l, top));
}

// ---- host checks ------------------------------------------------------------------
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
inline int dtype_bytes(int32_t dtype) { return dtype == MC_F32 ? 4 : dtype == MC_F16 || dtype == MC_BF16 ? 2 : 0; }

// The scale of scores in powers of two has to be a number.
inline bool scale_ok(float scale) { return isfinite(scale * kLog2e); }

// Memory of another device or pageable host memory is refused, for every
// pointer that is given (70 ns each); memory that CUDA says nothing about
// cannot be read by a kernel either.
inline mc_status on_current_device(std::initializer_list<const void*> pointers) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return MC_CUDA;
  for (const void* p : pointers) {
    if (!p) continue;
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
      cudaGetLastError();
      return MC_INVALID_INPUT;
    }
    const bool ours = a.type == cudaMemoryTypeDevice ? a.device == dev
                                                     : a.type == cudaMemoryTypeManaged ||
                                                           (a.type == cudaMemoryTypeHost && a.devicePointer == p);
    if (!ours) return MC_INVALID_INPUT;
  }
  return MC_OK;
}

// A launch's outcome; its error does not stay behind for the caller's own calls.
inline mc_status launched(cudaError_t e) {
  if (e == cudaSuccess) return MC_OK;
  cudaGetLastError();
  return MC_CUDA;
}

// Rows of head_dim values whose strides keep every 16-byte load aligned.  No
// rows need no address: an empty tensor's is often null.
constexpr int64_t kOpMaxStride = int64_t(1) << 40;
inline bool strides_ok(const void* base, int64_t rows, int64_t row_stride, int64_t head_stride, int bytes) {
  return (base || rows == 0) && aligned16(base) && row_stride >= 0 && head_stride >= 0 && row_stride < kOpMaxStride &&
         head_stride < kOpMaxStride && (row_stride * bytes) % 16 == 0 && (head_stride * bytes) % 16 == 0;
}

// Written rows must not overlap each other: either the heads of a row lie
// within the row's stride, or the rows of a head within the head's.  (2^31 rows
// or heads times a stride pass 64 bits.)
inline bool strides_apart(int64_t rows, int64_t heads, int64_t head_dim, int64_t row_stride, int64_t head_stride) {
  const bool head_ok = heads <= 1 || head_stride >= head_dim;
  const bool row_ok = rows <= 1 || row_stride >= head_dim;
  if (!head_ok || !row_ok) return false;
  if (rows <= 1 || heads <= 1) return true;
  return row_stride >= static_cast<__int128>(heads - 1) * head_stride + head_dim ||
         head_stride >= static_cast<__int128>(rows - 1) * row_stride + head_dim;
}

// Raises a kernel's dynamic shared memory limit, once per device.
template <typename K>
inline cudaError_t allow_smem(K kernel, size_t bytes, uint64_t* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (__atomic_load_n(done, __ATOMIC_ACQUIRE) >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < 64) __atomic_fetch_or(done, uint64_t(1) << dev, __ATOMIC_RELEASE);
  return e;
}

}  // namespace mc
