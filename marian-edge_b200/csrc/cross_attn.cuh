// cross_attn.cuh -- the launch parameters of mc_cross_attention's kernels.
#pragma once

#include "decode_ops.cuh"

namespace mc {

struct CrossParams {
  AttnRows rows;
  AttnSplit split;
  const void *k, *v;
  long long k_rs, k_hs, v_rs, v_hs;
  const uint8_t* mask;
  float scale;
  int row_tiles;
  uint32_t* status;
};

// Long sequences on the 5th-generation tensor cores (cross_attn_long.cu):
// 256 query rows and 128 keys a tile, 16-bit types, no mask, scale > 0.
constexpr int kLongRows = 256;
constexpr int kLongKeys = 128;

// Whether the rows of k and v can be described by a tensor map.
bool cross_long_strides(const mc_cross_attention_args* a);
// cudaErrorNotSupported: the driver took no tensor map of k or v; nothing ran.
cudaError_t launch_cross_long(const CrossParams& p, long long units, cudaStream_t s);

}  // namespace mc
