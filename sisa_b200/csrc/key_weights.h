// Host-side launch parameters of the prompt key-weight kernel (key_weights.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace sisa {

struct KeyWeightParams {
  CUtensorMap tm_k;    // (64, L, H, B) bf16/fp16, box (64, 128), 128B swizzle
  CUtensorMap tm_b;    // (32, L, H, B), box (32, 128), 64B swizzle
  CUtensorMap tm_q;    // box (64, 64), 128B swizzle
  CUtensorMap tm_c;    // box (32, 64), 64B swizzle
  CUtensorMap tm_pos;  // (L, 4, B*H) fp32 planes, box (64, 4, 1)
  const float* pos;    // (B*H, 4, Lp) planes {g, F, rowf, colf}
  const float* lam;
  const float* lse;    // (B, H, L) log2 units
  float* w;            // (B, H, L)
  int B, H, L, Lp, first, ntk;
  int32_t* status;
};

cudaError_t launch_key_weights(const KeyWeightParams& p, int dtype, cudaStream_t st);

}  // namespace sisa
