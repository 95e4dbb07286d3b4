// Host-side launch parameters of the prompt key-weight kernel (key_weights.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace sisa {

struct KeyWeightParams {
  const char* q; int64_t q_sb, q_sh, q_sl;   // (B, H, L, 64) views, low precision
  const char* k; int64_t k_sb, k_sh, k_sl;
  const char* c; int64_t c_sb, c_sh, c_sl;   // (B, H, L, 32)
  const char* b; int64_t b_sb, b_sh, b_sl;
  const float* pos;                          // (B*H, 4, Lp) planes {g, F, rowf, colf}
  const float* lam;
  const float* lse;                          // (B, H, L) log2 units
  float* w;                                  // (B, H, L)
  int B, H, L, Lp, first;
  int32_t* status;
};

cudaError_t launch_key_weights(const KeyWeightParams& p, int dtype, cudaStream_t st);

}  // namespace sisa
