// Log probabilities of tokens from logits: the kernels' launcher (k_logp.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace grx {

constexpr int kLogpMaxTop = 32;

struct LogpArgs {
  const void* x = nullptr;  // [rows], row r at r·stride
  int64_t stride = 0;
  int rows = 0, vocab = 0, top = 0;
  const int* targets = nullptr;  // [rows]
  float *logprob = nullptr, *entropy = nullptr;  // [rows]
  int* ids = nullptr;                            // [rows][top]
  float* lps = nullptr;                          // [rows][top]
};

// type: 0 float32, 1 float16, 30 bfloat16.
cudaError_t launch_logp(const LogpArgs& a, int type, cudaStream_t st);

}  // namespace grx
