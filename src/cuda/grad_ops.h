// Host-callable launchers of the kernels that work on a training step's
// gradients: the norm of a list of tensors, clipping, and the embedding table.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "ibcomm/tunables.h"

namespace ibcomm {

// A launch whose blocks wait for one another, refused where they do not fit on the
// GPU at once: a process may have been given a part of it.  The callers then take
// kernels that do not wait, or a smaller grid.  IBCOMM_COOPERATIVE_CTAS: the
// largest such grid, where the runtime does not know of the part.
template <typename... Params, typename... Args>
cudaError_t LaunchTogether(void (*kernel)(Params...), int blocks, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  const int most = Tunable("IBCOMM_COOPERATIVE_CTAS", -1);
  if (most >= 0 && blocks > 1 && blocks > most) return cudaErrorCooperativeLaunchTooLarge;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeCooperative;
  attribute.val.cooperative = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
  if (e == cudaErrorCooperativeLaunchTooLarge) cudaGetLastError();  // it is dealt with
  return e;
}

// ---- norm of a list of tensors, and clipping (grad_norm_kernel.cu) ----
// Partial sums that a call may need room for (doubles of its workspace).
constexpr int kNormPartials = 2048;

struct GradTensor {
  const void* in;
  void* out;  // of the clipped values; null where only the norm is asked for
  uint64_t n;
  int32_t dtype_in;
  int32_t dtype_out;
};

enum class GradPower : int32_t { kMax = 0, kTwo = 2 };

struct GradNormParams {
  const GradTensor* tensors;
  int count;
  GradPower power;
  double* work;           // kNormPartials doubles on the device
  const double* sums;     // `num_sums` sums (or maxima) to take instead of those of the tensors; null: the tensors'
  int num_sums;
  void* norm;             // where the norm goes (float, or double with norm_is_double); may be null
  int norm_is_double;
  double* sum;            // where the sum of squares (or the maximum) goes; may be null
  bool clip;
  double max_norm;
};
cudaError_t LaunchGradNorm(const GradNormParams& p, cudaStream_t stream);

// ---- embedding (embedding_kernel.cu) ----
struct EmbeddingParams {
  const void* tokens;
  int tokens_are_64;
  uint64_t num_tokens;
  const void* weight;
  uint64_t rows;
  uint64_t width;
  int dtype_weight;
  void* out;
  int dtype_out;
  double scale;
};
cudaError_t LaunchEmbedding(const EmbeddingParams& p, cudaStream_t stream);

struct EmbeddingGradParams {
  const void* tokens;
  int tokens_are_64;
  uint64_t num_tokens;
  const void* grad;  // num_tokens x width
  int dtype_grad;
  void* out;  // rows x width
  int dtype_out;
  uint64_t rows;
  uint64_t width;
  int64_t padding;  // row without a gradient, -1 = none
  double scale;
  bool accumulate;
  void* work;
  size_t work_bytes;
};
// Bytes of workspace that LaunchEmbeddingGrad needs.
size_t EmbeddingGradWorkBytes(uint64_t num_tokens, uint64_t rows, uint64_t width);
cudaError_t LaunchEmbeddingGrad(const EmbeddingGradParams& p, cudaStream_t stream);

}  // namespace ibcomm
