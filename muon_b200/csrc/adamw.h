// Internal interface of the multi-tensor AdamW kernels (adamw.cu): the step with 32-bit and with
// 8-bit moments, the global gradient norm, scaling by a device-side factor, and the conversion of
// moments between 32 and 8 bits. Tensor tables travel in the kernel arguments (up to 32764 bytes),
// so a call allocates nothing and copies nothing before its launch.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mb {

constexpr int kStateBlock = 256;  // elements of a flattened tensor that share one scale of 8-bit state

enum StateKind : int { STATE_EXP_AVG = 0, STATE_EXP_AVG_SQ = 1 };

// One AdamW call, all tensors of one parameter and one gradient type. Moments: 32-bit (exp_avg,
// exp_avg_sq point at floats) or 8-bit (codes, with the scales in *_scale).
struct AdamWCall {
  void* const* param;
  void* const* master;  // null: no master weights
  void* const* grad;
  void* const* exp_avg;
  void* const* exp_avg_scale;  // null: 32-bit moments
  void* const* exp_avg_sq;
  void* const* exp_avg_sq_scale;
  const int64_t* numel;
  const int64_t* steps;
  int count;
  int param_dtype, grad_dtype;
  double lr, weight_decay, beta1, beta2, eps;
  const float* grad_scale;  // device, or null
  uint32_t seed;
};
int run_adamw(const AdamWCall& c, cudaStream_t stream);

// Partial sums of squares go to `partials` (grad_norm_partials() doubles); out2 = {norm, factor}.
int grad_norm_partials(int* n);
int run_grad_norm(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double max_norm,
                  float* out2, double* partials, cudaStream_t stream);
int run_clip(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double max_norm,
             float* out2, double* partials, cudaStream_t stream);

int run_quantize(void* const* src, void* const* codes, void* const* scales, const int64_t* numel, int count,
                 int dtype, int kind, cudaStream_t stream);
int run_dequantize(void* const* codes, void* const* scales, void* const* dst, const int64_t* numel, int count,
                   int dtype, int kind, cudaStream_t stream);

}  // namespace mb
