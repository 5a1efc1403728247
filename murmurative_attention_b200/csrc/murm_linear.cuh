// murm_linear.cuh — the matrix product of the linear layer: description, epilogue math, entry.
#pragma once

#include "murm_kernels.cuh"

namespace murm {
namespace lin {

// D[m][n] = sum over k of A(m,k) B(n,k); z = D + bias[n]; out = act(z) + residual[m][n].
// A is a[m*lda + k], or with a_mn a[k*lda + m]; B likewise.
struct Gemm {
  int dtype;  // of a, b, out and the epilogue's tensors
  const void* a; int64_t lda; bool a_mn;
  const void* b; int64_t ldb; bool b_mn;
  int M, N, K;
  const void* bias;
  const void* res; int64_t ldr;
  void* out; int64_t ldo;
  void* preact;  // [M][N] contiguous, or NULL
  int act;       // murm_activation
};
size_t gemm_workspace(const Gemm& g);
murm_status gemm(const Gemm& g, void* workspace, cudaStream_t st);

// ---------------------------------------------------------------------------
// activations, in fp32
// ---------------------------------------------------------------------------
constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;

__device__ __forceinline__ float sigmoidf_(float x) { return 1.f / (1.f + expf(-x)); }

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case MURM_ACT_RELU: return z < 0.f ? 0.f : z;  // keeps NaN
    case MURM_ACT_SILU: return z * sigmoidf_(z);
    case MURM_ACT_GELU: return 0.5f * z * (1.f + erff(z * kSqrtHalf));
    case MURM_ACT_GELU_TANH:  // 0.5 (1 + tanh u) = sigmoid(2u)
      return z * sigmoidf_(2.f * kSqrt2OverPi * (z + 0.044715f * z * z * z));
  }
  return z;
}
// d act / dz
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case MURM_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case MURM_ACT_SILU: {
      const float s = sigmoidf_(z);
      return s * (1.f + z * (1.f - s));
    }
    case MURM_ACT_GELU:
      return 0.5f * (1.f + erff(z * kSqrtHalf)) + z * kInvSqrt2Pi * expf(-0.5f * z * z);
    case MURM_ACT_GELU_TANH: {
      const float s = sigmoidf_(2.f * kSqrt2OverPi * (z + 0.044715f * z * z * z));
      return s + z * s * (1.f - s) * (2.f * kSqrt2OverPi) * (1.f + 3.f * 0.044715f * z * z);
    }
  }
  return 1.f;
}

}  // namespace lin
}  // namespace murm
