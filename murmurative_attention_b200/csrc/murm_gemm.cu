// murm_gemm.cu — matrix product with the linear layer's epilogue.
#include "murm_linear.cuh"

namespace murm {
namespace lin {

// 64 x 64 tile per block, 4 x 4 outputs per thread, products and sums in fp32.
template <typename T>
__global__ void __launch_bounds__(256) k_gemm(Gemm g) {
  __shared__ float sa[16][65], sb[16][65];
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const T* a = static_cast<const T*>(g.a);
  const T* b = static_cast<const T*>(g.b);
  float acc[4][4] = {};
  for (int k0 = 0; k0 < g.K; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int ka = g.a_mn ? i >> 6 : i & 15, ma = g.a_mn ? i & 63 : i >> 4;
      const int kb = g.b_mn ? i >> 6 : i & 15, nb = g.b_mn ? i & 63 : i >> 4;
      const int64_t m = m0 + ma, n = n0 + nb, k1 = k0 + ka, k2 = k0 + kb;
      sa[ka][ma] = m < g.M && k1 < g.K ? Elem<T>::load(a + (g.a_mn ? k1 * g.lda + m : m * g.lda + k1)) : 0.f;
      sb[kb][nb] = n < g.N && k2 < g.K ? Elem<T>::load(b + (g.b_mn ? k2 * g.ldb + n : n * g.ldb + k2)) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][ty * 4 + i] * sb[k][tx + 16 * j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m >= g.M || n >= g.N) continue;
      float z = acc[i][j];
      if (g.bias) z += Elem<T>::load(static_cast<const T*>(g.bias) + n);
      if (g.preact) Elem<T>::store(static_cast<T*>(g.preact) + m * g.N + n, z);
      float y = act_value(z, g.act);
      if (g.res) y += Elem<T>::load(static_cast<const T*>(g.res) + m * g.ldr + n);
      Elem<T>::store(static_cast<T*>(g.out) + m * g.ldo + n, y);
    }
}

size_t gemm_workspace(const Gemm&) { return 0; }

murm_status gemm(const Gemm& g, void*, cudaStream_t st) {
  const dim3 grid((g.N + 63) / 64, (g.M + 63) / 64);
  switch (g.dtype) {
    case MURM_F32: MURM_LAUNCH("linear_gemm", k_gemm<float>, grid, 256, 0, st, g); break;
    case MURM_F16: MURM_LAUNCH("linear_gemm", k_gemm<__half>, grid, 256, 0, st, g); break;
    default: MURM_LAUNCH("linear_gemm", k_gemm<__nv_bfloat16>, grid, 256, 0, st, g);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MURM_OK : report_error(MURM_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace lin
}  // namespace murm
