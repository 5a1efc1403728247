// murm_linear_rows.cu — the linear layer for a few rows (decode steps).
//
// out[m][n] = epilogue(sum over k of x[m][k] W[n][k]) for groups of M <= 16 rows. Every element of W is
// read once per group and used M times, so the bound is W's bytes from HBM or L2 and, at a layer's usual sizes, the
// latency of one round of loads; a tensor-core tile would be 128 rows of which a few are there. A
// warp takes R rows of W: its lanes read 16 bytes each of those and of the rows of x, all of a
// stretch of K at once, and keep M x R partial sums in fp32, which a butterfly that halves the
// values with each step reduces to one per lane.
// 4 x 1024 -> 1024: 2.6 us (2 MB of W: 0.32 us at HBM's rate; launch and one latency are the rest).
#include "murm_linear.cuh"
#include "murm_sm100.cuh"

namespace murm {
namespace lin {

namespace {

constexpr int kWarps = 4;

template <typename T> struct Vec;  // 16 bytes of a row
template <> struct Vec<float> { static constexpr int n = 4; using bits = uint32_t; };
template <> struct Vec<__half> { static constexpr int n = 8; using bits = uint16_t; };
template <> struct Vec<__nv_bfloat16> { static constexpr int n = 8; using bits = uint16_t; };

// acc + the products of two runs of 16 bytes; each 16-bit product is exact and added with one
// rounding (fp32 fma on 16-bit operands).
__device__ __forceinline__ float dot16(const uint4& a, const uint4& b, float acc, const float*) {
  acc = fmaf(__uint_as_float(a.x), __uint_as_float(b.x), acc);
  acc = fmaf(__uint_as_float(a.y), __uint_as_float(b.y), acc);
  acc = fmaf(__uint_as_float(a.z), __uint_as_float(b.z), acc);
  return fmaf(__uint_as_float(a.w), __uint_as_float(b.w), acc);
}
#define MURM_DOT2(TY)                                                                                   \
  asm("{\n .reg .b16 a0, a1, b0, b1;\n mov.b32 {a0, a1}, %1;\n mov.b32 {b0, b1}, %2;\n"                 \
      " fma.rn.f32." TY " %0, a0, b0, %0;\n fma.rn.f32." TY " %0, a1, b1, %0;\n}"                       \
      : "+f"(acc)                                                                                       \
      : "r"(a), "r"(b))
__device__ __forceinline__ void dot2(uint32_t a, uint32_t b, float& acc, const __half*) { MURM_DOT2("f16"); }
__device__ __forceinline__ void dot2(uint32_t a, uint32_t b, float& acc, const __nv_bfloat16*) { MURM_DOT2("bf16"); }
#undef MURM_DOT2
template <typename T>
__device__ __forceinline__ float dot16(const uint4& a, const uint4& b, float acc, const T* t) {
  dot2(a.x, b.x, acc, t);
  dot2(a.y, b.y, acc, t);
  dot2(a.z, b.z, acc, t);
  dot2(a.w, b.w, acc, t);
  return acc;
}

struct RowsArgs {
  const void *x, *w, *bias, *res;
  void *out, *slope;
  int64_t ldx, ldw, ldr, ldo;
  int M, N, K, act;
};

// A lane's share of 32 V elements of a row from k on: 16 bytes in place, or, where rows are not 16-byte
// aligned, every 32nd element (the same ones of every row, so their order does not matter).
template <typename T, bool VEC, bool GUARD>
__device__ __forceinline__ uint4 share(const T* row, int k, int K) {
  constexpr int V = Vec<T>::n;
  const int lane = threadIdx.x & 31;
  if constexpr (VEC) {
    const int at = k + lane * V;
    return !GUARD || at < K ? __ldg(reinterpret_cast<const uint4*>(row + at)) : make_uint4(0, 0, 0, 0);
  } else {
    using E = typename Vec<T>::bits;
    alignas(16) E e[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = k + j * 32 + lane;
      e[j] = __ldg(reinterpret_cast<const E*>(row) + (GUARD ? min(at, K - 1) : at));
      if (GUARD && at >= K) e[j] = 0;
    }
    return *reinterpret_cast<const uint4*>(e);
  }
}

// One stretch of K: STEPS x 32 lanes x 16 bytes of R rows of W and M rows of x.
template <typename T, int M, int R, int STEPS, bool VEC, bool GUARD>
__device__ __forceinline__ void stretch(const RowsArgs& p, const T* x, const T* w, int k, int m_last, float (&acc)[M * R]) {
  uint4 wv[STEPS][R], xv[STEPS][M];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int at = k + s * 32 * Vec<T>::n;
#pragma unroll
    for (int r = 0; r < R; ++r) wv[s][r] = share<T, VEC, GUARD>(w + r * p.ldw, at, p.K);
#pragma unroll
    for (int m = 0; m < M; ++m)  // rows past the last repeat it; nothing reads their sums
      xv[s][m] = share<T, VEC, GUARD>(x + min(m, m_last) * p.ldx, at, p.K);
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) acc[m * R + r] = dot16(xv[s][m], wv[s][r], acc[m * R + r], (const T*)nullptr);
}

template <typename T, int M, int R, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) k_rows(const __grid_constant__ RowsArgs p) {
  constexpr int V = Vec<T>::n, C = M * R;
  constexpr int kSteps = M >= 8 ? 1 : M == 4 ? 2 : 4;
  sm100::pdl_wait();
  const int lane = threadIdx.x & 31;
  const int n0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * R;
  if (n0 >= p.N) return;
  const int m0 = blockIdx.y * M, rows = min(p.M - m0, M);
  const T* x = static_cast<const T*>(p.x) + m0 * p.ldx;
  const T* w = static_cast<const T*>(p.w) + (int64_t)min(n0, p.N - R) * p.ldw;  // the last warp steps back
  float acc[C];
#pragma unroll
  for (int i = 0; i < C; ++i) acc[i] = 0.f;
  int k = 0;
  constexpr int kWide = kSteps * 32 * V;
  const int k_full = p.K / kWide * kWide;
  for (; k < k_full; k += kWide) stretch<T, M, R, kSteps, VEC, false>(p, x, w, k, rows - 1, acc);
  for (; k < p.K; k += 32 * V) stretch<T, M, R, 1, VEC, true>(p, x, w, k, rows - 1, acc);
  // C sums over 32 lanes: each step a lane keeps one half of its values and adds its partner's
#pragma unroll
  for (int c = C, bit = 1; c > 1; c >>= 1, bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
      if (i >= c / 2) break;
      const float mine = up ? acc[i + c / 2] : acc[i], other = up ? acc[i] : acc[i + c / 2];
      acc[i] = mine + __shfl_xor_sync(0xffffffffu, other, bit);
    }
  }
#pragma unroll
  for (int o = C; o < 32; o <<= 1) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
  // lane bit j chose the upper half in step j: its value's index, most significant bit first
  int i = 0;
#pragma unroll
  for (int c = C / 2, bit = 1; c > 0; c >>= 1, bit <<= 1)
    if (lane & bit) i += c;
  const int m = m0 + i / R, n = min(n0, p.N - R) + i % R;
  if (lane >= C || i / R >= rows || n < n0) return;
  float z = acc[0];
  if (p.bias) z += Elem<T>::load(static_cast<const T*>(p.bias) + n);
  float slope, y = act_value<sizeof(T) == 2>(z, p.act, slope);
  if (p.slope) store_slope(static_cast<Slope<T>*>(p.slope) + (int64_t)m * p.N + n, slope);
  if (p.res) y += Elem<T>::load(static_cast<const T*>(p.res) + (int64_t)m * p.ldr + n);
  Elem<T>::store(static_cast<T*>(p.out) + m * p.ldo + n, y);
}

template <typename T, int M, bool VEC>
void launch(const RowsArgs& p, cudaStream_t st) {
  // two rows of W per warp, half the reads of x, where that leaves warps enough for every SM:
  // 8 x 4096 -> 4096 bf16 14.8 us with one, 11.6 with two; 2 x 1024 -> 4096 3.7 and 2.7
  const bool two = p.N >= 4096;
  const int per = kWarps * (two ? 2 : 1);
  const dim3 blocks((p.N + per - 1) / per, (p.M + M - 1) / M);
  if (two) MURM_LAUNCH_PDL("linear_rows", (k_rows<T, M, 2, VEC>), blocks, 32 * kWarps, 0, st, p);
  else MURM_LAUNCH_PDL("linear_rows", (k_rows<T, M, 1, VEC>), blocks, 32 * kWarps, 0, st, p);
}

template <typename T, bool VEC>
void by_rows(const RowsArgs& p, cudaStream_t st) {
  if (p.M == 1) launch<T, 1, VEC>(p, st);
  else if (p.M == 2) launch<T, 2, VEC>(p, st);
  else if (p.M <= 4) launch<T, 4, VEC>(p, st);
  else if (p.M <= 8) launch<T, 8, VEC>(p, st);
  else launch<T, 16, VEC>(p, st);
}

bool vectors(const murm_linear_args& a) {
  const size_t es = a.dtype == MURM_F32 ? 4 : 2;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.weight);
  return bits % 16 == 0 && a.x_stride * es % 16 == 0 && a.w_stride * es % 16 == 0 && a.in_features * es % 16 == 0;
}
template <typename T>
void forward(const murm_linear_args& a, const RowsArgs& p, cudaStream_t st) {
  if (vectors(a)) by_rows<T, true>(p, st);
  else by_rows<T, false>(p, st);
}

}  // namespace

// Up to 8 rows, and up to 16 of fp32 (the tensor path's three planes and their packing cost more); more
// rows, in groups of 16, as long as the groups' passes over W stay short: past that every warp's reads
// of 16 rows of x bind. A pass over few columns costs what 256 do, and the tensor path less with a short
// K. Measured, these kernels / the tensor cores, us:
//   bf16 4 x 1024 -> 1024 2.6 / 8.4, 16 x 1024 -> 1024 4.1 / 9.9, 32 rows 7.4 / 10.0, 64 rows 11.5 / 10.1;
//   128 x 256 -> 256 4.0 / 6.6, 500 rows 9.2 / 6.6; 8000 x 64 -> 16 9.1 / 4.5, 800 x 2560 -> 16 5.9 / 9.2;
//   8 x 4096 -> 4096 11.6 / 14.8, 16 rows 28 / 14.8;
//   fp32 48 x 1024 -> 1024 11.7 / 17.3, 64 x 512 -> 2048 17.1 / 15.4;
// where rows are not 16-byte aligned (the tensor path lays them out first):
//   bf16 16 x 1001 -> 1111 7.7 / 16.0, 48 rows 20 / 17.8; 32 x 513 -> 2047 17.8 / 16.3;
//   fp32 16 x 4095 -> 1023 19.4 / 27, 32 x 1001 -> 1111 12.6 / 17.8, 64 rows 19.4 / 18.3.
bool few_rows(const murm_linear_args& a) {
  const bool f32 = a.dtype == MURM_F32;
  const int64_t unit = f32 ? 1 << 20 : 1 << 19, by_k = unit + unit * a.in_features / 256;
  const int64_t cap = (f32 ? 3 : 4) * unit;
  int64_t most = by_k < cap ? by_k : cap;
  if (!vectors(a)) most -= most / 4;
  const int64_t passes = (a.rows + 15) / 16 * a.out_features * (a.in_features < 256 ? 256 : a.in_features);
  return a.rows <= (f32 ? 16 : 8) || passes <= most;
}

murm_status few_rows_forward(const murm_linear_args& a, cudaStream_t st) {
  const RowsArgs p{a.x, a.weight, a.bias, a.residual, a.out, a.slope, a.x_stride, a.w_stride, a.r_stride, a.out_stride,
                   (int)a.rows, a.out_features, a.in_features, a.activation};
  switch (a.dtype) {
    case MURM_F32: forward<float>(a, p, st); break;
    case MURM_F16: forward<__half>(a, p, st); break;
    default: forward<__nv_bfloat16>(a, p, st);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MURM_OK : report_error(MURM_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace lin
}  // namespace murm
