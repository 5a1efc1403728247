// murm_linear.cuh — the matrix product of the linear layer: description, epilogue math, entries.
#pragma once

#include "murm_kernels.cuh"

namespace murm {
namespace lin {

// A 16-bit matrix the tensor cores read through TMA: row-major [rows][cols] with a row stride of
// `ld` elements (a multiple of 8; base 16-byte aligned). fp32 data is three bf16 planes, `plane`
// elements apart, that add up to it exactly.
struct Operand {
  const void* p;
  int64_t ld, plane;
  int planes;
};

// D(m,n) = sum over k of A(m,k) B(n,k); z = D + bias[n]; out = act(z) + residual(m,n).
// The operand's rows are m (n) and its columns k; with a_mn (b_mn) its rows are k.
struct Gemm {
  int dtype;  // murm_dtype of out and of the epilogue's tensors
  Operand a, b;
  bool a_mn, b_mn;
  int M, N, K;
  const void* bias;
  const void* res; int64_t ldr;
  void* out; int64_t ldo;
  void* slope;   // [M][N] contiguous: act'(z) as Slope<T>, or NULL
  int act;       // murm_activation
};
// One product, or two that do not depend on each other (the backward's) in one launch where that is
// the shorter way: their tiles fill the SMs together.
size_t gemm_workspace(const Gemm* g, int count);
murm_status gemm(const Gemm* g, int count, void* workspace, cudaStream_t st);

// A slope beside elements of 16 bits T, in 16 bits. The activations' slopes lie between -0.13 and 1.13.
// - codes below 0xc000: (code - 8192) 2^-15, equal steps with 1 exact, within 2^-16; both ways are one
//   fma: added to 2^23, the number's last mantissa bits are the code.
// - from 0xc000 on: small slopes, as the T they round to. Bit 13 is the sign, the bits below it T's last 13:
//   fp16 below 2^-7, and bf16 below 2^-8 (held times 2^-55, so that 13 bits reach to 2^-71). In equal steps a
//   unit in its activation's tail would get a wrong gradient or none (gelu's slope 11 % off at -4.5, zero
//   from -5 on) where T can hold the right one.
// - 0xffff: NaN (a NaN's last bits are ones after the fma; the largest small slope is left out for it).
// fp16 slopes throughout, within 2^-12 of those near one, gave fp16 gradients 1.2 times the error.
template <typename T> struct SlopeCode { uint16_t code; };
constexpr float kSlopeScale = 32768.f, kSlopeZero = 8388608.f + 8192.f;
__device__ __forceinline__ uint32_t slope_bits(float s) { return __float_as_uint(fmaf(s, kSlopeScale, kSlopeZero)); }
__device__ __forceinline__ float slope_of(uint32_t bits) {  // 0x4b000000 | code
  return fmaf(__uint_as_float(bits), 1.f / kSlopeScale, -kSlopeZero / kSlopeScale);
}
constexpr float kSmallCodes = 1.25f;          // what the fma makes of 0xc000
constexpr uint32_t kSmallEnd = 0x1fff1fffu;   // in T's bits, twice
constexpr float kBf16Down = 0x1p-55f, kBf16Up = 0x1p55f;
// Two slopes as the T's of small ones, and 0xffff where they are small enough.
__device__ __forceinline__ uint32_t small_slopes(float a, float b, uint32_t& mask, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  uint32_t bits, end = kSmallEnd;
  __half2 limit;
  memcpy(&limit, &end, 4);
  mask = __hlt2_mask(__habs2(h), limit);
  memcpy(&bits, &h, 4);
  return bits;
}
__device__ __forceinline__ uint32_t small_slopes(float a, float b, uint32_t& mask, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a * kBf16Down, b * kBf16Down);
  uint32_t bits, end = kSmallEnd;
  __nv_bfloat162 limit;
  memcpy(&limit, &end, 4);
  mask = __hlt2_mask(__habs2(h), limit);
  memcpy(&bits, &h, 4);
  return bits;
}
__device__ __forceinline__ void small_values(uint32_t bits, float& a, float& b, const __half*) {
  __half2 h;
  memcpy(&h, &bits, 4);
  const float2 f = __half22float2(h);
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ void small_values(uint32_t bits, float& a, float& b, const __nv_bfloat16*) {
  a = __uint_as_float(bits << 16) * kBf16Up;
  b = __uint_as_float(bits & 0xffff0000u) * kBf16Up;
}
// Two slopes <-> two codes, the first in the low half.
__device__ __forceinline__ uint32_t slope_steps(float a, float b) {
  return __byte_perm(slope_bits(a), slope_bits(b), 0x5410);
}
template <typename T>
__device__ __forceinline__ uint32_t encode_slopes(float a, float b) {
  const uint32_t steps = slope_steps(a, b);
  uint32_t mask;
  const uint32_t bits = small_slopes(a, b, mask, (const T*)nullptr);
  return ((bits | ((bits >> 2) & 0x20002000u) | 0xc000c000u) & mask) | (steps & ~mask);
}
template <typename T>
__device__ __forceinline__ void decode_slopes(uint32_t w, float& a, float& b) {  // all but NaN
  float sa, sb;
  small_values((w & 0x1fff1fffu) | ((w << 2) & 0x80008000u), sa, sb, (const T*)nullptr);
  a = slope_of(__byte_perm(w, 0x4b00u, 0x5410));
  b = slope_of(__byte_perm(w, 0x4b00u, 0x5432));
  a = a >= kSmallCodes ? sa : a;
  b = b >= kSmallCodes ? sb : b;
}

// Type of the saved slopes: fp32 beside fp32, else codes.
template <typename T> struct SlopeOf { using type = SlopeCode<T>; };
template <> struct SlopeOf<float> { using type = float; };
template <typename T> using Slope = typename SlopeOf<T>::type;
__device__ __forceinline__ void store_slope(float* p, float s) { *p = s; }
template <typename T>
__device__ __forceinline__ void store_slope(SlopeCode<T>* p, float s) { p->code = (uint16_t)encode_slopes<T>(s, s); }
template <int V>
__device__ __forceinline__ void load_slopes(const float (&s)[V], float (&out)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = s[e];
}
// Two codes to a word. One maximum over all the words tells whether one of them is NaN (a comparison per code
// made 4096 x 1024 a microsecond slower).
template <typename T, int V>
__device__ __forceinline__ void load_slopes(const SlopeCode<T> (&s)[V], float (&out)[V]) {
  uint32_t most = 0;
  if constexpr (V == 1) {
    float unused;
    most = s[0].code;
    decode_slopes<T>(most, out[0], unused);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      uint32_t w;
      memcpy(&w, &s[e], sizeof(w));
      most = __vmaxu2(most, w);
      decode_slopes<T>(w, out[e], out[e + 1]);
    }
  }
  if ((most & 0xffffu) == 0xffffu || most >= 0xffff0000u) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (s[e].code == 0xffffu) out[e] = __uint_as_float(0x7fffffffu);
  }
}

// The forward for a few rows (murm_linear_rows.cu), where it takes the call: no workspace.
bool few_rows(const murm_linear_args& a);
murm_status few_rows_forward(const murm_linear_args& a, cudaStream_t st);

// Packing of a row-major matrix into an Operand: fp32 always (three planes), 16-bit data when its
// address or stride is not one TMA can take.
struct Matrix {
  const void* p;
  int64_t ld;
  int64_t rows;
  int cols;
};
bool needs_pack(int dtype, const Matrix& m);
size_t pack_bytes(int dtype, const Matrix& m);
Operand packed_at(int dtype, const Matrix& m, void* dst);  // the operand pack() writes at dst
constexpr int kMaxPack = 3;
// Up to kMaxPack matrices in one launch.
murm_status pack(int dtype, const Matrix* m, void* const* dst, int count, cudaStream_t st);

// ---------------------------------------------------------------------------
// activations, in fp32
// ---------------------------------------------------------------------------
constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kLog2e = 1.4426950408889634f;

// FAST: for results rounded to 16 bits, with the hardware's exp2 and reciprocal (relative errors
// near 2^-22); else CUDA's accurate functions.
__device__ __forceinline__ float ex2_(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / (1 + exp(-(a + b x^2) x)): the sigmoid (a = 1, b = 0) and gelu's tanh form
template <bool FAST>
__device__ __forceinline__ float sigmoid_(float x, float a, float b) {
  if (FAST) return rcp_(1.f + ex2_(x * fmaf(x * x, -b * kLog2e, -a * kLog2e)));
  return 1.f / (1.f + expf(-x * (a + b * (x * x))));
}
template <bool FAST>
__device__ __forceinline__ float silu_sigmoid(float x) {
  if (FAST) return rcp_(1.f + ex2_(-kLog2e * x));
  return 1.f / (1.f + expf(-x));
}
constexpr float kTanhA = 2.f * kSqrt2OverPi, kTanhB = 2.f * kSqrt2OverPi * 0.044715f;

// 0.5 erfc(a / sqrt 2) for a >= 0, the standard normal distribution's upper tail, and exp(-a^2/2)
// beside it: formula 7.1.26 of Abramowitz and Stegun (absolute error of erf at most 1.5e-7), with
// the argument's 1/sqrt 2 and the result's 1/2 folded into the coefficients.
__device__ __forceinline__ float normal_tail(float a, float& e) {
  const float t = rcp_(fmaf(0.3275911f * kSqrtHalf, a, 1.f));
  float q = fmaf(t, 0.5f * 1.061405429f, -0.5f * 1.453152027f);
  q = fmaf(q, t, 0.5f * 1.421413741f);
  q = fmaf(q, t, -0.5f * 0.284496736f);
  q = fmaf(q, t, 0.5f * 0.254829592f);
  e = ex2_(-0.5f * kLog2e * a * a);
  return q * t * e;
}
// max(z, 0), NaN for NaN
__device__ __forceinline__ float relu_(float z) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}

// act(z) and, beside it, its slope there (the forward saves slopes for the backward: they share
// the costly part, and a rounded slope is nearer than the slope at a rounded z). The compiler drops
// the slope where it is not used.
template <bool FAST>
__device__ __forceinline__ float act_value(float z, int act, float& slope) {
  switch (act) {
    case MURM_ACT_RELU:
      slope = z > 0.f ? 1.f : 0.f;
      return relu_(z);
    case MURM_ACT_SILU: {
      const float s = silu_sigmoid<FAST>(z), y = z * s;
      slope = fmaf(y, 1.f - s, s);
      return y;
    }
    case MURM_ACT_GELU: {
      if (FAST) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|); past 30 the second term is 0
        float e;
        const float a = fminf(fabsf(z), 30.f);
        const float q = normal_tail(a, e);
        slope = fmaf(z * kInvSqrt2Pi, e, z < 0.f ? q : 1.f - q);
        return fmaf(-a, q, relu_(z));
      }
      const float c = 0.5f * (1.f + erff(z * kSqrtHalf));
      slope = c + z * kInvSqrt2Pi * expf(-0.5f * z * z);
      return z * c;
    }
    case MURM_ACT_GELU_TANH: {  // 0.5 (1 + tanh u) = sigmoid(2u)
      const float s = sigmoid_<FAST>(z, kTanhA, kTanhB), y = z * s;
      slope = fmaf(y * (1.f - s), fmaf(3.f * kTanhB, fminf(z * z, 1e6f), kTanhA), s);
      return y;
    }
  }
  slope = 1.f;
  return z;
}

// The three bf16 terms of an fp32 value, each the leading 8 bits of what is left (cut, so that no
// term overflows): they add up to it exactly, as long as the last stays above bf16's smallest
// number. Infinities and NaN go to the first term alone.
__device__ __forceinline__ void split3(float x, uint16_t (&t)[3]) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    t[0] = (u & 0x007fffffu) ? 0x7fffu : (uint16_t)(u >> 16);
    t[1] = t[2] = 0;
    return;
  }
  t[0] = (uint16_t)(u >> 16);
  const float r = x - __uint_as_float(u & 0xffff0000u);
  const uint32_t v = __float_as_uint(r);
  t[1] = (uint16_t)(v >> 16);
  t[2] = (uint16_t)(__float_as_uint(r - __uint_as_float(v & 0xffff0000u)) >> 16);
}

}  // namespace lin
}  // namespace murm
