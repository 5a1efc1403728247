// murm_linear.cu — the linear layer's C ABI and its elementwise backward.
//
// Forward: one matrix product with bias, activation and residual in its epilogue (murm_gemm.cu).
// Backward: dz = dy * act'(z) and db = column sums of dz in one pass over dy and z, then
// dx = dz W and dW = dz^T x. Without an activation dz is dy itself and the pass only sums it.
#include <cstdarg>
#include <cstdio>

#include "murm_linear.cuh"

namespace murm {
namespace lin {

namespace {

murm_status bad(murm_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
murm_status bad(murm_status s, const char* fmt, ...) {
  char msg[384];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return report_error(s, msg);
}

// ---------------------------------------------------------------------------
// dz = dy * act'(z), db
// ---------------------------------------------------------------------------
constexpr int kDzCols = 32;     // column groups (of V columns) per block, a warp wide
constexpr int kDzRows = 8;      // rows a block has in flight
constexpr int kDzChunks = 128;  // most row chunks, each with one partial of db

template <typename T, int V> struct alignas(V * sizeof(T)) Pack { T e[V]; };

// Block (x, y): V * 32 columns, a chunk of rows; 8 warps take the chunk's rows in turn. dz is
// rounded to T, the type its products take it in; db sums it unrounded, in fp32, a thread's rows in
// order, then the block's 8 warps in order, then (k_col_sum) the chunks in order.
template <typename T, int V>
__global__ void __launch_bounds__(kDzCols * kDzRows)
    k_dz(const T* dy, int64_t ldy, const T* z, int M, int N, int act, int chunk, T* dz, float* part) {
  __shared__ float s[kDzRows][kDzCols * V + 1];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n = (blockIdx.x * kDzCols + tx) * V;
  const int m0 = blockIdx.y * chunk, m1 = min(M, m0 + chunk);
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  if (n < N) {  // V divides N
    using P = Pack<T, V>;
#pragma unroll 4
    for (int m = m0 + ty; m < m1; m += kDzRows) {
      const P g = *reinterpret_cast<const P*>(dy + (int64_t)m * ldy + n);
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = Elem<T>::load(g.e + e);
      if (z) {
        const P zz = *reinterpret_cast<const P*>(z + (int64_t)m * N + n);
        P o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          d[e] *= act_slope(Elem<T>::load(zz.e + e), act);
          Elem<T>::store(o.e + e, d[e]);
        }
        if (dz) *reinterpret_cast<P*>(dz + (int64_t)m * N + n) = o;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += d[e];
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < V; ++e) s[ty][tx * V + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < kDzCols * V; c += kDzCols * kDzRows) {
    const int col = blockIdx.x * kDzCols * V + c;
    if (col >= N) continue;
    float sum = 0.f;
    for (int r = 0; r < kDzRows; ++r) sum += s[r][c];
    part[(int64_t)blockIdx.y * N + col] = sum;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_col_sum(const float* part, int chunks, int N, T* out) {
  __shared__ float s[8][33];
  const int n = blockIdx.x * 32 + (threadIdx.x & 31), ty = threadIdx.x >> 5;
  float sum = 0.f;
  if (n < N)
    for (int c = ty; c < chunks; c += 8) sum += part[(int64_t)c * N + n];
  s[ty][threadIdx.x & 31] = sum;
  __syncthreads();
  if (ty == 0 && n < N) {
    sum = 0.f;
    for (int r = 0; r < 8; ++r) sum += s[r][threadIdx.x];
    Elem<T>::store(out + n, sum);
  }
}

int dz_chunks(int M, int N, int V) {
  // about four blocks per SM, chunks of 32 rows at least
  const int cols = (N + kDzCols * V - 1) / (kDzCols * V);
  int c = (148 * 4 + cols - 1) / cols;
  const int most = (M + 31) / 32;
  if (c > most) c = most;
  return c > kDzChunks ? kDzChunks : c;
}

template <typename T, int V>
void launch_dz(const murm_linear_bwd_args& a, T* dz, float* part, cudaStream_t st) {
  const int M = (int)a.rows, N = a.out_features;
  const int most = dz_chunks(M, N, V);
  const int chunk = (M + most - 1) / most;
  const int chunks = (M + chunk - 1) / chunk;
  const dim3 grid((N + kDzCols * V - 1) / (kDzCols * V), chunks);
  MURM_LAUNCH("linear_dz", (k_dz<T, V>), grid, kDzCols * kDzRows, 0, st, static_cast<const T*>(a.grad_out), a.go_stride,
              a.activation == MURM_ACT_NONE ? (const T*)nullptr : static_cast<const T*>(a.preact), M, N, a.activation,
              chunk, dz, part);
  if (part)
    MURM_LAUNCH("linear_col_sum", k_col_sum<T>, (N + 31) / 32, 256, 0, st, (const float*)part, chunks, N,
                static_cast<T*>(a.grad_bias));
}

template <typename T>
void run_dz(const murm_linear_bwd_args& a, void* dz, float* part, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.grad_out) | reinterpret_cast<uintptr_t>(a.preact);
  if (a.out_features % V == 0 && a.go_stride % V == 0 && bits % 16 == 0)
    launch_dz<T, V>(a, static_cast<T*>(dz), part, st);
  else
    launch_dz<T, 1>(a, static_cast<T*>(dz), part, st);
}

// ---------------------------------------------------------------------------
// checks, workspaces
// ---------------------------------------------------------------------------
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
size_t elem_size(int dtype) { return dtype == MURM_F32 ? 4 : 2; }

murm_status check_sizes(int64_t rows, int in, int out, int dtype, int act) {
  if (dtype < MURM_F32 || dtype > MURM_BF16) return bad(MURM_ERR_DTYPE, "unsupported dtype code %d", dtype);
  if (rows < 0 || in < 1 || out < 1)
    return bad(MURM_ERR_INVALID_ARGUMENT, "rows must be >= 0 and features >= 1 (got %lld, %d, %d)", (long long)rows, in,
               out);
  if (rows > 2147483647 - 1024 || in > 2147483647 - 1024 || out > 2147483647 - 1024)
    return bad(MURM_ERR_UNSUPPORTED, "rows and features must be below 2^31 - 1024");
  if (act < MURM_ACT_NONE || act > MURM_ACT_GELU_TANH)
    return bad(MURM_ERR_INVALID_ARGUMENT, "unknown activation code %d", act);
  return MURM_OK;
}

// A matrix argument: present (unless optional), aligned to its element, rows that do not overlap.
murm_status check_mat(const char* name, const void* p, int64_t stride, int64_t cols, int dtype, bool optional) {
  if (!p) return optional ? MURM_OK : bad(MURM_ERR_INVALID_ARGUMENT, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % elem_size(dtype))
    return bad(MURM_ERR_INVALID_ARGUMENT, "%s is not aligned to its element", name);
  if (stride < cols)
    return bad(MURM_ERR_INVALID_ARGUMENT, "%s row stride %lld is below its %lld columns", name, (long long)stride,
               (long long)cols);
  return MURM_OK;
}

murm_status check_fwd(const murm_linear_args* a) {
  if (!a) return bad(MURM_ERR_INVALID_ARGUMENT, "args is NULL");
  if (murm_status s = check_sizes(a->rows, a->in_features, a->out_features, a->dtype, a->activation)) return s;
  if (a->rows == 0) return MURM_OK;
  if (murm_status s = check_mat("x", a->x, a->x_stride, a->in_features, a->dtype, false)) return s;
  if (murm_status s = check_mat("weight", a->weight, a->w_stride, a->in_features, a->dtype, false)) return s;
  if (murm_status s = check_mat("bias", a->bias, a->out_features, a->out_features, a->dtype, true)) return s;
  if (murm_status s = check_mat("residual", a->residual, a->r_stride, a->out_features, a->dtype, true)) return s;
  if (murm_status s = check_mat("preact", a->preact, a->out_features, a->out_features, a->dtype, true)) return s;
  return check_mat("out", a->out, a->out_stride, a->out_features, a->dtype, false);
}

murm_status check_bwd(const murm_linear_bwd_args* a) {
  if (!a) return bad(MURM_ERR_INVALID_ARGUMENT, "args is NULL");
  if (murm_status s = check_sizes(a->rows, a->in_features, a->out_features, a->dtype, a->activation)) return s;
  const int in = a->in_features, out = a->out_features, dt = a->dtype;
  if (murm_status s = check_mat("grad_x", a->grad_x, a->gx_stride, in, dt, true)) return s;
  if (murm_status s = check_mat("grad_weight", a->grad_weight, a->gw_stride, in, dt, true)) return s;
  if (murm_status s = check_mat("grad_bias", a->grad_bias, out, out, dt, true)) return s;
  if (a->rows == 0) return MURM_OK;
  if (murm_status s = check_mat("x", a->x, a->x_stride, in, dt, a->grad_weight == nullptr)) return s;
  if (murm_status s = check_mat("weight", a->weight, a->w_stride, in, dt, a->grad_x == nullptr)) return s;
  if (murm_status s = check_mat("preact", a->preact, out, out, dt, a->activation == MURM_ACT_NONE)) return s;
  return check_mat("grad_out", a->grad_out, a->go_stride, out, dt, false);
}

murm_status check_ws(const void* ws, size_t have, size_t need) {
  if (need && (!ws || reinterpret_cast<uintptr_t>(ws) % 256 || have < need))
    return bad(MURM_ERR_WORKSPACE, "workspace needs %zu bytes, 256-byte aligned (got %zu)", need, have);
  return MURM_OK;
}

Gemm forward_gemm(const murm_linear_args& a) {
  Gemm g{};
  g.dtype = a.dtype;
  g.a = a.x; g.lda = a.x_stride;
  g.b = a.weight; g.ldb = a.w_stride;
  g.M = (int)a.rows; g.N = a.out_features; g.K = a.in_features;
  g.bias = a.bias;
  g.res = a.residual; g.ldr = a.r_stride;
  g.out = a.out; g.ldo = a.out_stride;
  g.preact = a.preact;
  g.act = a.activation;
  return g;
}

// dz as the products' operand: the pass's result, or grad_out itself without an activation.
struct BwdPlan {
  bool act, need_dz, need_db;
  size_t dz_at, part_at, gemm_at, bytes;
  Gemm gx, gw;
};
BwdPlan plan_bwd(const murm_linear_bwd_args& a) {
  BwdPlan p{};
  p.act = a.activation != MURM_ACT_NONE;
  p.need_dz = p.act && (a.grad_x || a.grad_weight);
  p.need_db = a.grad_bias != nullptr;
  size_t o = 0;
  auto take = [&o](size_t n) { const size_t at = o; o += align256(n); return at; };
  p.dz_at = take(p.need_dz ? (size_t)a.rows * a.out_features * elem_size(a.dtype) : 0);
  p.part_at = take(p.need_db ? (size_t)kDzChunks * a.out_features * sizeof(float) : 0);
  p.gemm_at = o;
  const char* ws = static_cast<const char*>(a.workspace);
  const void* dz = p.act ? ws + p.dz_at : a.grad_out;
  const int64_t ldz = p.act ? a.out_features : a.go_stride;
  Gemm g{};
  g.dtype = a.dtype;
  g.a = dz; g.lda = ldz;
  size_t most = 0;
  if (a.grad_x) {
    p.gx = g;
    p.gx.b = a.weight; p.gx.ldb = a.w_stride; p.gx.b_mn = true;
    p.gx.M = (int)a.rows; p.gx.N = a.in_features; p.gx.K = a.out_features;
    p.gx.out = a.grad_x; p.gx.ldo = a.gx_stride;
    most = gemm_workspace(p.gx);
  }
  if (a.grad_weight) {
    p.gw = g;
    p.gw.a_mn = true;
    p.gw.b = a.x; p.gw.ldb = a.x_stride; p.gw.b_mn = true;
    p.gw.M = a.out_features; p.gw.N = a.in_features; p.gw.K = (int)a.rows;
    p.gw.out = a.grad_weight; p.gw.ldo = a.gw_stride;
    const size_t w = gemm_workspace(p.gw);
    most = w > most ? w : most;
  }
  p.bytes = p.gemm_at + most;
  return p;
}

murm_status run_bwd(const murm_linear_bwd_args& a, cudaStream_t st) {
  if (a.rows == 0) {  // sums over no rows
    const size_t es = elem_size(a.dtype);
    cudaError_t e = cudaSuccess;
    if (a.grad_weight)
      e = cudaMemset2DAsync(a.grad_weight, a.gw_stride * es, 0, a.in_features * es, a.out_features, st);
    if (e == cudaSuccess && a.grad_bias) e = cudaMemsetAsync(a.grad_bias, 0, a.out_features * es, st);
    return e == cudaSuccess ? MURM_OK : bad(MURM_ERR_CUDA, "clearing gradients: %s", cudaGetErrorString(e));
  }
  const BwdPlan p = plan_bwd(a);
  if (murm_status s = check_ws(a.workspace, a.workspace_bytes, p.bytes)) return s;
  char* ws = static_cast<char*>(a.workspace);
  if (p.need_dz || p.need_db) {
    void* dz = p.need_dz ? ws + p.dz_at : nullptr;
    float* part = p.need_db ? reinterpret_cast<float*>(ws + p.part_at) : nullptr;
    switch (a.dtype) {
      case MURM_F32: run_dz<float>(a, dz, part, st); break;
      case MURM_F16: run_dz<__half>(a, dz, part, st); break;
      default: run_dz<__nv_bfloat16>(a, dz, part, st);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bad(MURM_ERR_CUDA, "linear backward launch: %s", cudaGetErrorString(e));
  }
  if (a.grad_x)
    if (murm_status s = gemm(p.gx, ws + p.gemm_at, st)) return s;
  if (a.grad_weight)
    if (murm_status s = gemm(p.gw, ws + p.gemm_at, st)) return s;
  return MURM_OK;
}

}  // namespace
}  // namespace lin
}  // namespace murm

using namespace murm::lin;

extern "C" {

murm_status murm_linear_workspace(const murm_linear_args* args, size_t* bytes) {
  if (!bytes) return bad(MURM_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (murm_status s = check_fwd(args)) return s;
  *bytes = args->rows ? gemm_workspace(forward_gemm(*args)) : 0;
  return MURM_OK;
}
murm_status murm_linear_fwd(const murm_linear_args* args, void* stream) {
  if (murm_status s = check_fwd(args)) return s;
  if (args->rows == 0) return MURM_OK;
  const Gemm g = forward_gemm(*args);
  if (murm_status s = check_ws(args->workspace, args->workspace_bytes, gemm_workspace(g))) return s;
  return gemm(g, args->workspace, static_cast<cudaStream_t>(stream));
}
murm_status murm_linear_bwd_workspace(const murm_linear_bwd_args* args, size_t* bytes) {
  if (!bytes) return bad(MURM_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (murm_status s = check_bwd(args)) return s;
  *bytes = args->rows ? plan_bwd(*args).bytes : 0;
  return MURM_OK;
}
murm_status murm_linear_bwd(const murm_linear_bwd_args* args, void* stream) {
  if (murm_status s = check_bwd(args)) return s;
  return run_bwd(*args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
