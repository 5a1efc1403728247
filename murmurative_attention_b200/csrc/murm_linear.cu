// murm_linear.cu — the linear layer's C ABI and its elementwise backward.
//
// Forward: one matrix product with bias, activation and residual in its epilogue (murm_gemm.cu).
// Backward: dz = dy * act'(z), from the slopes the forward saved, and db = column sums of dz in one
// pass over both, then dx = dz W and dW = dz^T x. Without an activation dz is dy itself and the pass only sums it.
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "murm_linear.cuh"
#include "murm_sm100.cuh"

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
// dz = dy * slope, db
// ---------------------------------------------------------------------------
constexpr int kDzThreads = 256;
constexpr int kDzChunks = 512;  // most row chunks, each with one partial of db

template <typename T, int V> struct alignas(V * sizeof(T)) Pack { T e[V]; };

// dz becomes the products' operand: rounded to T where that is 16 bits wide, three bf16 planes
// that hold it exactly for fp32.
template <typename T, int V>
__device__ __forceinline__ void store_operand(const Operand& o, int64_t at, const float (&d)[V]) {
  if constexpr (sizeof(T) == 2) {
    Pack<T, V> r;
#pragma unroll
    for (int e = 0; e < V; ++e) Elem<T>::store(r.e + e, d[e]);
    *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(const_cast<void*>(o.p)) + at) = r;
  } else {
    Pack<uint16_t, V> r[3];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      uint16_t t[3];
      split3(d[e], t);
      for (int q = 0; q < 3; ++q) r[q].e[e] = t[q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<Pack<uint16_t, V>*>(static_cast<uint16_t*>(const_cast<void*>(o.p)) + q * o.plane + at) = r[q];
  }
}

// Block (x, y): `cols` threads side by side (a power of two, as many as a row has groups of V
// columns, up to the block), the others on further rows; a chunk of rows. db sums dz unrounded, in
// fp32: a thread's rows in order, then the block's row groups in order, then (k_col_sum, if there are several) the chunks.
//
// Bound by memory: dy and the slopes read once, dz written once; 32768 x 4096 bf16 takes 135 us
// (6.0 TB/s; 127 with slopes in equal steps alone). A row's columns go to neighbouring threads and a thread issues kDzDepth rows' loads
// together; with a bounds check at each of them they went out one by one (180 us), so full batches
// run without and single rows follow.
constexpr int kDzDepth = 4;

template <typename T, int V, bool SLOPE>
__global__ void __launch_bounds__(kDzThreads, 3)
    k_dz(const T* dy, int64_t ldy, const Slope<T>* slope, int M, int N, int cols, int chunk, Operand dz, float* part,
         T* db) {
  __shared__ float s[kDzThreads * V];  // [row group][column]
  sm100::pdl_wait();
  sm100::pdl_trigger();
  const int tx = threadIdx.x & (cols - 1), ty = threadIdx.x / cols, rows = kDzThreads / cols;
  const uint32_t n = (blockIdx.x * cols + tx) * (uint32_t)V;  // the last block's may pass 2^31
  const int m1 = (int)min((int64_t)M, (int64_t)(blockIdx.y + 1) * chunk);
  constexpr int kDepth = SLOPE ? kDzDepth : 2 * kDzDepth;
  using P = Pack<T, V>;
  using PS = Pack<Slope<T>, V>;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  auto row = [&](int r, const P& g, const PS& sl) {
    float d[V], s[V];
    if (SLOPE) load_slopes(sl.e, s);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      d[e] = Elem<T>::load(g.e + e);
      if (SLOPE) d[e] *= s[e];
      acc[e] += d[e];
    }
    if (SLOPE && dz.p) store_operand<T, V>(dz, (int64_t)r * dz.ld + n, d);
  };
  if (n < (uint32_t)N) {  // V divides N
    int m = blockIdx.y * chunk + ty;
    const T* pg = dy + (int64_t)m * ldy + n;
    const Slope<T>* ps = slope + (int64_t)m * N + n;
    for (; m + (kDepth - 1) * rows < m1; m += kDepth * rows) {
      P g[kDepth];
      PS sl[kDepth];
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        g[i] = *reinterpret_cast<const P*>(pg);
        if (SLOPE) sl[i] = *reinterpret_cast<const PS*>(ps);
        pg += (int64_t)rows * ldy;
        ps += (int64_t)rows * N;
      }
#pragma unroll
      for (int i = 0; i < kDepth; ++i) row(m + i * rows, g[i], sl[i]);
    }
    for (; m < m1; m += rows) {
      const P g = *reinterpret_cast<const P*>(pg);
      PS sl{};
      if (SLOPE) sl = *reinterpret_cast<const PS*>(ps);
      row(m, g, sl);
      pg += (int64_t)rows * ldy;
      ps += (int64_t)rows * N;
    }
  }
  if (!part && !db) return;
#pragma unroll
  for (int e = 0; e < V; ++e) s[(ty * cols + tx) * V + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < cols * V; c += kDzThreads) {
    const uint32_t col = blockIdx.x * cols * (uint32_t)V + c;
    if (col >= (uint32_t)N) continue;
    float sum = 0.f;
    for (int r = 0; r < rows; ++r) sum += s[r * cols * V + c];
    if (db) Elem<T>::store(db + col, sum);  // the only chunk
    else part[(int64_t)blockIdx.y * N + col] = sum;
  }
}

// out[n] = the chunks' sums of column n: a warp takes every 32nd chunk of 32 neighbouring columns, then
// a column's 32 sums go to the lanes of one warp.
template <typename T>
__global__ void __launch_bounds__(1024) k_col_sum(const float* part, int chunks, int N, T* out) {
  __shared__ float s[32][33];
  sm100::pdl_wait();
  sm100::pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (n < N) {
#pragma unroll 4
    for (int c = warp; c < chunks; c += 32) sum += part[(int64_t)c * N + n];
  }
  s[warp][lane] = sum;
  __syncthreads();
  sum = s[lane][warp];
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0 && blockIdx.x * 32 + warp < N) Elem<T>::store(out + blockIdx.x * 32 + warp, sum);
}

// The pass's blocks: `cols` threads side by side with V columns each, chunks of `chunk` rows.
struct DzShape {
  int v, cols, blocks_x, chunk, chunks;
};
DzShape dz_shape(const murm_linear_bwd_args& a) {
  const int M = (int)a.rows, N = a.out_features, v = 16 / (a.dtype == MURM_F32 ? 4 : 2);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.grad_out) | reinterpret_cast<uintptr_t>(a.slope);
  DzShape s{};
  s.v = N % v == 0 && a.go_stride % v == 0 && bits % 16 == 0 ? v : 1;
  s.cols = 32;
  while (s.cols < kDzThreads && s.cols * s.v < N) s.cols *= 2;
  s.blocks_x = (int)(((int64_t)N + s.cols * s.v - 1) / (s.cols * s.v));
  // Two rounds of three blocks per SM, so that the last ones leave little idle. With slopes one round
  // where two would leave a thread less than 64 rows, and 24 rows per chunk at least (bf16 8192 x 4096,
  // gradients of 64 inputs with it: one round of 37 rows 71 us, 32 rows in 1.15 rounds 8 more; 4096 x 1024:
  // chunks of 24 rows 19.0, of 32 and 48 0.9 and 2.4 more). Without them, half the bytes, 32 rows and two rounds
  // (8192 x 4096: 41.2, one round 1.5 more).
  const bool slopes = a.activation != MURM_ACT_NONE;
  const int wave = 148 * 3 / s.blocks_x, least = slopes ? 24 : 32;
  int most = 2 * wave;
  if (slopes && (int64_t)most * 64 * (kDzThreads / s.cols) > M) most = wave;
  if (most < 1) most = 1;
  if (most > kDzChunks) most = kDzChunks;
  if (most > (M + least - 1) / least) most = (M + least - 1) / least;
  // few rows per thread in all: one chunk, whose block writes db itself (a launch less)
  if (M <= 16 * (kDzThreads / s.cols)) most = 1;
  s.chunk = (M + most - 1) / most;
  s.chunks = (M + s.chunk - 1) / s.chunk;
  return s;
}
// Partial sums of db: one chunk writes db itself.
size_t dz_part_bytes(const murm_linear_bwd_args& a) {
  const int chunks = a.grad_bias ? dz_shape(a).chunks : 0;
  return chunks > 1 ? (size_t)chunks * a.out_features * sizeof(float) : 0;
}

template <typename T, int V>
void launch_dz(const murm_linear_bwd_args& a, const DzShape& s, const Operand& dz, float* part, cudaStream_t st) {
  const int M = (int)a.rows, N = a.out_features, cols = s.cols, chunk = s.chunk, chunks = s.chunks;
  const dim3 grid(s.blocks_x, chunks);
  const T* dy = static_cast<const T*>(a.grad_out);
  T* db = chunks == 1 ? static_cast<T*>(a.grad_bias) : nullptr;
  if (db) part = nullptr;
  if (a.activation == MURM_ACT_NONE)
    MURM_LAUNCH_PDL("linear_col_part", (k_dz<T, V, false>), grid, kDzThreads, 0, st, dy, a.go_stride,
                (const Slope<T>*)nullptr, M, N, cols, chunk, dz, part, db);
  else
    MURM_LAUNCH_PDL("linear_dz", (k_dz<T, V, true>), grid, kDzThreads, 0, st, dy, a.go_stride,
                static_cast<const Slope<T>*>(a.slope), M, N, cols, chunk, dz, part, db);
  if (part)
    MURM_LAUNCH_PDL("linear_col_sum", k_col_sum<T>, (N + 31) / 32, 1024, 0, st, (const float*)part, chunks, N,
                static_cast<T*>(a.grad_bias));
}

template <typename T>
void run_dz(const murm_linear_bwd_args& a, const Operand& dz, float* part, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const DzShape s = dz_shape(a);
  if (s.v == V) launch_dz<T, V>(a, s, dz, part, st);
  else launch_dz<T, 1>(a, s, dz, part, st);
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
  if (murm_status s = check_mat("slope", a->slope, a->out_features, a->out_features, a->dtype, true)) return s;
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
  if (murm_status s = check_mat("slope", a->slope, out, out, dt, a->activation == MURM_ACT_NONE)) return s;
  return check_mat("grad_out", a->grad_out, a->go_stride, out, dt, false);
}

murm_status check_ws(const void* ws, size_t have, size_t need) {
  if (need && (!ws || reinterpret_cast<uintptr_t>(ws) % 256 || have < need))
    return bad(MURM_ERR_WORKSPACE, "workspace needs %zu bytes, 256-byte aligned (got %zu)", need, have);
  return MURM_OK;
}

// A matrix as an operand: in place where TMA can read it, else packed at an offset of the workspace.
struct Source {
  Matrix m;
  bool packed;
  size_t at;
  Operand op;
};
struct Layout {
  size_t bytes = 0;
  char* ws;
  int dtype;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += align256(n);
    return at;
  }
  Source source(const void* p, int64_t ld, int64_t rows, int cols) {
    Source s{Matrix{p, ld, rows, cols}, false, 0, {}};
    s.packed = needs_pack(dtype, s.m);
    if (s.packed) {
      s.at = take(pack_bytes(dtype, s.m));
      s.op = packed_at(dtype, s.m, ws + s.at);
    } else {
      s.op = Operand{p, ld, 0, 1};
    }
    return s;
  }
};
murm_status fill(std::initializer_list<const Source*> all, const Layout& l, cudaStream_t st) {
  Matrix m[kMaxPack];
  void* dst[kMaxPack];
  int count = 0;
  for (const Source* s : all) {
    if (!s->packed) continue;
    m[count] = s->m;
    dst[count++] = l.ws + s->at;
  }
  return count ? pack(l.dtype, m, dst, count, st) : MURM_OK;
}

struct FwdPlan {
  Layout l;
  Source x, w;
  Gemm g;
  size_t gemm_at;
};
FwdPlan plan_fwd(const murm_linear_args& a) {
  FwdPlan p{};
  p.l.ws = static_cast<char*>(a.workspace);
  p.l.dtype = a.dtype;
  p.x = p.l.source(a.x, a.x_stride, a.rows, a.in_features);
  p.w = p.l.source(a.weight, a.w_stride, a.out_features, a.in_features);
  Gemm& g = p.g;
  g.dtype = a.dtype;
  g.a = p.x.op;
  g.b = p.w.op;
  g.M = (int)a.rows; g.N = a.out_features; g.K = a.in_features;
  g.bias = a.bias;
  g.res = a.residual; g.ldr = a.r_stride;
  g.out = a.out; g.ldo = a.out_stride;
  g.slope = a.slope;
  g.act = a.activation;
  p.gemm_at = p.l.take(gemm_workspace(&g, 1));
  return p;
}

struct BwdPlan {
  Layout l;
  bool act, products;
  Source x, w, dy;  // dy: dz itself without an activation
  Operand dz;
  size_t part_at, gemm_at;
  Gemm g[2];  // dx, dW: those that are wanted
  int count;
};
BwdPlan plan_bwd(const murm_linear_bwd_args& a) {
  BwdPlan p{};
  p.l.ws = static_cast<char*>(a.workspace);
  p.l.dtype = a.dtype;
  p.act = a.activation != MURM_ACT_NONE;
  p.products = a.grad_x || a.grad_weight;
  if (p.products) {
    if (p.act) {
      const Matrix m{nullptr, 0, a.rows, a.out_features};
      const size_t at = p.l.take(pack_bytes(a.dtype, m));
      p.dz = packed_at(a.dtype, m, p.l.ws + at);
    } else {
      p.dy = p.l.source(a.grad_out, a.go_stride, a.rows, a.out_features);
      p.dz = p.dy.op;
    }
  }
  if (a.grad_x) p.w = p.l.source(a.weight, a.w_stride, a.out_features, a.in_features);
  if (a.grad_weight) p.x = p.l.source(a.x, a.x_stride, a.rows, a.in_features);
  p.part_at = p.l.take(dz_part_bytes(a));
  Gemm g{};
  g.dtype = a.dtype;
  g.a = p.dz;
  g.N = a.in_features;
  g.b_mn = true;
  if (a.grad_x) {
    Gemm& x = p.g[p.count++];
    x = g;
    x.b = p.w.op;
    x.M = (int)a.rows; x.K = a.out_features;
    x.out = a.grad_x; x.ldo = a.gx_stride;
  }
  if (a.grad_weight) {
    Gemm& w = p.g[p.count++];
    w = g;
    w.a_mn = true;
    w.b = p.x.op;
    w.M = a.out_features; w.K = (int)a.rows;
    w.out = a.grad_weight; w.ldo = a.gw_stride;
  }
  p.gemm_at = p.l.take(p.count ? gemm_workspace(p.g, p.count) : 0);
  return p;
}

murm_status run_fwd(const murm_linear_args& a, cudaStream_t st) {
  if (few_rows(a)) return few_rows_forward(a, st);
  const FwdPlan p = plan_fwd(a);
  if (murm_status s = check_ws(a.workspace, a.workspace_bytes, p.l.bytes)) return s;
  if (murm_status s = fill({&p.x, &p.w}, p.l, st)) return s;
  return gemm(&p.g, 1, p.l.ws + p.gemm_at, st);
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
  if (murm_status s = check_ws(a.workspace, a.workspace_bytes, p.l.bytes)) return s;
  if ((p.act && p.products) || a.grad_bias) {
    const Operand dz = p.act ? p.dz : Operand{};
    float* part = a.grad_bias ? reinterpret_cast<float*>(p.l.ws + p.part_at) : nullptr;
    switch (a.dtype) {
      case MURM_F32: run_dz<float>(a, dz, part, st); break;
      case MURM_F16: run_dz<__half>(a, dz, part, st); break;
      default: run_dz<__nv_bfloat16>(a, dz, part, st);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bad(MURM_ERR_CUDA, "linear backward launch: %s", cudaGetErrorString(e));
  }
  if (murm_status s = fill({&p.dy, &p.w, &p.x}, p.l, st)) return s;
  return p.count ? gemm(p.g, p.count, p.l.ws + p.gemm_at, st) : MURM_OK;
}

}  // namespace
}  // namespace lin
}  // namespace murm

using namespace murm::lin;

extern "C" {

murm_status murm_linear_workspace(const murm_linear_args* args, size_t* bytes) {
  if (!bytes) return bad(MURM_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (murm_status s = check_fwd(args)) return s;
  *bytes = args->rows && !few_rows(*args) ? plan_fwd(*args).l.bytes : 0;
  return MURM_OK;
}
murm_status murm_linear_fwd(const murm_linear_args* args, void* stream) {
  if (murm_status s = check_fwd(args)) return s;
  if (args->rows == 0) return MURM_OK;
  return run_fwd(*args, static_cast<cudaStream_t>(stream));
}
murm_status murm_linear_bwd_workspace(const murm_linear_bwd_args* args, size_t* bytes) {
  if (!bytes) return bad(MURM_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (murm_status s = check_bwd(args)) return s;
  *bytes = args->rows ? plan_bwd(*args).l.bytes : 0;
  return MURM_OK;
}
murm_status murm_linear_bwd(const murm_linear_bwd_args* args, void* stream) {
  if (murm_status s = check_bwd(args)) return s;
  return run_bwd(*args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
