// murm_rope.cu — per-head RMS norm and position rotation in one pass, and the rotation alone,
// forward and backward.
//
// For a row x of d elements with gain w, position p and pair frequencies f:
//   y = R(p f) (x * r * w),  r = rsqrt(mean(x^2) + eps),
// R turning each pair of elements by its angle. With g = R^T dy the backward is
//   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x)).
// r is recomputed from x, so the forward saves nothing.
//
// Both directions read each input element once and write each output element once: the bound is
// HBM. A row belongs to L lanes of a warp (L a power of two), each of which holds both members of
// V pairs (two loads of V elements), so the rotation needs no exchange and the norm log2(L)
// shuffles. A lane's pairs are the same in every row it takes, and a group of L lanes takes
// several heads of one token: the angles (64-bit products reduced to a turn, then sincospif)
// are formed once for all of them.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "murm_kernels.cuh"
#include "murm_sm100.cuh"

namespace murm {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;
constexpr int kMaxD = 256;
constexpr int kSms = 148;
constexpr int kBwdBlocks = kSms * 3;  // blocks of the norm's backward, each with one partial of dw
constexpr int kRowsInFlight = 4;      // heads whose loads a forward group issues together

struct Rows {
  const void* x; Strides3 xs;
  const void* g; Strides3 gs;
  void* y;       Strides3 ys;
  const void* w;
  int w_f32;
  int heads;    // heads of the tensor
  int chunk;    // heads per group and item
  int items;    // (token, head chunk) items
  int blocks;   // blocks of the launch that work on this tensor
};
struct Params {
  Rows t[2];               // q, k: the first t[0].blocks blocks take q's items, the rest k's
  float* part;             // backward: [blocks][d] partial sums of dw
  int B, N, d, rd, L;      // L lanes per row
  int units, rot_units;    // units of 2V elements per row; those below rot_units are rotated
  int inverse, pos_type;
  float eps;
  const void* pos; int64_t ps[3];
  const float* freqs;      // the caller's frequencies, or NULL: turns below
  int sec_end[3];          // pair p is of the first axis a with p < sec_end[a], else of axis 3
  double turns[kMaxPairs]; // frequency of each pair / 2 pi
};

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <typename T, int V> using Raw = typename RawOf<V * (int)sizeof(T)>::type;

// The elements of one unit of a row: a[e], b[e] are the members of its e-th pair.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void unpack(const Raw<T, V>& lo, const Raw<T, V>& hi, float (&a)[V], float (&b)[V]) {
  const T* pl = reinterpret_cast<const T*>(&lo);
  const T* ph = reinterpret_cast<const T*>(&hi);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (INTER) {
      a[e] = Elem<T>::load(2 * e < V ? pl + 2 * e : ph + 2 * e - V);
      b[e] = Elem<T>::load(2 * e + 1 < V ? pl + 2 * e + 1 : ph + 2 * e + 1 - V);
    } else {
      a[e] = Elem<T>::load(pl + e);
      b[e] = Elem<T>::load(ph + e);
    }
  }
}
template <typename T, int V, bool INTER>
__device__ __forceinline__ void pack(const float (&a)[V], const float (&b)[V], Raw<T, V>& lo, Raw<T, V>& hi) {
  T* pl = reinterpret_cast<T*>(&lo);
  T* ph = reinterpret_cast<T*>(&hi);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (INTER) {
      Elem<T>::store(2 * e < V ? pl + 2 * e : ph + 2 * e - V, a[e]);
      Elem<T>::store(2 * e + 1 < V ? pl + 2 * e + 1 : ph + 2 * e + 1 - V, b[e]);
    } else {
      Elem<T>::store(pl + e, a[e]);
      Elem<T>::store(ph + e, b[e]);
    }
  }
}

// Lane `lane` of a row owns the units lane + L*j, j < UPL.
template <int V> struct UnitsPerLane { static constexpr int v = V >= 4 ? 1 : 4; };

struct UnitAt {
  int lo, hi;  // element offsets of the unit's two runs of V elements
  bool on;
};
template <int V, bool INTER>
__device__ __forceinline__ UnitAt unit_at(const Params& p, int u) {
  UnitAt r;
  r.on = u < p.units;
  if (!INTER && u < p.rot_units) {
    r.lo = u * V;
    r.hi = p.rd / 2 + u * V;
  } else {
    r.lo = u * 2 * V;  // the same for interleaved pairs and for elements past the rotated part
    r.hi = r.lo + V;
  }
  return r;
}

__device__ __forceinline__ double load_pos(const Params& p, int b, int n, int axis) {
  const int64_t at = b * p.ps[0] + n * p.ps[1] + axis * p.ps[2];
  if (p.pos_type == MURM_POS_I64) return (double)static_cast<const int64_t*>(p.pos)[at];
  if (p.pos_type == MURM_POS_I32) return (double)static_cast<const int32_t*>(p.pos)[at];
  return (double)static_cast<const float*>(p.pos)[at];
}
__device__ __forceinline__ int axis_of(const Params& p, int pair) {
  return (pair >= p.sec_end[0]) + (pair >= p.sec_end[1]) + (pair >= p.sec_end[2]);
}
__device__ __forceinline__ double turns_of(const Params& p, int pair) {
  constexpr double kInvTwoPi = 0.15915494309189533576888;
  return p.freqs ? (double)p.freqs[pair] * kInvTwoPi : p.turns[pair];
}
// cos and sin of the angle, from its turns. The product and its reduction are in 64 bits (a 32-bit
// angle of position 100000 is off by 0.004 rad), to the nearest quarter turn: the remainder's own
// rounding to 32 bits then moves the angle by at most 2^-28 turns (2.3e-8 rad), less than the
// rounding of the sine itself; reduced to a half turn only it would be 2^-26 turns.
__device__ __forceinline__ void cos_sin(double pos, double turns, float& c, float& s) {
  double t = pos * turns;
  t -= rint(t);
  const double quarter = rint(4.0 * t);
  float c0, s0;
  sincospif(2.0f * (float)(t - 0.25 * quarter), &s0, &c0);
  const int m = (int)quarter;  // -2..2
  const bool swap = m & 1;
  c = swap ? s0 : c0;
  s = swap ? c0 : s0;
  if ((m + 1) & 2) c = -c;  // a quarter or half turn on: cos(a + pi/2) = -sin a, cos(a + pi) = -cos a
  if (m & 2) s = -s;        // sin(a + pi) = -sin a, sin(a + 3 pi/2) = -cos a
}

__device__ __forceinline__ float load_weight(const Rows& r, int i, const __half*) {
  return r.w_f32 ? static_cast<const float*>(r.w)[i] : __half2float(static_cast<const __half*>(r.w)[i]);
}
__device__ __forceinline__ float load_weight(const Rows& r, int i, const __nv_bfloat16*) {
  return r.w_f32 ? static_cast<const float*>(r.w)[i]
                 : __bfloat162float(static_cast<const __nv_bfloat16*>(r.w)[i]);
}
__device__ __forceinline__ float load_weight(const Rows& r, int i, const float*) {
  return static_cast<const float*>(r.w)[i];
}

__device__ __forceinline__ float row_sum(float v, int L) {
  for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a lane keeps for the rows of one token: its units, gains and angles.
template <typename T, int V, bool INTER, bool NORM>
struct LaneState {
  static constexpr int U = UnitsPerLane<V>::v;
  UnitAt at[U];
  float wa[NORM ? U : 1][V], wb[NORM ? U : 1][V];
  float c[U][V], s[U][V];

  __device__ __forceinline__ void init(const Params& p, const Rows& r, int lane) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      at[j] = unit_at<V, INTER>(p, lane + p.L * j);
      if (NORM) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int ia = INTER ? at[j].lo + 2 * e : at[j].lo + e;
          const int ib = INTER ? ia + 1 : at[j].hi + e;
          wa[j][e] = r.w && at[j].on ? load_weight(r, ia, (const T*)nullptr) : 1.f;
          wb[j][e] = r.w && at[j].on ? load_weight(r, ib, (const T*)nullptr) : 1.f;
        }
      }
    }
  }
  __device__ __forceinline__ void angles(const Params& p, int lane, int b, int n) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int u = lane + p.L * j;
#pragma unroll
      for (int e = 0; e < V; ++e) { c[j][e] = 1.f; s[j][e] = 0.f; }
      if (u < p.rot_units) {
        int axis = -1;
        double pos = 0.0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int pair = u * V + e;
          const int ax = axis_of(p, pair);
          if (ax != axis) pos = load_pos(p, b, n, ax);
          axis = ax;
          cos_sin(pos, turns_of(p, pair), c[j][e], s[j][e]);
          if (p.inverse) s[j][e] = -s[j][e];
        }
      }
    }
  }
};

template <typename T, int V, bool INTER, bool NORM>
__global__ void __launch_bounds__(kThreads) k_rope_fwd(const __grid_constant__ Params p) {
  constexpr int U = UnitsPerLane<V>::v;
  constexpr int F = U == 1 ? kRowsInFlight : 1;
  using R = Raw<T, V>;
  const bool second = blockIdx.x >= p.t[0].blocks;
  const Rows& r = p.t[second];
  const int block = blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & (p.L - 1);
  const int item = block * (kThreads / p.L) + threadIdx.x / p.L;
  // consecutive groups take consecutive tokens of one head chunk
  const int tokens = p.B * p.N;
  const bool live = item < r.items;
  const int chunk = live ? item / tokens : 0;
  const int bn = live ? item - chunk * tokens : 0;
  const int b = bn / p.N, n = bn - b * p.N;
  LaneState<T, V, INTER, NORM> st;
  st.init(p, r, lane);
  st.angles(p, lane, b, n);
  const float inv_d = 1.f / (float)p.d;
  const T* x = row_ptr(static_cast<const T*>(r.x), r.xs, b, 0, n);
  T* y = row_ptr(static_cast<T*>(r.y), r.ys, b, 0, n);
  const int h0 = chunk * r.chunk;
  const int h1 = min(r.heads, h0 + r.chunk);
  for (int hb = 0; hb < r.chunk; hb += F) {  // the same trip count in every lane: the norm shuffles
    R lo[F][U], hi[F][U];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int h = h0 + hb + f;
      const T* row = x + (int64_t)h * r.xs.s[1];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        lo[f][j] = R{};
        hi[f][j] = R{};
        if (live && h < h1 && st.at[j].on) {
          lo[f][j] = __ldg(reinterpret_cast<const R*>(row + st.at[j].lo));
          hi[f][j] = __ldg(reinterpret_cast<const R*>(row + st.at[j].hi));
        }
      }
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int h = h0 + hb + f;
      float a[U][V], bb[U][V];
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        unpack<T, V, INTER>(lo[f][j], hi[f][j], a[j], bb[j]);
        if (NORM) {
#pragma unroll
          for (int e = 0; e < V; ++e) ss += a[j][e] * a[j][e] + bb[j][e] * bb[j][e];
        }
      }
      float rn = 1.f;
      if (NORM) rn = rsqrtf(row_sum(ss, p.L) * inv_d + p.eps);
      T* row = y + (int64_t)h * r.ys.s[1];
#pragma unroll
      for (int j = 0; j < U; ++j) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float ua = a[j][e], ub = bb[j][e];
          if (NORM) {
            ua *= rn * st.wa[j][e];
            ub *= rn * st.wb[j][e];
          }
          a[j][e] = ua * st.c[j][e] - ub * st.s[j][e];
          bb[j][e] = ua * st.s[j][e] + ub * st.c[j][e];
        }
        if (live && h < h1 && st.at[j].on) {
          R l, u;
          pack<T, V, INTER>(a[j], bb[j], l, u);
          *reinterpret_cast<R*>(row + st.at[j].lo) = l;
          *reinterpret_cast<R*>(row + st.at[j].hi) = u;
        }
      }
    }
  }
}

// The norm's backward. A group strides over items of one tensor and sums dw of its own pairs in
// registers; the block adds its groups up in shared memory, in group order, into one partial.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads) k_norm_rope_bwd(const __grid_constant__ Params p) {
  constexpr int U = UnitsPerLane<V>::v;
  constexpr int F = U == 1 ? 2 : 1;
  using R = Raw<T, V>;
  extern __shared__ float s_dw[];  // [groups][d]
  const bool second = blockIdx.x >= p.t[0].blocks;
  const Rows& r = p.t[second];
  const int block = blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & (p.L - 1);
  const int groups = kThreads / p.L, group = threadIdx.x / p.L;
  const int tokens = p.B * p.N;
  LaneState<T, V, INTER, true> st;
  st.init(p, r, lane);
  const float inv_d = 1.f / (float)p.d;
  float da[U][V], db[U][V];
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) da[j][e] = db[j][e] = 0.f;
  for (int base = block * groups; base < r.items; base += r.blocks * groups) {  // uniform in the block
    const int item = base + group;
    const bool live = item < r.items;
    const int chunk = live ? item / tokens : 0;
    const int bn = live ? item - chunk * tokens : 0;
    const int b = bn / p.N, n = bn - b * p.N;
    st.angles(p, lane, b, n);
    const T* x = row_ptr(static_cast<const T*>(r.x), r.xs, b, 0, n);
    const T* g = row_ptr(static_cast<const T*>(r.g), r.gs, b, 0, n);
    T* y = row_ptr(static_cast<T*>(r.y), r.ys, b, 0, n);
    const int h0 = chunk * r.chunk;
    const int h1 = min(r.heads, h0 + r.chunk);
    for (int hb = 0; hb < r.chunk; hb += F) {
      R xl[F][U], xh[F][U], gl[F][U], gh[F][U];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int h = h0 + hb + f;
        const T* xr = x + (int64_t)h * r.xs.s[1];
        const T* gr = g + (int64_t)h * r.gs.s[1];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          xl[f][j] = R{}; xh[f][j] = R{}; gl[f][j] = R{}; gh[f][j] = R{};
          if (live && h < h1 && st.at[j].on) {
            xl[f][j] = __ldg(reinterpret_cast<const R*>(xr + st.at[j].lo));
            xh[f][j] = __ldg(reinterpret_cast<const R*>(xr + st.at[j].hi));
            gl[f][j] = __ldg(reinterpret_cast<const R*>(gr + st.at[j].lo));
            gh[f][j] = __ldg(reinterpret_cast<const R*>(gr + st.at[j].hi));
          }
        }
      }
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int h = h0 + hb + f;
        float xa[U][V], xb[U][V], ga[U][V], gb[U][V];
        float ss = 0.f, sx = 0.f;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          unpack<T, V, INTER>(xl[f][j], xh[f][j], xa[j], xb[j]);
          unpack<T, V, INTER>(gl[f][j], gh[f][j], ga[j], gb[j]);
#pragma unroll
          for (int e = 0; e < V; ++e) {  // g = R^T dy
            const float u = ga[j][e], v = gb[j][e];
            ga[j][e] = u * st.c[j][e] + v * st.s[j][e];
            gb[j][e] = v * st.c[j][e] - u * st.s[j][e];
            ss += xa[j][e] * xa[j][e] + xb[j][e] * xb[j][e];
            sx += ga[j][e] * st.wa[j][e] * xa[j][e] + gb[j][e] * st.wb[j][e] * xb[j][e];
          }
        }
        ss = row_sum(ss, p.L);
        sx = row_sum(sx, p.L);
        const float rn = rsqrtf(ss * inv_d + p.eps);
        const float k = rn * rn * (sx * inv_d);
        const bool on = live && h < h1;
        T* row = y + (int64_t)h * r.ys.s[1];
#pragma unroll
        for (int j = 0; j < U; ++j) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (on) {  // rows past the end would add 0 * rsqrt(eps), NaN when eps is 0
              da[j][e] += ga[j][e] * (xa[j][e] * rn);
              db[j][e] += gb[j][e] * (xb[j][e] * rn);
            }
            ga[j][e] = rn * (ga[j][e] * st.wa[j][e] - xa[j][e] * k);
            gb[j][e] = rn * (gb[j][e] * st.wb[j][e] - xb[j][e] * k);
          }
          if (on && st.at[j].on) {
            R l, u;
            pack<T, V, INTER>(ga[j], gb[j], l, u);
            *reinterpret_cast<R*>(row + st.at[j].lo) = l;
            *reinterpret_cast<R*>(row + st.at[j].hi) = u;
          }
        }
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (!st.at[j].on) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int ia = INTER ? st.at[j].lo + 2 * e : st.at[j].lo + e;
      const int ib = INTER ? ia + 1 : st.at[j].hi + e;
      s_dw[group * p.d + ia] = da[j][e];
      s_dw[group * p.d + ib] = db[j][e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.d; i += kThreads) {
    float sum = 0.f;
    for (int q = 0; q < groups; ++q) sum += s_dw[q * p.d + i];
    p.part[(int64_t)blockIdx.x * p.d + i] = sum;
  }
}

// dw = sum of the blocks' partials, in a fixed order: 32 columns per block, 32 strided slices of
// the partials per column. blockIdx.y: q or k.
struct Finish {
  void* gw[2];
  int f32[2], first[2], blocks[2];
};
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_weight_sum(const float* part, int d, Finish f) {
  __shared__ float s[32][33];
  const int t = blockIdx.y, col = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.f;
  if (f.gw[t] && col < d)
    for (int i = threadIdx.y; i < f.blocks[t]; i += 32) sum += part[(int64_t)(f.first[t] + i) * d + col];
  s[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && f.gw[t] && col < d) {
    sum = 0.f;
    for (int i = 0; i < 32; ++i) sum += s[i][threadIdx.x];
    if (f.f32[t]) static_cast<float*>(f.gw[t])[col] = sum;
    else Elem<T>::store(static_cast<T*>(f.gw[t]) + col, sum);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
murm_status bad(murm_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
murm_status bad(murm_status s, const char* fmt, ...) {
  char msg[384];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return report_error(s, msg);
}

size_t elem_size(int dtype) { return dtype == MURM_F32 ? 4 : 2; }

murm_status check_rows(const murm_norm_rope_args& a, const murm_head_rows& r, const char* name, bool backward) {
  if (r.heads < 0) return bad(MURM_ERR_INVALID_ARGUMENT, "%s heads must be >= 0, got %d", name, r.heads);
  if (r.heads == 0) return MURM_OK;
  const bool empty = a.batch == 0 || a.tokens == 0;
  if (!empty && (!r.x || !r.out)) return bad(MURM_ERR_INVALID_ARGUMENT, "%s: x or out is NULL", name);
  if (!empty && backward && !r.grad) return bad(MURM_ERR_INVALID_ARGUMENT, "%s: grad is NULL", name);
  const size_t es = elem_size(a.dtype);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.out) |
                         (backward ? reinterpret_cast<uintptr_t>(r.grad) : 0);
  if (bits % es) return bad(MURM_ERR_INVALID_ARGUMENT, "%s: a pointer is not aligned to its element", name);
  for (int i = 0; i < 3; ++i)
    if (r.out_stride[i] == 0 && (i == 0 ? a.batch : i == 1 ? r.heads : a.tokens) > 1)
      return bad(MURM_ERR_INVALID_ARGUMENT, "%s: out stride[%d] is zero", name, i);
  if ((r.weight || r.grad_weight) && r.weight_dtype != MURM_F32 && r.weight_dtype != a.dtype)
    return bad(MURM_ERR_DTYPE, "%s weight must be fp32 or of the rows' dtype, got code %d", name, r.weight_dtype);
  const double rows = (double)a.batch * r.heads * a.tokens;
  if (rows > 2146435072.0) return bad(MURM_ERR_UNSUPPORTED, "%s: batch*heads*tokens exceeds 2^31 - 2^20 rows", name);
  return MURM_OK;
}

murm_status check_args(const murm_norm_rope_args* a, bool backward) {
  if (!a) return bad(MURM_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->dtype < MURM_F32 || a->dtype > MURM_BF16) return bad(MURM_ERR_DTYPE, "unsupported dtype code %d", a->dtype);
  if (a->batch < 0 || a->tokens < 0)
    return bad(MURM_ERR_INVALID_ARGUMENT, "batch and tokens must be >= 0 (got %d, %d)", a->batch, a->tokens);
  if (a->head_dim < 2 || a->head_dim > kMaxD || a->head_dim % 2)
    return bad(MURM_ERR_UNSUPPORTED, "head_dim must be even and in 2..%d, got %d", kMaxD, a->head_dim);
  if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 2)
    return bad(MURM_ERR_INVALID_ARGUMENT, "rotary_dim must be even and in 0..head_dim=%d, got %d", a->head_dim,
               a->rotary_dim);
  if (a->axes < 1 || a->axes > 4) return bad(MURM_ERR_INVALID_ARGUMENT, "axes must be 1..4, got %d", a->axes);
  if (a->axes > 1) {
    int64_t sum = 0;
    for (int i = 0; i < a->axes; ++i) {
      if (a->sections[i] < 0) return bad(MURM_ERR_INVALID_ARGUMENT, "sections[%d] is negative", i);
      sum += a->sections[i];
    }
    if (sum != a->rotary_dim / 2)
      return bad(MURM_ERR_INVALID_ARGUMENT, "sections must add up to rotary_dim/2 = %d pairs, got %lld",
                 a->rotary_dim / 2, (long long)sum);
  }
  if (a->position_type < MURM_POS_I64 || a->position_type > MURM_POS_F32)
    return bad(MURM_ERR_DTYPE, "unsupported position type code %d", a->position_type);
  if (a->rotary_dim > 0 && !a->positions && a->batch > 0 && a->tokens > 0)
    return bad(MURM_ERR_INVALID_ARGUMENT, "positions is NULL");
  if (!a->freqs && !(a->base > 0 && std::isfinite(a->base)))
    return bad(MURM_ERR_INVALID_ARGUMENT, "base must be positive and finite");
  if (a->normalize && !(a->eps >= 0 && std::isfinite(a->eps)))
    return bad(MURM_ERR_INVALID_ARGUMENT, "eps must be >= 0 and finite");
  if (backward && !a->normalize)
    return bad(MURM_ERR_INVALID_ARGUMENT, "the rotation's backward is murm_norm_rope_fwd with `inverse` set");
  if (murm_status s = check_rows(*a, a->q, "q", backward)) return s;
  if (murm_status s = check_rows(*a, a->k, "k", backward)) return s;
  return MURM_OK;
}

// Widest run of elements (V) that every row, stride and unit boundary allows.
int pick_v(const murm_norm_rope_args& a, bool backward) {
  const size_t es = elem_size(a.dtype);
  for (int v = (int)(16 / es); v > 1; v = v == 8 ? 4 : 1) {
    bool ok = a.rotary_dim % (2 * v) == 0 && (a.head_dim - a.rotary_dim) % (2 * v) == 0;
    for (const murm_head_rows* r : {&a.q, &a.k}) {
      if (r->heads == 0) continue;
      const uintptr_t bits = reinterpret_cast<uintptr_t>(r->x) | reinterpret_cast<uintptr_t>(r->out) |
                             (backward ? reinterpret_cast<uintptr_t>(r->grad) : 0);
      ok = ok && bits % (v * es) == 0;
      for (int i = 0; i < 3; ++i)
        ok = ok && r->x_stride[i] % v == 0 && r->out_stride[i] % v == 0 &&
             (!backward || r->grad_stride[i] % v == 0);
    }
    if (ok) return v;
  }
  return 1;
}

Strides3 s3(const int64_t* s) { return Strides3{{s[0], s[1], s[2]}}; }

// Heads per item of a tensor: all of them when the tokens alone give every SM `threads` threads
// (the angles are then formed once per token), else as many as keep that many threads busy.
int pick_chunk(int64_t tokens, int heads, int L, int threads, int step) {
  const int64_t want = ((int64_t)kSms * threads / L + tokens - 1) / tokens;  // items per token
  int64_t chunks = want < 1 ? 1 : want > heads ? heads : want;
  int chunk = (int)((heads + chunks - 1) / chunks);
  if (chunk > step) chunk = (chunk + step - 1) / step * step;
  return chunk < heads ? chunk : heads;
}

void fill(const murm_norm_rope_args& a, int v, bool backward, Params* p) {
  p->B = a.batch; p->N = a.tokens; p->d = a.head_dim; p->rd = a.rotary_dim;
  p->units = a.head_dim / (2 * v);
  p->rot_units = a.rotary_dim / (2 * v);
  const int per_lane = v >= 4 ? 1 : 4;
  int L = 1;
  while (L * per_lane < p->units) L *= 2;
  p->L = L;
  p->inverse = a.inverse ? 1 : 0;
  p->pos_type = a.position_type;
  p->eps = (float)a.eps;
  p->pos = a.positions;
  for (int i = 0; i < 3; ++i) p->ps[i] = a.position_stride[i];
  p->freqs = a.freqs;
  const int pairs = a.rotary_dim / 2;
  int end = 0;
  for (int i = 0; i < 3; ++i) {
    if (a.axes > 1 && i < a.axes) end += a.sections[i];
    p->sec_end[i] = (a.axes > 1 && i < a.axes - 1) ? end : pairs;
  }
  if (!a.freqs) {
    constexpr double kTwoPi = 6.283185307179586476925;
    if (a.axes > 1 && a.own_spectrum) {
      int at = 0;
      for (int i = 0; i < a.axes; ++i) {
        const double ratio = a.sections[i] ? std::pow(a.base, -1.0 / a.sections[i]) : 1.0;
        double f = 1.0 / kTwoPi;
        for (int j = 0; j < a.sections[i]; ++j, f *= ratio) p->turns[at++] = f;
      }
    } else {
      const double ratio = pairs ? std::pow(a.base, -1.0 / pairs) : 1.0;
      double f = 1.0 / kTwoPi;
      for (int i = 0; i < pairs; ++i, f *= ratio) p->turns[i] = f;
    }
  }
  const int groups = kThreads / L;
  const int64_t tokens = (int64_t)a.batch * a.tokens;
  const murm_head_rows* in[2] = {&a.q, &a.k};
  for (int t = 0; t < 2; ++t) {
    Rows& r = p->t[t];
    r = Rows{};
    const murm_head_rows& s = *in[t];
    if (s.heads == 0) continue;
    r.x = s.x; r.xs = s3(s.x_stride);
    r.g = s.grad; r.gs = s3(s.grad_stride);
    r.y = s.out; r.ys = s3(s.out_stride);
    r.w = s.weight;
    r.w_f32 = s.weight_dtype == MURM_F32;
    r.heads = s.heads;
    r.chunk = pick_chunk(tokens, s.heads, L, 1024, backward ? 2 : kRowsInFlight);
    r.items = (int)(tokens * ((s.heads + r.chunk - 1) / r.chunk));
    r.blocks = (r.items + groups - 1) / groups;
  }
  if (backward) {  // at most kBwdBlocks blocks, shared out by heads
    const int heads = a.q.heads + a.k.heads;
    for (int t = 0; t < 2; ++t) {
      Rows& r = p->t[t];
      if (!r.heads) continue;
      int cap = (int)((int64_t)kBwdBlocks * r.heads / heads);
      if (cap < 1) cap = 1;
      if (t == 1 && cap > kBwdBlocks - p->t[0].blocks) cap = kBwdBlocks - p->t[0].blocks;
      if (r.blocks > cap) r.blocks = cap;
    }
  }
}

template <typename T, int V, bool INTER>
murm_status launch(const murm_norm_rope_args& a, bool backward, cudaStream_t st) {
  Params p{};
  fill(a, V, backward, &p);
  const int blocks = p.t[0].blocks + p.t[1].blocks;
  if (!backward) {
    if (a.normalize) MURM_LAUNCH("norm_rope_fwd", (k_rope_fwd<T, V, INTER, true>), blocks, kThreads, 0, st, p);
    else MURM_LAUNCH("rope_fwd", (k_rope_fwd<T, V, INTER, false>), blocks, kThreads, 0, st, p);
  } else {
    const bool sums = a.q.grad_weight || a.k.grad_weight;
    p.part = sums ? static_cast<float*>(a.workspace) : nullptr;
    const size_t smem = sums ? (size_t)(kThreads / p.L) * a.head_dim * sizeof(float) : 0;
    MURM_LAUNCH("norm_rope_bwd", (k_norm_rope_bwd<T, V, INTER>), blocks, kThreads, smem, st, p);
    if (sums) {
      Finish f{};
      const murm_head_rows* in[2] = {&a.q, &a.k};
      for (int t = 0; t < 2; ++t) {
        f.gw[t] = in[t]->heads ? in[t]->grad_weight : nullptr;
        f.f32[t] = in[t]->weight_dtype == MURM_F32;
        f.first[t] = t ? p.t[0].blocks : 0;
        f.blocks[t] = p.t[t].blocks;
      }
      MURM_LAUNCH("norm_weight_sum", (k_norm_weight_sum<T>), dim3((a.head_dim + 31) / 32, 2), dim3(32, 32), 0, st,
                  (const float*)p.part, a.head_dim, f);
    }
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MURM_OK : bad(MURM_ERR_CUDA, "norm_rope launch: %s", cudaGetErrorString(e));
}

template <typename T>
murm_status by_width(const murm_norm_rope_args& a, bool backward, cudaStream_t st) {
  const int v = pick_v(a, backward);
  if constexpr (sizeof(T) == 2)
    if (v == 8) return a.interleaved ? launch<T, 8, true>(a, backward, st) : launch<T, 8, false>(a, backward, st);
  if (v == 4) return a.interleaved ? launch<T, 4, true>(a, backward, st) : launch<T, 4, false>(a, backward, st);
  return a.interleaved ? launch<T, 1, true>(a, backward, st) : launch<T, 1, false>(a, backward, st);
}

murm_status run(const murm_norm_rope_args* a, bool backward, cudaStream_t st) {
  if (murm_status s = check_args(a, backward)) return s;
  if (backward && (a->q.grad_weight || a->k.grad_weight)) {
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 ||
        a->workspace_bytes < murm_norm_rope_workspace())
      return bad(MURM_ERR_WORKSPACE, "the backward's workspace needs %zu bytes, 256-byte aligned (got %zu)",
                 murm_norm_rope_workspace(), a->workspace_bytes);
  }
  if (a->batch == 0 || a->tokens == 0 || a->q.heads + a->k.heads == 0) {
    // no rows: the sums over rows are zero
    for (const murm_head_rows* r : {&a->q, &a->k})
      if (backward && r->heads && r->grad_weight &&
          cudaMemsetAsync(r->grad_weight, 0, elem_size(r->weight_dtype) * a->head_dim, st) != cudaSuccess)
        return bad(MURM_ERR_CUDA, "clearing grad_weight failed");
    return MURM_OK;
  }
  switch (a->dtype) {
    case MURM_F32: return by_width<float>(*a, backward, st);
    case MURM_F16: return by_width<__half>(*a, backward, st);
    default: return by_width<__nv_bfloat16>(*a, backward, st);
  }
}

}  // namespace rope
}  // namespace murm

extern "C" {

size_t murm_norm_rope_workspace(void) {
  return (size_t)murm::rope::kBwdBlocks * murm::rope::kMaxD * sizeof(float);
}
murm_status murm_norm_rope_fwd(const murm_norm_rope_args* args, void* stream) {
  return murm::rope::run(args, false, static_cast<cudaStream_t>(stream));
}
murm_status murm_norm_rope_bwd(const murm_norm_rope_args* args, void* stream) {
  return murm::rope::run(args, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
