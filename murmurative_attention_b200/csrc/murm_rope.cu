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
// HBM. A row belongs to L lanes of a warp (with the norm a power of two), each of which holds both
// members of V pairs (two loads of V elements), so the rotation needs no exchange and the norm
// log2(L) shuffles. A lane's pairs are the same in every row it takes, and a group of L lanes takes
// several heads of one token: the angles (64-bit products, reduced to an eighth of a turn) are formed
// once for all of them. The norm's kernels walk over their items with a ring of asynchronous copies
// in shared memory ahead of them; the rotation, with a third of the arithmetic, takes an item per
// group and several rows at once.
// Measured: norm and rotation of q and k, 8 x 8192 tokens, 16 + 4 heads of 128, bf16: 121 us
// (671 MB, 5.5 TB/s), backward 198 us (1.0 GB, 5.1 TB/s); rotation of 2 x 23400 x 24 rows of 128:
// 91 us (575 MB, 6.3 TB/s).
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
// Launch shapes, by measurement (q and k of 8 x 8192 tokens, 16 + 4 heads of 128, bf16):
// forward: 8 pairs per lane, 1 row at a time, rings of 4, 2 blocks per SM: 121 us; rings of 8
//   126, 2 rows side by side and rings of 6 121 (but 24 + 8 heads, 4 x 8192: 105 against 95 us),
//   3 blocks 181, 1 block 164, 4 pairs per lane 158 (more shuffles and addresses per byte);
// backward: 8 pairs, 1 row, rings of 4, 2 blocks: 198 us; 2 rows 340 (128 registers are too few), 1 block 212,
//   4 pairs and 4 rows 290.
// rotation (2 x 23400 tokens, 24 heads of 128): 4 pairs, 4 rows, 4 blocks: 91 us; 8 pairs 93, 2 rows 99.
constexpr int kFwdV = 8, kFwdRows = 1, kFwdDepth = 4, kFwdPerSm = 2;
constexpr int kBwdV = 8, kBwdRows = 1, kBwdDepth = 4, kBwdPerSm = 2;
constexpr int kRotV = 4, kRotRows = 4, kRotPerSm = 4;
constexpr int kFwdBlocks = kSms * kFwdPerSm;
constexpr int kBwdBlocks = kSms * kBwdPerSm;  // each with a partial of dw
// an item's angles cost about as much as this many rows: with 3 the call above takes 129 us, with 5 117,
// but 24 + 8 heads 95 and 99, 12 + 3 heads of 80 94 and 98
constexpr int kAngleRows = 4;

struct Rows {
  const void* x; Strides3 xs;
  const void* g; Strides3 gs;
  void* y;       Strides3 ys;
  const void* w;
  int w_f32;
  int heads;    // heads of the tensor
  int chunk;    // heads per group and item
  int chunks;   // head chunks: items per token
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

// ---------------------------------------------------------------------------
// pairs of fp32 values: one instruction for two (the kernels are close to the issue rate)
// ---------------------------------------------------------------------------
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f2 both(float v) { return pair(v, v); }
__device__ __forceinline__ void halves(f2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 neg2(f2 a) { return a ^ 0x8000000080000000ull; }
__device__ __forceinline__ float sum2(f2 v) {
  float lo, hi;
  halves(v, lo, hi);
  return lo + hi;
}

// Two neighbouring elements of a row <-> two fp32 values.
__device__ __forceinline__ void expand(uint32_t u, float& lo, float& hi, const __nv_bfloat16*) {
  lo = __uint_as_float(u << 16);
  hi = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void expand(uint32_t u, float& lo, float& hi, const __half*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ uint32_t shrink(float lo, float hi, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t shrink(float lo, float hi, const __half*) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The pairs of one unit of a row, two to an f2 (V = 1: one, and a zero).
template <int V> struct Pairs { static constexpr int v = V == 1 ? 1 : V / 2; };

// a, b: the first and second members of the unit's pairs. lo and hi hold its 2V elements; pairs are
// (lo[e], hi[e]), or with INTER neighbours in the order lo, hi.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void unpack(const Raw<T, V>& lo, const Raw<T, V>& hi, f2 (&a)[Pairs<V>::v],
                                       f2 (&b)[Pairs<V>::v]) {
  float x[V], y[V];  // the elements of lo, of hi
  if constexpr (sizeof(T) == 2 && V > 1) {
    const uint32_t* pl = reinterpret_cast<const uint32_t*>(&lo);
    const uint32_t* ph = reinterpret_cast<const uint32_t*>(&hi);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      expand(pl[e / 2], x[e], x[e + 1], (const T*)nullptr);
      expand(ph[e / 2], y[e], y[e + 1], (const T*)nullptr);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x[e] = Elem<T>::load(reinterpret_cast<const T*>(&lo) + e);
      y[e] = Elem<T>::load(reinterpret_cast<const T*>(&hi) + e);
    }
  }
  if constexpr (V == 1) {
    a[0] = pair(x[0], 0.f);
    b[0] = pair(y[0], 0.f);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      if (INTER) {
        const float* q = 2 * e < V ? x + 2 * e : y + 2 * e - V;
        a[e / 2] = pair(q[0], q[2]);
        b[e / 2] = pair(q[1], q[3]);
      } else {
        a[e / 2] = pair(x[e], x[e + 1]);
        b[e / 2] = pair(y[e], y[e + 1]);
      }
    }
  }
}
template <typename T, int V, bool INTER>
__device__ __forceinline__ void pack(const f2 (&a)[Pairs<V>::v], const f2 (&b)[Pairs<V>::v], Raw<T, V>& lo,
                                     Raw<T, V>& hi) {
  float x[V], y[V];
  if constexpr (V == 1) {
    float z;
    halves(a[0], x[0], z);
    halves(b[0], y[0], z);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      if (INTER) {
        float* q = 2 * e < V ? x + 2 * e : y + 2 * e - V;
        halves(a[e / 2], q[0], q[2]);
        halves(b[e / 2], q[1], q[3]);
      } else {
        halves(a[e / 2], x[e], x[e + 1]);
        halves(b[e / 2], y[e], y[e + 1]);
      }
    }
  }
  if constexpr (sizeof(T) == 2 && V > 1) {
    uint32_t* pl = reinterpret_cast<uint32_t*>(&lo);
    uint32_t* ph = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      pl[e / 2] = shrink(x[e], x[e + 1], (const T*)nullptr);
      ph[e / 2] = shrink(y[e], y[e + 1], (const T*)nullptr);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      Elem<T>::store(reinterpret_cast<T*>(&lo) + e, x[e]);
      Elem<T>::store(reinterpret_cast<T*>(&hi) + e, y[e]);
    }
  }
}

// Lane `lane` of a row owns the units lane + L*j, j < UPL.
template <int V> struct UnitsPerLane { static constexpr int v = V >= 4 ? 1 : 4; };

struct UnitAt {
  int lo, hi;  // element offsets of the unit's two runs of V elements
  bool on;     // lanes past the row's units read its last one and write nothing
};
template <int V, bool INTER>
__device__ __forceinline__ UnitAt unit_at(const Params& p, int lane_unit) {
  UnitAt r;
  r.on = lane_unit < p.units;
  const int u = min(lane_unit, p.units - 1);
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
// rounding of the sine itself; reduced to a half turn only it would be 2^-26 turns. Within the eighth
// of a turn that is left (x = pi/4 at most) the Taylor series to x^9 and x^10 leave x^11 / 11! < 2e-9
// and x^12 / 12! < 2e-10.
__device__ __forceinline__ void cos_sin(double pos, double turns, float& c, float& s) {
  double t = pos * turns;
  t -= rint(t);
  const double quarter = rint(4.0 * t);
  const float x = 6.2831853071795865f * (float)(t - 0.25 * quarter), x2 = x * x;
  float s0 = fmaf(x2, 1.f / 362880.f, -1.f / 5040.f);
  s0 = fmaf(s0, x2, 1.f / 120.f);
  s0 = fmaf(s0, x2, -1.f / 6.f);
  s0 = fmaf(s0 * x2, x, x);
  float c0 = fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f);
  c0 = fmaf(c0, x2, -1.f / 720.f);
  c0 = fmaf(c0, x2, 1.f / 24.f);
  c0 = fmaf(c0, x2, -0.5f);
  c0 = fmaf(c0, x2, 1.f);
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

// Sums over a row's lanes, F rows side by side.
template <int F>
__device__ __forceinline__ void row_sums(float (&v)[F], int L) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < L) {
#pragma unroll
      for (int f = 0; f < F; ++f) v[f] += __shfl_xor_sync(0xffffffffu, v[f], o);
    }
}

// What a lane keeps beside the rows: its units, their gains, and the angles of the current token.
template <typename T, int V, bool INTER>
struct LaneState {
  static constexpr int U = UnitsPerLane<V>::v, P = Pairs<V>::v;
  UnitAt at[U];
  f2 wa[U][P], wb[U][P];

  __device__ __forceinline__ void gains(const Rows& r) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float a[2 * P], b[2 * P];
#pragma unroll
      for (int e = 0; e < 2 * P; ++e) {
        const int k = e < V ? e : 0;  // V = 1 fills the idle half with a copy
        const int ia = INTER ? at[j].lo + 2 * k : at[j].lo + k;
        const int ib = INTER ? ia + 1 : at[j].hi + k;
        a[e] = r.w ? load_weight(r, ia, (const T*)nullptr) : 1.f;
        b[e] = r.w ? load_weight(r, ib, (const T*)nullptr) : 1.f;
      }
#pragma unroll
      for (int q = 0; q < P; ++q) {
        wa[j][q] = pair(a[2 * q], a[2 * q + 1]);
        wb[j][q] = pair(b[2 * q], b[2 * q + 1]);
      }
    }
  }
  // cos and sin of the pairs of unit j of token (b, n); 1 and 0 past the rotated part
  __device__ __forceinline__ void angles(const Params& p, int lane, int b, int n, int j, f2 (&c)[P], f2 (&s)[P]) const {
    const int u = lane + p.L * j;
    float cs[2 * P], sn[2 * P];
#pragma unroll
    for (int e = 0; e < 2 * P; ++e) { cs[e] = 1.f; sn[e] = 0.f; }
    if (u < p.rot_units) {
      int axis = -1;
      double pos = 0.0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int pr = u * V + e;
        const int ax = axis_of(p, pr);
        if (ax != axis) pos = load_pos(p, b, n, ax);
        axis = ax;
        cos_sin(pos, turns_of(p, pr), cs[e], sn[e]);
        if (p.inverse) sn[e] = -sn[e];
      }
    }
#pragma unroll
    for (int q = 0; q < P; ++q) {
      c[q] = pair(cs[2 * q], cs[2 * q + 1]);
      s[q] = pair(sn[2 * q], sn[2 * q + 1]);
    }
  }
};

// A group's walk over its rows: items (a token and `chunk` of its heads) `stride` apart, head by
// head. Consecutive items are consecutive tokens of one head chunk: item = (c * B + b) * N + n; the
// walk adds the stride digit by digit. Groups past the last item stay at their last one, heads past
// the chunk's last at that, so that no load has a condition of its own; neither writes.
struct Walk {
  int c, b, n;     // head chunk, batch, token
  int dc, db, dn;  // the stride's digits
  int h, count;    // head within the chunk, heads in it
  bool live;
  __device__ __forceinline__ void start(const Params& p, const Rows& r, int item, int stride) {
    live = item < r.items;
    if (!live) item = r.items - 1;
    c = item / p.N;
    n = item - c * p.N;
    b = c % p.B;
    c /= p.B;
    dc = stride / p.N;
    dn = stride - dc * p.N;
    db = dc % p.B;
    dc /= p.B;
    enter(r);
  }
  __device__ __forceinline__ void enter(const Rows& r) {
    h = 0;
    count = min(r.chunk, r.heads - c * r.chunk);
  }
  // F rows on (F divides the chunk); true when that begins another item.
  template <int F>
  __device__ __forceinline__ bool step(const Params& p, const Rows& r) {
    h += F;
    if (h < r.chunk) return false;
    int c1 = c + dc, b1 = b + db, n1 = n + dn;
    if (n1 >= p.N) { n1 -= p.N; ++b1; }
    if (b1 >= p.B) { b1 -= p.B; ++c1; }
    live = live && c1 < r.chunks;
    if (live) { c = c1; b = b1; n = n1; }
    enter(r);
    return true;
  }
  __device__ __forceinline__ const void* position(const Params& p) const {
    const int64_t at = b * p.ps[0] + n * p.ps[1];
    return static_cast<const char*>(p.pos) + at * (p.pos_type == MURM_POS_I64 ? 8 : 4);
  }
};

__device__ __forceinline__ void async_copy(uint32_t dst, const void* src, uint4*) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_copy(uint32_t dst, const void* src, uint2*) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {  // all but the newest N groups have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The rows of A arrays (x; x and dy) on their way to a lane: a ring of S slots in shared memory that
// only this lane writes and reads, filled by asynchronous copies S - F rows ahead, so that the bytes
// in flight cost no registers and need no barrier. F rows are taken at a time. Without wide accesses
// (V = 1) rows are loaded when they are due.
template <typename T, int V, int U, int A, int S, int F>
struct Ring {
  using R = Raw<T, V>;
  static constexpr bool kAsync = V >= 4;
  static constexpr uint32_t kHalf = kThreads * sizeof(R);  // the block's lanes side by side
  static constexpr uint32_t kSlot = A * 2 * kHalf;
  static constexpr int kBytes = kAsync ? S * (int)kSlot : 0;
  const Params& p;
  const Rows& r;
  const UnitAt (&at)[U];
  const T* row[A];
  Walk w;            // the next row to fetch
  int left;
  uint32_t smem, slot;  // this lane's place in slot 0; the slot to fill next, in bytes

  __device__ __forceinline__ Ring(const Params& p_, const Rows& r_, const UnitAt (&at_)[U], void* sm, int first,
                                  int stride, int total)
      : p(p_), r(r_), at(at_), left(total), smem(sm100::smem_u32(sm) + threadIdx.x * (uint32_t)sizeof(R)), slot(0) {
    w.start(p, r, first, stride);
    enter();
    if constexpr (kAsync)
      for (int i = 0; i < S - F; ++i) fetch();
  }
  __device__ __forceinline__ void enter() {
    row[0] = row_ptr(static_cast<const T*>(r.x), r.xs, w.b, w.c * r.chunk, w.n);
    if (A == 2) row[A - 1] = row_ptr(static_cast<const T*>(r.g), r.gs, w.b, w.c * r.chunk, w.n);
    if (p.rot_units) asm volatile("prefetch.global.L1 [%0];" ::"l"(w.position(p)));  // else there may be none
  }
  __device__ __forceinline__ void step() {
    if (w.template step<1>(p, r)) {
      enter();
    } else if (w.h < w.count) {
      row[0] += r.xs.s[1];
      if (A == 2) row[A - 1] += r.gs.s[1];
    }
  }
  __device__ __forceinline__ void fetch() {
    if (left > 0) {
      --left;
#pragma unroll
      for (int a = 0; a < A; ++a) {
        async_copy(smem + slot + a * 2 * kHalf, row[a] + at[0].lo, (R*)nullptr);
        async_copy(smem + slot + (a * 2 + 1) * kHalf, row[a] + at[0].hi, (R*)nullptr);
      }
      step();
    }
    async_commit();
    slot += kSlot;
    if (slot == S * kSlot) slot = 0;
  }
  // The next F rows' units.
  __device__ __forceinline__ void next(void* sm, R (&lo)[F][A][U], R (&hi)[F][A][U]) {
    if constexpr (kAsync) {
#pragma unroll
      for (int f = 0; f < F; ++f) fetch();
      async_wait<S - F>();
      const uint8_t* s = static_cast<const uint8_t*>(sm) + threadIdx.x * sizeof(R);
      uint32_t at_slot = slot;  // all slots are taken: the next one to fill holds the oldest row
#pragma unroll
      for (int f = 0; f < F; ++f, at_slot += kSlot) {
        if (at_slot == S * kSlot) at_slot = 0;
#pragma unroll
        for (int a = 0; a < A; ++a) {
          lo[f][a][0] = *reinterpret_cast<const R*>(s + at_slot + a * 2 * kHalf);
          hi[f][a][0] = *reinterpret_cast<const R*>(s + at_slot + (a * 2 + 1) * kHalf);
        }
      }
    } else {
#pragma unroll
      for (int f = 0; f < F; ++f) {
#pragma unroll
        for (int a = 0; a < A; ++a)
#pragma unroll
          for (int j = 0; j < U; ++j) {
            lo[f][a][j] = __ldg(reinterpret_cast<const R*>(row[a] + at[j].lo));
            hi[f][a][j] = __ldg(reinterpret_cast<const R*>(row[a] + at[j].hi));
          }
        step();
      }
    }
  }
};

// The rounds of a block over its tensor's items.
__device__ __forceinline__ int block_rounds(const Rows& r, int first, int stride) {
  return first < r.items ? (r.items - first + stride - 1) / stride : 0;
}

// The rotation alone: an item per group, its first heads' loads on their way while the angles are
// formed. No sums over the row, so L is the row's number of units whatever it is (9 lanes for a row of
// 72: 26 us for 516096 rows of bf16; in groups of 16 lanes 37 us).
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads, kRotPerSm) k_rotate(const __grid_constant__ Params p) {
  constexpr int U = UnitsPerLane<V>::v, F = U == 1 ? kRotRows : 1, P = Pairs<V>::v;
  using R = Raw<T, V>;
  const bool second = blockIdx.x >= p.t[0].blocks;
  const Rows& r = p.t[second];
  const int block = blockIdx.x - (second ? p.t[0].blocks : 0);
  const int groups = kThreads / p.L, group = threadIdx.x / p.L, lane = threadIdx.x - group * p.L;
  if (group >= groups) return;
  LaneState<T, V, INTER> st;
#pragma unroll
  for (int j = 0; j < U; ++j) st.at[j] = unit_at<V, INTER>(p, lane + p.L * j);
  Walk w;
  w.start(p, r, block * groups + group, 0);
  const T* x = row_ptr(static_cast<const T*>(r.x), r.xs, w.b, w.c * r.chunk, w.n);
  T* y = row_ptr(static_cast<T*>(r.y), r.ys, w.b, w.c * r.chunk, w.n);
  R lo[F][U], hi[F][U];
  auto load = [&](int h) {  // past the last head: that one again
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const T* row = x + (int64_t)min(h + f, w.count - 1) * r.xs.s[1];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        lo[f][j] = __ldg(reinterpret_cast<const R*>(row + st.at[j].lo));
        hi[f][j] = __ldg(reinterpret_cast<const R*>(row + st.at[j].hi));
      }
    }
  };
  load(0);
  f2 c[U][P], s[U][P], ns[U][P];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    st.angles(p, lane, w.b, w.n, j, c[j], s[j]);
#pragma unroll
    for (int q = 0; q < P; ++q) ns[j][q] = neg2(s[j][q]);
  }
  for (int h = 0; h < w.count; h += F) {
    if (h > 0) load(h);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      T* row = y + (int64_t)(h + f) * r.ys.s[1];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        f2 xa[P], xb[P], ya[P], yb[P];
        unpack<T, V, INTER>(lo[f][j], hi[f][j], xa, xb);
#pragma unroll
        for (int q = 0; q < P; ++q) {
          ya[q] = fma2(xa[q], c[j][q], mul2(xb[q], ns[j][q]));
          yb[q] = fma2(xa[q], s[j][q], mul2(xb[q], c[j][q]));
        }
        if (w.live && h + f < w.count && st.at[j].on) {
          R l, u;
          pack<T, V, INTER>(ya, yb, l, u);
          *reinterpret_cast<R*>(row + st.at[j].lo) = l;
          *reinterpret_cast<R*>(row + st.at[j].hi) = u;
        }
      }
    }
  }
}

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads, kFwdPerSm) k_norm_rope_fwd(const __grid_constant__ Params p) {
  constexpr int U = UnitsPerLane<V>::v, F = U == 1 ? kFwdRows : 1;
  using R = Raw<T, V>;
  extern __shared__ __align__(16) uint8_t smem[];
  const bool second = blockIdx.x >= p.t[0].blocks;
  const Rows& r = p.t[second];
  const int block = blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & (p.L - 1);
  const int groups = kThreads / p.L, group = threadIdx.x / p.L, stride = r.blocks * groups;
  const int total = block_rounds(r, block * groups, stride) * r.chunk;  // rows per group, uniform in the block
  constexpr int P = Pairs<V>::v;
  LaneState<T, V, INTER> st;
#pragma unroll
  for (int j = 0; j < U; ++j) st.at[j] = unit_at<V, INTER>(p, lane + p.L * j);
  Ring<T, V, U, 1, kFwdDepth, F> ring(p, r, st.at, smem, block * groups + group, stride, total);
  st.gains(r);
  const float inv_d = 1.f / (float)p.d;
  // y = (x r w) turned: a' = r (xa (wa cos) - xb (wb sin)), b' = r (xa (wa sin) + xb (wb cos)); the
  // four products of gain and angle hold for all of a token's heads
  f2 aa[U][P], ab[U][P], ba[U][P], bb[U][P];
  Walk w;
  w.start(p, r, block * groups + group, stride);
  T* row = nullptr;
  for (int i = 0; i < total; i += F) {
    if (w.h == 0) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        f2 c[P], s[P];
        st.angles(p, lane, w.b, w.n, j, c, s);
#pragma unroll
        for (int q = 0; q < P; ++q) {
          aa[j][q] = mul2(st.wa[j][q], c[q]);
          ab[j][q] = neg2(mul2(st.wb[j][q], s[q]));
          ba[j][q] = mul2(st.wa[j][q], s[q]);
          bb[j][q] = mul2(st.wb[j][q], c[q]);
        }
      }
      row = row_ptr(static_cast<T*>(r.y), r.ys, w.b, w.c * r.chunk, w.n);
    }
    R lo[F][1][U], hi[F][1][U];
    ring.next(smem, lo, hi);
    f2 xa[F][U][P], xb[F][U][P];
    float ss[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      ss[f] = 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        unpack<T, V, INTER>(lo[f][0][j], hi[f][0][j], xa[f][j], xb[f][j]);
        f2 q2 = 0;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          q2 = fma2(xa[f][j][q], xa[f][j][q], q2);
          q2 = fma2(xb[f][j][q], xb[f][j][q], q2);
        }
        ss[f] += st.at[j].on ? sum2(q2) : 0.f;
      }
    }
    row_sums<F>(ss, p.L);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const f2 rn = both(rsqrtf(ss[f] * inv_d + p.eps));
      const bool on = w.live && w.h + f < w.count;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        f2 ya[P], yb[P];
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const f2 u = mul2(xa[f][j][q], rn), v = mul2(xb[f][j][q], rn);
          ya[q] = fma2(u, aa[j][q], mul2(v, ab[j][q]));
          yb[q] = fma2(u, ba[j][q], mul2(v, bb[j][q]));
        }
        if (on && st.at[j].on) {
          R l, u;
          pack<T, V, INTER>(ya, yb, l, u);
          *reinterpret_cast<R*>(row + st.at[j].lo) = l;
          *reinterpret_cast<R*>(row + st.at[j].hi) = u;
        }
      }
      row += r.ys.s[1];
    }
    w.template step<F>(p, r);
  }
}

// The norm's backward. A group sums dw of its own pairs in registers over all its rows; the block
// adds its groups up in shared memory, in group order, into one partial.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads, kBwdPerSm) k_norm_rope_bwd(const __grid_constant__ Params p) {
  constexpr int U = UnitsPerLane<V>::v, F = U == 1 ? kBwdRows : 1;
  using R = Raw<T, V>;
  extern __shared__ __align__(16) uint8_t smem[];
  const bool second = blockIdx.x >= p.t[0].blocks;
  const Rows& r = p.t[second];
  const int block = blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & (p.L - 1);
  const int groups = kThreads / p.L, group = threadIdx.x / p.L, stride = r.blocks * groups;
  const int total = block_rounds(r, block * groups, stride) * r.chunk;
  constexpr int P = Pairs<V>::v;
  LaneState<T, V, INTER> st;
#pragma unroll
  for (int j = 0; j < U; ++j) st.at[j] = unit_at<V, INTER>(p, lane + p.L * j);
  Ring<T, V, U, 2, kBwdDepth, F> ring(p, r, st.at, smem, block * groups + group, stride, total);
  st.gains(r);
  const float inv_d = 1.f / (float)p.d;
  f2 da[U][P], db[U][P], c[U][P], s[U][P];
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int q = 0; q < P; ++q) da[j][q] = db[j][q] = 0;
  Walk w;
  w.start(p, r, block * groups + group, stride);
  T* row = nullptr;
  for (int i = 0; i < total; i += F) {
    if (w.h == 0) {
#pragma unroll
      for (int j = 0; j < U; ++j) st.angles(p, lane, w.b, w.n, j, c[j], s[j]);
      row = row_ptr(static_cast<T*>(r.y), r.ys, w.b, w.c * r.chunk, w.n);
    }
    R lo[F][2][U], hi[F][2][U];
    ring.next(smem, lo, hi);
    f2 xa[F][U][P], xb[F][U][P], ga[F][U][P], gb[F][U][P];
    float ss[F], sx[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      ss[f] = sx[f] = 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        unpack<T, V, INTER>(lo[f][0][j], hi[f][0][j], xa[f][j], xb[f][j]);
        unpack<T, V, INTER>(lo[f][1][j], hi[f][1][j], ga[f][j], gb[f][j]);
        f2 q2 = 0, x2 = 0;
#pragma unroll
        for (int q = 0; q < P; ++q) {  // g = R^T dy
          const f2 u = ga[f][j][q], v = gb[f][j][q];
          ga[f][j][q] = fma2(u, c[j][q], mul2(v, s[j][q]));
          gb[f][j][q] = fma2(v, c[j][q], mul2(neg2(u), s[j][q]));
          q2 = fma2(xa[f][j][q], xa[f][j][q], q2);
          q2 = fma2(xb[f][j][q], xb[f][j][q], q2);
          x2 = fma2(mul2(ga[f][j][q], st.wa[j][q]), xa[f][j][q], x2);
          x2 = fma2(mul2(gb[f][j][q], st.wb[j][q]), xb[f][j][q], x2);
        }
        ss[f] += st.at[j].on ? sum2(q2) : 0.f;
        sx[f] += st.at[j].on ? sum2(x2) : 0.f;
      }
    }
    row_sums<F>(ss, p.L);
    row_sums<F>(sx, p.L);
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const float rn = rsqrtf(ss[f] * inv_d + p.eps);
      const f2 r2 = both(rn), k2 = both(-rn * rn * (sx[f] * inv_d));
      if (w.live && w.h + f < w.count) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
          f2 ya[P], yb[P];
#pragma unroll
          for (int q = 0; q < P; ++q) {
            da[j][q] = fma2(ga[f][j][q], mul2(xa[f][j][q], r2), da[j][q]);
            db[j][q] = fma2(gb[f][j][q], mul2(xb[f][j][q], r2), db[j][q]);
            ya[q] = mul2(r2, fma2(xa[f][j][q], k2, mul2(ga[f][j][q], st.wa[j][q])));
            yb[q] = mul2(r2, fma2(xb[f][j][q], k2, mul2(gb[f][j][q], st.wb[j][q])));
          }
          if (st.at[j].on) {
            R l, u;
            pack<T, V, INTER>(ya, yb, l, u);
            *reinterpret_cast<R*>(row + st.at[j].lo) = l;
            *reinterpret_cast<R*>(row + st.at[j].hi) = u;
          }
        }
      }
      row += r.ys.s[1];
    }
    w.template step<F>(p, r);
  }
  if (!p.part) return;
  float* s_dw = reinterpret_cast<float*>(smem);  // [groups][d], over the rings
  __syncthreads();
#pragma unroll
  for (int j = 0; j < U; ++j) {
    if (!st.at[j].on) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int ia = INTER ? st.at[j].lo + 2 * e : st.at[j].lo + e;
      const int ib = INTER ? ia + 1 : st.at[j].hi + e;
      float a[2], b[2];
      halves(da[j][e / 2], a[0], a[1]);
      halves(db[j][e / 2], b[0], b[1]);
      s_dw[group * p.d + ia] = a[e & 1];
      s_dw[group * p.d + ib] = b[e & 1];
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
    if (!empty && r.out_stride[i] == 0 && (i == 0 ? a.batch : i == 1 ? r.heads : a.tokens) > 1)
      return bad(MURM_ERR_INVALID_ARGUMENT, "%s: out stride[%d] is zero", name, i);
  if ((r.weight || r.grad_weight) && r.weight_dtype != MURM_F32 && r.weight_dtype != a.dtype)
    return bad(MURM_ERR_DTYPE, "%s weight must be fp32 or of the rows' dtype, got code %d", name, r.weight_dtype);
  if ((reinterpret_cast<uintptr_t>(r.weight) | reinterpret_cast<uintptr_t>(r.grad_weight)) % elem_size(r.weight_dtype))
    return bad(MURM_ERR_INVALID_ARGUMENT, "%s: a weight pointer is not aligned to its element", name);
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
  if (reinterpret_cast<uintptr_t>(a->positions) % (a->position_type == MURM_POS_I64 ? 8 : 4) ||
      reinterpret_cast<uintptr_t>(a->freqs) % 4)
    return bad(MURM_ERR_INVALID_ARGUMENT, "positions or freqs is not aligned to its element");
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
  const int most = !a.normalize ? kRotV : backward ? kBwdV : kFwdV;
  for (int v = (int)(16 / es) < most ? (int)(16 / es) : most; v > 1; v = v == 8 ? 4 : 1) {
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

// Heads per item of a tensor, a multiple of `rows`: the fewest rounds of the resident groups over the
// items, each as long as its heads and its angles.
int pick_chunk(int64_t tokens, int heads, double groups, int rows) {
  int best = rows;
  double best_cost = 0;
  for (int c = rows;; c += rows) {
    const int64_t items = tokens * ((heads + c - 1) / c);
    const double cost = std::ceil(items / groups) * (c + kAngleRows);
    if (best_cost == 0 || cost < best_cost) {
      best_cost = cost;
      best = c;
    }
    if (c >= heads || c >= 64) return best;
  }
}

void fill(const murm_norm_rope_args& a, int v, bool backward, Params* p) {
  p->B = a.batch; p->N = a.tokens; p->d = a.head_dim; p->rd = a.rotary_dim;
  p->units = a.head_dim / (2 * v);
  p->rot_units = a.rotary_dim / (2 * v);
  const int per_lane = v >= 4 ? 1 : 4;
  int L = 1;
  while (L * per_lane < p->units) L *= 2;
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
  p->L = a.normalize ? L : (p->units + per_lane - 1) / per_lane;
  const int groups = kThreads / p->L;
  const int64_t tokens = (int64_t)a.batch * a.tokens;
  const int most = backward ? kBwdBlocks : kFwdBlocks;
  const int rows = v < 4 ? 1 : !a.normalize ? kRotRows : backward ? kBwdRows : kFwdRows;
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
    r.chunk = pick_chunk(tokens, s.heads, (double)most * groups * s.heads / (a.q.heads + a.k.heads), rows);
    r.chunks = (s.heads + r.chunk - 1) / r.chunk;
    r.items = (int)(tokens * r.chunks);
    r.blocks = (r.items + groups - 1) / groups;
  }
  if (!a.normalize) return;
  // no more blocks than are resident at once, shared out by work: an item's angles cost about as
  // much as kAngleRows rows
  double work[2] = {0, 0};
  for (int t = 0; t < 2; ++t)
    if (p->t[t].heads) work[t] = (double)p->t[t].items * (p->t[t].chunk + kAngleRows);
  for (int t = 0; t < 2; ++t) {
    Rows& r = p->t[t];
    if (!r.heads) continue;
    int cap = (int)(most * work[t] / (work[0] + work[1]));
    if (cap < 1) cap = 1;
    if (t == 1 && cap > most - p->t[0].blocks) cap = most - p->t[0].blocks;
    if (t == 0 && cap == most && work[1] > 0) cap = most - 1;
    if (r.blocks > cap) r.blocks = cap;
  }
}

template <typename T, int V, bool INTER>
murm_status launch(const murm_norm_rope_args& a, bool backward, cudaStream_t st) {
  Params p{};
  fill(a, V, backward, &p);
  const int blocks = p.t[0].blocks + p.t[1].blocks;
  constexpr int U = UnitsPerLane<V>::v;
  cudaError_t e = cudaSuccess;
  if (!a.normalize) {
    MURM_LAUNCH("rotate", (k_rotate<T, V, INTER>), blocks, kThreads, 0, st, p);
  } else if (!backward) {
    constexpr int smem = Ring<T, V, U, 1, kFwdDepth, U == 1 ? kFwdRows : 1>::kBytes;
    auto* kernel = k_norm_rope_fwd<T, V, INTER>;
    if (smem > 48 * 1024) e = smem_opt_in(kernel, smem);
    if (e == cudaSuccess) MURM_LAUNCH("norm_rope_fwd", kernel, blocks, kThreads, smem, st, p);
  } else {
    const bool sums = a.q.grad_weight || a.k.grad_weight;
    p.part = sums ? static_cast<float*>(a.workspace) : nullptr;
    const int rings = Ring<T, V, U, 2, kBwdDepth, U == 1 ? kBwdRows : 1>::kBytes, dw = (kThreads / p.L) * a.head_dim * (int)sizeof(float);
    const int smem = rings > dw ? rings : dw;
    auto* kernel = k_norm_rope_bwd<T, V, INTER>;
    if (smem > 48 * 1024) e = smem_opt_in(kernel, smem);
    if (e == cudaSuccess) MURM_LAUNCH("norm_rope_bwd", kernel, blocks, kThreads, smem, st, p);
    if (sums && e == cudaSuccess) {
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
  if (e == cudaSuccess) e = cudaGetLastError();
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
