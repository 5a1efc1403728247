// murm_gemm.cu — the linear layer's matrix products on tcgen05, with their epilogue.
//
// D = A B^T with A [M][K], B [N][K] read as they lie in memory: the tensor cores take either
// operand K-major (rows of K) or MN-major (rows of M or N), so the forward (x W^T) and both
// gradients (dz W, dz^T x) need no transposed copy.
//
// k_gemm_tc: a pair of CTAs (cta_group::2) per 256 x BN tile, each holding 128 rows of A, half the
// rows of B and a 128 x BN fp32 accumulator in TMEM (two accumulators: a tile's epilogue runs under
// the next tile's products). Persistent over the tiles. Warps 0, 2 and 3 load the operands by TMA into
// a ring of 64-deep stages, a stage each in turn (one thread needs some 490 clocks to wait for a stage
// and issue its copies, as long as the MMAs take), warp 1 of the first CTA issues the MMAs of both
// CTAs, warps 4-19 run the
// epilogue, each on 32 rows and a quarter of the columns: TMEM -> registers -> bias, activation,
// residual -> 64-byte swizzled rows in shared memory -> TMA store (or plain stores where the
// result's rows are not 16-byte aligned).
//
// fp32 operands are three bf16 planes, the terms cut and not rounded; the products of planes (i, j) with
// i + j <= 2 are added smallest first into the same fp32 accumulator. The pairs left out, (1,2) and (2,1)
// before all, are up to 2^-21 of a product and 2^-24.7 on average, always with its sign. Products with few tiles and a long K split
// K; the parts' fp32 sums go to the workspace and k_split_sum adds them in order and runs the epilogue. So
// do fp32 products of a long K, whose items change accumulators on the way (kSegment).
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdio>

#include "murm_linear.cuh"
#include "murm_sm100.cuh"

namespace murm {

extern __device__ int g_device_error;
PFN_cuTensorMapEncodeTiled_v12000 tc_tensor_map_encoder();  // murm_tc.cu

namespace lin {
using namespace sm100;

constexpr int kErrLinear = 64;  // device error bit: a copy or an MMA of a linear product never completed
constexpr int kSms = 148;
constexpr int kPairs = kSms / 2;     // CTA pairs resident at once
constexpr int kBK = 64;              // depth of a stage: one 128-byte swizzled row
constexpr uint32_t kABytes = 128 * kBK * 2;
constexpr int kLoaders = 3;
constexpr int kEpiWarps = 16;        // 4 row groups (TMEM lanes) x 4 column groups
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr uint32_t kBuf = 32 * 64;   // one epilogue warp's 32 rows of 64 bytes

template <int BN> struct Tile {
  static constexpr uint32_t kBBytes = BN / 2 * kBK * 2;
  static constexpr uint32_t kStage = kABytes + kBBytes;
  static constexpr int kStages = BN == 256 ? 6 : 8;  // of 256: 6 and 5 alike, 4 3 % slower
  static constexpr uint32_t OFF_OUT = kStages * kStage;  // one buffer per epilogue warp
  static constexpr uint32_t OFF_BAR = OFF_OUT + kEpiWarps * kBuf;
  static constexpr uint32_t kSmem = OFF_BAR + 256 + 1024;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static_assert(kSmem <= 232448, "shared memory budget");
};

struct Bars {  // in shared memory at OFF_BAR
  uint64_t full[8], empty[8];         // operand stages; `full` of the pair's first CTA counts both loads
  uint64_t acc_full[2], acc_free[2];  // accumulators; acc_free is used in the pair's first CTA
  uint32_t tmem;
};
static_assert(sizeof(Bars) <= 256, "barrier area");

struct Args {
  int M, N;
  int iters, total, splits, seg;          // stages per split, in all; K splits; stages per accumulator
  int tiles_m, tiles_n, tiles, items;     // items: tiles * splits
  uint32_t idesc;
  int a_mn, b_mn;
  int fp32;  // operands are three planes
  const void* bias; int bias_vec;         // *_vec: 16-byte accesses are aligned and stay inside the row
  int act;
  const void* res; int64_t ldr; int res_vec;
  void* out; int64_t ldo; int out_tma;
  void* slope; int slope_tma;
  int partial;     // out: fp32 sums of K splits, tiles side by side, splits `split_rows` rows apart
  int split_rows;
  int join;        // an item's last segment reads what the earlier ones left in out, then runs the epilogue
};
struct Problem {
  CUtensorMap a, b, out, slope;
  Args p;
};
// One launch: the items of one or two products. Pair j takes the positions j, j + pairs, ...; with
// `tabled` a position's item is order[position] (kNone: nothing).
constexpr int kMaxOrder = 8 * kPairs;
constexpr uint16_t kNone = 0xffff;
constexpr int kAdd = 2;  // a tile's rows are added to what its item's earlier segments left
struct Launch {
  Problem q[2];
  int items, positions, tabled;
  uint16_t order[kMaxOrder];
};
static_assert(sizeof(Launch) <= 4000, "kernel parameters");

// Plane pairs of an fp32 product, smallest terms first: (0,2) (2,0) (1,1) (0,1) (1,0) (0,0).
constexpr int kPlanePairs = 6;
__device__ __forceinline__ int plane_a(int pair) { return (0x021010 >> (4 * (5 - pair))) & 15; }
__device__ __forceinline__ int plane_b(int pair) { return (0x201100 >> (4 * (5 - pair))) & 15; }

// ---------------------------------------------------------------------------
// PTX of the CTA pair
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Both CTAs have come here. Relaxed: what has to be seen across (barrier initialisation) has a fence
// of its own; a releasing arrival waits some 1000 clocks for the thread's global stores.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of the first CTA's copy of a shared-memory object.
__device__ __forceinline__ uint32_t map_to_first(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
// Says that this warp's reads of TMEM are done (ordered by the tcgen05 fence before it; relaxed for
// the same reason as above).
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Load into this CTA's shared memory that counts on a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                              uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
      "%3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The same with fp32 sums into what is there.
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// This thread's stores have reached global memory: its later ones to the same place come after them.
__device__ __forceinline__ void tma_store_wait_done() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  fence_proxy_async_global();
}
// This thread's stores have read their shared memory.
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once this thread's MMAs are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  if (mbar_timed_wait(bar, parity)) return true;
  atomicOr(&g_device_error, kErrLinear);
  return false;
}

// ---------------------------------------------------------------------------
// epilogue pieces
// ---------------------------------------------------------------------------
template <typename T> struct Out {  // an epilogue step: 64 bytes of a row
  static constexpr int kCols = 64 / sizeof(T);
  static constexpr bool kFast = sizeof(T) == 2;
};

__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b, const SlopeCode<T>*) {
  return encode_slopes<T>(a, b);
}
__device__ __forceinline__ float2 unpack2(uint32_t u, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, const __nv_bfloat16*) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Chunk j of 16 bytes of row r in a buffer of 64-byte rows (the tensor engine's 64-byte swizzle).
__device__ __forceinline__ uint32_t chunk_at(int r, int j) { return r * 64 + ((j ^ ((r >> 1) & 3)) << 4); }

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {  // 16 bytes of elements
  if constexpr (sizeof(T) == 2)
    return make_uint4(pack2(v[0], v[1], (const T*)nullptr), pack2(v[2], v[3], (const T*)nullptr),
                      pack2(v[4], v[5], (const T*)nullptr), pack2(v[6], v[7], (const T*)nullptr));
  else
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
// A lane's own row.
template <typename T>
__device__ __forceinline__ void write_row(uint32_t buf, int lane, const float (&v)[Out<T>::kCols]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) sts128(buf + chunk_at(lane, j), pack16<T>(v + j * (16 / sizeof(T))));
}
template <typename T>
__device__ __forceinline__ void add16(const uint4& u, float* v) {  // v += the elements of 16 bytes
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const float2 f = unpack2(w[i], (const T*)nullptr);
      v[2 * i] += f.x;
      v[2 * i + 1] += f.y;
    } else {
      v[i] += __uint_as_float(w[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void add_row(uint32_t buf, int lane, float (&v)[Out<T>::kCols]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) add16<T>(lds128(buf + chunk_at(lane, j)), v + j * (16 / sizeof(T)));
}
// A warp's 32 rows of a buffer in global memory, four lanes to a row: coalesced 16-byte accesses.
// OWN: rows that this kernel has written (not to be had from the read-only cache).
template <typename T, bool OWN = false>
__device__ __forceinline__ void load_rows(const T* g, int64_t ld, int rows, int cols, int lane, uint4 (&v)[4]) {
  const int c = (lane & 3) * (16 / (int)sizeof(T));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    v[i] = make_uint4(0, 0, 0, 0);
    if (r < rows && c < cols) {
      const uint4* at = reinterpret_cast<const uint4*>(g + r * ld + c);
      v[i] = OWN ? __ldcg(at) : __ldg(at);
    }
  }
}
__device__ __forceinline__ void put_rows(uint32_t buf, int lane, const uint4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sts128(buf + chunk_at(i * 8 + (lane >> 2), lane & 3), v[i]);
}
// The same rows where 16-byte accesses are not aligned: element by element, columns side by side. Global
// reads go out four together, rows past the last from that one (777 x 1001 -> 1111 bf16 with a residual:
// 21.0 us one by one, 19.6 so, 17.8 eight together, which spills: 8192 x 1024 -> 4096 63 us for 61.8).
template <typename T, bool STORE>
__device__ __forceinline__ void copy_rows(uint8_t* buf, T* g, int64_t ld, int rows, int cols, int lane) {
  constexpr int kCols = Out<T>::kCols, kRows = 32 / kCols;  // columns of a row, rows side by side
  const int c = lane % kCols;
  if (c >= cols) return;
  auto at = [&](int r) {
    return reinterpret_cast<T*>(buf + chunk_at(r, (c * (int)sizeof(T)) >> 4) + ((c * (int)sizeof(T)) & 15));
  };
  if (STORE) {
    for (int r = lane / kCols; r < rows; r += kRows) g[r * ld + c] = *at(r);
    return;
  }
#pragma unroll 4
  for (int r = lane / kCols; r < 32; r += kRows) *at(r) = __ldg(g + min(r, rows - 1) * ld + c);
}
// The bias of a step's columns: the same address in every lane, from L1. With `vec`, b holds it
// (loaded early, while the accumulator is on its way).
template <typename T>
__device__ __forceinline__ void load_bias(const T* bias, int cols, uint4 (&b)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[j] = make_uint4(0, 0, 0, 0);
    if (j * (16 / (int)sizeof(T)) < cols) b[j] = __ldg(reinterpret_cast<const uint4*>(bias) + j);
  }
}
template <typename T>
__device__ __forceinline__ void add_bias(const T* bias, int vec, const uint4 (&b)[4], int cols,
                                         float (&v)[Out<T>::kCols]) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) add16<T>(b[j], v + j * (16 / sizeof(T)));
  } else {
#pragma unroll
    for (int j = 0; j < Out<T>::kCols; ++j)
      if (j < cols) v[j] += Elem<T>::load(bias + j);
  }
}
// v = act(v); SLOPE: the slopes go to the lane's row of the buffer, 16 bytes at a time.
template <typename T, bool SLOPE, int ACT>
__device__ __forceinline__ void activate_as(float (&v)[Out<T>::kCols], uint32_t buf, int lane) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float d[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[j * kPer + i] = act_value<Out<T>::kFast>(v[j * kPer + i], ACT, d[i]);
    if constexpr (SLOPE && ACT == MURM_ACT_RELU && sizeof(T) == 2)  // 0 and 1 are steps
      sts128(buf + chunk_at(lane, j), make_uint4(slope_steps(d[0], d[1]), slope_steps(d[2], d[3]),
                                                 slope_steps(d[4], d[5]), slope_steps(d[6], d[7])));
    else if (SLOPE) sts128(buf + chunk_at(lane, j), pack16<Slope<T>>(d));
  }
}
template <typename T, bool SLOPE>
__device__ __forceinline__ void activate(float (&v)[Out<T>::kCols], int act, uint32_t buf, int lane) {
  switch (act) {  // one loop per activation: the choice is made once
    case MURM_ACT_NONE: break;
    case MURM_ACT_RELU: activate_as<T, SLOPE, MURM_ACT_RELU>(v, buf, lane); break;
    case MURM_ACT_SILU: activate_as<T, SLOPE, MURM_ACT_SILU>(v, buf, lane); break;
    case MURM_ACT_GELU: activate_as<T, SLOPE, MURM_ACT_GELU>(v, buf, lane); break;
    default: activate_as<T, SLOPE, MURM_ACT_GELU_TANH>(v, buf, lane);
  }
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
struct Item {
  int which;  // the product; -1: nothing at this position
  int m0, n0, split, i0, i1;
};
// Tiles run down kGroupM tile rows before the next tile column, so that the tiles in flight at once
// read few rows of A and few of B from L2.
constexpr int kGroupM = 8;
template <int BN, bool TWO>
__device__ __forceinline__ Item item_at(const Launch& l, int position) {
  Item r;
  int item = TWO && l.tabled ? l.order[position] : position;
  r.which = -1;
  if (item >= l.items) return r;
  r.which = TWO && item >= l.q[0].p.items;
  const Args& p = l.q[TWO ? r.which : 0].p;
  if (TWO && r.which) item -= l.q[0].p.items;
  r.split = item / p.tiles;
  const int t = item - r.split * p.tiles;
  const int g = t / (kGroupM * p.tiles_n), in = t - g * kGroupM * p.tiles_n;
  const int gm = min(kGroupM, p.tiles_m - g * kGroupM);
  const int n = in / gm;
  r.m0 = (g * kGroupM + in - n * gm) * 256;
  r.n0 = n * BN;
  r.i0 = r.split * p.iters;
  r.i1 = min(p.total, r.i0 + p.iters);
  return r;
}

// TWO: a launch of two products, whose epilogues only store. With one, its parameters are at fixed
// places; with two, what the loops need of them is read once per item (read by a computed place in
// every round they cost a fifth of the time).
template <typename T, int BN, bool TWO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_gemm_tc(const __grid_constant__ Launch l) {
  using L = Tile<BN>;
  constexpr int kCols = Out<T>::kCols;
  constexpr bool kSegs = sizeof(T) == 4;  // an item may take several accumulators (fp32)
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + L::OFF_BAR);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->acc_full[i], 1);
      mbar_init(&bars->acc_free[i], 2 * kEpiWarps);
    }
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc_pair(&bars->tmem, L::kTmemCols);
  if (warp == 3 && lane < (TWO ? 2 : 1)) {
    prefetch_map(&l.q[lane].a);
    prefetch_map(&l.q[lane].b);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are up before any remote arrival
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  pdl_trigger();

  if (warp < 4 && warp != 1 && lane == 0) {
    // ------------------------------------------------------------ operand loads
    const int mine = warp ? warp - 1 : 0;  // this loader's stages: mine, mine + kLoaders, ...
    const uint32_t full0 = map_to_first(&bars->full[0]);
    int base = 0;  // stages of the items before
    bool ok = true;
    Item t = item_at<BN, TWO>(l, first);  // the parameters come from a cold constant cache: before the wait
    pdl_wait();
    for (int at = first; ok && at < l.positions; at += step) {
      if (at != first) t = item_at<BN, TWO>(l, at);
      if (t.which < 0) continue;
      const Problem& pr = l.q[TWO ? t.which : 0];
      const CUtensorMap *map_a = &pr.a, *map_b = &pr.b;
      const int a_mn = pr.p.a_mn, b_mn = pr.p.b_mn, fp32 = pr.p.fp32;
      const int ma = t.m0 + (int)rank * 128, nb = t.n0 + (int)rank * (BN / 2), seg = pr.p.seg;
      for (int i0 = t.i0, i1; ok && i0 < t.i1; base += i1 - i0, i0 = i1) {
        i1 = kSegs ? min(t.i1, i0 + seg) : t.i1;
        // fp32: a segment of K goes through all plane pairs, `per` stages each
        const int per = fp32 ? (i1 - i0) / kPlanePairs : 0, k0 = fp32 ? i0 / kPlanePairs : i0;
        const int skip = (mine + kLoaders - base % kLoaders) % kLoaders;
        int s = (base + skip) % L::kStages;
        uint32_t ph = ((base + skip) / L::kStages) & 1;  // the parity of the stage's round
        int pair = fp32 ? skip / per : 0;
        int kb = k0 + skip - pair * per;
        for (int i = i0 + skip; i < i1; i += kLoaders) {
          if (!(ok = wait(&bars->empty[s], ph ^ 1))) break;
          if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * L::kStage);
          const uint32_t bar = full0 + s * 8;
          const uint32_t sa = sbase + s * L::kStage, sb = sa + kABytes;
          const int k = kb * kBK;
          const int pa = fp32 ? plane_a(pair) : 0, pb = fp32 ? plane_b(pair) : 0;
          if (a_mn) {
            tma_load_pair(sa, map_a, ma, k, pa, bar);
            tma_load_pair(sa + 8192, map_a, ma + 64, k, pa, bar);
          } else {
            tma_load_pair(sa, map_a, k, ma, pa, bar);
          }
          if (b_mn) {
#pragma unroll
            for (int c = 0; c < BN / 128; ++c) tma_load_pair(sb + c * 8192, map_b, nb + c * 64, k, pb, bar);
          } else {
            tma_load_pair(sb, map_b, k, nb, pb, bar);
          }
          kb += kLoaders;
          while (fp32 && kb >= k0 + per) { kb -= per; ++pair; }
          s += kLoaders;
          if (s >= L::kStages) { s -= L::kStages; ph ^= 1; }
        }
      }
    }
    // the last stages' loads and releases must have arrived before the CTAs may exit
    for (int j = max(0, base - L::kStages); mine == 0 && j < base; ++j) {
      const int st = j % L::kStages, par = (j / L::kStages) & 1;
      if (rank == 0 && !wait(&bars->full[st], par)) break;
      if (ok) ok = wait(&bars->empty[st], par);
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ------------------------------------------------------------ MMAs of both CTAs
    // Operand descriptors: K-major steps through 16 of a row's 64 elements (32 bytes), MN-major
    // through 16 of 64 rows (2 KB), its 64-wide column blocks 8 KB apart. Only the low word, which
    // holds the address, changes.
    uint32_t s = 0, ph = 0;
    int t = 0;
    bool ok = true;
    for (int at = first; ok && at < l.positions; at += step) {
      const Item w = item_at<BN, TWO>(l, at);
      if (w.which < 0) continue;
      const Args& p = l.q[TWO ? w.which : 0].p;
      const uint64_t da = smem_desc(sbase, p.a_mn ? 8192 : 16, 1024, kSwizzle128B);
      const uint64_t db = smem_desc(sbase + kABytes, p.b_mn ? 8192 : 16, 1024, kSwizzle128B);
      const uint32_t a_hi = (uint32_t)(da >> 32), b_hi = (uint32_t)(db >> 32);
      const uint32_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4, idesc = p.idesc;
      const int seg = p.seg;
      for (int i0 = w.i0, i1; ok && i0 < w.i1; i0 = i1, ++t) {
        i1 = kSegs ? min(w.i1, i0 + seg) : w.i1;
        const int buf = t & 1;
        if (!(ok = wait(&bars->acc_free[buf], ((t >> 1) & 1) ^ 1))) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        uint32_t more = 0;
        for (int i = i0; i < i1; ++i) {
          if (!(ok = wait(&bars->full[s], ph))) break;
          tc_fence_after();
          uint32_t a_lo = (uint32_t)da + s * (L::kStage >> 4), b_lo = (uint32_t)db + s * (L::kStage >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            mma_pair(d, ((uint64_t)a_hi << 32) | a_lo, ((uint64_t)b_hi << 32) | b_lo, idesc, more);
            a_lo += a_step;
            b_lo += b_step;
            more = 1;
          }
          commit_pair(&bars->empty[s]);
          if (++s == L::kStages) { s = 0; ph ^= 1; }
        }
        if (ok) commit_pair(&bars->acc_full[buf]);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int w = warp & 3, quarter = (warp - 4) >> 2;  // TMEM lanes 32w.., columns quarter * BN/4..
    const uint32_t sbuf = sbase + L::OFF_OUT + (warp - 4) * kBuf;
    uint8_t* pbuf = smem + L::OFF_OUT + (warp - 4) * kBuf;
    pdl_wait();
    int t = 0;
    bool ok = true;
    // sends the buffer's rows out (tma = kAdd: adds them), once every lane has written its own
    auto send = [&](const CUtensorMap* map, int tma, T* base, int64_t ld, int row, int n, int store_row, int M, int N) {
      if (tma) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) kSegs && tma == kAdd ? tma_add_2d(map, sbuf, n, store_row) : tma_store_2d(map, sbuf, n, store_row);
      } else {
        __syncwarp();
        copy_rows<T, true>(pbuf, base + (int64_t)row * ld + n, ld, min(32, M - row), N - n, lane);
      }
    };
    auto buffer_free = [&]() {  // its last store, or the warp's own copies, have read it
      if (lane == 0) tma_store_wait_read();
      __syncwarp();
    };
    for (int at = first; ok && at < l.positions; at += step) {
      const Item it = item_at<BN, TWO>(l, at);
      if (it.which < 0) continue;
      const Problem& pr = l.q[TWO ? it.which : 0];
      const Args& p = pr.p;
      const CUtensorMap* map_out = &pr.out;
      const int M = p.M, N = p.N, partial = p.partial, split_row = it.split * p.split_rows;
      for (int i0 = it.i0; ok && i0 < it.i1; i0 = kSegs ? i0 + p.seg : it.i1) {
        const bool later = kSegs && i0 > it.i0, last = !kSegs || i0 + p.seg >= it.i1;
        const bool join = !TWO && later && last && p.join;
        const int out_tma = later && !join ? kAdd : p.out_tma;
        const int buf = t & 1;
        const int row = it.m0 + (int)rank * 128 + w * 32;
        const int n_first = it.n0 + quarter * (BN / 4);
        const int n_end = row < M ? min(N, n_first + BN / 4) : 0;
        const T* res = TWO ? nullptr : static_cast<const T*>(p.res) + (int64_t)row * p.ldr;
        const bool res_vec = !TWO && p.res && p.res_vec;
        uint4 rv[4], bv[4];
        if (last && res_vec && n_first < n_end)
          load_rows(res + n_first, p.ldr, M - row, N - n_first, lane, rv);
        if (!TWO && last && p.bias_vec && n_first < n_end) load_bias(static_cast<const T*>(p.bias) + n_first, N - n_first, bv);
        ok = wait(&bars->acc_full[buf], (t >> 1) & 1);
        ++t;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (later) {
          if (lane == 0) tma_store_wait_done();
          __syncwarp();
        }
        tc_fence_after();
        const uint32_t acc = tmem + buf * BN + quarter * (BN / 4) + ((uint32_t)(w * 32) << 16);
        for (int n = n_first; n < n_end; n += kCols) {
          float v[kCols];
          if constexpr (kCols == 32) tmem_ld32(acc + (n - n_first), v);
          else tmem_ld16(acc + (n - n_first), v);
          tmem_wait_ld();
          if constexpr (sizeof(T) == 2) {
            if (partial) {  // 32 columns of fp32: two rows' worth of the buffer
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                buffer_free();
                write_row<float>(sbuf, lane, *reinterpret_cast<const float(*)[16]>(v + 16 * h));
                send(map_out, 1, static_cast<T*>(nullptr), 0, row, n + 16 * h, split_row + row, M, N);
              }
              continue;
            }
          }
          if constexpr (kSegs && !TWO) {
            if (!last) {
              buffer_free();
              write_row<T>(sbuf, lane, v);
              send(map_out, out_tma, static_cast<T*>(nullptr), 0, row, n, split_row + row, M, N);
              continue;
            }
            if (join) {
              uint4 earlier[4];
              load_rows<T, true>(static_cast<const T*>(p.out) + (int64_t)row * p.ldo + n, p.ldo, M - row, N - n, lane,
                                 earlier);
              buffer_free();
              put_rows(sbuf, lane, earlier);
              __syncwarp();
              add_row<T>(sbuf, lane, v);
            }
          }
          if (!TWO && p.bias) {
            add_bias<T>(static_cast<const T*>(p.bias) + n, p.bias_vec, bv, N - n, v);
            if (p.bias_vec && n + kCols < n_end)
              load_bias(static_cast<const T*>(p.bias) + n + kCols, N - n - kCols, bv);
          }
          if (!TWO && p.slope) {
            buffer_free();
            activate<T, true>(v, p.act, sbuf, lane);
            send(&pr.slope, p.slope_tma, static_cast<T*>(p.slope), N, row, n, row, M, N);  // by size alone
          } else if (!TWO) {
            activate<T, false>(v, p.act, sbuf, lane);
          }
          buffer_free();
          if (!TWO && p.res) {
            if (res_vec) {
              put_rows(sbuf, lane, rv);
              if (n + kCols < n_end)
                load_rows(res + n + kCols, p.ldr, M - row, N - n - kCols, lane, rv);
            } else {
              copy_rows<T, false>(pbuf, const_cast<T*>(res) + n, p.ldr, min(32, M - row), N - n, lane);
            }
            __syncwarp();
            add_row<T>(sbuf, lane, v);
          }
          write_row<T>(sbuf, lane, v);
          send(map_out, out_tma, static_cast<T*>(p.out), p.ldo, row, n, split_row + row, M, N);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_remote(map_to_first(&bars->acc_free[buf]));
      }
    }
    if (lane == 0) tma_store_wait_read();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no arrival, load or MMA of the pair is outstanding past this point
  tc_fence_after();
  if (warp == 2) tmem_free_pair(tmem, L::kTmemCols);
}

// out = epilogue of the K splits' sums, added in order. Four columns per thread; bias and residual are
// read first, beside the sums, at clamped columns (2048 x 1024 -> 1024 fp32 with both: 35.9 us, 38.0 where
// they were read one by one between the stores).
template <typename T>
__global__ void __launch_bounds__(256)
    k_split_sum(const float* part, int64_t split_stride, int ldp, const __grid_constant__ Args p) {
  pdl_wait();
  pdl_trigger();
  const int n = (blockIdx.y * 64 + (threadIdx.x & 63)) * 4;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.N || m >= p.M) return;
  float b[4] = {}, r[4] = {};
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = Elem<T>::load(static_cast<const T*>(p.bias) + min(n + j, p.N - 1));
  }
  if (p.res) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = Elem<T>::load(static_cast<const T*>(p.res) + m * p.ldr + min(n + j, p.N - 1));
  }
  const float* src = part + m * ldp + n;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < p.splits; i += 4) {  // four splits' loads together, added in order
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = *reinterpret_cast<const float4*>(src + (int64_t)min(i + j, p.splits - 1) * split_stride);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i + j >= p.splits) break;
      s.x += v[j].x; s.y += v[j].y; s.z += v[j].z; s.w += v[j].w;
    }
  }
  float z[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j >= p.N) break;
    float slope;
    const float y = act_value<Out<T>::kFast>(z[j] + b[j], p.act, slope) + r[j];
    if (p.slope) store_slope(static_cast<Slope<T>*>(p.slope) + m * p.N + n + j, slope);
    Elem<T>::store(static_cast<T*>(p.out) + m * p.ldo + n + j, y);
  }
}

// ---------------------------------------------------------------------------
// packing
// ---------------------------------------------------------------------------
struct PackOne {
  const void* src;
  uint16_t* dst;  // rows of `pitch` elements, the columns past `cols` zero
  int64_t ld, rows, plane;
  int cols, pitch, vec, first;  // vec: 16-byte loads; first: the matrix's first block
};
struct PackArgs {
  PackOne m[kMaxPack];
  int count;
};
// Eight columns per thread and step; a run of blocks per matrix.
template <typename T>
__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ PackArgs args) {
  sm100::pdl_wait();
  sm100::pdl_trigger();
  int which = 0;
  while (which + 1 < args.count && (int)blockIdx.x >= args.m[which + 1].first) ++which;
  const PackOne& p = args.m[which];
  const int blocks = (which + 1 < args.count ? args.m[which + 1].first : (int)gridDim.x) - p.first;
  const int per_row = p.pitch / 8;
  const int64_t groups = p.rows * per_row;
  for (int64_t i = ((int)blockIdx.x - p.first) * 256ll + threadIdx.x; i < groups; i += blocks * 256ll) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row) * 8;
    const T* s = static_cast<const T*>(p.src) + r * p.ld + c;
    uint16_t* dst = p.dst + r * p.pitch + c;
    alignas(16) uint16_t o[3][8];
    if constexpr (sizeof(T) == 4) {
      float v[8];
      if (p.vec) {
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(s);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(s + 4);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s[min(e, p.cols - 1 - c)];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e >= p.cols) v[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint16_t t[3];
        split3(v[e], t);
        o[0][e] = t[0]; o[1][e] = t[1]; o[2][e] = t[2];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
        *reinterpret_cast<uint4*>(dst + q * p.plane) = *reinterpret_cast<const uint4*>(o[q]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[0][e] = *reinterpret_cast<const uint16_t*>(s + min(e, p.cols - 1 - c));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e >= p.cols) o[0][e] = 0;
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o[0]);
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

int64_t pitch_of(int cols) { return ((int64_t)cols + 7) / 8 * 8; }

struct Config {
  int bn, splits, iters, total, tiles_m, tiles_n;
  int seg;       // stages per accumulator
  bool partial;  // fp32 sums in the workspace, then k_split_sum
  bool direct;   // fp32 sums in the result itself
};

bool tma_rows(const void* p, int64_t ld, size_t es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0;
}
bool bare(const Gemm& g) { return !g.bias && !g.res && !g.slope && g.act == MURM_ACT_NONE; }

// The tensor cores cut each partial sum to 24 bits. So that fp32 keeps its accuracy whatever K is, an
// accumulator of fp32 takes at most kSegment stages of K. An item's first segment is stored, each further
// one added to it in global memory in fp32 (rounded; by the pair that stored it, in order; sums below
// 2^-126 count as 0): in the result itself where K is not split and 16-byte rows allow it, and there the
// last segment reads what the others left, if an epilogue follows. Error in parts of its norm and time, by
// the most of K a segment takes (512, 768, 1024; all of it): 4096^3 5.2e-7 666 us, 7.0e-7 651, 1.05e-6 637,
// 4.5e-6 613 (plain fp32 1.1e-6); 4096 x 1024 -> 4096 5.2e-7 165, the same, 1.05e-6 157 (5.7e-7); dW of 64 x 64
// over 40000 rows 5.3e-7, 6.5e-7, 8.8e-7, all 86 us (8.4e-7).
constexpr int kSegment = 768 / kBK;

Config config(const Gemm& g, int bn, int splits) {
  const bool fp32 = g.a.planes == 3;
  const int kblocks = (g.K + kBK - 1) / kBK, pairs = fp32 ? kPlanePairs : 1;
  const int blocks = (kblocks + splits - 1) / splits;  // of a split
  const int segments = fp32 ? (blocks + kSegment - 1) / kSegment : 1;
  Config c{};
  c.bn = bn;
  c.total = kblocks * pairs;
  c.iters = blocks * pairs;
  c.splits = (c.total + c.iters - 1) / c.iters;
  c.tiles_m = (g.M + 255) / 256;
  c.tiles_n = (g.N + bn - 1) / bn;
  c.seg = (blocks + segments - 1) / segments * pairs;
  c.direct = c.splits == 1 && segments > 1 && tma_rows(g.out, g.ldo, 4) && g.N % 4 == 0 && g.res != g.out;
  c.partial = !c.direct && (c.splits > 1 || segments > 1);
  return c;
}

// Tile width and K splits by estimated time, in microseconds measured on B200:
// - with all pairs busy a 64-deep stage takes 0.35 of a 256-wide tile and 0.31 of a 128-wide one (its
//   MMAs take half as long, but the wait for a stage, its MMAs' issue and its release do not). So 128
//   pays only where it leaves fewer rounds: 512 x 1024 x 1024: 8.9 us at 128, 9.8 at 256;
//   8192 x 1024 x 1024: 25.9 and 16.7.
// - a split costs a second launch, and its fp32 sums about 4.8 MB per us:
//   1024 x 1024 x 8192 (dW): 24 us in three parts, 21 in four, 24 in eight.
// - a launch of its own costs about 5 (prologue, first loads, last epilogue).
constexpr double kLaunchUs = 5.0;
double stage_us(int bn) { return bn == 256 ? 0.35 : 0.31; }
double split_us(const Config& c) {
  const double tiles = (double)c.tiles_m * c.tiles_n * 256 * c.bn * 4 / 9.6e6;  // one pass over all
  const double rest = c.partial ? 4.0 + tiles * c.splits : 0.0;  // k_split_sum
  return c.partial || c.direct ? rest + tiles * ((c.total + c.seg - 1) / c.seg) : 0.0;
}
// fp32 items are six times as long, so that splits may pay for more of them (both gradients of 4200 x 1100
// -> 4100: 470 us so, 550 with two rounds at most; of 4096^3 1180, with eight 1400).
bool split_fits(const Gemm& g, const Config& c, int splits) {
  const int most = (g.a.planes == 3 ? 4 : 2) * kPairs;
  return splits == 1 || (c.total / splits >= 2 && (int64_t)c.tiles_m * c.tiles_n * splits <= most);
}
double choose_one(const Gemm& g, Config* best) {
  double best_t = 0;
  for (int bn : {256, 128})
    for (int splits = 1; splits <= 16; ++splits) {
      const Config c = config(g, bn, splits);
      if (!split_fits(g, c, splits)) break;
      const int64_t rounds = ((int64_t)c.tiles_m * c.tiles_n * c.splits + kPairs - 1) / kPairs;
      const double t = rounds * c.iters * stage_us(bn) + split_us(c);
      if (best_t == 0 || t < best_t) {
        best_t = t;
        *best = c;
      }
    }
  return best_t + kLaunchUs;
}

struct Plan {
  Config c[2];
  bool together;
};
// Two products together: no shorter than their work over all pairs, than the longest item, or than
// what the last item of a pair leaves idle (about a quarter of the shorter ones); side by side they
// also run a tenth slower than alone (two sets of operands in L2, and no SM left idle whose power the
// others could use). Both gradients of 2048 x 1024 x 1024: 15.3 us, apart 23.9; of 8192 x 1024 x 1024
// 33.7 and 39.3, of 4096 x 1024 x 4096 48.0 and 52.5, of 32768 x 1024 x 4096 406 and 378.
constexpr double kTogether = 1.1;
Plan choose(const Gemm* g, int count) {
  Plan p{};
  double apart = 0;
  for (int i = 0; i < count; ++i) apart += choose_one(g[i], &p.c[i]);
  if (count < 2) return p;
  constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};
  struct Option {
    Config c;
    double item, work, extra;
  } opt[2][8];
  for (int bn : {256, 128}) {
    int n[2] = {0, 0};
    for (int i = 0; i < 2; ++i)
      for (int splits : kSplits) {
        Option& o = opt[i][n[i]];
        o.c = config(g[i], bn, splits);
        if (!split_fits(g[i], o.c, splits)) break;
        o.item = o.c.iters * stage_us(bn);
        o.work = o.item * o.c.tiles_m * o.c.tiles_n * o.c.splits;
        o.extra = split_us(o.c);
        ++n[i];
      }
    for (int a = 0; a < n[0]; ++a)
      for (int b = 0; b < n[1]; ++b) {
        const Option &x = opt[0][a], &y = opt[1][b];
        const double work = kTogether * (x.work + y.work) / kPairs + (x.item < y.item ? x.item : y.item) / 4;
        const double longest = x.item > y.item ? x.item : y.item;
        const double t = kLaunchUs + x.extra + y.extra + (work > longest ? work : longest);
        if (t < apart) {
          apart = t;
          p.c[0] = x.c;
          p.c[1] = y.c;
          p.together = true;
        }
      }
  }
  return p;
}

// The items of both products over the pairs, the longer ones (the first n0) first, then the others to
// the pairs with the least to do so far. All items of a product are taken to be of one length, so the
// pairs are of two kinds at any time: those with one more of the long items and the rest.
void fill_order(Launch* l, int n0, int len0, int n1, int len1, int pairs) {
  for (int i = 0; i < kMaxOrder; ++i) l->order[i] = kNone;
  int slot[2] = {n0 / pairs + (n0 % pairs ? 1 : 0), n0 / pairs};  // rows of the table taken, per kind
  const int cut = n0 % pairs;                                     // pairs below it have one more
  for (int i = 0; i < n0; ++i) l->order[i] = (uint16_t)i;
  int load[2] = {slot[0] * len0, slot[1] * len0};
  int next = n0;
  const int end = n0 + n1;
  while (next < end) {
    const int kind = cut && load[0] < load[1] ? 0 : 1;
    const int from = kind ? cut : 0, to = kind ? pairs : cut;
    for (int j = from; j < to && next < end; ++j) {
      const int at = slot[kind] * pairs + j;
      if (at >= kMaxOrder) {  // too uneven for the table: in plain order
        l->tabled = 0;
        l->positions = l->items;
        return;
      }
      l->order[at] = (uint16_t)next++;
    }
    ++slot[kind];
    load[kind] += len1;
  }
  const int rows = slot[0] > slot[1] ? slot[0] : slot[1];
  l->tabled = 1;
  l->positions = rows * pairs;
}

// Operands: three dimensions (the planes) and 128-byte swizzled rows; results (planes = 0): two
// dimensions and the epilogue's 64-byte rows.
CUresult encode(CUtensorMap* map, CUtensorMapDataType type, size_t es, const void* p, int64_t cols, int64_t rows,
                int64_t ld, int planes, int64_t plane, int box_cols, int box_rows) {
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * es), (cuuint64_t)((planes > 1 ? plane : ld) * es)};
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  cuuint32_t unit[3] = {1, 1, 1};
  return tc_tensor_map_encoder()(map, type, planes ? 3 : 2, const_cast<void*>(p), dims, strides, box, unit,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 planes ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == MURM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                           : dtype == MURM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

template <typename... KArgs, typename... Args>
void launch(const char* name, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st,
            Args&&... args) {
  MURM_LAUNCH_PDL(name, kernel, grid, threads, smem, st, args...);
}

// Fills a launch's product.
template <typename T, int BN>
CUresult describe(const Gemm& g, const Config& c, void* workspace, Problem* q) {
  const size_t es = sizeof(T);
  constexpr int kCols = Out<T>::kCols;
  Args& p = q->p;
  p = Args{};
  p.M = g.M; p.N = g.N;
  p.iters = c.iters; p.total = c.total; p.splits = c.splits; p.seg = c.seg;
  p.tiles_m = c.tiles_m;
  p.tiles_n = c.tiles_n;
  p.tiles = c.tiles_m * c.tiles_n;
  p.items = p.tiles * c.splits;
  p.idesc = idesc_f16(g.dtype == MURM_F16 ? 0 : 1, 256, c.bn, g.a_mn, g.b_mn);
  p.a_mn = g.a_mn; p.b_mn = g.b_mn;
  p.fp32 = g.a.planes == 3;
  const CUtensorMapDataType op = g.dtype == MURM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapDataType ot = map_type(g.dtype);
  CUresult r;
  if (g.a_mn) r = encode(&q->a, op, 2, g.a.p, g.M, g.K, g.a.ld, g.a.planes, g.a.plane, 64, 64);
  else r = encode(&q->a, op, 2, g.a.p, g.K, g.M, g.a.ld, g.a.planes, g.a.plane, 64, 128);
  if (r != CUDA_SUCCESS) return r;
  if (g.b_mn) r = encode(&q->b, op, 2, g.b.p, g.N, g.K, g.b.ld, g.b.planes, g.b.plane, 64, 64);
  else r = encode(&q->b, op, 2, g.b.p, g.K, g.N, g.b.ld, g.b.planes, g.b.plane, 64, BN / 2);
  if (r != CUDA_SUCCESS) return r;
  if (c.partial) {  // partial sums alone; the epilogue follows in k_split_sum
    p.partial = 1;
    p.M = p.split_rows = c.tiles_m * 256;
    p.N = c.tiles_n * BN;
    p.out = workspace;
    p.ldo = p.N;
    p.out_tma = 1;
    return encode(&q->out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, workspace, p.N, (int64_t)p.M * c.splits, p.ldo, 0, 0, 16,
                  32);
  }
  p.bias = g.bias; p.act = g.act;
  p.res = g.res; p.ldr = g.ldr;
  p.out = g.out; p.ldo = g.ldo;
  p.slope = g.slope;
  p.join = c.direct && !bare(g);
  const int per = 16 / (int)es;
  p.res_vec = p.res && tma_rows(p.res, p.ldr, es) && g.N % per == 0;
  p.bias_vec = p.bias && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0 && g.N % per == 0;
  p.out_tma = tma_rows(g.out, g.ldo, es);
  if (p.out_tma) r = encode(&q->out, ot, es, g.out, g.N, g.M, g.ldo, 0, 0, kCols, 32);
  if (r == CUDA_SUCCESS && p.slope) {
    p.slope_tma = tma_rows(p.slope, g.N, es);
    if (p.slope_tma) r = encode(&q->slope, ot, es, p.slope, g.N, g.M, g.N, 0, 0, kCols, 32);
  }
  return r;
}

size_t split_bytes(const Config& c) {
  return !c.partial ? 0 : (size_t)c.splits * c.tiles_m * 256 * c.tiles_n * c.bn * sizeof(float);
}

// One launch of one or two products with the same tile width, then the sums of those with splits.
template <typename T, int BN>
murm_status launch_tc(const Gemm* g, const Config* c, int count, char* workspace, cudaStream_t st) {
  Launch l;
  l.items = l.tabled = 0;
  // the product with the longer items comes first
  const int swap = count == 2 && c[1].iters > c[0].iters;
  float* part[2];
  for (int i = 0; i < count; ++i) {
    part[i] = reinterpret_cast<float*>(workspace);
    workspace += split_bytes(c[i]);
    const CUresult r = describe<T, BN>(g[i], c[i], part[i], &l.q[i ^ swap]);
    if (r != CUDA_SUCCESS) {
      char msg[96];
      snprintf(msg, sizeof msg, "linear: a tensor map was refused (%d)", (int)r);
      return report_error(MURM_ERR_CUDA, msg);
    }
    l.items += l.q[i ^ swap].p.items;
  }
  l.positions = l.items;
  const int pairs = l.items < kPairs ? l.items : kPairs;
  if (count == 2 && l.items <= kMaxOrder)
    fill_order(&l, l.q[0].p.items, l.q[0].p.iters, l.q[1].p.items, l.q[1].p.iters, pairs);
  auto* kernel = count == 2 ? k_gemm_tc<T, BN, true> : k_gemm_tc<T, BN, false>;
  if (cudaError_t e = smem_opt_in(kernel, Tile<BN>::kSmem)) return report_error(MURM_ERR_CUDA, cudaGetErrorString(e));
  launch("linear_gemm", kernel, dim3(2 * pairs), kThreads, Tile<BN>::kSmem, st, l);
  for (int i = 0; i < count; ++i) {
    if (!c[i].partial) continue;
    Args p = l.q[i ^ swap].p;
    const int ldp = p.N;
    const int64_t stride = (int64_t)p.M * p.N;
    p.M = g[i].M; p.N = g[i].N;
    p.bias = g[i].bias; p.act = g[i].act;
    p.res = g[i].res; p.ldr = g[i].ldr;
    p.out = g[i].out; p.ldo = g[i].ldo;
    p.slope = g[i].slope;
    launch("linear_split_sum", k_split_sum<T>, dim3((p.M + 3) / 4, (p.N + 255) / 256), 256, 0, st,
           const_cast<const float*>(part[i]), stride, ldp, p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MURM_OK : report_error(MURM_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T>
murm_status run(const Gemm* g, int count, char* workspace, cudaStream_t st) {
  const Plan p = choose(g, count);
  auto go = [&](const Gemm* gs, const Config* cs, int n, char* ws) {
    return cs[0].bn == 256 ? launch_tc<T, 256>(gs, cs, n, ws, st) : launch_tc<T, 128>(gs, cs, n, ws, st);
  };
  if (p.together) return go(g, p.c, 2, workspace);
  for (int i = 0; i < count; ++i) {
    if (murm_status s = go(g + i, p.c + i, 1, workspace)) return s;
    workspace += split_bytes(p.c[i]);
  }
  return MURM_OK;
}

}  // namespace

size_t gemm_workspace(const Gemm* g, int count) {
  const Plan p = choose(g, count);
  return split_bytes(p.c[0]) + (count > 1 ? split_bytes(p.c[1]) : 0);
}

murm_status gemm(const Gemm* g, int count, void* workspace, cudaStream_t st) {
  if (!tc_tensor_map_encoder()) return report_error(MURM_ERR_CUDA, "linear: cuTensorMapEncodeTiled is not available");
  char* ws = static_cast<char*>(workspace);
  switch (g[0].dtype) {
    case MURM_F32: return run<float>(g, count, ws, st);
    case MURM_F16: return run<__half>(g, count, ws, st);
    default: return run<__nv_bfloat16>(g, count, ws, st);
  }
}

bool needs_pack(int dtype, const Matrix& m) { return dtype == MURM_F32 || !tma_rows(m.p, m.ld, 2); }

size_t pack_bytes(int dtype, const Matrix& m) {
  return (size_t)m.rows * pitch_of(m.cols) * 2 * (dtype == MURM_F32 ? 3 : 1);
}

Operand packed_at(int dtype, const Matrix& m, void* dst) {
  return Operand{dst, pitch_of(m.cols), m.rows * pitch_of(m.cols), dtype == MURM_F32 ? 3 : 1};
}

murm_status pack(int dtype, const Matrix* m, void* const* dst, int count, cudaStream_t st) {
  PackArgs a{};
  a.count = count;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    const int pitch = (int)pitch_of(m[i].cols);
    a.m[i] = PackOne{m[i].p, static_cast<uint16_t*>(dst[i]), m[i].ld, m[i].rows, m[i].rows * pitch, m[i].cols, pitch,
                     dtype == MURM_F32 && m[i].cols % 8 == 0 && tma_rows(m[i].p, m[i].ld, 4), (int)blocks};
    const int64_t need = (m[i].rows * (pitch / 8) + 255) / 256;
    blocks += need < kSms * 16 ? need : kSms * 16;
  }
  if (dtype == MURM_F32) launch("linear_pack", k_pack<float>, dim3((unsigned)blocks), 256, 0, st, a);
  else launch("linear_pack", k_pack<__half>, dim3((unsigned)blocks), 256, 0, st, a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MURM_OK : report_error(MURM_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace lin
}  // namespace murm
