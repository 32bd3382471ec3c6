// What a training step does to a list of gradients around the codecs: the global norm, clipping by it, and for the
// sparsifier momentum correction and momentum factor masking.
//
//   norm      S = sum over all tensors of g^2 (or the largest |g|), N = sqrt(S) (or S)
//   clip      c = scale * min(1, max_norm / (|scale| N + 1e-6)); out = c g
//   momentum  u = m u + c g; where asked for, d = m u + c g (Nesterov's direction)
//   mask      u[i] = 0 for every index i of a sparsifier message
//
// All four are streams over lists of tensors described by a table in the kernel-argument segment, as in the codecs.  What a
// call needs beyond its tensors lies in the caller's result block, so nothing is allocated, nothing waits, and two graphs
// that were captured on one stream share nothing.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <vector>

#include "hpx_common.h"
#include "hpx_tables.h"

namespace {
using namespace hpx;

constexpr int kThreads = 256;

// ---- the result block --------------------------------------------------------
// doubles: [0] S, [1] norm, [2] coefficient, [3] arrivals, [16 ...] a partial sum per workgroup, then the arrivals of each group
// of workgroups, a cache line each.  All arrivals are zero between calls.
constexpr int kArrivals = 3;
constexpr int kSlots = 16;
constexpr int kMaxGrid = 512;  // two workgroups of 512 lanes on each of 256 CUs
constexpr int kGroups = 16;
constexpr int kGroupArrivals = kSlots + kMaxGrid;
constexpr int kLineDoubles = 16;
static_assert(kGroupArrivals + kGroups * kLineDoubles <= HPX_GRAD_RESULT, "result block too small");

// ---- tables ------------------------------------------------------------------
// An element count and its type share a word.  (The limit of a count, far beyond any memory, keeps sums of them in 64 bits and the
// tiles of a tensor in the norm, which takes it as a whole, in 32.)
constexpr int kTypeShift = 56;
constexpr int64_t kMaxSize = int64_t(1) << 40;
__host__ __device__ inline int64_t seg_size(uint64_t nt) { return int64_t(nt & ((uint64_t(1) << kTypeShift) - 1)); }
__host__ __device__ inline int seg_type(uint64_t nt) { return int(nt >> kTypeShift); }

struct NormSeg {
  const void* g;
  uint64_t nt;
  static constexpr int kCapLarge = 448;
};
struct ClipSeg {
  const void* g;
  void* out;  // in place: g itself, in its type; else fp32
  uint64_t nt;
  static constexpr int kCapLarge = 320;
};
struct MomentumSeg {
  const void* g;
  float* u;
  float* d;
  uint64_t nt;
  static constexpr int kCapLarge = 256;
};
struct MaskSeg {
  const uint8_t* in;
  float* u;
  int32_t in_size;
  int32_t n;
  static constexpr int kCapLarge = 320;
};
constexpr int kCapSmall = 8;

static_assert(sizeof(Table<NormSeg, NormSeg::kCapLarge>) <= 9600 && sizeof(Table<ClipSeg, ClipSeg::kCapLarge>) <= 9600 &&
                  sizeof(Table<MomentumSeg, MomentumSeg::kCapLarge>) <= 9600 && sizeof(Table<MaskSeg, MaskSeg::kCapLarge>) <= 9600,
              "kernel-argument budget");

// ---- element types -----------------------------------------------------------
template <int TYPE>
struct Elem;
template <>
struct Elem<HPX_F32> {
  using raw = uint32_t;
  __device__ static float to(raw v) { return __uint_as_float(v); }
  __device__ static raw from(float v) { return __float_as_uint(v); }
};
template <>
struct Elem<HPX_BF16> {
  using raw = uint16_t;
  __device__ static float to(raw v) { return __uint_as_float(uint32_t(v) << 16); }
  __device__ static raw from(float v) {  // to nearest, ties to even; a NaN stays one
    const uint32_t b = __float_as_uint(v);
    return raw(v != v ? (b >> 16) | 0x40u : (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);
  }
};
template <>
struct Elem<HPX_F16> {
  using raw = uint16_t;
  __device__ static float to(raw v) { return float(__builtin_bit_cast(_Float16, v)); }
  __device__ static raw from(float v) { return __builtin_bit_cast(raw, _Float16(v)); }
};

// Four consecutive elements as they lie in memory; a tensor may start at any element.
template <typename Raw>
struct __attribute__((packed, aligned(sizeof(Raw)))) Raw4 {
  uint32_t w[sizeof(Raw)];
};
template <int TYPE>
using raw4 = Raw4<typename Elem<TYPE>::raw>;

// STREAM: with the non-temporal hint (see ld4_stream), which a list larger than kPlainBytes wants; one that is smaller may lie in the
// caches, and stays there.
template <int TYPE, bool STREAM>
__device__ __forceinline__ raw4<TYPE> load4(const void* base, int64_t e) {
  const raw4<TYPE>* q = reinterpret_cast<const raw4<TYPE>*>(static_cast<const typename Elem<TYPE>::raw*>(base) + e);
  if constexpr (!STREAM) return *q;
  raw4<TYPE> r;
#pragma unroll
  for (unsigned i = 0; i < sizeof(typename Elem<TYPE>::raw); i++) r.w[i] = __builtin_nontemporal_load(&q->w[i]);
  return r;
}
// Bytes that a writing pass reads.  Plain / streaming loads: clipping 16 M fp32 elements 33.0 / 34.2 us, 32 M 61.4 / 60.4, 64 M bf16
// 79.6 / 78.6; momentum of 4 M fp32 elements 9.5 / 10.1, 12 M (96 MB) 24.1 / 24.8, 16 M 34.8 / 31.7, 138 M 297 / 258.  Stores stream at
// every size: clipping 4 M elements 13.0 us against 14.1 with plain ones, 64 M 117 against 139.
constexpr int64_t kPlainBytes = int64_t(96) << 20;
template <int TYPE>
__device__ __forceinline__ void store4_stream(void* base, int64_t e, float4 x) {
  using E = Elem<TYPE>;
  uint32_t w[sizeof(typename E::raw)];
  if constexpr (TYPE == HPX_F32) {
    w[0] = E::from(x.x); w[1] = E::from(x.y); w[2] = E::from(x.z); w[3] = E::from(x.w);
  } else {
    w[0] = E::from(x.x) | uint32_t(E::from(x.y)) << 16;
    w[1] = E::from(x.z) | uint32_t(E::from(x.w)) << 16;
  }
  raw4<TYPE>* q = reinterpret_cast<raw4<TYPE>*>(static_cast<typename E::raw*>(base) + e);
#pragma unroll
  for (unsigned i = 0; i < sizeof(typename E::raw); i++) __builtin_nontemporal_store(w[i], &q->w[i]);
}
template <int TYPE>
__device__ __forceinline__ float4 value4(const raw4<TYPE>& r) {
  using E = Elem<TYPE>;
  if constexpr (TYPE == HPX_F32) return make_float4(E::to(r.w[0]), E::to(r.w[1]), E::to(r.w[2]), E::to(r.w[3]));
  else return make_float4(E::to(uint16_t(r.w[0])), E::to(uint16_t(r.w[0] >> 16)), E::to(uint16_t(r.w[1])), E::to(uint16_t(r.w[1] >> 16)));
}
template <int TYPE>
__device__ __forceinline__ float load1(const void* base, int64_t e) { return Elem<TYPE>::to(static_cast<const typename Elem<TYPE>::raw*>(base)[e]); }
template <int TYPE>
__device__ __forceinline__ void store1(void* base, int64_t e, float x) { static_cast<typename Elem<TYPE>::raw*>(base)[e] = Elem<TYPE>::from(x); }

// ---- norm --------------------------------------------------------------------
// Squares and their sums are fp64: a square of a large or small fp32 value leaves fp32's range, and the sum of 10^8 of them its
// precision.  (|g| is taken as its bit pattern: patterns order as magnitudes do, and a NaN's lies above infinity's.)
template <int ORDER>
struct Sum;
template <>
struct Sum<2> {
  double v = 0.0;
  __device__ void add(float x) { const double d = double(x); v = fma(d, d, v); }
  __device__ double value() const { return v; }
  __device__ static double join(double a, double b) { return a + b; }
};
template <>
struct Sum<HPX_NORM_MAX> {
  uint32_t v = 0u;
  __device__ void add(float x) { const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu; v = b > v ? b : v; }
  __device__ double value() const { return double(__uint_as_float(v)); }
  __device__ static double join(double a, double b) {
    const int64_t x = __double_as_longlong(a) & INT64_MAX, y = __double_as_longlong(b) & INT64_MAX;
    return __longlong_as_double(x > y ? x : y);
  }
};

// Tiles of 32 KiB are counted from the tensor's first element, not from a boundary of memory: which elements a partial sum is
// made of, and so every bit of the result, then depends on types, sizes and values alone, and ranks that hold the same gradients
// at other addresses find the same norm.
constexpr int kNormThreads = 512;
constexpr uint32_t kNormTileBytes = 32768;
constexpr int kNormIters = kNormTileBytes / (kNormThreads * 16);
inline int64_t norm_tiles(int64_t n, int type) {
  const int64_t per = kNormTileBytes / (type == HPX_F32 ? 4 : 2);
  return (n + per - 1) / per;
}

// Sixteen bytes of a tensor that may start at any element.
template <typename Raw>
struct __attribute__((packed, aligned(sizeof(Raw)))) Chunk {
  uint32_t w[4];
};

template <int ORDER, int TYPE>
__device__ __forceinline__ void norm_chunk(Sum<ORDER>& s, const Chunk<typename Elem<TYPE>::raw>& c) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (TYPE == HPX_F32) {
      s.add(__uint_as_float(c.w[i]));
    } else {
      s.add(Elem<TYPE>::to(uint16_t(c.w[i])));
      s.add(Elem<TYPE>::to(uint16_t(c.w[i] >> 16)));
    }
  }
}

// Tiles t, t + step, ... below t1 of one tensor.  Those below `keep` are loaded streaming, the others so that they stay in the
// Infinity Cache (see kKeepBytes).
template <int ORDER, int TYPE>
__device__ __forceinline__ void norm_tiles_of(Sum<ORDER>& s, const void* p, int64_t n, int64_t t, int64_t t1, int step, int64_t keep) {
  using Raw = typename Elem<TYPE>::raw;
  constexpr int kPer = 16 / sizeof(Raw);  // elements of a chunk
  constexpr int64_t kTile = kNormTileBytes / sizeof(Raw);
  const Raw* at = static_cast<const Raw*>(p) + t * kTile + threadIdx.x * kPer;
  const int64_t whole = n / kTile < t1 ? n / kTile : t1;
  // (two loops: of both kinds of load in one the compiler makes plain ones)
  for (; t < whole && t < keep; t += step, at += step * kTile) {
    Chunk<Raw> c[kNormIters];
#pragma unroll
    for (int k = 0; k < kNormIters; k++) {
      const Chunk<Raw>* q = reinterpret_cast<const Chunk<Raw>*>(at + k * kNormThreads * kPer);
#pragma unroll
      for (int i = 0; i < 4; i++) c[k].w[i] = __builtin_nontemporal_load(&q->w[i]);
    }
#pragma unroll
    for (int k = 0; k < kNormIters; k++) norm_chunk<ORDER, TYPE>(s, c[k]);
  }
  for (; t < whole; t += step, at += step * kTile) {
    Chunk<Raw> c[kNormIters];
#pragma unroll
    for (int k = 0; k < kNormIters; k++) c[k] = *reinterpret_cast<const Chunk<Raw>*>(at + k * kNormThreads * kPer);
#pragma unroll
    for (int k = 0; k < kNormIters; k++) norm_chunk<ORDER, TYPE>(s, c[k]);
  }
  if (t < t1) {
    // The tensor's last tile: whole chunks, and what is left of the last one an element to a lane; all requested together.
    const int64_t left = n - t * kTile;
    const int chunks = int(left / kPer), rest = int(left % kPer);
    Chunk<Raw> c[kNormIters];
    float one = 0.f;
    if (int(threadIdx.x) < rest) one = load1<TYPE>(p, n - rest + threadIdx.x);
#pragma unroll
    for (int k = 0; k < kNormIters; k++)
      if (k * kNormThreads + int(threadIdx.x) < chunks) c[k] = *reinterpret_cast<const Chunk<Raw>*>(at + k * kNormThreads * kPer);
#pragma unroll
    for (int k = 0; k < kNormIters; k++)
      if (k * kNormThreads + int(threadIdx.x) < chunks) norm_chunk<ORDER, TYPE>(s, c[k]);
    s.add(one);
  }
}

// Over a wave and over a workgroup of WAVES waves, the same order of additions whatever the timing.  By lane permutes, as
// wave_reduce: few and short instructions, for at the end of a launch they come from memory one cache line after the other (the
// hand-over of a norm took 2.5 us longer with four of these unrolled side by side).
template <int ORDER>
__device__ __forceinline__ double wave_join(double v) {
  auto perm = [](double x, auto ctrl, auto rows) {
    const uint64_t b = __double_as_longlong(x);
    const int lo = int(uint32_t(b)), hi = int(uint32_t(b >> 32));
    const uint32_t l = uint32_t(__builtin_amdgcn_update_dpp(lo, lo, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    const uint32_t h = uint32_t(__builtin_amdgcn_update_dpp(hi, hi, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    return __longlong_as_double(int64_t(uint64_t(h) << 32 | l));
  };
  using std::integral_constant;
  using J = Sum<ORDER>;
  v = J::join(v, perm(v, integral_constant<int, 0xB1>{}, integral_constant<int, 0xF>{}));   // quad_perm [1,0,3,2]
  v = J::join(v, perm(v, integral_constant<int, 0x4E>{}, integral_constant<int, 0xF>{}));   // quad_perm [2,3,0,1]
  v = J::join(v, perm(v, integral_constant<int, 0x141>{}, integral_constant<int, 0xF>{}));  // row_half_mirror
  v = J::join(v, perm(v, integral_constant<int, 0x140>{}, integral_constant<int, 0xF>{}));  // row_mirror
  v = J::join(v, perm(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{}));  // row_bcast:15 into rows 1 and 3
  v = J::join(v, perm(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{}));  // row_bcast:31 into rows 2 and 3
  const uint64_t b = __double_as_longlong(v);
  const uint32_t l = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), kWave - 1)), h = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b >> 32)), kWave - 1));
  return __longlong_as_double(int64_t(uint64_t(h) << 32 | l));
}
template <int ORDER, int WAVES>
__device__ __forceinline__ double block_join(double v, double* lds) {
  v = wave_join<ORDER>(v);
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; w++) v = Sum<ORDER>::join(v, lds[w]);
  return v;
}

// The partial sums of all workgroups.  One wave that takes them all, and the four waves of a workgroup that request a quarter each
// and exchange them through LDS, add them in the same order.
constexpr int kQuarters = 4;
template <int ORDER>
__device__ __forceinline__ double slots_quarter(const double* slots, int used, int quarter) {
  constexpr int kEach = kMaxGrid / kQuarters / kWave;
  const int first = quarter * kEach * kWave + (threadIdx.x & (kWave - 1));
  // (every slot is loaded, whoever may have written it: a load behind a branch of its own waits for the one before)
  double v[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i++) v[i] = __hip_atomic_load(&slots[first + i * kWave], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  double sum = first < used ? v[0] : 0.0;
#pragma unroll
  for (int i = 1; i < kEach; i++) sum = Sum<ORDER>::join(sum, first + i * kWave < used ? v[i] : 0.0);
  return sum;
}
template <int ORDER>
__device__ __forceinline__ double slots_join(const double* slots, int used) {
  double v = slots_quarter<ORDER>(slots, used, 0);
#pragma unroll
  for (int i = 1; i < kQuarters; i++) v = Sum<ORDER>::join(v, slots_quarter<ORDER>(slots, used, i));
  return wave_join<ORDER>(v);
}
template <int ORDER>
__device__ __forceinline__ double slots_join(const double* slots, int used, double (&lds)[kQuarters][kWave]) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  lds[wave][lane] = slots_quarter<ORDER>(slots, used, wave);
  __syncthreads();
  double v = lds[0][lane];
#pragma unroll
  for (int i = 1; i < kQuarters; i++) v = Sum<ORDER>::join(v, lds[i][lane]);
  return wave_join<ORDER>(v);
}

template <int ORDER>
__device__ __forceinline__ void norm_result(double* result, double v, int add) {
  if (add) v = Sum<ORDER>::join(result[0], v);
  result[0] = v;
  result[1] = ORDER == 2 ? sqrt(v) : v;
}

// What a later call reads again should still be in the 256 MB Infinity Cache: the last kKeepBytes of a list are loaded so that they
// stay there, what lies before them streaming.  302 M bf16 elements (604 MB) clipped into fp32: norm 96 us and clipping 269, with
// streaming loads throughout 94 and 283, with plain ones 106 and 271.
constexpr int64_t kKeepBytes = int64_t(192) << 20;

// One pass over the list.  A workgroup sums every gridDim.x-th tile and leaves one partial sum; the last to arrive joins them in
// their order, so the result does not depend on who that is.  Bound by memory: 604 MB at 6.3 TB/s, 102 MB in 161 tensors 20.1 us
// (5.1 TB/s, of which about 4 us are the launch and the hand-over), and 18.3 where the Infinity Cache holds them.  The hand-over is a store, a wait and an atomic of agent scope.
// Stores of that scope are written through, so the wait for their acknowledgement orders them before the atomic; a release fence,
// which also writes the L2 cache back, took 45 us more with 2048 workgroups.  Atomics on one address are served about 10 ns apart,
// hence groups: 102 MB took 28 us with 1024 arrivals at one counter, 20.5 with 16 counters and another for them.  (512 workgroups of 512
// lanes: 19.8 then, of 256 lanes with twice the loads 21.2; 256 of 1024: 21.4.)
// Lists of more tensors than a table holds take several launches, whose workgroups add to the slots of the one before (the first
// `valid` of them); only the last joins.
template <int ORDER, int CAP>
__global__ __launch_bounds__(kNormThreads) void grad_norm_kernel(const Table<NormSeg, CAP> a, double* result, int valid, int last, int add) {
  __shared__ double lds[kNormThreads / kWave];
  Sum<ORDER> s;
  const int tiles = a.tile_start[a.nseg], step = gridDim.x;
  const int keep = tiles - int(kKeepBytes / kNormTileBytes);
  for (int tile = blockIdx.x; tile < tiles;) {
    const int k = find_segment<CAP>(a.tile_start, a.nseg, tile);
    const uint64_t nt = a.seg[k].nt;
    const int from = a.tile_start[k], to = a.tile_start[k + 1];
    switch (seg_type(nt)) {
      case HPX_F32: norm_tiles_of<ORDER, HPX_F32>(s, a.seg[k].g, seg_size(nt), tile - from, to - from, step, int64_t(keep) - from); break;
      case HPX_BF16: norm_tiles_of<ORDER, HPX_BF16>(s, a.seg[k].g, seg_size(nt), tile - from, to - from, step, int64_t(keep) - from); break;
      default: norm_tiles_of<ORDER, HPX_F16>(s, a.seg[k].g, seg_size(nt), tile - from, to - from, step, int64_t(keep) - from); break;
    }
    tile += (to - tile + step - 1) / step * step;
  }
  double v = block_join<ORDER, kNormThreads / kWave>(s.value(), lds);
  if (threadIdx.x >= kWave) return;  // the first wave does the rest
  if (last && gridDim.x == 1 && valid == 0) {
    if (threadIdx.x == 0) norm_result<ORDER>(result, v, add);
    return;
  }
  double* slots = result + kSlots;
  int am_last = 0;
  if (threadIdx.x == 0) {
    if (int(blockIdx.x) < valid) v = Sum<ORDER>::join(slots[blockIdx.x], v);
    __hip_atomic_store(&slots[blockIdx.x], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (last) {
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const uint32_t group = blockIdx.x % kGroups, groups = gridDim.x < kGroups ? gridDim.x : kGroups;
      const uint32_t members = (gridDim.x - group + kGroups - 1) / kGroups;
      uint32_t* here = reinterpret_cast<uint32_t*>(result + kGroupArrivals + group * kLineDoubles);
      uint32_t* all = reinterpret_cast<uint32_t*>(result + kArrivals);
      if (members == 1 || __hip_atomic_fetch_add(here, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == members - 1) {
        if (members > 1) __hip_atomic_store(here, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        am_last = __hip_atomic_fetch_add(all, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
        if (am_last) __hip_atomic_store(all, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  if (!__builtin_amdgcn_readfirstlane(am_last)) return;
  v = slots_join<ORDER>(slots, int(gridDim.x) > valid ? int(gridDim.x) : valid);
  if (threadIdx.x == 0) norm_result<ORDER>(result, v, add);
}

// ---- the coefficient ---------------------------------------------------------
struct Clip {
  const double* result;  // null: the coefficient is `scale`
  double max_norm;
  double scale;
  int32_t order;
  int32_t tell;  // the first workgroup writes norm and coefficient into the block
};

// The factor for the gradients, from the sum that a norm call, and perhaps an all-reduce behind it, has left.  A norm that
// is not finite gives 0, and a factor of 0 means that nothing of the gradient is taken, whatever it holds.
__device__ __forceinline__ float clip_coefficient(const Clip& a, double s, double* norm) {
  const double n = fabs(a.scale) * (a.order == 2 ? sqrt(s) : s);
  *norm = n;
  if (!(n <= DBL_MAX)) return 0.f;
  const double c = a.max_norm / (n + 1e-6);
  return float(a.scale * (c < 1.0 ? c : 1.0));
}
__device__ __forceinline__ float clip_coefficient(const Clip& a, double* norm) {
  if (!a.result) return float(a.scale);
  return clip_coefficient(a, a.result[0], norm);
}
__device__ __forceinline__ float4 times(float c, float4 g) {
  if (c == 0.f) return make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(c * g.x, c * g.y, c * g.z, c * g.w);
}

// ---- tiles of the writers ----------------------------------------------------
// ITERS x 1024 elements, on boundaries of as many elements of the array that is written: a lane's four elements are aligned there.
template <int ITERS>
__host__ __device__ inline int64_t tile_lead(const void* p, int item) {  // elements between the boundary below and p
  return int64_t((reinterpret_cast<uintptr_t>(p) / item) & (kThreads * 4 * ITERS - 1));
}
template <int ITERS>
inline int64_t write_tiles(const void* p, int64_t n, int item) { return (tile_lead<ITERS>(p, item) + n + kThreads * 4 * ITERS - 1) / (kThreads * 4 * ITERS); }

// The lane's part of a tile: groups of four elements k * 1024 behind e0, those of them that has(k), and at the tensor's ends, where
// less than a group is left before the first or behind the last, an element of its own (one >= 0).
template <int ITERS>
struct Part {
  int64_t e0, one;
  int64_t n;
  bool whole;
  __device__ Part(const void* p, int item, int64_t size, int64_t tile) : n(size) {
    constexpr int64_t kTile = kThreads * 4 * ITERS;
    const int64_t lead = tile_lead<ITERS>(p, item), first = tile * kTile - lead;
    e0 = first + threadIdx.x * 4;
    whole = first >= 0 && first + kTile <= n;
    one = -1;
    if (!whole) {
      const int64_t to_group = (4 - (lead & 3)) & 3, head = to_group < n ? to_group : n, tail = (n - head) & 3;
      if (first <= 0 && threadIdx.x < head) one = threadIdx.x;
      if (threadIdx.x >= kWave && threadIdx.x < kWave + tail && n - tail >= first && n - tail < first + kTile) one = n - tail + (threadIdx.x - kWave);
    }
  }
  __device__ int64_t at(int k) const { return e0 + k * kThreads * 4; }
  __device__ bool has(int k) const { return whole || (at(k) >= 0 && at(k) + 4 <= n); }
};

// The gradient is requested first; coefficient() is called by every lane of the workgroup.
constexpr int kClipIters = 2;
template <int TYPE, int OUT, bool STREAM, typename Coefficient>
__device__ __forceinline__ void clip_tile(const ClipSeg& sg, int64_t n, int64_t tile, Coefficient coefficient) {
  const Part<kClipIters> part(sg.out, sizeof(typename Elem<OUT>::raw), n, tile);
  raw4<TYPE> g[kClipIters];
  if (part.whole) {
#pragma unroll
    for (int k = 0; k < kClipIters; k++) g[k] = load4<TYPE, STREAM>(sg.g, part.at(k));
    const float c = coefficient();
#pragma unroll
    for (int k = 0; k < kClipIters; k++) store4_stream<OUT>(sg.out, part.at(k), times(c, value4<TYPE>(g[k])));
    return;
  }
  float one = 0.f;
  if (part.one >= 0) one = load1<TYPE>(sg.g, part.one);
#pragma unroll
  for (int k = 0; k < kClipIters; k++)
    if (part.has(k)) g[k] = load4<TYPE, STREAM>(sg.g, part.at(k));
  const float c = coefficient();
#pragma unroll
  for (int k = 0; k < kClipIters; k++)
    if (part.has(k)) store4_stream<OUT>(sg.out, part.at(k), times(c, value4<TYPE>(g[k])));
  if (part.one >= 0) store1<OUT>(sg.out, part.one, c == 0.f ? 0.f : c * one);
}

// Second pass of a clipping call.  With `slots` the pass before has left its partial sums and nobody has joined them: every
// workgroup does that for itself while its gradients are on the way, which saves the hand-over at the end of that pass and costs 4 KiB
// of loads in each.  With / without, norm and clipping: 3 M fp16 elements (1500 tiles) 9.7 / 10.9 us, 10 M fp32 (4900) 22.0 / 23.5, 22 M
// (10 700) 41.7 / 43.1, 100 M (48 800) 178.6 / 180.1, bf16 116.7 / 118.4; 134 M (65 400) 239.6 / 242.5, bf16 160.1 / 160.7; 160 M (78 100)
// 286.8 / 287.3, bf16 192.5 / 192.3; 200 M (97 700) 360.0 / 359.5, bf16 243.8 / 241.9; 302 M (147 500) 550.5 / 545.7, bf16 378.6 / 370.0.  (In place the
// few workgroups join at every size: 134 M 258.9 / 259.3, 302 M 602.2 / 605.2, bf16 297.4 / 298.7, a gain that a rule of its own is not worth.)
// Bound by what Infinity Cache and memory deliver together: 25.6 M fp32 elements 28.8 us behind their norm (7.1 TB/s read and written),
// 35.0 where they come from memory (5.8); 110 M of a mixed list 92 (7.2 TB/s) and 109.7 (6.0).
constexpr int64_t kJoinTiles = 65536;
//
// In place there may be nothing to do, so the coefficient comes first and the tiles are shared by few workgroups: 110 M elements of a mixed
// list that is short enough already took 77 us with a workgroup for each tile, 38 of them to start workgroups that end at once, and take
// 41; one that is not, 117 and 107.  (1024: 40.5 and 116; 4096: 42 and 108.  Written elsewhere, 131 with a workgroup for each tile, 135 to
// 137 so.)
constexpr int kInPlaceGrid = 2048;
template <int ORDER, bool STREAM, int CAP>
__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const Table<ClipSeg, CAP> a, const Clip clip, double* result, int slots, int in_place) {
  static_assert(kThreads / kWave == kQuarters, "a quarter of the slots to a wave");
  __shared__ double lds[kQuarters][kWave];
  auto coefficient = [&]() -> float {
    const double s = slots ? slots_join<ORDER>(result + kSlots, slots, lds) : result[0];
    double norm = 0.0;
    const float c = clip_coefficient(clip, s, &norm);
    if (clip.tell && blockIdx.x == 0 && threadIdx.x == 0) {
      if (slots) result[0] = s;
      result[1] = norm;
      result[2] = double(c);
    }
    return c;
  };
  if (in_place) {
    const float c = coefficient();
    if (c == 1.f) return;
    auto known = [c]() { return c; };
    for (int tile = blockIdx.x; tile < a.tile_start[a.nseg]; tile += gridDim.x) {
      const int k = find_segment<CAP>(a.tile_start, a.nseg, tile);
      const ClipSeg sg = a.seg[k];
      const int64_t n = seg_size(sg.nt), t = tile - a.tile_start[k];
      switch (seg_type(sg.nt)) {
        case HPX_F32: clip_tile<HPX_F32, HPX_F32, STREAM>(sg, n, t, known); break;
        case HPX_BF16: clip_tile<HPX_BF16, HPX_BF16, STREAM>(sg, n, t, known); break;
        default: clip_tile<HPX_F16, HPX_F16, STREAM>(sg, n, t, known); break;
      }
    }
    return;
  }
  if (a.nseg == 0) {  // norm and coefficient are told all the same
    coefficient();
    return;
  }
  const int tile = blockIdx.x, k = find_segment<CAP>(a.tile_start, a.nseg, tile);
  const ClipSeg sg = a.seg[k];
  const int64_t n = seg_size(sg.nt), t = tile - a.tile_start[k];
  switch (seg_type(sg.nt)) {
    case HPX_F32: clip_tile<HPX_F32, HPX_F32, STREAM>(sg, n, t, coefficient); break;
    case HPX_BF16: clip_tile<HPX_BF16, HPX_F32, STREAM>(sg, n, t, coefficient); break;
    default: clip_tile<HPX_F16, HPX_F32, STREAM>(sg, n, t, coefficient); break;
  }
}

// A short list in one launch of one workgroup, which keeps it in registers between the norm and the product: a wave takes 1024
// elements of one tensor at a time, three times at most.  One CU moves some 100 GB/s, so what the second launch costs is the limit:
// 16 thousand elements 4.7 us against 8.1 in two launches, 33 thousand 6.1 against 8.2, 47 thousand 7.1 against 8.2 (and 60 thousand, in
// four rounds, took as long as in two launches).  The order of additions is its own, not that of grad_norm_kernel, whose lanes take
// 16 bytes at a time 8 KiB apart: to follow it, a wave would hold 256 of a short tensor's elements where it holds 1024.
constexpr int kShortThreads = 1024;
constexpr int kShortTile = kWave * 16;
constexpr int kShortRounds = 3;
constexpr int kShortTiles = kShortRounds * kShortThreads / kWave;  // 48, so at most as many tensors
static_assert(kShortTiles <= kWave, "the table is read by one wave");

struct ShortPart {  // the lane's elements of a tile: four groups of four, and one of those behind the last whole group
  float4 v[4];
  float one;
};
template <int TYPE>
__device__ __forceinline__ void short_load(ShortPart& p, const void* g, int64_t n, int64_t first) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t rest = n & 3, e0 = first + lane * 4;
  raw4<TYPE> r[4];
  p.one = n - rest < first + kShortTile && lane < rest ? load1<TYPE>(g, n - rest + lane) : 0.f;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int64_t e = e0 + k * kWave * 4;
    if (e + 4 <= n) r[k] = load4<TYPE, false>(g, e);
  }
#pragma unroll
  for (int k = 0; k < 4; k++) p.v[k] = e0 + k * kWave * 4 + 4 <= n ? value4<TYPE>(r[k]) : make_float4(0.f, 0.f, 0.f, 0.f);
}
template <int OUT>
__device__ __forceinline__ void short_store(const ShortPart& p, void* out, int64_t n, int64_t first, float c) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t rest = n & 3, e0 = first + lane * 4;
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (e0 + k * kWave * 4 + 4 <= n) store4_stream<OUT>(out, e0 + k * kWave * 4, times(c, p.v[k]));
  if (n - rest < first + kShortTile && lane < rest) store1<OUT>(out, n - rest + lane, c == 0.f ? 0.f : c * p.one);
}

template <int ORDER>
__global__ __launch_bounds__(kShortThreads) void grad_clip_short_kernel(const Table<ClipSeg, kShortTiles> a, const Clip clip, double* result, int in_place) {
  __shared__ double lds[kShortThreads / kWave];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), tiles = a.tile_start[a.nseg];
  ShortPart part[kShortRounds];
  int seg[kShortRounds];
  Sum<ORDER> s;
#pragma unroll
  for (int r = 0; r < kShortRounds; r++) {
    const int tile = r * (kShortThreads / kWave) + wave;
    if (tile < tiles) {
      const int k = __builtin_amdgcn_readfirstlane(find_segment<kShortTiles>(a.tile_start, a.nseg, tile));
      const uint64_t nt = a.seg[k].nt;
      const int64_t n = seg_size(nt), first = int64_t(tile - a.tile_start[k]) * kShortTile;
      seg[r] = k;
      switch (seg_type(nt)) {
        case HPX_F32: short_load<HPX_F32>(part[r], a.seg[k].g, n, first); break;
        case HPX_BF16: short_load<HPX_BF16>(part[r], a.seg[k].g, n, first); break;
        default: short_load<HPX_F16>(part[r], a.seg[k].g, n, first); break;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kShortRounds; r++)
    if (r * (kShortThreads / kWave) + wave < tiles) {
#pragma unroll
      for (int k = 0; k < 4; k++) { s.add(part[r].v[k].x); s.add(part[r].v[k].y); s.add(part[r].v[k].z); s.add(part[r].v[k].w); }
      s.add(part[r].one);
    }
  const double sum = block_join<ORDER, kShortThreads / kWave>(s.value(), lds);
  double norm = 0.0;
  const float c = clip_coefficient(clip, sum, &norm);
  if (threadIdx.x == 0) {
    result[0] = sum;
    result[1] = norm;
    result[2] = double(c);
  }
  if (in_place && c == 1.f) return;
#pragma unroll
  for (int r = 0; r < kShortRounds; r++) {
    const int tile = r * (kShortThreads / kWave) + wave;
    if (tile < tiles) {
      const int k = seg[r];
      const ClipSeg sg = a.seg[k];
      const int64_t n = seg_size(sg.nt), first = int64_t(tile - a.tile_start[k]) * kShortTile;
      switch (in_place ? seg_type(sg.nt) : HPX_F32) {
        case HPX_F32: short_store<HPX_F32>(part[r], sg.out, n, first, c); break;
        case HPX_BF16: short_store<HPX_BF16>(part[r], sg.out, n, first, c); break;
        default: short_store<HPX_F16>(part[r], sg.out, n, first, c); break;
      }
    }
  }
}

// ---- momentum ----------------------------------------------------------------
// u' = m u + c g with the product c g rounded once and one rounding for the rest (fma), d = m u' + c g likewise.
__device__ __forceinline__ float4 axpy(float m, float4 x, float4 y) { return make_float4(fmaf(m, x.x, y.x), fmaf(m, x.y, y.y), fmaf(m, x.z, y.z), fmaf(m, x.w, y.w)); }

// Tiles of 4096 elements; with a direction to write as well, tiles of 2048.  Bound by memory: 138 M fp32 elements 258 us (6.4 TB/s; 275
// with tiles of 2048), 100 M 183 (196); with a direction, 100 M bf16 elements 225 us (6.2 TB/s; 243 with tiles of 4096), 25.6 M in
// 161 tensors 58.7 (61.7).  Streaming launches ask for LDS they do not touch, so that a CU holds three workgroups (see
// kWriteStreamPadLds3): 302 M bf16 elements 463 us, 477 with four, 482 with eight; 130 M in 100 tensors 202, 206, 207; one fp32 tensor of
// 25 M 49.0, 47.7, 47.6.
template <bool DIRECTION>
constexpr int kMomentumIters = DIRECTION ? 2 : 4;
template <int TYPE, bool DIRECTION, bool STREAM, typename Coefficient>
__device__ __forceinline__ void momentum_tile(const MomentumSeg& sg, int64_t n, int64_t tile, float m, Coefficient coefficient) {
  constexpr int kIters = kMomentumIters<DIRECTION>;
  const Part<kIters> part(sg.u, 4, n, tile);
  raw4<TYPE> g[kIters];
  raw4<HPX_F32> u[kIters];
  if (part.whole) {
#pragma unroll
    for (int k = 0; k < kIters; k++) {
      g[k] = load4<TYPE, STREAM>(sg.g, part.at(k));
      u[k] = load4<HPX_F32, STREAM>(sg.u, part.at(k));
    }
    const float c = coefficient();
#pragma unroll
    for (int k = 0; k < kIters; k++) {
      const float4 cg = times(c, value4<TYPE>(g[k])), v = axpy(m, value4<HPX_F32>(u[k]), cg);
      store4_stream<HPX_F32>(sg.u, part.at(k), v);
      if (DIRECTION) store4_stream<HPX_F32>(sg.d, part.at(k), axpy(m, v, cg));
    }
    return;
  }
  float g1 = 0.f, u1 = 0.f;
  if (part.one >= 0) {
    g1 = load1<TYPE>(sg.g, part.one);
    u1 = sg.u[part.one];
  }
#pragma unroll
  for (int k = 0; k < kIters; k++)
    if (part.has(k)) {
      g[k] = load4<TYPE, STREAM>(sg.g, part.at(k));
      u[k] = load4<HPX_F32, STREAM>(sg.u, part.at(k));
    }
  const float c = coefficient();
#pragma unroll
  for (int k = 0; k < kIters; k++)
    if (part.has(k)) {
      const float4 cg = times(c, value4<TYPE>(g[k])), v = axpy(m, value4<HPX_F32>(u[k]), cg);
      store4_stream<HPX_F32>(sg.u, part.at(k), v);
      if (DIRECTION) store4_stream<HPX_F32>(sg.d, part.at(k), axpy(m, v, cg));
    }
  if (part.one >= 0) {
    const float cg = c == 0.f ? 0.f : c * g1, v = fmaf(m, u1, cg);
    sg.u[part.one] = v;
    if (DIRECTION) sg.d[part.one] = fmaf(m, v, cg);
  }
}

template <bool DIRECTION, bool STREAM, int CAP>
__global__ __launch_bounds__(kThreads) void gd_momentum_kernel(const Table<MomentumSeg, CAP> a, const Clip clip, double* result, float m) {
  const int tile = blockIdx.x;
  auto coefficient = [&]() -> float {
    double norm = 0.0;
    const float c = clip_coefficient(clip, &norm);
    if (clip.tell && tile == 0 && threadIdx.x == 0) {
      result[1] = norm;
      result[2] = double(c);
    }
    return c;
  };
  if (a.nseg == 0) {
    coefficient();
    return;
  }
  // Requested behind the loads it costs a short list nothing (4 M elements 8.8 us against 9.4, 12 M 23.2 against 24.1); in a streaming list
  // other workgroups fill the time, and first is better (25.6 M bf16 with a direction 58.2 against 59.1, 138 M 259.4 against 261.4).
  const float first = STREAM ? coefficient() : 0.f;
  auto factor = [&]() -> float { return STREAM ? first : coefficient(); };
  const int k = find_segment<CAP>(a.tile_start, a.nseg, tile);
  const MomentumSeg sg = a.seg[k];
  const int64_t n = seg_size(sg.nt), t = tile - a.tile_start[k];
  switch (seg_type(sg.nt)) {
    case HPX_F32: momentum_tile<HPX_F32, DIRECTION, STREAM>(sg, n, t, m, factor); break;
    case HPX_BF16: momentum_tile<HPX_BF16, DIRECTION, STREAM>(sg, n, t, m, factor); break;
    default: momentum_tile<HPX_F16, DIRECTION, STREAM>(sg, n, t, m, factor); break;
  }
}

// ---- mask --------------------------------------------------------------------
// A lane takes an entry of the message: it requests the header and its index together (both lie within the message's room)
// and stores a zero if the header counts the entry in and the index lies in the tensor.
constexpr int kMaskTile = kThreads;
__host__ __device__ inline int mask_room(int32_t in_size) { return in_size < 4 ? 0 : (in_size - 4) / 8; }

template <int CAP>
__global__ __launch_bounds__(kThreads) void gd_mask_kernel(const Table<MaskSeg, CAP> a, int32_t* counts) {
  const int tile = blockIdx.x;
  const int s = find_segment<CAP>(a.tile_start, a.nseg, tile);
  const MaskSeg sg = a.seg[s];
  const int32_t* words = reinterpret_cast<const int32_t*>(sg.in);
  const int64_t i = int64_t(tile - a.tile_start[s]) * kMaskTile + threadIdx.x;
  const int room = mask_room(sg.in_size);
  const int32_t bytes = sg.in_size >= 4 ? words[0] : 0;
  const int32_t at = i < room ? words[1 + i] : -1;
  const bool good = bytes >= 4 && bytes <= sg.in_size && (bytes & 7) == 4;
  const int k = good ? (bytes - 4) / 8 : 0;
  if (i < k && uint32_t(at) < uint32_t(sg.n)) sg.u[at] = 0.f;
  if (counts && i == 0) counts[s] = good ? k : -1;
}

// ---- host --------------------------------------------------------------------
int item_size(int type) { return type == HPX_F32 ? 4 : 2; }
bool aligned(const void* p, int item) { return reinterpret_cast<uintptr_t>(p) % item == 0; }

int64_t list_bytes(int count, const int64_t* sizes, const int32_t* types) {
  int64_t b = 0;
  for (int i = 0; i < count; i++) b += sizes[i] * item_size(types ? types[i] : HPX_F32);
  return b;
}
// f with two truth values as types.
template <typename F>
int with_constants(bool a, bool b, F f) {
  if (a) return b ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
  return b ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

struct Span {
  uintptr_t b, e;
};
Span span(const void* p, int64_t bytes) { return {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + uintptr_t(bytes)}; }
// The memory of a list of tensors.
class Spans {
 public:
  explicit Spans(size_t room) { v_.reserve(room); }
  void add(const Span& x) { v_.push_back(x); }
  // Whether any of them overlap; sorts them and joins those that do.  Before meets().
  bool close() {
    bool sorted = true, found = false;
    for (size_t i = 1; i < v_.size() && sorted; i++) sorted = v_[i - 1].b <= v_[i].b;
    if (!sorted) std::sort(v_.begin(), v_.end(), [](const Span& x, const Span& y) { return x.b < y.b; });
    for (size_t i = 1; i < v_.size() && !found; i++) found = v_[i].b < v_[i - 1].e;
    if (!found) return false;
    size_t n = 0;
    for (const Span& x : v_) {
      if (n > 0 && x.b < v_[n - 1].e) v_[n - 1].e = std::max(v_[n - 1].e, x.e);
      else v_[n++] = x;
    }
    v_.resize(n);
    return true;
  }
  // Whether x overlaps any of them.  Lists mostly ascend side by side, so the first span that ends behind x's begin is looked
  // for where the last call found it and one further, which costs a list of 161 tensors 1 us less than searching each time.
  bool meets(const Span& x) {
    if (!first_behind(at_, x.b)) {
      if (at_ < v_.size() && first_behind(at_ + 1, x.b)) at_++;
      else at_ = size_t(std::upper_bound(v_.begin(), v_.end(), x.b, [](uintptr_t b, const Span& s) { return b < s.e; }) - v_.begin());
    }
    return at_ < v_.size() && v_[at_].b < x.e;
  }

 private:
  bool first_behind(size_t k, uintptr_t b) const { return (k == 0 || v_[k - 1].e <= b) && (k == v_.size() || b < v_[k].e); }
  std::vector<Span> v_;
  size_t at_ = 0;
};

int check_list(const char* who, int count, const void* const* grads, const int64_t* sizes, const int32_t* types) {
  for (int i = 0; i < count; i++) {
    HPX_ARG(sizes[i] >= 0 && sizes[i] < kMaxSize, "%s: tensor %d has size %lld", who, i, static_cast<long long>(sizes[i]));
    const int type = types ? types[i] : HPX_F32;
    HPX_ARG(type == HPX_F32 || type == HPX_BF16 || type == HPX_F16, "%s: tensor %d has type %d", who, i, type);
    HPX_ARG(sizes[i] == 0 || grads[i], "%s: tensor %d has a null pointer", who, i);
    HPX_ARG(sizes[i] == 0 || aligned(grads[i], item_size(type)), "%s: tensor %d does not start at a multiple of its element size", who, i);
  }
  return HPX_OK;
}
int check_result(const char* who, const double* result) {
  HPX_ARG(result && aligned(result, 8), "%s: the result block is null or does not start at a multiple of 8 bytes", who);
  return HPX_OK;
}
Span block_span(const double* result) { return span(result, HPX_GRAD_RESULT * int64_t(sizeof(double))); }
// A tensor that shares memory with the block would be read while sums are stored there, or overwrite its counters of arrivals, which
// later calls rely on.
int check_apart(const char* who, const char* what, int count, const void* const* p, const int64_t* sizes, const int32_t* types, const double* result) {
  const Span block = block_span(result);
  for (int i = 0; i < count; i++) {
    if (sizes[i] == 0) continue;
    const Span s = span(p[i], sizes[i] * item_size(types ? types[i] : HPX_F32));
    HPX_ARG(s.e <= block.b || block.e <= s.b, "%s: %s %d overlaps the result block", who, what, i);
  }
  return HPX_OK;
}
int check_clip(const char* who, int order, double max_norm, double scale) {
  HPX_ARG(order == 2 || order == HPX_NORM_MAX, "%s: order %d is neither 2 nor HPX_NORM_MAX", who, order);
  HPX_ARG(max_norm >= 0.0, "%s: max_norm %g is negative or not a number", who, max_norm);
  HPX_ARG(std::isfinite(scale) && std::fabs(scale) <= FLT_MAX, "%s: scale %g is not finite", who, scale);
  return HPX_OK;
}

// `elements` of `item` bytes behind p.
const void* behind(const void* p, int64_t elements, int item) { return static_cast<const uint8_t*>(p) + elements * item; }
void* behind(void* p, int64_t elements, int item) { return static_cast<uint8_t*>(p) + elements * item; }

// slots: not null where the caller joins the partial sums itself; gets their number.
template <int ORDER, int CAP>
int launch_norm(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, int add, double* result, int* slots, hipStream_t st) {
  int valid = 0;
  const int rc = for_tables<NormSeg, CAP>(
      count, INT32_MAX - kMaxGrid,  // a fixed grid walks over the tiles: only their number has to stay in 32 bits
      [&](int i, int64_t*, NormSeg& sg) -> int64_t {
        if (sizes[i] == 0) return 0;
        const int type = types ? types[i] : HPX_F32;
        sg = NormSeg{grads[i], uint64_t(sizes[i]) | uint64_t(type) << kTypeShift};
        return norm_tiles(sizes[i], type);
      },
      [&](const Table<NormSeg, CAP>& a, int tiles, bool last) -> int {
        const int grid = std::max(1, std::min(tiles, kMaxGrid));
        HPX_LAUNCH("grad_norm_kernel", (grad_norm_kernel<ORDER, CAP>), dim3(grid), dim3(kNormThreads), st, a, result, valid, int(last && !slots), add);
        HPX_HIP(hipGetLastError());
        valid = std::max(valid, grid);
        return HPX_OK;
      });
  if (slots) *slots = valid;
  return rc;
}
template <int ORDER>
int norm(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, int add, double* result, int* slots, hipStream_t st) {
  return count <= kCapSmall ? launch_norm<ORDER, kCapSmall>(count, grads, sizes, types, add, result, slots, st)
                            : launch_norm<ORDER, NormSeg::kCapLarge>(count, grads, sizes, types, add, result, slots, st);
}

ClipSeg clip_seg(const void* g, void* out, int64_t size, int type) { return ClipSeg{g, out, uint64_t(size) | uint64_t(type) << kTypeShift}; }

// Outputs of a clipping call: null where it works in place.
struct Outs {
  float* const* p;
  void* at(const void* const* grads, int i) const { return p ? static_cast<void*>(p[i]) : const_cast<void*>(grads[i]); }
  int item(int type) const { return p ? 4 : item_size(type); }
};

static_assert(kPartElements % (kThreads * 4 * kClipIters) == 0 && kPartElements % (kThreads * 4 * kMomentumIters<false>) == 0 &&
                  kPartElements / (kThreads * 4 * std::min(kClipIters, kMomentumIters<true>)) + 1 <= most_tiles(kThreads),
              "a part begins on the tensor's place in a tile, and goes into a table");
template <int ORDER, bool STREAM, int CAP>
int launch_clip(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, Outs outs, Clip clip, double* result, int slots, hipStream_t st) {
  return for_tables<ClipSeg, CAP>(
      count, most_tiles(kThreads),
      [&](int i, int64_t* at, ClipSeg& sg) -> int64_t {
        if (sizes[i] == 0) return 0;
        const int type = types ? types[i] : HPX_F32;
        const int64_t from = *at, n = next_part(sizes[i], at);
        sg = clip_seg(behind(grads[i], from, item_size(type)), behind(outs.at(grads, i), from, outs.item(type)), n, type);
        return write_tiles<kClipIters>(sg.out, n, outs.item(type));
      },
      [&](const Table<ClipSeg, CAP>& a, int tiles, bool) -> int {
        const int grid = std::max(1, outs.p ? tiles : std::min(tiles, kInPlaceGrid));
        HPX_LAUNCH("grad_clip_kernel", (grad_clip_kernel<ORDER, STREAM, CAP>), dim3(grid), dim3(kThreads), st, a, clip, result, slots, int(!outs.p));
        HPX_HIP(hipGetLastError());
        clip.tell = 0;
        return HPX_OK;
      });
}

// Lists of up to kShortTiles tiles of 1024 elements: one launch of one workgroup.
template <int ORDER>
int launch_clip_short(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, Outs outs, const Clip& clip, double* result, hipStream_t st) {
  return for_tables<ClipSeg, kShortTiles>(
      count, kShortTiles,
      [&](int i, int64_t*, ClipSeg& sg) -> int64_t {
        sg = clip_seg(grads[i], outs.at(grads, i), sizes[i], types ? types[i] : HPX_F32);
        return (sizes[i] + kShortTile - 1) / kShortTile;
      },
      [&](const Table<ClipSeg, kShortTiles>& a, int, bool) -> int {
        HPX_LAUNCH("grad_clip_short_kernel", (grad_clip_short_kernel<ORDER>), dim3(1), dim3(kShortThreads), st, a, clip, result, int(!outs.p));
        HPX_HIP(hipGetLastError());
        return HPX_OK;
      });
}

template <int ORDER>
int clip(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, Outs outs, bool measured, const Clip& clip, double* result, hipStream_t st) {
  int slots = 0;
  if (!measured) {
    int64_t short_tiles = 0, tiles = 0;
    for (int i = 0; i < count; i++) {
      short_tiles += (sizes[i] + kShortTile - 1) / kShortTile;
      tiles += sizes[i] / (kThreads * 4 * kClipIters) + 1;
    }
    if (short_tiles <= kShortTiles) return launch_clip_short<ORDER>(count, grads, sizes, types, outs, clip, result, st);
    if (const int rc = norm<ORDER>(count, grads, sizes, types, 0, result, tiles <= kJoinTiles ? &slots : nullptr, st)) return rc;
  }
  return with_constants(list_bytes(count, sizes, types) > kPlainBytes, count <= kCapSmall, [&](auto stream, auto small) {
    constexpr int CAP = decltype(small)::value ? kCapSmall : ClipSeg::kCapLarge;
    return launch_clip<ORDER, decltype(stream)::value, CAP>(count, grads, sizes, types, outs, clip, result, slots, st);
  });
}

template <bool DIRECTION, bool STREAM, int CAP>
int launch_momentum(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, float* const* us, float* const* outs, float m, Clip clip, double* result,
                    hipStream_t st) {
  return for_tables<MomentumSeg, CAP>(
      count, most_tiles(kThreads),
      [&](int i, int64_t* at, MomentumSeg& sg) -> int64_t {
        if (sizes[i] == 0) return 0;
        const int type = types ? types[i] : HPX_F32;
        const int64_t from = *at, n = next_part(sizes[i], at);
        sg = MomentumSeg{behind(grads[i], from, item_size(type)), us[i] + from, outs ? outs[i] + from : nullptr, uint64_t(n) | uint64_t(type) << kTypeShift};
        return write_tiles<kMomentumIters<DIRECTION>>(sg.u, n, 4);
      },
      [&](const Table<MomentumSeg, CAP>& a, int tiles, bool) -> int {
        HPX_LAUNCH_LDS("gd_momentum_kernel", hpx::g_prof_on, (gd_momentum_kernel<DIRECTION, STREAM, CAP>), dim3(std::max(1, tiles)), dim3(kThreads), STREAM ? kWriteStreamPadLds3 : 0, st, a, clip, result, m);
        HPX_HIP(hipGetLastError());
        clip.tell = 0;
        return HPX_OK;
      });
}

template <int CAP>
int launch_mask(int count, const uint8_t* const* ins, const int32_t* in_sizes, float* const* us, const int32_t* sizes, int32_t* counts, hipStream_t st) {
  int first = 0;
  return for_tables<MaskSeg, CAP>(
      count, most_tiles(kThreads),
      [&](int i, int64_t*, MaskSeg& sg) -> int64_t {
        sg = MaskSeg{ins[i], us[i], in_sizes[i], sizes[i]};
        return std::max(1, (mask_room(in_sizes[i]) + kMaskTile - 1) / kMaskTile);
      },
      [&](const Table<MaskSeg, CAP>& a, int tiles, bool) -> int {
        if (tiles == 0) return HPX_OK;
        HPX_LAUNCH("gd_mask_kernel", (gd_mask_kernel<CAP>), dim3(tiles), dim3(kThreads), st, a, counts ? counts + first : nullptr);
        HPX_HIP(hipGetLastError());
        first += a.nseg;
        return HPX_OK;
      });
}

// Refuses lists in which an element is written twice, or written through one tensor and read through another, and tensors that
// overlap the result block (null: there is none).  `a`, which `a_name` names, and `outs` (null: there are none) are written; the
// tensors of `in_place` (one of the two lists) may be the gradients themselves.
int check_writes(const char* who, int count, const void* const* grads, const int64_t* sizes, const int32_t* types, const void* const* a, const char* a_name,
                 const void* const* outs, const void* const* in_place, const double* result) {
  Spans w(size_t(count) * (outs ? 2 : 1));
  for (int i = 0; i < count; i++) {
    if (sizes[i] == 0) continue;
    w.add(span(a[i], sizes[i] * (a[i] == grads[i] ? item_size(types ? types[i] : HPX_F32) : 4)));
  }
  for (int i = 0; outs && i < count; i++) {
    if (sizes[i] == 0) continue;
    w.add(span(outs[i], sizes[i] * 4));
  }
  HPX_ARG(!w.close(), "%s: two of the tensors that are written overlap", who);
  for (int i = 0; i < count; i++) {
    if (sizes[i] == 0) continue;
    if (in_place && in_place[i] == grads[i]) continue;
    HPX_ARG(!w.meets(span(grads[i], sizes[i] * item_size(types ? types[i] : HPX_F32))), "%s: gradient %d overlaps a tensor that is written", who, i);
  }
  if (!result) return HPX_OK;
  const bool written = w.meets(block_span(result));
  if (written || a != grads)
    if (const int rc = check_apart(who, "gradient", count, grads, sizes, types, result)) return rc;
  if (!written) return HPX_OK;
  if (const int rc = check_apart(who, a_name, count, a, sizes, nullptr, result)) return rc;
  return outs ? check_apart(who, "output", count, outs, sizes, nullptr, result) : HPX_OK;
}

// A C entry point lets no C++ exception out.
template <typename F>
int guarded(const char* who, F f) {
  hpx::clear_error();
  try {
    return f();
  } catch (...) {
    hpx::set_error("%s: out of host memory", who);
    return HPX_ERR_HIP;
  }
}
}  // namespace

HPX_API int hpx_grad_norm(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, int order, int is_add_to,
                          double* result, hpx_stream_t stream) {
  const char* who = "hpx_grad_norm";
  return guarded(who, [&]() -> int {
    HPX_ARG(count >= 0, "%s: negative count", who);
    HPX_ARG(count == 0 || (grads && sizes), "%s: null argument array", who);
    if (const int rc = check_clip(who, order, 0.0, 1.0)) return rc;
    if (const int rc = check_result(who, result)) return rc;
    if (const int rc = check_list(who, count, grads, sizes, types)) return rc;
    if (const int rc = check_apart(who, "gradient", count, grads, sizes, types, result)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return order == 2 ? norm<2>(count, grads, sizes, types, is_add_to != 0, result, nullptr, st)
                      : norm<HPX_NORM_MAX>(count, grads, sizes, types, is_add_to != 0, result, nullptr, st);
  });
}

HPX_API int hpx_grad_clip(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, float* const* outs, int is_measured,
                          int order, double max_norm, double scale, double* result, hpx_stream_t stream) {
  const char* who = "hpx_grad_clip";
  return guarded(who, [&]() -> int {
    HPX_ARG(count >= 0, "%s: negative count", who);
    HPX_ARG(count == 0 || (grads && sizes), "%s: null argument array", who);
    if (const int rc = check_clip(who, order, max_norm, scale)) return rc;
    if (const int rc = check_result(who, result)) return rc;
    if (const int rc = check_list(who, count, grads, sizes, types)) return rc;
    for (int i = 0; outs && i < count; i++) {
      if (sizes[i] == 0) continue;
      HPX_ARG(outs[i] && aligned(outs[i], 4), "%s: output %d is null or does not start at a multiple of its element size", who, i);
      HPX_ARG(!types || types[i] == HPX_F32 || outs[i] != grads[i], "%s: output %d is fp32 and cannot take the place of a gradient of another type", who, i);
    }
    const void* const* to = outs ? reinterpret_cast<const void* const*>(outs) : grads;
    if (const int rc = check_writes(who, count, grads, sizes, types, to, "output", nullptr, to, result)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Clip how{result, max_norm, scale, order, 1};
    return order == 2 ? clip<2>(count, grads, sizes, types, Outs{outs}, is_measured != 0, how, result, st)
                      : clip<HPX_NORM_MAX>(count, grads, sizes, types, Outs{outs}, is_measured != 0, how, result, st);
  });
}

HPX_API int hpx_gd_momentum(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, float* const* momenta,
                            float* const* outs, float momentum, int order, double max_norm, double scale, double* result, hpx_stream_t stream) {
  const char* who = "hpx_gd_momentum";
  return guarded(who, [&]() -> int {
    HPX_ARG(count >= 0, "%s: negative count", who);
    HPX_ARG(count == 0 || (grads && sizes && momenta), "%s: null argument array", who);
    HPX_ARG(std::isfinite(momentum), "%s: momentum %g is not finite", who, double(momentum));
    if (const int rc = check_clip(who, order, max_norm, scale)) return rc;
    HPX_ARG(aligned(result, 8), "%s: the result block does not start at a multiple of 8 bytes", who);
    if (const int rc = check_list(who, count, grads, sizes, types)) return rc;
    for (int i = 0; i < count; i++) {
      if (sizes[i] == 0) continue;
      HPX_ARG(momenta[i] && aligned(momenta[i], 4), "%s: momentum %d is null or does not start at a multiple of its element size", who, i);
      HPX_ARG(!outs || (outs[i] && aligned(outs[i], 4)), "%s: output %d is null or does not start at a multiple of its element size", who, i);
      HPX_ARG(!outs || !types || types[i] == HPX_F32 || outs[i] != grads[i], "%s: output %d is fp32 and cannot take the place of a gradient of another type", who, i);
    }
    const void* const *us = reinterpret_cast<const void* const*>(momenta), *const *ds = reinterpret_cast<const void* const*>(outs);
    if (const int rc = check_writes(who, count, grads, sizes, types, us, "momentum", ds, ds, result)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Clip clip{result, max_norm, scale, order, result != nullptr};
    int64_t elements = 0;
    for (int i = 0; i < count; i++) elements += sizes[i];
    const bool large = list_bytes(count, sizes, types) + 4 * elements > kPlainBytes;
    return with_constants(large, count <= kCapSmall, [&](auto streaming, auto small) {
      constexpr bool S = decltype(streaming)::value;
      constexpr int CAP = decltype(small)::value ? kCapSmall : MomentumSeg::kCapLarge;
      if (outs) return launch_momentum<true, S, CAP>(count, grads, sizes, types, momenta, outs, momentum, clip, result, st);
      return launch_momentum<false, S, CAP>(count, grads, sizes, types, momenta, outs, momentum, clip, result, st);
    });
  });
}

HPX_API int hpx_gd_mask(int count, const uint8_t* const* ins, const int32_t* in_sizes, float* const* momenta, const int32_t* sizes,
                        int32_t* counts, hpx_stream_t stream) {
  const char* who = "hpx_gd_mask";
  return guarded(who, [&]() -> int {
    HPX_ARG(count >= 0, "%s: negative count", who);
    if (count == 0) return HPX_OK;
    HPX_ARG(ins && in_sizes && momenta && sizes, "%s: null argument array", who);
    HPX_ARG(aligned(counts, 4), "%s: the counts do not start at a multiple of 4 bytes", who);
    const Span nothing{UINTPTR_MAX, 0};
    Span read = nothing, written = nothing;  // from the lowest to the highest address
    auto widen = [](Span& all, const Span& x) { all = Span{std::min(all.b, x.b), std::max(all.e, x.e)}; };
    for (int i = 0; i < count; i++) {
      HPX_ARG(in_sizes[i] >= 0 && sizes[i] >= 0, "%s: message %d has a negative size", who, i);
      HPX_ARG(in_sizes[i] < 4 || (ins[i] && aligned(ins[i], 4)), "%s: message %d is null or does not start at a multiple of 4 bytes", who, i);
      HPX_ARG(sizes[i] == 0 || (momenta[i] && aligned(momenta[i], 4)), "%s: momentum %d is null or does not start at a multiple of 4 bytes", who, i);
      if (in_sizes[i] >= 4) widen(read, span(ins[i], in_sizes[i]));
      if (sizes[i] > 0) widen(written, span(momenta[i], int64_t(sizes[i]) * 4));
    }
    // Zeros are all that is stored to momenta, so several messages may name one; what is read must not be among it, nor the counts.
    // (Messages from one buffer and momenta from another need no look at each.)
    auto cross = [](const Span& x, const Span& y) { return x.b < y.e && y.b < x.e; };
    const Span told = counts ? span(counts, int64_t(count) * 4) : nothing;
    if (cross(read, written) || cross(told, written) || cross(told, read)) {
      Spans w{size_t(count)};
      for (int i = 0; i < count; i++)
        if (sizes[i] > 0) w.add(span(momenta[i], int64_t(sizes[i]) * 4));
      w.close();
      HPX_ARG(!counts || !w.meets(told), "%s: the counts overlap a momentum", who);
      for (int i = 0; i < count; i++) {
        if (in_sizes[i] < 4) continue;
        const Span in = span(ins[i], in_sizes[i]);
        HPX_ARG(!w.meets(in), "%s: message %d overlaps a momentum", who, i);
        HPX_ARG(!counts || !cross(in, told), "%s: the counts overlap message %d", who, i);
      }
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (count <= kCapSmall) return launch_mask<kCapSmall>(count, ins, in_sizes, momenta, sizes, counts, st);
    return launch_mask<MaskSeg::kCapLarge>(count, ins, in_sizes, momenta, sizes, counts, st);
  });
}
