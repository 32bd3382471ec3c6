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

namespace {
using namespace hpx;

constexpr int kThreads = 256;

// ---- the result block --------------------------------------------------------
// doubles: [0] S, [1] norm, [2] coefficient, [3] arrivals (zero between calls), [16 ...] one partial sum per workgroup
constexpr int kArrivals = 3;
constexpr int kSlots = 16;
constexpr int kMaxGrid = HPX_GRAD_RESULT - kSlots;
static_assert(kMaxGrid == 2048, "eight workgroups of 256 lanes on each of 256 CUs");

// ---- tables ------------------------------------------------------------------
// An element count and its type share a word: the count needs 48 bits.
constexpr int kTypeShift = 56;
constexpr int64_t kMaxSize = int64_t(1) << 48;
__host__ __device__ inline int64_t seg_size(uint64_t nt) { return int64_t(nt & ((uint64_t(1) << kTypeShift) - 1)); }
__host__ __device__ inline int seg_type(uint64_t nt) { return int(nt >> kTypeShift); }

struct NormSeg {
  const void* g;
  uint64_t nt;
  static constexpr int kCapLarge = 448;
};
struct ClipSeg {
  const void* g;
  void* out;  // g itself: in place, in g's type; else fp32
  uint64_t nt;
  static constexpr int kCapLarge = 320;
};
struct MomentumSeg {
  const void* g;
  float* u;
  float* d;  // null: no direction
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

template <typename Seg, int CAP>
struct Table {
  int32_t nseg;
  int32_t tile_start[CAP + 1];
  Seg seg[CAP];
};
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
  Raw v[4];
};
template <int TYPE>
__device__ __forceinline__ float4 load4(const void* base, int64_t e) {
  using E = Elem<TYPE>;
  const Raw4<typename E::raw> r = *reinterpret_cast<const Raw4<typename E::raw>*>(static_cast<const typename E::raw*>(base) + e);
  return make_float4(E::to(r.v[0]), E::to(r.v[1]), E::to(r.v[2]), E::to(r.v[3]));
}
template <int TYPE>
__device__ __forceinline__ void store4(void* base, int64_t e, float4 x) {
  using E = Elem<TYPE>;
  Raw4<typename E::raw> r;
  r.v[0] = E::from(x.x); r.v[1] = E::from(x.y); r.v[2] = E::from(x.z); r.v[3] = E::from(x.w);
  *reinterpret_cast<Raw4<typename E::raw>*>(static_cast<typename E::raw*>(base) + e) = r;
}

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

// Tiles of 16 KiB are counted from the tensor's first element, not from a boundary of memory: which elements a partial sum is
// made of, and so every bit of the result, then depends on types, sizes and values alone, and ranks that hold the same gradients
// at other addresses find the same norm.
constexpr uint32_t kNormTileBytes = 16384;
constexpr int kNormIters = kNormTileBytes / (kThreads * 16);
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

template <int ORDER, int TYPE>
__device__ __forceinline__ void norm_tile(Sum<ORDER>& s, const void* p, int64_t n, int64_t tile) {
  using Raw = typename Elem<TYPE>::raw;
  constexpr int kPer = 16 / sizeof(Raw);  // elements of a chunk
  const Raw* g = static_cast<const Raw*>(p);
  const int64_t first = tile * (kNormTileBytes / sizeof(Raw)), e0 = first + threadIdx.x * kPer;
  if (first + int64_t(kNormTileBytes / sizeof(Raw)) <= n) {
    Chunk<Raw> c[kNormIters];
#pragma unroll
    for (int k = 0; k < kNormIters; k++) c[k] = *reinterpret_cast<const Chunk<Raw>*>(g + e0 + k * kThreads * kPer);
#pragma unroll
    for (int k = 0; k < kNormIters; k++) norm_chunk<ORDER, TYPE>(s, c[k]);
    return;
  }
#pragma unroll
  for (int k = 0; k < kNormIters; k++) {
    const int64_t e = e0 + k * kThreads * kPer;
    if (e + kPer <= n) {
      norm_chunk<ORDER, TYPE>(s, *reinterpret_cast<const Chunk<Raw>*>(g + e));
    } else {
      for (int64_t x = e; x < n; x++) s.add(Elem<TYPE>::to(g[x]));
    }
  }
}

// Over the workgroup, the same order of additions whatever the timing; every lane gets the result of thread 0's wave.
template <int ORDER>
__device__ __forceinline__ double block_join(double v, double* lds) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = Sum<ORDER>::join(v, __shfl_xor(v, o, kWave));
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; w++) v = Sum<ORDER>::join(v, lds[w]);
  __syncthreads();
  return v;
}

// A workgroup sums every gridDim.x-th tile and leaves one partial sum; the last one to arrive joins them in their order, so
// the result does not depend on who that is.  Lists of more tensors than a table holds take several launches, whose workgroups
// add to the slots of the one before (the first `valid` of them); only the last joins.
template <int ORDER, int CAP>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const Table<NormSeg, CAP> a, double* result, int valid, int last, int add) {
  __shared__ double lds[kThreads / kWave];
  __shared__ int am_last;
  Sum<ORDER> s;
  const int tiles = a.tile_start[a.nseg];
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int k = find_segment<CAP>(a.tile_start, a.nseg, tile);
    const uint64_t nt = a.seg[k].nt;
    const int64_t t = tile - a.tile_start[k];
    switch (seg_type(nt)) {
      case HPX_F32: norm_tile<ORDER, HPX_F32>(s, a.seg[k].g, seg_size(nt), t); break;
      case HPX_BF16: norm_tile<ORDER, HPX_BF16>(s, a.seg[k].g, seg_size(nt), t); break;
      default: norm_tile<ORDER, HPX_F16>(s, a.seg[k].g, seg_size(nt), t); break;
    }
  }
  double v = block_join<ORDER>(s.value(), lds);
  double* slots = result + kSlots;
  if (threadIdx.x == 0) {
    if (int(blockIdx.x) < valid) v = Sum<ORDER>::join(slots[blockIdx.x], v);
    __hip_atomic_store(&slots[blockIdx.x], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    am_last = 0;
    if (last) {
      uint32_t* arrivals = reinterpret_cast<uint32_t*>(result + kArrivals);
      am_last = __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
      if (am_last) __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  if (!am_last) return;
  const int used = int(gridDim.x) > valid ? int(gridDim.x) : valid;
  v = 0.0;
  for (int i = threadIdx.x; i < used; i += kThreads)
    v = Sum<ORDER>::join(v, __hip_atomic_load(&slots[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  v = block_join<ORDER>(v, lds);
  if (threadIdx.x == 0) {
    if (add) v = Sum<ORDER>::join(result[0], v);
    result[0] = v;
    result[1] = ORDER == 2 ? sqrt(v) : v;
  }
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
__device__ __forceinline__ float clip_coefficient(const Clip& a, double* norm) {
  if (!a.result) return float(a.scale);
  const double s = a.result[0];
  const double n = fabs(a.scale) * (a.order == 2 ? sqrt(s) : s);
  *norm = n;
  if (!(n <= DBL_MAX)) return 0.f;
  const double c = a.max_norm / (n + 1e-6);
  return float(a.scale * (c < 1.0 ? c : 1.0));
}
__device__ __forceinline__ float4 times(float c, float4 g) {
  if (c == 0.f) return make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(c * g.x, c * g.y, c * g.z, c * g.w);
}

// ---- tiles of the writers ----------------------------------------------------
// 4096 elements, on boundaries of 4096 elements of the array that is written: a lane's four elements are aligned there.
constexpr int kIters = 4;
constexpr int kTileElems = kThreads * 4 * kIters;
__host__ __device__ inline int64_t tile_lead(const void* p, int item) {  // elements between the boundary below and p
  return int64_t((reinterpret_cast<uintptr_t>(p) / item) & (kTileElems - 1));
}
inline int64_t write_tiles(const void* p, int64_t n, int item) { return (tile_lead(p, item) + n + kTileElems - 1) / kTileElems; }

// Calls whole(e) for each of the lane's groups of four elements e ... e + 3 that lies in the tensor, one(e) for single ones at
// the ends.
template <typename Whole, typename One>
__device__ __forceinline__ void for_tile(const void* p, int item, int64_t n, int64_t tile, Whole whole, One one) {
  const int64_t e0 = tile * kTileElems - tile_lead(p, item) + threadIdx.x * 4;
#pragma unroll
  for (int k = 0; k < kIters; k++) {
    const int64_t e = e0 + k * kThreads * 4;
    if (e >= 0 && e + 4 <= n) {
      whole(e);
    } else {
      for (int64_t x = e; x < e + 4; x++)
        if (x >= 0 && x < n) one(x);
    }
  }
}

template <int TYPE, int OUT>
__device__ __forceinline__ void clip_tile(const ClipSeg& sg, int64_t n, int64_t tile, float c) {
  using G = typename Elem<TYPE>::raw;
  using O = typename Elem<OUT>::raw;
  for_tile(
      sg.out, sizeof(O), n, tile, [&](int64_t e) { store4<OUT>(sg.out, e, times(c, load4<TYPE>(sg.g, e))); },
      [&](int64_t e) {
        const float g = Elem<TYPE>::to(static_cast<const G*>(sg.g)[e]);
        static_cast<O*>(sg.out)[e] = Elem<OUT>::from(c == 0.f ? 0.f : c * g);
      });
}

template <int CAP>
__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const Table<ClipSeg, CAP> a, const Clip clip, double* result) {
  const int tile = blockIdx.x;
  double norm = 0.0;
  const float c = clip_coefficient(clip, &norm);
  if (clip.tell && tile == 0 && threadIdx.x == 0) {
    result[1] = norm;
    result[2] = double(c);
  }
  const int k = find_segment<CAP>(a.tile_start, a.nseg, tile);
  const ClipSeg sg = a.seg[k];
  const int64_t n = seg_size(sg.nt), t = tile - a.tile_start[k];
  if (n == 0) return;
  if (sg.out == sg.g) {
    if (c == 1.f) return;
    switch (seg_type(sg.nt)) {
      case HPX_F32: clip_tile<HPX_F32, HPX_F32>(sg, n, t, c); break;
      case HPX_BF16: clip_tile<HPX_BF16, HPX_BF16>(sg, n, t, c); break;
      default: clip_tile<HPX_F16, HPX_F16>(sg, n, t, c); break;
    }
  } else {
    switch (seg_type(sg.nt)) {
      case HPX_F32: clip_tile<HPX_F32, HPX_F32>(sg, n, t, c); break;
      case HPX_BF16: clip_tile<HPX_BF16, HPX_F32>(sg, n, t, c); break;
      default: clip_tile<HPX_F16, HPX_F32>(sg, n, t, c); break;
    }
  }
}

// ---- momentum ----------------------------------------------------------------
// u' = m u + c g with the product c g rounded once and one rounding for the rest (fma), d = m u' + c g likewise.
template <int TYPE>
__device__ __forceinline__ void momentum_tile(const MomentumSeg& sg, int64_t n, int64_t tile, float m, float c) {
  using G = typename Elem<TYPE>::raw;
  for_tile(
      sg.u, 4, n, tile,
      [&](int64_t e) {
        const float4 g = times(c, load4<TYPE>(sg.g, e));
        float4 u = ld4(sg.u + e);
        u = make_float4(fmaf(m, u.x, g.x), fmaf(m, u.y, g.y), fmaf(m, u.z, g.z), fmaf(m, u.w, g.w));
        st4(sg.u + e, u);
        if (sg.d) st4(sg.d + e, make_float4(fmaf(m, u.x, g.x), fmaf(m, u.y, g.y), fmaf(m, u.z, g.z), fmaf(m, u.w, g.w)));
      },
      [&](int64_t e) {
        const float g = c == 0.f ? 0.f : c * Elem<TYPE>::to(static_cast<const G*>(sg.g)[e]);
        const float u = fmaf(m, sg.u[e], g);
        sg.u[e] = u;
        if (sg.d) sg.d[e] = fmaf(m, u, g);
      });
}

template <int CAP>
__global__ __launch_bounds__(kThreads) void gd_momentum_kernel(const Table<MomentumSeg, CAP> a, const Clip clip, double* result, float m) {
  const int tile = blockIdx.x;
  double norm = 0.0;
  const float c = clip_coefficient(clip, &norm);
  if (clip.tell && tile == 0 && threadIdx.x == 0) {
    result[1] = norm;
    result[2] = double(c);
  }
  const int k = find_segment<CAP>(a.tile_start, a.nseg, tile);
  const MomentumSeg sg = a.seg[k];
  const int64_t n = seg_size(sg.nt), t = tile - a.tile_start[k];
  if (n == 0) return;
  switch (seg_type(sg.nt)) {
    case HPX_F32: momentum_tile<HPX_F32>(sg, n, t, m, c); break;
    case HPX_BF16: momentum_tile<HPX_BF16>(sg, n, t, m, c); break;
    default: momentum_tile<HPX_F16>(sg, n, t, m, c); break;
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

struct Span {
  uintptr_t b, e;
};
// Whether the spans, in any order, overlap anywhere; sorts them.
bool overlap(std::vector<Span>& v) {
  bool sorted = true;
  for (size_t i = 1; i < v.size() && sorted; i++) sorted = v[i - 1].b <= v[i].b;
  if (!sorted) std::sort(v.begin(), v.end(), [](const Span& x, const Span& y) { return x.b < y.b; });
  for (size_t i = 1; i < v.size(); i++)
    if (v[i].b < v[i - 1].e) return true;
  return false;
}

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
int check_clip(const char* who, int order, double max_norm, double scale) {
  HPX_ARG(order == 2 || order == HPX_NORM_MAX, "%s: order %d is neither 2 nor HPX_NORM_MAX", who, order);
  HPX_ARG(max_norm >= 0.0, "%s: max_norm %g is negative or not a number", who, max_norm);
  HPX_ARG(std::isfinite(scale) && std::fabs(scale) <= FLT_MAX, "%s: scale %g is not finite", who, scale);
  return HPX_OK;
}

// Fills tables from items [0, count) and hands each to `launch(table, tiles, last)`.  fill(i, seg) returns the number of
// tiles of item i, 0 to leave it out.  At least one launch is made, of an empty table if need be.
template <typename Seg, int CAP, typename Fill, typename Launch>
int for_tables(int count, Fill fill, Launch launch) {
  Table<Seg, CAP> a;
  int i = 0;
  do {
    a.nseg = 0;
    a.tile_start[0] = 0;
    while (i < count && a.nseg < CAP) {
      const int64_t tiles = fill(i, a.seg[a.nseg]);
      if (tiles == 0) { i++; continue; }
      if (int64_t(a.tile_start[a.nseg]) + tiles > INT32_MAX - kMaxGrid) {
        if (a.nseg) break;
        set_error("tensor %d is too large for one launch", i);
        return HPX_ERR_ARG;
      }
      a.tile_start[a.nseg + 1] = a.tile_start[a.nseg] + int32_t(tiles);
      a.nseg++;
      i++;
    }
    const int rc = launch(a, a.tile_start[a.nseg], i == count);
    if (rc != HPX_OK) return rc;
  } while (i < count);
  return HPX_OK;
}

template <int ORDER, int CAP>
int launch_norm(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, int add, double* result, hipStream_t st) {
  int valid = 0;
  return for_tables<NormSeg, CAP>(
      count,
      [&](int i, NormSeg& sg) -> int64_t {
        if (sizes[i] == 0) return 0;
        const int type = types ? types[i] : HPX_F32;
        sg = NormSeg{grads[i], uint64_t(sizes[i]) | uint64_t(type) << kTypeShift};
        return norm_tiles(sizes[i], type);
      },
      [&](const Table<NormSeg, CAP>& a, int tiles, bool last) -> int {
        const int grid = std::max(1, std::min(tiles, kMaxGrid));
        HPX_LAUNCH("grad_norm_kernel", (grad_norm_kernel<ORDER, CAP>), dim3(grid), dim3(kThreads), st, a, result, valid, int(last), add);
        HPX_HIP(hipGetLastError());
        valid = std::max(valid, grid);
        return HPX_OK;
      });
}
int norm(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, int order, int add, double* result, hipStream_t st) {
  if (order == 2)
    return count <= kCapSmall ? launch_norm<2, kCapSmall>(count, grads, sizes, types, add, result, st)
                              : launch_norm<2, NormSeg::kCapLarge>(count, grads, sizes, types, add, result, st);
  return count <= kCapSmall ? launch_norm<HPX_NORM_MAX, kCapSmall>(count, grads, sizes, types, add, result, st)
                            : launch_norm<HPX_NORM_MAX, NormSeg::kCapLarge>(count, grads, sizes, types, add, result, st);
}

template <int CAP>
int launch_clip(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, void* const* outs, Clip clip, double* result, hipStream_t st) {
  return for_tables<ClipSeg, CAP>(
      count,
      [&](int i, ClipSeg& sg) -> int64_t {
        if (sizes[i] == 0) return 0;
        const int type = types ? types[i] : HPX_F32;
        sg = ClipSeg{grads[i], outs[i], uint64_t(sizes[i]) | uint64_t(type) << kTypeShift};
        return write_tiles(outs[i], sizes[i], outs[i] == grads[i] ? item_size(type) : 4);
      },
      [&](Table<ClipSeg, CAP>& a, int tiles, bool) -> int {
        if (tiles == 0) {  // norm and coefficient are told all the same
          if (!clip.tell) return HPX_OK;
          a.seg[0] = ClipSeg{nullptr, nullptr, 0};
          a.nseg = 1;
          a.tile_start[1] = 1;
          tiles = 1;
        }
        HPX_LAUNCH("grad_clip_kernel", (grad_clip_kernel<CAP>), dim3(tiles), dim3(kThreads), st, a, clip, result);
        HPX_HIP(hipGetLastError());
        clip.tell = 0;
        return HPX_OK;
      });
}

template <int CAP>
int launch_momentum(int count, const void* const* grads, const int64_t* sizes, const int32_t* types, float* const* us, float* const* outs, float m, Clip clip, double* result,
                    hipStream_t st) {
  return for_tables<MomentumSeg, CAP>(
      count,
      [&](int i, MomentumSeg& sg) -> int64_t {
        if (sizes[i] == 0) return 0;
        const int type = types ? types[i] : HPX_F32;
        sg = MomentumSeg{grads[i], us[i], outs ? outs[i] : nullptr, uint64_t(sizes[i]) | uint64_t(type) << kTypeShift};
        return write_tiles(us[i], sizes[i], 4);
      },
      [&](Table<MomentumSeg, CAP>& a, int tiles, bool) -> int {
        if (tiles == 0) {
          if (!clip.tell) return HPX_OK;
          a.seg[0] = MomentumSeg{nullptr, nullptr, nullptr, 0};
          a.nseg = 1;
          a.tile_start[1] = 1;
          tiles = 1;
        }
        HPX_LAUNCH("gd_momentum_kernel", (gd_momentum_kernel<CAP>), dim3(tiles), dim3(kThreads), st, a, clip, result, m);
        HPX_HIP(hipGetLastError());
        clip.tell = 0;
        return HPX_OK;
      });
}

template <int CAP>
int launch_mask(int count, const uint8_t* const* ins, const int32_t* in_sizes, float* const* us, const int32_t* sizes, int32_t* counts, hipStream_t st) {
  int first = 0;
  return for_tables<MaskSeg, CAP>(
      count,
      [&](int i, MaskSeg& sg) -> int64_t {
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

// Refuses lists in which an element is written twice, or written through one tensor and read through another; the tensors of
// `in_place` (one of the two lists) may be the gradients themselves.
int check_writes(const char* who, int count, const void* const* grads, const int64_t* sizes, const int32_t* types, const void* const* a, const void* const* b,
                 const void* const* in_place) {
  std::vector<Span> w;
  w.reserve(size_t(count) * (b ? 2 : 1));
  for (int i = 0; i < count; i++) {
    if (sizes[i] == 0) continue;
    const int item = a[i] == grads[i] ? item_size(types ? types[i] : HPX_F32) : 4;
    const uintptr_t p = reinterpret_cast<uintptr_t>(a[i]);
    w.push_back({p, p + uintptr_t(sizes[i]) * item});
  }
  for (int i = 0; b && i < count; i++) {
    if (sizes[i] == 0) continue;
    const uintptr_t p = reinterpret_cast<uintptr_t>(b[i]);
    w.push_back({p, p + uintptr_t(sizes[i]) * 4});
  }
  HPX_ARG(!overlap(w), "%s: two of the tensors that are written overlap", who);
  for (int i = 0; i < count; i++) {
    if (sizes[i] == 0) continue;
    const uintptr_t p = reinterpret_cast<uintptr_t>(grads[i]), e = p + uintptr_t(sizes[i]) * item_size(types ? types[i] : HPX_F32);
    if (in_place && in_place[i] == grads[i]) continue;
    // the first written span that ends behind p
    auto it = std::upper_bound(w.begin(), w.end(), p, [](uintptr_t x, const Span& s) { return x < s.e; });
    HPX_ARG(it == w.end() || it->b >= e, "%s: gradient %d overlaps a tensor that is written", who, i);
  }
  return HPX_OK;
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
    return norm(count, grads, sizes, types, order, is_add_to != 0, result, static_cast<hipStream_t>(stream));
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
    std::vector<void*> to(static_cast<size_t>(count));
    for (int i = 0; i < count; i++) {
      to[size_t(i)] = outs ? outs[i] : const_cast<void*>(grads[i]);
      HPX_ARG(sizes[i] == 0 || (to[size_t(i)] && (!outs || aligned(outs[i], 4))), "%s: output %d is null or does not start at a multiple of its element size", who, i);
      HPX_ARG(sizes[i] == 0 || !outs || !types || types[i] == HPX_F32 || outs[i] != grads[i], "%s: output %d is fp32 and cannot take the place of a gradient of another type", who, i);
    }
    if (const int rc = check_writes(who, count, grads, sizes, types, to.data(), nullptr, to.data())) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!is_measured)
      if (const int rc = norm(count, grads, sizes, types, order, 0, result, st)) return rc;
    const Clip clip{result, max_norm, scale, order, 1};
    if (count <= kCapSmall) return launch_clip<kCapSmall>(count, grads, sizes, types, to.data(), clip, result, st);
    return launch_clip<ClipSeg::kCapLarge>(count, grads, sizes, types, to.data(), clip, result, st);
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
    const void* const* ds = reinterpret_cast<const void* const*>(outs);
    if (const int rc = check_writes(who, count, grads, sizes, types, reinterpret_cast<const void* const*>(momenta), ds, ds)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const Clip clip{result, max_norm, scale, order, result != nullptr};
    if (count <= kCapSmall) return launch_momentum<kCapSmall>(count, grads, sizes, types, momenta, outs, momentum, clip, result, st);
    return launch_momentum<MomentumSeg::kCapLarge>(count, grads, sizes, types, momenta, outs, momentum, clip, result, st);
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
    for (int i = 0; i < count; i++) {
      HPX_ARG(in_sizes[i] >= 0 && sizes[i] >= 0, "%s: message %d has a negative size", who, i);
      HPX_ARG(in_sizes[i] < 4 || (ins[i] && aligned(ins[i], 4)), "%s: message %d is null or does not start at a multiple of 4 bytes", who, i);
      HPX_ARG(sizes[i] == 0 || (momenta[i] && aligned(momenta[i], 4)), "%s: momentum %d is null or does not start at a multiple of 4 bytes", who, i);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (count <= kCapSmall) return launch_mask<kCapSmall>(count, ins, in_sizes, momenta, sizes, counts, st);
    return launch_mask<MaskSeg::kCapLarge>(count, ins, in_sizes, momenta, sizes, counts, st);
  });
}
