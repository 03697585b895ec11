// luma_grad.cu — the gradient operators of include/luma_b200.h: norms over
// many tensors, the clip coefficient, scaling in place and the accumulation
// of micro-batches.
//
// The tensors of a call reach the kernels as a table in the launch's own
// parameters (addresses, sizes and types by value): no table in device
// memory, no copy, nothing that outlives the call, and a captured launch
// replays with the table it was captured with.  More tensors than a table
// holds are worked on by several launches.  Every tensor is cut into tiles of
// one size; which tiles a CTA works on, where its partial result goes and in
// which order the partial results are joined follow from the tensors' sizes,
// types and alignments (tiles begin at 32-byte lines, or where eight
// accumulators do) and from how many CTAs the device holds: the same tensors
// give the same bits on every call.  The same values at another alignment may
// be summed in another order.
//
// All of it is bound by memory: one or two operations per element against 2 to
// 12 bytes.  Figures below are CUDA-event times on one B200 of passes captured
// in a graph over three sets of inputs (copy bandwidth 6.55 TB/s; pure reads
// reach 7.4).  "Layer" is one Llama-3-8B decoder layer, 9 tensors with 218 M
// elements in bf16.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <mutex>
#include <utility>
#include <vector>

#include "luma_b200.h"
#include "luma_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kVec = 32;                   // bytes of the widest load
constexpr int kBatch = 4;                  // loads in flight per thread
// The norm: two loads with five CTAs on an SM (46 registers) against four with
// two (90 registers): a layer 67.6 against 97.6 us, 42 MB 13.4 against 13.7 us,
// 16 GB 2,155 against 2,209 us.  Six or eight CTAs spill.
constexpr int kNormBatch = 2;
constexpr int kNormCtas = 5;
// tiles, as powers of two: one batch of a CTA, of a warp in the small kernel
constexpr int kNormTile = 14;        // bytes
constexpr int kScaleTile = 15;       // bytes
constexpr int kAccumulateTile = 13;  // elements
constexpr int kWarpTile = 11;        // bytes
static_assert(1 << kNormTile == kNormBatch * kThreads * kVec &&
              1 << kScaleTile == kBatch * kThreads * kVec &&
              1 << kAccumulateTile == kBatch * kThreads * 8 &&
              1 << kWarpTile == kNormBatch * 32 * kVec);

// Tensors of one launch, at most N.  Tile t belongs to the last entry i with
// first[i] <= t; entries without elements have no tiles.
template <int N>
struct Table {
  static constexpr int kMost = N;
  uint64_t ptr[N];
  int64_t numel[N];
  uint32_t first[N + 1];
  uint8_t dtype[N];
  int32_t n;
  int32_t shift;           // a tile is 2^shift bytes
};

// The same with the gradients that are added to ptr; tiles are 2^shift elements.
template <int N>
struct PairTable : Table<N> {
  uint64_t src[N];
  uint8_t src_dtype[N];
};

// A launch's parameters end at 32,764 bytes; calls with few tensors carry few
// (a norm of 84 MB 17.8 us with the small table, 18.3 us with one of 20 KB).
using Big = Table<1280>;
using Small = Table<128>;
using BigPair = PairTable<960>;
using SmallPair = PairTable<128>;

struct FinishArgs {
  const double* partials;
  int64_t n;
  int kind;
  double max_norm;
  const float* inv_scale;
  float* found_inf;
  float* norm;
  float* coef;
  double* power;
};

// The kernels of a call follow one another in a chain: each lets the next one
// be set up on the SMs it leaves free (start_next), and the next one waits for
// it to have ended, with all it wrote visible, before it touches what it needs
// from it (wait_for_previous).  Every kernel of a chain waits before it ends,
// so one that has ended has all before it behind it.  The first one is an
// ordinary launch, for which the wait returns at once.  Against ordinary
// launches: coefficient of 84 MB 18.2 against 19.7 us, norms of 10,000 tensors
// 473 against 484 us.
__device__ __forceinline__ void start_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <class T>
__device__ __forceinline__ int find_entry(const T& t, uint32_t tile) {
  int lo = 0, hi = t.n;  // first[lo] <= tile < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= tile) lo = mid; else hi = mid;
  }
  return lo;
}

// -- elements -----------------------------------------------------------------

template <int DT> struct Elem { static constexpr int kSize = DT == LUMA_F32 ? 4 : 2; };

template <int DT>
__device__ __forceinline__ float to_float(uint32_t bits) {
  if constexpr (DT == LUMA_F32) return __uint_as_float(bits);
  else if constexpr (DT == LUMA_BF16) return __uint_as_float(bits << 16);
  else return __half2float(__ushort_as_half((unsigned short)bits));
}

template <int DT>
__device__ __forceinline__ uint32_t to_bits(float v) {
  if constexpr (DT == LUMA_F32) return __float_as_uint(v);
  else if constexpr (DT == LUMA_BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  else return __half_as_ushort(__float2half_rn(v));
}

template <int DT>
__device__ __forceinline__ float load_elem(const char* p) {
  if constexpr (DT == LUMA_F32) return *reinterpret_cast<const float*>(p);
  else return to_float<DT>(*reinterpret_cast<const uint16_t*>(p));
}

template <int DT>
__device__ __forceinline__ void store_elem(char* p, float v) {
  if constexpr (DT == LUMA_F32) *reinterpret_cast<float*>(p) = v;
  else *reinterpret_cast<uint16_t*>(p) = (uint16_t)to_bits<DT>(v);
}

// The elements of a 32-bit word: one float32, or two 16-bit ones.
template <int DT>
__device__ __forceinline__ void unpack(uint32_t w, float* v) {
  if constexpr (DT == LUMA_F32) {
    v[0] = __uint_as_float(w);
  } else if constexpr (DT == LUMA_BF16) {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    v[0] = f.x;
    v[1] = f.y;
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack(const float* v) {
  if constexpr (DT == LUMA_F32) {
    return __float_as_uint(v[0]);
  } else if constexpr (DT == LUMA_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(v[0], v[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 32 bytes read once: past L1, and from memory that nothing writes meanwhile.
__device__ __forceinline__ void load_once(const char* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                 "=r"(w[6]), "=r"(w[7]) : "l"(p));
}

__device__ __forceinline__ void load32(const char* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                 "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
}

__device__ __forceinline__ void store32(char* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               :: "l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                  "r"(w[6]), "r"(w[7]) : "memory");
}

// -- sums ---------------------------------------------------------------------

// max that keeps NaN, as the norm of a tensor with a NaN has to
__device__ __forceinline__ double max_nan(double a, double b) {
  return (a != a || a > b) ? a : b;
}

__device__ __forceinline__ double join(int kind, double a, double b) {
  return kind == LUMA_NORM_MAX ? max_nan(a, b) : a + b;
}

__device__ __forceinline__ double power_of(int kind, float x) {
  const double a = fabs((double)x);
  return kind == LUMA_NORM_2 ? a * a : a;
}

// The powers of N elements joined onto `acc`: in float32, in four chains of
// N / 4 additions (2 to 8 in the kernels below), then in float64.  A float32 sum in [2^-100, 2^126] has
// not overflowed, and what its squares lost below 2^-149 is less than 2^-40 of
// it; a sum outside (all zeros excepted) is taken again in float64.  The
// maximum is taken on the magnitudes' bits, whose order has NaN above inf.
template <int KIND, int N>
__device__ __forceinline__ double join_batch(double acc, const float (&v)[N]) {
  if constexpr (KIND == LUMA_NORM_MAX) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return max_nan(acc, (double)__uint_as_float(m));
  } else {
    static_assert(N <= 64 && N % 4 == 0, "four chains of at most 16");
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i)
      s[i & 3] = KIND == LUMA_NORM_2 ? fmaf(v[i], v[i], s[i & 3]) : s[i & 3] + fabsf(v[i]);
    const float sum = (s[0] + s[1]) + (s[2] + s[3]);
    if (sum >= 0x1.0p-100f && sum <= 0x1.0p126f) return acc + (double)sum;
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= __float_as_uint(v[i]);
    if ((any & 0x7FFFFFFFu) != 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) acc += power_of(KIND, v[i]);
    }
    return acc;
  }
}

// Lanes joined in pairs, then pairs of pairs: result in lane 0 of the warp.
template <int LANES>
__device__ __forceinline__ double warp_join(int kind, double v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = join(kind, v, __shfl_down_sync(0xFFFFFFFFu, v, o));
  return v;
}

// Result in thread 0.  32 warps' values are joined like lanes (a norm of 8 KB
// of bf16 2.90 us, against 3.07 with one thread that takes them one by one); for
// 8 warps the shuffles cost the norm kernel two registers too many, and with the
// spills norms of 10,000 tensors 464 in place of 449 us.
template <int THREADS>
__device__ __forceinline__ double block_join(int kind, double v) {
  constexpr int kWarps = THREADS / 32;
  __shared__ double s[kWarps];
  v = warp_join<32>(kind, v);
  __syncthreads();  // the call before is done with s
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if constexpr (kWarps > 8) {
    if (threadIdx.x < 32) v = warp_join<kWarps>(kind, s[threadIdx.x % kWarps]);
  } else if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) v = join(kind, v, s[w]);
  }
  return v;
}

// -- tiles of one tensor --------------------------------------------------------

// Tiles of the norm and the scaling are cut at multiples of 32 bytes of the
// address space, so that whatever a tensor's alignment all but its first and
// last 32-byte line is read with full loads: [lo, hi) is the tensor's part of
// the tiles [r0, r1), [v0, v1) its full lines.
struct Span {
  char *lo, *hi, *v0, *v1;
};

template <int DT, class T>
__device__ __forceinline__ Span span_of(const T& t, int e, uint32_t r0, uint32_t r1) {
  const uint64_t p = t.ptr[e], end = p + (uint64_t)t.numel[e] * Elem<DT>::kSize;
  const uint64_t from = p & ~(uint64_t)(kVec - 1);
  const uint64_t lo = max(p, from + ((uint64_t)(r0 - t.first[e]) << t.shift));
  const uint64_t hi = min(end, from + ((uint64_t)(r1 - t.first[e]) << t.shift));
  const uint64_t v0 = (lo + kVec - 1) & ~(uint64_t)(kVec - 1);
  const uint64_t v1 = max(v0, hi & ~(uint64_t)(kVec - 1));
  return {(char*)lo, (char*)hi, (char*)v0, (char*)v1};
}

// fn(address) for the elements outside the full lines: at most 30 of them, one
// for each of the first threads of a team (`i` is the thread's place in it).
template <int DT, class F>
__device__ __forceinline__ void for_edges(const Span& s, int i, F&& fn) {
  constexpr int kSize = Elem<DT>::kSize;
  const int head = (int)(((s.v0 < s.hi ? s.v0 : s.hi) - s.lo) / kSize);
  const int tail = s.hi > s.v1 ? (int)((s.hi - s.v1) / kSize) : 0;
  if (i < head) fn(s.lo + i * kSize);
  else if (i < head + tail) fn(s.v1 + (i - head) * kSize);
}

// The powers of the tiles [r0, r1) joined onto `acc`, by a team of TEAM
// threads.  Per element a conversion (none for float32) and a multiply-add:
// the float32 sums keep float64 off the path of the data, where its conversions
// bound the kernel (a layer 380 us with float64 per element and scalar loads).
template <int DT, int KIND, int TEAM, class T>
__device__ __forceinline__ double norm_tiles(const T& t, int e, uint32_t r0, uint32_t r1, int me,
                                             double acc) {
  constexpr int kPer = 4 / Elem<DT>::kSize;  // elements per word
  const Span s = span_of<DT>(t, e, r0, r1);
#pragma unroll 1
  for (const char* p = s.v0 + me * kVec; p < s.v1; p += kNormBatch * TEAM * kVec) {
    uint32_t w[kNormBatch][8];
#pragma unroll
    for (int u = 0; u < kNormBatch; ++u) {
      if (p + u * TEAM * kVec < s.v1) {
        // a team of one warp is luma_grad_small_kernel's, which may write later
        if constexpr (TEAM == 32) load32(p + u * TEAM * kVec, w[u]);
        else load_once(p + u * TEAM * kVec, w[u]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[u][k] = 0;
      }
    }
    float v[kNormBatch * 8 * kPer];
#pragma unroll
    for (int u = 0; u < kNormBatch; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) unpack<DT>(w[u][k], v + (u * 8 + k) * kPer);
    acc = join_batch<KIND>(acc, v);
  }
  for_edges<DT>(s, me, [&](const char* p) { acc = join(KIND, acc, power_of(KIND, load_elem<DT>(p))); });
  return acc;
}

// The same by the tensor's type.
template <int KIND, int TEAM, class T>
__device__ __forceinline__ double norm_any(const T& t, int e, uint32_t r0, uint32_t r1, int me,
                                           double acc) {
  switch (t.dtype[e]) {
    case LUMA_F32: return norm_tiles<LUMA_F32, KIND, TEAM>(t, e, r0, r1, me, acc);
    case LUMA_BF16: return norm_tiles<LUMA_BF16, KIND, TEAM>(t, e, r0, r1, me, acc);
    default: return norm_tiles<LUMA_F16, KIND, TEAM>(t, e, r0, r1, me, acc);
  }
}

// The first tile of a team's share, and the team whose share holds tile r: the
// first c with r < floor(tiles (c + 1) / teams), that is r + 1 <= tiles (c + 1) /
// teams.
__device__ __forceinline__ uint32_t share_begin(uint32_t team, uint32_t teams, uint32_t tiles) {
  return (uint32_t)((uint64_t)tiles * team / teams);
}

__device__ __forceinline__ uint32_t team_of(uint32_t r, uint32_t teams, uint32_t tiles) {
  return (uint32_t)((((uint64_t)r + 1) * teams - 1) / tiles);
}

// fn(entry, r0, r1) for the tiles of one of `teams` teams: an equal share of
// all tiles of the table, one behind the other, entry by entry.  As many teams
// as the GPU holds, so there are few partials to join and no CTA starts late:
// a layer 65.4 us, against 67.6 with a CTA per tile and 65.1 with CTAs taking
// turns, which loses 2% at 16 GB (2,168 and 2,220 us).  Tiles smaller than a
// batch even the shares out and lose more in half-empty batches (42 MB 16.5 us
// with 2 KB, 12.7 with 16 KB).
template <class T, class F>
__device__ __forceinline__ void for_share(const T& t, uint32_t team, uint32_t teams, F&& fn) {
  const uint32_t tiles = t.first[t.n];
  uint32_t r = share_begin(team, teams, tiles);
  const uint32_t end = share_begin(team + 1, teams, tiles);
  if (r == end) return;
#pragma unroll 1
  for (int e = find_entry(t, r); r < end; ++e) {
    const uint32_t stop = min(end, t.first[e + 1]);
    if (r < stop) fn(e, r, stop);
    r = stop;
  }
}

// fn(entry, r, r + 1) for every tile of one CTA, CTAs taking turns.
template <class T, class F>
__device__ __forceinline__ void for_turns(const T& t, F&& fn) {
  const uint32_t tiles = t.first[t.n];
#pragma unroll 1
  for (uint32_t r = blockIdx.x; r < tiles; r += gridDim.x) fn(find_entry(t, r), r, r + 1);
}

// partials[CTA], or with TENSORS partials[CTA + entry] for every entry that the
// CTA's share touches: along the tiles one or both of the two numbers grow, so
// no two partials share a place and those of an entry lie side by side.
template <int KIND, bool TENSORS, class T>
__global__ void __launch_bounds__(kThreads, kNormCtas) luma_grad_norm_kernel(
    const __grid_constant__ T t, double* partials) {
  start_next();
  double acc = 0.0;
  for_share(t, blockIdx.x, gridDim.x, [&](int e, uint32_t r0, uint32_t r1) {
    acc = norm_any<KIND, kThreads>(t, e, r0, r1, threadIdx.x, acc);
    if constexpr (TENSORS) {
      acc = block_join<kThreads>(KIND, acc);
      if (threadIdx.x == 0) partials[blockIdx.x + e] = acc;
      acc = 0.0;
    }
  });
  if constexpr (!TENSORS) {
    acc = block_join<kThreads>(KIND, acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
  }
  wait_for_previous();  // the table before this one: other tensors, other partials
}

// partials[0, n) joined by the CTA, result in thread 0.  Eight loads in flight
// per thread: a chain of single ones costs a memory latency each (35 us of an
// 80 us call for a tensor of 3,584 tiles).
template <int THREADS>
__device__ __forceinline__ double join_partials(int kind, const double* partials, int64_t n) {
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 8 * THREADS) {
    double v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = i + u * THREADS < n ? __ldcg(partials + i + u * THREADS) : 0.0;
#pragma unroll
    for (int u = 0; u < 8; ++u) acc = join(kind, acc, v[u]);
  }
  return block_join<THREADS>(kind, acc);
}

constexpr int kTensorThreads = 128;

// One CTA per tensor: its norm, and its power for the total.  `ctas` is the
// grid that left the partials.
template <class T>
__global__ void __launch_bounds__(kTensorThreads) luma_grad_tensor_finish_kernel(
    const __grid_constant__ T t, int kind, uint32_t ctas, const double* partials, double* powers,
    float* norms) {
  wait_for_previous();
  start_next();
  const int e = blockIdx.x;
  const uint32_t tiles = t.first[t.n], r0 = t.first[e], r1 = t.first[e + 1];
  double acc = 0.0;
  if (r0 < r1) {  // no CTA has an empty share: there are no more of them than tiles
    const uint32_t c0 = team_of(r0, ctas, tiles), c1 = team_of(r1 - 1, ctas, tiles);
    acc = join_partials<kTensorThreads>(kind, partials + c0 + e, c1 - c0 + 1);
  }
  if (threadIdx.x != 0) return;
  powers[e] = acc;
  norms[e] = (float)(kind == LUMA_NORM_2 ? sqrt(acc) : acc);
}

// One thread's work on the joined partials; returns the coefficient.
__device__ __forceinline__ float write_results(const FinishArgs& a, double power) {
  if (a.power != nullptr) *a.power = power;
  // sums in 64 bits of finite float32 values are finite
  if (a.found_inf != nullptr && !isfinite(power)) *a.found_inf = 1.0f;
  const double inv = a.inv_scale != nullptr ? (double)*a.inv_scale : 1.0;
  const double r = (a.kind == LUMA_NORM_2 ? sqrt(power) : power) * fabs(inv);
  if (a.norm != nullptr) *a.norm = (float)r;
  if (a.coef == nullptr) return 1.0f;
  double c = a.max_norm / (r + 1e-6);
  if (c > 1.0) c = 1.0;  // NaN stays NaN
  *a.coef = (float)(c * inv);
  return (float)(c * inv);
}

__global__ void __launch_bounds__(1024) luma_grad_finish_kernel(const FinishArgs a) {
  wait_for_previous();
  start_next();
  const double acc = join_partials<1024>(a.kind, a.partials, a.n);
  if (threadIdx.x == 0) write_results(a, acc);
}

template <int DT, int TEAM, class T>
__device__ __forceinline__ void scale_tiles(const T& t, int e, uint32_t r0, uint32_t r1, int me,
                                            float c) {
  constexpr int kPer = 4 / Elem<DT>::kSize;
  const Span s = span_of<DT>(t, e, r0, r1);
#pragma unroll 1
  for (char* p = s.v0 + me * kVec; p < s.v1; p += kBatch * TEAM * kVec) {
    uint32_t w[kBatch][8];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (p + u * TEAM * kVec < s.v1) {
        load32(p + u * TEAM * kVec, w[u]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[u][k] = 0;
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (p + u * TEAM * kVec >= s.v1) break;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float v[kPer];
        unpack<DT>(w[u][k], v);
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] *= c;
        w[u][k] = pack<DT>(v);
      }
      store32(p + u * TEAM * kVec, w[u]);
    }
  }
  for_edges<DT>(s, me, [&](char* p) { store_elem<DT>(p, load_elem<DT>(p) * c); });
}

template <int TEAM, class T>
__device__ __forceinline__ void scale_any(const T& t, int e, uint32_t r0, uint32_t r1, int me,
                                          float c) {
  switch (t.dtype[e]) {
    case LUMA_F32: scale_tiles<LUMA_F32, TEAM>(t, e, r0, r1, me, c); break;
    case LUMA_BF16: scale_tiles<LUMA_BF16, TEAM>(t, e, r0, r1, me, c); break;
    default: scale_tiles<LUMA_F16, TEAM>(t, e, r0, r1, me, c); break;
  }
}

// Reads and writes at 7.2 TB/s (84 MB of float32 in 23.4 us).  No more CTAs
// than the GPU holds: most calls find a factor of 1 and end here, and 13,000
// CTAs that only end cost 24 us (a layer within its bound 91 against 67 us).
// Going through the tiles from the end, whose reads the norm before left in L2,
// changed nothing (51.4 and 52.3 us for norm and scaling of 84 MB).
template <class T>
__global__ void __launch_bounds__(kThreads) luma_grad_scale_kernel(
    const __grid_constant__ T t, float host_scale, const float* scale) {
  wait_for_previous();
  start_next();
  const float c = scale != nullptr ? host_scale * __ldcg(scale) : host_scale;
  if (c == 1.0f) return;  // x * 1 is x: nothing to write
  for_turns(t, [&](int e, uint32_t r0, uint32_t r1) {
    scale_any<kThreads>(t, e, r0, r1, threadIdx.x, c);
  });
}

// A small call as a whole: the norm, its results and with `clip` the scaling.
// One cluster of eight CTAs whose warps share the tiles; the warps' sums are
// joined in a fixed order, the CTAs' through distributed shared memory.  One
// launch in place of two (norm) or three (clip), one fp32 tensor that L2 holds, 30
// passes in a graph: norm of 8 KB 2.6 against 3.3 us, 128 KB 3.3 against 3.1, equal at
// 512 KB (3.4), 1 MB 3.9 against 3.6; fill and clip of 8 KB 5.9 against 6.4 us,
// equal at 128 KB (7.3), 512 KB 8.6 against 8.0, 1 MB 10.7 against 8.1, where eight
// SMs cannot read fast enough.
constexpr int kClusterCtas = 8;
constexpr int kClusterThreads = 1024;

template <int KIND>
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kClusterThreads)
luma_grad_small_kernel(const __grid_constant__ Small t, const FinishArgs a, int clip) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  cg::cluster_group::arrival_token started = cluster.barrier_arrive();
  __shared__ double sums[kClusterCtas];  // CTA 0's: one from each
  __shared__ float coef;
  constexpr uint32_t kWarps = kClusterThreads / 32;
  // neighbouring warps of a CTA get tiles that lie next to one another
  const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  double acc = 0.0;
  for_share(t, warp, kClusterCtas * kWarps, [&](int e, uint32_t r0, uint32_t r1) {
    acc = norm_any<KIND, 32>(t, e, r0, r1, lane, acc);
  });
  acc = block_join<kClusterThreads>(KIND, acc);
  cluster.barrier_wait(std::move(started));  // every CTA has its shared memory
  if (threadIdx.x == 0) *cluster.map_shared_rank(sums + blockIdx.x, 0) = acc;
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    for (int k = 1; k < kClusterCtas; ++k) acc = join(KIND, acc, sums[k]);
    const float c = write_results(a, acc);
    if (clip)
      for (int k = 0; k < kClusterCtas; ++k) *cluster.map_shared_rank(&coef, k) = c;
  }
  if (!clip) return;
  cluster.sync();
  const float c = coef;
  if (c == 1.0f) return;  // x * 1 is x: nothing to write
  for_share(t, warp, kClusterCtas * kWarps, [&](int e, uint32_t r0, uint32_t r1) {
    scale_any<32>(t, e, r0, r1, lane, c);
  });
}

// The same with a norm for each tensor: in place of three launches (20 bf16
// tensors with 8 KB 4.3 against 5.4 us, with 512 KB 5.1 against 5.5, with 1 MB 5.8
// against 5.5).  A warp leaves a
// partial at [warp + entry] for every entry that its share touches, as the CTAs
// of luma_grad_norm_kernel do.
template <int KIND>
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kClusterThreads)
luma_grad_small_tensors_kernel(const __grid_constant__ Small t, const FinishArgs a,
                               float* norms) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  constexpr uint32_t kWarps = kClusterThreads / 32, kTeams = kClusterCtas * kWarps;
  __shared__ double partials[kTeams + Small::kMost];  // CTA 0's
  __shared__ double powers[Small::kMost];
  cluster.sync();  // every CTA has its shared memory
  const uint32_t warp = blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  for_share(t, warp, kTeams, [&](int e, uint32_t r0, uint32_t r1) {
    const double acc = warp_join<32>(KIND, norm_any<KIND, 32>(t, e, r0, r1, lane, 0.0));
    if (lane == 0) *cluster.map_shared_rank(partials + warp + e, 0) = acc;
  });
  cluster.sync();
  if (blockIdx.x != 0) return;
  const uint32_t tiles = t.first[t.n];
  for (int e = warp; e < t.n; e += kWarps) {
    const uint32_t r0 = t.first[e], r1 = t.first[e + 1];
    double acc = 0.0;
    if (r0 < r1) {
      const uint32_t c0 = team_of(r0, kTeams, tiles), c1 = team_of(r1 - 1, kTeams, tiles);
      for (uint32_t c = c0 + lane; c <= c1; c += 32)
        if (share_begin(c, kTeams, tiles) < share_begin(c + 1, kTeams, tiles))
          acc = join(KIND, acc, partials[c + e]);
    }
    acc = warp_join<32>(KIND, acc);
    if (lane == 0) {
      powers[e] = acc;
      norms[e] = (float)(KIND == LUMA_NORM_2 ? sqrt(acc) : acc);
    }
  }
  __syncthreads();
  if (warp != 0) return;
  double acc = 0.0;
  for (int e = lane; e < t.n; e += 32) acc = join(KIND, acc, powers[e]);
  acc = warp_join<32>(KIND, acc);
  if (lane == 0) write_results(a, acc);
}

// Eight elements of consecutive memory, aligned to their size, as loaded.
template <int DT> struct Eight { uint32_t w[DT == LUMA_F32 ? 8 : 4]; };

template <int DT>
__device__ __forceinline__ Eight<DT> load8(const char* p) {
  Eight<DT> x;
  if constexpr (DT == LUMA_F32) {
    load32(p, x.w);
  } else {
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]) : "l"(p) : "memory");
  }
  return x;
}

template <int DT>
__device__ __forceinline__ void unpack8(const Eight<DT>& x, float (&v)[8]) {
  constexpr int kPer = 4 / Elem<DT>::kSize;
#pragma unroll
  for (int k = 0; k < 8 / kPer; ++k) unpack<DT>(x.w[k], v + k * kPer);
}

// Stores eight values; v becomes what was stored.
template <int DT>
__device__ __forceinline__ void store8(char* p, float (&v)[8]) {
  constexpr int kPer = 4 / Elem<DT>::kSize;
  Eight<DT> x;
#pragma unroll
  for (int k = 0; k < 8 / kPer; ++k) x.w[k] = pack<DT>(v + k * kPer);
  if constexpr (DT == LUMA_F32) {
    store32(p, x.w);
  } else {
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};"
                 :: "l"(p), "r"(x.w[0]), "r"(x.w[1]), "r"(x.w[2]), "r"(x.w[3]) : "memory");
    unpack8<DT>(x, v);
  }
}

// The product is rounded before it is added, not fused: for a gradient that is
// a multiple of three, fl32(fl32(1/3) * g) is g/3 itself and ties of the sum in
// bfloat16 are the ties of the definition, while the unrounded product lies a
// hair above and tips them (1 of 1,300 elements of such a sum was a step off).
struct Accumulate {
  float c;
  bool overwrite;
  __device__ __forceinline__ float operator()(float acc, float g) const {
    const float x = __fmul_rn(c, g);
    return overwrite ? x : __fadd_rn(acc, x);
  }
};

// The tiles [r0, r1) of one tensor.  Where accumulator and gradient reach a multiple
// of eight of their elements together, a thread works on eight consecutive
// elements with one load each; elsewhere (a view at an odd offset) neighbouring
// threads work on neighbouring elements.
template <int AT, int GT, int KIND, class T>
__device__ __forceinline__ double accumulate_tiles(const T& t, int e, uint32_t r0, uint32_t r1,
                                                   const Accumulate f, double sum) {
  constexpr int kA = Elem<AT>::kSize, kG = Elem<GT>::kSize;
  const int64_t n = t.numel[e];
  char* const a0 = (char*)t.ptr[e];
  const char* const g0 = (const char*)t.src[e];
  int64_t lo = (int64_t)(r0 - t.first[e]) << t.shift;
  int64_t hi = min((int64_t)(r1 - t.first[e]) << t.shift, n);
  const auto one = [&](int64_t i) {
    const float old = f.overwrite ? 0.0f : load_elem<AT>(a0 + i * kA);
    float v = f(old, load_elem<GT>(g0 + i * kG));
    store_elem<AT>(a0 + i * kA, v);
    if constexpr (KIND != LUMA_NORM_NONE) {
      v = to_float<AT>(to_bits<AT>(v));
      sum = join(KIND, sum, power_of(KIND, v));
    }
  };
  // elements before acc is at a multiple of eight elements
  const int head = (int)((8 - (t.ptr[e] / kA) % 8) % 8);
  if ((t.src[e] + (uint64_t)head * kG) % (8 * kG) == 0) {
    lo = lo == 0 ? 0 : lo + head;  // tiles move with the alignment
    hi = min(hi + head, n);
    const int64_t v0 = lo == 0 ? min((int64_t)head, n) : min(lo, n);
    const int64_t v1 = hi == n ? v0 + (max(hi - v0, (int64_t)0) & ~(int64_t)7) : hi;
#pragma unroll 1
    for (int64_t i = v0 + threadIdx.x * 8; i < v1; i += kBatch * kThreads * 8) {
      Eight<AT> x[kBatch];
      Eight<GT> y[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t j = i + u * kThreads * 8;
        x[u] = Eight<AT>{};
        y[u] = Eight<GT>{};
        if (j < v1) {
          if (!f.overwrite) x[u] = load8<AT>(a0 + j * kA);
          y[u] = load8<GT>(g0 + j * kG);
        }
      }
      float all[kBatch * 8];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t j = i + u * kThreads * 8;
        float v[8], g[8];
        unpack8<AT>(x[u], v);
        unpack8<GT>(y[u], g);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = f(v[k], g[k]);
        if (j < v1) store8<AT>(a0 + j * kA, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) all[u * 8 + k] = j < v1 ? v[k] : 0.0f;
      }
      if constexpr (KIND != LUMA_NORM_NONE) sum = join_batch<KIND>(sum, all);
    }
    const int64_t before = lo == 0 ? v0 : 0, behind = hi == n ? max(n - v1, (int64_t)0) : 0;
    const int k = threadIdx.x;
    if (k < before) one(k);
    else if (k < before + behind) one(v1 + (k - before));
  } else {
#pragma unroll 1
    for (int64_t i = lo + threadIdx.x; i < hi; i += 8 * kThreads) {
      float v[8], g[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t j = i + u * kThreads;
        v[u] = g[u] = 0.0f;
        if (j < hi) {
          if (!f.overwrite) v[u] = load_elem<AT>(a0 + j * kA);
          g[u] = load_elem<GT>(g0 + j * kG);
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t j = i + u * kThreads;
        v[u] = f(v[u], g[u]);
        if (j < hi) store_elem<AT>(a0 + j * kA, v[u]);
        v[u] = j < hi ? to_float<AT>(to_bits<AT>(v[u])) : 0.0f;
      }
      if constexpr (KIND != LUMA_NORM_NONE) sum = join_batch<KIND>(sum, v);
    }
  }
  return sum;
}

// A CTA per tile: a layer in two micro-batches, the second with the norm, 514 us
// (6.8 TB/s over both calls), against 583 us with as many CTAs as the GPU holds
// taking turns and 585 us with equal shares.  Neighbouring CTAs of one wave read
// and write neighbouring memory.
template <int KIND, class T>
__global__ void __launch_bounds__(kThreads) luma_grad_accumulate_kernel(
    const __grid_constant__ T t, float host_scale, const float* scale, int overwrite,
    double* partials) {
  start_next();
  const Accumulate f{scale != nullptr ? host_scale * __ldcg(scale) : host_scale, overwrite != 0};
  double acc = 0.0;
  for_turns(t, [&](int e, uint32_t r0, uint32_t r1) {
    switch (t.dtype[e] * 4 + t.src_dtype[e]) {
#define LUMA_CASE(A, G) \
  case A * 4 + G: acc = accumulate_tiles<A, G, KIND>(t, e, r0, r1, f, acc); break;
      LUMA_CASE(LUMA_F32, LUMA_F32)
      LUMA_CASE(LUMA_F32, LUMA_BF16)
      LUMA_CASE(LUMA_F32, LUMA_F16)
      LUMA_CASE(LUMA_BF16, LUMA_F32)
      LUMA_CASE(LUMA_BF16, LUMA_BF16)
      LUMA_CASE(LUMA_BF16, LUMA_F16)
#undef LUMA_CASE
      default: break;  // the host lets no other types through
    }
  });
  if constexpr (KIND != LUMA_NORM_NONE) {
    acc = block_join<kThreads>(KIND, acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
  }
  wait_for_previous();  // the table before this one: other tensors, other partials
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

constexpr int kMaxDevices = 64;

// What is known of each device: 0 nothing yet, 1 usable, 2 another
// architecture; and the CTAs it holds at once of each kernel.
int g_usable[kMaxDevices];
std::vector<std::pair<const void*, int>> g_resident[kMaxDevices];
std::mutex g_devices_mu;

// Makes a device current for one call and puts the caller's back.
struct DeviceScope {
  int before = -1;
  bool changed = false;
  int status = LUMA_OK;
  explicit DeviceScope(int dev) {
    cudaError_t e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != dev) {
      e = cudaSetDevice(dev);
      changed = e == cudaSuccess;
    }
    if (e != cudaSuccess) {
      status = luma_cuda_fail(e, "cudaSetDevice");
      return;
    }
    if (dev >= kMaxDevices) {
      status = luma_fail(LUMA_ERR_INVALID, "device index %d out of range", dev);
      return;
    }
    std::lock_guard<std::mutex> lk(g_devices_mu);
    if (g_usable[dev] == 0) {
      int major = 0;
      e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
      if (e != cudaSuccess) {
        status = luma_cuda_fail(e, "cudaDeviceGetAttribute");
        return;
      }
      g_usable[dev] = major == 10 ? 1 : 2;
    }
    if (g_usable[dev] == 2)
      status = luma_fail(LUMA_ERR_UNSUPPORTED, "device %d is not an sm_100 device", dev);
  }
  ~DeviceScope() {
    if (changed) cudaSetDevice(before);
  }
};

int elem_size(int dtype) { return dtype == LUMA_F32 ? 4 : 2; }

int check_list(const char* what, const uint64_t* ptr, const uint8_t* dtype, const int64_t* numel,
               int64_t n) {
  if (n > 0 && (ptr == nullptr || dtype == nullptr || numel == nullptr))
    return luma_fail(LUMA_ERR_INVALID, "%s: NULL list", what);
  for (int64_t i = 0; i < n; ++i) {
    if (numel[i] < 0)
      return luma_fail(LUMA_ERR_INVALID, "%s: entry %lld has a negative size", what, (long long)i);
    if (dtype[i] > LUMA_F16)
      return luma_fail(LUMA_ERR_INVALID, "%s: entry %lld has unknown type %d", what, (long long)i,
                       (int)dtype[i]);
    if (numel[i] > 0 && (ptr[i] == 0 || (ptr[i] & (elem_size(dtype[i]) - 1)) != 0))
      return luma_fail(LUMA_ERR_INVALID, "%s: entry %lld has a NULL or misaligned address", what,
                       (long long)i);
    if (numel[i] > (int64_t)1 << 48)
      return luma_fail(LUMA_ERR_INVALID, "%s: entry %lld is too large", what, (long long)i);
  }
  return LUMA_OK;
}

struct Range {
  uint64_t lo, hi;
  int64_t i;
};

// Tensors a call writes must not overlap one another, nor what the call reads
// for another element, the factor among it: the elements of a launch are
// worked on in no order.  src[i] may be the very elements of ptr[i].
int check_disjoint(const char* what, const LumaGradArgs* a, const uint64_t* ptr,
                   const uint8_t* dtype, const uint64_t* src, const uint8_t* src_dtype) {
  std::vector<Range> w;
  w.reserve((size_t)a->n);
  bool sorted = true;
  for (int64_t i = 0; i < a->n; ++i) {
    if (a->numel[i] == 0) continue;
    const uint64_t hi = ptr[i] + (uint64_t)a->numel[i] * elem_size(dtype[i]);
    if (!w.empty() && ptr[i] < w.back().hi) sorted = false;
    w.push_back({ptr[i], hi, i});
  }
  auto by_lo = [](const Range& x, const Range& y) { return x.lo < y.lo; };
  if (!sorted) {
    std::sort(w.begin(), w.end(), by_lo);
    for (size_t k = 1; k < w.size(); ++k)
      if (w[k].lo < w[k - 1].hi)
        return luma_fail(LUMA_ERR_INVALID, "%s: tensors %lld and %lld overlap in memory", what,
                         (long long)w[k - 1].i, (long long)w[k].i);
  }
  if (w.empty()) return LUMA_OK;
  const uint64_t s0 = (uint64_t)(uintptr_t)a->scale, s1 = s0 + sizeof(float);
  for (const Range& r : w)
    if (s0 != 0 && r.lo < s1 && s0 < r.hi)
      return luma_fail(LUMA_ERR_INVALID, "%s: the factor lies in tensor %lld", what,
                       (long long)r.i);
  if (src == nullptr) return LUMA_OK;
  const uint64_t all_lo = w.front().lo, all_hi = w.back().hi;
  for (int64_t i = 0; i < a->n; ++i) {
    if (a->numel[i] == 0) continue;
    const uint64_t lo = src[i], hi = lo + (uint64_t)a->numel[i] * elem_size(src_dtype[i]);
    if (hi <= all_lo || lo >= all_hi || (lo == ptr[i] && src_dtype[i] == dtype[i])) continue;
    // the first written range that ends behind lo
    size_t x = 0, y = w.size();
    while (x < y) {
      const size_t m = (x + y) / 2;
      if (w[m].hi > lo) y = m; else x = m + 1;
    }
    if (x < w.size() && w[x].lo < hi)
      return luma_fail(LUMA_ERR_INVALID, "%s: gradient %lld overlaps accumulator %lld in memory",
                       what, (long long)i, (long long)w[x].i);
  }
  return LUMA_OK;
}

// A tile's size as a power of two: `least`, or more where that would give more
// than `most` tiles.
int tile_shift(double total, int least, int64_t most) {
  int shift = least;
  while (std::ldexp((double)most, shift) < total) ++shift;
  return shift;
}

// Accumulation has a partial for each tile, about LUMA_GRAD_TILES at most;
// elsewhere their number only has to stay within 32 bits.
constexpr int64_t kManyTiles = (int64_t)1 << 30;

double total_bytes(const LumaGradArgs* a) {
  double total = 0.0;
  for (int64_t i = 0; i < a->n; ++i) total += (double)a->numel[i] * elem_size(a->dtypes[i]);
  return total;
}

// Fills an entry and returns its tiles.  Norm and scaling: from the 32-byte
// line that the tensor begins in.
template <int N>
int64_t fill(Table<N>& t, int k, const LumaGradArgs* a, int64_t i) {
  t.ptr[k] = a->grads[i];
  t.numel[k] = a->numel[i];
  t.dtype[k] = a->dtypes[i];
  if (a->numel[i] == 0) return 0;
  const int64_t bytes = a->numel[i] * elem_size(a->dtypes[i]) + (int64_t)(a->grads[i] % kVec);
  return ((bytes - 1) >> t.shift) + 1;
}

template <int N>
int64_t fill(PairTable<N>& t, int k, const LumaGradArgs* a, int64_t i) {
  t.ptr[k] = a->accs[i];
  t.numel[k] = a->numel[i];
  t.dtype[k] = a->acc_dtypes[i];
  t.src[k] = a->grads[i];
  t.src_dtype[k] = a->dtypes[i];
  return a->numel[i] == 0 ? 0 : ((a->numel[i] - 1) >> t.shift) + 1;
}

// Calls launch(table, index of its first tensor, its tiles) for every table of
// the call.
template <class T, class F>
int for_tables(const LumaGradArgs* a, int shift, F&& launch) {
  static thread_local T t;
  t.shift = shift;
  for (int64_t i = 0; i < a->n;) {
    const int64_t begin = i;
    int64_t tiles = 0;
    int k = 0;
    for (; i < a->n && k < T::kMost; ++i, ++k) {
      t.first[k] = (uint32_t)tiles;
      tiles += fill(t, k, a, i);
    }
    t.first[k] = (uint32_t)tiles;
    t.n = k;
    const int st = launch(t, begin, tiles);
    if (st != LUMA_OK) return st;
  }
  return LUMA_OK;
}

// The launches of one call, in order on one stream.
struct Chain {
  int device;
  cudaStream_t stream;
  bool first = true;

  Chain(int dev, void* st) : device(dev), stream(static_cast<cudaStream_t>(st)) {}

  // CTAs for so many tiles: at most what the device holds at once of a kernel.
  template <class K>
  int64_t grid(K* kernel, int64_t tiles) {
    int64_t most = 0;
    {
      std::lock_guard<std::mutex> lk(g_devices_mu);
      std::vector<std::pair<const void*, int>>& known = g_resident[device];
      for (const auto& [k, n] : known)
        if (k == (const void*)kernel) most = n;
      if (most == 0) {
        int sms = 0, per = 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kThreads, 0) !=
                cudaSuccess || sms * per == 0) {
          cudaGetLastError();
          sms = 148, per = 1;  // a guess is as right, only slower
        }
        most = sms * per;
        known.emplace_back((const void*)kernel, (int)most);
      }
    }
    return std::min(tiles, most);
  }

  template <class... P, class... A>
  int launch(const char* what, void (*kernel)(P...), int64_t grid, int threads, A&&... args) {
    if (grid == 0) return LUMA_OK;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = first ? 0 : 1;
    first = false;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
    if (e == cudaSuccess) return LUMA_OK;
    cudaGetLastError();  // reported here, not by a later call
    return luma_cuda_fail(e, what);
  }
};

FinishArgs finish_args(const LumaGradArgs* a, int64_t n_partials) {
  return {a->partials, n_partials, a->norm_kind, a->max_norm, a->inv_scale,
          a->found_inf, a->norm, a->coef, a->power};
}

int finish(const LumaGradArgs* a, int64_t n_partials, Chain& chain) {
  return chain.launch("luma_grad_finish_kernel", luma_grad_finish_kernel, 1, 1024,
                      finish_args(a, n_partials));
}

int check_norm(const char* what, const LumaGradArgs* a) {
  if (a->norm_kind != LUMA_NORM_1 && a->norm_kind != LUMA_NORM_2 && a->norm_kind != LUMA_NORM_MAX)
    return luma_fail(LUMA_ERR_INVALID, "%s: unknown norm kind %d", what, (int)a->norm_kind);
  if (a->partials == nullptr) return luma_fail(LUMA_ERR_INVALID, "%s: NULL workspace", what);
  if (a->n_partials < LUMA_GRAD_PARTIALS(a->n))
    return luma_fail(LUMA_ERR_INVALID, "%s: a workspace of %lld doubles, %lld are needed", what,
                     (long long)a->n_partials, (long long)LUMA_GRAD_PARTIALS(a->n));
  if (a->coef != nullptr && !(a->max_norm >= 0.0))
    return luma_fail(LUMA_ERR_INVALID, "%s: max_norm must be 0 or more", what);
  return LUMA_OK;
}

// The instance of a kernel template for a norm kind.
#define LUMA_BY_KIND(kind, K, ...)                             \
  ((kind) == LUMA_NORM_1   ? K<LUMA_NORM_1 __VA_OPT__(,) __VA_ARGS__>   \
   : (kind) == LUMA_NORM_2 ? K<LUMA_NORM_2 __VA_OPT__(,) __VA_ARGS__>   \
                           : K<LUMA_NORM_MAX __VA_OPT__(,) __VA_ARGS__>)

template <class T>
int norm_of(const LumaGradArgs* a, Chain& chain) {
  const bool tensors = a->norms != nullptr;
  const int shift = tile_shift(total_bytes(a), kNormTile, kManyTiles);
  auto* kernel = tensors ? LUMA_BY_KIND(a->norm_kind, luma_grad_norm_kernel, true, T)
                         : LUMA_BY_KIND(a->norm_kind, luma_grad_norm_kernel, false, T);
  int64_t partials = tensors ? a->n : 0;  // behind the tensors' powers
  int s = for_tables<T>(a, shift, [&](const T& t, int64_t, int64_t tiles) {
    const int64_t grid = chain.grid(kernel, tiles);
    double* const to = a->partials + partials;
    partials += grid + (tensors ? t.n : 0);
    return chain.launch("luma_grad_norm_kernel", kernel, grid, kThreads, t, to);
  });
  if (s != LUMA_OK) return s;
  if (!tensors) return finish(a, partials, chain);
  // behind all the norms, so that those follow one another without a gap
  partials = a->n;
  s = for_tables<T>(a, shift, [&](const T& t, int64_t begin, int64_t tiles) {
    const int64_t grid = chain.grid(kernel, tiles);
    const double* const from = a->partials + partials;
    partials += grid + t.n;
    return chain.launch("luma_grad_tensor_finish_kernel", luma_grad_tensor_finish_kernel<T>, t.n,
                        kTensorThreads, t, a->norm_kind, (uint32_t)grid, from,
                        a->partials + begin, a->norms + begin);
  });
  return s == LUMA_OK ? finish(a, a->n, chain) : s;
}

template <class T>
int scale_of(const LumaGradArgs* a, float host_scale, const float* scale, Chain& chain) {
  const int shift = tile_shift(total_bytes(a), kScaleTile, kManyTiles);
  auto* kernel = luma_grad_scale_kernel<T>;
  return for_tables<T>(a, shift, [&](const T& t, int64_t, int64_t tiles) {
    return chain.launch("luma_grad_scale_kernel", kernel, chain.grid(kernel, tiles), kThreads, t,
                        host_scale, scale);
  });
}

template <class T>
int accumulate_of(const LumaGradArgs* a, Chain& chain) {
  double total = 0.0;
  for (int64_t i = 0; i < a->n; ++i) total += (double)a->numel[i];
  const bool norm = a->norm_kind != LUMA_NORM_NONE;
  auto* kernel = norm ? LUMA_BY_KIND(a->norm_kind, luma_grad_accumulate_kernel, T)
                      : luma_grad_accumulate_kernel<LUMA_NORM_NONE, T>;
  int64_t partials = 0;
  int s = for_tables<T>(a, tile_shift(total, kAccumulateTile, LUMA_GRAD_TILES),
                        [&](const T& t, int64_t, int64_t tiles) {
    double* const to = norm ? a->partials + partials : nullptr;
    partials += tiles;
    return chain.launch("luma_grad_accumulate_kernel", kernel, tiles, kThreads, t, a->host_scale,
                        a->scale, a->overwrite, to);
  });
  if (s == LUMA_OK && norm) s = finish(a, partials, chain);
  return s;
}

// Whether a call is one for luma_grad_small_kernel (its comment has both sides).
constexpr double kSmallBytes = 1 << 19;
bool small(const LumaGradArgs* a) {
  return a->n > 0 && a->n <= Small::kMost && total_bytes(a) <= kSmallBytes;
}

int small_of(const LumaGradArgs* a, int clip, Chain& chain) {
  auto* kernel = LUMA_BY_KIND(a->norm_kind, luma_grad_small_kernel);
  auto* tensors = LUMA_BY_KIND(a->norm_kind, luma_grad_small_tensors_kernel);
  return for_tables<Small>(a, kWarpTile, [&](const Small& t, int64_t, int64_t) {
    if (a->norms != nullptr)
      return chain.launch("luma_grad_small_tensors_kernel", tensors, kClusterCtas,
                          kClusterThreads, t, finish_args(a, 0), a->norms);
    return chain.launch("luma_grad_small_kernel", kernel, kClusterCtas, kClusterThreads, t,
                        finish_args(a, 0), clip);
  });
}

int norm_call(const LumaGradArgs* a, Chain& chain) {
  if (small(a)) return small_of(a, 0, chain);
  return a->n <= Small::kMost ? norm_of<Small>(a, chain) : norm_of<Big>(a, chain);
}

int scale_call(const LumaGradArgs* a, float host_scale, const float* scale, Chain& chain) {
  return a->n <= Small::kMost ? scale_of<Small>(a, host_scale, scale, chain)
                              : scale_of<Big>(a, host_scale, scale, chain);
}

int check_args(const char* what, const LumaGradArgs* a) {
  if (a == nullptr) return luma_fail(LUMA_ERR_INVALID, "%s: NULL args", what);
  if (a->n < 0 || a->n > (int64_t)1 << 24)
    return luma_fail(LUMA_ERR_INVALID, "%s: %lld tensors", what, (long long)a->n);
  if (a->device < 0) return luma_fail(LUMA_ERR_INVALID, "%s: device %d", what, (int)a->device);
  return check_list(what, a->grads, a->dtypes, a->numel, a->n);
}

int grad_norm(const LumaGradArgs* a, void* stream) {
  int s = check_args("luma_grad_norm", a);
  if (s == LUMA_OK) s = check_norm("luma_grad_norm", a);
  if (s != LUMA_OK) return s;
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  Chain chain(a->device, stream);
  return norm_call(a, chain);
}

int grad_finish(const LumaGradArgs* a, void* stream) {
  if (a == nullptr) return luma_fail(LUMA_ERR_INVALID, "luma_grad_finish: NULL args");
  if (a->partials == nullptr || a->n_partials < 0)
    return luma_fail(LUMA_ERR_INVALID, "luma_grad_finish: no partials");
  if (a->norm_kind != LUMA_NORM_1 && a->norm_kind != LUMA_NORM_2 && a->norm_kind != LUMA_NORM_MAX)
    return luma_fail(LUMA_ERR_INVALID, "luma_grad_finish: unknown norm kind %d",
                     (int)a->norm_kind);
  if (a->coef != nullptr && !(a->max_norm >= 0.0))
    return luma_fail(LUMA_ERR_INVALID, "luma_grad_finish: max_norm must be 0 or more");
  if (a->device < 0)
    return luma_fail(LUMA_ERR_INVALID, "luma_grad_finish: device %d", (int)a->device);
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  Chain chain(a->device, stream);
  return finish(a, a->n_partials, chain);
}

int grad_scale(const LumaGradArgs* a, void* stream) {
  int s = check_args("luma_grad_scale", a);
  if (s == LUMA_OK)
    s = check_disjoint("luma_grad_scale", a, a->grads, a->dtypes, nullptr, nullptr);
  if (s != LUMA_OK) return s;
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  Chain chain(a->device, stream);
  return scale_call(a, a->host_scale, a->scale, chain);
}

int grad_clip(const LumaGradArgs* a, void* stream) {
  int s = check_args("luma_grad_clip", a);
  if (s == LUMA_OK) s = check_norm("luma_grad_clip", a);
  if (s == LUMA_OK && a->coef == nullptr)
    s = luma_fail(LUMA_ERR_INVALID, "luma_grad_clip: NULL coef");
  if (s == LUMA_OK)
    s = check_disjoint("luma_grad_clip", a, a->grads, a->dtypes, nullptr, nullptr);
  if (s != LUMA_OK) return s;
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  Chain chain(a->device, stream);
  if (a->norms == nullptr && small(a)) return small_of(a, 1, chain);
  s = norm_call(a, chain);
  if (s == LUMA_OK) s = scale_call(a, 1.0f, a->coef, chain);
  return s;
}

int grad_accumulate(const LumaGradArgs* a, void* stream) {
  const char* what = "luma_grad_accumulate";
  int s = check_args(what, a);
  if (s == LUMA_OK) s = check_list(what, a->accs, a->acc_dtypes, a->numel, a->n);
  if (s == LUMA_OK && a->norm_kind != LUMA_NORM_NONE) s = check_norm(what, a);
  if (s == LUMA_OK) s = check_disjoint(what, a, a->accs, a->acc_dtypes, a->grads, a->dtypes);
  if (s != LUMA_OK) return s;
  for (int64_t i = 0; i < a->n; ++i)
    if (a->acc_dtypes[i] == LUMA_F16)
      return luma_fail(LUMA_ERR_INVALID, "%s: accumulator %lld is float16", what, (long long)i);
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  Chain chain(a->device, stream);
  return a->n <= SmallPair::kMost ? accumulate_of<SmallPair>(a, chain)
                                  : accumulate_of<BigPair>(a, chain);
}

// No exception leaves a C entry.
int guarded(const char* what, int (*fn)(const LumaGradArgs*, void*), const LumaGradArgs* a,
            void* stream) {
  luma_g_err[0] = '\0';
  try {
    return fn(a, stream);
  } catch (const std::exception& e) {
    return luma_fail(LUMA_ERR_INVALID, "%s: %s", what, e.what());
  }
}

}  // namespace

extern "C" {

int luma_grad_norm(const LumaGradArgs* args, void* stream) {
  return guarded("luma_grad_norm", grad_norm, args, stream);
}

int luma_grad_finish(const LumaGradArgs* args, void* stream) {
  return guarded("luma_grad_finish", grad_finish, args, stream);
}

int luma_grad_scale(const LumaGradArgs* args, void* stream) {
  return guarded("luma_grad_scale", grad_scale, args, stream);
}

int luma_grad_clip(const LumaGradArgs* args, void* stream) {
  return guarded("luma_grad_clip", grad_clip, args, stream);
}

int luma_grad_accumulate(const LumaGradArgs* args, void* stream) {
  return guarded("luma_grad_accumulate", grad_accumulate, args, stream);
}

}  // extern "C"
