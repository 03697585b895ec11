// luma_grad.cu — the gradient operators of include/luma_b200.h: norms over
// many tensors, the clip coefficient, scaling in place and the accumulation
// of micro-batches.
//
// The tensors of a call reach the kernels as a table in the launch's own
// parameters (addresses, sizes and types by value): no table in device
// memory, no copy, nothing that outlives the call, and a captured launch
// replays with the table it was captured with.  More tensors than a table
// holds are worked on by several launches.  Every tensor is cut into tiles of
// one size and a CTA works on one tile, so a partial result belongs to one
// tensor, sits at a fixed place in the workspace and is summed in a fixed
// order: the same tensors give the same bits on every call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <vector>

#include "luma_b200.h"
#include "luma_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTable = 1024;               // tensors per launch
constexpr int64_t kMinTileElems = 1 << 14;

// Tensors of one launch.  Tile t belongs to the last entry i with
// first[i] <= t; entries without elements have no tiles.
struct Table {
  uint64_t ptr[kTable];
  uint64_t src[kTable];    // accumulate: the gradient added to ptr
  int64_t numel[kTable];
  uint32_t first[kTable + 1];
  uint8_t dtype[kTable];
  uint8_t src_dtype[kTable];
  int32_t n;
  int64_t tile;            // elements per tile
};

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

__device__ __forceinline__ int find_entry(const Table& t, uint32_t tile) {
  int lo = 0, hi = t.n;  // first[lo] <= tile < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= tile) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float load_elem(uint64_t p, int dtype, int64_t i) {
  if (dtype == LUMA_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == LUMA_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_elem(uint64_t p, int dtype, int64_t i, float v) {
  if (dtype == LUMA_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == LUMA_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// The value a store of v leaves behind.
__device__ __forceinline__ float stored(int dtype, float v) {
  if (dtype == LUMA_F32) return v;
  if (dtype == LUMA_BF16) return __bfloat162float(__float2bfloat16_rn(v));
  return __half2float(__float2half_rn(v));
}

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

// Result in thread 0.  Lanes and warps are joined in a fixed order.
__device__ __forceinline__ double block_join(int kind, double v) {
  __shared__ double s[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(kind, v, __shfl_down_sync(0xFFFFFFFFu, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = join(kind, v, s[w]);
  return v;
}

__global__ void __launch_bounds__(kThreads) luma_grad_norm_kernel(
    const __grid_constant__ Table t, int kind, double* partials) {
  const int e = find_entry(t, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - t.first[e]) * t.tile;
  const int64_t hi = min(lo + t.tile, t.numel[e]);
  double acc = 0.0;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads)
    acc = join(kind, acc, power_of(kind, load_elem(t.ptr[e], t.dtype[e], i)));
  acc = block_join(kind, acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// One warp per tensor: its partials joined in order.
__global__ void __launch_bounds__(kThreads) luma_grad_tensor_finish_kernel(
    const __grid_constant__ Table t, int kind, const double* partials, float* norms) {
  const int e = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= t.n) return;
  double acc = 0.0;
  for (uint32_t k = t.first[e] + lane; k < t.first[e + 1]; k += 32)
    acc = join(kind, acc, partials[k]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc = join(kind, acc, __shfl_down_sync(0xFFFFFFFFu, acc, o));
  if (lane == 0) norms[e] = (float)(kind == LUMA_NORM_2 ? sqrt(acc) : acc);
}

__global__ void __launch_bounds__(1024) luma_grad_finish_kernel(const FinishArgs a) {
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < a.n; i += 1024) acc = join(a.kind, acc, a.partials[i]);
  acc = block_join(a.kind, acc);
  if (threadIdx.x != 0) return;
  if (a.power != nullptr) *a.power = acc;
  // sums in 64 bits of finite float32 values are finite
  if (a.found_inf != nullptr && !isfinite(acc)) *a.found_inf = 1.0f;
  const double inv = a.inv_scale != nullptr ? (double)*a.inv_scale : 1.0;
  const double r = (a.kind == LUMA_NORM_2 ? sqrt(acc) : acc) * fabs(inv);
  if (a.norm != nullptr) *a.norm = (float)r;
  if (a.coef != nullptr) {
    double c = a.max_norm / (r + 1e-6);
    if (c > 1.0) c = 1.0;  // NaN stays NaN
    *a.coef = (float)(c * inv);
  }
}

__global__ void __launch_bounds__(kThreads) luma_grad_scale_kernel(
    const __grid_constant__ Table t, float host_scale, const float* scale) {
  const float c = scale != nullptr ? host_scale * *scale : host_scale;
  if (c == 1.0f) return;  // x * 1 is x: nothing to write
  const int e = find_entry(t, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - t.first[e]) * t.tile;
  const int64_t hi = min(lo + t.tile, t.numel[e]);
  for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads)
    store_elem(t.ptr[e], t.dtype[e], i, load_elem(t.ptr[e], t.dtype[e], i) * c);
}

__global__ void __launch_bounds__(kThreads) luma_grad_accumulate_kernel(
    const __grid_constant__ Table t, float host_scale, const float* scale, int overwrite, int kind,
    double* partials) {
  const float c = scale != nullptr ? host_scale * *scale : host_scale;
  const int e = find_entry(t, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - t.first[e]) * t.tile;
  const int64_t hi = min(lo + t.tile, t.numel[e]);
  double acc = 0.0;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
    const float g = load_elem(t.src[e], t.src_dtype[e], i);
    const float v = overwrite ? c * g : fmaf(c, g, load_elem(t.ptr[e], t.dtype[e], i));
    store_elem(t.ptr[e], t.dtype[e], i, v);
    if (kind != LUMA_NORM_NONE) acc = join(kind, acc, power_of(kind, stored(t.dtype[e], v)));
  }
  if (kind == LUMA_NORM_NONE) return;
  acc = block_join(kind, acc);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

constexpr int kMaxDevices = 64;

// 0: not looked at yet, 1: usable, 2: another architecture
int g_usable[kMaxDevices];
std::mutex g_usable_mu;

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
    std::lock_guard<std::mutex> lk(g_usable_mu);
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
    if (numel[i] > 0 && (ptr[i] == 0 || ptr[i] % elem_size(dtype[i]) != 0))
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
// for another element: the elements of a launch are worked on in no order.
// src[i] may be the very elements of ptr[i].
int check_disjoint(const char* what, const LumaGradArgs* a, const uint64_t* ptr,
                   const uint8_t* dtype, const uint64_t* src, const uint8_t* src_dtype) {
  try {
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
    if (src == nullptr) return LUMA_OK;
    for (int64_t i = 0; i < a->n; ++i) {
      if (a->numel[i] == 0) continue;
      const uint64_t lo = src[i], hi = lo + (uint64_t)a->numel[i] * elem_size(src_dtype[i]);
      if (lo == ptr[i] && src_dtype[i] == dtype[i]) continue;
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
  } catch (const std::bad_alloc&) {
    return luma_fail(LUMA_ERR_INVALID, "%s: out of host memory", what);
  }
  return LUMA_OK;
}

// Elements per tile: enough tiles to fill the GPU, at most about
// LUMA_GRAD_TILES in all.
int64_t tile_elems(const LumaGradArgs* a) {
  double total = 0.0;
  for (int64_t i = 0; i < a->n; ++i) total += (double)a->numel[i];
  int64_t tile = kMinTileElems;
  while ((double)tile * LUMA_GRAD_TILES < total) tile *= 2;
  return tile;
}

int64_t tiles_of(int64_t numel, int64_t tile) { return (numel + tile - 1) / tile; }

// Calls launch(table, index of its first tensor, its tiles, index of its first
// tile) for every table of the call.
template <class F>
int for_tables(const LumaGradArgs* a, const uint64_t* ptr, const uint8_t* dtype,
               const uint64_t* src, const uint8_t* src_dtype, int64_t* n_tiles, F&& launch) {
  static thread_local Table t;
  t.tile = tile_elems(a);
  int64_t done = 0;
  for (int64_t i = 0; i < a->n;) {
    const int64_t begin = i;
    int64_t tiles = 0;
    int k = 0;
    for (; i < a->n && k < kTable; ++i, ++k) {
      const int64_t m = tiles_of(a->numel[i], t.tile);
      if (tiles + m > 0x7FFFFFFF) break;
      t.ptr[k] = ptr[i];
      t.src[k] = src != nullptr ? src[i] : 0;
      t.numel[k] = a->numel[i];
      t.dtype[k] = dtype[i];
      t.src_dtype[k] = src != nullptr ? src_dtype[i] : 0;
      t.first[k] = (uint32_t)tiles;
      tiles += m;
    }
    t.first[k] = (uint32_t)tiles;
    t.n = k;
    const int st = launch(t, begin, tiles, done);
    if (st != LUMA_OK) return st;
    done += tiles;
  }
  *n_tiles = done;
  return LUMA_OK;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LUMA_OK : luma_cuda_fail(e, what);
}

int finish(const LumaGradArgs* a, int64_t n_partials, cudaStream_t st) {
  FinishArgs f{a->partials, n_partials, a->norm_kind, a->max_norm, a->inv_scale,
               a->found_inf, a->norm, a->coef, a->power};
  luma_grad_finish_kernel<<<1, 1024, 0, st>>>(f);
  return launched("luma_grad_finish_kernel");
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

int norm_of(const LumaGradArgs* a, cudaStream_t st) {
  int64_t tiles_all = 0;
  int s = for_tables(a, a->grads, a->dtypes, nullptr, nullptr, &tiles_all,
                     [&](const Table& t, int64_t begin, int64_t tiles, int64_t first) {
    if (tiles > 0)
      luma_grad_norm_kernel<<<(unsigned)tiles, kThreads, 0, st>>>(t, a->norm_kind,
                                                                  a->partials + first);
    int r = launched("luma_grad_norm_kernel");
    if (r == LUMA_OK && a->norms != nullptr) {
      luma_grad_tensor_finish_kernel<<<(t.n + kWarps - 1) / kWarps, kThreads, 0, st>>>(
          t, a->norm_kind, a->partials + first, a->norms + begin);
      r = launched("luma_grad_tensor_finish_kernel");
    }
    return r;
  });
  if (s == LUMA_OK) s = finish(a, tiles_all, st);
  return s;
}

int scale_of(const LumaGradArgs* a, float host_scale, const float* scale, cudaStream_t st) {
  int64_t tiles_all = 0;
  return for_tables(a, a->grads, a->dtypes, nullptr, nullptr, &tiles_all,
                    [&](const Table& t, int64_t, int64_t tiles, int64_t) {
    if (tiles > 0)
      luma_grad_scale_kernel<<<(unsigned)tiles, kThreads, 0, st>>>(t, host_scale, scale);
    return launched("luma_grad_scale_kernel");
  });
}

int check_args(const char* what, const LumaGradArgs* a) {
  if (a == nullptr) return luma_fail(LUMA_ERR_INVALID, "%s: NULL args", what);
  if (a->n < 0 || a->n > (int64_t)1 << 24)
    return luma_fail(LUMA_ERR_INVALID, "%s: %lld tensors", what, (long long)a->n);
  if (a->device < 0) return luma_fail(LUMA_ERR_INVALID, "%s: device %d", what, (int)a->device);
  return check_list(what, a->grads, a->dtypes, a->numel, a->n);
}

}  // namespace

extern "C" {

int luma_grad_norm(const LumaGradArgs* a, void* stream) {
  luma_g_err[0] = '\0';
  int s = check_args("luma_grad_norm", a);
  if (s == LUMA_OK) s = check_norm("luma_grad_norm", a);
  if (s != LUMA_OK) return s;
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  return norm_of(a, static_cast<cudaStream_t>(stream));
}

int luma_grad_finish(const LumaGradArgs* a, void* stream) {
  luma_g_err[0] = '\0';
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
  return finish(a, a->n_partials, static_cast<cudaStream_t>(stream));
}

int luma_grad_scale(const LumaGradArgs* a, void* stream) {
  luma_g_err[0] = '\0';
  int s = check_args("luma_grad_scale", a);
  if (s == LUMA_OK)
    s = check_disjoint("luma_grad_scale", a, a->grads, a->dtypes, nullptr, nullptr);
  if (s != LUMA_OK) return s;
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  return scale_of(a, a->host_scale, a->scale, static_cast<cudaStream_t>(stream));
}

int luma_grad_clip(const LumaGradArgs* a, void* stream) {
  luma_g_err[0] = '\0';
  int s = check_args("luma_grad_clip", a);
  if (s == LUMA_OK) s = check_norm("luma_grad_clip", a);
  if (s == LUMA_OK && a->coef == nullptr)
    s = luma_fail(LUMA_ERR_INVALID, "luma_grad_clip: NULL coef");
  if (s == LUMA_OK)
    s = check_disjoint("luma_grad_clip", a, a->grads, a->dtypes, nullptr, nullptr);
  if (s != LUMA_OK) return s;
  DeviceScope dev(a->device);
  if (dev.status != LUMA_OK) return dev.status;
  s = norm_of(a, static_cast<cudaStream_t>(stream));
  if (s == LUMA_OK) s = scale_of(a, 1.0f, a->coef, static_cast<cudaStream_t>(stream));
  return s;
}

int luma_grad_accumulate(const LumaGradArgs* a, void* stream) {
  luma_g_err[0] = '\0';
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int64_t tiles_all = 0;
  s = for_tables(a, a->accs, a->acc_dtypes, a->grads, a->dtypes, &tiles_all,
                 [&](const Table& t, int64_t, int64_t tiles, int64_t first) {
    if (tiles > 0)
      luma_grad_accumulate_kernel<<<(unsigned)tiles, kThreads, 0, st>>>(
          t, a->host_scale, a->scale, a->overwrite, a->norm_kind,
          a->partials != nullptr ? a->partials + first : nullptr);
    return launched("luma_grad_accumulate_kernel");
  });
  if (s == LUMA_OK && a->norm_kind != LUMA_NORM_NONE) s = finish(a, tiles_all, st);
  return s;
}

}  // extern "C"
