// Norm over all gradients of a model, and their clipping (jk_clip_grad_norm).
//
//   total = sqrt(sum_i sum_e g_ie^2)  or  max |g_ie|,   g_ie <- g_ie * min(1, max_norm / (total + eps))
//
// Two kernels: the first reads every gradient and leaves one partial per block, the second adds
// the partials (every block in the same order, so all have the same coefficient) and scales. The
// squares are summed in f64: neither their range nor the count of elements can spoil the sum.
// The tensors' addresses go into the kernels' parameters, so a call copies no table to the
// device and can be captured into a graph.
#include "jk_host.h"
#include "jk_rows.cuh"

namespace jk {
namespace clip {

constexpr int kThreads = 512;
constexpr int kMaxBlocks = 148 * 2;
constexpr int kTable = 640;                 // tensors of one launch
constexpr int64_t kChunk = 16384;           // elements that a block takes at a time
constexpr int kMaxGroups = 64;              // launches of the first kernel whose partials fit the workspace

struct Table {
  const void* in[kTable];
  void* out[kTable];
  int64_t numel[kTable];
  uint32_t first[kTable + 1];  // chunk number at which a tensor begins
  uint8_t in_type[kTable], out_type[kTable];
  int count;
};

// What the partials hold: sums of squares (f64), or maxima.
__device__ __forceinline__ double join(double a, double b, int kind) {
  if (kind == JK_NORM_2) return a + b;
  return a != a || a > b ? a : b;  // NaN stays
}

__device__ __forceinline__ double block_join(double v, int kind, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < kThreads / 32; ++i) v = join(v, scratch[i], kind);
  __syncthreads();
  return v;
}

__device__ __forceinline__ int find(const Table& t, uint32_t chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float load(const void* p, int64_t i, int type) {
  if (type == JK_F32) return static_cast<const float*>(p)[i];
  if (type == JK_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store(void* p, int64_t i, int type, float v) {
  if (type == JK_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == JK_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Table t, int kind, double* partials) {
  __shared__ double scratch[kThreads / 32];
  double acc = 0.0;
  const uint32_t chunks = t.first[t.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find(t, c);
    const int64_t begin = (c - t.first[i]) * kChunk;
    const int64_t end = min(begin + kChunk, t.numel[i]);
    for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
      const double v = load(t.in[i], e, t.in_type[i]);
      acc = join(acc, kind == JK_NORM_2 ? v * v : fabs(v), kind);
    }
  }
  acc = block_join(acc, kind, scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// total over `n` partials; every block computes it, block 0 of the first group writes it.
__device__ __forceinline__ float total_norm(const double* partials, int n, int kind, double* scratch) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = join(v, partials[i], kind);
  v = block_join(v, kind, scratch);
  return static_cast<float>(kind == JK_NORM_2 ? sqrt(v) : v);
}

__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table t, int kind, const double* partials, int n, float max_norm, float eps,
                 float* total) {
  __shared__ double scratch[kThreads / 32];
  const float norm = total_norm(partials, n, kind, scratch);
  if (total != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *total = norm;
  float coef = max_norm / (norm + eps);
  coef = coef > 1.f ? 1.f : coef;  // a NaN stays
  const uint32_t chunks = t.first[t.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find(t, c);
    if (coef == 1.f && t.in[i] == t.out[i]) continue;
    const int64_t begin = (c - t.first[i]) * kChunk;
    const int64_t end = min(begin + kChunk, t.numel[i]);
    for (int64_t e = begin + threadIdx.x; e < end; e += kThreads)
      store(t.out[i], e, t.out_type[i], load(t.in[i], e, t.in_type[i]) * coef);
  }
}

__global__ void __launch_bounds__(kThreads) total_kernel(int kind, const double* partials, int n, float* total) {
  __shared__ double scratch[kThreads / 32];
  const float norm = total_norm(partials, n, kind, scratch);
  if (threadIdx.x == 0) *total = norm;
}

// Tensors [from, ...) into the table until it is full; returns the next tensor.
inline int64_t fill(Table& t, const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes,
                    const int* out_dtypes, int64_t count, int64_t from) {
  int n = 0;
  uint32_t chunk = 0;
  for (; from < count && n < kTable; ++from) {
    if (numels[from] == 0) continue;
    const int64_t chunks = (numels[from] + kChunk - 1) / kChunk;
    if (n > 0 && chunk + chunks > 0x7fffffff) break;
    t.in[n] = grads[from];
    t.out[n] = outs == nullptr ? const_cast<void*>(grads[from]) : outs[from];
    t.numel[n] = numels[from];
    t.in_type[n] = static_cast<uint8_t>(dtypes[from]);
    t.out_type[n] = static_cast<uint8_t>(outs == nullptr ? dtypes[from] : out_dtypes[from]);
    t.first[n++] = chunk;
    chunk += static_cast<uint32_t>(chunks);
  }
  t.first[n] = chunk;
  t.count = n;
  return from;
}

inline int blocks_for(const Table& t) {
  const uint32_t chunks = t.first[t.count];
  return static_cast<int>(chunks < kMaxBlocks ? chunks : kMaxBlocks);
}

}  // namespace clip
}  // namespace jk

extern "C" int64_t jk_clip_grad_norm_workspace(void) {
  return static_cast<int64_t>(sizeof(double)) * jk::clip::kMaxBlocks * jk::clip::kMaxGroups;
}

extern "C" int jk_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes,
                                 const int* out_dtypes, int64_t count, int norm_kind, int clip_on, float max_norm,
                                 float eps, float* total, void* workspace, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::clip;
  if (count < 0 || count > static_cast<int64_t>(kTable) * kMaxGroups) return JK_ERR_BAD_SHAPE;
  if (norm_kind != JK_NORM_2 && norm_kind != JK_NORM_INF) return JK_ERR_UNSUPPORTED_KIND;
  if (total == nullptr || workspace == nullptr) return JK_ERR_BAD_ARG;
  if (count > 0 && (grads == nullptr || numels == nullptr || dtypes == nullptr || (outs != nullptr && out_dtypes == nullptr)))
    return JK_ERR_BAD_ARG;
  if (!aligned16(workspace)) return JK_ERR_ALIGNMENT;
  for (int64_t i = 0; i < count; ++i) {
    if (numels[i] < 0) return JK_ERR_BAD_SHAPE;
    if (!float_dtype(dtypes[i]) || (outs != nullptr && !float_dtype(out_dtypes[i]))) return JK_ERR_BAD_DTYPE;
    if (numels[i] > 0 && (grads[i] == nullptr || (outs != nullptr && outs[i] == nullptr))) return JK_ERR_BAD_ARG;
  }
  int st = check_device();
  if (st != JK_OK) return st;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  auto* partials = static_cast<double*>(workspace);
  Table t;
  int n = 0, groups = 0;
  for (int64_t at = 0; at < count;) {
    at = fill(t, grads, outs, numels, dtypes, out_dtypes, count, at);
    if (t.count == 0) break;
    if (++groups > kMaxGroups) return JK_ERR_BAD_SHAPE;
    norm_kernel<<<blocks_for(t), kThreads, 0, s>>>(t, norm_kind, partials + n);
    n += blocks_for(t);
  }
  if (clip_on && n > 0) {
    for (int64_t at = 0, g = 0; at < count; ++g) {
      if (groups > 1 || g > 0) at = fill(t, grads, outs, numels, dtypes, out_dtypes, count, at); else at = count;
      if (t.count == 0) break;
      scale_kernel<<<blocks_for(t), kThreads, 0, s>>>(t, norm_kind, partials, n, max_norm, eps, g == 0 ? total : nullptr);
    }
  } else {
    total_kernel<<<1, kThreads, 0, s>>>(norm_kind, partials, n, total);
  }
  return launch_status();
}
