// Norm over all gradients of a model, and their clipping (jk_clip_grad_norm).
//
//   total = sqrt(sum_i sum_e g_ie^2)  or  max |g_ie|,   g_ie <- g_ie * min(1, max_norm / (total + eps))
//
// Two kernels: the first reads every gradient and leaves one partial per block, the second adds
// the partials (every block in the same order, so all have the same coefficient) and scales. The
// tensors' addresses go into the kernels' parameters, so a call copies no table to the device
// and can be captured into a graph.
//
// Bound: memory. A tensor is cut into chunks of 32 KB; a block takes a chunk at a time, each
// thread four 16-byte loads at once. The second kernel takes the chunks from the last to the
// first, as the last ones that the first kernel read are still in L2.
#include "jk_host.h"
#include "jk_rows.cuh"

#include <type_traits>

namespace jk {
namespace clip {

constexpr int kThreads = 512;
constexpr int kPacks = 4;                                        // 16-byte packs of a thread's turn
constexpr int64_t kChunkPacks = static_cast<int64_t>(kThreads) * kPacks;
constexpr int kMaxBlocks = 148 * 2;
constexpr int kSmall = 64, kLarge = 640;  // tensors of one launch: the parameters of a launch are copied, so few tensors take the small table
constexpr int kMaxGroups = 64;            // launches of the first kernel whose partials fit the workspace

template <int N>
struct Table {
  const void* in[N];
  void* out[N];
  int64_t numel[N];
  uint32_t first[N + 1];  // chunk number at which a tensor begins
  uint8_t in_type[N], out_type[N];
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
  v = scratch[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
  for (int o = kThreads / 64; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  return v;
}

template <int N>
__device__ __forceinline__ int find(const Table<N>& t, uint32_t chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// The part of a tensor that is one chunk: elements [head, head + packs * kPack) from a 16-byte
// boundary on, `lead` elements before the first boundary (first chunk) and `trail` after the
// last whole pack (last chunk).
template <typename T>
struct Part {
  const T* body;
  int64_t at;  // body's first element in the tensor
  int packs, lead, trail;

  __device__ __forceinline__ Part(const void* base, int64_t numel, uint32_t chunk) {
    const T* p = static_cast<const T*>(base);
    int64_t head = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
    if (head > numel) head = numel;
    const int64_t all = (numel - head) / kPack<T>, from = chunk * kChunkPacks;
    const int64_t left = all - from;
    packs = static_cast<int>(left < kChunkPacks ? left : kChunkPacks);
    at = head + from * kPack<T>;
    body = p + at;
    lead = chunk == 0 ? static_cast<int>(head) : 0;
    trail = left <= kChunkPacks ? static_cast<int>(numel - head - all * kPack<T>) : 0;
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum of the squares of a thread's packs, in f32: at most 32 squares, so the sum is good to
// 2^-19; where it leaves f32's range, or comes near its lower end, the squares are taken again
// in f64 (f16 cannot get there). Zeros, common in the gradients of an embedding, do not.
template <typename T>
__device__ __forceinline__ double squares(const uint4 (&raw)[kPacks]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    float f[kPack<T>];
    unpack<T>(raw[i], f);
#pragma unroll
    for (int j = 0; j < kPack<T>; ++j) s = fmaf(f[j], f[j], s);
  }
  if constexpr (sizeof(T) == 4 || std::is_same<T, __nv_bfloat16>::value) {
    if (!(s > 1e-25f && s < 1e35f)) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < kPacks; ++i) bits |= raw[i].x | raw[i].y | raw[i].z | raw[i].w;
      if ((bits & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu)) == 0) return 0.0;
      double d = 0.0;
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        float f[kPack<T>];
        unpack<T>(raw[i], f);
#pragma unroll
        for (int j = 0; j < kPack<T>; ++j) d += static_cast<double>(f[j]) * static_cast<double>(f[j]);
      }
      return d;
    }
  }
  return static_cast<double>(s);
}

template <typename T>
__device__ __forceinline__ double part_norm(const Part<T>& p, int kind, double acc) {
  uint4 raw[kPacks];
  const uint4* src = reinterpret_cast<const uint4*>(p.body);
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    const int k = i * kThreads + threadIdx.x;
    raw[i] = k < p.packs ? src[k] : make_uint4(0, 0, 0, 0);
  }
  float edge = 0.f;
  const int t = threadIdx.x;
  if (t < p.lead) edge = to_f32(p.body[t - p.lead]);
  if (t >= 32 && t < 32 + p.trail) edge = to_f32(p.body[static_cast<int64_t>(p.packs) * kPack<T> + t - 32]);
  if (kind == JK_NORM_2) {
    acc += squares<T>(raw);
    if (edge != 0.f) acc += static_cast<double>(edge) * static_cast<double>(edge);
    return acc;
  }
  float m = fabsf(edge);
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    float f[kPack<T>];
    unpack<T>(raw[i], f);
#pragma unroll
    for (int j = 0; j < kPack<T>; ++j) m = max_nan(m, fabsf(f[j]));
  }
  return join(acc, static_cast<double>(m), kind);
}

template <int N>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Table<N> t, int kind, double* partials) {
  __shared__ double scratch[kThreads / 32];
  double acc = 0.0;
  const uint32_t chunks = t.first[t.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find(t, c);
    const int type = t.in_type[i];
    const uint32_t k = c - t.first[i];
    JK_WITH_TYPE(type, T, acc = part_norm<T>(Part<T>(t.in[i], t.numel[i], k), kind, acc));
  }
  acc = block_join(acc, kind, scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// total over `n` partials, the same in every block.
__device__ __forceinline__ float total_norm(const double* partials, int n, int kind, double* scratch) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = join(v, partials[i], kind);
  v = block_join(v, kind, scratch);
  return static_cast<float>(kind == JK_NORM_2 ? sqrt(v) : v);
}

// B bytes of memory in registers.
template <int B>
struct Raw;
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<16> { using type = uint4; };

// The unit of a thread's turn is what fills 16 bytes of the wider of the two types, so that
// neighbouring threads read and write neighbouring addresses on both sides.
template <typename T, typename O>
__device__ __forceinline__ void part_scale(const Part<T>& p, O* out, float coef) {
  constexpr int kUnit = sizeof(T) >= sizeof(O) ? kPack<T> : kPack<O>;  // elements
  constexpr int kTurns = kPacks * kPack<T> / kUnit;
  using In = typename Raw<kUnit * sizeof(T)>::type;
  using Out = typename Raw<kUnit * sizeof(O)>::type;
  const int units = p.packs * (kPack<T> / kUnit);
  In raw[kTurns];
  const In* src = reinterpret_cast<const In*>(p.body);
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int k = i * kThreads + threadIdx.x;
    if (k < units) raw[i] = __ldcs(src + k);
  }
  const int t = threadIdx.x;
  O* dst = out + p.at;
  if (t < p.lead) dst[t - p.lead] = from_f32<O>(to_f32(p.body[t - p.lead]) * coef);
  if (t >= 32 && t < 32 + p.trail) {
    const int64_t e = static_cast<int64_t>(p.packs) * kPack<T> + t - 32;
    dst[e] = from_f32<O>(to_f32(p.body[e]) * coef);
  }
  const bool vector = reinterpret_cast<uintptr_t>(dst) % sizeof(Out) == 0;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int k = i * kThreads + threadIdx.x;
    if (k >= units) continue;
    const T* in = reinterpret_cast<const T*>(&raw[i]);
    Out wide;
    O* f = reinterpret_cast<O*>(&wide);
#pragma unroll
    for (int j = 0; j < kUnit; ++j) f[j] = from_f32<O>(to_f32(in[j]) * coef);
    if (vector) {
      __stcs(reinterpret_cast<Out*>(dst) + k, wide);
    } else {
#pragma unroll
      for (int j = 0; j < kUnit; ++j) dst[static_cast<int64_t>(k) * kUnit + j] = f[j];
    }
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table<N> t, int kind, const double* partials, int n, float max_norm, float eps,
                 float* total) {
  __shared__ double scratch[kThreads / 32];
  const float norm = total_norm(partials, n, kind, scratch);
  if (total != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *total = norm;
  float coef = max_norm / (norm + eps);
  coef = coef > 1.f ? 1.f : coef;  // a NaN stays
  const uint32_t chunks = t.first[t.count];
  for (uint32_t back = blockIdx.x; back < chunks; back += gridDim.x) {
    const uint32_t c = chunks - 1 - back;
    const int i = find(t, c);
    if (coef == 1.f && t.in[i] == t.out[i]) continue;
    const int type = t.in_type[i], out_type = t.out_type[i];
    const uint32_t k = c - t.first[i];
    JK_WITH_TYPE(type, T, {
      const Part<T> part(t.in[i], t.numel[i], k);
      JK_WITH_TYPE(out_type, O, part_scale<T, O>(part, static_cast<O*>(t.out[i]), coef));
    });
  }
}

__global__ void __launch_bounds__(kThreads) total_kernel(int kind, const double* partials, int n, float* total) {
  __shared__ double scratch[kThreads / 32];
  const float norm = total_norm(partials, n, kind, scratch);
  if (threadIdx.x == 0) *total = norm;
}

// The call's tensors.
struct Call {
  const void* const* grads;
  void* const* outs;
  const int64_t* numels;
  const int* dtypes;
  const int* out_dtypes;
  int64_t count;
};

inline int64_t chunks_of(const Call& q, int64_t i) {
  const int64_t size = dtype_bytes(q.dtypes[i]);
  int64_t head = ((16 - (reinterpret_cast<uintptr_t>(q.grads[i]) & 15)) & 15) / size;  // as Part has it
  if (head > q.numels[i]) head = q.numels[i];
  const int64_t packs = (q.numels[i] - head) * size / 16;
  return packs <= kChunkPacks ? 1 : (packs + kChunkPacks - 1) / kChunkPacks;
}

// Tensors [from, ...) into the table until it is full; returns the next tensor.
template <int N>
int64_t fill(Table<N>& t, const Call& q, int64_t from) {
  int n = 0;
  uint32_t chunk = 0;
  for (; from < q.count && n < N; ++from) {
    if (q.numels[from] == 0) continue;
    const int64_t chunks = chunks_of(q, from);
    if (n > 0 && chunk + chunks > 0x7fffffff) break;
    t.in[n] = q.grads[from];
    t.out[n] = q.outs == nullptr ? const_cast<void*>(q.grads[from]) : q.outs[from];
    t.numel[n] = q.numels[from];
    t.in_type[n] = static_cast<uint8_t>(q.dtypes[from]);
    t.out_type[n] = static_cast<uint8_t>(q.outs == nullptr ? q.dtypes[from] : q.out_dtypes[from]);
    t.first[n++] = chunk;
    chunk += static_cast<uint32_t>(chunks);
  }
  t.first[n] = chunk;
  t.count = n;
  return from;
}

template <int N>
int blocks_for(const Table<N>& t) {
  const uint32_t chunks = t.first[t.count];
  return static_cast<int>(chunks < kMaxBlocks ? chunks : kMaxBlocks);
}

template <int N>
int launch(const Call& q, int kind, bool clip_on, float max_norm, float eps, float* total, double* partials,
           cudaStream_t s) {
  Table<N> t;
  int n = 0, groups = 0;
  for (int64_t at = 0; at < q.count;) {
    at = fill(t, q, at);
    if (t.count == 0) break;
    if (++groups > kMaxGroups) return JK_ERR_BAD_SHAPE;
    norm_kernel<N><<<blocks_for(t), kThreads, 0, s>>>(t, kind, partials + n);
    n += blocks_for(t);
  }
  if (!clip_on || n == 0) {
    total_kernel<<<1, kThreads, 0, s>>>(kind, partials, n, total);
    return launch_status();
  }
  for (int64_t at = 0, g = 0; at < q.count; ++g) {
    if (groups == 1) at = q.count;  // the table holds them all
    else at = fill(t, q, at);
    if (t.count == 0) break;
    scale_kernel<N><<<blocks_for(t), kThreads, 0, s>>>(t, kind, partials, n, max_norm, eps, g == 0 ? total : nullptr);
  }
  return launch_status();
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
  if (count < 0 || count > static_cast<int64_t>(kLarge) * kMaxGroups) return JK_ERR_BAD_SHAPE;
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
  const Call q{grads, outs, numels, dtypes, out_dtypes, count};
  auto* partials = static_cast<double*>(workspace);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (count <= kSmall) return launch<kSmall>(q, norm_kind, clip_on != 0, max_norm, eps, total, partials, s);
  return launch<kLarge>(q, norm_kind, clip_on != 0, max_norm, eps, total, partials, s);
}
