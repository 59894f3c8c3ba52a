// Norm over all gradients of a model, and their clipping (jk_clip_grad_norm).
//
//   total = sqrt(sum_i sum_e g_ie^2)  or  max |g_ie|,   g_ie <- g_ie * min(1, max_norm / (total + eps))
//
// Two kernels: the first reads every gradient and leaves one partial per block, the second adds
// the partials (every block in the same order, so all have the same coefficient) and scales. The
// tensors' addresses go into the kernels' parameters, so a call copies no table to the device
// and can be captured into a graph.
//
// Bound: memory. A tensor is cut into chunks of 16 KB. In each block one warp finds the block's
// chunks in the table and keeps kStages bulk copies in flight into a ring in shared memory, so
// that neither the search nor the sums stop the loads; the other warps take a chunk out of the ring
// at a time. (218M bf16 into f32: 82 + 222 us with four blocks of two stages per SM, 87 + 228 with two
// of six, 142 + 229 with one of thirteen.) The second kernel takes the chunks from
// the last to the first, as the last ones that the first kernel read are still in L2, and fills
// its ring while the first one ends.
#include "jk_host.h"
#include "jk_rows.cuh"
#include "jk_sm100.cuh"

#include <type_traits>

namespace jk {
namespace clip {

constexpr int kWorkers = 256;             // threads that take chunks; one more warp loads them
constexpr int kThreads = kWorkers + 32;
constexpr int kPacks = 4;                 // 16-byte packs of a thread's turn
constexpr int kChunkPacks = kWorkers * kPacks;
constexpr int kStages = 2;
constexpr int kBlocksPerSm = 4;
constexpr int kMaxBlocks = 148 * kBlocksPerSm;
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

// Over the workers (the loading warp takes no part).
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

__device__ __forceinline__ double workers_join(double v, int kind, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  workers_sync();
  v = scratch[0];
  for (int i = 1; i < kWorkers / 32; ++i) v = join(v, scratch[i], kind);
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

// One chunk, as the loading warp leaves it beside its data: elements [at, at + packs * kPack) of
// a tensor, from a 16-byte boundary on, `lead` elements before the first boundary (first chunk)
// and `trail` after the last whole pack (last chunk), which are read where they lie.
struct Part {
  const void* body;
  void* out;  // the element of the output that corresponds to *body
  int packs;
  uint8_t type, out_type, lead, trail;
};

template <int N>
__device__ __forceinline__ Part part_of(const Table<N>& t, uint32_t chunk) {
  const int i = find(t, chunk);
  Part p;
  p.type = t.in_type[i], p.out_type = t.out_type[i];
  const int size = p.type == JK_F32 ? 4 : 2, out_size = p.out_type == JK_F32 ? 4 : 2;
  const char* in = static_cast<const char*>(t.in[i]);
  const int64_t numel = t.numel[i];
  int64_t head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / size;
  if (head > numel) head = numel;
  const uint32_t k = chunk - t.first[i];
  const int per = 16 / size;
  const int64_t all = (numel - head) / per, from = static_cast<int64_t>(k) * kChunkPacks, left = all - from;
  p.packs = static_cast<int>(left < kChunkPacks ? left : kChunkPacks);
  const int64_t at = head + from * per;
  p.body = in + at * size;
  p.out = static_cast<char*>(t.out[i]) + at * out_size;
  p.lead = k == 0 ? static_cast<uint8_t>(head) : 0;
  p.trail = left <= kChunkPacks ? static_cast<uint8_t>(numel - head - all * per) : 0;
  return p;
}

struct Ring {
  uint4 data[kStages][kChunkPacks];
  Part part[kStages];
  uint64_t full[kStages], empty[kStages];
  double scratch[kWorkers / 32];
  bool idle;
};

__device__ __forceinline__ void ring_init(Ring& ring) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], kWorkers / 32);
    }
    fence_barrier_init();
  }
  __syncthreads();
}

// The loading warp's one thread: chunks block, block + grid, ... (counted from the end when
// `backwards`) into the ring. A stage whose workers do not come back in time ends the kernel with
// an error, after the copies in flight have landed.
template <int N>
__device__ __forceinline__ void ring_load(const Table<N>& t, Ring& ring, bool backwards) {
  const uint32_t chunks = t.first[t.count];
  int n = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x, ++n) {
    const int s = n % kStages;
    if (n >= kStages && !mbar_wait(&ring.empty[s], (n / kStages - 1) & 1)) {
      g_device_error = JK_ERR_DEVICE_TIMEOUT;
      break;
    }
    const Part p = part_of(t, backwards ? chunks - 1 - c : c);
    ring.part[s] = p;
    mbar_arrive_expect_tx(&ring.full[s], p.packs * 16);
    if (p.packs > 0) bulk_load(ring.data[s], p.body, p.packs * 16, &ring.full[s]);
  }
  for (int back = n < kStages ? n : kStages; back > 0; --back) {
    const int k = n - back;
    mbar_wait(&ring.full[k % kStages], (k / kStages) & 1);
  }
}

// What a worker does with each chunk of its block.
template <int N, typename F>
__device__ __forceinline__ void ring_take(const Table<N>& t, Ring& ring, F&& take) {
  const uint32_t chunks = t.first[t.count];
  int n = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x, ++n) {
    const int s = n % kStages;
    if (!mbar_wait(&ring.full[s], (n / kStages) & 1)) {
      g_device_error = JK_ERR_DEVICE_TIMEOUT;
      return;
    }
    take(ring.part[s], ring.data[s]);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[s]);
  }
}

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
__device__ __forceinline__ double part_norm(const Part& p, const uint4* data, int kind, double acc) {
  uint4 raw[kPacks];
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    const int k = i * kWorkers + threadIdx.x;
    raw[i] = k < p.packs ? data[k] : make_uint4(0, 0, 0, 0);
  }
  float edge = 0.f;
  const int t = threadIdx.x;
  const T* body = static_cast<const T*>(p.body);
  if (t < p.lead) edge = to_f32(body[t - p.lead]);
  if (t >= 32 && t < 32 + p.trail) edge = to_f32(body[p.packs * kPack<T> + t - 32]);
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
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    norm_kernel(const __grid_constant__ Table<N> t, int kind, double* partials) {
  extern __shared__ __align__(128) unsigned char memory[];
  Ring& ring = *reinterpret_cast<Ring*>(memory);
  ring_init(ring);
  double acc = 0.0;
  if (threadIdx.x < kWorkers) {
    ring_take(t, ring, [&](const Part& p, const uint4* data) {
      JK_WITH_TYPE(p.type, T, acc = part_norm<T>(p, data, kind, acc));
    });
    grid_dependency_launch();
    acc = workers_join(acc, kind, ring.scratch);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
  } else if (threadIdx.x == kWorkers) {
    ring_load(t, ring, false);
  }
}

// total over `n` partials, the same in every block.
__device__ __forceinline__ float total_norm(const double* partials, int n, int kind, double* scratch) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kWorkers) v = join(v, partials[i], kind);
  v = workers_join(v, kind, scratch);
  return static_cast<float>(kind == JK_NORM_2 ? sqrt(v) : v);
}

// A turn's unit is what fills 16 bytes of the wider of the two types, so that neighbouring
// threads read and write neighbouring addresses on both sides.
template <typename T, typename O>
__device__ __forceinline__ void part_scale(const Part& p, const uint4* data, float coef) {
  constexpr int kUnit = sizeof(T) >= sizeof(O) ? kPack<T> : kPack<O>;  // elements
  constexpr int kTurns = kPacks * kPack<T> / kUnit;
  const int units = p.packs * (kPack<T> / kUnit);
  const T* body = static_cast<const T*>(p.body);
  O* out = static_cast<O*>(p.out);
  const int t = threadIdx.x;
  if (t < p.lead) out[t - p.lead] = from_f32<O>(to_f32(body[t - p.lead]) * coef);
  if (t >= 32 && t < 32 + p.trail) {
    const int e = p.packs * kPack<T> + t - 32;
    out[e] = from_f32<O>(to_f32(body[e]) * coef);
  }
  const bool vector = reinterpret_cast<uintptr_t>(out) % (kUnit * sizeof(O)) == 0;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int k = i * kWorkers + t;
    if (k >= units) continue;
    float f[kUnit];
    if constexpr (kUnit == kPack<T>) {
      unpack<T>(data[k], f);
    } else {  // half a pack
      const uint2 h = reinterpret_cast<const uint2*>(data)[k];
      float both[kPack<T>];
      unpack<T>(make_uint4(h.x, h.y, 0, 0), both);
#pragma unroll
      for (int j = 0; j < kUnit; ++j) f[j] = both[j];
    }
#pragma unroll
    for (int j = 0; j < kUnit; ++j) f[j] *= coef;
    if (vector) {
      if constexpr (kUnit == kPack<O>) {
        __stcs(reinterpret_cast<uint4*>(out) + k, pack<O>(f));
      } else {
        float both[kPack<O>] = {};
#pragma unroll
        for (int j = 0; j < kUnit; ++j) both[j] = f[j];
        const uint4 u = pack<O>(both);
        __stcs(reinterpret_cast<uint2*>(out) + k, make_uint2(u.x, u.y));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kUnit; ++j) out[k * kUnit + j] = from_f32<O>(f[j]);
    }
  }
}

// With outputs of their own, the ring fills before the norm is known. In place it does not: a
// coefficient of 1 then leaves every gradient as it is, unread.
template <int N>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    scale_kernel(const __grid_constant__ Table<N> t, int kind, const double* partials, int n, float max_norm, float eps,
                 bool in_place, float* total) {
  extern __shared__ __align__(128) unsigned char memory[];
  Ring& ring = *reinterpret_cast<Ring*>(memory);
  ring_init(ring);
  float coef = 0.f;
  if (threadIdx.x < kWorkers) {
    grid_dependency_wait();
    const float norm = total_norm(partials, n, kind, ring.scratch);
    coef = max_norm / (norm + eps);
    coef = coef > 1.f ? 1.f : coef;  // a NaN stays
    if (threadIdx.x == 0) {
      ring.idle = coef == 1.f;
      if (total != nullptr && blockIdx.x == 0) *total = norm;
    }
  }
  if (in_place) {
    __syncthreads();
    if (ring.idle) return;
  }
  if (threadIdx.x < kWorkers) {
    ring_take(t, ring, [&](const Part& p, const uint4* data) {
      JK_WITH_TYPE(p.type, T, JK_WITH_TYPE(p.out_type, O, (part_scale<T, O>(p, data, coef))));
    });
  } else if (threadIdx.x == kWorkers) {
    ring_load(t, ring, true);
  }
}

__global__ void __launch_bounds__(kWorkers) total_kernel(int kind, const double* partials, int n, float* total) {
  __shared__ double scratch[kWorkers / 32];
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

// Tensors [from, ...) into the table until it is full; returns the next one that is not empty, or
// `count`: another call for the rest would find something, and leaves a table that holds all as it is.
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
  while (from < q.count && q.numels[from] == 0) ++from;
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
  if (cudaFuncSetAttribute(norm_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Ring)) != cudaSuccess ||
      cudaFuncSetAttribute(scale_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Ring)) != cudaSuccess) {
    cudaGetLastError();
    return JK_ERR_LAUNCH;
  }
  Table<N> t;
  int n = 0, groups = 0;
  for (int64_t at = 0; at < q.count;) {
    at = fill(t, q, at);
    if (t.count == 0) break;
    if (++groups > kMaxGroups) return JK_ERR_BAD_SHAPE;
    norm_kernel<N><<<blocks_for(t), kThreads, sizeof(Ring), s>>>(t, kind, partials + n);
    n += blocks_for(t);
  }
  if (!clip_on || n == 0) {
    total_kernel<<<1, kWorkers, 0, s>>>(kind, partials, n, total);
    return launch_status();
  }
  for (int64_t at = 0, g = 0; at < q.count; ++g) {
    if (groups == 1) at = q.count;  // the table holds them all
    else at = fill(t, q, at);
    if (t.count == 0) break;
    const bool in_place = q.outs == nullptr;
    // only the first of them follows the kernel whose partials it waits for
    if (g == 0)
      launch_dependent(scale_kernel<N>, blocks_for(t), kThreads, sizeof(Ring), s, t, kind, partials, n, max_norm, eps,
                       in_place, total);
    else
      scale_kernel<N><<<blocks_for(t), kThreads, sizeof(Ring), s>>>(t, kind, partials, n, max_norm, eps, in_place, nullptr);
  }
  return launch_status();
}

}  // namespace clip

JK_ERROR_READER(read_error_clip)

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
