// Softmax cross entropy over a vocabulary and its gradient (jk_cross_entropy_forward / _backward).
//
//   lse = m + log sum_j exp(z_j - m), m = max_j z_j
//   loss = lse - (1 - a) z_t - a E_j[z_j]
//   grad_j = c (exp(z_j - lse) - (1 - a) [j = t] - a / V),  c = scale / number of rows that count
//
// With the maximum at hand, loss = log sum exp(z - m) + (1 - a) (m - z_t) + a E_j[m - z_j] and
// softmax_j = exp(z_j - m) / sum: differences from m keep their digits where m is large, which
// lse = m + log(sum), one f32 number, does not. exp(z - m) is taken of the difference: with z * log2(e) - m * log2(e) in one fma, logits of the
// type's lowest value would overflow both products and meet as inf - inf.
#include "jk_host.h"
#include "jk_rows.cuh"

namespace jk {
namespace loss {

constexpr int kThreads = 512;
constexpr int kMaxBlocks = 148 * 4;

// What a block leaves for the reduction over rows.
struct Partial {
  double sum;
  long long rows;
};

// Sum of one value per thread, and the maximum of another, over the block (NaN is kept by the
// sum; the maximum ignores it).
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = warp_sum32(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < kThreads / 32; ++i) v += scratch[i];
  __syncthreads();
  return v;
}

__device__ __forceinline__ float block_max(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < kThreads / 32; ++i) v = fmaxf(v, scratch[i]);
  __syncthreads();
  return v;
}

// Rows that count, over all rows (every block counts for itself).
__device__ __forceinline__ int count_rows(const int64_t* targets, int64_t rows, int64_t ignore_index, int* scratch) {
  if (threadIdx.x == 0) *scratch = 0;
  __syncthreads();
  int n = 0;
  for (int64_t r = threadIdx.x; r < rows; r += kThreads) n += targets[r] != ignore_index;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) atomicAdd(scratch, n);
  __syncthreads();
  return *scratch;
}

template <typename T>
__device__ __forceinline__ void write_grad(const T* z, T* grad, int64_t vocab, float base, float inv, float c,
                                           int64_t target, float smoothing) {
  const float share = smoothing / static_cast<float>(vocab), hit = 1.f - smoothing;
  for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
    float p = expf(to_f32(z[j]) - base) * inv - share;
    if (j == target) p -= hit;
    grad[j] = from_f32<T>(c * p);
  }
}

// One block per row at a time; the row is read three times.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    forward_kernel(const T* logits, int64_t stride, const int64_t* targets, int64_t rows, int64_t vocab,
                   int64_t ignore_index, float smoothing, int reduction, float grad_scale, float* losses, float* lse_out,
                   T* grad, int64_t grad_stride, Partial* partials) {
  __shared__ float scratch[kThreads / 32];
  __shared__ int counted;
  float c = grad_scale;
  if (grad != nullptr && reduction == JK_REDUCE_MEAN)
    c = grad_scale / static_cast<float>(count_rows(targets, rows, ignore_index, &counted));
  Partial part{0.0, 0};
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t target = targets[r];
    const T* z = logits + r * stride;
    T* g = grad == nullptr ? nullptr : grad + r * grad_stride;
    if (target == ignore_index) {
      if (threadIdx.x == 0) {
        if (losses != nullptr) losses[r] = 0.f;
        if (lse_out != nullptr) lse_out[r] = 0.f;
      }
      if (g != nullptr)
        for (int64_t j = threadIdx.x; j < vocab; j += kThreads) g[j] = from_f32<T>(0.f);
      continue;
    }
    float m = -INFINITY;
    for (int64_t j = threadIdx.x; j < vocab; j += kThreads) m = fmaxf(m, to_f32(z[j]));
    m = block_max(m, scratch);
    float a = 0.f, all = 0.f;
    for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
      const float d = to_f32(z[j]) - m;
      a += expf(d);
      all -= d;
    }
    a = block_sum(a, scratch);
    const float lse = m + logf(a);
    const bool inside = target >= 0 && target < vocab;
    float l = inside ? logf(a) + (1.f - smoothing) * (m - to_f32(z[target])) : NAN;
    if (smoothing != 0.f) l += smoothing * (block_sum(all, scratch) / static_cast<float>(vocab));
    __syncthreads();  // z[target] is read before an in-place gradient replaces it
    if (threadIdx.x == 0) {
      if (losses != nullptr) losses[r] = l;
      if (lse_out != nullptr) lse_out[r] = lse;
    }
    part.sum += l;
    part.rows += 1;
    if (g != nullptr) write_grad(z, g, vocab, m, 1.f / a, inside ? c : NAN, target, smoothing);
    __syncthreads();
  }
  if (threadIdx.x == 0) partials[blockIdx.x] = part;
}

// The blocks' partial sums, in their order.
__global__ void reduce_kernel(const Partial* partials, int blocks, int reduction, float* loss) {
  double sum = 0.0;
  long long n = 0;
  for (int i = threadIdx.x; i < blocks; i += 32) {
    sum += partials[i].sum;
    n += partials[i].rows;
  }
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (threadIdx.x == 0) *loss = static_cast<float>(reduction == JK_REDUCE_MEAN ? sum / static_cast<double>(n) : sum);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    backward_kernel(const float* grad_loss, const T* logits, int64_t stride, const int64_t* targets, const float* lse,
                    int64_t rows, int64_t vocab, int64_t ignore_index, float smoothing, int reduction, T* grad,
                    int64_t grad_stride) {
  __shared__ int counted;
  float w = 1.f;
  if (reduction == JK_REDUCE_MEAN) w = 1.f / static_cast<float>(count_rows(targets, rows, ignore_index, &counted));
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t target = targets[r];
    T* g = grad + r * grad_stride;
    if (target == ignore_index) {
      for (int64_t j = threadIdx.x; j < vocab; j += kThreads) g[j] = from_f32<T>(0.f);
      continue;
    }
    const float c = target >= 0 && target < vocab ? w * grad_loss[reduction == JK_REDUCE_NONE ? r : 0] : NAN;
    write_grad(logits + r * stride, g, vocab, lse[r], 1.f, c, target, smoothing);
  }
}

inline int blocks_for(int64_t rows) { return static_cast<int>(rows < kMaxBlocks ? rows : kMaxBlocks); }

}  // namespace loss

JK_ERROR_READER(read_error_loss)

}  // namespace jk

extern "C" int64_t jk_cross_entropy_workspace(int64_t rows) {
  return rows <= 0 ? 0 : jk::loss::blocks_for(rows) * static_cast<int64_t>(sizeof(jk::loss::Partial));
}

extern "C" int jk_cross_entropy_forward(const void* logits, int64_t logits_stride, const int64_t* targets, int64_t rows,
                                        int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                                        int reduction, float grad_scale, float* losses, float* lse, float* loss,
                                        void* grad, int64_t grad_stride, void* workspace, jk_stream_t stream) {
  using namespace jk;
  if (rows < 0 || vocab <= 0 || logits_stride < 0 || grad_stride < 0) return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype)) return JK_ERR_BAD_DTYPE;
  if (reduction < JK_REDUCE_NONE || reduction > JK_REDUCE_SUM) return JK_ERR_UNSUPPORTED_KIND;
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f)) return JK_ERR_BAD_ARG;
  if ((loss == nullptr) != (reduction == JK_REDUCE_NONE) || (grad != nullptr && reduction == JK_REDUCE_NONE))
    return JK_ERR_BAD_ARG;
  if (rows > 0 && (logits == nullptr || targets == nullptr || workspace == nullptr)) return JK_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(workspace) & 7u) != 0) return JK_ERR_ALIGNMENT;
  int st = check_device();
  if (st != JK_OK) return st;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  auto* partials = static_cast<loss::Partial*>(workspace);
  const int blocks = rows == 0 ? 0 : loss::blocks_for(rows);
  if (rows > 0) {
    JK_WITH_TYPE(dtype, T, {
      loss::forward_kernel<T><<<blocks, loss::kThreads, 0, s>>>(
          static_cast<const T*>(logits), logits_stride, targets, rows, vocab, ignore_index, label_smoothing, reduction,
          grad_scale, losses, lse, static_cast<T*>(grad), grad_stride, partials);
    });
  }
  if (loss != nullptr) loss::reduce_kernel<<<1, 32, 0, s>>>(partials, blocks, reduction, loss);
  return launch_status();
}

extern "C" int jk_cross_entropy_backward(const float* grad_loss, const void* logits, int64_t logits_stride,
                                         const int64_t* targets, const float* lse, int64_t rows, int64_t vocab, int dtype,
                                         int64_t ignore_index, float label_smoothing, int reduction, void* grad,
                                         int64_t grad_stride, jk_stream_t stream) {
  using namespace jk;
  if (rows < 0 || vocab <= 0 || logits_stride < 0 || grad_stride < 0) return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype)) return JK_ERR_BAD_DTYPE;
  if (reduction < JK_REDUCE_NONE || reduction > JK_REDUCE_SUM) return JK_ERR_UNSUPPORTED_KIND;
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f)) return JK_ERR_BAD_ARG;
  if (rows == 0) return JK_OK;
  if (grad_loss == nullptr || logits == nullptr || targets == nullptr || lse == nullptr || grad == nullptr)
    return JK_ERR_BAD_ARG;
  int st = check_device();
  if (st != JK_OK) return st;
  JK_WITH_TYPE(dtype, T, {
    loss::backward_kernel<T><<<loss::blocks_for(rows), loss::kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        grad_loss, static_cast<const T*>(logits), logits_stride, targets, lse, rows, vocab, ignore_index, label_smoothing,
        reduction, static_cast<T*>(grad), grad_stride);
  });
  return launch_status();
}
