// Layer norm of an apply step, forward and backward (jk_layer_norm_forward / _backward).
//
//   sum = x + s * delta,  mean = E[sum],  rstd = 1 / sqrt(E[(sum - mean)^2] + eps),
//   n = (sum - mean) * rstd,  y = n * weight + bias
//   u = grad_y * weight,  grad_x = rstd * (u - E[u] - n * E[u * n]) + grad_sum,  grad_delta = s * grad_x
//   grad_weight = sum_rows grad_y * n,  grad_bias = sum_rows grad_y
//
// The variance is the mean of the squared distances from the mean (two sums over the row), not
// E[sum^2] - mean^2, which cancels where the mean is large against the spread.
#include "jk_host.h"
#include "jk_rows.cuh"

namespace jk {
namespace norm {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 148 * 4;

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = warp_sum32(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < kThreads / 32; ++i) v += scratch[i];
  __syncthreads();
  return v;
}

template <typename T>
__device__ __forceinline__ float sum_at(const T* x, const T* delta, float scale, int64_t c) {
  const float v = to_f32(x[c]);
  return delta == nullptr ? v : fmaf(scale, to_f32(delta[c]), v);
}

// One block per row, the row read three times.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads)
    forward_kernel(const T* x, int64_t x_stride, const T* delta, int64_t delta_stride, float scale, const W* weight,
                   const W* bias, int64_t rows, int64_t dim, float eps, T* y, T* sum, float* mean, float* rstd) {
  __shared__ float scratch[kThreads / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    const T* dr = delta == nullptr ? nullptr : delta + r * delta_stride;
    float a = 0.f;
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) a += sum_at(xr, dr, scale, c);
    const float mu = block_sum(a, scratch) / static_cast<float>(dim);
    a = 0.f;
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
      const float d = sum_at(xr, dr, scale, c) - mu;
      a = fmaf(d, d, a);
    }
    const float rs = rsqrtf(block_sum(a, scratch) / static_cast<float>(dim) + eps);
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
      const float h = sum_at(xr, dr, scale, c);
      const float n = (h - mu) * rs;
      const float w = weight == nullptr ? 1.f : to_f32(weight[c]), b = bias == nullptr ? 0.f : to_f32(bias[c]);
      y[r * dim + c] = from_f32<T>(fmaf(n, w, b));
      if (sum != nullptr) sum[r * dim + c] = from_f32<T>(h);
    }
    if (threadIdx.x == 0 && mean != nullptr) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

// One block per row at a time; the block's share of the parameter gradients goes to its own
// part of the workspace [blocks][2][dim], each column by one thread.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads)
    backward_kernel(const T* grad_y, int64_t gy_stride, const T* sum, int64_t sum_stride, const float* mean,
                    const float* rstd, const W* weight, const T* grad_sum, int64_t gs_stride, float scale, int64_t rows,
                    int64_t dim, T* grad_x, T* grad_delta, float* workspace) {
  __shared__ float scratch[kThreads / 32];
  float* part = workspace == nullptr ? nullptr : workspace + static_cast<int64_t>(blockIdx.x) * 2 * dim;
  if (part != nullptr)
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) part[c] = part[dim + c] = 0.f;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* gy = grad_y + r * gy_stride;
    const T* h = sum + r * sum_stride;
    const float mu = mean[r], rs = rstd[r];
    float a = 0.f, b = 0.f;
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
      const float g = to_f32(gy[c]), n = (to_f32(h[c]) - mu) * rs;
      const float u = weight == nullptr ? g : g * to_f32(weight[c]);
      a += u;
      b = fmaf(u, n, b);
      if (part != nullptr) {
        part[c] = fmaf(g, n, part[c]);
        part[dim + c] += g;
      }
    }
    a = block_sum(a, scratch) / static_cast<float>(dim);
    b = block_sum(b, scratch) / static_cast<float>(dim);
    for (int64_t c = threadIdx.x; c < dim; c += kThreads) {
      const float g = to_f32(gy[c]), n = (to_f32(h[c]) - mu) * rs;
      const float u = weight == nullptr ? g : g * to_f32(weight[c]);
      float d = rs * (u - a - n * b);
      if (grad_sum != nullptr) d += to_f32(grad_sum[r * gs_stride + c]);
      grad_x[r * dim + c] = from_f32<T>(d);
      if (grad_delta != nullptr) grad_delta[r * dim + c] = from_f32<T>(scale * d);
    }
  }
}

template <typename W>
__global__ void __launch_bounds__(kThreads)
    parameters_kernel(const float* workspace, int blocks, int64_t dim, W* grad_weight, W* grad_bias) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= 2 * dim) return;
  float a = 0.f;
  for (int i = 0; i < blocks; ++i) a += workspace[static_cast<int64_t>(i) * 2 * dim + c];
  if (c < dim)
    grad_weight[c] = from_f32<W>(a);
  else
    grad_bias[c - dim] = from_f32<W>(a);
}

inline int blocks_for(int64_t rows) { return static_cast<int>(rows < kMaxBlocks ? rows : kMaxBlocks); }

}  // namespace norm
}  // namespace jk

extern "C" int jk_layer_norm_forward(const void* x, int64_t x_stride, const void* delta, int64_t delta_stride,
                                     float delta_scale, const void* weight, const void* bias, int param_dtype,
                                     int64_t rows, int64_t dim, int dtype, float eps, void* y, void* sum, float* mean,
                                     float* rstd, jk_stream_t stream) {
  using namespace jk;
  if (rows < 0 || dim <= 0 || x_stride < 0 || delta_stride < 0) return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype) || !float_dtype(param_dtype)) return JK_ERR_BAD_DTYPE;
  if (rows == 0) return JK_OK;
  if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) return JK_ERR_BAD_ARG;
  int st = check_device();
  if (st != JK_OK) return st;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  JK_WITH_TYPE(dtype, T, JK_WITH_TYPE(param_dtype, W, {
    norm::forward_kernel<T, W><<<norm::blocks_for(rows), norm::kThreads, 0, s>>>(
        static_cast<const T*>(x), x_stride, static_cast<const T*>(delta), delta_stride, delta_scale,
        static_cast<const W*>(weight), static_cast<const W*>(bias), rows, dim, eps, static_cast<T*>(y),
        static_cast<T*>(sum), mean, rstd);
  }));
  return launch_status();
}

extern "C" int64_t jk_layer_norm_backward_workspace(int64_t rows, int64_t dim) {
  return rows <= 0 || dim <= 0 ? 0 : 2 * dim * jk::norm::blocks_for(rows);
}

extern "C" int jk_layer_norm_backward(const void* grad_y, int64_t grad_y_stride, const void* sum, int64_t sum_stride,
                                      const float* mean, const float* rstd, const void* weight, int param_dtype,
                                      const void* grad_sum, int64_t grad_sum_stride, float delta_scale, int64_t rows,
                                      int64_t dim, int dtype, void* grad_x, void* grad_delta, void* grad_weight,
                                      void* grad_bias, float* workspace, jk_stream_t stream) {
  using namespace jk;
  if (rows < 0 || dim <= 0 || grad_y_stride < 0 || sum_stride < 0 || grad_sum_stride < 0) return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype) || !float_dtype(param_dtype)) return JK_ERR_BAD_DTYPE;
  const bool params = grad_weight != nullptr;
  if (params != (grad_bias != nullptr)) return JK_ERR_BAD_ARG;
  if (rows > 0 && (grad_y == nullptr || sum == nullptr || mean == nullptr || rstd == nullptr || grad_x == nullptr ||
                   (params && workspace == nullptr)))
    return JK_ERR_BAD_ARG;
  if (params && !aligned16(workspace)) return JK_ERR_ALIGNMENT;
  int st = check_device();
  if (st != JK_OK) return st;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const int blocks = rows == 0 ? 0 : norm::blocks_for(rows);
  JK_WITH_TYPE(param_dtype, W, {
    if (rows > 0) {
      JK_WITH_TYPE(dtype, T, {
        norm::backward_kernel<T, W><<<blocks, norm::kThreads, 0, s>>>(
            static_cast<const T*>(grad_y), grad_y_stride, static_cast<const T*>(sum), sum_stride, mean, rstd,
            static_cast<const W*>(weight), static_cast<const T*>(grad_sum), grad_sum_stride, delta_scale, rows, dim,
            static_cast<T*>(grad_x), static_cast<T*>(grad_delta), params ? workspace : nullptr);
      });
    }
    if (params)
      norm::parameters_kernel<W><<<static_cast<unsigned>((2 * dim + norm::kThreads - 1) / norm::kThreads), norm::kThreads, 0,
                                   s>>>(workspace, blocks, dim, static_cast<W*>(grad_weight),
                                        static_cast<W*>(grad_bias));
  });
  return launch_status();
}
