// Layer norm of an apply step, forward and backward (jk_layer_norm_forward / _backward).
//
//   sum = x + s * delta,  mean = E[sum],  rstd = 1 / sqrt(E[(sum - mean)^2] + eps),
//   n = (sum - mean) * rstd,  y = n * weight + bias
//   u = grad_y * weight,  grad_x = rstd * (u - E[u] - n * E[u * n]) + grad_sum,  grad_delta = s * grad_x
//   grad_weight = sum_rows grad_y * n,  grad_bias = sum_rows grad_y
//
// The variance is the mean of the squared distances from the mean (two sums over the row), not
// E[sum^2] - mean^2, which cancels where the mean is large against the spread.
//
// Bound: memory, every row read once and written once. A row of up to 16384 elements stays in the
// registers of the 8 to 1024 threads that share it, each with up to 16 elements, in 16-byte packs. A
// thread keeps its columns for all rows it comes to, so the parameters and, backward, the sums of
// their gradients stay in its registers too, and the next row is on its way while one is worked on.
//
// Rows of an odd width begin anywhere within a 16-byte block, but those a multiple of 8 (16-bit) or 4
// rows apart begin alike: the rows of a group of threads are that far apart, so its packs lie on
// 16-byte boundaries all the same (SHIFTED), whole but for a row's first and last. Where the tensors
// lie differently from each other, elements are taken one by one. Longer rows are read again for
// each sum.
#include "jk_host.h"
#include "jk_rows.cuh"

namespace jk {
namespace norm {

constexpr int kMaxParts = 148 * 4;  // blocks that leave their share of the parameter gradients

struct Forward {
  const void *x, *delta;
  int64_t x_stride, delta_stride;
  float scale;
  const void *weight, *bias;
  int param_type;
  int64_t rows;
  int64_t dim;
  float eps;
  void *y, *sum;
  float *mean, *rstd;
};

struct Backward {
  const void *grad_y, *sum, *grad_sum;
  int64_t grad_y_stride, sum_stride, grad_sum_stride;
  const float *mean, *rstd;
  const void* weight;
  int param_type;
  float scale;
  int64_t rows;
  int64_t dim;
  void *grad_x, *grad_delta;
  float* parts;  // [blocks][2][dim], or null
};

__device__ __forceinline__ float param_at(const void* p, int64_t c, int type, float none) {
  if (p == nullptr) return none;
  if (type == JK_F32) return static_cast<const float*>(p)[c];
  if (type == JK_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[c]);
  return to_f32(static_cast<const __half*>(p)[c]);
}

// VEC neighbouring elements as they lie in memory: a 16-byte pack, or one.
template <typename T, int VEC>
struct Raw {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ T* elements() { return reinterpret_cast<T*>(&v); }
  __device__ __forceinline__ void floats(float (&f)[VEC]) const { unpack<T>(v, f); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) { *reinterpret_cast<uint4*>(p) = pack<T>(f); }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void clear() { v = from_f32<T>(0.f); }
  __device__ __forceinline__ T* elements() { return &v; }
  __device__ __forceinline__ void floats(float (&f)[1]) const { f[0] = to_f32(v); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};

// Threads of a block, and rows that it has at a time, with `TPR` threads to a row.
template <int TPR>
constexpr int kBlock = TPR > 256 ? TPR : (TPR > 32 ? TPR : 256);
template <int TPR>
constexpr int kGroups = kBlock<TPR> / TPR;

// The least power of two from n on.
template <int n>
constexpr int kPowerOfTwo = n <= 1 ? 1 : 2 * kPowerOfTwo<(n + 1) / 2>;

// Sums over the threads of a row, in all of them. With more than a warp to a row the row has the
// whole block; `turn` alternates, so that one barrier does.
template <int TPR, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], float (*scratch)[COUNT][32], int turn) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < COUNT; ++i) scratch[turn][i][threadIdx.x >> 5] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      v[i] = lane < TPR / 32 ? scratch[turn][i][lane] : 0.f;
#pragma unroll
      for (int o = kPowerOfTwo<TPR / 32> / 2; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      if constexpr (TPR < 1024) v[i] = __shfl_sync(0xffffffffu, v[i], 0);
    }
  }
}

// How far row r is from a 16-byte boundary, in elements, for the rows that a group of threads has.
template <typename T, bool SHIFTED>
__device__ __forceinline__ int shift_of(const T* p, int64_t r, int64_t stride) {
  return SHIFTED ? static_cast<int>(reinterpret_cast<uintptr_t>(p + r * stride) & 15) / static_cast<int>(sizeof(T)) : 0;
}

// Which of a pack's columns from c on the row has, a bit for each.
template <int VEC>
__device__ __forceinline__ uint32_t columns_of(int c, int dim) {
  const int from = min(max(-c, 0), VEC), to = min(max(dim - c, 0), VEC);
  return ((1u << to) - 1u) & ~((1u << from) - 1u);
}
template <int VEC>
constexpr uint32_t kWhole = (1u << VEC) - 1u;

// A pack at p. Columns that the row does not have are read as they come (they are another row's), but
// not past an end of the tensor (`first`, `last` row).
template <typename T, int VEC, bool SHIFTED>
__device__ __forceinline__ void load_pack(Raw<T, VEC>& raw, const T* p, uint32_t columns, bool first, bool last) {
  if (SHIFTED && ((first && !(columns & 1u)) || (last && !(columns >> (VEC - 1))))) {
    Raw<T, VEC> some;  // a rare case: in local memory, so that it takes no registers from the others
    some.clear();
#pragma unroll 1
    for (int j = 0; j < VEC; ++j)
      if ((columns >> j) & 1u) some.elements()[j] = p[j];
    raw = some;
  } else {
    raw.load(p);
  }
}

// Clears what a pack has of columns outside the row.
template <int VEC, bool SHIFTED>
__device__ __forceinline__ void clear_outside(float (&f)[VEC], uint32_t columns) {
  if (SHIFTED && columns != kWhole<VEC>) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = (columns >> j) & 1u ? f[j] : 0.f;
  }
}

// A pack's columns [0, m) or, `tail` false, its last m, in halves, quarters and one element: the pack
// lies on a 16-byte boundary, and m is less than a pack.
__device__ __forceinline__ void store_some(void* p, const uint4& u, int m, bool tail, int size) {
  char* to = static_cast<char*>(p);
  const int bytes = m * size;
  if (bytes & 8) *reinterpret_cast<uint2*>(to + (tail ? 0 : 8)) = tail ? make_uint2(u.x, u.y) : make_uint2(u.z, u.w);
  if (bytes & 4) {
    const int at = tail ? bytes & 8 : 12 - (bytes & 8);
    *reinterpret_cast<uint32_t*>(to + at) = tail ? (at == 0 ? u.x : u.z) : (at == 12 ? u.w : u.y);
  }
  if (bytes & 2) {
    const int at = tail ? bytes - 2 : 16 - bytes;
    const uint32_t low = at & 4 ? u.y : u.x, high = at & 4 ? u.w : u.z, word = at & 8 ? high : low;
    *reinterpret_cast<uint16_t*>(to + at) = static_cast<uint16_t>(at & 2 ? word >> 16 : word);
  }
}

template <typename T, int VEC, bool SHIFTED>
__device__ __forceinline__ void store_pack(T* p, uint32_t columns, const float (&f)[VEC]) {
  if (!SHIFTED || columns == kWhole<VEC>) {
    Raw<T, VEC>::store(p, f);
  } else if (columns & (1u | 1u << (VEC - 1))) {
    uint4 u;
    Raw<T, VEC>::store(reinterpret_cast<T*>(&u), f);
    store_some(p, u, __popc(columns), columns & 1u, static_cast<int>(sizeof(T)));
  } else {  // a row within a pack
    Raw<T, VEC> some;
    Raw<T, VEC>::store(some.elements(), f);
#pragma unroll 1
    for (int j = 0; j < VEC; ++j)
      if ((columns >> j) & 1u) p[j] = some.elements()[j];
  }
}

// (f - a) * b, element by element; two at a time where there are two.
template <int VEC>
__device__ __forceinline__ void centre(float (&f)[VEC], float a, float b) {
  if constexpr (VEC == 1) {
    f[0] = (f[0] - a) * b;
  } else {
    const uint64_t minus = pair(-a, -a), by = pair(b, b);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float2 v = unpair(mul2(add2(pair(f[j], f[j + 1]), minus), by));
      f[j] = v.x, f[j + 1] = v.y;
    }
  }
}

// a * b + c
template <int VEC>
__device__ __forceinline__ void multiply_add(float (&o)[VEC], const float (&a)[VEC], const float (&b)[VEC], const float (&c)[VEC]) {
  if constexpr (VEC == 1) {
    o[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float2 v = unpair(fma2(pair(a[j], a[j + 1]), pair(b[j], b[j + 1]), pair(c[j], c[j + 1])));
      o[j] = v.x, o[j + 1] = v.y;
    }
  }
}

// a * s + c, with one factor
template <int VEC>
__device__ __forceinline__ void scale_add(float (&o)[VEC], const float (&a)[VEC], float s, const float (&c)[VEC]) {
  if constexpr (VEC == 1) {
    o[0] = fmaf(a[0], s, c[0]);
  } else {
    const uint64_t by = pair(s, s);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const float2 v = unpair(fma2(pair(a[j], a[j + 1]), by, pair(c[j], c[j + 1])));
      o[j] = v.x, o[j + 1] = v.y;
    }
  }
}

// A sum in two halves, and what is added to it: f, and a * b.
struct Two {
  uint64_t v;
  __device__ __forceinline__ Two() : v(0) {}
  template <int VEC>
  __device__ __forceinline__ void add(const float (&f)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) v = add2(v, pair(f[j], VEC > 1 ? f[j + (VEC > 1)] : 0.f));
  }
  template <int VEC>
  __device__ __forceinline__ void add(const float (&a)[VEC], const float (&b)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2)
      v = fma2(pair(a[j], VEC > 1 ? a[j + (VEC > 1)] : 0.f), pair(b[j], VEC > 1 ? b[j + (VEC > 1)] : 0.f), v);
  }
  __device__ __forceinline__ float sum() const {
    const float2 f = unpair(v);
    return f.x + f.y;
  }
};

template <typename T, int VEC, int N, int TPR, bool SHIFTED, bool DELTA>
__global__ void __launch_bounds__(kBlock<TPR>, kBlock<TPR> <= 512 ? (N == 1 && TPR > 32 ? 768 : 512) / kBlock<TPR> : 1) forward_kernel(const Forward a) {
  __shared__ float scratch[2][1][32];
  const int dim = static_cast<int>(a.dim), thread = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups<TPR>;
  int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups<TPR> + threadIdx.x / TPR;
  const int first_column = thread * VEC - shift_of<T, SHIFTED>(static_cast<const T*>(a.x), r, a.x_stride);
  constexpr int kNext = TPR * VEC;  // columns from one pack of a thread to its next
  const T *x = static_cast<const T*>(a.x) + r * a.x_stride + first_column,
          *delta = static_cast<const T*>(a.delta) + (DELTA ? r * a.delta_stride + first_column : 0);
  const int64_t out = r * dim + first_column;
  T *y = static_cast<T*>(a.y) + out, *sum = a.sum == nullptr ? nullptr : static_cast<T*>(a.sum) + out;
  float w[N][VEC], b[N][VEC];
  uint32_t columns[N];
#pragma unroll
  for (int i = 0; i < N; ++i) columns[i] = columns_of<VEC>(first_column + i * kNext, dim);
  // two rows are on their way: an SM has 64 KB of loads in flight (32768 x 512 bf16 with a residual:
  // 25.2 us on the device, 26.4 with one row)
  Raw<T, VEC> next_x[N], next_d[DELTA ? N : 1], now_x[N], now_d[DELTA ? N : 1];
  const auto load = [&](int64_t r) {  // row r, at x
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (columns[i] != 0) {
        load_pack<T, VEC, SHIFTED>(next_x[i], x + i * kNext, columns[i], r == 0, r == a.rows - 1);
        if (DELTA) load_pack<T, VEC, SHIFTED>(next_d[DELTA ? i : 0], delta + i * kNext, columns[i], r == 0, r == a.rows - 1);
      }
    }
    x += step * a.x_stride;
    if (DELTA) delta += step * a.delta_stride;
  };
  const auto advance = [&] {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      now_x[i] = next_x[i];
      if (DELTA) now_d[DELTA ? i : 0] = next_d[DELTA ? i : 0];
    }
  };
  if (r < a.rows) load(r);
  advance();
  if (r + step < a.rows) load(r + step);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const bool has = (columns[i] >> j) & 1u;
      w[i][j] = has ? param_at(a.weight, first_column + i * kNext + j, a.param_type, 1.f) : 0.f;
      b[i][j] = has ? param_at(a.bias, first_column + i * kNext + j, a.param_type, 0.f) : 0.f;
    }
  const float inv = 1.f / static_cast<float>(dim);
  // all groups of a block take as many turns, as they may share a warp
  for (int64_t base = r - threadIdx.x / TPR; base < a.rows; base += step, r += step) {
    const bool here = r < a.rows;
    float f[N][VEC], s[1];
    Two total;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (here && columns[i] != 0) {
        now_x[i].floats(f[i]);
        if (DELTA) {
          float d[VEC];
          now_d[DELTA ? i : 0].floats(d);
          scale_add<VEC>(f[i], d, a.scale, f[i]);
        }
        clear_outside<VEC, SHIFTED>(f[i], columns[i]);
        total.add(f[i]);
      }
    }
    advance();
    if (r + 2 * step < a.rows) load(r + 2 * step);
    s[0] = total.sum();
    row_sums<TPR, 1>(s, scratch, 0);
    const float mu = s[0] * inv;
    Two squares;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (here && columns[i] != 0) {
        float d[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[j] = f[i][j];
        centre<VEC>(d, mu, 1.f);
        clear_outside<VEC, SHIFTED>(d, columns[i]);
        squares.add(d, d);
      }
    }
    s[0] = squares.sum();
    row_sums<TPR, 1>(s, scratch, 1);
    const float rs = rsqrtf(fmaf(s[0], inv, a.eps));
    if (here) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (columns[i] != 0) {
          float o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = f[i][j];
          centre<VEC>(o, mu, rs);
          multiply_add<VEC>(o, o, w[i], b[i]);
          store_pack<T, VEC, SHIFTED>(y + i * kNext, columns[i], o);
          if (sum != nullptr) store_pack<T, VEC, SHIFTED>(sum + i * kNext, columns[i], f[i]);
        }
      }
      if (thread == 0 && a.mean != nullptr) {
        a.mean[r] = mu;
        a.rstd[r] = rs;
      }
    }
    y += step * dim;
    if (sum != nullptr) sum += step * dim;
  }
}

// Columns that a group of threads can have.
template <int VEC, int N, int TPR>
constexpr int kColumns = N * VEC * TPR;

// The block's share of the parameter gradients: its groups' sums, which all have every column, joined
// in their order.
template <int VEC, int N, int TPR>
__device__ __forceinline__ void leave_parts(const float (&dw)[N][VEC], const float (&db)[N][VEC], int first_column, int dim,
                                            float* parts, float* shared) {
  float* mine = parts + static_cast<int64_t>(blockIdx.x) * 2 * dim;
  // shared memory [group][2][kColumns], a column's place such that neighbouring threads write neighbouring words
  const auto place = [&](int c) { return (c % VEC) * (kColumns<VEC, N, TPR> / VEC) + c / VEC; };
  float* of_group = shared + threadIdx.x / TPR * (2 * kColumns<VEC, N, TPR>);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = i * TPR * VEC + first_column + j;
      if (c >= 0 && c < dim) {
        if constexpr (kGroups<TPR> == 1) {
          mine[c] = dw[i][j];
          mine[dim + c] = db[i][j];
        } else {
          of_group[place(c)] = dw[i][j];
          of_group[kColumns<VEC, N, TPR> + place(c)] = db[i][j];
        }
      }
    }
  if constexpr (kGroups<TPR> > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * dim; c += kBlock<TPR>) {
      const float* at = shared + (c < dim ? place(c) : kColumns<VEC, N, TPR> + place(c - dim));
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups<TPR>; ++g) s += at[g * 2 * kColumns<VEC, N, TPR>];
      mine[c] = s;
    }
  }
}

template <typename T, int VEC, int N, int TPR, bool SHIFTED, bool SUM, bool PARAMS>
__global__ void __launch_bounds__(kBlock<TPR>, kBlock<TPR> <= 512 ? 512 / kBlock<TPR> : 1) backward_kernel(const Backward a) {
  __shared__ float scratch[2][2][32];
  __shared__ float shared[PARAMS && kGroups<TPR> > 1 ? kGroups<TPR> * 2 * kColumns<VEC, N, TPR> : 1];
  const int dim = static_cast<int>(a.dim), thread = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups<TPR>;
  const T *gy = static_cast<const T*>(a.grad_y), *h = static_cast<const T*>(a.sum), *gs = static_cast<const T*>(a.grad_sum);
  int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups<TPR> + threadIdx.x / TPR;
  const int first_column = thread * VEC - shift_of<T, SHIFTED>(gy, r, a.grad_y_stride);
  const auto columns = [&](int c) { return SHIFTED ? columns_of<VEC>(c, dim) : kWhole<VEC>; };
  float w[N][VEC], dw[N][VEC] = {}, db[N][VEC] = {};
  Raw<T, VEC> next_y[N], next_h[N], next_s[SUM ? N : 1];
  float next_mean = 0.f, next_rstd = 0.f;
  const auto load = [&](int64_t r) {
    next_mean = a.mean[r];
    next_rstd = a.rstd[r];
    const bool first = r == 0, last = r == a.rows - 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR * VEC + first_column;
      if (c < dim) {
        load_pack<T, VEC, SHIFTED>(next_y[i], gy + r * a.grad_y_stride + c, columns(c), first, last);
        load_pack<T, VEC, SHIFTED>(next_h[i], h + r * a.sum_stride + c, columns(c), first, last);
        if (SUM) load_pack<T, VEC, SHIFTED>(next_s[SUM ? i : 0], gs + r * a.grad_sum_stride + c, columns(c), first, last);
      }
    }
  };
  if (r < a.rows) load(r);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = i * TPR * VEC + first_column + j;
      w[i][j] = c >= 0 && c < dim ? param_at(a.weight, c, a.param_type, 1.f) : 0.f;
    }
  const float inv = 1.f / static_cast<float>(dim);
  int turn = 0;
  for (int64_t base = r - threadIdx.x / TPR; base < a.rows; base += step, r += step, turn ^= 1) {
    const bool here = r < a.rows;
    Raw<T, VEC> y[N], hh[N], ss[SUM ? N : 1];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      y[i] = next_y[i], hh[i] = next_h[i];
      if (SUM) ss[SUM ? i : 0] = next_s[SUM ? i : 0];
    }
    const float mu = next_mean, rs = next_rstd;
    if (r + step < a.rows) load(r + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR * VEC + first_column;
      if (here && c < dim) {
        float g[VEC], n[VEC];
        y[i].floats(g);
        hh[i].floats(n);
#pragma unroll
        for (int j = 0; j < VEC; ++j) n[j] = (n[j] - mu) * rs;
        clear_outside<VEC, SHIFTED>(g, columns(c));
        clear_outside<VEC, SHIFTED>(n, columns(c));  // another row's may be infinite, or be so against this row's mean
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float u = g[j] * w[i][j];
          s[0] += u;
          s[1] = fmaf(u, n[j], s[1]);
          if (PARAMS) {
            dw[i][j] = fmaf(g[j], n[j], dw[i][j]);
            db[i][j] += g[j];
          }
        }
      }
    }
    row_sums<TPR, 2>(s, scratch, turn);
    if (!here) continue;
    const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR * VEC + first_column;
      if (c < dim) {
        float g[VEC], n[VEC], o[VEC], q[VEC];
        y[i].floats(g);
        hh[i].floats(n);
        if (SUM) ss[SUM ? i : 0].floats(q);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          n[j] = (n[j] - mu) * rs;
          o[j] = fmaf(g[j], w[i][j], -fmaf(n[j], c1, c0));
          o[j] = SUM ? fmaf(rs, o[j], q[j]) : rs * o[j];
        }
        store_pack<T, VEC, SHIFTED>(static_cast<T*>(a.grad_x) + r * dim + c, columns(c), o);
        if (a.grad_delta != nullptr) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] *= a.scale;
          store_pack<T, VEC, SHIFTED>(static_cast<T*>(a.grad_delta) + r * dim + c, columns(c), o);
        }
      }
    }
  }
  if constexpr (PARAMS) {
    grid_dependency_launch();
    leave_parts<VEC, N, TPR>(dw, db, first_column, dim, a.parts, shared);
  }
}

// ---------------------------------------------------------------- rows of any length
constexpr int kLongThreads = 512;

__device__ __forceinline__ float long_sum(float v, float* scratch) {
  v = warp_sum32(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum32((threadIdx.x & 31) < kLongThreads / 32 ? scratch[threadIdx.x & 31] : 0.f);
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) long_forward_kernel(const Forward a) {
  __shared__ float scratch[kLongThreads / 32];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* d = a.delta == nullptr ? nullptr : static_cast<const T*>(a.delta) + r * a.delta_stride;
    const auto at = [&](int64_t c) { return d == nullptr ? to_f32(x[c]) : fmaf(a.scale, to_f32(d[c]), to_f32(x[c])); };
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < a.dim; c += kLongThreads) s += at(c);
    const float mu = long_sum(s, scratch) / static_cast<float>(a.dim);
    s = 0.f;
    for (int64_t c = threadIdx.x; c < a.dim; c += kLongThreads) {
      const float v = at(c) - mu;
      s = fmaf(v, v, s);
    }
    const float rs = rsqrtf(long_sum(s, scratch) / static_cast<float>(a.dim) + a.eps);
    for (int64_t c = threadIdx.x; c < a.dim; c += kLongThreads) {
      const float v = at(c);
      static_cast<T*>(a.y)[r * a.dim + c] =
          from_f32<T>(fmaf((v - mu) * rs, param_at(a.weight, c, a.param_type, 1.f), param_at(a.bias, c, a.param_type, 0.f)));
      if (a.sum != nullptr) static_cast<T*>(a.sum)[r * a.dim + c] = from_f32<T>(v);
    }
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[r] = mu;
      a.rstd[r] = rs;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) long_backward_kernel(const Backward a) {
  __shared__ float scratch[kLongThreads / 32];
  float* part = a.parts == nullptr ? nullptr : a.parts + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* gy = static_cast<const T*>(a.grad_y) + r * a.grad_y_stride;
    const T* h = static_cast<const T*>(a.sum) + r * a.sum_stride;
    const float mu = a.mean[r], rs = a.rstd[r];
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < a.dim; c += kLongThreads) {
      const float g = to_f32(gy[c]), n = (to_f32(h[c]) - mu) * rs, u = g * param_at(a.weight, c, a.param_type, 1.f);
      s0 += u;
      s1 = fmaf(u, n, s1);
      if (part != nullptr) {  // a column is always the same thread's
        part[c] = r == blockIdx.x ? g * n : fmaf(g, n, part[c]);
        part[a.dim + c] = r == blockIdx.x ? g : part[a.dim + c] + g;
      }
    }
    s0 = long_sum(s0, scratch) / static_cast<float>(a.dim);
    s1 = long_sum(s1, scratch) / static_cast<float>(a.dim);
    for (int64_t c = threadIdx.x; c < a.dim; c += kLongThreads) {
      const float n = (to_f32(h[c]) - mu) * rs;
      float d = rs * (to_f32(gy[c]) * param_at(a.weight, c, a.param_type, 1.f) - s0 - n * s1);
      if (a.grad_sum != nullptr) d += to_f32(static_cast<const T*>(a.grad_sum)[r * a.grad_sum_stride + c]);
      static_cast<T*>(a.grad_x)[r * a.dim + c] = from_f32<T>(d);
      if (a.grad_delta != nullptr) static_cast<T*>(a.grad_delta)[r * a.dim + c] = from_f32<T>(a.scale * d);
    }
  }
}

// ---------------------------------------------------------------- parameter gradients
// 32 columns to a block, 32 threads to a column; the blocks' shares are added in a fixed order.
template <typename W>
__global__ void __launch_bounds__(1024) parameters_kernel(const float* parts, int count, int64_t dim, W* grad_weight, W* grad_bias) {
  __shared__ float sums[32][33];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;
  const int slice = threadIdx.x / 32;
  grid_dependency_wait();
  float s = 0.f;
  if (c < 2 * dim)
    for (int i = slice; i < count; i += 32) s += parts[static_cast<int64_t>(i) * 2 * dim + c];
  sums[slice][threadIdx.x % 32] = s;
  __syncthreads();
  s = warp_sum32(sums[threadIdx.x % 32][slice]);  // thread (slice, lane) now has column `slice`
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * 32 + slice;
  if (threadIdx.x % 32 != 0 || mine >= 2 * dim) return;
  if (mine < dim)
    grad_weight[mine] = from_f32<W>(s);
  else
    grad_bias[mine - dim] = from_f32<W>(s);
}

// ---------------------------------------------------------------- launches
inline int64_t groups_to_blocks(int64_t rows, int groups, int64_t most) {
  const int64_t want = (rows + groups - 1) / groups;
  return want < most ? want : most;
}

// Blocks of a kernel that an SM holds, asked for once (the devices are alike).
template <auto KERNEL>
int blocks_per_sm(int threads) {
  static const int per_sm = [threads] {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    return n;
  }();
  return per_sm;
}

// Rows of one group are `step` apart; with SHIFTED they have to begin alike against 16-byte blocks, so
// the step is a multiple of what a block has elements, or a group has one row only.
template <int VEC, int TPR, bool SHIFTED>
int64_t blocks_of(int64_t rows, int64_t most) {
  const int64_t blocks = groups_to_blocks(rows, kGroups<TPR>, most);
  if (!SHIFTED || blocks * kGroups<TPR> >= rows) return blocks;
  constexpr int64_t kUnit = kGroups<TPR> % VEC == 0 ? 1 : VEC / kGroups<TPR>;  // groups: 1, or 8 and more
  return blocks / kUnit * kUnit;
}

template <auto KERNEL, int VEC, int TPR, bool SHIFTED>
int run_forward(const Forward& a, cudaStream_t s) {
  const int64_t blocks = blocks_of<VEC, TPR, SHIFTED>(a.rows, 148ll * blocks_per_sm<KERNEL>(kBlock<TPR>));
  KERNEL<<<static_cast<unsigned>(blocks), kBlock<TPR>, 0, s>>>(a);
  return 0;
}

template <typename T, int VEC, bool SHIFTED, int N, int TPR>
int pick_forward(const Forward& a, cudaStream_t s) {
  return a.delta != nullptr ? run_forward<forward_kernel<T, VEC, N, TPR, SHIFTED, true>, VEC, TPR, SHIFTED>(a, s)
                            : run_forward<forward_kernel<T, VEC, N, TPR, SHIFTED, false>, VEC, TPR, SHIFTED>(a, s);
}

template <auto KERNEL, int VEC, int TPR, bool SHIFTED>
int run_backward(const Backward& a, cudaStream_t s) {
  int64_t most = 148ll * blocks_per_sm<KERNEL>(kBlock<TPR>);
  const int64_t parts = kBlock<TPR> <= 128 ? kMaxParts : kBlock<TPR> <= 256 ? kMaxParts / 4 * 3 : kMaxParts / 2;
  if (a.parts != nullptr && most > parts) most = parts;
  const int blocks = static_cast<int>(blocks_of<VEC, TPR, SHIFTED>(a.rows, most));
  KERNEL<<<blocks, kBlock<TPR>, 0, s>>>(a);
  return blocks;
}

template <typename T, int VEC, bool SHIFTED, int N, int TPR>
int pick_backward(const Backward& a, cudaStream_t s) {
  if (a.grad_sum != nullptr)
    return a.parts != nullptr ? run_backward<backward_kernel<T, VEC, N, TPR, SHIFTED, true, true>, VEC, TPR, SHIFTED>(a, s)
                              : run_backward<backward_kernel<T, VEC, N, TPR, SHIFTED, true, false>, VEC, TPR, SHIFTED>(a, s);
  return a.parts != nullptr ? run_backward<backward_kernel<T, VEC, N, TPR, SHIFTED, false, true>, VEC, TPR, SHIFTED>(a, s)
                            : run_backward<backward_kernel<T, VEC, N, TPR, SHIFTED, false, false>, VEC, TPR, SHIFTED>(a, s);
}

// The threads of a row and their turns: a warp or less as long as 16 elements a thread do, so that no
// barrier is needed; beyond, 8 to 16 elements of a 16-byte pack or two each, which leaves an SM 512
// threads or more. Four packs to fewer threads are no better (us a call, forward and backward; f32,
// 8192 x 2048: 25.5 and 42.1 with two, 23.5 and 43.6 with four; 8192 x 2047: 59.9 and 63.9, either way).
// Rows of 4097 to 5113 16-bit elements that begin anywhere take one pack of 640 threads (3000 x 4501
// f16: 29.2 and 39.5, 31.2 and 41.6 with two of 384), those that begin on a 16-byte boundary two
// (3000 x 4608 f16: 23.0 and 30.7, 23.0 and 31.7 with one of 640); above, one pack is slower for both
// (3000 x 6001 f16: 31.2 and 47.7 with two, 32.8 and 48.2 with one of 768).
#define JK_NORM_SHAPES(RUN)                                             \
  if constexpr (VEC == 8) {                                             \
    if (turns <= 8) return RUN(1, 8);                                   \
    if (turns <= 16) return RUN(1, 16);                                 \
    if (turns <= 32) return RUN(1, 32);                                 \
    if (turns <= 64) return RUN(2, 32);                                 \
    if (turns <= 128) return RUN(1, 128);                               \
    if (turns <= 256) return RUN(2, 128);                               \
    if (turns <= 512) return RUN(2, 256);                               \
    if constexpr (SHIFTED) {                                            \
      if (turns <= 640) return RUN(1, 640);                             \
    }                                                                   \
    if (turns <= 768) return RUN(2, 384);                               \
    if (turns <= 1024) return RUN(2, 512);                              \
    return RUN(2, 1024);                                                \
  } else if constexpr (VEC == 4) {                                      \
    if (turns <= 8) return RUN(1, 8);                                   \
    if (turns <= 16) return RUN(1, 16);                                 \
    if (turns <= 32) return RUN(1, 32);                                 \
    if (turns <= 64) return RUN(2, 32);                                 \
    if (turns <= 128) return RUN(4, 32);                                \
    if (turns <= 256) return RUN(2, 128);                               \
    if (turns <= 512) return RUN(2, 256);                               \
    if (turns <= 768) return RUN(2, 384);                               \
    if (turns <= 1024) return RUN(2, 512);                              \
    if (turns <= 1536) return RUN(2, 768);                              \
    if (turns <= 2048) return RUN(2, 1024);                             \
    return RUN(4, 1024);                                                \
  } else {                                                              \
    if (turns <= 128) return RUN(4, 32);                                \
    if (turns <= 512) return RUN(16, 32);                               \
    if (turns <= 2048) return RUN(16, 128);                             \
    if (turns <= 4096) return RUN(16, 256);                             \
    if (turns <= 8192) return RUN(16, 512);                             \
    return RUN(16, 1024);                                               \
  }

// Whether rows stay in registers: 16384 elements, with room for a start within a pack.
template <typename T>
bool in_registers(int64_t dim) {
  return dim + (dim % kPack<T> != 0 ? kPack<T> : 0) <= 16384;
}

template <typename T, int VEC, bool SHIFTED>
int shape_forward(const Forward& a, cudaStream_t s) {
  const int64_t turns = (a.dim + (SHIFTED ? 2 : 1) * (VEC - 1)) / VEC;
#define JK_RUN(N, TPR) pick_forward<T, VEC, SHIFTED, N, TPR>(a, s)
  JK_NORM_SHAPES(JK_RUN)
#undef JK_RUN
}

template <typename T, int VEC, bool SHIFTED>
int shape_backward(const Backward& a, cudaStream_t s) {
  const int64_t turns = (a.dim + (SHIFTED ? 2 : 1) * (VEC - 1)) / VEC;
#define JK_RUN(N, TPR) pick_backward<T, VEC, SHIFTED, N, TPR>(a, s)
  JK_NORM_SHAPES(JK_RUN)
#undef JK_RUN
}

// Whether a tensor's rows can be taken in packs: they begin where those of a contiguous one on a 16-byte
// boundary do and, where packs hold parts of two rows, only the first and the last row's packs reach past
// the tensor (an earlier row's would where the rows after it are no longer than what it reaches).
template <typename T>
bool lies_plain(const void* p, int64_t stride, int64_t dim) {
  return p == nullptr || (aligned16(p) && (stride - dim) % kPack<T> == 0 && (dim % kPack<T> == 0 || stride >= kPack<T> - 1));
}

template <typename T>
void forward(const Forward& a, cudaStream_t s) {
  if (!in_registers<T>(a.dim)) {
    long_forward_kernel<T><<<static_cast<unsigned>(a.rows < 148 * 4 ? a.rows : 148 * 4), kLongThreads, 0, s>>>(a);
  } else if (lies_plain<T>(a.x, a.x_stride, a.dim) && lies_plain<T>(a.delta, a.delta_stride, a.dim) && aligned16(a.y) &&
             aligned16(a.sum)) {
    if (a.dim % kPack<T> == 0) shape_forward<T, kPack<T>, false>(a, s);
    else shape_forward<T, kPack<T>, true>(a, s);
  } else {
    shape_forward<T, 1, false>(a, s);
  }
}

// Returns the blocks that left a share of the parameter gradients.
template <typename T>
int backward(const Backward& a, cudaStream_t s) {
  if (!in_registers<T>(a.dim)) {
    const int blocks = static_cast<int>(a.rows < kMaxParts ? a.rows : kMaxParts);
    long_backward_kernel<T><<<blocks, kLongThreads, 0, s>>>(a);
    return blocks;
  }
  if (lies_plain<T>(a.grad_y, a.grad_y_stride, a.dim) && lies_plain<T>(a.sum, a.sum_stride, a.dim) &&
      lies_plain<T>(a.grad_sum, a.grad_sum_stride, a.dim) && aligned16(a.grad_x) && aligned16(a.grad_delta))
    return a.dim % kPack<T> == 0 ? shape_backward<T, kPack<T>, false>(a, s) : shape_backward<T, kPack<T>, true>(a, s);
  return shape_backward<T, 1, false>(a, s);
}

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
  const norm::Forward a{x, delta, x_stride, delta_stride, delta_scale, weight, bias, param_dtype,
                        rows, dim, eps, y, sum, mean, rstd};
  JK_WITH_TYPE(dtype, T, norm::forward<T>(a, reinterpret_cast<cudaStream_t>(stream)));
  return launch_status();
}

extern "C" int64_t jk_layer_norm_backward_workspace(int64_t rows, int64_t dim) {
  return rows <= 0 || dim <= 0 ? 0 : 2 * dim * (rows < jk::norm::kMaxParts ? rows : jk::norm::kMaxParts);
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
  const norm::Backward a{grad_y, sum, grad_sum, grad_y_stride, sum_stride, grad_sum_stride, mean, rstd, weight, param_dtype,
                         delta_scale, rows, dim, grad_x, grad_delta, params ? workspace : nullptr};
  int parts = 0;
  if (rows > 0) JK_WITH_TYPE(dtype, T, parts = norm::backward<T>(a, s));
  if (params)
    JK_WITH_TYPE(param_dtype, W, launch_dependent(norm::parameters_kernel<W>, static_cast<unsigned>((2 * dim + 31) / 32), 1024, 0, s,
                                                  workspace, parts, dim, static_cast<W*>(grad_weight), static_cast<W*>(grad_bias)));
  return launch_status();
}
