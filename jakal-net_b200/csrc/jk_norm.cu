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
// registers of the 8 to 1024 threads that share it, each with up to 16 elements; a thread keeps its
// columns for all rows it comes to, so the parameters and, backward, the sums of their gradients stay
// in its registers too. Three forms:
//   * forward_kernel, backward_kernel: rows that lie in 16-byte packs, a pack at a time, the next row
//     on its way in registers while one is worked on;
//   * staged_forward_kernel, staged_backward_kernel: rows that do not (an odd width, an odd offset).
//     One warp has tiles of rows copied to shared memory as they lie, in 16-byte blocks, tiles ahead;
//     the others take their elements from there one by one, whatever their alignment;
//   * long_*: longer rows, read again for each sum.
#include "jk_host.h"
#include "jk_rows.cuh"
#include "jk_sm100.cuh"

namespace jk {
namespace norm {

constexpr int kMaxParts = 148 * 2;  // blocks that leave their share of the parameter gradients

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
  __device__ __forceinline__ void floats(float (&f)[VEC]) const { unpack<T>(v, f); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) { *reinterpret_cast<uint4*>(p) = pack<T>(f); }
};
// Threads of a block, and rows that it has at a time, with `TPR` threads to a row.
template <int TPR>
constexpr int kBlock = TPR > 256 ? TPR : (TPR > 32 ? TPR : 256);
template <int TPR>
constexpr int kGroups = kBlock<TPR> / TPR;

// Sums over the threads of a row, in all of them. With more than a warp to a row the row has the
// whole block; `turn` alternates, so that one barrier does.
template <int TPR, int COUNT, bool STAGED = false>
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
    if constexpr (STAGED)
      asm volatile("bar.sync 1, %0;" ::"n"(TPR) : "memory");  // not the loading warp
    else
      __syncthreads();
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      v[i] = lane < TPR / 32 ? scratch[turn][i][lane] : 0.f;
#pragma unroll
      for (int o = TPR / 64; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      if constexpr (TPR < 1024) v[i] = __shfl_sync(0xffffffffu, v[i], 0);
    }
  }
}

template <typename T, int VEC, int N, int TPR, bool DELTA>
__global__ void __launch_bounds__(kBlock<TPR>) forward_kernel(const Forward a) {
  __shared__ float scratch[2][1][32];
  const int dim = static_cast<int>(a.dim), thread = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups<TPR>;
  const T *x = static_cast<const T*>(a.x), *delta = static_cast<const T*>(a.delta);
  float w[N][VEC], b[N][VEC];
  Raw<T, VEC> next_x[N], next_d[DELTA ? N : 1];
  const auto load = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + thread) * VEC;
      if (c < dim) {
        next_x[i].load(x + r * a.x_stride + c);
        if (DELTA) next_d[DELTA ? i : 0].load(delta + r * a.delta_stride + c);
      }
    }
  };
  int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups<TPR> + threadIdx.x / TPR;
  if (r < a.rows) load(r);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (i * TPR + thread) * VEC + j;
      w[i][j] = c < dim ? param_at(a.weight, c, a.param_type, 1.f) : 0.f;
      b[i][j] = c < dim ? param_at(a.bias, c, a.param_type, 0.f) : 0.f;
    }
  const float inv = 1.f / static_cast<float>(dim);
  // all groups of a block take as many turns, as they may share a warp
  for (int64_t base = r - threadIdx.x / TPR; base < a.rows; base += step, r += step) {
    const bool here = r < a.rows;
    float f[N][VEC], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + thread) * VEC;
      if (here && c < dim) {
        next_x[i].floats(f[i]);
        if (DELTA) {
          float d[VEC];
          next_d[DELTA ? i : 0].floats(d);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[i][j] = fmaf(a.scale, d[j], f[i][j]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[0] += f[i][j];
      }
    }
    if (r + step < a.rows) load(r + step);
    row_sums<TPR, 1>(s, scratch, 0);
    const float mu = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + thread) * VEC;
      if (here && c < dim) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = f[i][j] - mu;
          s[0] = fmaf(d, d, s[0]);
        }
      }
    }
    row_sums<TPR, 1>(s, scratch, 1);
    const float rs = rsqrtf(fmaf(s[0], inv, a.eps));
    if (!here) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + thread) * VEC;
      if (c < dim) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = fmaf((f[i][j] - mu) * rs, w[i][j], b[i][j]);
        Raw<T, VEC>::store(static_cast<T*>(a.y) + r * dim + c, o);
        if (a.sum != nullptr) Raw<T, VEC>::store(static_cast<T*>(a.sum) + r * dim + c, f[i]);
      }
    }
    if (thread == 0 && a.mean != nullptr) {
      a.mean[r] = mu;
      a.rstd[r] = rs;
    }
  }
}

// The block's share of the parameter gradients: the groups' sums joined, in their order.
template <int VEC, int N, int TPR, bool STAGED = false>
__device__ __forceinline__ void leave_parts(float (&dw)[N][VEC], float (&db)[N][VEC], int dim, float* parts, float* shared) {
  const int thread = threadIdx.x % TPR;
  float* mine = parts + static_cast<int64_t>(blockIdx.x) * 2 * dim;
  if constexpr (TPR < 32) {  // the groups of a warp
#pragma unroll
    for (int o = 16; o >= TPR; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          dw[i][j] += __shfl_xor_sync(0xffffffffu, dw[i][j], o);
          db[i][j] += __shfl_xor_sync(0xffffffffu, db[i][j], o);
        }
  }
  constexpr int kShare = TPR <= 32 ? kBlock<TPR> / 32 : 1;  // warps that have the same columns
  const bool speaks = TPR >= 32 || (threadIdx.x & 31) < TPR;
  for (int g = 0; g < kShare; ++g) {
    if (speaks && (kShare == 1 || static_cast<int>(threadIdx.x >> 5) == g)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int c = (i * TPR + thread) * VEC + j;
          if (c < dim) {
            if (kShare == 1) {
              mine[c] = dw[i][j];
              mine[dim + c] = db[i][j];
            } else {
              // an element's place: its turn, its place in the pack, its thread; neighbouring threads, neighbouring words
              float* at = shared + ((i * VEC + j) * TPR + thread) * 2;
              const float2 before = g == 0 ? make_float2(0.f, 0.f) : *reinterpret_cast<float2*>(at);
              const float2 now = make_float2(before.x + dw[i][j], before.y + db[i][j]);
              if (g == kShare - 1) {
                mine[c] = now.x;
                mine[dim + c] = now.y;
              } else {
                *reinterpret_cast<float2*>(at) = now;
              }
            }
          }
        }
    }
    if constexpr (kShare > 1) {
      if constexpr (STAGED)
        asm volatile("bar.sync 1, %0;" ::"n"(kBlock<TPR>) : "memory");
      else
        __syncthreads();
    }
  }
}

template <typename T, int VEC, int N, int TPR, bool SUM, bool PARAMS>
__global__ void __launch_bounds__(kBlock<TPR>, kBlock<TPR> <= 512 ? 512 / kBlock<TPR> : 1) backward_kernel(const Backward a) {
  __shared__ float scratch[2][2][32];
  constexpr bool kShared = PARAMS && TPR <= 32;
  __shared__ float shared[kShared ? N * VEC * TPR * 2 : 1];
  const int dim = static_cast<int>(a.dim), thread = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups<TPR>;
  const T *gy = static_cast<const T*>(a.grad_y), *h = static_cast<const T*>(a.sum), *gs = static_cast<const T*>(a.grad_sum);
  float w[N][VEC], dw[N][VEC] = {}, db[N][VEC] = {};
  Raw<T, VEC> next_y[N], next_h[N], next_s[SUM ? N : 1];
  float next_mean = 0.f, next_rstd = 0.f;
  const auto load = [&](int64_t r) {
    next_mean = a.mean[r];
    next_rstd = a.rstd[r];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * TPR + thread) * VEC;
      if (c < dim) {
        next_y[i].load(gy + r * a.grad_y_stride + c);
        next_h[i].load(h + r * a.sum_stride + c);
        if (SUM) next_s[SUM ? i : 0].load(gs + r * a.grad_sum_stride + c);
      }
    }
  };
  int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups<TPR> + threadIdx.x / TPR;
  if (r < a.rows) load(r);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (i * TPR + thread) * VEC + j;
      w[i][j] = c < dim ? param_at(a.weight, c, a.param_type, 1.f) : 0.f;
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
      const int c = (i * TPR + thread) * VEC;
      if (here && c < dim) {
        float g[VEC], n[VEC];
        y[i].floats(g);
        hh[i].floats(n);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          n[j] = (n[j] - mu) * rs;
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
      const int c = (i * TPR + thread) * VEC;
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
        Raw<T, VEC>::store(static_cast<T*>(a.grad_x) + r * dim + c, o);
        if (a.grad_delta != nullptr) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] *= a.scale;
          Raw<T, VEC>::store(static_cast<T*>(a.grad_delta) + r * dim + c, o);
        }
      }
    }
  }
  if constexpr (PARAMS) {
    grid_dependency_launch();
    leave_parts<VEC, N, TPR>(dw, db, dim, a.parts, shared);
  }
}

// ---------------------------------------------------------------- rows off 16-byte boundaries
constexpr int kMaxFeeds = 5;
constexpr int kMaxStages = 8;
constexpr int kMaxTileRows = 128;

// An input as the loading warp sees it: rows of bytes, `stride` apart. Rows without a gap are copied
// as one piece, others one by one, each to a place `pitch` after the one before.
struct Feed {
  const char* p;
  int64_t stride;
  int row_bytes;
  uint32_t offset;  // in a stage
  int pitch;        // 0: one piece
};

struct Plan {
  Feed feed[kMaxFeeds];
  int feeds, tile_rows, stages;
  uint32_t stage_bytes;
};

// Where row `i` of the tile that begins at row r0 lies in a stage.
__device__ __forceinline__ const char* staged(const Feed& f, const unsigned char* stage, int64_t r0, int i) {
  const uint32_t first = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(f.p) + r0 * f.stride) & 15u;
  const uint32_t at = f.pitch == 0 ? first + i * f.row_bytes
                                   : i * f.pitch + (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(f.p) + (r0 + i) * f.stride) & 15u);
  return reinterpret_cast<const char*>(stage) + f.offset + at;
}

// Bytes [from, to) of an input into shared memory at `dst` (which stands for the 16-byte block that
// `from` lies in). Whole blocks by one bulk copy; where the first or the last block reaches outside
// the input, its bytes one element's half or whole at a time, before the copies are announced.
// Returns the bytes of the bulk copy.
__device__ __forceinline__ uint32_t copy_piece(const Feed& f, int64_t rows, const char* from, const char* to, unsigned char* dst,
                                               bool issue, uint64_t* bar) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(from), end = reinterpret_cast<uintptr_t>(to);
  const uintptr_t low = begin & ~uintptr_t(15);
  uintptr_t a = low, b = (end + 15) & ~uintptr_t(15);
  if (a < reinterpret_cast<uintptr_t>(f.p)) a += 16;
  if (b > reinterpret_cast<uintptr_t>(f.p) + (rows - 1) * f.stride + f.row_bytes) b -= 16;
  if (b < a) b = a;  // nothing but ends
  if (!issue) {
    const uintptr_t head = a < end ? a : end, tail = b > head ? b : head;
    for (uintptr_t p = begin; p < head; p += 2) *reinterpret_cast<uint16_t*>(dst + (p - low)) = *reinterpret_cast<const uint16_t*>(p);
    for (uintptr_t p = tail; p < end; p += 2) *reinterpret_cast<uint16_t*>(dst + (p - low)) = *reinterpret_cast<const uint16_t*>(p);
  } else if (b > a) {
    bulk_load(dst + (a - low), reinterpret_cast<const void*>(a), static_cast<uint32_t>(b - a), bar);
  }
  return static_cast<uint32_t>(b - a);
}

struct Ring {
  uint64_t full[kMaxStages], empty[kMaxStages];
};

__device__ __forceinline__ void ring_init(Ring& ring, int stages, int workers) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], workers / 32);
    }
    fence_barrier_init();
  }
  __syncthreads();
}

// The loading warp: tiles block, block + grid, ... A wait that runs out is recorded, and no later one
// is waited for: the kernel then ends soon, with an error that jk_device_status reports.
__device__ __forceinline__ void load_tiles(const Plan& plan, Ring& ring, unsigned char* memory, int64_t rows) {
  const int lane = threadIdx.x & 31;
  bool good = true;
  int stage = 0;
  uint32_t turn = 0;
  const int64_t tiles = (rows + plan.tile_rows - 1) / plan.tile_rows;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    if (turn > 0 && good) good = mbar_wait(&ring.empty[stage], (turn - 1) & 1);
    const int64_t r0 = tile * plan.tile_rows;
    const int n = static_cast<int>(rows - r0 < plan.tile_rows ? rows - r0 : plan.tile_rows);
    unsigned char* base = memory + static_cast<size_t>(stage) * plan.stage_bytes;
    uint32_t bytes = 0;
    for (int issue = 0; issue < 2; ++issue) {
      for (int k = 0; k < plan.feeds; ++k) {
        const Feed& f = plan.feed[k];
        if (f.pitch == 0) {
          if (lane == k) {
            const char* from = f.p + r0 * f.stride;
            bytes += copy_piece(f, rows, from, from + static_cast<int64_t>(n) * f.row_bytes, base + f.offset, issue != 0, &ring.full[stage]);
          }
        } else {
          for (int i = lane; i < n; i += 32) {
            const char* from = f.p + (r0 + i) * f.stride;
            bytes += copy_piece(f, rows, from, from + f.row_bytes, base + f.offset + i * f.pitch, issue != 0, &ring.full[stage]);
          }
        }
      }
      if (issue == 0) {
        bytes = __reduce_add_sync(0xffffffffu, bytes);
        if (lane == 0) mbar_arrive_expect_tx(&ring.full[stage], bytes);
        __syncwarp();
      }
    }
    if (++stage == plan.stages) stage = 0, ++turn;
  }
  // copies in flight land before the block's memory is given back
  for (int i = 0; i < plan.stages; ++i) {
    const uint32_t loads = turn + (i < stage ? 1 : 0);
    if (loads > 0 && good) good = mbar_wait(&ring.full[i], (loads - 1) & 1);
  }
  if (!good) g_device_error = JK_ERR_DEVICE_TIMEOUT;
}

// `take(i, r, stage)` for the tiles' rows that this thread's group has: i in the tile, r in all.
template <int TPR, typename F>
__device__ __forceinline__ void take_tiles(const Plan& plan, Ring& ring, const unsigned char* memory, int64_t rows, F&& take) {
  bool good = true;
  int stage = 0;
  uint32_t turn = 0;
  const int64_t tiles = (rows + plan.tile_rows - 1) / plan.tile_rows;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    if (good) good = mbar_wait(&ring.full[stage], turn & 1);
    const int64_t r0 = tile * plan.tile_rows;
    const int n = static_cast<int>(rows - r0 < plan.tile_rows ? rows - r0 : plan.tile_rows);
    const unsigned char* base = memory + static_cast<size_t>(stage) * plan.stage_bytes;
    for (int i = threadIdx.x / TPR; i < n; i += kGroups<TPR>) take(i, r0, base);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[stage]);
    if (++stage == plan.stages) stage = 0, ++turn;
  }
  if (!good) g_device_error = JK_ERR_DEVICE_TIMEOUT;
}

template <typename T, int N, int TPR, bool DELTA>
__global__ void __launch_bounds__(kBlock<TPR> + 32) staged_forward_kernel(const Forward a, const __grid_constant__ Plan plan) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ Ring ring;
  __shared__ float scratch[2][1][32];
  ring_init(ring, plan.stages, kBlock<TPR>);
  if (threadIdx.x >= kBlock<TPR>) {
    load_tiles(plan, ring, memory, a.rows);
    return;
  }
  const int dim = static_cast<int>(a.dim), thread = threadIdx.x % TPR;
  float w[N], b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = i * TPR + thread;
    w[i] = c < dim ? param_at(a.weight, c, a.param_type, 1.f) : 0.f;
    b[i] = c < dim ? param_at(a.bias, c, a.param_type, 0.f) : 0.f;
  }
  const float inv = 1.f / static_cast<float>(dim);
  take_tiles<TPR>(plan, ring, memory, a.rows, [&](int row, int64_t r0, const unsigned char* stage) {
    const T* x = reinterpret_cast<const T*>(staged(plan.feed[0], stage, r0, row));
    const T* d = DELTA ? reinterpret_cast<const T*>(staged(plan.feed[1], stage, r0, row)) : nullptr;
    float f[N], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR + thread;
      f[i] = 0.f;
      if (c < dim) {
        f[i] = to_f32(x[c]);
        if (DELTA) f[i] = fmaf(a.scale, to_f32(d[c]), f[i]);
      }
      s[0] += f[i];
    }
    row_sums<TPR, 1, true>(s, scratch, 0);
    const float mu = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = i * TPR + thread < dim ? f[i] - mu : 0.f;
      s[0] = fmaf(v, v, s[0]);
    }
    row_sums<TPR, 1, true>(s, scratch, 1);
    const float rs = rsqrtf(fmaf(s[0], inv, a.eps));
    const int64_t r = r0 + row;
    T *y = static_cast<T*>(a.y) + r * dim, *sum = a.sum == nullptr ? nullptr : static_cast<T*>(a.sum) + r * dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR + thread;
      if (c < dim) {
        y[c] = from_f32<T>(fmaf((f[i] - mu) * rs, w[i], b[i]));
        if (sum != nullptr) sum[c] = from_f32<T>(f[i]);
      }
    }
    if (thread == 0 && a.mean != nullptr) {
      a.mean[r] = mu;
      a.rstd[r] = rs;
    }
  });
}

template <typename T, int N, int TPR, bool SUM, bool PARAMS>
__global__ void __launch_bounds__(kBlock<TPR> + 32) staged_backward_kernel(const Backward a, const __grid_constant__ Plan plan) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ Ring ring;
  __shared__ float scratch[2][2][32];
  constexpr bool kShared = PARAMS && TPR <= 32;
  __shared__ float shared[kShared ? N * TPR * 2 : 1];
  ring_init(ring, plan.stages, kBlock<TPR>);
  if (threadIdx.x >= kBlock<TPR>) {
    load_tiles(plan, ring, memory, a.rows);
    return;
  }
  const int dim = static_cast<int>(a.dim), thread = threadIdx.x % TPR;
  float w[N], dw[N][1] = {}, db[N][1] = {};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = i * TPR + thread;
    w[i] = c < dim ? param_at(a.weight, c, a.param_type, 1.f) : 0.f;
  }
  const float inv = 1.f / static_cast<float>(dim);
  int turn = 0;
  take_tiles<TPR>(plan, ring, memory, a.rows, [&](int row, int64_t r0, const unsigned char* stage) {
    const float mu = *reinterpret_cast<const float*>(staged(plan.feed[0], stage, r0, row));
    const float rs = *reinterpret_cast<const float*>(staged(plan.feed[1], stage, r0, row));
    const T* gy = reinterpret_cast<const T*>(staged(plan.feed[2], stage, r0, row));
    const T* h = reinterpret_cast<const T*>(staged(plan.feed[3], stage, r0, row));
    float g[N], n[N], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR + thread;
      g[i] = n[i] = 0.f;
      if (c < dim) {
        g[i] = to_f32(gy[c]);
        n[i] = (to_f32(h[c]) - mu) * rs;
      }
      if (PARAMS) {
        dw[i][0] = fmaf(g[i], n[i], dw[i][0]);
        db[i][0] += g[i];
      }
      const float u = g[i] * w[i];
      s[0] += u;
      s[1] = fmaf(u, n[i], s[1]);
    }
    row_sums<TPR, 2, true>(s, scratch, turn);
    turn ^= 1;
    const float c0 = s[0] * inv, c1 = s[1] * inv;
    const T* gs = SUM ? reinterpret_cast<const T*>(staged(plan.feed[4], stage, r0, row)) : nullptr;
    const int64_t r = r0 + row;
    T *gx = static_cast<T*>(a.grad_x) + r * dim, *gd = a.grad_delta == nullptr ? nullptr : static_cast<T*>(a.grad_delta) + r * dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * TPR + thread;
      if (c < dim) {
        float o = fmaf(g[i], w[i], -fmaf(n[i], c1, c0));
        o = SUM ? fmaf(rs, o, to_f32(gs[c])) : rs * o;
        gx[c] = from_f32<T>(o);
        if (gd != nullptr) gd[c] = from_f32<T>(a.scale * o);
      }
    }
  });
  if constexpr (PARAMS) {
    grid_dependency_launch();
    leave_parts<1, N, TPR, true>(dw, db, dim, a.parts, shared);
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

template <auto KERNEL, int TPR>
int run_forward(const Forward& a, cudaStream_t s) {
  const int64_t blocks = groups_to_blocks(a.rows, kGroups<TPR>, 148ll * blocks_per_sm<KERNEL>(kBlock<TPR>));
  KERNEL<<<static_cast<unsigned>(blocks), kBlock<TPR>, 0, s>>>(a);
  return 0;
}

template <typename T, int VEC, int N, int TPR>
int pick_forward(const Forward& a, cudaStream_t s) {
  return a.delta != nullptr ? run_forward<forward_kernel<T, VEC, N, TPR, true>, TPR>(a, s)
                            : run_forward<forward_kernel<T, VEC, N, TPR, false>, TPR>(a, s);
}

template <auto KERNEL, int TPR>
int run_backward(const Backward& a, cudaStream_t s) {
  int64_t most = 148ll * blocks_per_sm<KERNEL>(kBlock<TPR>);
  if (a.parts != nullptr && most > kMaxParts) most = kMaxParts;
  const int blocks = static_cast<int>(groups_to_blocks(a.rows, kGroups<TPR>, most));
  KERNEL<<<blocks, kBlock<TPR>, 0, s>>>(a);
  return blocks;
}

template <typename T, int VEC, int N, int TPR>
int pick_backward(const Backward& a, cudaStream_t s) {
  if (a.grad_sum != nullptr)
    return a.parts != nullptr ? run_backward<backward_kernel<T, VEC, N, TPR, true, true>, TPR>(a, s)
                              : run_backward<backward_kernel<T, VEC, N, TPR, true, false>, TPR>(a, s);
  return a.parts != nullptr ? run_backward<backward_kernel<T, VEC, N, TPR, false, true>, TPR>(a, s)
                            : run_backward<backward_kernel<T, VEC, N, TPR, false, false>, TPR>(a, s);
}

constexpr int kNoRoom = -1000;  // no status

// A plan for rows off boundaries: tiles of some 8 KB, as many in flight as fill an SM's shared memory
// with the blocks that it holds. False if two tiles of one row do not fit.
struct Tiles {
  int blocks_per_sm;
  size_t smem;
};
inline bool plan_tiles(Plan& plan, int64_t rows, int groups, int want_blocks, Tiles& tiles) {
  int64_t row = 0;
  for (int k = 0; k < plan.feeds; ++k) row += plan.feed[k].row_bytes;
  int64_t tile_rows = groups;
  while (tile_rows * 2 <= kMaxTileRows && tile_rows * 2 * row <= 8192) tile_rows *= 2;
  const int64_t least = (rows + 148 * want_blocks - 1) / (148 * want_blocks);  // rows of a block
  while (tile_rows > groups && tile_rows > least) tile_rows /= 2;
  plan.tile_rows = static_cast<int>(tile_rows);
  uint32_t at = 0;
  for (int k = 0; k < plan.feeds; ++k) {
    Feed& f = plan.feed[k];
    f.offset = at;
    f.pitch = f.stride == f.row_bytes ? 0 : (f.row_bytes + 15 + 15) / 16 * 16;
    at += f.pitch == 0 ? static_cast<uint32_t>((tile_rows * f.row_bytes + 15 + 15) / 16 * 16) : static_cast<uint32_t>(tile_rows * f.pitch);
  }
  plan.stage_bytes = at;
  constexpr int64_t kRoom = 200 * 1024;
  int blocks = want_blocks;
  while (blocks > 1 && kRoom / blocks < 3 * static_cast<int64_t>(at)) --blocks;
  const int64_t fit = kRoom / blocks / at;
  if (fit < 2) return false;
  plan.stages = static_cast<int>(fit < kMaxStages ? fit : kMaxStages);
  tiles = {blocks, static_cast<size_t>(plan.stages) * at};
  return true;
}

template <typename T>
Feed feed_of(const void* p, int64_t stride, int64_t dim) {
  return {static_cast<const char*>(p), stride * static_cast<int64_t>(sizeof(T)), static_cast<int>(dim * sizeof(T)), 0, 0};
}

template <auto KERNEL>
bool allow(size_t smem) {
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}

template <auto KERNEL, typename T, int TPR>
int run_staged_forward(const Forward& a, cudaStream_t s) {
  Plan plan = {};
  plan.feed[plan.feeds++] = feed_of<T>(a.x, a.x_stride, a.dim);
  if (a.delta != nullptr) plan.feed[plan.feeds++] = feed_of<T>(a.delta, a.delta_stride, a.dim);
  Tiles tiles;
  if (!plan_tiles(plan, a.rows, kGroups<TPR>, blocks_per_sm<KERNEL>(kBlock<TPR> + 32), tiles)) return kNoRoom;
  if (!allow<KERNEL>(tiles.smem)) return JK_ERR_LAUNCH;
  const int64_t blocks = groups_to_blocks(a.rows, plan.tile_rows, 148ll * tiles.blocks_per_sm);
  KERNEL<<<static_cast<unsigned>(blocks), kBlock<TPR> + 32, tiles.smem, s>>>(a, plan);
  return 0;
}

template <auto KERNEL, typename T, int TPR>
int run_staged_backward(const Backward& a, cudaStream_t s) {
  Plan plan = {};
  plan.feed[plan.feeds++] = feed_of<float>(a.mean, 1, 1);
  plan.feed[plan.feeds++] = feed_of<float>(a.rstd, 1, 1);
  plan.feed[plan.feeds++] = feed_of<T>(a.grad_y, a.grad_y_stride, a.dim);
  plan.feed[plan.feeds++] = feed_of<T>(a.sum, a.sum_stride, a.dim);
  if (a.grad_sum != nullptr) plan.feed[plan.feeds++] = feed_of<T>(a.grad_sum, a.grad_sum_stride, a.dim);
  Tiles tiles;
  if (!plan_tiles(plan, a.rows, kGroups<TPR>, blocks_per_sm<KERNEL>(kBlock<TPR> + 32), tiles)) return kNoRoom;
  if (!allow<KERNEL>(tiles.smem)) return JK_ERR_LAUNCH;
  int64_t most = 148ll * tiles.blocks_per_sm;
  if (a.parts != nullptr && most > kMaxParts) most = kMaxParts;
  const int blocks = static_cast<int>(groups_to_blocks(a.rows, plan.tile_rows, most));
  KERNEL<<<blocks, kBlock<TPR> + 32, tiles.smem, s>>>(a, plan);
  return blocks;
}

template <typename T, int N, int TPR>
int pick_staged_forward(const Forward& a, cudaStream_t s) {
  return a.delta != nullptr ? run_staged_forward<staged_forward_kernel<T, N, TPR, true>, T, TPR>(a, s)
                            : run_staged_forward<staged_forward_kernel<T, N, TPR, false>, T, TPR>(a, s);
}

template <typename T, int N, int TPR>
int pick_staged_backward(const Backward& a, cudaStream_t s) {
  if (a.grad_sum != nullptr)
    return a.parts != nullptr ? run_staged_backward<staged_backward_kernel<T, N, TPR, true, true>, T, TPR>(a, s)
                              : run_staged_backward<staged_backward_kernel<T, N, TPR, true, false>, T, TPR>(a, s);
  return a.parts != nullptr ? run_staged_backward<staged_backward_kernel<T, N, TPR, false, true>, T, TPR>(a, s)
                            : run_staged_backward<staged_backward_kernel<T, N, TPR, false, false>, T, TPR>(a, s);
}

// The threads of a row and their turns: as few threads as hold it with 16 elements each (fewer where
// a warp has room), a warp's or less while that does, so that no barrier is needed.
#define JK_NORM_SHAPES(RUN)                                             \
  if constexpr (VEC == 8) {                                             \
    if (turns <= 8) return RUN(1, 8);                                   \
    if (turns <= 16) return RUN(1, 16);                                 \
    if (turns <= 32) return RUN(1, 32);                                 \
    if (turns <= 64) return RUN(2, 32);                                 \
    if (turns <= 256) return RUN(2, 128);                               \
    if (turns <= 512) return RUN(2, 256);                               \
    if (turns <= 1024) return RUN(2, 512);                              \
    return RUN(2, 1024);                                                \
  } else if constexpr (VEC == 4) {                                      \
    if (turns <= 8) return RUN(1, 8);                                   \
    if (turns <= 16) return RUN(1, 16);                                 \
    if (turns <= 32) return RUN(1, 32);                                 \
    if (turns <= 64) return RUN(2, 32);                                 \
    if (turns <= 128) return RUN(4, 32);                                \
    if (turns <= 512) return RUN(4, 128);                               \
    if (turns <= 1024) return RUN(4, 256);                              \
    if (turns <= 2048) return RUN(4, 512);                              \
    return RUN(4, 1024);                                                \
  } else {                                                              \
    if (turns <= 32) return RUN(1, 32);                                 \
    if (turns <= 64) return RUN(2, 32);                                 \
    if (turns <= 128) return RUN(4, 32);                                \
    if (turns <= 256) return RUN(8, 32);                                \
    if (turns <= 512) return RUN(16, 32);                               \
    if (turns <= 1024) return RUN(8, 128);                              \
    if (turns <= 2048) return RUN(8, 256);                              \
    if (turns <= 4096) return RUN(8, 512);                              \
    return RUN(16, 512);                                                \
  }

constexpr int64_t kMaxDim = 16384, kMaxStagedDim = 8192;  // of the rows that stay in registers

template <typename T, int VEC>
int shape_forward(const Forward& a, cudaStream_t s) {
  const int64_t turns = a.dim / VEC;
#define JK_RUN(N, TPR) pick_forward<T, VEC, N, TPR>(a, s)
  JK_NORM_SHAPES(JK_RUN)
#undef JK_RUN
}

template <typename T>
int shape_staged_forward(const Forward& a, cudaStream_t s) {
  constexpr int VEC = 1;
  const int64_t turns = a.dim;
#define JK_RUN(N, TPR) pick_staged_forward<T, N, TPR>(a, s)
  JK_NORM_SHAPES(JK_RUN)
#undef JK_RUN
}

template <typename T, int VEC>
int shape_backward(const Backward& a, cudaStream_t s) {
  const int64_t turns = a.dim / VEC;
#define JK_RUN(N, TPR) pick_backward<T, VEC, N, TPR>(a, s)
  JK_NORM_SHAPES(JK_RUN)
#undef JK_RUN
}

template <typename T>
int shape_staged_backward(const Backward& a, cudaStream_t s) {
  constexpr int VEC = 1;
  const int64_t turns = a.dim;
#define JK_RUN(N, TPR) pick_staged_backward<T, N, TPR>(a, s)
  JK_NORM_SHAPES(JK_RUN)
#undef JK_RUN
}

template <typename T>
bool in_packs(const void* p, int64_t stride) {
  return p == nullptr || (aligned16(p) && stride % kPack<T> == 0);
}

template <typename T>
int forward(const Forward& a, cudaStream_t s) {
  if (a.dim <= kMaxDim && in_packs<T>(a.x, a.x_stride) && in_packs<T>(a.delta, a.delta_stride) && in_packs<T>(a.y, a.dim) &&
      in_packs<T>(a.sum, a.dim))
    return shape_forward<T, kPack<T>>(a, s);
  if (a.dim <= kMaxStagedDim) {
    const int done = shape_staged_forward<T>(a, s);
    if (done != kNoRoom) return done;
  }
  long_forward_kernel<T><<<static_cast<unsigned>(a.rows < 148 * 4 ? a.rows : 148 * 4), kLongThreads, 0, s>>>(a);
  return 0;
}

// Returns the blocks that left a share of the parameter gradients, or a status.
template <typename T>
int backward(const Backward& a, cudaStream_t s) {
  if (a.dim <= kMaxDim && in_packs<T>(a.grad_y, a.grad_y_stride) && in_packs<T>(a.sum, a.sum_stride) &&
      in_packs<T>(a.grad_sum, a.grad_sum_stride) && in_packs<T>(a.grad_x, a.dim) && in_packs<T>(a.grad_delta, a.dim))
    return shape_backward<T, kPack<T>>(a, s);
  if (a.dim <= kMaxStagedDim) {
    const int done = shape_staged_backward<T>(a, s);
    if (done != kNoRoom) return done;
  }
  const int blocks = static_cast<int>(a.rows < kMaxParts ? a.rows : kMaxParts);
  long_backward_kernel<T><<<blocks, kLongThreads, 0, s>>>(a);
  return blocks;
}

}  // namespace norm

JK_ERROR_READER(read_error_norm)

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
  JK_WITH_TYPE(dtype, T, st = norm::forward<T>(a, reinterpret_cast<cudaStream_t>(stream)));
  return st < 0 ? st : launch_status();
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
  if (parts < 0) return parts;
  if (params)
    JK_WITH_TYPE(param_dtype, W, launch_dependent(norm::parameters_kernel<W>, static_cast<unsigned>((2 * dim + 31) / 32), 1024, 0, s,
                                                  workspace, parts, dim, static_cast<W*>(grad_weight), static_cast<W*>(grad_bias)));
  return launch_status();
}
