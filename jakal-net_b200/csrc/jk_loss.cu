// Softmax cross entropy over a vocabulary and its gradient (jk_cross_entropy_forward / _backward).
//
//   lse = m + log sum_j exp(z_j - m), m = max_j z_j
//   loss = lse - (1 - a) z_t - a E_j[z_j]
//   grad_j = c (exp(z_j - lse) - (1 - a) [j = t] - a / V),  c = scale / number of rows that count
//
// With the maximum at hand, loss = log sum exp(z - m) + (1 - a) (m - z_t) + a E_j[m - z_j] and
// softmax_j = exp(z_j - m) / sum: differences from m keep their digits where m is large, which
// lse = m + log(sum), one f32 number, does not. exp(z - m) is 2^(z log2(e) - r), one fma and the
// hardware's exponential, with r = m log2(e) rounded once and carried along. What r is short of that
// product is a factor of the whole sum, of up to 2^(half a unit in r's last place): beyond |m| = 2^23
// it would be more than 2 (and out of range from 2^31 on), so there it is taken of z - m instead. The
// mean distance from m comes from the same exponents (4096 x 16384 bf16 with gradient and smoothing:
// 62 us, 104 when it took the logits once more; f32: 104 against 106).
//
// Bound: memory, one read of the logits and one write of the gradient; for 16-bit logits with a
// gradient the exponentials, two a logit, come near it. Three forms:
//   * warp_kernel, rows of up to 1024 logits: a warp has a row in its registers;
//   * rows_kernel, loss and gradient of longer rows: a block has a row (of few rows, a cluster of
//     blocks shares each) in shared memory, brought there by bulk copies that run rows ahead of the
//     arithmetic, and takes the gradient from the same copy, so the logits are read once;
//   * stream_kernel, the loss alone, or the gradient from the lse, and both one after the other where
//     rows_kernel does not have the room: the packs of all rows in equal runs, one for each warp.
#include "jk_host.h"
#include "jk_rows.cuh"
#include "jk_sm100.cuh"

#include <type_traits>

namespace jk {
namespace loss {

enum Mode { kLoss, kBoth, kBackward, kLater };  // kLater: kBackward within the forward call

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int64_t kMaxVocab = int64_t(1) << 30;  // columns are counted in 32 bits
constexpr int kMaxBlocks = 148 * 8;    // blocks that leave a partial
constexpr int kCounts = 64;            // blocks of the counting kernel
constexpr int64_t kCountRows = 4096;   // up to so many rows every block counts for itself

// What a block leaves for the reduction over rows.
struct Partial {
  double sum;
  long long rows;
};

template <typename T>
struct Args {
  const T* logits;
  int64_t stride;
  const int64_t* targets;
  int64_t rows, vocab, ignore_index;
  float smoothing;
  int reduction;
  float scale;             // of the gradient (forward)
  const float* grad_loss;  // backward
  const float *lse_in, *low_in;  // low: what an lse in one f32 is short of the log-sum (null: 0)
  float* losses;
  float *lse_out, *low_out;
  T* grad;
  int64_t grad_stride;
  Partial* partials;
  const int* counts;  // of kCounts blocks, or null: count here
  float* loss_now;    // not null where one block has all rows: it writes the reduced loss itself
};

// A product that is rounded by itself, whatever it is added to.
__device__ __forceinline__ float product(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The largest of N packs, NaN aside; 16-bit types two at a time.
template <typename T, int N>
__device__ __forceinline__ float pack_max(const uint4 (&raw)[N]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float f[4];
      unpack<T>(raw[i], f);
      m = fmaxf(m, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])));
    }
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m = *reinterpret_cast<const T2*>(&raw[0].x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const T2* h = reinterpret_cast<const T2*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) m = __hmax2(m, h[j]);
    }
    return fmaxf(to_f32(m.x), to_f32(m.y));
  }
}

// The reference of a sum of exponentials: exp(z - m) as 2^(z log2(e) - r) while r is good to one half.
constexpr float kFar = 8388608.f;  // r < 2^24
struct Base {
  float m, r;
  bool near;

  __device__ __forceinline__ explicit Base(float m_) : m(m_), r(product(m_, kLog2e)), near(fabsf(m_) < kFar) {}
  __device__ __forceinline__ float exp_near(float z) const { return exp2_approx(fmaf(z, kLog2e, -r)); }
  __device__ __forceinline__ float exp_far(float z) const { return exp2_approx((z - m) * kLog2e); }
  __device__ __forceinline__ float exp(float z) const { return near ? exp_near(z) : exp_far(z); }
  // What 2^-r is short of exp(-m), as a power of 2 (near only) and of e.
  __device__ __forceinline__ float short_of() const { return fmaf(-m, kLog2e, r); }
  __device__ __forceinline__ float rest() const { return near ? kLn2 * short_of() : 0.f; }
};

// Replaces N logits by their exponentials.
template <int N>
__device__ __forceinline__ void exponentials(float (&z)[N], const Base& b) {
  if (b.near) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = b.exp_near(z[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = b.exp_far(z[i]);
  }
}

// (m, s): a maximum and the sum of the exponentials on it; -inf and 0 for nothing.
struct Sum {
  float m, s;
};

// What a sum on maximum `from` is worth on a larger one: 2^-r counts for a near one, exp(-m) for a far one.
__device__ __forceinline__ float factor_to(float from, float to) {
  const Base a(from), b(to);
  if (b.near) return exp2_approx(a.near ? a.r - b.r : fmaf(from, kLog2e, -b.r));
  return exp2_approx(fmaf(from - to, kLog2e, a.near ? fmaf(-from, kLog2e, a.r) : 0.f));
}

__device__ __forceinline__ float warp_max32(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Over a warp: one maximum, one factor per lane, one sum. Every lane gets the same bits.
__device__ __forceinline__ Sum warp_join(Sum v) {
  const float m = warp_max32(v.m);
  // a lane without a finite value has s = 0 or NaN, and neither needs a factor
  return {m, warp_sum32(v.m == m ? v.s : v.s * factor_to(v.m, m))};
}

template <int N>
__device__ __forceinline__ float top_of(const float (&z)[N]) {
  float top = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
  return top;
}

// Adds N values to a thread's sum.
template <int N>
__device__ __forceinline__ void take(Sum& v, float (&z)[N]) {
  const float top = top_of(z);
  if (top > v.m) {
    v.s *= factor_to(v.m, top);  // from -inf: 0
    v.m = top;
  }
  exponentials(z, Base(v.m == -INFINITY ? 0.f : v.m));
#pragma unroll
  for (int i = 0; i < N; ++i) v.s += z[i];
}

// The scale of a Gap, a power of two that is less than 1 / (2 vocab): the sum stays in f32's range.
__device__ __forceinline__ float gap_scale(int vocab) { return __uint_as_float(static_cast<uint32_t>(94 + __clz(vocab)) << 23); }

// For label smoothing: the sum of (z - m) * scale over n logits, m being their maximum so far. All terms
// have one sign, so the sum keeps its digits wherever m is, which a sum of logits would not.
struct Gap {
  float sum;
  int n;

  // m has grown
  __device__ __forceinline__ void move(float from, float to, float scale) {
    if (n > 0 && from != to) sum = fmaf(static_cast<float>(n), fmaf(from, scale, -to * scale), sum);
  }
  __device__ __forceinline__ void add(float z, float m, float scale) {
    sum += fmaf(z, scale, m == -INFINITY ? 0.f : -m * scale);  // where all are -inf, so is the sum
    ++n;
  }
  // Over a warp whose lanes had maxima `from`.
  __device__ __forceinline__ void join(float from, float to, float scale) {
    move(from, to, scale);
    sum = warp_sum32(sum);
    n = __reduce_add_sync(0xffffffffu, n);
  }
};

// Adds N packs to a thread's sum and, with GAP, the first `whole` of them to its gap (the others are
// all -inf); again(i) is pack i once more. All maxima first: 16 logits or more share one comparison
// and one factor.
template <typename T, bool GAP, int N, typename Again>
__device__ __forceinline__ void take_packs(Sum& v, const uint4 (&raw)[N], Gap& gap, float scale, int whole, Again&& again) {
  const float top = pack_max<T>(raw);
  if (top > v.m) {
    v.s *= factor_to(v.m, top);
    if (GAP) gap.move(v.m, top, scale);
    v.m = top;
  }
  const float m = v.m == -INFINITY ? 0.f : v.m;
  const Base b(m);
  float g = -INFINITY;  // of the gap, in powers of 2: the exponents are at hand
  if (b.near) {
    const uint64_t l2e = pair(kLog2e, kLog2e), minus_r = pair(-b.r, -b.r);
    uint64_t s = pair(v.s, 0.f), x_sum = 0;
    const auto take_pack = [&](const uint4& u) {
      float f[kPack<T>];
      unpack<T>(u, f);
#pragma unroll
      for (int j = 0; j < kPack<T>; j += 2) {
        const uint64_t x2 = fma2(pair(f[j], f[j + 1]), l2e, minus_r);
        const float2 x = unpair(x2);
        s = add2(s, pair(exp2_approx(x.x), exp2_approx(x.y)));
        if (GAP) x_sum = add2(x_sum, x2);
      }
    };
    if (!GAP || whole == N) {
#pragma unroll
      for (int i = 0; i < N; ++i) take_pack(raw[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < whole) take_pack(raw[i]);
    }
    float2 both = unpair(s);
    v.s = both.x + both.y;
    both = unpair(x_sum);
    if (GAP) g = fmaf(static_cast<float>(whole * kPack<T>), b.short_of(), both.x + both.y);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float f[kPack<T>];
      unpack<T>(raw[i], f);
#pragma unroll
      for (int j = 0; j < kPack<T>; ++j) v.s += b.exp_far(f[j]);
    }
  }
  if (GAP) {
    gap.n += whole * kPack<T>;
    if (g > -1e38f) {
      gap.sum = fmaf(g, kLn2 * scale, gap.sum);
    } else {  // the exponents have left f32's range, or are not at hand
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i >= whole) continue;
        float f[kPack<T>];
        unpack<T>(again(i), f);
#pragma unroll
        for (int j = 0; j < kPack<T>; ++j) gap.sum += fmaf(f[j], scale, -m * scale);
      }
    }
  }
}

// f = scale * exp(f - m) + other for a pack.
template <typename T>
__device__ __forceinline__ void gradient_pack(float (&f)[kPack<T>], const Base& b, float scale, float other) {
  if (b.near) {
    const uint64_t l2e = pair(kLog2e, kLog2e), minus_r = pair(-b.r, -b.r), by = pair(scale, scale), to = pair(other, other);
#pragma unroll
    for (int j = 0; j < kPack<T>; j += 2) {
      const float2 x = unpair(fma2(pair(f[j], f[j + 1]), l2e, minus_r));
      const float2 y = unpair(fma2(pair(exp2_approx(x.x), exp2_approx(x.y)), by, to));
      f[j] = y.x, f[j + 1] = y.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPack<T>; ++j) f[j] = fmaf(b.exp_far(f[j]), scale, other);
  }
}

// Rows that count, over all rows, by the block's threads [0, n).
__device__ __forceinline__ int count_rows(const int64_t* targets, int64_t rows, int64_t ignore_index, int threads) {
  int n = 0;
  for (int64_t r = threadIdx.x; r < rows; r += threads) n += targets[r] != ignore_index;
  return __reduce_add_sync(0xffffffffu, n);
}

__global__ void __launch_bounds__(256) count_kernel(const int64_t* targets, int64_t rows, int64_t ignore_index, int* counts) {
  __shared__ int part[8];
  const int64_t per = (rows + gridDim.x - 1) / gridDim.x, from = per * blockIdx.x;
  const int64_t n = rows - from < per ? rows - from : per;
  const int mine = n > 0 ? count_rows(targets + from, n, ignore_index, 256) : 0;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    int all = 0;
    for (int i = 0; i < 8; ++i) all += part[i];
    counts[blockIdx.x] = all;
  }
}

// The factor of a row's gradient, without the row's own grad_loss, for all of the block's threads
// [0, threads); `sync` is their barrier.
template <typename T, typename Sync>
__device__ __forceinline__ float gradient_factor(const Args<T>& a, bool forward, int threads, int* scratch, Sync&& sync) {
  float c = forward ? a.scale : (a.reduction == JK_REDUCE_NONE ? 1.f : *a.grad_loss);
  if (a.reduction != JK_REDUCE_MEAN) return c;
  int n = 0;
  if (a.counts != nullptr) {
    for (int i = threadIdx.x & 31; i < kCounts; i += 32) n += a.counts[i];
    n = __reduce_add_sync(0xffffffffu, n);
  } else {
    const int mine = count_rows(a.targets, a.rows, a.ignore_index, threads);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = mine;
    sync();
    for (int i = 0; i < threads / 32; ++i) n += scratch[i];
  }
  return c / static_cast<float>(n);
}

// A row's loss and log-sum (lse + low) from its sum, target logit and Gap's sum.
struct RowLoss {
  float loss, lse, low;
  __device__ __forceinline__ RowLoss(Sum v, float zt, float gap, float smoothing, int vocab) {
    const float log_sum = logf(v.s) + Base(v.m).rest();  // ln sum exp(z - m)
    loss = log_sum + (1.f - smoothing) * (v.m - zt);
    if (smoothing != 0.f) loss -= smoothing * gap / (gap_scale(vocab) * static_cast<float>(vocab));
    lse = v.m + log_sum;
    const float t = lse - v.m;
    low = (v.m - (lse - t)) + (log_sum - t);
  }
};

// Row r's results, of those that are asked for (LOW: of a loss alone, whose gradient may follow).
template <bool LOW, typename T>
__device__ __forceinline__ void leave_row(const Args<T>& a, int64_t r, float loss, float lse, float low) {
  if (a.losses != nullptr) a.losses[r] = loss;
  if (a.lse_out != nullptr) a.lse_out[r] = lse;
  if (LOW && a.low_out != nullptr) a.low_out[r] = low;
}

// ---------------------------------------------------------------- short rows
// A warp per row, N turns of VEC neighbouring elements per lane. So few rows as kOneBlockRows are one
// block's, which then needs no second kernel for their sum.
constexpr int kWarpThreads = 256, kOneBlockThreads = 512;
constexpr int64_t kOneBlockRows = 2 * kOneBlockThreads / 32;

template <typename T, int VEC>
__device__ __forceinline__ void load_row(float (&f)[VEC], const T* p) {
  if constexpr (VEC == 1)
    f[0] = to_f32(*p);
  else
    unpack<T>(*reinterpret_cast<const uint4*>(p), f);
}

template <typename T, int MODE, int VEC, int N, int THREADS>
__global__ void __launch_bounds__(THREADS) warp_kernel(const Args<T> a) {
  __shared__ int scratch[THREADS / 32];
  __shared__ Partial parts[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int vocab = static_cast<int>(a.vocab);
  float factor = 0.f;
  if (MODE != kLoss) factor = gradient_factor(a, MODE == kBoth, THREADS, scratch, [] { __syncthreads(); });
  const float share = a.smoothing / static_cast<float>(vocab), hit = 1.f - a.smoothing;
  Partial part{0.0, 0};
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + warp; r < a.rows;
       r += static_cast<int64_t>(gridDim.x) * (THREADS / 32)) {
    const int64_t target = a.targets[r];
    const T* z = a.logits + r * a.stride;
    T* g = MODE == kLoss ? nullptr : a.grad + r * a.grad_stride;
    const bool ignored = target == a.ignore_index;
    const bool inside = target >= 0 && target < vocab;
    float f[N][VEC];
    if (!ignored) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * 32 + lane) * VEC;
        if (c < vocab) {
          load_row<T, VEC>(f[i], z + c);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[i][j] = -INFINITY;
        }
      }
    }
    float m = 0.f, scale = 0.f;
    if (!ignored && MODE != kBackward) {
      const float zt = inside ? to_f32(z[target]) : NAN;
      Sum v{-INFINITY, 0.f};
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) top = fmaxf(top, f[i][j]);
      v.m = top = warp_max32(top);
      const Base base(top == -INFINITY ? 0.f : top);  // the sum of nothing but exp(-inf) is 0, its log -inf
      float gap = 0.f;  // of the exponents, then of the logits
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const bool has = (i * 32 + lane) * VEC + j < vocab;
          if (a.smoothing != 0.f) gap += has ? fmaf(f[i][j], kLog2e, -base.r) : 0.f;
          f[i][j] = base.exp(f[i][j]);
          v.s += has ? f[i][j] : 0.f;
        }
      }
      v.s = warp_sum32(v.s);
      if (a.smoothing != 0.f) {
        const float by = gap_scale(vocab);
        gap = fmaf(static_cast<float>(vocab), base.short_of(), warp_sum32(gap));
        if (base.near && gap > -1e38f) {
          gap *= kLn2 * by;
        } else {  // the exponents have left f32's range
          gap = 0.f;
          for (int c = lane; c < vocab; c += 32) gap += fmaf(to_f32(z[c]), by, -top * by);
          gap = warp_sum32(gap);
        }
      }
      const RowLoss l(v, zt, gap, a.smoothing, vocab);
      if (lane == 0) leave_row<MODE == kLoss>(a, r, l.loss, l.lse, l.low);
      part.sum += l.loss;
      part.rows += 1;
      scale = factor / v.s;
      __syncwarp();  // z[target] is read before an in-place gradient replaces it
    } else if (ignored && MODE != kBackward && lane == 0) {
      leave_row<MODE == kLoss>(a, r, 0.f, 0.f, 0.f);
    }
    if (MODE == kLoss) continue;
    float c0 = ignored ? 0.f : factor;
    if (MODE == kBackward && !ignored) {
      m = a.lse_in[r];
      if (a.reduction == JK_REDUCE_NONE) c0 = a.grad_loss[r];
      scale = c0 * expf(Base(m).rest() - (a.low_in != nullptr ? a.low_in[r] : 0.f));
    }
    if (!ignored && !inside) scale = c0 = NAN;
    const Base from(m);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * 32 + lane) * VEC;
      if (c >= vocab) continue;
      float o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float e = ignored ? 0.f : MODE == kBackward ? from.exp(f[i][j]) : f[i][j];
        o[j] = ignored ? 0.f : fmaf(e, scale, -(c + j == target ? hit + share : share) * c0);
      }
      if constexpr (VEC == 1)
        g[c] = from_f32<T>(o[0]);
      else
        *reinterpret_cast<uint4*>(g + c) = pack<T>(o);
    }
  }
  if (MODE == kBackward) return;
  grid_dependency_launch();
  if (lane == 0) parts[warp] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) part.sum += parts[i].sum, part.rows += parts[i].rows;
    if (a.loss_now != nullptr)
      *a.loss_now = static_cast<float>(a.reduction == JK_REDUCE_MEAN ? part.sum / static_cast<double>(part.rows) : part.sum);
    else
      a.partials[blockIdx.x] = part;
  }
}

// ---------------------------------------------------------------- a row as 16-byte packs
constexpr int kTurn = 6;  // packs that a thread takes at once

// Where a row lies against 16-byte packs: pack k holds columns k * kPack - shift ..., the first
// and the last one perhaps in part.
template <typename T>
struct Window {
  const T* z;
  int shift, packs;

  __device__ __forceinline__ Window(const Args<T>& a, int64_t row) {
    z = a.logits + row * a.stride;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(z) & 15) / static_cast<int>(sizeof(T));
    packs = (shift + static_cast<int>(a.vocab) + kPack<T> - 1) / kPack<T>;
  }
};

template <typename T>
__device__ __forceinline__ T minus_inf() {
  return from_f32<T>(-INFINITY);
}

// ---------------------------------------------------------------- loss, and gradient from the lse
// Warps on their own. The packs of all rows, in pieces of 32 x kTurn, are cut into equal runs, one
// for each warp, so that no SM ends late; a lane has the next piece on its way while it works on
// one. A row that more than one warp has part of leaves a record for each, and the reduction over
// rows joins them.
constexpr int kStreamThreads = 256;
// Loss of 4096 x 50001 bf16: 70 us with six packs and two blocks on an SM, 73 with four and three, 160
// with two and six: what a piece costs apart from its packs is spread over more of them.
constexpr int kStreamBlocksPerSm = 2;
constexpr int kMaxWarps = 148 * kStreamBlocksPerSm * (kStreamThreads / 32);
constexpr int kPiece = 32 * kTurn;  // packs

struct Record {
  int64_t row;  // -1: none
  float m, s, gap;
  int n;  // logits in it, if smoothing asks
};

// A piece of a row.
template <typename T>
struct Item {
  int64_t row, target;
  const T* z;
  int piece, shift;
  float value, low, grad_loss;  // the target's logit (kLoss), or the row's lse
  bool ignored, inside;
};

template <typename T, int MODE, bool SMOOTH>
__global__ void __launch_bounds__(kStreamThreads, kStreamBlocksPerSm)
    stream_kernel(const Args<T> a, int pieces, Record* records, int* come) {
  __shared__ int scratch[kStreamThreads / 32];
  constexpr int kP = kPack<T>;
  const int lane = threadIdx.x & 31, vocab = static_cast<int>(a.vocab);
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kStreamThreads / 32);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kStreamThreads / 32) + (threadIdx.x >> 5);
  const int64_t all_items = a.rows * pieces;
  int64_t item = all_items / warps * warp + min(warp, all_items % warps);
  const int64_t end = item + all_items / warps + (warp < all_items % warps ? 1 : 0);
  const float hit = 1.f - a.smoothing, share = a.smoothing / static_cast<float>(vocab);
  float factor = 0.f;
  if (MODE != kLoss) factor = gradient_factor(a, MODE == kLater, kStreamThreads, scratch, [] { __syncthreads(); });
  if (MODE == kLoss && blockIdx.x == 0 && threadIdx.x == 0) *come = 0;  // for the reduction that follows

  // the piece that is next, and what it needs beside its packs
  int64_t row = item / pieces;
  int piece = static_cast<int>(item - row * pieces);
  const int64_t first_row = row;
  int64_t targets_from = row, some_targets = 0;  // of 32 rows, a row per lane
  if (item < end) some_targets = a.targets[min(row + lane, a.rows - 1)];
  uint4 next[kTurn];
  Item<T> it{};
  const auto enter_row = [&] {
    if (row - targets_from >= 32) {
      targets_from = row;
      some_targets = a.targets[min(row + lane, a.rows - 1)];
    }
    it.row = row;
    it.target = __shfl_sync(0xffffffffu, static_cast<long long>(some_targets), static_cast<int>(row - targets_from));
    it.ignored = it.target == a.ignore_index;
    const Window<T> w(a, row);
    it.z = w.z;
    it.shift = w.shift;
    it.inside = it.target >= 0 && it.target < vocab;
    if (it.ignored) return;
    if (MODE == kLoss && piece == 0) it.value = it.inside ? to_f32(w.z[it.target]) : NAN;
    if (MODE != kLoss) {
      it.value = a.lse_in[row];
      it.low = a.low_in != nullptr ? a.low_in[row] : 0.f;
      if (MODE == kBackward && a.reduction == JK_REDUCE_NONE) it.grad_loss = a.grad_loss[row];
    }
  };
  // whether all packs of a piece are whole
  const auto interior = [&](const Item<T>& q) { return q.piece > 0 && (q.piece + 1) * kPiece * kP <= vocab + q.shift; };
  const auto load = [&] {
    it.piece = piece;
    if (it.ignored) return;
    const int c0 = (piece * kPiece + lane) * kP - it.shift;
    if (interior(it)) {
      const uint4* from = reinterpret_cast<const uint4*>(it.z + c0);
#pragma unroll
      for (int i = 0; i < kTurn; ++i) next[i] = __ldcs(from + i * 32);
    } else {
#pragma unroll
      for (int i = 0; i < kTurn; ++i) {
        const int c = c0 + i * 32 * kP;
        if (c >= 0 && c + kP <= vocab) {
          next[i] = __ldcs(reinterpret_cast<const uint4*>(it.z + c));
        } else {  // -inf where there is no column
          T* e = reinterpret_cast<T*>(&next[i]);
#pragma unroll
          for (int j = 0; j < kP; ++j) e[j] = c + j >= 0 && c + j < vocab ? it.z[c + j] : minus_inf<T>();
        }
      }
    }
  };
  if (item < end) {
    enter_row();
    load();
  }

  Sum v{-INFINITY, 0.f};
  Gap gap{0.f, 0};
  const float gap_by = gap_scale(vocab);
  float zt = 0.f;
  bool from_start = false, recorded[2] = {false, false};
  Partial part{0.0, 0};
  while (item < end) {
    uint4 raw[kTurn];
#pragma unroll
    for (int i = 0; i < kTurn; ++i) raw[i] = next[i];
    const Item<T> q = it;
    if (q.piece == 0) {
      from_start = true;
      zt = q.value;
    }
    ++item;
    if (++piece == pieces) {
      piece = 0;
      ++row;
    }
    if (item < end) {
      if (piece == 0) enter_row();
      load();
    }
    const int c0 = (q.piece * kPiece + lane) * kP - q.shift;
    const bool last = q.piece == pieces - 1;
    if (MODE == kLoss) {
      if (!q.ignored) {
        const bool whole = interior(q);
        const float before = v.m;
        if (SMOOTH && whole) {
          take_packs<T, true>(v, raw, gap, gap_by, kTurn, [&](int i) { return raw[i]; });
        } else {
          take_packs<T, false>(v, raw, gap, 0.f, 0, [&](int i) { return raw[i]; });
        }
        if (SMOOTH && !whole) {
          gap.move(before, v.m, gap_by);
#pragma unroll
          for (int i = 0; i < kTurn; ++i) {
            float f[kP];
            unpack<T>(raw[i], f);
#pragma unroll
            for (int j = 0; j < kP; ++j) {
              const int c = c0 + i * 32 * kP + j;
              if (c >= 0 && c < vocab) gap.add(f[j], v.m, gap_by);
            }
          }
        }
        if (last || item == end) {
          const float mine = v.m;
          v = warp_join(v);
          if (SMOOTH) gap.join(mine, v.m, gap_by);
          if (last && from_start) {
            const RowLoss l(v, zt, gap.sum, a.smoothing, vocab);
            if (lane == 0) leave_row<true>(a, q.row, l.loss, l.lse, l.low);
            part.sum += l.loss;
            part.rows += 1;
          } else {
            const int slot = q.row == first_row ? 0 : 1;
            recorded[slot] = true;
            if (lane == 0) records[2 * warp + slot] = {q.row, v.m, v.s, gap.sum, gap.n};
          }
          v = {-INFINITY, 0.f};
          gap = {0.f, 0};
        }
      } else if (last && lane == 0) {
        leave_row<true>(a, q.row, 0.f, 0.f, 0.f);
      }
    } else {
      T* g = a.grad + q.row * a.grad_stride;
      const bool alike = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(q.z)) & 15) == 0;
      const Base base(q.value);
      const float k0 = !q.inside ? NAN : MODE == kBackward && a.reduction == JK_REDUCE_NONE ? q.grad_loss : factor;
      const float scale = k0 * expf(base.rest() - q.low), other = -share * k0;
      const bool whole = alike && interior(q);
#pragma unroll
      for (int i = 0; i < kTurn; ++i) {
        const int c = c0 + i * 32 * kP;
        if (!whole && c >= vocab) continue;
        float f[kP] = {};
        if (!q.ignored) {
          unpack<T>(raw[i], f);
          gradient_pack<T>(f, base, scale, other);
          if (q.inside && static_cast<uint32_t>(static_cast<int>(q.target) - c) < static_cast<uint32_t>(kP)) {
#pragma unroll
            for (int j = 0; j < kP; ++j) f[j] -= c + j == static_cast<int>(q.target) ? hit * k0 : 0.f;
          }
        }
        if (whole || (alike && c >= 0 && c + kP <= vocab)) {
          __stcs(reinterpret_cast<uint4*>(g + c), pack<T>(f));
        } else {
#pragma unroll
          for (int j = 0; j < kP; ++j)
            if (c + j >= 0 && c + j < vocab) g[c + j] = from_f32<T>(f[j]);
        }
      }
    }
    if (last) from_start = false;
  }
  if (MODE != kLoss) return;
  grid_dependency_launch();
  if (lane == 0) {
    for (int i = 0; i < 2; ++i)
      if (!recorded[i]) records[2 * warp + i].row = -1;
    a.partials[warp] = part;
  }
}

// ---------------------------------------------------------------- loss and gradient at once
// A cluster of blocks has a row, each block a slice of it in shared memory. One warp of the block
// has the next rows' slices copied there and finds out how they lie; the others (workers) take a
// slice twice, for the sum and for the gradient.
constexpr int kMaxWorkers = 480;
constexpr int kMaxStages = 6;
constexpr int kMaxCluster = 8;

// A slice, in positions from the first element of its first pack.
struct Slice {
  int64_t row;
  const void* in;        // position 0 of the logits
  void* out;             // and of the gradient
  int whole, whole_end;  // packs that are whole and in shared memory
  int end;               // pack 0 (whole = 1) and pack whole_end (< end) are the row's ends
  int low, high;         // positions that have a column
  int at, owner;         // position of the target, or -1, and which thread has its pack, if whole, or -1
  bool ignored, inside;  // target
  bool head_outside, tail_outside;  // an end's pack reaches outside the logits: it is not in shared memory
};

struct Shared {
  uint64_t full[kMaxStages], empty[kMaxStages], joined[2];
  Slice slice[kMaxStages];
  float4 warp[2][kMaxWorkers / 32];  // (m, s, target logit, gap) of each warp
  float4 peer[2][kMaxCluster];    // and of each block of the cluster
  int counts[kMaxWorkers / 32];
};

__device__ __forceinline__ uint32_t map_peer(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_peer(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void store_peer(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void arrive_peer(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity) {
  const long long start = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok != 0) return true;
    if (clock64() - start > JK_WAIT_LIMIT_CYCLES) return false;
  }
}

// No block of a cluster ends while another may still write to its shared memory.
__device__ __forceinline__ void leave(int cluster) {
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// The loading warp: slices of rows first, first + step, ... A wait that runs out is recorded and ends the
// loading, after the copies in flight have landed; the workers wait no more after one that runs out of
// theirs. The kernel then ends soon, with an error that jk_device_status reports.
template <typename T, int WORKERS>
__device__ __forceinline__ void load_slices(const Args<T>& a, Shared& sh, unsigned char* memory, int stages, int slice_packs,
                                            int rank, int cluster, int64_t first, int64_t step) {
  constexpr int kP = kPack<T>;
  const int lane = threadIdx.x & 31, vocab = static_cast<int>(a.vocab);
  bool good = true;
  int n = 0, stage = 0;
  uint32_t turn = 0;
  int64_t ahead = 0;
  for (int64_t r = first; r < a.rows; r += step, ++n) {
    if (n % 32 == 0 && r + lane * step < a.rows) ahead = a.targets[r + lane * step];  // of the next 32 rows
    const int64_t target = __shfl_sync(0xffffffffu, static_cast<long long>(ahead), n % 32);
    if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait(&sh.empty[stage], (turn - 1) & 1))) {
      good = false;
      break;
    }
    if (lane == 0) {
      const Window<T> w(a, r);
      const int per = (w.packs + cluster - 1) / cluster;
      const int begin = min(per * rank, w.packs), end = min(begin + per, w.packs);
      const int origin = begin * kP - w.shift;  // column of position 0
      Slice s;
      s.row = r;
      s.in = w.z + origin;
      s.out = a.grad + r * a.grad_stride + origin;
      s.end = end - begin;
      s.low = max(0, -origin);
      s.high = min(s.end * kP, vocab - origin);
      s.whole = s.low > 0 ? 1 : 0;
      s.whole_end = s.end > s.whole && s.high < s.end * kP ? s.end - 1 : s.end;
      s.head_outside = s.whole == 1 && w.z - w.shift < a.logits;
      s.tail_outside = s.whole_end < s.end && w.z - w.shift + w.packs * kP > a.logits + (a.rows - 1) * a.stride + vocab;
      // a row of one pack may leave the logits at both ends
      if (s.whole == 1 && s.end == 1) s.head_outside |= w.z - w.shift + kP > a.logits + (a.rows - 1) * a.stride + vocab;
      s.ignored = target == a.ignore_index;
      s.inside = target >= 0 && target < vocab;
      const int at = s.inside ? static_cast<int>(target) - origin : -1;
      s.at = at >= s.low && at < s.high ? at : -1;
      const int pack = s.at / kP;
      s.owner = s.at >= 0 && pack >= s.whole && pack < s.whole_end ? (pack - s.whole) % WORKERS : -1;
      sh.slice[stage] = s;
      const int from = s.head_outside ? 1 : 0, to = s.tail_outside ? s.whole_end : s.end;
      const uint32_t bytes = !s.ignored && to > from ? static_cast<uint32_t>(to - from) * 16 : 0;
      mbar_arrive_expect_tx(&sh.full[stage], bytes);
      if (bytes > 0)
        bulk_load(memory + (static_cast<size_t>(stage) * slice_packs + from) * 16, static_cast<const T*>(s.in) + from * kP, bytes,
                  &sh.full[stage]);
    }
    __syncwarp();
    if (++stage == stages) stage = 0, ++turn;
  }
  // copies in flight land before the block's memory is given back
  for (int i = 0; i < stages; ++i) {
    const uint32_t loads = turn + (i < stage ? 1 : 0);
    if (loads > 0 && !mbar_wait(&sh.full[i], (loads - 1) & 1)) good = false;
  }
  if (!good) g_device_error = JK_ERR_DEVICE_TIMEOUT;
}

// Adds packs k, k + WORKERS, ... (N of them, those before `end`) to a thread's sum.
template <typename T, int WORKERS, bool SMOOTH, int N>
__device__ __forceinline__ void sum_turn(Sum& v, Gap& gap, float gap_by, const uint4* packs, int k, int end) {
  const T low = minus_inf<T>();
  uint32_t two;
  if constexpr (sizeof(T) == 4) two = __float_as_uint(low);
  else two = *reinterpret_cast<const uint16_t*>(&low) * 0x10001u;
  uint4 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) raw[i] = k + i * WORKERS < end ? packs[k + i * WORKERS] : make_uint4(two, two, two, two);
  const int left = end - k;  // packs of this thread lie WORKERS apart
  take_packs<T, SMOOTH>(v, raw, gap, gap_by, left <= 0 ? 0 : min((left + WORKERS - 1) / WORKERS, N),
                        [&](int i) { return packs[k + i * WORKERS]; });
}

template <typename T, int WORKERS, int PER_SM, bool CLUSTER, bool SMOOTH>
__global__ void __launch_bounds__(WORKERS + 32, PER_SM)
    rows_kernel(const Args<T> a, int stages, int slice_packs, int cluster_size) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ Shared sh;
  __shared__ int gap_counts[SMOOTH ? 2 : 1][kMaxWorkers / 32 + kMaxCluster];  // of the gaps in sh.warp and sh.peer
  constexpr int kP = kPack<T>, kWarps = WORKERS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cluster = CLUSTER ? cluster_size : 1;
  const int rank = CLUSTER ? blockIdx.x % cluster : 0;
  const int64_t first = blockIdx.x / cluster, step = gridDim.x / cluster;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], kWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&sh.joined[i], cluster);
    fence_barrier_init();
  }
  __syncthreads();
  if (CLUSTER) {  // no block reaches for another's barriers before they are set up
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (warp == kWarps) {
    load_slices<T, WORKERS>(a, sh, memory, stages, slice_packs, rank, cluster, first, step);
    leave(cluster);
    return;
  }
  const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory"); };
  const float factor = gradient_factor(a, true, WORKERS, sh.counts, sync);
  const float hit = 1.f - a.smoothing, share = SMOOTH ? a.smoothing / static_cast<float>(a.vocab) : 0.f;
  const float gap_by = SMOOTH ? gap_scale(static_cast<int>(a.vocab)) : 0.f;
  bool good = true;
  double sum = 0.0;
  int counted = 0, stage = 0, joins = 0;
  uint32_t turn = 0;
  for (int64_t r = first; r < a.rows; r += step) {
    if (good) good = mbar_wait(&sh.full[stage], turn & 1);
    const Slice& sl = sh.slice[stage];
    const uint4* packs = reinterpret_cast<const uint4*>(memory) + static_cast<size_t>(stage) * slice_packs;
    const int whole = sl.whole, whole_end = sl.whole_end;
    uint4* out = static_cast<uint4*>(sl.out);
    // the row's ends, an element to a thread: the first pack's for threads 0-7, the last one's for 8-15
    const int in_pack = threadIdx.x & 7;
    int end_at = -1;
    if (threadIdx.x < 16 && in_pack < kP) {
      if (threadIdx.x < 8 ? whole > 0 : whole_end < sl.end) end_at = (threadIdx.x < 8 ? 0 : whole_end * kP) + in_pack;
      if (end_at < sl.low || end_at >= sl.high) end_at = -1;
    }
    const bool outside = threadIdx.x < 8 ? sl.head_outside : sl.tail_outside;
    const auto element = [&](int pos, bool from_logits) {
      return to_f32(from_logits ? static_cast<const T*>(sl.in)[pos] : reinterpret_cast<const T*>(packs)[pos]);
    };
    if (sl.ignored) {
      for (int k = whole + threadIdx.x; k < whole_end; k += WORKERS) out[k] = make_uint4(0, 0, 0, 0);
      if (end_at >= 0) static_cast<T*>(sl.out)[end_at] = from_f32<T>(0.f);
      if (threadIdx.x == 0 && rank == 0) leave_row<false>(a, r, 0.f, 0.f, 0.f);
    } else {
      Sum v{-INFINITY, 0.f};
      Gap gap{0.f, 0};
      float zt = 0.f;
      // turns of kTurn packs while they are mostly full, then of two
      int k = whole + threadIdx.x, left = (whole_end - whole + WORKERS - 1) / WORKERS;
      for (; left > kTurn / 2; left -= kTurn, k += kTurn * WORKERS) sum_turn<T, WORKERS, SMOOTH, kTurn>(v, gap, gap_by, packs, k, whole_end);
      for (; left > 0; left -= 2, k += 2 * WORKERS) sum_turn<T, WORKERS, SMOOTH, 2>(v, gap, gap_by, packs, k, whole_end);
      if (end_at >= 0) {
        const float z = element(end_at, outside), before = v.m;
        float f[1] = {z};
        take(v, f);
        if (SMOOTH) {
          gap.move(before, v.m, gap_by);
          gap.add(z, v.m, gap_by);
        }
      }
      if (threadIdx.x == 0 && sl.at >= 0)
        zt = element(sl.at, (sl.at < kP && sl.head_outside) || (sl.at >= whole_end * kP && sl.tail_outside));
      const float mine = v.m;
      v = warp_join(v);
      if (SMOOTH) gap.join(mine, v.m, gap_by);
      // of three rows that count, the warps of a block are never in the first and the third at once
      if (lane == 0) {
        sh.warp[joins & 1][warp] = make_float4(v.m, v.s, zt, gap.sum);
        if (SMOOTH) gap_counts[joins & 1][warp] = gap.n;
      }
      sync();
      float4 q = lane < kWarps ? sh.warp[joins & 1][lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      v = warp_join({q.x, q.y});
      if (SMOOTH) {
        gap = {q.w, lane < kWarps ? gap_counts[joins & 1][lane] : 0};
        gap.join(q.x, v.m, gap_by);
      }
      zt = q.z;  // of the first warp's first thread
      if (CLUSTER) {  // neither are the blocks of a cluster, so a slot and a barrier are free again
        zt = __shfl_sync(0xffffffffu, zt, 0);
        if (threadIdx.x < cluster) {
          store_peer(map_peer(&sh.peer[joins & 1][rank], threadIdx.x), make_float4(v.m, v.s, zt, gap.sum));
          if (SMOOTH) store_peer(map_peer(&gap_counts[joins & 1][kMaxWorkers / 32 + rank], threadIdx.x), gap.n);
          arrive_peer(map_peer(&sh.joined[joins & 1], threadIdx.x));
        }
        if (good) good = wait_cluster(&sh.joined[joins & 1], (joins >> 1) & 1);
        q = lane < cluster ? sh.peer[joins & 1][lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
        v = warp_join({q.x, q.y});
        zt = warp_sum32(q.z);
        if (SMOOTH) {
          gap = {q.w, lane < cluster ? gap_counts[joins & 1][kMaxWorkers / 32 + lane] : 0};
          gap.join(q.x, v.m, gap_by);
        }
      }
      ++joins;
      if (threadIdx.x == 0 && rank == 0) {
        const RowLoss l(v, sl.inside ? zt : NAN, gap.sum, a.smoothing, static_cast<int>(a.vocab));
        leave_row<false>(a, r, l.loss, l.lse, l.low);
        sum += l.loss;
        ++counted;
      }
      const Base base(v.m);
      const float c0 = sl.inside ? factor : NAN, scale = __fdividef(c0, v.s), other = -share * c0;
      for (k = whole + threadIdx.x; k < whole_end; k += 3 * WORKERS) {
        uint4 raw[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) raw[i] = packs[min(k + i * WORKERS, whole_end - 1)];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (k + i * WORKERS >= whole_end) continue;
          float f[kP];
          unpack<T>(raw[i], f);
          gradient_pack<T>(f, base, scale, other);
          out[k + i * WORKERS] = pack<T>(f);
        }
      }
      if (threadIdx.x == sl.owner)  // after its pack
        static_cast<T*>(sl.out)[sl.at] = from_f32<T>(fmaf(base.exp(element(sl.at, false)), scale, other) - hit * c0);
      if (end_at >= 0)
        static_cast<T*>(sl.out)[end_at] =
            from_f32<T>(fmaf(base.exp(element(end_at, outside)), scale, other) - (end_at == sl.at ? hit * c0 : 0.f));
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[stage]);
    if (++stage == stages) stage = 0, ++turn;
  }
  if (!good) g_device_error = JK_ERR_DEVICE_TIMEOUT;
  grid_dependency_launch();
  if (threadIdx.x == 0) a.partials[blockIdx.x] = {sum, counted};
  leave(cluster);
}

// ---------------------------------------------------------------- reduction over rows
// The partial sums in their order, and the rows that warps have left in parts. The last block to
// come adds up what the blocks have (the order of the sum does not depend on which that is).
constexpr int kReduceBlocks = 32;  // a lane for each

__device__ __forceinline__ Partial warp_add(Partial p) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    p.sum += __shfl_xor_sync(0xffffffffu, p.sum, o);
    p.rows += __shfl_xor_sync(0xffffffffu, p.rows, o);
  }
  return p;
}

struct Ticket {
  Partial blocks[kReduceBlocks];
  int come;
};

template <typename T>
__global__ void __launch_bounds__(256)
    reduce_kernel(const Args<T> a, int partials, const Record* records, int record_count, float* loss, Ticket* ticket) {
  __shared__ Partial parts[8];
  grid_dependency_wait();
  const int at = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  Partial p{0.0, 0};
  for (int i = at; i < partials; i += step) {
    p.sum += a.partials[i].sum;
    p.rows += a.partials[i].rows;
  }
  for (int i = at; i < record_count; i += step) {
    const Record head = records[i];
    if (head.row < 0) continue;
    const int64_t target = a.targets[head.row];
    const float zt = target >= 0 && target < a.vocab ? to_f32(a.logits[head.row * a.stride + target]) : NAN;
    // the records of a row follow one another, with one unused between two of them at most
    const bool begun = (i >= 1 && records[i - 1].row == head.row) || (i >= 2 && records[i - 2].row == head.row);
    if (begun) continue;
    Sum v{head.m, head.s};
    Gap gap{head.gap, head.n};
    const float gap_by = gap_scale(static_cast<int>(a.vocab));
    for (int j = i + 1, unused = 0; j < record_count && unused < 2; ++j) {
      const Record q = records[j];
      if (q.row < 0) {
        ++unused;
        continue;
      }
      if (q.row != head.row) break;
      unused = 0;
      const float m = fmaxf(v.m, q.m);
      const float f = v.m == m ? 1.f : factor_to(v.m, m), g = q.m == m ? 1.f : factor_to(q.m, m);
      Gap other{q.gap, q.n};
      gap.move(v.m, m, gap_by);
      other.move(q.m, m, gap_by);
      gap.sum += other.sum;
      gap.n += other.n;
      v = {m, v.s * f + q.s * g};
    }
    const RowLoss l(v, zt, gap.sum, a.smoothing, static_cast<int>(a.vocab));
    leave_row<true>(a, head.row, l.loss, l.lse, l.low);
    p.sum += l.loss;
    p.rows += 1;
  }
  p = warp_add(p);
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = p;
  __syncthreads();
  if (threadIdx.x >= 32 || loss == nullptr) return;
  p = warp_add(threadIdx.x < 8 ? parts[threadIdx.x] : Partial{0.0, 0});
  if (gridDim.x > 1) {
    int order = 0;
    if (threadIdx.x == 0) {
      ticket->blocks[blockIdx.x] = p;
      __threadfence();
      order = atomicAdd(&ticket->come, 1);
    }
    if (__shfl_sync(0xffffffffu, order, 0) != static_cast<int>(gridDim.x) - 1) return;
    __threadfence();
    const volatile Partial* q = &ticket->blocks[threadIdx.x];
    p.sum = q->sum;
    p.rows = q->rows;
    p = warp_add(p);
  }
  if (threadIdx.x == 0) *loss = static_cast<float>(a.reduction == JK_REDUCE_MEAN ? p.sum / static_cast<double>(p.rows) : p.sum);
}

// ---------------------------------------------------------------- launches
// The caller's workspace. (With one record for each of a warp's runs' ends.)
struct Workspace {
  Partial partials[kMaxWarps > kMaxBlocks ? kMaxWarps : kMaxBlocks];
  Record records[2 * kMaxWarps];
  Ticket ticket;
  int counts[kCounts];
};

constexpr int kWarpColumns = 1024;  // of the rows that a warp holds

template <typename T, int MODE, int VEC, int THREADS>
void launch_warps(const Args<T>& a, int blocks, cudaStream_t s) {
  const int64_t turns = (a.vocab + 32 * VEC - 1) / (32 * VEC);
  constexpr int kMost = kWarpColumns / 32 / VEC;
  if constexpr (VEC == 1) {
    if (turns <= 2) warp_kernel<T, MODE, VEC, 2, THREADS><<<blocks, THREADS, 0, s>>>(a);
    else if (turns <= 8) warp_kernel<T, MODE, VEC, 8, THREADS><<<blocks, THREADS, 0, s>>>(a);
    else warp_kernel<T, MODE, VEC, kMost, THREADS><<<blocks, THREADS, 0, s>>>(a);
  } else {
    if (turns <= 1) warp_kernel<T, MODE, VEC, 1, THREADS><<<blocks, THREADS, 0, s>>>(a);
    else if (turns <= 2) warp_kernel<T, MODE, VEC, 2, THREADS><<<blocks, THREADS, 0, s>>>(a);
    else warp_kernel<T, MODE, VEC, kMost, THREADS><<<blocks, THREADS, 0, s>>>(a);
  }
}

// What the reduction over rows will find.
struct Left {
  int partials = 0, records = 0;
};

template <typename T, int MODE>
Left launch_stream(const Args<T>& a, Workspace* ws, cudaStream_t s) {
  const int packs = static_cast<int>((a.vocab + 2 * (kPack<T> - 1)) / kPack<T>);  // of a row, wherever it begins
  const int pieces = (packs + kPiece - 1) / kPiece;
  // a run of four pieces or more keeps the records of a row few
  const int64_t want = (a.rows * pieces + 4 * (kStreamThreads / 32) - 1) / (4 * (kStreamThreads / 32));
  const int blocks = static_cast<int>(want < 148 * kStreamBlocksPerSm ? want : 148 * kStreamBlocksPerSm);
  if (MODE == kLoss && a.smoothing != 0.f)
    stream_kernel<T, MODE, MODE == kLoss><<<blocks, kStreamThreads, 0, s>>>(a, pieces, ws->records, &ws->ticket.come);
  else
    stream_kernel<T, MODE, false><<<blocks, kStreamThreads, 0, s>>>(a, pieces, ws->records, &ws->ticket.come);
  return {blocks * (kStreamThreads / 32), 2 * blocks * (kStreamThreads / 32)};
}

constexpr int64_t kRoom = 212 * 1024;  // of an SM's shared memory, for the slices of all its blocks
constexpr int64_t kFewRows = 74;       // so few rows leave half of the SMs without a block

template <typename T, int WORKERS, int PER_SM, bool CLUSTER, bool SMOOTH>
bool launch_rows(const Args<T>& a, int64_t blocks, int stages, int slice_packs, int cluster, cudaStream_t s) {
  auto kernel = rows_kernel<T, WORKERS, PER_SM, CLUSTER, SMOOTH>;
  const size_t smem = static_cast<size_t>(stages) * slice_packs * 16;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) return false;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(WORKERS + 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CLUSTER ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, stages, slice_packs, cluster) == cudaSuccess;
}

// Slices of this many packs, WORKERS threads and up to PER_SM blocks on an SM. Returns the blocks.
template <typename T, int WORKERS, int PER_SM>
int run_rows(const Args<T>& a, int slice, int cluster, cudaStream_t s) {
  int per_sm = PER_SM;
  while (per_sm > 1 && 2 * 16ll * slice * per_sm > kRoom) --per_sm;
  const int64_t fit = kRoom / per_sm / (16ll * slice);
  const int stages = static_cast<int>(fit < kMaxStages ? fit : kMaxStages);
  int64_t clusters = 148 * per_sm / cluster;
  if (clusters > a.rows) clusters = a.rows;
  const int64_t blocks = clusters * cluster;
  const bool smooth = a.smoothing != 0.f;
  bool done;
  if (cluster > 1) done = smooth ? launch_rows<T, WORKERS, PER_SM, true, true>(a, blocks, stages, slice, cluster, s) : launch_rows<T, WORKERS, PER_SM, true, false>(a, blocks, stages, slice, cluster, s);
  else done = smooth ? launch_rows<T, WORKERS, PER_SM, false, true>(a, blocks, stages, slice, cluster, s) : launch_rows<T, WORKERS, PER_SM, false, false>(a, blocks, stages, slice, cluster, s);
  return done ? static_cast<int>(blocks) : -1;
}

// Returns the blocks that left a partial.
template <typename T, int MODE>
int launch_warp_rows(const Args<T>& a, cudaStream_t s) {
  const bool aligned = a.vocab % kPack<T> == 0 && a.stride % kPack<T> == 0 && aligned16(a.logits) &&
                       (MODE == kLoss || (a.grad_stride % kPack<T> == 0 && aligned16(a.grad)));
  if constexpr (MODE != kBackward) {
    if (a.loss_now != nullptr) {
      if (aligned) launch_warps<T, MODE, kPack<T>, kOneBlockThreads>(a, 1, s);
      else launch_warps<T, MODE, 1, kOneBlockThreads>(a, 1, s);
      return 0;
    }
  }
  const int64_t want = (a.rows + kWarpThreads / 32 - 1) / (kWarpThreads / 32);
  const int blocks = static_cast<int>(want < kMaxBlocks ? want : kMaxBlocks);
  if (aligned) launch_warps<T, MODE, kPack<T>, kWarpThreads>(a, blocks, s);
  else launch_warps<T, MODE, 1, kWarpThreads>(a, blocks, s);
  return blocks;
}

// Both at once, where rows_kernel can: gradient and logits lie alike against 16 bytes, and two slices
// (one that is worked on, one on its way) fit the block's shared memory. A row is one block's, but for
// few rows, which a cluster of blocks shares; longer rows in greater number are read twice instead
// (1500 x 60000 f32: 186 us, 236 with clusters of eight). Returns the partials, or 0.
template <typename T>
int launch_both(const Args<T>& a, cudaStream_t s) {
  const bool alike = (a.stride - a.grad_stride) % kPack<T> == 0 &&
                     ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0;
  const int64_t packs = (a.vocab + 2 * (kPack<T> - 1)) / kPack<T>;
  if (!alike || 2 * 16 * packs > kRoom * (a.rows <= kFewRows ? kMaxCluster : 1)) return 0;
  int cluster = 1;
  while (cluster < kMaxCluster && a.rows * cluster <= kFewRows &&
         (2 * 16 * ((packs + cluster - 1) / cluster) > kRoom || packs >= 1024 * cluster))
    cluster *= 2;
  const int slice = static_cast<int>((packs + cluster - 1) / cluster);
  if (2 * 16ll * slice > kRoom) return 0;
  // Threads by the slice's length: some eight packs each, so that what a row costs apart from its packs
  // is spread over them, and as many blocks as an SM then holds. (4096 x 16384 bf16: 52.5 us with 256
  // threads and three blocks, 57.8 with 128 and six, 66 with 480 and two; 16000 x 2500: 53 with 64 and
  // eight, 69 with 128 and six, 105 with 256 and three.)
  if (slice <= 600) return run_rows<T, 64, 8>(a, slice, cluster, s);
  if (slice <= 1200) return run_rows<T, 128, 6>(a, slice, cluster, s);
  if (slice <= 2400) return run_rows<T, 256, 3>(a, slice, cluster, s);
  return run_rows<T, 480, 2>(a, slice, cluster, s);
}

// Where many rows have to be counted for the gradient's factor, a kernel of its own does it first.
template <typename T>
void count_apart(Args<T>& a, Workspace* ws, cudaStream_t s) {
  if (a.reduction != JK_REDUCE_MEAN || a.rows <= kCountRows) return;
  count_kernel<<<kCounts, 256, 0, s>>>(a.targets, a.rows, a.ignore_index, ws->counts);
  a.counts = ws->counts;
}

template <typename T>
int backward(Args<T> a, Workspace* ws, cudaStream_t s) {
  count_apart(a, ws, s);
  if (a.vocab <= kWarpColumns) launch_warp_rows<T, kBackward>(a, s);
  else launch_stream<T, kBackward>(a, ws, s);
  return launch_status();
}

template <typename T>
int forward(Args<T> a, float* loss, Workspace* ws, cudaStream_t s) {
  Left left;
  bool gradient_later = false;
  a.partials = ws == nullptr ? nullptr : ws->partials;
  if (a.rows > 0) {
    if (a.grad != nullptr) count_apart(a, ws, s);
    if (a.vocab <= kWarpColumns) {
      if (a.rows <= kOneBlockRows) a.loss_now = loss;
      left.partials = a.grad != nullptr ? launch_warp_rows<T, kBoth>(a, s) : launch_warp_rows<T, kLoss>(a, s);
      if (a.loss_now != nullptr) loss = nullptr;
    } else {
      if (a.grad != nullptr) left.partials = launch_both(a, s);
      if (left.partials < 0) {
        cudaGetLastError();
        return JK_ERR_LAUNCH;
      }
      if (left.partials == 0) {
        gradient_later = a.grad != nullptr;
        if (gradient_later) {  // from the log-sum, kept in two parts: one f32 does not tell its neighbours apart far from 0
          if (a.lse_out == nullptr) a.lse_out = reinterpret_cast<float*>(ws + 1);
          a.low_out = reinterpret_cast<float*>(ws + 1) + a.rows;
        }
        left = launch_stream<T, kLoss>(a, ws, s);
      }
    }
  }
  if (loss != nullptr || left.records > 0) {
    launch_dependent(reduce_kernel<T>, left.records > 0 ? kReduceBlocks : 1, 256, 0, s, a, left.partials, ws == nullptr ? nullptr : ws->records, left.records, loss,
                     ws == nullptr ? nullptr : &ws->ticket);
  }
  if (gradient_later) {
    a.lse_in = a.lse_out;
    a.low_in = a.low_out;
    launch_stream<T, kLater>(a, ws, s);
  }
  return launch_status();
}

}  // namespace loss

JK_ERROR_READER(read_error_loss)

}  // namespace jk

namespace jk {
namespace loss {

int checked_forward(const void* logits, int64_t logits_stride, const int64_t* targets, int64_t rows, int64_t vocab, int dtype,
                    int64_t ignore_index, float label_smoothing, int reduction, float grad_scale, float* losses, float* lse,
                    float* lse_low, float* loss, void* grad, int64_t grad_stride, void* workspace, jk_stream_t stream) {
  if (rows < 0 || vocab <= 0 || vocab > kMaxVocab || logits_stride < 0 || grad_stride < 0) return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype)) return JK_ERR_BAD_DTYPE;
  if (reduction < JK_REDUCE_NONE || reduction > JK_REDUCE_SUM) return JK_ERR_UNSUPPORTED_KIND;
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f)) return JK_ERR_BAD_ARG;
  if ((loss == nullptr) != (reduction == JK_REDUCE_NONE) || (grad != nullptr && reduction == JK_REDUCE_NONE))
    return JK_ERR_BAD_ARG;
  if (rows > 0 && (logits == nullptr || targets == nullptr || workspace == nullptr)) return JK_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(workspace) & 7u) != 0) return JK_ERR_ALIGNMENT;
  int st = check_device();
  if (st != JK_OK) return st;
  JK_WITH_TYPE(dtype, T, {
    const Args<T> a{static_cast<const T*>(logits), logits_stride, targets, rows, vocab, ignore_index,
                    label_smoothing, reduction, grad_scale, nullptr, nullptr, nullptr, losses, lse, lse_low,
                    static_cast<T*>(grad), grad_stride, nullptr, nullptr, nullptr};
    st = forward<T>(a, loss, static_cast<Workspace*>(workspace), reinterpret_cast<cudaStream_t>(stream));
  });
  return st;
}

int checked_backward(const float* grad_loss, const void* logits, int64_t logits_stride, const int64_t* targets, const float* lse,
                     const float* lse_low, int64_t rows, int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                     int reduction, void* grad, int64_t grad_stride, void* workspace, jk_stream_t stream) {
  if (rows < 0 || vocab <= 0 || vocab > kMaxVocab || logits_stride < 0 || grad_stride < 0) return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype)) return JK_ERR_BAD_DTYPE;
  if (reduction < JK_REDUCE_NONE || reduction > JK_REDUCE_SUM) return JK_ERR_UNSUPPORTED_KIND;
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f)) return JK_ERR_BAD_ARG;
  if (rows == 0) return JK_OK;
  if (grad_loss == nullptr || logits == nullptr || targets == nullptr || lse == nullptr || grad == nullptr ||
      workspace == nullptr)
    return JK_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(workspace) & 7u) != 0) return JK_ERR_ALIGNMENT;
  int st = check_device();
  if (st != JK_OK) return st;
  JK_WITH_TYPE(dtype, T, {
    const Args<T> a{static_cast<const T*>(logits), logits_stride, targets, rows, vocab, ignore_index,
                    label_smoothing, reduction, 1.f, grad_loss, lse, lse_low, nullptr, nullptr, nullptr, static_cast<T*>(grad),
                    grad_stride, nullptr, nullptr, nullptr};
    st = backward<T>(a, static_cast<Workspace*>(workspace), reinterpret_cast<cudaStream_t>(stream));
  });
  return st;
}

}  // namespace loss
}  // namespace jk

extern "C" int64_t jk_cross_entropy_workspace(int64_t rows) {
  // and a log-sum of each row, in two parts, for a gradient that is taken in a second pass
  return rows <= 0 ? 0 : static_cast<int64_t>(sizeof(jk::loss::Workspace)) + rows * 8;
}

extern "C" int jk_cross_entropy_forward(const void* logits, int64_t logits_stride, const int64_t* targets, int64_t rows,
                                        int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                                        int reduction, float grad_scale, float* losses, float* lse, float* loss,
                                        void* grad, int64_t grad_stride, void* workspace, jk_stream_t stream) {
  return jk::loss::checked_forward(logits, logits_stride, targets, rows, vocab, dtype, ignore_index, label_smoothing, reduction,
                                   grad_scale, losses, lse, nullptr, loss, grad, grad_stride, workspace, stream);
}

extern "C" int jk_cross_entropy_forward_split(const void* logits, int64_t logits_stride, const int64_t* targets, int64_t rows,
                                              int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                                              int reduction, float* losses, float* lse, float* lse_low, float* loss,
                                              void* workspace, jk_stream_t stream) {
  return jk::loss::checked_forward(logits, logits_stride, targets, rows, vocab, dtype, ignore_index, label_smoothing, reduction,
                                   1.f, losses, lse, lse_low, loss, nullptr, 0, workspace, stream);
}

extern "C" int jk_cross_entropy_backward(const float* grad_loss, const void* logits, int64_t logits_stride,
                                         const int64_t* targets, const float* lse, int64_t rows, int64_t vocab, int dtype,
                                         int64_t ignore_index, float label_smoothing, int reduction, void* grad,
                                         int64_t grad_stride, void* workspace, jk_stream_t stream) {
  return jk::loss::checked_backward(grad_loss, logits, logits_stride, targets, lse, nullptr, rows, vocab, dtype, ignore_index,
                                    label_smoothing, reduction, grad, grad_stride, workspace, stream);
}

extern "C" int jk_cross_entropy_backward_split(const float* grad_loss, const void* logits, int64_t logits_stride,
                                               const int64_t* targets, const float* lse, const float* lse_low, int64_t rows,
                                               int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                                               int reduction, void* grad, int64_t grad_stride, void* workspace,
                                               jk_stream_t stream) {
  return jk::loss::checked_backward(grad_loss, logits, logits_stride, targets, lse, lse_low, rows, vocab, dtype, ignore_index,
                                    label_smoothing, reduction, grad, grad_stride, workspace, stream);
}
