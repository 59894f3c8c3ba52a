// Verification of drafted tokens from given random numbers (jk_verify_draft).
//
// Token i of a sequence, drawn from the draft's q_i, is accepted while u_i q_i(x_i) < p_i(x_i). With
// the first place a that is not, the new token is drawn from r = max(p_a - q_a, 0), which makes the
// sequence one of the target's: it is the least j at which the running sum of r passes u r's total.
// Where all are accepted r is the target's next distribution.
//
// A comparison of a product or of a running sum decides a token, so both are in f64: products of two
// f32 are exact there, and a running sum is off by less than 2^-40 + m 2^-53 of the total (m:
// entries that a lane adds up, at most 2^18 for a few sequences and 2^23 for many), where f32 would
// give another token in one of some thousand draws over a vocabulary of 100,000. Conversions to f64
// are the slowest part (16 a cycle and SM), so a difference takes one: d = x - y in f32, whose
// rounding error (x - d) - y is exact there for x >= y >= 0, and errors are added up on their own,
// in f32 up to 128 of them.
//
// Of the draft's and the target's rows only place a's are read, once: a cluster of blocks per
// sequence adds them up by warps, each a run of 16-byte packs; the run that holds the draw is cut
// into runs again, one for each warp of its block, until one warp finds the token (the second look
// at a run comes from L2). Bound: for a batch the issue of instructions (14.5 an entry) and, in the end,
// the steps that find the token: 25 us on the device for 256 sequences of 100003 bf16 entries, of which
// 14 for the memory; for a few sequences the latency of these steps (8.6 us for one of 131072 f32
// entries, 5.6 for one of 1000).
#include <cooperative_groups.h>

#include "jk_host.h"
#include "jk_rows.cuh"

#include <type_traits>

namespace jk {
namespace verify {

constexpr int kFew = 512, kMany = 128;  // threads of a block, for few sequences and for many
constexpr int kManyPerSm = 7;
constexpr int kLoads = 2;               // packs of a lane whose loads are on their way together
constexpr int kMaxCluster = 8;
constexpr int kSms = 148;

struct Args {
  const void *target, *draft;
  int64_t target_b, target_t, draft_b, draft_t;
  const int64_t* tokens;
  const float* uniform;
  const int32_t* counts;
  int32_t drafted, vocab;
  int64_t* out;
  int32_t* accepted;
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// NaN and negative values count as 0.
__device__ __forceinline__ float mass(float v) { return fmaxf(v, 0.0f); }

// Packs of both as 0 <= y <= x: 16-bit types two at a time.
template <typename T>
__device__ __forceinline__ void bounded(const uint4& u, const uint4& v, float (&x)[kPack<T>], float (&y)[kPack<T>]) {
  if constexpr (sizeof(T) == 4) {
    unpack<T>(u, x);
    unpack<T>(v, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = mass(x[e]), y[e] = fminf(mass(y[e]), x[e]);
  } else {
    using P = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    uint4 a = u, b = v;
    P *pa = reinterpret_cast<P*>(&a), *pb = reinterpret_cast<P*>(&b);
    const uint32_t none = 0;
    const P zero = *reinterpret_cast<const P*>(&none);
#pragma unroll
    for (int i = 0; i < 4; ++i) pa[i] = __hmax2(pa[i], zero), pb[i] = __hmin2(__hmax2(pb[i], zero), pa[i]);
    unpack<T>(a, x);
    unpack<T>(b, y);
  }
}

// One place's r: packs of E entries on the 16-byte blocks of the target's row.
template <typename T>
struct Rest {
  static constexpr int E = kPack<T>;
  const T *p, *q;   // q null: 0 throughout
  int32_t without;  // this entry is 0 (the token that a certain draft had), -1: none
  int32_t vocab, head, packs;
  uint32_t apart;   // bytes by which the draft's packs begin inside a 16-byte block

  __device__ __forceinline__ Rest(const T* p_, const T* q_, int32_t without_, int32_t vocab_)
      : p(p_), q(q_), without(without_), vocab(vocab_) {
    head = static_cast<int32_t>((reinterpret_cast<uintptr_t>(p_) & 15) / sizeof(T));
    packs = (head + vocab + E - 1) / E;
    apart = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(q_) - reinterpret_cast<uintptr_t>(p_)) & 15u;
  }

  // Entries [E k - head, E k - head + E) of both, as 0 <= y <= x; those outside the row, and `without`, are 0.
  __device__ __forceinline__ void load(int32_t k, float (&x)[E], float (&y)[E]) const {
    const int32_t j = k * E - head;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = j + e >= 0 && j + e < vocab && j + e != without;
      x[e] = mass(in ? to_f32(p[j + e]) : 0.0f);
      y[e] = fminf(mass(in && q != nullptr ? to_f32(q[j + e]) : 0.0f), x[e]);
    }
  }

  // s + lost: the sum of x - y; two differences at a time.
  static __device__ __forceinline__ void add(const float (&x)[E], const float (&y)[E], double& s, uint64_t& lost) {
    const uint64_t minus = pair(-1.0f, -1.0f);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const uint64_t x2 = pair(x[e], x[e + 1]), y2 = pair(y[e], y[e + 1]);
      const uint64_t d = fma2(y2, minus, x2);
      lost = add2(lost, fma2(y2, minus, fma2(d, minus, x2)));
      const float2 f = unpair(d);
      s += static_cast<double>(f.x);
      s += static_cast<double>(f.y);
    }
  }

  // Over packs [from, to), a warp. WORDS: apart / 4, known where the loop is compiled, as selecting
  // words would take most of its time; 4: there is no draft.
  template <int WORDS>
  __device__ __forceinline__ double sum_of(int32_t from, int32_t to) const {
    const int lane = threadIdx.x & 31;
    double s = 0.0;
    uint64_t lost = 0;
    // packs that lie in the row as a whole, [low, high): their loads go out kLoads at a time
    const int32_t first = head > 0 ? 1 : 0, past = (head + vocab) / E;
    const int32_t low = from > first ? from : first, high = to < past ? to : past;
    const int32_t odd = without >= 0 ? (without + head) / E : -1;
    auto fetch = [&](int32_t k, uint4& u, uint4& v, uint4& n) {
      const int32_t j = k * E - head;
      u = *reinterpret_cast<const uint4*>(p + j);
      v = n = make_uint4(0, 0, 0, 0);
      if (WORDS < 4) {
        const uint4* block = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(q + j) - apart);
        v = block[0];
        if (WORDS > 0 || apart != 0) n = block[1];
      }
    };
    auto take = [&](int32_t k, const uint4& u, uint4 v, const uint4& n) {
      if (WORDS < 4) {
        const uint32_t w[8] = {v.x, v.y, v.z, v.w, n.x, n.y, n.z, n.w}, bits = (apart & 3) * 8;
        constexpr int W = WORDS & 3;
        v = make_uint4(__funnelshift_r(w[W], w[W + 1], bits), __funnelshift_r(w[W + 1], w[W + 2], bits),
                       __funnelshift_r(w[W + 2], w[W + 3], bits), __funnelshift_r(w[W + 3], w[W + 4], bits));
      }
      float x[E], y[E];
      bounded<T>(u, v, x, y);
      if (WORDS == 4 && k == odd) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (odd * E - head + e == without) x[e] = 0.0f;
      }
      add(x, y, s, lost);
    };
    int32_t k = low + lane;
    // errors go over into the sum after at most 128 of them, so that their own rounding does not
    // grow with the vocabulary
    auto over = [&] {
      const float2 some = unpair(lost);
      s += static_cast<double>(some.x) + static_cast<double>(some.y);
      lost = 0;
    };
    int pending = 0;
    for (; k + 32 * (kLoads - 1) < high; k += 32 * kLoads) {
      if (++pending > 128 / (kLoads * E / 2)) over(), pending = 1;
      uint4 u[kLoads], v[kLoads], n[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) fetch(k + 32 * i, u[i], v[i], n[i]);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) take(k + 32 * i, u[i], v[i], n[i]);
    }
#pragma unroll 1
    for (; k < high; k += 32) {
      uint4 u, v, n;
      fetch(k, u, v, n);
      take(k, u, v, n);
    }
    // the row's first and last pack, where other data share them
    const int32_t edge = lane == 0 ? 0 : packs - 1;
    if (lane < 2 && edge >= from && edge < to && (edge < first || edge >= past) && (lane == 0 || packs > 1)) {
      float x[E], y[E];
      load(edge, x, y);
      add(x, y, s, lost);
    }
    over();
    return warp_sum64(s);
  }

  // Over packs [from, to), a warp.
  __device__ __forceinline__ double sum(int32_t from, int32_t to) const {
    if (q == nullptr) return sum_of<4>(from, to);
    switch (apart >> 2) {
      case 0: return sum_of<0>(from, to);
      case 1: return sum_of<1>(from, to);
      case 2: return sum_of<2>(from, to);
      default: return sum_of<3>(from, to);
    }
  }
};

// The part (of n, their sums given) that holds `draw` when the parts are laid one after the other
// from `before`: the first whose end passes it, else (the sums' rounding) the last that is not empty;
// -1: all are empty. before: receives where that part begins.
__device__ __forceinline__ int part_of(const double* sums, int n, double draw, double& before) {
  int best = -1;
  double at = before, begin = before;
  for (int i = 0; i < n; ++i) {
    if (sums[i] > 0.0) {
      best = i, begin = at;
      if (at + sums[i] > draw) break;
    }
    at += sums[i];
  }
  before = begin;
  return best;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == kMany ? kManyPerSm : 2) verify_kernel(const Args g) {
  constexpr int kWarps = THREADS / 32;
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  __shared__ double sums[kWarps];
  __shared__ double totals[kMaxCluster];
  __shared__ int32_t first, token;
  cluster.barrier_arrive();  // before another block writes here, this one has begun
  const int rank = cluster.block_rank(), size = cluster.num_blocks();
  const int64_t b = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int32_t n = g.counts == nullptr ? g.drafted : g.counts[b];
  n = n < 0 ? 0 : n > g.drafted ? g.drafted : n;
  const T* target = static_cast<const T*>(g.target) + b * g.target_b;
  const T* draft = g.draft == nullptr ? nullptr : static_cast<const T*>(g.draft) + b * g.draft_b;
  const int64_t* tokens = g.tokens + b * g.drafted;
  const float* uniform = g.uniform + b * (g.drafted + 1);
  if (tid == 0) first = n;
  __syncthreads();
  for (int32_t i = tid; i < n; i += THREADS) {
    const int64_t x = tokens[i];
    bool ok = false;
    if (x >= 0 && x < g.vocab) {
      const float q = draft == nullptr ? 1.0f : mass(to_f32(draft[i * g.draft_t + x]));
      ok = static_cast<double>(uniform[i]) * static_cast<double>(q) < static_cast<double>(mass(to_f32(target[i * g.target_t + x])));
    }
    if (!ok) atomicMin(&first, i);
  }
  __syncthreads();
  const int32_t a = first;
  const bool rejected = a < n;
  const int64_t x = rejected ? tokens[a] : -1;
  Rest<T> rest(target + a * g.target_t, rejected && draft != nullptr ? draft + a * g.draft_t : nullptr,
               rejected && draft == nullptr && x >= 0 && x < g.vocab ? static_cast<int32_t>(x) : -1, g.vocab);
  const double u = static_cast<double>(uniform[g.drafted]);
  // this block's run of packs, and each warp's of it
  const int32_t mine = (rest.packs + size - 1) / size;
  int32_t from = rank * mine < rest.packs ? rank * mine : rest.packs;
  int32_t to = from + mine < rest.packs ? from + mine : rest.packs;
  double total = 0.0;
  for (int turn = 0; turn < 2; ++turn) {
    const int32_t each = (to - from + kWarps - 1) / kWarps;
    const int32_t low = from + warp * each < to ? from + warp * each : to;
    const double s = rest.sum(low, low + each < to ? low + each : to);
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    if (turn == 0) cluster.barrier_wait();
    if (tid < size) {
      double all = 0.0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) all += sums[w];
      *cluster.map_shared_rank(&totals[rank], tid) = all;
    }
    cluster.sync();
    total = 0.0;
    for (int i = 0; i < size; ++i) total += totals[i];
    // without mass (the target is nowhere above the draft): the target itself
    if (total > 0.0 || !rejected || turn == 1) break;
    rest.q = nullptr, rest.without = -1;
    cluster.sync();  // the totals have been read
  }
  double draw = u * total, before = 0.0;
  const int owner = part_of(totals, size, draw, before);
  if (owner == rank) {
    // the run that holds the draw, cut into the warps' runs until it is a few packs
    double begin = before;
    while (true) {
      const int32_t each = (to - from + kWarps - 1) / kWarps;
      const int w = part_of(sums, kWarps, draw, begin);
      from = from + w * each < to ? from + w * each : to;  // w >= 0: the run has mass
      to = from + each < to ? from + each : to;
      if (to - from <= 64) break;
      __syncthreads();  // the sums have been read
      const int32_t next = (to - from + kWarps - 1) / kWarps;
      const int32_t low = from + warp * next < to ? from + warp * next : to;
      const double s = rest.sum(low, low + next < to ? low + next : to);
      if (lane == 0) sums[warp] = s;
      __syncthreads();
    }
    if (warp == 0) {
      int32_t found = -1, last = -1;
      for (int32_t k0 = from; k0 < to && found < 0; k0 += 32) {
        float x[Rest<T>::E] = {}, y[Rest<T>::E] = {};
        if (k0 + lane < to) rest.load(k0 + lane, x, y);
        double r[Rest<T>::E];
#pragma unroll
        for (int e = 0; e < Rest<T>::E; ++e) r[e] = static_cast<double>(x[e]) - static_cast<double>(y[e]);
        double own = 0.0;
#pragma unroll
        for (int e = 0; e < Rest<T>::E; ++e) own += r[e];
        double upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        const double all = __shfl_sync(0xffffffffu, upto, 31);
        double at = begin + (upto - own);
        int32_t here = -1, positive = -1;
#pragma unroll
        for (int e = 0; e < Rest<T>::E; ++e) {
          at += r[e];
          if (r[e] > 0.0) {
            positive = (k0 + lane) * Rest<T>::E - rest.head + e;
            if (here < 0 && at > draw) here = positive;
          }
        }
        const unsigned hits = __ballot_sync(0xffffffffu, here >= 0), some = __ballot_sync(0xffffffffu, positive >= 0);
        if (hits != 0) found = __shfl_sync(0xffffffffu, here, __ffs(hits) - 1);
        if (some != 0) last = __shfl_sync(0xffffffffu, positive, 31 - __clz(some));
        begin += all;
      }
      if (lane == 0) token = found >= 0 ? found : last;
    }
  } else if (tid == 0) {
    token = -1;
  }
  __syncthreads();
  if (owner == rank || (owner < 0 && rank == 0)) {
    int64_t* out = g.out + b * (g.drafted + 1);
    for (int32_t i = tid; i <= g.drafted; i += THREADS) out[i] = i < a ? tokens[i] : i == a ? token : -1;
    if (tid == 0) g.accepted[b] = a;
  }
}

template <typename T, int THREADS>
int launch_one(const Args& g, int64_t batch, int size, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * size));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(size);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, verify_kernel<T, THREADS>, g);
  return launch_status();
}

template <typename T>
int launch(const Args& g, int64_t batch, cudaStream_t s) {
  // Blocks of a sequence: a power of 2, none for less than 2048 entries. Up to two sequences an SM:
  // large blocks, of which an SM holds two, 128 at most in clusters, as clusters of 8 do not fill
  // every SM. More sequences: small ones, whose number the SMs share out more evenly. On the
  // device, large and small: 8.6 and 11.1 us for 1 x 131072 f32, 16 and 20 for 128 x 100003 bf16,
  // 25 and 29 for 256 x 100003, 41 and 37 for 320 x 100003, 53 and 33 for 1000 x 20000 f32, 39 and
  // 14 for 2000 x 1000.
  const bool few = batch <= 2 * kSms;
  const int64_t slots = few ? 128 : kSms * kManyPerSm;
  int size = 1;
  while (size < kMaxCluster && batch * size * 2 <= slots && g.vocab / (size * 2) >= 2048) size *= 2;
  return few ? launch_one<T, kFew>(g, batch, size, s) : launch_one<T, kMany>(g, batch, size, s);
}

}  // namespace verify
}  // namespace jk

extern "C" int jk_verify_draft(const jk_draft_t* q, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::verify;
  if (q == nullptr) return JK_ERR_BAD_ARG;
  const int64_t batch = q->batch, drafted = q->drafted, vocab = q->vocab;
  if (batch < 0 || drafted < 0 || vocab < 1 || batch > (1 << 24) || drafted > (1 << 30) || vocab > (1 << 30)) return JK_ERR_BAD_SHAPE;
  const int dtype = q->dtype == JK_F32 || q->dtype == JK_BF16 || q->dtype == JK_F16 ? static_cast<int>(q->dtype) : -1;
  if (dtype < 0) return JK_ERR_BAD_DTYPE;
  if (batch > 0 && (q->target == nullptr || q->uniform == nullptr || q->out_tokens == nullptr || q->accepted == nullptr)) return JK_ERR_BAD_ARG;
  if (batch > 0 && drafted > 0 && q->tokens == nullptr) return JK_ERR_BAD_ARG;
  if (int st = check_device()) return st;
  if (batch == 0) return JK_OK;
  const Args g{q->target, q->draft, q->target_stride[0], q->target_stride[1], q->draft_stride[0], q->draft_stride[1], q->tokens, q->uniform,
               q->counts, static_cast<int32_t>(drafted), static_cast<int32_t>(vocab), q->out_tokens, q->accepted};
  auto s = reinterpret_cast<cudaStream_t>(stream);
  JK_WITH_TYPE(dtype, T, return launch<T>(g, batch, s));
}
