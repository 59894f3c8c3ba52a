// Pages of a cache: room for new nodes and their rows written, sequences that branch, end and are
// cut back, pages copied and moved together (jk_cache_*).
//
// The pages' bookkeeping (table, lengths, references) stays on the device, so that a step of a model
// needs no read-back and can be captured into a graph. What is decided one sequence after the other
// (who gets which of the free pages) is a prefix sum over the sequences and one over the pages,
// which one block of 1024 threads takes in rounds; what moves bytes is a launch of its own that
// fills the GPU. Whole numbers throughout: results do not depend on the order in which blocks run
// (references are added to, never read, where blocks share them).
//
// Bound: bookkeeping by the latency of a few dependent reads and a launch or two (room for a node
// in each of 32 sequences, its rows written and given back: 9.8 us on the device, 45 as calls),
// copies by memory (the 70 us of 460 MB moved together are what they take at the measured copy
// rate; 76 MB of new rows 16 us, of which 12 for the memory). A copy has 16-byte stores to aligned
// blocks whatever the alignment of its two sides: where they differ, a block is put together from
// the two aligned blocks of the source that hold its bytes (so rows of 65 bf16 cost two loads a
// block instead of eight).
#include "jk_host.h"
#include "jk_rows.cuh"

namespace jk {
namespace cache {

constexpr int kOne = 1024;          // threads of the bookkeeping block
constexpr int kThreads = 256;       // threads of a copying block
constexpr int kLoads = 8;           // 16-byte blocks of a lane in one piece of a page
constexpr int kPiece = 32 * kLoads; // 16-byte blocks of a piece: a warp's turn
constexpr int kMaxBlocks = 148 * 8;
constexpr int kSmall = 8, kLarge = 512;  // pools of a launch: its parameters are copied, so few take the small table
constexpr int kMaxWrite = 64;
constexpr int64_t kMaxLength = 0x7fffffff - 64;  // nodes of a sequence: what the propagation sees

// ---- copies of any alignment

// Bytes [from, to) of dst from src, both multiples of `unit` (1, 2, 4, 8) apart and aligned to it.
__device__ __forceinline__ void copy_units(char* dst, const char* src, int64_t from, int64_t to, uint32_t unit) {
  if (unit == 8) {
    for (; from < to; from += 8) *reinterpret_cast<uint64_t*>(dst + from) = *reinterpret_cast<const uint64_t*>(src + from);
  } else if (unit == 4) {
    for (; from < to; from += 4) *reinterpret_cast<uint32_t*>(dst + from) = *reinterpret_cast<const uint32_t*>(src + from);
  } else if (unit == 2) {
    for (; from < to; from += 2) *reinterpret_cast<uint16_t*>(dst + from) = *reinterpret_cast<const uint16_t*>(src + from);
  } else {
    for (; from < to; ++from) dst[from] = src[from];
  }
}

__device__ __forceinline__ uint32_t address16(const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u; }

// Aligned 16-byte blocks that [p, p + bytes) has a part of.
__device__ __forceinline__ int64_t blocks16(const void* p, int64_t bytes) { return (address16(p) + bytes + 15) >> 4; }

// Blocks first, first + step, ... (N of them) of dst's; those past its end are left out.
template <int N>
__device__ __forceinline__ void copy_blocks(char* dst, const char* src, int64_t bytes, uint32_t unit, int64_t first, int step) {
  const uint32_t head = address16(dst), a = (address16(src) - head) & 15u;
  const int64_t at = first * 16 - head;
  uint4 v[N];
  if (((head | a | static_cast<uint32_t>(bytes)) & 15u) == 0) {  // 16-byte blocks on both sides: what caches mostly have
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (at + j * step * 16 < bytes) v[j] = *reinterpret_cast<const uint4*>(src + at + j * step * 16);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (at + j * step * 16 < bytes) *reinterpret_cast<uint4*>(dst + at + j * step * 16) = v[j];
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int64_t off = at + int64_t(j) * step * 16;
    if (off >= 0 && off + 16 <= bytes) v[j] = load16(src + off, a);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int64_t off = at + int64_t(j) * step * 16;
    if (off >= 0 && off + 16 <= bytes) {
      *reinterpret_cast<uint4*>(dst + off) = v[j];
    } else if (off < bytes) {
      copy_units(dst, src, off < 0 ? 0 : off, off + 16 < bytes ? off + 16 : bytes, unit);
    }
  }
}

// ---- a block's prefix sums

// Inclusive prefix sum over the block's kOne threads; total: of all of them. scratch: 33 elements.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* scratch, V& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  __syncthreads();  // scratch may still be read from the round before
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  if (warp == 0) {
    V w = scratch[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    scratch[lane] = w;
  }
  __syncthreads();
  total = scratch[31];
  return warp == 0 ? v : v + scratch[warp - 1];
}

// refs[4 * i .. 4 * i + 4) as one load where they lie in a 16-byte block; entries past the end as `pad`.
__device__ __forceinline__ int4 refs4(const int32_t* refs, int64_t at, int64_t pages, int pad, bool aligned) {
  if (aligned && at + 4 <= pages) return *reinterpret_cast<const int4*>(refs + at);
  int4 r = make_int4(pad, pad, pad, pad);
  if (at < pages) r.x = refs[at];
  if (at + 1 < pages) r.y = refs[at + 1];
  if (at + 2 < pages) r.z = refs[at + 2];
  if (at + 3 < pages) r.w = refs[at + 3];
  return r;
}

struct Table {
  int32_t* at;
  int64_t stride;
  int64_t batch, columns, pages;
};

__device__ __forceinline__ bool in_cache(int32_t page, int64_t pages) { return static_cast<uint32_t>(page) < static_cast<uint64_t>(pages); }

// ---- copies of whole pages

template <int N>
struct Pools {
  char* data[N];
  int64_t stride[N], bytes[N];
  uint32_t first[N + 1];  // the piece at which a pool's page begins, of the pieces of a page in all pools
  int count;
};

// dst[step * i] <- src[step * i] for pairs i < n; n_dev: n is read there.
struct Pairs {
  const int32_t *src, *dst;
  int step;
  int64_t n;
  const int32_t* n_dev;
};

template <int N>
__device__ __forceinline__ void copy_pairs(const Pools<N>& pools, const Pairs& q, int64_t pages) {
  const int64_t n = q.n_dev == nullptr ? q.n : *q.n_dev;
  const uint32_t per = pools.first[pools.count];
  const int64_t items = n * per, step = int64_t(gridDim.x) * (kThreads / 32);
  for (int64_t item = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); item < items; item += step) {
    const int64_t i = item / per;
    const uint32_t piece = static_cast<uint32_t>(item - i * per);
    const int32_t s = q.src[i * q.step], d = q.dst[i * q.step];
    if (!in_cache(s, pages) || !in_cache(d, pages) || s == d) continue;
    int low = 0, high = pools.count - 1;
    while (low < high) {
      const int mid = (low + high + 1) >> 1;
      if (pools.first[mid] <= piece) low = mid;
      else high = mid - 1;
    }
    char* to = pools.data[low] + d * pools.stride[low];
    const char* from = pools.data[low] + s * pools.stride[low];
    const int64_t bytes = pools.bytes[low];
    const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to) | reinterpret_cast<uintptr_t>(from) | bytes) | 8u;
    copy_blocks<kLoads>(to, from, bytes, odd & -odd, int64_t(piece - pools.first[low]) * kPiece + (threadIdx.x & 31), 32);
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads) copy_kernel(const __grid_constant__ Pools<N> pools, const Pairs q, int64_t pages) {
  grid_dependency_wait();
  copy_pairs(pools, q, pages);
}

// ---- room for new nodes

struct Reserve {
  int64_t* from;    // [batch] number of the sequence's first page among those that all ask for
  int32_t* need;    // [batch] pages that it asks for
  int32_t* begin;   // [batch] column that takes the first of them
  int32_t* pairs;   // [batch][2] page to copy and its copy, -1: none
  int32_t* free;    // [pages] the free pages, lowest first
};

__global__ void __launch_bounds__(kOne) reserve_kernel(Table t, int32_t* lengths, int32_t* refs, const int32_t* counts, int64_t page_size,
                                                       int32_t* added, Reserve w) {
  __shared__ int64_t scratch[33];
  __shared__ int32_t scratch32[33];
  const int tid = threadIdx.x;
  // who asks for how many
  int64_t asked = 0;
  for (int64_t base = 0; base < t.batch; base += kOne) {
    const int64_t b = base + tid;
    int32_t need = 0, shared = -1;
    int64_t have = 0;
    bool fits = false;
    if (b < t.batch) {
      const int64_t n = lengths[b], c = counts[b];
      fits = n >= 0 && c >= 0 && n + c <= t.columns * page_size && n + c <= kMaxLength;
      if (fits && c > 0) {
        have = (n + page_size - 1) / page_size;
        need = static_cast<int32_t>((n + c + page_size - 1) / page_size - have);
        if (n % page_size != 0) {
          const int32_t last = t.at[b * t.stride + have - 1];
          if (in_cache(last, t.pages) && refs[last] > 1) shared = last, ++need, --have;
        }
      }
    }
    int64_t total;
    const int64_t upto = block_scan<int64_t>(need, scratch, total);
    if (b < t.batch) {
      w.from[b] = asked + upto - need;
      w.need[b] = fits ? need : -1;
      w.begin[b] = static_cast<int32_t>(have);
      w.pairs[2 * b] = shared;
    }
    asked += total;
  }
  // the free pages, as many as are asked for
  const int64_t wanted = asked < t.pages ? asked : t.pages;
  const bool aligned = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
  int64_t found = 0;
  for (int64_t base = 0; base < t.pages && found < wanted; base += 4 * kOne) {
    const int64_t at = base + 4 * tid;
    const int4 r = refs4(refs, at, t.pages, 1, aligned);
    const int32_t mine = (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
    int32_t total;
    int64_t k = found + block_scan<int32_t>(mine, scratch32, total) - mine;
    if (r.x == 0 && k < wanted) w.free[k++] = static_cast<int32_t>(at);
    if (r.y == 0 && k < wanted) w.free[k++] = static_cast<int32_t>(at + 1);
    if (r.z == 0 && k < wanted) w.free[k++] = static_cast<int32_t>(at + 2);
    if (r.w == 0 && k < wanted) w.free[k++] = static_cast<int32_t>(at + 3);
    found += total;
  }
  __syncthreads();
  // a warp a sequence
  const int lane = tid & 31;
  for (int64_t b = tid >> 5; b < t.batch; b += kOne / 32) {
    const int32_t need = w.need[b], begin = w.begin[b];
    const int64_t from = w.from[b];
    const bool given = need >= 0 && (need == 0 || from + need <= found);
    const int32_t shared = w.pairs[2 * b];
    __syncwarp();
    if (lane == 0) {
      const int32_t c = counts[b];
      added[b] = given ? c : 0;
      if (given) lengths[b] += c;
      const bool copies = given && shared >= 0;
      if (!copies) w.pairs[2 * b] = -1;
      else atomicSub(refs + shared, 1);
      w.pairs[2 * b + 1] = copies ? w.free[from] : -1;
    }
    if (given) {
      for (int32_t k = lane; k < need; k += 32) {
        const int32_t page = w.free[from + k];
        t.at[b * t.stride + begin + k] = page;
        refs[page] = 1;
      }
    }
  }
}

// ---- rows of new nodes

struct Write {
  char* pages[kMaxWrite];
  const char* rows[kMaxWrite];
  int64_t page_stride[kMaxWrite][3], row_stride[kMaxWrite][3];  // bytes
  int64_t bytes[kMaxWrite];                                     // of a row
  uint8_t lanes_log2[kMaxWrite], unit[kMaxWrite];
};

__global__ void __launch_bounds__(kThreads) write_kernel(const __grid_constant__ Write w, const int32_t* table, int64_t table_stride,
                                                         const int32_t* lengths, const int32_t* counts, uint32_t rows, uint32_t new_nodes,
                                                         uint32_t heads, int64_t pages, uint32_t page_size, int64_t columns) {
  const int i = blockIdx.y;
  const int log2 = w.lanes_log2[i], lanes = 1 << log2;
  const uint64_t row = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) >> log2;
  if (row >= rows) return;
  const uint32_t h = static_cast<uint32_t>(row) % heads, bt = static_cast<uint32_t>(row) / heads;
  const uint32_t t = bt % new_nodes, b = bt / new_nodes;
  int32_t n = counts == nullptr ? static_cast<int32_t>(new_nodes) : counts[b];
  n = n > static_cast<int32_t>(new_nodes) ? static_cast<int32_t>(new_nodes) : n;
  const int64_t place = int64_t(lengths[b]) - n + t;
  if (static_cast<int32_t>(t) >= n || place < 0) return;
  const uint32_t c = static_cast<uint32_t>(place) / page_size, off = static_cast<uint32_t>(place) - c * page_size;
  if (c >= columns) return;
  const int32_t page = table[b * table_stride + c];
  if (!in_cache(page, pages)) return;
  char* to = w.pages[i] + page * w.page_stride[i][0] + h * w.page_stride[i][1] + off * w.page_stride[i][2];
  const char* from = w.rows[i] + b * w.row_stride[i][0] + t * w.row_stride[i][1] + h * w.row_stride[i][2];
  const int64_t bytes = w.bytes[i], blocks = blocks16(to, bytes);
  for (int64_t k = threadIdx.x & (lanes - 1); k < blocks; k += 4 * lanes) copy_blocks<4>(to, from, bytes, w.unit[i], k, lanes);
}

// ---- sequences that branch, and that are cut back

// Row of the child: a copy of the parent's, whose pages get one more reference; a parent that was
// empty (it may be a child of this call, whose row another thread is writing) gives an empty row.
__device__ __forceinline__ void fork_row(const Table& t, int32_t* refs, int32_t parent, int32_t child, int32_t length, int64_t first, int64_t step) {
  for (int64_t c = first; c < t.columns; c += step) {
    const int32_t page = length > 0 ? t.at[parent * t.stride + c] : -1;
    t.at[child * t.stride + c] = page;
    if (in_cache(page, t.pages)) atomicAdd(refs + page, 1);
  }
}

// taken: [batch], of which only the children's entries are used; copied: [forks] the parent's
// length, -1: not done.
__global__ void __launch_bounds__(kOne) fork_kernel(Table t, int32_t* lengths, int32_t* refs, const int32_t* parents, const int32_t* children,
                                                    int64_t forks, uint8_t* done, int32_t* taken, int32_t* copied, bool rows_too) {
  auto inside = [&](int64_t i) {
    return in_cache(children[i], t.batch) && in_cache(parents[i], t.batch);
  };
  for (int64_t i = threadIdx.x; i < forks; i += kOne)
    if (in_cache(children[i], t.batch)) taken[children[i]] = 0x7fffffff;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < forks; i += kOne)
    if (in_cache(children[i], t.batch)) atomicMin(taken + children[i], static_cast<int32_t>(i));
  __syncthreads();
  for (int64_t i = threadIdx.x; i < forks; i += kOne) {
    const bool ok = inside(i) && taken[children[i]] == i && lengths[children[i]] == 0;
    const int32_t n = ok ? lengths[parents[i]] : -1;
    copied[i] = n < 0 ? -1 : n;
    done[i] = n >= 0;
  }
  __syncthreads();  // lengths are read above and written below
  for (int64_t i = threadIdx.x; i < forks; i += kOne)
    if (copied[i] >= 0) lengths[children[i]] = copied[i];
  if (!rows_too) return;
  for (int64_t i = threadIdx.x >> 5; i < forks; i += kOne / 32)
    if (copied[i] >= 0) fork_row(t, refs, parents[i], children[i], copied[i], threadIdx.x & 31, 32);
}

__global__ void __launch_bounds__(kThreads) fork_rows_kernel(Table t, int32_t* refs, const int32_t* parents, const int32_t* children,
                                                             int64_t forks, const int32_t* copied) {
  grid_dependency_wait();
  for (int64_t i = blockIdx.x; i < forks; i += gridDim.x)
    if (copied[i] >= 0) fork_row(t, refs, parents[i], children[i], copied[i], threadIdx.x, kThreads);
}

__global__ void __launch_bounds__(kThreads) release_kernel(Table t, int32_t* lengths, int32_t* refs, const int32_t* new_lengths,
                                                           int64_t page_size) {
  for (int64_t b = blockIdx.x; b < t.batch; b += gridDim.x) {
    const int32_t n = lengths[b], asked = new_lengths[b];
    const int32_t keep = asked < 0 ? 0 : asked < n ? asked : n;
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) lengths[b] = keep;
    const int64_t first = keep > 0 ? (keep + page_size - 1) / page_size : 0;
    for (int64_t c = first + threadIdx.x; c < t.columns; c += kThreads) {
      const int32_t page = t.at[b * t.stride + c];
      if (page < 0) continue;
      if (in_cache(page, t.pages)) atomicSub(refs + page, 1);
      t.at[b * t.stride + c] = -1;
    }
  }
}

// ---- pages moved together

// sum over the workspace: moves[0] pages, from[i] -> to[i], map[page]: the i of a page that moved
// (of the others, any number).
struct Compact {
  int32_t *moves, *from, *to, *map;
};

__global__ void __launch_bounds__(kOne) compact_kernel(int32_t* refs, int64_t pages, int32_t* live_out, Compact w) {
  __shared__ int32_t scratch[33];
  const bool aligned = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
  const int tid = threadIdx.x;
  int32_t mine = 0;
  for (int64_t at = 4 * tid; at < pages; at += 4 * kOne) {
    const int4 r = refs4(refs, at, pages, 0, aligned);
    mine += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0);
  }
  int32_t live;
  block_scan<int32_t>(mine, scratch, live);
  int32_t holes = 0, moves = 0;
  for (int64_t base = 0; base < pages; base += 4 * kOne) {
    const int64_t at = base + 4 * tid;
    const int4 r = refs4(refs, at, pages, 0, aligned);
    const int32_t v[4] = {r.x, r.y, r.z, r.w};
    bool hole[4], move[4];
    int32_t packed = 0;  // at most 4096 of each in a round
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hole[j] = at + j < live && v[j] <= 0;
      move[j] = at + j >= live && v[j] > 0;
      packed += (hole[j] ? 1 : 0) + (move[j] ? 1 << 16 : 0);
    }
    int32_t total;
    const int32_t upto = block_scan<int32_t>(packed, scratch, total) - packed;
    int32_t h = holes + (upto & 0xffff), m = moves + (upto >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (hole[j]) w.to[h++] = static_cast<int32_t>(at + j);
      if (move[j]) w.from[m++] = static_cast<int32_t>(at + j);
    }
    holes += total & 0xffff;
    moves += total >> 16;
  }
  __syncthreads();
  for (int32_t i = tid; i < moves; i += kOne) {
    const int32_t from = w.from[i], to = w.to[i];
    w.map[from] = i;
    refs[to] = refs[from];
    refs[from] = 0;
  }
  if (tid == 0) {
    *w.moves = moves;
    *live_out = live;
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ Pools<N> pools, Table t, const int32_t* live_at, Compact w) {
  grid_dependency_wait();
  const int32_t live = *live_at, moves = *w.moves;
  const int64_t entries = t.batch * t.columns;
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < entries; i += int64_t(gridDim.x) * kThreads) {
    int32_t* at = t.at + (i / t.columns) * t.stride + i % t.columns;
    const int32_t page = *at;
    // an entry past the pages in use names one that moved, if the references are right; one that
    // has none stays as it is
    if (page >= live && in_cache(page, t.pages)) {
      const int32_t k = w.map[page];
      if (static_cast<uint32_t>(k) < static_cast<uint32_t>(moves) && w.from[k] == page) *at = w.to[k];
    }
  }
  copy_pairs(pools, Pairs{w.from, w.to, 1, 0, w.moves}, t.pages);
}

// ---- host

template <int N>
int fill(Pools<N>& p, const jk_pools_t& q) {
  uint64_t first = 0;
  for (int64_t i = 0; i < q.count; ++i) {
    p.data[i] = static_cast<char*>(q.data[i]);
    p.stride[i] = q.stride_bytes[i];
    p.bytes[i] = q.page_bytes[i];
    p.first[i] = static_cast<uint32_t>(first);
    // a page that begins inside a 16-byte block has a part of one more
    const int64_t head = ((reinterpret_cast<uintptr_t>(q.data[i]) | q.stride_bytes[i]) & 15) == 0 ? 0 : 15;
    first += ((q.page_bytes[i] + head + 15) / 16 + kPiece - 1) / kPiece;
    if (first > 0x7fffffff) return JK_ERR_BAD_SHAPE;
  }
  p.first[q.count] = static_cast<uint32_t>(first);
  p.count = static_cast<int>(q.count);
  return JK_OK;
}

inline int check_pools(const jk_pools_t* q, int64_t pages) {
  if (q == nullptr || q->count < 0 || q->count > kLarge) return q == nullptr ? JK_ERR_BAD_ARG : JK_ERR_BAD_SHAPE;
  if (q->count > 0 && (q->data == nullptr || q->page_bytes == nullptr || q->stride_bytes == nullptr)) return JK_ERR_BAD_ARG;
  for (int64_t i = 0; i < q->count; ++i) {
    if (q->page_bytes[i] < 0 || q->stride_bytes[i] < q->page_bytes[i]) return JK_ERR_BAD_SHAPE;
    if (pages > 0 && q->page_bytes[i] > 0 && q->data[i] == nullptr) return JK_ERR_BAD_ARG;
  }
  return JK_OK;
}

inline int check_cache(const jk_cache_t* c) {
  if (c == nullptr) return JK_ERR_BAD_ARG;
  constexpr int64_t most = 0x7fffffff;
  if (c->batch < 0 || c->columns < 0 || c->pages < 0 || c->batch > most || c->columns > most || c->pages > most || c->table_stride < 0 ||
      c->page_size < 1 || c->page_size > most)
    return JK_ERR_BAD_SHAPE;
  if (c->batch > 1 && c->table_stride < c->columns) return JK_ERR_BAD_SHAPE;  // rows would overlap
  if (c->batch > 0 && c->columns > 0 && c->table == nullptr) return JK_ERR_BAD_ARG;
  return JK_OK;
}

inline Table table_of(const jk_cache_t* c) { return Table{c->table, c->table_stride, c->batch, c->columns, c->pages}; }

inline unsigned copy_grid(int64_t pairs, uint32_t per) {
  const int64_t warps = pairs > (int64_t(1) << 30) / (per + 1) ? int64_t(1) << 30 : pairs * per;
  const int64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
  return static_cast<unsigned>(blocks < 1 ? 1 : blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

template <int N>
int launch_copy(const jk_pools_t& q, const Pairs& pairs, int64_t at_most, int64_t pages, cudaStream_t s) {
  Pools<N> p;
  if (const int st = fill(p, q)) return st;
  launch_dependent(copy_kernel<N>, copy_grid(at_most, p.first[p.count]), kThreads, 0, s, p, pairs, pages);
  return launch_status();
}

template <int N>
int launch_move(const jk_pools_t& q, const Table& t, const int32_t* live, const Compact& w, cudaStream_t s) {
  Pools<N> p;
  if (const int st = fill(p, q)) return st;
  // at most half of the pages move
  const unsigned copies = copy_grid(t.pages / 2, p.first[p.count]);
  const int64_t entries = (t.batch * t.columns + kThreads - 1) / kThreads;
  const unsigned grid = entries > copies ? static_cast<unsigned>(entries < kMaxBlocks ? entries : kMaxBlocks) : copies;
  launch_dependent(move_kernel<N>, grid, kThreads, 0, s, p, t, live, w);
  return launch_status();
}

inline int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace cache
}  // namespace jk

extern "C" {

int64_t jk_cache_reserve_workspace(int64_t batch, int64_t pages) {
  if (batch < 0 || pages < 0) return 0;
  return jk::cache::round16(batch * 8) + 2 * jk::cache::round16(batch * 4) + jk::cache::round16(batch * 8) + jk::cache::round16(pages * 4);
}

int jk_cache_reserve(const jk_pools_t* pools, const jk_cache_t* cache, const int32_t* counts, int32_t* added, void* workspace,
                     jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cache;
  if (int st = check_cache(cache)) return st;
  const int64_t batch = cache->batch, pages = cache->pages;
  if (int st = check_pools(pools, pages)) return st;
  if (batch > 0 && (cache->lengths == nullptr || counts == nullptr || added == nullptr || workspace == nullptr)) return JK_ERR_BAD_ARG;
  if (pages > 0 && cache->refs == nullptr) return JK_ERR_BAD_ARG;
  if (!aligned16(workspace)) return JK_ERR_ALIGNMENT;
  if (int st = check_device()) return st;
  if (batch == 0) return JK_OK;
  char* p = static_cast<char*>(workspace);
  Reserve w;
  w.from = reinterpret_cast<int64_t*>(p), p += round16(batch * 8);
  w.need = reinterpret_cast<int32_t*>(p), p += round16(batch * 4);
  w.begin = reinterpret_cast<int32_t*>(p), p += round16(batch * 4);
  w.pairs = reinterpret_cast<int32_t*>(p), p += round16(batch * 8);
  w.free = reinterpret_cast<int32_t*>(p);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  reserve_kernel<<<1, kOne, 0, s>>>(table_of(cache), cache->lengths, cache->refs, counts, cache->page_size, added, w);
  if (int st = launch_status()) return st;
  if (pools->count == 0) return JK_OK;
  const Pairs pairs{w.pairs, w.pairs + 1, 2, batch, nullptr};
  return pools->count <= kSmall ? launch_copy<kSmall>(*pools, pairs, batch, pages, s) : launch_copy<kLarge>(*pools, pairs, batch, pages, s);
}

int jk_cache_write(const jk_rows_t* q, const jk_cache_t* cache, const int32_t* counts, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cache;
  if (q == nullptr) return JK_ERR_BAD_ARG;
  const int64_t count = q->count, new_nodes = q->new_nodes, heads = q->heads;
  if (count < 0 || count > kMaxWrite) return JK_ERR_BAD_SHAPE;
  if (int st = check_cache(cache)) return st;
  if (new_nodes < 0 || heads < 0 || new_nodes > 0x7fffffff || heads > 0x7fffffff) return JK_ERR_BAD_SHAPE;
  if (count > 0 && (q->pages_data == nullptr || q->pages_strides == nullptr || q->rows_data == nullptr || q->rows_strides == nullptr ||
                    q->widths == nullptr || q->element_bytes == nullptr))
    return JK_ERR_BAD_ARG;
  const int64_t nodes = cache->batch * new_nodes;  // below 2^62
  if (nodes > 0 && heads > 0x7fffffff / nodes) return JK_ERR_BAD_SHAPE;
  const int64_t rows = nodes * heads, pages = cache->pages;
  Write w;
  int most = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t size = q->element_bytes[i];
    if (size != 1 && size != 2 && size != 4 && size != 8) return JK_ERR_BAD_DTYPE;
    if (q->widths[i] < 0 || q->widths[i] > 0x7fffffff) return JK_ERR_BAD_SHAPE;
    if (rows > 0 && q->widths[i] > 0 && (q->rows_data[i] == nullptr || (pages > 0 && q->pages_data[i] == nullptr))) return JK_ERR_BAD_ARG;
    w.pages[i] = static_cast<char*>(q->pages_data[i]);
    w.rows[i] = static_cast<const char*>(q->rows_data[i]);
    w.bytes[i] = q->widths[i] * size;
    for (int j = 0; j < 3; ++j) {
      w.page_stride[i][j] = q->pages_strides[3 * i + j] * size;
      w.row_stride[i][j] = q->rows_strides[3 * i + j] * size;
    }
    w.unit[i] = static_cast<uint8_t>(size);
    // lanes of a row: as many as it has blocks (one more where it begins inside a block), a power
    // of 2, but four blocks a lane in rows of 512 bytes and more, so that each table entry that is
    // waited for is followed by that many loads (32 x 1024 nodes of 64 + 512 + 1 bf16, with room
    // and release: 24.4 us with two blocks a lane in all rows, 21.7 with four)
    int64_t blocks = (w.bytes[i] + 15) / 16 + (w.bytes[i] % 16 != 0 && w.bytes[i] > 16 ? 1 : 0);
    if (blocks >= 32) blocks = (blocks + 3) / 4;
    int log2 = 0;
    while (log2 < 5 && (int64_t(1) << log2) < blocks) ++log2;
    w.lanes_log2[i] = static_cast<uint8_t>(log2);
    if (log2 > most) most = log2;
  }
  if (rows > 0 && cache->lengths == nullptr) return JK_ERR_BAD_ARG;
  if (int st = check_device()) return st;
  if (rows == 0 || count == 0 || pages == 0 || cache->columns == 0) return JK_OK;
  const int64_t grid = ((rows << most) + kThreads - 1) / kThreads;
  if (grid > 0x7fffffff) return JK_ERR_BAD_SHAPE;
  write_kernel<<<dim3(static_cast<unsigned>(grid), static_cast<unsigned>(count)), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      w, cache->table, cache->table_stride, cache->lengths, counts, static_cast<uint32_t>(rows), static_cast<uint32_t>(new_nodes),
      static_cast<uint32_t>(heads), pages, static_cast<uint32_t>(cache->page_size), cache->columns);
  return launch_status();
}

int64_t jk_cache_fork_workspace(int64_t batch, int64_t forks) {
  if (batch < 0 || forks < 0) return 0;
  return jk::cache::round16(batch * 4) + jk::cache::round16(forks * 4);
}

int jk_cache_fork(const jk_cache_t* cache, const int32_t* parents, const int32_t* children, int64_t forks, uint8_t* done, void* workspace,
                  jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cache;
  if (int st = check_cache(cache)) return st;
  const int64_t batch = cache->batch, columns = cache->columns;
  if (forks < 0 || forks > 0x7ffffffe) return JK_ERR_BAD_SHAPE;
  if (forks > 0 && (parents == nullptr || children == nullptr || done == nullptr || workspace == nullptr)) return JK_ERR_BAD_ARG;
  if ((batch > 0 && cache->lengths == nullptr) || (cache->pages > 0 && cache->refs == nullptr)) return JK_ERR_BAD_ARG;
  if (!aligned16(workspace)) return JK_ERR_ALIGNMENT;
  if (int st = check_device()) return st;
  if (forks == 0) return JK_OK;
  const Table t = table_of(cache);
  int32_t *lengths = cache->lengths, *refs = cache->refs;
  auto* taken = static_cast<int32_t*>(workspace);
  auto* copied = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + round16(batch * 4));
  auto s = reinterpret_cast<cudaStream_t>(stream);
  // few table entries: the block that decides copies them as well, which saves a launch (forks and
  // entries each, together with the release that undoes them, a call and on the device: 63 x 128
  // 19.0 and 6.2 us so, 20.9 and 5.7 with a launch for the rows; 63 x 512 18.7 and 12.0, 21.0 and
  // 6.3)
  const bool rows_too = columns == 0 || forks <= 8192 / columns;
  fork_kernel<<<1, kOne, 0, s>>>(t, lengths, refs, parents, children, forks, done, taken, copied, rows_too);
  if (!rows_too)
    launch_dependent(fork_rows_kernel, static_cast<unsigned>(forks < kMaxBlocks ? forks : kMaxBlocks), kThreads, 0, s, t, refs, parents, children,
                     forks, copied);
  return launch_status();
}

int jk_cache_release(const jk_cache_t* cache, const int32_t* new_lengths, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cache;
  if (int st = check_cache(cache)) return st;
  const int64_t batch = cache->batch;
  if (batch > 0 && (cache->lengths == nullptr || new_lengths == nullptr)) return JK_ERR_BAD_ARG;
  if (cache->pages > 0 && cache->refs == nullptr) return JK_ERR_BAD_ARG;
  if (int st = check_device()) return st;
  if (batch == 0) return JK_OK;
  release_kernel<<<static_cast<unsigned>(batch < kMaxBlocks ? batch : kMaxBlocks), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      table_of(cache), cache->lengths, cache->refs, new_lengths, cache->page_size);
  return launch_status();
}

int64_t jk_cache_compact_workspace(int64_t pages) {
  if (pages < 0) return 0;
  return 16 + 3 * jk::cache::round16(pages * 4);
}

int jk_cache_compact(const jk_pools_t* pools, const jk_cache_t* cache, int32_t* live, void* workspace, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cache;
  if (int st = check_cache(cache)) return st;
  const int64_t pages = cache->pages;
  if (int st = check_pools(pools, pages)) return st;
  if (live == nullptr || workspace == nullptr || (pages > 0 && cache->refs == nullptr)) return JK_ERR_BAD_ARG;
  if (!aligned16(workspace)) return JK_ERR_ALIGNMENT;
  if (int st = check_device()) return st;
  char* p = static_cast<char*>(workspace);
  Compact w;
  w.moves = reinterpret_cast<int32_t*>(p), p += 16;
  w.from = reinterpret_cast<int32_t*>(p), p += round16(pages * 4);
  w.to = reinterpret_cast<int32_t*>(p), p += round16(pages * 4);
  w.map = reinterpret_cast<int32_t*>(p);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  compact_kernel<<<1, kOne, 0, s>>>(cache->refs, pages, live, w);
  if (int st = launch_status()) return st;
  const Table t = table_of(cache);
  return pools->count <= kSmall ? launch_move<kSmall>(*pools, t, live, w, s) : launch_move<kLarge>(*pools, t, live, w, s);
}

int jk_cache_copy(const jk_pools_t* pools, const int32_t* src, const int32_t* dst, int64_t n, int64_t pages, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cache;
  if (int st = check_pools(pools, pages)) return st;
  if (n < 0 || n > 0x7fffffff || pages < 0 || pages > 0x7fffffff) return JK_ERR_BAD_SHAPE;
  if (n > 0 && (src == nullptr || dst == nullptr)) return JK_ERR_BAD_ARG;
  if (int st = check_device()) return st;
  if (n == 0 || pools->count == 0) return JK_OK;
  const Pairs pairs{src, dst, 1, n, nullptr};
  auto s = reinterpret_cast<cudaStream_t>(stream);
  return pools->count <= kSmall ? launch_copy<kSmall>(*pools, pairs, n, pages, s) : launch_copy<kLarge>(*pools, pairs, n, pages, s);
}

}  // extern "C"
