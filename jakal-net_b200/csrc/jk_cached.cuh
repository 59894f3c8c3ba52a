// Propagation of a few new nodes over the nodes of a paged cache (jk_cached_propagation).
//
//   s_j = scale q . k_j + bias over the places j that a node sees,  w = compress(s),
//   value = sum_j w_j v_j,  state = sum_j w_j st_j
//
// A unit is one sequence, one head of the cache, and the rows (new node, head) that read it: they
// share every key and value that is loaded. Bound: memory, so the kernel reads the seen part of the
// cache once and keeps loads on their way all the time:
//   * The units' places are laid one after the other in tiles of 64 and cut into as many equal runs
//     as blocks fit the GPU, whatever the sequences' lengths (which only the device knows; every block
//     adds them up for itself). A unit that several blocks have parts of is joined by a second kernel
//     from what they leave: reference, sum and unnormalised values. Few tiles a unit: a block each, and
//     no second kernel.
//   * A warp has every fourth 16 places of the run to itself: its own ring of shared memory fed by
//     asynchronous copies, its own running maximum and sums, no barrier between warps until the run's
//     end, where the four are joined in shared memory.
// 16-bit types: both products are warp matrix instructions with the places (scores) and the value's
// columns (sums) as their 16 rows, and the unit's rows as their 8 columns, of which one node of one head
// fills one: S^T = K Q^T, O^T = V^T W^T. W^T leaves the first product with places across the wrong
// lanes; a matrix transpose within the warp turns it. Weights go into the second product as two planes,
// high + low, so their rounding (2^-16 and less) is far below that of the result.
// f32: the same walk with fused multiply-adds, which keep f32's rounding.
// Exponentials are base 2 on a reference that is itself rounded, so partial sums with different
// references join without a rounding of their own.
//
// What is not seen has no part in a result, whatever it holds: places past the last node and places
// without a page arrive as zeros, and a tile of which rows see different parts (the newest nodes of a
// draft, the far end of their windows) adds up its values row by row.
#pragma once

#include "jk_host.h"
#include "jk_rows.cuh"

#include <type_traits>

namespace jk {
namespace cached {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kKeys = 16;               // places of a warp's turn
constexpr int kTile = kWarps * kKeys;   // places of a block's turn
constexpr int kSms = 148;
constexpr int kMaxBatch = 1024;         // sequences of a launch
constexpr int kMaxRank = 256, kMaxDim = 512, kMaxNew = 64;
constexpr int kUnitTiles = 8;           // units of at most so many tiles get a block each
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const char *query, *keys, *values, *states;  // states null: none
  int64_t query_stride[3];                     // bytes: sequence, node, head
  int64_t key_stride[3], value_stride[3], state_stride[3];  // bytes: page, head, place
  const int32_t *table, *lengths, *counts;
  int64_t table_stride, pages, columns;
  int32_t batch, new_nodes, heads, kv_heads, group, rank, dim;
  uint32_t page_size;
  int32_t window, compress;
  float scale, bias;
  char *out_value, *out_state;
  // layout
  int32_t blocks, row_blocks, rows;       // blocks of the grid; row blocks of a unit's rows, and rows of one
  int32_t key_chunk, value_chunk;         // bytes of one asynchronous copy (16, 8, 4), 0: element by element
  int32_t key_row, value_row;             // elements of a row in shared memory
  int32_t stages, stage_bytes, ring_bytes;
  int32_t part_row;                       // floats of a row that a block leaves: dim rounded up to 4, reference, sum, state
  int64_t* plan;                          // [batch + 2]: tiles of a block, tiles before each sequence
  float* parts;                           // [blocks][2][rows][part_row]
  bool split;
};

// ---- a sequence's places

struct Span {
  int32_t n;         // new nodes that count
  int32_t first;     // place of the first of them (may be negative)
  int32_t low, end;  // places that any of them sees: [low, end)
};

__device__ __forceinline__ Span span_of(const Args& a, int32_t b) {
  Span s;
  const int32_t length = a.lengths[b];
  int32_t n = a.counts == nullptr ? a.new_nodes : a.counts[b];
  s.n = n < 0 ? 0 : n > a.new_nodes ? a.new_nodes : n;
  s.first = length - s.n;
  const int64_t room = a.columns * a.page_size;
  const int32_t most = room < 0x7fffffff - kTile ? static_cast<int32_t>(room) : 0x7fffffff - kTile;
  s.end = s.n == 0 || length < 0 ? 0 : length < most ? length : most;
  const int64_t low = a.window < 0 ? 0 : int64_t(s.first) - a.window;
  s.low = low < 0 ? 0 : low < s.end ? static_cast<int32_t>(low) : s.end;
  return s;
}

__device__ __forceinline__ int32_t tiles_of(const Span& s) { return (s.end - s.low + kTile - 1) / kTile; }

// ---- small pieces

template <typename T>
struct Two;
template <>
struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type of(float a, float b) { return __floats2bfloat162_rn(a, b); }
  static __device__ __forceinline__ float2 back(type v) { return __bfloat1622float2(v); }
};
template <>
struct Two<__half> {
  using type = __half2;
  static __device__ __forceinline__ type of(float a, float b) { return __floats2half2_rn(a, b); }
  static __device__ __forceinline__ float2 back(type v) { return __half22float2(v); }
};

__device__ __forceinline__ uint32_t shared_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix2(uint32_t& r0, uint32_t& r1, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// `bytes` of src, or zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src, bool there) {
  const int n = there ? BYTES : 0;
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until at most `pending` of this thread's groups are on their way.
__device__ __forceinline__ void copy_wait(int pending) {
  if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// ---- compressors

// A score (the bare product) as the compressor takes it: z, whose maximum is the reference (log2 units).
__device__ __forceinline__ float level(int compress, float dot, float scale, float bias) {
  if (compress == JK_SOFTMAX) return dot * scale;  // scale has log2(e) in it
  return fabsf(fmaf(dot, scale, bias)) * kLog2e;
}
// Its weight before normalisation, on reference `ref` (unused by softsign).
__device__ __forceinline__ float weight(int compress, float dot, float scale, float bias, float ref) {
  if (compress == JK_SOFTMAX) return exp2f(fmaf(dot, scale, -ref));
  const float s = fmaf(dot, scale, bias);
  if (compress == JK_SOFTSIGN) return s / (1.0f + fabsf(s));
  return exp2f(fmaf(fabsf(s), kLog2e, -ref));  // the sign is put on after the sum
}
__device__ __forceinline__ float signed_weight(int compress, float dot, float scale, float bias, float w) {
  if (compress != JK_SIGNED_ABS_SOFTMAX) return w;
  const float s = fmaf(dot, scale, bias);
  return s > 0.0f ? w : s < 0.0f ? -w : s == 0.0f ? 0.0f : s;  // NaN stays
}

// What one warp has of a tile: shared memory of one stage, then the walk's own words.
struct Stage {
  char* keys;
  char* values;
  float* states;   // [kKeys]
  uint32_t* seen;  // bit i: place i of the tile is in the cache
};

struct Layout {
  char* base;
  int32_t key_bytes, value_bytes, stage_bytes;
  __device__ __forceinline__ Stage at(int i) const {
    char* p = base + i * stage_bytes;
    char* words = p + key_bytes + value_bytes;
    return Stage{p, p + key_bytes, reinterpret_cast<float*>(words), reinterpret_cast<uint32_t*>(words + 4 * kKeys)};
  }
};

template <typename T, int BYTES>
__device__ __forceinline__ void load_chunks(char* dst, int32_t dst_row, const char* src, int64_t offset, uint32_t there, int32_t row_bytes, int lane) {
  const uint32_t to = shared_at(dst);
#pragma unroll
  for (int q = 0; q < 4; ++q) {  // 8 lanes a row
    const int row = 4 * q + (lane >> 3);
    const char* from = src + __shfl_sync(0xffffffffu, offset, row);
    const bool ok = (there >> row) & 1;
    for (int c = (lane & 7) * BYTES; c < row_bytes; c += 8 * BYTES) copy_async<BYTES>(to + row * dst_row + c, from + c, ok);
  }
}

template <typename T>
__device__ __forceinline__ void load_rows(char* dst, int32_t dst_row, const char* src, int64_t offset, uint32_t there, int32_t row_bytes, int chunk,
                                          int lane) {
  if (chunk == 16) return load_chunks<T, 16>(dst, dst_row, src, offset, there, row_bytes, lane);
  if (chunk == 8) return load_chunks<T, 8>(dst, dst_row, src, offset, there, row_bytes, lane);
  if (chunk == 4) return load_chunks<T, 4>(dst, dst_row, src, offset, there, row_bytes, lane);
  if constexpr (sizeof(T) == 2) {  // 16-bit rows of an odd width, or that begin anywhere
    const int n = row_bytes / 2;
#pragma unroll 4
    for (int row = 0; row < kKeys; ++row) {
      const char* from = src + __shfl_sync(0xffffffffu, offset, row);
      const bool ok = (there >> row) & 1;
      for (int c = lane; c < n; c += 32)
        reinterpret_cast<uint16_t*>(dst + row * dst_row)[c] = ok ? reinterpret_cast<const uint16_t*>(from)[c] : uint16_t(0);
    }
  }
}

// ---- the kernel

// ROWS: rows of a unit that a block takes (a multiple of 8 for 16-bit types); DIM: columns of the value at most.
template <typename T, int ROWS, int DIM>
__global__ void __launch_bounds__(kThreads) cached_kernel(const __grid_constant__ Args a) {
  constexpr bool kWide = std::is_same_v<T, float>;
  constexpr int NT = kWide ? 1 : ROWS / 8;             // 8-row tiles of the matrix instructions
  constexpr int MT = kWide ? 1 : DIM / 16;             // 16-column tiles of the value
  constexpr int CT = kWide ? DIM / 32 : 1;             // f32: columns of a lane
  constexpr int OWN = kWide ? ROWS : 2 * NT;           // rows whose reference and sum a thread keeps
  extern __shared__ __align__(16) char memory[];
  __shared__ int64_t before[kMaxBatch + 1];
  __shared__ int64_t scan[kWarps];
  __shared__ float ref_s[kWarps][ROWS], sum_s[kWarps][ROWS], state_s[kWarps][ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // tiles before each sequence
  {
    int64_t carry = 0;
    if (tid == 0) before[0] = 0;
    for (int32_t base = 0; base < a.batch; base += kThreads) {
      const int32_t b = base + tid;
      int64_t v = b < a.batch ? int64_t(tiles_of(span_of(a, b))) * a.kv_heads * a.row_blocks : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
      }
      __syncthreads();
      if (lane == 31) scan[warp] = v;
      __syncthreads();
      int64_t add = carry;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) add += scan[w];
        carry += scan[w];
      }
      if (b < a.batch) before[b + 1] = v + add;
    }
    __syncthreads();
  }
  grid_dependency_launch();
  const int64_t total = before[a.batch];
  int64_t chunk, at, until;
  int32_t unit = 0;
  if (a.split) {
    chunk = (total + a.blocks - 1) / a.blocks;
    at = chunk * blockIdx.x < total ? chunk * blockIdx.x : total;
    until = at + chunk < total ? at + chunk : total;
    if (blockIdx.x == 0) {
      if (tid == 0) a.plan[0] = chunk;
      for (int32_t b = tid; b <= a.batch; b += kThreads) a.plan[1 + b] = before[b];
    }
  } else {
    unit = blockIdx.x;
    chunk = 1, at = 0, until = 1;
  }

  // shared memory: queries, the f32 weights of a tile, then the rings
  const int query_row = a.key_row;
  T* query = reinterpret_cast<T*>(memory);
  constexpr int kWeightRow = kWide ? kKeys : kKeys + 1;
  float* weights = reinterpret_cast<float*>(memory + ((ROWS * query_row * sizeof(T) + 15) & ~size_t(15))) + warp * (ROWS * kWeightRow);
  char* rings = memory + ((ROWS * query_row * sizeof(T) + 15) & ~size_t(15)) + ((kWarps * ROWS * kWeightRow * 4 + 15) & ~15);
  const Layout ring{rings + warp * a.stages * a.stage_bytes, kKeys * a.key_row * int(sizeof(T)), kKeys * a.value_row * int(sizeof(T)), a.stage_bytes};
  float* joined = reinterpret_cast<float*>(rings);  // [kWarps][ROWS][DIM + 4], once the rings are drained

  while (at < until) {
    // ---- the unit and the run of its tiles
    int32_t b, inner, tile = 0, tiles, unit_tiles;
    int64_t unit_begin = 0;
    if (a.split) {
      int32_t low = 0, high = a.batch - 1;
      while (low < high) {  // the last sequence that begins at or before `at`, and is not empty
        const int32_t mid = (low + high) >> 1;
        if (before[mid + 1] > at) high = mid;
        else low = mid + 1;
      }
      b = low;
    } else {
      b = unit / (a.kv_heads * a.row_blocks);
    }
    const Span span = span_of(a, b);
    unit_tiles = tiles_of(span);
    if (a.split) {
      const int64_t in = at - before[b];
      inner = static_cast<int32_t>(in / unit_tiles);
      tile = static_cast<int32_t>(in - int64_t(inner) * unit_tiles);
      unit_begin = at - tile;
      const int64_t left = until - at;
      tiles = unit_tiles - tile < left ? unit_tiles - tile : static_cast<int32_t>(left);
    } else {
      inner = unit - b * (a.kv_heads * a.row_blocks);
      tiles = unit_tiles;
    }
    const int32_t kv = inner / a.row_blocks, row0 = (inner - kv * a.row_blocks) * ROWS;
    const int32_t unit_rows = a.group * a.new_nodes;
    const int32_t rows = unit_rows - row0 < ROWS ? unit_rows - row0 : ROWS;
    // what every node that counts sees
    const int32_t t_first = row0 / a.group;
    int32_t t_last = (row0 + rows - 1) / a.group;
    if (t_last > span.n - 1) t_last = span.n - 1;
    const int32_t all_end = span.first + t_first + 1 < span.end ? span.first + t_first + 1 : span.end;
    const int64_t far = int64_t(span.first) + t_last - a.window;
    const int32_t all_low = a.window < 0 || far < span.low ? span.low : far < span.end ? static_cast<int32_t>(far) : span.end;

    // ---- queries
    for (int i = tid; i < ROWS * query_row; i += kThreads) {
      const int r = i / query_row, c = i - r * query_row;
      float v = 0.0f;
      if (r < rows && c < a.rank) {
        const int t = (row0 + r) / a.group, g = (row0 + r) - t * a.group;
        if (t < span.n)
          v = to_f32(reinterpret_cast<const T*>(a.query + b * a.query_stride[0] + t * a.query_stride[1] + (kv * a.group + g) * a.query_stride[2])[c]);
      }
      query[i] = from_f32<T>(v);
    }
    // pads of the rings' rows: 0, and not written again before the rings are used to join
    for (int i = lane; i < a.stages * kKeys; i += 32) {
      const Stage s = ring.at(i / kKeys);
      T* k = reinterpret_cast<T*>(s.keys) + (i % kKeys) * a.key_row;
      T* v = reinterpret_cast<T*>(s.values) + (i % kKeys) * a.value_row;
      for (int c = a.rank; c < a.key_row; ++c) k[c] = from_f32<T>(0.0f);
      for (int c = a.dim; c < a.value_row; ++c) v[c] = from_f32<T>(0.0f);
    }
    __syncthreads();

    // ---- this thread's rows: the places they see, [row_low, row_end)
    int32_t row_low[OWN], row_end[OWN];
    float ref[OWN], sum[OWN], state[OWN];
    bool any[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int r = kWide ? i : (i >> 1) * 8 + 2 * (lane & 3) + (i & 1);
      const int t = (row0 + r) / a.group;
      const bool counts = r < rows && t < span.n;
      const int32_t place = span.first + t;
      row_end[i] = !counts ? 0 : place + 1 < span.end ? place + 1 : span.end;
      row_low[i] = a.window < 0 || place < a.window ? 0 : place - a.window;
      ref[i] = a.compress == JK_SOFTSIGN ? 0.0f : -INFINITY;
      sum[i] = state[i] = 0.0f;
      any[i] = false;
    }
    float out[kWide ? ROWS : MT][kWide ? CT : NT * 4];
#pragma unroll
    for (int i = 0; i < (kWide ? ROWS : MT); ++i)
#pragma unroll
      for (int j = 0; j < (kWide ? CT : NT * 4); ++j) out[i][j] = 0.0f;

    const char* keys = a.keys + kv * a.key_stride[1];
    const char* values = a.values + kv * a.value_stride[1];
    const char* states = a.states == nullptr ? nullptr : a.states + kv * a.state_stride[1];
    const int32_t key0 = span.low + tile * kTile + warp * kKeys;

    // the page of this lane's place (lanes 16.. as lanes 0..) of turn i, -1: none
    auto page_of = [&](int32_t i) -> int32_t {
      const int64_t j = int64_t(key0) + int64_t(i) * kTile + (lane & 15);
      if (i >= tiles || j >= span.end) return -1;
      const int32_t page = a.table[b * a.table_stride + static_cast<uint32_t>(j) / a.page_size];
      return static_cast<uint32_t>(page) < static_cast<uint64_t>(a.pages) ? page : -1;
    };
    float state_next = 0.0f;  // of the turn that was issued last
    auto issue = [&](int32_t i, int32_t page) {
      if (i < tiles) {
        const Stage s = ring.at(i % a.stages);
        const uint32_t j = static_cast<uint32_t>(key0 + i * kTile + (lane & 15));
        const uint32_t off = page < 0 ? 0 : j % a.page_size;
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
        const int64_t p = page < 0 ? 0 : page;
        load_rows<T>(s.keys, a.key_row * int(sizeof(T)), keys, p * a.key_stride[0] + off * a.key_stride[2], there, a.rank * int(sizeof(T)), a.key_chunk, lane);
        load_rows<T>(s.values, a.value_row * int(sizeof(T)), values, p * a.value_stride[0] + off * a.value_stride[2], there, a.dim * int(sizeof(T)),
                     a.value_chunk, lane);
        if (lane == 0) *s.seen = there;
        if (states != nullptr && lane < kKeys)
          state_next = page < 0 ? 0.0f : to_f32(*reinterpret_cast<const T*>(states + p * a.state_stride[0] + off * a.state_stride[2]));
      }
      copy_commit();
    };
    auto put_state = [&](int32_t i) {  // of turn i, read when it was issued
      if (states != nullptr && i >= 0 && i < tiles && lane < kKeys) ring.at(i % a.stages).states[lane] = state_next;
    };

    int32_t page = page_of(0);
    for (int i = 0; i < a.stages - 1; ++i) {
      const int32_t next = page_of(i + 1);
      issue(i, page);
      put_state(i);
      page = next;
    }
    for (int32_t i = 0; i < tiles; ++i) {
      __syncwarp();  // the stage to fill has been read by all lanes
      const int32_t ahead = i + a.stages - 1;
      if (a.stages > 1 && i > 0) put_state(ahead - 1);
      const int32_t next = page_of(ahead + 1);
      issue(ahead, page);
      if (a.stages == 1) put_state(ahead);
      page = next;
      copy_wait(a.stages - 1);
      __syncwarp();
      const Stage s = ring.at(i % a.stages);
      const uint32_t there = *s.seen;
      const int32_t k0 = key0 + i * kTile;
      if (there == 0) continue;
      // rows see different parts of it
      const int32_t tile_end = k0 + kKeys < span.end ? k0 + kKeys : span.end;
      const bool mixed = tile_end > all_end || k0 < all_low;

      if constexpr (!kWide) {
        float c[NT][4], c2[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[n][e] = c2[n][e] = 0.0f;
        // K: matrices (places 0-7 | 8-15) x (columns 0-7 | 8-15)
        const uint32_t k_at = shared_at(reinterpret_cast<T*>(s.keys) + (lane & 15) * a.key_row + (lane >> 4) * 8);
        const uint32_t q_at = shared_at(query + (lane & 7) * query_row + ((lane >> 3) & 1) * 8);
        const int steps = (a.rank + 15) / 16;
        for (int k = 0; k < steps; k += 2) {
          uint32_t ka[4], kb[4];
          ldmatrix4(ka, k_at + k * 32);
          const bool more = k + 1 < steps;
          if (more) ldmatrix4(kb, k_at + (k + 1) * 32);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t b0, b1;
            ldmatrix2(b0, b1, q_at + n * 8 * query_row * 2 + k * 32);
            mma<T>(c[n], ka, b0, b1);
            if (more) {
              ldmatrix2(b0, b1, q_at + n * 8 * query_row * 2 + (k + 1) * 32);
              mma<T>(c2[n], kb, b0, b1);
            }
          }
        }
        // c[n][e]: place (lane / 4) + 8 (e / 2), row 8 n + 2 (lane % 4) + e % 2
        const int place = lane >> 2;
        const float st0 = states == nullptr ? 0.0f : s.states[place], st1 = states == nullptr ? 0.0f : s.states[place + 8];
        uint32_t high[NT][2], low[NT][2];
        bool moved = false;
        float factor[OWN];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i2 = 2 * n + e;
            const float d0 = c[n][e] + c2[n][e], d1 = c[n][e + 2] + c2[n][e + 2];
            const int32_t j0 = k0 + place, j1 = j0 + 8;
            const bool v0 = ((there >> place) & 1) && j0 < row_end[i2] && j0 >= row_low[i2];
            const bool v1 = ((there >> (place + 8)) & 1) && j1 < row_end[i2] && j1 >= row_low[i2];
            any[i2] |= v0 || v1;
            factor[i2] = 1.0f;
            float r = 0.0f;
            if (a.compress != JK_SOFTSIGN) {
              float top = v0 ? level(a.compress, d0, a.scale, a.bias) : -INFINITY;
              if (v1) top = fmaxf(top, level(a.compress, d1, a.scale, a.bias));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              top = fmaxf(top, ref[i2]);
              r = top == -INFINITY ? 0.0f : top;
              if (top != ref[i2]) {
                factor[i2] = exp2f(ref[i2] - r);
                ref[i2] = top;
                moved = true;
              }
            }
            const float w0 = v0 ? weight(a.compress, d0, a.scale, a.bias, r) : 0.0f;
            const float w1 = v1 ? weight(a.compress, d1, a.scale, a.bias, r) : 0.0f;
            sum[i2] = fmaf(sum[i2], factor[i2], w0 + w1);
            w[e] = v0 ? signed_weight(a.compress, d0, a.scale, a.bias, w0) : 0.0f;
            w[e + 2] = v1 ? signed_weight(a.compress, d1, a.scale, a.bias, w1) : 0.0f;
            if (states != nullptr) {
              float x = state[i2] * factor[i2];
              if (v0) x = fmaf(w[e], st0, x);
              if (v1) x = fmaf(w[e + 2], st1, x);
              state[i2] = x;
            }
          }
          if (mixed) {
#pragma unroll
            for (int e = 0; e < 4; ++e) weights[(8 * n + 2 * (lane & 3) + (e & 1)) * kWeightRow + place + 8 * (e >> 1)] = w[e];
          } else {
            using P = Two<T>;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const typename P::type hi = P::of(w[2 * h], w[2 * h + 1]);
              const float2 f = P::back(hi);
              const typename P::type lo = P::of(w[2 * h] - f.x, w[2 * h + 1] - f.y);
              high[n][h] = transpose8(*reinterpret_cast<const uint32_t*>(&hi));
              low[n][h] = transpose8(*reinterpret_cast<const uint32_t*>(&lo));
            }
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) out[m][4 * n + e] *= factor[2 * n + (e & 1)];
        }
        if (!mixed) {
          // V^T: matrices (columns 0-7 | 8-15) x (places 0-7 | 8-15), read transposed
          const uint32_t v_at = shared_at(reinterpret_cast<T*>(s.values) + ((lane & 7) + ((lane >> 4) & 1) * 8) * a.value_row + ((lane >> 3) & 1) * 8);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (m * 16 < a.dim) {
              uint32_t va[4];
              ldmatrix4_trans(va, v_at + m * 32);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float(&o)[4] = *reinterpret_cast<float(*)[4]>(&out[m][4 * n]);
                mma<T>(o, va, high[n][0], high[n][1]);
                mma<T>(o, va, low[n][0], low[n][1]);
              }
            }
          }
        } else {
          __syncwarp();
          const T* v = reinterpret_cast<const T*>(s.values);
          for (int k = 0; k < kKeys; ++k) {
            if (!((there >> k) & 1)) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (k0 + k < row_low[2 * n + e] || k0 + k >= row_end[2 * n + e]) continue;
                const float w = weights[(8 * n + 2 * (lane & 3) + e) * kWeightRow + k];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                  if (m * 16 < a.dim) {
                    out[m][4 * n + e] = fmaf(w, to_f32(v[k * a.value_row + m * 16 + place]), out[m][4 * n + e]);
                    out[m][4 * n + e + 2] = fmaf(w, to_f32(v[k * a.value_row + m * 16 + place + 8]), out[m][4 * n + e + 2]);
                  }
                }
              }
          }
        }
      } else {
        // f32: a lane has half a place's columns, lanes 16.. the second half
        const int place = lane & 15;
        const int half = a.key_row / 2 / 4 * 4;  // key_row is a multiple of 4; the two halves need not be equal
        const int begin = lane < 16 ? 0 : half, end = lane < 16 ? half : a.key_row - 4;
        const float* k = reinterpret_cast<const float*>(s.keys) + place * a.key_row;
        const float* q = reinterpret_cast<const float*>(query);
        float dot[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) dot[r] = 0.0f;
        for (int x = begin; x < end; x += 4) {
          const float4 kv4 = *reinterpret_cast<const float4*>(k + x);
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            if (r < rows) {
              const float4 q4 = *reinterpret_cast<const float4*>(q + r * query_row + x);
              dot[r] = fmaf(kv4.x, q4.x, fmaf(kv4.y, q4.y, fmaf(kv4.z, q4.z, fmaf(kv4.w, q4.w, dot[r]))));
            }
          }
        }
        const int32_t j = k0 + place;
        const float st = states == nullptr ? 0.0f : s.states[place];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          if (r < rows) {
            const float d = dot[r] + __shfl_xor_sync(0xffffffffu, dot[r], 16);
            const bool v = ((there >> place) & 1) && j < row_end[r] && j >= row_low[r];
            any[r] |= v;
            float factor = 1.0f, base = 0.0f;
            if (a.compress != JK_SOFTSIGN) {
              float top = v ? level(a.compress, d, a.scale, a.bias) : -INFINITY;
#pragma unroll
              for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              top = fmaxf(top, ref[r]);
              base = top == -INFINITY ? 0.0f : top;
              if (top != ref[r]) {
                factor = exp2f(ref[r] - base);
                ref[r] = top;
#pragma unroll
                for (int x = 0; x < CT; ++x) out[r][x] *= factor;
              }
            }
            float w = v ? weight(a.compress, d, a.scale, a.bias, base) : 0.0f;
            sum[r] = fmaf(sum[r], factor, lane < 16 ? w : 0.0f);
            w = v ? signed_weight(a.compress, d, a.scale, a.bias, w) : 0.0f;
            if (states != nullptr) {
              state[r] *= factor;
              if (v && lane < 16) state[r] = fmaf(w, st, state[r]);
            }
            if (lane < 16) weights[r * kWeightRow + place] = w;
          }
        }
        __syncwarp();
        const float* v = reinterpret_cast<const float*>(s.values);
#pragma unroll 1
        for (int k4 = 0; k4 < kKeys; k4 += 4) {
          float x[4][CT];
#pragma unroll
          for (int k1 = 0; k1 < 4; ++k1)
#pragma unroll
            for (int y = 0; y < CT; ++y) x[k1][y] = lane + 32 * y < a.dim ? v[(k4 + k1) * a.value_row + lane + 32 * y] : 0.0f;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            if (r < rows) {
              const float4 w4 = *reinterpret_cast<const float4*>(weights + r * kWeightRow + k4);
              const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int k1 = 0; k1 < 4; ++k1) {
                const int32_t jj = k0 + k4 + k1;
                if (!mixed || (jj >= row_low[r] && jj < row_end[r])) {
#pragma unroll
                  for (int y = 0; y < CT; ++y) out[r][y] = fmaf(w[k1], x[k1][y], out[r][y]);
                }
              }
            }
          }
        }
      }
    }
    copy_wait(0);

    // ---- the warps' sums, then the block's
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      bool seen = any[i];
#pragma unroll
      for (int o = kWide ? 1 : 4; o < 32; o <<= 1) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        state[i] += __shfl_xor_sync(0xffffffffu, state[i], o);
        seen |= __shfl_xor_sync(0xffffffffu, int(seen), o) != 0;
      }
      // scores that are all -inf: their softmax is NaN, unlike that of no score at all
      if (seen && ref[i] == -INFINITY) sum[i] = NAN;
    }
    __syncthreads();  // the rings are drained
    constexpr int kJoinRow = DIM + 4;
    if constexpr (!kWide) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int r = (i >> 1) * 8 + 2 * (lane & 3) + (i & 1);
        if (lane < 4) ref_s[warp][r] = ref[i], sum_s[warp][r] = sum[i], state_s[warp][r] = state[i];
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (m * 16 < a.dim) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 8 * n + 2 * (lane & 3) + (e & 1), d = m * 16 + (lane >> 2) + 8 * (e >> 1);
              joined[(warp * ROWS + r) * kJoinRow + d] = out[m][4 * n + e];
            }
        }
    } else {
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) ref_s[warp][r] = ref[r], sum_s[warp][r] = sum[r], state_s[warp][r] = state[r];
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int y = 0; y < CT; ++y) joined[(warp * ROWS + r) * kJoinRow + lane + 32 * y] = out[r][y];
    }
    __syncthreads();
    const bool whole = tiles == unit_tiles;
    float* part = nullptr;
    if (!whole) {
      const int slot = unit_begin < chunk * blockIdx.x ? 0 : 1;  // a unit that began before this block's run, or one that goes on after it
      part = a.parts + (int64_t(blockIdx.x) * 2 + slot) * ROWS * a.part_row;
    }
    for (int r = warp; r < rows; r += kWarps) {
      float top = ref_s[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ref_s[w][r]);
      float f[kWarps], all = 0.0f, st = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const bool none = top != -INFINITY && ref_s[w][r] == -INFINITY;  // a warp that saw nothing, or only -inf
        f[w] = top == -INFINITY ? 1.0f : exp2f(ref_s[w][r] - top);
        if (!none) all = fmaf(sum_s[w][r], f[w], all), st = fmaf(state_s[w][r], f[w], st);
      }
      float norm = 1.0f;
      if (whole && a.compress != JK_SOFTSIGN) norm = top == -INFINITY ? (all != all ? NAN : 0.0f) : 1.0f / all;
      const int t = (row0 + r) / a.group, g = (row0 + r) - t * a.group;
      const int64_t row = (int64_t(b) * a.new_nodes + t) * a.heads + kv * a.group + g;
      const bool zero = whole && (t >= span.n || (top == -INFINITY && norm == 0.0f));
      for (int d = lane; d < a.dim; d += 32) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) x = fmaf(f[w], joined[(w * ROWS + r) * kJoinRow + d], x);
        if (whole) reinterpret_cast<T*>(a.out_value)[row * a.dim + d] = from_f32<T>(zero ? 0.0f : x * norm);
        else part[r * a.part_row + d] = x;
      }
      if (lane == 0) {
        if (!whole) {
          float* words = part + r * a.part_row + a.part_row - 4;
          words[0] = top, words[1] = all, words[2] = st;
        } else if (a.out_state != nullptr) {
          reinterpret_cast<T*>(a.out_state)[row] = from_f32<T>(zero ? 0.0f : st * norm);
        }
      }
    }
    __syncthreads();  // before the next unit's queries, and before the rings are filled again
    if (a.split) at += tiles;
    else at = until;
  }
}

// Joins the parts of a unit's row that several blocks left; a unit without tiles has zeros.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  __shared__ float factor[2 * kSms];
  __shared__ float scratch[8][4];
  __shared__ __align__(16) float columns[8][128];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t unit_rows = a.group * a.new_nodes;
  const int64_t unit = blockIdx.x / unit_rows;  // sequence and head of the cache
  const int32_t b = static_cast<int32_t>(unit / a.kv_heads), kv = static_cast<int32_t>(unit - int64_t(b) * a.kv_heads);
  const int32_t row_of = blockIdx.x - static_cast<uint32_t>(unit * unit_rows);
  const int32_t t = row_of / a.group, g = row_of - t * a.group;
  const int64_t row = (int64_t(b) * a.new_nodes + t) * a.heads + kv * a.group + g;
  const Span span = span_of(a, b);
  const int32_t tiles = tiles_of(span);
  T* out = reinterpret_cast<T*>(a.out_value) + row * a.dim;
  grid_dependency_wait();
  if (tiles == 0) {
    for (int d = tid; d < a.dim; d += 256) out[d] = from_f32<T>(0.0f);
    if (tid == 0 && a.out_state != nullptr) reinterpret_cast<T*>(a.out_state)[row] = from_f32<T>(0.0f);
    return;
  }
  const int64_t chunk = a.plan[0];
  const int32_t row_block = row_of / a.rows, r = row_of - row_block * a.rows;
  const int64_t begin = a.plan[1 + b] + (int64_t(kv) * a.row_blocks + row_block) * tiles;
  const int32_t first = static_cast<int32_t>(begin / chunk), last = static_cast<int32_t>((begin + tiles - 1) / chunk);
  if (first == last) return;  // one block had all of it
  const int32_t n = last - first + 1;
  // part i: of block first + i; only the first block's can be one that began there
  auto part_at = [&](int32_t i) {
    const int64_t block = first + i;
    return a.parts + ((block * 2 + (begin < chunk * block ? 0 : 1)) * a.rows + r) * a.part_row;
  };
  const int32_t words = a.part_row - 4;
  float top = -INFINITY;
  for (int32_t i = tid; i < n; i += 256) top = fmaxf(top, part_at(i)[words]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) scratch[warp][0] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, scratch[w][0]);
  float all = 0.0f, st = 0.0f;
  for (int32_t i = tid; i < n; i += 256) {
    const float* p = part_at(i) + words;
    const float ref = p[0];
    const float f = top == -INFINITY ? 1.0f : exp2f(ref - top);
    factor[i] = f;
    if (top == -INFINITY || ref != -INFINITY) all = fmaf(p[1], f, all), st = fmaf(p[2], f, st);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    st += __shfl_xor_sync(0xffffffffu, st, o);
  }
  if (lane == 0) scratch[warp][1] = all, scratch[warp][2] = st;
  __syncthreads();
  all = st = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) all += scratch[w][1], st += scratch[w][2];
  float norm = 1.0f;
  if (a.compress != JK_SOFTSIGN) norm = top == -INFINITY ? (all != all ? NAN : 0.0f) : 1.0f / all;
  const bool zero = t >= span.n || (top == -INFINITY && norm == 0.0f);
  if (tid == 0 && a.out_state != nullptr) reinterpret_cast<T*>(a.out_state)[row] = from_f32<T>(zero ? 0.0f : st * norm);
  // a warp has every eighth part, a lane four columns
  for (int32_t d0 = 0; d0 < a.dim; d0 += 128) {
    const int32_t d = d0 + 4 * lane;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < words) {
#pragma unroll 4
      for (int32_t i = warp; i < n; i += 8) {
        const float4 v = *reinterpret_cast<const float4*>(part_at(i) + d);
        const float f = factor[i];
        x.x = fmaf(f, v.x, x.x), x.y = fmaf(f, v.y, x.y), x.z = fmaf(f, v.z, x.z), x.w = fmaf(f, v.w, x.w);
      }
    }
    *reinterpret_cast<float4*>(&columns[warp][4 * lane]) = x;
    __syncthreads();
    if (tid < 128 && d0 + tid < a.dim) {
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) y += columns[w][tid];
      out[d0 + tid] = from_f32<T>(zero ? 0.0f : y * norm);
    }
    __syncthreads();
  }
}

// ---- host

struct Shape {
  int rows, dim;     // template arguments
  int row_blocks;
  size_t shared;
  int stages, stage_bytes, per_sm;
};

// Rows of a block and its shared memory, from sizes alone (the workspace's size depends on them).
inline Shape shape_of(int64_t unit_rows, int64_t rank, int64_t dim, int dtype) {
  Shape s;
  const bool wide = dtype == JK_F32;
  const int size = wide ? 4 : 2;
  s.dim = dim <= 128 ? 128 : dim <= 256 ? 256 : 512;
  // 128 registers of sums a thread at most
  if (wide) s.rows = unit_rows == 1 ? 1 : 8;
  else s.rows = unit_rows <= 8 || s.dim == 512 ? 8 : unit_rows <= 16 || s.dim == 256 ? 16 : 32;
  s.row_blocks = static_cast<int>((unit_rows + s.rows - 1) / s.rows);
  const int64_t key_row = wide ? (rank + 7) / 8 * 8 + 4 : (rank + 15) / 16 * 16 + 8;
  const int64_t value_row = wide ? (dim + 3) / 4 * 4 : (dim + 15) / 16 * 16 + 8;
  s.stage_bytes = static_cast<int>(kKeys * (key_row + value_row) * size + 4 * kKeys + 16);
  const size_t fixed = ((s.rows * key_row * size + 15) & ~15) + ((kWarps * s.rows * (wide ? kKeys : kKeys + 1) * 4 + 15) & ~15);
  const size_t join = size_t(kWarps) * s.rows * (s.dim + 4) * 4;
  auto bytes = [&](int stages) {
    const size_t rings = size_t(kWarps) * stages * s.stage_bytes;
    return fixed + (rings > join ? rings : join);
  };
  // two blocks of an SM with three stages each, else one with as many (up to three) as fit
  const size_t half = 102 * 1024, whole = 212 * 1024;
  s.stages = 3, s.per_sm = 2;
  if (bytes(3) > half) {
    if (bytes(2) <= half) s.stages = 2;
    else {
      s.per_sm = 1;
      while (s.stages > 1 && bytes(s.stages) > whole) --s.stages;
    }
  }
  s.shared = bytes(s.stages);
  return s;
}

template <typename T, int ROWS, int DIM>
int launch_one(const Args& a, const Shape& s, int64_t units, cudaStream_t stream) {
  if (cudaFuncSetAttribute(cached_kernel<T, ROWS, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(s.shared)) != cudaSuccess) {
    cudaGetLastError();
    return JK_ERR_LAUNCH;
  }
  cached_kernel<T, ROWS, DIM><<<static_cast<unsigned>(a.split ? a.blocks : units), kThreads, s.shared, stream>>>(a);
  if (int st = launch_status()) return st;
  if (!a.split) return JK_OK;
  launch_dependent(join_kernel<T>, static_cast<unsigned>(int64_t(a.batch) * a.kv_heads * a.group * a.new_nodes), 256, 0, stream, a);
  return launch_status();
}

// One launch, for at most kMaxBatch sequences; defined for each type in a unit of its own.
template <typename T>
int launch(const Args& a, const Shape& s, int64_t units, cudaStream_t stream) {
  if constexpr (std::is_same_v<T, float>) {
    if (s.rows == 1) {
      if (s.dim == 128) return launch_one<T, 1, 128>(a, s, units, stream);
      if (s.dim == 256) return launch_one<T, 1, 256>(a, s, units, stream);
      return launch_one<T, 1, 512>(a, s, units, stream);
    }
    if (s.dim == 128) return launch_one<T, 8, 128>(a, s, units, stream);
    if (s.dim == 256) return launch_one<T, 8, 256>(a, s, units, stream);
    return launch_one<T, 8, 512>(a, s, units, stream);
  } else {
    if (s.dim == 128) {
      if (s.rows == 8) return launch_one<T, 8, 128>(a, s, units, stream);
      if (s.rows == 16) return launch_one<T, 16, 128>(a, s, units, stream);
      return launch_one<T, 32, 128>(a, s, units, stream);
    }
    if (s.dim == 256) {
      if (s.rows == 8) return launch_one<T, 8, 256>(a, s, units, stream);
      return launch_one<T, 16, 256>(a, s, units, stream);
    }
    return launch_one<T, 8, 512>(a, s, units, stream);
  }
}

int launch_f32(const Args& a, const Shape& s, int64_t units, cudaStream_t stream);
int launch_bf16(const Args& a, const Shape& s, int64_t units, cudaStream_t stream);
int launch_f16(const Args& a, const Shape& s, int64_t units, cudaStream_t stream);

}  // namespace cached
}  // namespace jk
