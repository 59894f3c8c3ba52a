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
//   * A warp has every fourth 16 places of the run to itself: its own ring of shared memory, its own
//     reference and sums, no barrier between warps until the run's end, where the four are joined in
//     shared memory. Where pages hold a multiple of 16 places in 16-byte rows, one lane fetches the 16 by
//     tiled copies of 128-byte columns (4 for rank and dim 128 in 16 bits); else all lanes copy pieces
//     of 16, 8 or 4 bytes (7.0 and 8.8 us for 256 places of 8 heads of rank and dim 64, 13.3 and 14.4 for 4 x
//     4097 of dim 512, 222 and 225 for 32 x 10240 of 8 heads of 128, on the device). One bulk copy a row took
//     326 for the latter: 32 of them are issued one by one.
//   * Few warps fit an SM beside their rings, so a turn is short of instructions: places that all rows see
//     need no masks, and a reference that follows the maximum only once that is 8 (a factor of 256)
//     above it needs a vote a turn in place of a maximum over the warp.
// 16-bit types: both products are warp matrix instructions with the places (scores) and the value's
// columns (sums) as their 16 rows, and the unit's rows as their 8 columns, of which one node of one head
// fills one: S^T = K Q^T, O^T = V^T W^T. W^T leaves the first product with places across the wrong
// lanes; a matrix transpose within the warp turns it. Weights go into the second product as two planes,
// high + low, so their rounding (2^-16 and less) is far below that of the result. f16 has few exponents
// for that, so its weights are 2^7 times as large (softmaxes, whose weights are 2^8 at most then 2^15) or 2^15
// (softsign, below 1), and what they leave is below 2^-32 of a weight of 1 on the reference, or 2^-40.
// f32: the same walk with fused multiply-adds, which keep f32's rounding.
// Exponentials are base 2, of one fused multiply-add: a score times a rate less a reference, which is such a
// product rounded. From references of 2^24 on that rounding is a power of 2 and more (an exponent's
// whole range from 2^31 on), so the product is rounded before the difference too, as the score
// itself has been.
//
// What is not seen has no part in a result, whatever it holds: places past the last node and places
// without a page arrive as zeros, and a tile of which rows see different parts (the newest nodes of a
// draft, the far end of their windows) adds up its values row by row.
#pragma once

#include "jk_host.h"
#include "jk_rows.cuh"
#include "jk_sm100.cuh"

#include <type_traits>

namespace jk {
namespace cached {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kKeys = 16;               // places of a warp's turn
constexpr int kColumn = 2048;           // bytes of 16 places x 128 bytes of their rows: what a tiled copy fetches
constexpr int kTile = kWarps * kKeys;   // places of a block's turn
constexpr int kSms = 148;
constexpr int kMaxPerSm = 3;            // blocks of an SM
constexpr int kMaxBatch = 256;          // sequences of a launch
constexpr int kMaxStages = 2;           // of a warp's ring
constexpr int kMaxRank = 256, kMaxDim = 512, kMaxNew = 64;
// Units of at most so many tiles get a block each, which saves a launch (8 heads of 512 places:
// 13.4 us a call and 11.4 on the device so, 17.7 and 8.4 split; of 1024 places 21.2 and 18.3, 17.6
// and 8.5).
constexpr int kUnitTiles = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;          // by which a score may pass its row's reference, as a power of 2
constexpr float kFar = 16777216.0f;     // references from which a product with the rate is rounded before they are subtracted

struct Args {
  const char *query, *keys, *values, *states;  // states null: none
  int64_t query_stride[3];                     // bytes: sequence, node, head
  int64_t key_stride[3], value_stride[3], state_stride[3];  // bytes: page, head, place
  const int32_t *table, *lengths, *counts;
  int64_t table_stride, pages, columns;
  int32_t batch, new_nodes, heads, kv_heads, group, rank, dim;
  uint32_t page_size;
  int32_t window, compress;
  float scale, bias;                           // softmax: the rate (its scale and log2(e)), which the bias has no part in
  char *out_value, *out_state;
  // layout
  int32_t blocks, row_blocks, rows;       // blocks of the grid; row blocks of a unit's rows, and rows of one
  int32_t key_piece, value_piece;         // bytes of a piece that rows are copied in (16, 8, 4, 2)
  int32_t key_cols;                       // of a key's row read: rank rounded up to the product's steps
  int32_t query_row;                      // elements from one query to the next in shared memory
  int32_t key_bytes, stage_bytes, stages; // of a ring: keys of a stage, a stage, their number
  int32_t ring_bytes;                     // of all rings (and of what is joined in their place)
  int32_t part_row;                       // floats of a row that a block leaves: dim rounded up to 4, reference, sum, state, whether it saw any
  float* parts;                           // [blocks][2][rows][part_row]
  int32_t units;
  bool split, tiled;
  bool whole_runs;                        // a block's run is of one unit: units are few, so that what is left empty is little
};

// ---- a sequence's places

struct Span {
  int32_t n;         // new nodes that count
  int32_t first;     // place of the first of them (may be negative)
  int32_t low, end;  // places that any of them sees: [low, end)
  int32_t base;      // where the tiles begin
};

template <bool TILED>
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
  s.base = TILED ? s.low & ~(kKeys - 1) : s.low;  // a tiled copy's places are of one page
  return s;
}

__device__ __forceinline__ int32_t tiles_of(const Span& s) { return s.low < s.end ? (s.end - s.base + kTile - 1) / kTile : 0; }

__device__ __forceinline__ Span span_as(const Args& a, int32_t b) { return a.tiled ? span_of<true>(a, b) : span_of<false>(a, b); }

// Tiles of a block's run, of `total` tiles.
__device__ __forceinline__ int32_t run_of(const Args& a, int32_t total) {
  const int32_t runs = a.whole_runs ? a.blocks - a.units : a.blocks;
  return total <= runs ? 1 : (total + runs - 1) / runs;
}

__device__ __forceinline__ int32_t filled_up(int32_t tiles, int32_t run) { return run == 1 ? tiles : (tiles + run - 1) / run * run; }

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

// `BYTES` of src, or zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src, bool there) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until at most `pending` of this thread's groups are on their way.
__device__ __forceinline__ void copy_wait(int pending) {
  if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// ---- compressors

__device__ __forceinline__ float power2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What a product becomes: for the softmax nothing yet (its scale is in the rate), else the score.
template <int COMPRESS>
__device__ __forceinline__ float score_of(float dot, float scale, float bias) {
  return COMPRESS == JK_SOFTMAX ? dot : fmaf(dot, scale, bias);
}
// What is compared with the reference.
template <int COMPRESS>
__device__ __forceinline__ float height_of(float s) {
  return COMPRESS == JK_SOFTMAX ? s : fabsf(s);
}
// The power of 2 that all weights are multiplied by, in the sums too.
template <typename T, int COMPRESS>
constexpr float kUp = !std::is_same_v<T, __half> ? 0.0f : COMPRESS == JK_SOFTSIGN ? 15.0f : 7.0f;
constexpr float kSoftsignDown = 1.0f / 32768.0f;  // f16: what takes it out of the softsign's (the softmaxes' sum has it too)

// Its level above the reference, as a power of 2.
template <int COMPRESS>
__device__ __forceinline__ float level_of(float s, float rate, float ref) {
  return fmaf(height_of<COMPRESS>(s), rate, -ref);
}
template <int COMPRESS>
__device__ __forceinline__ float far_level_of(float s, float rate, float ref) {
  return __fsub_rn(__fmul_rn(height_of<COMPRESS>(s), rate), ref);
}
// Its part of the sum (softsign: the weight itself).
template <typename T, int COMPRESS>
__device__ __forceinline__ float mass_of(float s, float level) {
  if (COMPRESS != JK_SOFTSIGN) return power2(level);
  const float w = s / (1.0f + fabsf(s));
  return kUp<T, COMPRESS> == 0.0f ? w : w * (1.0f / kSoftsignDown);
}
// Its weight.
template <int COMPRESS>
__device__ __forceinline__ float weight_of(float s, float mass) {
  if (COMPRESS != JK_SIGNED_ABS_SOFTMAX) return mass;
  return s == 0.0f ? 0.0f : copysignf(mass, s);
}

// A stage holds columns of 128 bytes of its 16 rows, 2048 bytes each, in which the 16-byte block c
// of row r lies at 128 r + 16 (c ^ (r mod 8)): eight rows' blocks c are in different banks. (Tiled
// copies write it so.)
__device__ __forceinline__ int block_at(int row, int c) { return row * 128 + ((c ^ (row & 7)) << 4); }

// Rows of the 16 lanes' places in pieces of 16, 8 or 4 bytes, as their alignment allows, with as
// many lanes a row as have 128 bytes of it; rows that are not `there` arrive as zeros.
template <int BYTES>
__device__ __forceinline__ void load_pieces(char* stage, const char* src, int64_t offset, uint32_t there, int32_t row_bytes, int lane) {
  constexpr int kLanes = 128 / BYTES, kStep = 32 / kLanes;
  const int byte = lane % kLanes * BYTES;
#pragma unroll
  for (int row0 = 0; row0 < kKeys; row0 += kStep) {
    const int row = row0 + lane / kLanes;
    const char* from = src + __shfl_sync(0xffffffffu, offset, row) + byte;
    uint32_t to = shared_at(stage) + block_at(row, byte >> 4) + (byte & 15);
    const bool ok = (there >> row) & 1;
    for (int c = byte; c < row_bytes; c += 128) {
      copy_async<BYTES>(to, from, ok);
      to += kColumn;
      from += 128;
    }
  }
}

// The same for 16-bit rows that begin at any element: 16-byte blocks are put together from the two
// that hold their bytes, through registers. (These loads are waited for. 32 sequences of 10240 f16
// nodes, rank 128: 222 us with a dim of 128, 306 with 124 in pieces of 8, 404 with 126 in pieces of
// 4, 801 with 127 so, 1355 element by element; 126 so would take 762.)
template <typename T>
__device__ __forceinline__ void load_odd_rows(char* dst, const char* src, int64_t offset, uint32_t there, int32_t row_bytes, int lane) {
  const char* from[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) from[q] = src + __shfl_sync(0xffffffffu, offset, 4 * q + (lane >> 3));
#pragma unroll 1
  for (int c = (lane & 7) * 16; c < row_bytes; c += 128) {
    char* to = dst + (c >> 7) * kColumn;
    if (c + 16 <= row_bytes) {
      uint4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[q] = make_uint4(0, 0, 0, 0);
        if ((there >> (4 * q + (lane >> 3))) & 1) v[q] = load16(from[q] + c, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from[q])) & 15u);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(to + block_at(4 * q + (lane >> 3), lane & 7)) = v[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = 4 * q + (lane >> 3);
#pragma unroll 1
        for (int e = c; e < row_bytes; e += sizeof(T))
          *reinterpret_cast<T*>(to + block_at(row, lane & 7) + (e & 15)) = (there >> row) & 1 ? *reinterpret_cast<const T*>(from[q] + e) : from_f32<T>(0.0f);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_rows(char* stage, const char* src, int64_t offset, uint32_t there, int32_t row_bytes, int piece, int lane) {
  if (piece == 16) return load_pieces<16>(stage, src, offset, there, row_bytes, lane);
  if (piece == 8) return load_pieces<8>(stage, src, offset, there, row_bytes, lane);
  if (piece == 4) return load_pieces<4>(stage, src, offset, there, row_bytes, lane);
  if constexpr (sizeof(T) == 2) load_odd_rows<T>(stage, src, offset, there, row_bytes, lane);
}

// One column of 128 bytes of the 16 places from `place` on of a page: a tiled copy, counted on `bar`.
__device__ __forceinline__ void load_column(char* dst, const CUtensorMap* map, uint64_t* bar, int element, int place, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(shared_at(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(shared_at(bar)), "r"(element), "r"(place), "r"(head), "r"(page)
      : "memory");
}

// ---- the kernel

// A turn on its way: which of its places are in the cache and count, and the state of this lane's (lane % 16).
struct Turn {
  uint32_t there;
  float state;
};

// The tensor maps of the tiled copies: dims (columns of a row, places, heads, pages).
struct Maps {
  CUtensorMap keys, values;
};

// 16-bit types: an infinite value times a low plane that is 0 or of the other sign is NaN. A warp whose
// sums `joined` (a row every `join_row` floats) have NaN looks for the values that are none or infinite,
// which alone decide such a sum, and adds those up with their weights in one piece. (Rows with a score
// that is NaN have it in their `masses` too, and stay as they are.) This is a function of its own,
// whose registers the loop does not pay for. (32 sequences of 10240 f16 nodes: 225 us, with an infinity
// in every page 610; 8 new nodes 430 and 3600. Adding up every place again instead: 14 and 160 ms.)
// kOpen: a NaN, of a sum that no infinity has come to yet (sums of finite values may pass f32's range).
constexpr uint32_t kOpen = 0x7fc0beefu;
template <typename T, int COMPRESS, bool TILED>
__device__ __noinline__ void add_infinities(const Args& a, const T* query, const float* refs, const float* masses, float* joined, int join_row,
                                            int32_t b, int32_t kv, int32_t row0, int32_t rows, int32_t key0, int32_t tiles) {
  const int lane = threadIdx.x & 31;
  const float rate = COMPRESS == JK_SOFTMAX ? a.scale : kLog2e;
  const Span span = span_of<TILED>(a, b);
  const int32_t* table = a.table + b * a.table_stride;
  const char *keys = a.keys + kv * a.key_stride[1], *values = a.values + kv * a.value_stride[1];
  uint32_t some = 0;  // rows to mend
  for (int32_t r = 0; r < rows; ++r) {
    if ((row0 + r) / a.group >= span.n || masses[r] != masses[r]) continue;
    bool none = false;
    for (int d = lane; d < a.dim; d += 32) {
      float& sum = joined[r * join_row + d];
      if (sum != sum) none = true, sum = __uint_as_float(kOpen);
    }
    if (__any_sync(0xffffffffu, none)) some |= 1u << r;
  }
  if (some == 0) return;
  for (int32_t i = 0; i < tiles; ++i) {
    // a lane has the place lane % 16 of the turn
    const int32_t place0 = key0 + i * kTile, own = place0 + (lane & 15);
    bool there = own >= span.low && own < span.end;
    int64_t key_at = 0, value_at = 0;
    if (there) {
      const uint32_t column = static_cast<uint32_t>(own) / a.page_size, off = static_cast<uint32_t>(own) - column * a.page_size;
      const int32_t page = table[column];
      there = static_cast<uint32_t>(page) < static_cast<uint64_t>(a.pages);
      if (there) key_at = page * a.key_stride[0] + off * a.key_stride[2], value_at = page * a.value_stride[0] + off * a.value_stride[2];
    }
    const uint32_t in = __ballot_sync(0xffffffffu, there) & 0xffffu;
    uint32_t odd = 0;  // places with a value that is not finite
    if (a.value_piece == 16) {  // eight lanes a row, 16 bytes each
      const char* from[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) from[q] = values + __shfl_sync(0xffffffffu, value_at, 4 * q + (lane >> 3));
      const uint32_t mask = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;  // an exponent of ones: none, or infinite
      for (int c = (lane & 7) * 16; c < a.dim * 2; c += 128) {
        uint4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = (in >> (4 * q + (lane >> 3))) & 1 ? *reinterpret_cast<const uint4*>(from[q] + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t ones = __vcmpeq2(v[q].x & mask, mask) | __vcmpeq2(v[q].y & mask, mask) | __vcmpeq2(v[q].z & mask, mask) |
                                __vcmpeq2(v[q].w & mask, mask);
          odd |= ones != 0 ? 1u << (4 * q + (lane >> 3)) : 0u;
        }
      }
    } else {
      for (int d0 = 0; d0 < a.dim; d0 += 32) {
        const int d = d0 + lane;
        float x[kKeys];
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const T* value = reinterpret_cast<const T*>(values + __shfl_sync(0xffffffffu, value_at, k));
          x[k] = ((in >> k) & 1) && d < a.dim ? to_f32(value[d]) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kKeys; ++k) odd |= fabsf(x[k]) < INFINITY ? 0u : 1u << k;
      }
    }
    odd = __reduce_or_sync(0xffffffffu, odd);
    for (; odd != 0; odd &= odd - 1) {
      const int k = __ffs(odd) - 1;
      const T* value = reinterpret_cast<const T*>(values + __shfl_sync(0xffffffffu, value_at, k));
      const T* key = reinterpret_cast<const T*>(keys + __shfl_sync(0xffffffffu, key_at, k));
      float x[kMaxDim / 32];
#pragma unroll
      for (int e = 0; e < kMaxDim / 32; ++e) x[e] = lane + 32 * e < a.dim ? to_f32(value[lane + 32 * e]) : 0.0f;
      for (uint32_t left = some; left != 0; left &= left - 1) {
        const int r = __ffs(left) - 1;
        const int32_t place = span.first + (row0 + r) / a.group;
        if (place0 + k > place || (a.window >= 0 && place0 + k < int64_t(place) - a.window)) continue;
        // a weight is needed for an infinity that meets a sum that it may change: not NaN, and under the softmax not itself
        bool ask = false;
#pragma unroll
        for (int e = 0; e < kMaxDim / 32; ++e) {
          if (fabsf(x[e]) < INFINITY) continue;
          float& sum = joined[r * join_row + lane + 32 * e];
          if (x[e] != x[e]) sum = NAN;
          else if (__float_as_uint(sum) == kOpen || (sum == sum && !(COMPRESS == JK_SOFTMAX && sum == x[e]))) ask = true;
        }
        if (!__any_sync(0xffffffffu, ask)) continue;
        float dot = 0.0f;
        for (int c = lane; c < a.rank; c += 32) dot = fmaf(to_f32(query[r * a.query_row + c]), to_f32(key[c]), dot);
        const float score = score_of<COMPRESS>(warp_sum32(dot), a.scale, a.bias), ref = refs[r] == -INFINITY ? 0.0f : refs[r];
        const float level = fabsf(ref) >= kFar ? far_level_of<COMPRESS>(score, rate, ref) : level_of<COMPRESS>(score, rate, ref);
        const float w = weight_of<COMPRESS>(score, mass_of<T, COMPRESS>(score, level));
#pragma unroll
        for (int e = 0; e < kMaxDim / 32; ++e) {
          if (fabsf(x[e]) != INFINITY) continue;
          float& sum = joined[r * join_row + lane + 32 * e];
          const float part = w * x[e], both = __float_as_uint(sum) == kOpen ? part : sum + part;
          sum = both == both ? both : NAN;
        }
      }
    }
  }
}

// ROWS: rows of a unit that a block takes (a multiple of 8 for 16-bit types); DIM: columns of the
// value at most. TILED: pages hold a multiple of 16 places, and the maps fetch them.
template <typename T, int ROWS, int DIM, int COMPRESS, bool TILED>
__global__ void __launch_bounds__(kThreads, ROWS * DIM <= 1024 ? kMaxPerSm : 2) cached_kernel(const __grid_constant__ Args a,
                                                                                             const __grid_constant__ Maps maps) {
  constexpr bool kWide = std::is_same_v<T, float>;
  constexpr int NT = kWide ? 1 : ROWS / 8;             // 8-row tiles of the matrix instructions
  constexpr int MT = kWide ? 1 : DIM / 16;             // 16-column tiles of the value
  constexpr int CP = kWide ? DIM / 64 : 1;             // f32: pairs of columns of a lane, 64 columns apart
  // rows whose reference and sum a thread keeps (f32: half of them, lanes 16.. the other half)
  constexpr int OWN = kWide ? (ROWS + 1) / 2 : 2 * NT;
  constexpr int SIZE = sizeof(T);
  constexpr int COLUMN = 128 / SIZE;                   // elements of a 128-byte column
  const float rate = COMPRESS == JK_SOFTMAX ? a.scale : kLog2e;
  extern __shared__ char memory_[];
  __shared__ int32_t before[kMaxBatch + 1];
  __shared__ int32_t scan[kWarps];
  __shared__ float ref_s[kWarps][ROWS], sum_s[kWarps][ROWS], state_s[kWarps][ROWS];
  __shared__ bool seen_s[kWarps][ROWS];
  __shared__ uint64_t landed[kWarps][kMaxStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int fill = 0, take = 0;          // TILED: the stage that the next turn fills, and the one that is taken next, of all units
  uint32_t phase = 0, issued = 0;  // and the phase of the latter; turns that copied something
  bool late = false;               // a wait gave up
  if (TILED && lane == 0) {
    if (warp == 0) prefetch_tmap(&maps.keys), prefetch_tmap(&maps.values);
    for (int i = 0; i < kMaxStages; ++i) mbar_init(&landed[warp][i], 1);
    fence_barrier_init();
  }
  __syncwarp();

  int32_t chunk = 1, at = 0, until = 1;  // (the host sees to it that all tiles are fewer than 2^30)
  if (a.split) {
    // tiles before each sequence; where runs end with a unit, of units that are filled up to whole runs
    int32_t carry = 0;
    for (int turn = 0; turn < (a.whole_runs ? 2 : 1); ++turn) {
      if (turn == 1) chunk = run_of(a, carry), carry = 0;
      if (tid == 0) before[0] = 0;
      for (int32_t base = 0; base < a.batch; base += kThreads) {
        const int32_t b = base + tid;
        int32_t v = b < a.batch ? filled_up(tiles_of(span_of<TILED>(a, b)), chunk) * (a.kv_heads * a.row_blocks) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int32_t up = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += up;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        int32_t add = carry;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) add += scan[w];
          carry += scan[w];
        }
        if (b < a.batch) before[b + 1] = v + add;
      }
    }
    __syncthreads();
    grid_dependency_launch();
    if (!a.whole_runs) chunk = run_of(a, carry);
    at = chunk * int32_t(blockIdx.x) < carry ? chunk * int32_t(blockIdx.x) : carry;
    until = at + chunk < carry ? at + chunk : carry;
  }

  // shared memory: the rings (whose columns begin at multiples of 1024 bytes), queries, and the
  // weights of a tile that is added up row by row
  char* const memory = memory_ + ((1024u - (shared_at(memory_) & 1023u)) & 1023u);
  char* const ring = memory + warp * a.stages * a.stage_bytes;
  float* const joined = reinterpret_cast<float*>(memory);  // [kWarps][ROWS][DIM + 4], once the rings are drained
  T* const query = reinterpret_cast<T*>(memory + a.ring_bytes);
  constexpr int kWeightRow = kWide ? 2 * kKeys : kKeys + 1;  // f32: each weight twice, as its product is with two columns
  float* const weights = reinterpret_cast<float*>(memory + a.ring_bytes + ROWS * a.query_row * SIZE) + warp * (ROWS * kWeightRow);

  while (at < until) {
    // ---- the unit and the run of its tiles
    int32_t b, inner, tile = 0, tiles, unit_tiles;
    int32_t unit_begin = 0;
    if (a.split) {
      int32_t low = 0, high = a.batch - 1;
      while (low < high) {  // the sequence that tile `at` is of: the first that ends after it
        const int32_t mid = (low + high) >> 1;
        if (before[mid + 1] > at) high = mid;
        else low = mid + 1;
      }
      b = low;
    } else {
      b = blockIdx.x / (a.kv_heads * a.row_blocks);
    }
    const Span span = span_of<TILED>(a, b);
    unit_tiles = tiles_of(span);
    if (a.split) {
      const uint32_t in = at - before[b], room = a.whole_runs ? filled_up(unit_tiles, chunk) : unit_tiles;
      inner = in / room;
      tile = in - inner * room;
      unit_begin = at - tile;
      tiles = unit_tiles - tile < until - at ? unit_tiles - tile : until - at;
    } else {
      inner = blockIdx.x - b * (a.kv_heads * a.row_blocks);
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

    // ---- loads
    const char* keys = a.keys + kv * a.key_stride[1];
    const char* values = a.values + kv * a.value_stride[1];
    const char* states = a.states == nullptr ? nullptr : a.states + kv * a.state_stride[1];
    const int32_t* table = a.table + b * a.table_stride;
    const int32_t key0 = span.base + tile * kTile + warp * kKeys;
    const int own_place = lane & 15;
    struct Place {
      int32_t page;  // what the table says, -1: past the end
      uint32_t offset;
    };
    auto page_of = [&](int64_t j, Place& p) {  // of place j (64 bits: turns after the last may lie past 2^31)
      p.page = -1;
      if (j < span.end) {
        const uint32_t column = static_cast<uint32_t>(j) / a.page_size;
        p.offset = static_cast<uint32_t>(j) - column * a.page_size;
        p.page = table[column];
      }
    };
    // TILED: lane l has turn l's of the 32 turns at hand, looked up together; else a lane has that
    // of its place of the next turn
    Place looked_up{-1, 0};
    if (TILED) page_of(int64_t(key0) + lane * kTile, looked_up);
    else page_of(int64_t(key0) + own_place, looked_up);
    auto issue = [&](int32_t i) {
      Turn made{0, 0.0f};
      Place p = looked_up;
      if (TILED) {
        p.page = __shfl_sync(0xffffffffu, looked_up.page, i & 31);
        p.offset = __shfl_sync(0xffffffffu, looked_up.offset, i & 31);
        if ((i & 31) == 31) page_of(int64_t(key0) + (int64_t(i) + 1 + lane) * kTile, looked_up);
      } else {
        page_of(int64_t(key0) + (int64_t(i) + 1) * kTile + own_place, looked_up);
      }
      const bool there = static_cast<uint32_t>(p.page) < static_cast<uint64_t>(a.pages);
      if (i < tiles && !late) {
        if (TILED) {
          const int32_t k0 = key0 + i * kTile;
          const int low = span.low - k0, high = span.end - k0;  // places of this turn that count: [low, high), low < 16
          if (there && high > 0) {
            made.there = (high >= kKeys ? 0xffffu : (1u << high) - 1) & (low <= 0 ? 0xffffu : 0xffffu << low);
            if (lane == 0) {
              char* stage = ring + fill * a.stage_bytes;
              uint64_t* bar = &landed[warp][fill];
              mbar_arrive_expect_tx(bar, a.stage_bytes);
              for (int c = 0; c < a.rank; c += COLUMN, stage += kColumn) load_column(stage, &maps.keys, bar, c, p.offset, kv, p.page);
              for (int c = 0; c < a.dim; c += COLUMN, stage += kColumn) load_column(stage, &maps.values, bar, c, p.offset, kv, p.page);
            }
            fill ^= 1;
            ++issued;
          }
          p.offset += own_place;
        } else {
          made.there = __ballot_sync(0xffffffffu, there) & 0xffffu;
          char* stage = ring + (a.stages == 1 ? 0 : i & 1) * a.stage_bytes;
          const int64_t page = there ? p.page : 0, off = there ? p.offset : 0;
          const int64_t key_at = page * a.key_stride[0] + off * a.key_stride[2], value_at = page * a.value_stride[0] + off * a.value_stride[2];
          load_rows<T>(stage, keys, key_at, made.there, a.rank * SIZE, a.key_piece, lane);
          load_rows<T>(stage + a.key_bytes, values, value_at, made.there, a.dim * SIZE, a.value_piece, lane);
        }
        if (states != nullptr && ((made.there >> own_place) & 1))
          made.state = to_f32(*reinterpret_cast<const T*>(states + p.page * a.state_stride[0] + p.offset * a.state_stride[2]));
      }
      if (!TILED) copy_commit();
      return made;
    };
    const int lead = TILED || a.stages > 1 ? 1 : 0;  // turns on their way while one is worked on
    // ---- this thread's rows: the places they see, [row_low, row_end)
    const int own_row = kWide && ROWS > 1 && lane >= 16 ? OWN : 0;
    int32_t row_low[OWN], row_end[OWN];
    float ref[OWN], base[OWN], sum[OWN], state[OWN];  // base: the reference, 0 while there is none
    bool any[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int r = kWide ? own_row + i : (i >> 1) * 8 + 2 * (lane & 3) + (i & 1);
      const int t = (row0 + r) / a.group;
      const bool counts = r < rows && t < span.n;
      const int32_t place = span.first + t;
      row_end[i] = !counts ? 0 : place + 1 < span.end ? place + 1 : span.end;
      row_low[i] = a.window < 0 || place < a.window ? 0 : place - a.window;
      ref[i] = COMPRESS == JK_SOFTSIGN || !counts ? 0.0f : -INFINITY;
      base[i] = sum[i] = state[i] = 0.0f;
      any[i] = false;
    }
    bool unset = true;  // a row that counts has no reference yet, or one of kFar and more, and is looked at in every turn
    float out[MT][NT * 4];
    uint64_t pairs[kWide ? ROWS : 1][CP];  // f32's sums
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT * 4; ++j) out[i][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < (kWide ? ROWS : 1); ++i)
#pragma unroll
      for (int j = 0; j < CP; ++j) pairs[i][j] = 0;
    Turn first{0, 0.0f};
    for (int32_t i = -lead; i < tiles; ++i) {
      __syncwarp();  // the stage to fill has been read by all lanes
      const Turn made = issue(i + lead);
      const Turn now = lead ? first : made;
      first = made;
      if (i < 0) continue;
      if (i == 0) {
        // ---- queries, and the keys' columns that no copy fills: 0
        for (int r = warp; r < ROWS; r += kWarps) {
          const int t = (row0 + r) / a.group, g = (row0 + r) - t * a.group;
          const bool counts = r < rows && t < span.n;
          const T* from = reinterpret_cast<const T*>(a.query + b * a.query_stride[0] + t * a.query_stride[1] + (kv * a.group + g) * a.query_stride[2]);
          // (f32: columns first)
          for (int c = lane; c < a.key_cols; c += 32) query[kWide ? c * ROWS + r : r * a.query_row + c] = counts && c < a.rank ? from[c] : from_f32<T>(0.0f);
        }
        if (!TILED && a.key_cols > a.rank) {
          for (int i = lane; i < a.stages * kKeys; i += 32) {
            char* k = ring + i / kKeys * a.stage_bytes;
            for (int c = a.rank; c < a.key_cols; ++c)
              *reinterpret_cast<T*>(k + c / COLUMN * kColumn + block_at(i % kKeys, c % COLUMN * SIZE / 16) + c * SIZE % 16) = from_f32<T>(0.0f);
          }
        }
        __syncthreads();
      }
      const uint32_t there = now.there;
      if (!TILED) copy_wait(lead);
      if (there == 0) continue;
      char* const stage = ring + (TILED ? take : a.stages == 1 ? 0 : i & 1) * a.stage_bytes;
      if (TILED) {
        if (!late && !mbar_wait(&landed[warp][take], phase)) {
          late = true;
          g_device_error = JK_ERR_DEVICE_TIMEOUT;
        }
        late = __any_sync(0xffffffffu, late);
        take ^= 1;
        if (take == 0) phase ^= 1;
      }
      __syncwarp();
      char* const stage_values = stage + a.key_bytes;
      const int32_t k0 = key0 + i * kTile;
      // rows see different parts of it
      const bool mixed = (k0 + kKeys < span.end ? k0 + kKeys : span.end) > all_end || (k0 > span.low ? k0 : span.low) < all_low;
      const bool full = there == 0xffffu && !mixed;
      if (TILED && there != 0xffffu) {  // rows of values that do not count: 0, as a weight of 0 is no help against NaN
        for (int r = lane >> 3; r < kKeys; r += 4)
          if (!((there >> r) & 1))
            for (int c = lane & 7; c < (a.stage_bytes - a.key_bytes) / kColumn * 8; c += 8)
              *reinterpret_cast<uint4*>(stage_values + (c >> 3) * kColumn + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // before the next copy into them
        __syncwarp();
      }

      if constexpr (!kWide) {
        // c2: with 8 rows every other step has sums of its own, as the steps wait for one another
        float c[NT][4], c2[4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) c[n][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) c2[e] = 0.0f;
        {
          // K: matrices (places 0-7 | 8-15) x (columns 0-7 | 8-15); Q: rows 0-7 x four times 8
          // columns; two steps at a time, four in a column of 128 bytes
          uint32_t k_at = shared_at(stage) + block_at(lane & 15, lane >> 4);
          uint32_t q_at = shared_at(query + (lane & 7) * a.query_row + (lane >> 3) * 8);
#pragma unroll 2
          for (int k = 0; k < a.key_cols; k += 32) {
            uint32_t ka[4], kb[4];
            ldmatrix4(ka, k_at);
            ldmatrix4(kb, k_at ^ 32);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t q[4];
              ldmatrix4(q, q_at + n * 16 * a.query_row);
              mma<T>(c[n], ka, q[0], q[1]);
              mma<T>(NT == 1 ? c2 : c[n], kb, q[2], q[3]);
            }
            k_at = (k & 32) ? (k_at ^ 64) + kColumn : k_at ^ 64;
            q_at += 64;
          }
        }
        // c[n][e]: place (lane / 4) + 8 (e / 2), row 8 n + 2 (lane % 4) + e % 2
        const int place = lane >> 2;
        float st[2] = {0.0f, 0.0f};
        if (states != nullptr) {
          st[0] = __shfl_sync(0xffffffffu, now.state, place);
          st[1] = __shfl_sync(0xffffffffu, now.state, place + 8);
        }
        // weights in c; FULL: every row sees every place
        auto weigh = [&](auto whole) {
          constexpr bool FULL = decltype(whole)::value;
          bool sees[NT][4];
          float level[NT][4], highest = -INFINITY;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i2 = 2 * n + (e & 1), p = place + 8 * (e >> 1);
              c[n][e] = score_of<COMPRESS>(NT == 1 ? c[n][e] + c2[e] : c[n][e], a.scale, a.bias);
              sees[n][e] = FULL || (((there >> p) & 1) && k0 + p < row_end[i2] && k0 + p >= row_low[i2]);
              any[i2] |= sees[n][e];
              level[n][e] = level_of<COMPRESS>(c[n][e], rate, base[i2]);
              highest = fmaxf(highest, sees[n][e] ? level[n][e] : -INFINITY);
            }
          if (COMPRESS != JK_SOFTSIGN && __any_sync(0xffffffffu, unset || highest > kSlack + kUp<T, COMPRESS>)) {
            unset = false;
#pragma unroll
            for (int i2 = 0; i2 < OWN; ++i2) {
              const int n = i2 >> 1, e = i2 & 1;
              float top = sees[n][e] ? far_level_of<COMPRESS>(c[n][e], rate, kUp<T, COMPRESS>) : -INFINITY;
              if (sees[n][e + 2]) top = fmaxf(top, far_level_of<COMPRESS>(c[n][e + 2], rate, kUp<T, COMPRESS>));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              top = fmaxf(top, ref[i2]);
              const float factor = top == -INFINITY ? 1.0f : power2(ref[i2] - top);
              ref[i2] = top;
              base[i2] = top == -INFINITY ? 0.0f : top;
              unset |= top == -INFINITY;
              sum[i2] *= factor;
              state[i2] *= factor;
              const bool away = fabsf(base[i2]) >= kFar;
              unset |= away;
              level[n][e] = away ? far_level_of<COMPRESS>(c[n][e], rate, base[i2]) : level_of<COMPRESS>(c[n][e], rate, base[i2]);
              level[n][e + 2] = away ? far_level_of<COMPRESS>(c[n][e + 2], rate, base[i2]) : level_of<COMPRESS>(c[n][e + 2], rate, base[i2]);
#pragma unroll
              for (int m = 0; m < MT; ++m) out[m][4 * n + e] *= factor, out[m][4 * n + e + 2] *= factor;
            }
            unset = __any_sync(0xffffffffu, unset);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i2 = 2 * n + (e & 1);
              float w = mass_of<T, COMPRESS>(c[n][e], level[n][e]);
              if (!FULL && !sees[n][e]) w = 0.0f;
              sum[i2] += w;  // (the softsign has no use for it but to see a NaN)
              w = weight_of<COMPRESS>(c[n][e], w);
              if (!FULL && !sees[n][e]) w = 0.0f;
              if (states != nullptr && sees[n][e]) state[i2] = fmaf(w, st[e >> 1], state[i2]);
              c[n][e] = w;
            }
        };
        if (full) weigh(std::true_type());
        else weigh(std::false_type());
        if (!mixed) {
          uint32_t high[NT][2], low[NT][2];
          using P = Two<T>;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const typename P::type hi = P::of(c[n][2 * h], c[n][2 * h + 1]);
              const float2 f = P::back(hi);
              const typename P::type lo = P::of(c[n][2 * h] - f.x, c[n][2 * h + 1] - f.y);
              high[n][h] = transpose8(*reinterpret_cast<const uint32_t*>(&hi));
              low[n][h] = transpose8(*reinterpret_cast<const uint32_t*>(&lo));
            }
          // V^T: matrices (columns 0-7 | 8-15) x (places 0-7 | 8-15), read transposed
          const uint32_t v_at = shared_at(stage_values) + block_at((lane & 7) + ((lane >> 4) & 1) * 8, (lane >> 3) & 1);
#pragma unroll
          for (int m4 = 0; m4 < MT; m4 += 4) {
            if (m4 * 16 < a.dim) {  // (columns past the value's are read and added up for nothing)
#pragma unroll
              for (int m = m4; m < m4 + 4; ++m) {
                uint32_t va[4];
                ldmatrix4_trans(va, (v_at ^ (32 * (m & 3))) + (m >> 2) * kColumn);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  float(&o)[4] = *reinterpret_cast<float(*)[4]>(&out[m][4 * n]);
                  mma<T>(o, va, high[n][0], high[n][1]);
                  mma<T>(o, va, low[n][0], low[n][1]);
                }
              }
            }
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) weights[(8 * n + 2 * (lane & 3) + (e & 1)) * kWeightRow + place + 8 * (e >> 1)] = c[n][e];
          __syncwarp();
#pragma unroll 1
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
                    const uint32_t at0 = static_cast<uint32_t>(32 * (m & 3)), column0 = (m >> 2) * kColumn;
                    const T x0 = *reinterpret_cast<const T*>(stage_values + column0 + k * 128 + ((at0 ^ ((k & 7) << 4)) + 2 * place));
                    const T x1 = *reinterpret_cast<const T*>(stage_values + column0 + k * 128 + (((at0 + 16) ^ ((k & 7) << 4)) + 2 * place));
                    out[m][4 * n + e] = fmaf(w, to_f32(x0), out[m][4 * n + e]);
                    out[m][4 * n + e + 2] = fmaf(w, to_f32(x1), out[m][4 * n + e + 2]);
                  }
                }
              }
          }
        }
      } else {
        // f32: a lane has a place and half of the rows, lanes 16.. the other half; columns in
        // order, one sum a row
        const int place = own_place;
        const float* q = reinterpret_cast<const float*>(query) + own_row;
        uint64_t dots[(OWN + 1) / 2];  // rows in pairs
#pragma unroll
        for (int j = 0; j < (OWN + 1) / 2; ++j) dots[j] = 0;
#pragma unroll 2
        for (int x = 0; x < a.key_cols; x += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(stage + (x >> 5) * kColumn + block_at(place, (x >> 2) & 7));
          const float k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
          for (int x1 = 0; x1 < 4; ++x1) {
            const float* at_x = q + (x + x1) * ROWS;
            if constexpr (OWN == 1) {
              dots[0] = pair(fmaf(k[x1], *at_x, unpair(dots[0]).x), 0.0f);
            } else {
              const uint64_t kk = pair(k[x1], k[x1]);
              if constexpr (OWN == 4) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(at_x);
                dots[0] = fma2(kk, two.x, dots[0]);
                dots[1] = fma2(kk, two.y, dots[1]);
              } else {
                dots[0] = fma2(kk, *reinterpret_cast<const uint64_t*>(at_x), dots[0]);
              }
            }
          }
        }
        float score[OWN], level[OWN];
        bool sees[OWN];
        bool higher = unset;
#pragma unroll
        for (int i2 = 0; i2 < OWN; ++i2) {
          const float2 two = unpair(dots[i2 / 2]);
          score[i2] = score_of<COMPRESS>(i2 % 2 == 0 ? two.x : two.y, a.scale, a.bias);
          sees[i2] = full || (((there >> place) & 1) && k0 + place < row_end[i2] && k0 + place >= row_low[i2]);
          any[i2] |= sees[i2];
          level[i2] = level_of<COMPRESS>(score[i2], rate, base[i2]);
          higher |= sees[i2] && level[i2] > kSlack;  // (kUp is 0)
        }
        if (COMPRESS != JK_SOFTSIGN && __any_sync(0xffffffffu, higher)) {
          float factor[OWN];
          unset = false;
#pragma unroll
          for (int i2 = 0; i2 < OWN; ++i2) {
            float top = sees[i2] ? far_level_of<COMPRESS>(score[i2], rate, 0.0f) : -INFINITY;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, ref[i2]);
            factor[i2] = top == -INFINITY ? 1.0f : power2(ref[i2] - top);
            ref[i2] = top;
            base[i2] = top == -INFINITY ? 0.0f : top;
            unset |= top == -INFINITY;
            sum[i2] *= factor[i2];
            state[i2] *= factor[i2];
            const bool away = fabsf(base[i2]) >= kFar;
            unset |= away;
            level[i2] = away ? far_level_of<COMPRESS>(score[i2], rate, base[i2]) : level_of<COMPRESS>(score[i2], rate, base[i2]);
          }
          unset = __any_sync(0xffffffffu, unset);
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float f = __shfl_sync(0xffffffffu, factor[r % OWN], r < OWN ? 0 : 16);
#pragma unroll
            for (int y = 0; y < CP; ++y) pairs[r][y] = mul2(pairs[r][y], pair(f, f));
          }
        }
#pragma unroll
        for (int i2 = 0; i2 < OWN; ++i2) {
          float w = mass_of<T, COMPRESS>(score[i2], level[i2]);
          w = sees[i2] ? w : 0.0f;
          if (COMPRESS != JK_SOFTSIGN) sum[i2] += w;
          w = sees[i2] ? weight_of<COMPRESS>(score[i2], w) : 0.0f;
          if (states != nullptr && sees[i2]) state[i2] = fmaf(w, now.state, state[i2]);
          *reinterpret_cast<float2*>(weights + (own_row + i2) * kWeightRow + 2 * place) = make_float2(w, w);
        }
        __syncwarp();
        // a lane's columns 2 lane and 2 lane + 1 of every 64
        const char* v = stage_values + (lane >> 4) * kColumn + (lane & 1) * 8;
        const int block = (lane & 15) >> 1;
        if (!mixed) {
          constexpr int AT_ONCE = DIM == 512 ? 2 : 4;  // places whose values are in registers together
#pragma unroll 1
          for (int k4 = 0; k4 < kKeys; k4 += AT_ONCE) {
            uint64_t x[AT_ONCE][CP];
#pragma unroll
            for (int k1 = 0; k1 < AT_ONCE; ++k1)
#pragma unroll
              for (int y = 0; y < CP; ++y) x[k1][y] = *reinterpret_cast<const uint64_t*>(v + 2 * y * kColumn + block_at(k4 + k1, block));
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
              for (int k1 = 0; k1 < AT_ONCE; k1 += 2) {
                const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(weights + r * kWeightRow + 2 * (k4 + k1));
#pragma unroll
                for (int y = 0; y < CP; ++y) pairs[r][y] = fma2(x[k1 + 1][y], w.y, fma2(x[k1][y], w.x, pairs[r][y]));
              }
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < kKeys; ++k) {
            uint64_t x[CP];
#pragma unroll
            for (int y = 0; y < CP; ++y) x[y] = *reinterpret_cast<const uint64_t*>(v + 2 * y * kColumn + block_at(k, block));
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
              const int from = __shfl_sync(0xffffffffu, row_low[r % OWN], r < OWN ? 0 : 16), to = __shfl_sync(0xffffffffu, row_end[r % OWN], r < OWN ? 0 : 16);
              if (k0 + k >= from && k0 + k < to) {
                const uint64_t w = *reinterpret_cast<const uint64_t*>(weights + r * kWeightRow + 2 * k);
#pragma unroll
                for (int y = 0; y < CP; ++y) pairs[r][y] = fma2(x[y], w, pairs[r][y]);
              }
            }
          }
        }
      }
    }
    if (!TILED) copy_wait(0);
    // what gave up waiting still lets its copies land
    for (uint32_t q = issued < 2 ? 0 : issued - 2; TILED && late && q != issued; ++q) mbar_wait(&landed[warp][q & 1], (q >> 1) & 1);

    // ---- the warps' sums, then the block's
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
#pragma unroll
      for (int o = kWide ? 1 : 4; o < (kWide ? 16 : 32); o <<= 1) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        state[i] += __shfl_xor_sync(0xffffffffu, state[i], o);
        any[i] |= __shfl_xor_sync(0xffffffffu, int(any[i]), o) != 0;
      }
    }
    __syncthreads();  // the rings are drained
    constexpr int kJoinRow = DIM + 4;
    if constexpr (!kWide) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int r = (i >> 1) * 8 + 2 * (lane & 3) + (i & 1);
        if (lane < 4) ref_s[warp][r] = ref[i], sum_s[warp][r] = sum[i], state_s[warp][r] = state[i], seen_s[warp][r] = any[i];
      }
      bool none = false;
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (m * 16 < a.dim) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 8 * n + 2 * (lane & 3) + (e & 1), d = m * 16 + (lane >> 2) + 8 * (e >> 1);
              joined[(warp * ROWS + r) * kJoinRow + d] = out[m][4 * n + e];
              none |= out[m][4 * n + e] != out[m][4 * n + e] && d < a.dim;
            }
        }
      if (__any_sync(0xffffffffu, none)) {
        __syncwarp();
        add_infinities<T, COMPRESS, TILED>(a, query, ref_s[warp], sum_s[warp], joined + warp * ROWS * kJoinRow, kJoinRow, b, kv, row0, rows, key0, tiles);
      }
    } else {
#pragma unroll
      for (int i = 0; i < OWN; ++i)
        if ((lane & 15) == 0) {
          const int r = own_row + i;
          ref_s[warp][r] = ref[i], sum_s[warp][r] = sum[i], state_s[warp][r] = state[i], seen_s[warp][r] = any[i];
        }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int y = 0; y < CP; ++y) *reinterpret_cast<uint64_t*>(joined + (warp * ROWS + r) * kJoinRow + 2 * lane + 64 * y) = pairs[r][y];
    }
    __syncthreads();
    const bool whole = tiles == unit_tiles;
    float* part = nullptr;
    if (!whole) {
      const int slot = unit_begin < chunk * int32_t(blockIdx.x) ? 0 : 1;  // a unit that began before this block's run, or one that goes on after it
      part = a.parts + (int64_t(blockIdx.x) * 2 + slot) * ROWS * a.part_row;
    }
    // a warp a row, or where there are few rows all warps
    const int step = rows < kWarps ? kThreads : 32, lane_of = rows < kWarps ? tid : lane;
    for (int r = rows < kWarps ? 0 : warp; r < rows; r += rows < kWarps ? 1 : kWarps) {
      float top = ref_s[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ref_s[w][r]);
      // A reference of -inf: nothing seen, or scores of -inf and NaN alone. Its factor is 0, which
      // leaves a sum of 0 out and keeps NaN.
      float f[kWarps], all = 0.0f, st = 0.0f;
      bool seen = false;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        f[w] = top == -INFINITY ? 1.0f : power2(ref_s[w][r] - top);
        all = fmaf(sum_s[w][r], f[w], all), st = fmaf(state_s[w][r], f[w], st);
        seen |= seen_s[w][r];
      }
      // a softmax of scores that are all -inf is NaN, unlike that of no score at all
      const bool none = top == -INFINITY && !seen;
      float norm = std::is_same_v<T, __half> ? kSoftsignDown : 1.0f;
      if (whole && COMPRESS != JK_SOFTSIGN) norm = top == -INFINITY ? NAN : 1.0f / all;
      const int t = (row0 + r) / a.group, g = (row0 + r) - t * a.group;
      const int64_t row = (int64_t(b) * a.new_nodes + t) * a.heads + kv * a.group + g;
      const bool zero = whole && (t >= span.n || none);
      for (int d = lane_of; d < a.dim; d += step) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) x = fmaf(f[w], joined[(w * ROWS + r) * kJoinRow + d], x);
        if (whole) reinterpret_cast<T*>(a.out_value)[row * a.dim + d] = from_f32<T>(zero ? 0.0f : x * norm);
        else part[r * a.part_row + d] = x;
      }
      if (lane_of == 0) {
        if (!whole) {
          float* words = part + r * a.part_row + a.part_row - 4;
          words[0] = top, words[1] = all, words[2] = st, words[3] = none ? 0.0f : 1.0f;
        } else if (a.out_state != nullptr) {
          reinterpret_cast<T*>(a.out_state)[row] = from_f32<T>(zero ? 0.0f : st * norm);
        }
      }
    }
    if (TILED) fence_proxy_async_smem();
    __syncthreads();  // before the next unit's queries, and before the rings are filled again
    if (a.split && !a.whole_runs) at += tiles;
    else at = until;
  }
}

// Joins the parts of a unit's row that several blocks left, 128 columns a block; a unit without
// tiles has zeros.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  __shared__ int32_t counted[8][2];
  __shared__ float words_s[8][4];
  __shared__ __align__(16) float columns[8][128];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t unit_rows = a.group * a.new_nodes, slices = (a.dim + 127) / 128;
  const int64_t at = blockIdx.x / slices;
  const int32_t d0 = (blockIdx.x - static_cast<uint32_t>(at * slices)) * 128;
  const int64_t unit = at / unit_rows;  // sequence and head of the cache
  const int32_t b = static_cast<int32_t>(unit / a.kv_heads), kv = static_cast<int32_t>(unit - int64_t(b) * a.kv_heads);
  const int32_t row_of = static_cast<int32_t>(at - unit * unit_rows);
  const int32_t t = row_of / a.group, g = row_of - t * a.group;
  const int64_t row = (int64_t(b) * a.new_nodes + t) * a.heads + kv * a.group + g;
  // the blocks' runs, as the first kernel has them (while it runs)
  const Span span = span_as(a, b);
  const int32_t tiles = tiles_of(span);
  int32_t mine = 0, all_tiles = 0, chunk = 1;
  for (int turn = 0; turn < (a.whole_runs ? 2 : 1); ++turn) {
    if (turn == 1) {
      chunk = run_of(a, all_tiles);
      __syncthreads();  // the counts have been read
    }
    mine = all_tiles = 0;
    for (int32_t i = tid; i < a.batch; i += 256) {
      const int32_t n = filled_up(tiles_of(span_as(a, i)), chunk) * (a.kv_heads * a.row_blocks);
      all_tiles += n;
      if (i < b) mine += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
      all_tiles += __shfl_xor_sync(0xffffffffu, all_tiles, o);
    }
    if (lane == 0) counted[warp][0] = mine, counted[warp][1] = all_tiles;
    __syncthreads();
    mine = all_tiles = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) mine += counted[w][0], all_tiles += counted[w][1];
  }
  if (!a.whole_runs) chunk = run_of(a, all_tiles);
  T* out = reinterpret_cast<T*>(a.out_value) + row * a.dim + d0;
  const bool first_slice = tid == 0 && d0 == 0 && a.out_state != nullptr;
  if (tiles == 0) {
    if (tid < 128 && d0 + tid < a.dim) out[tid] = from_f32<T>(0.0f);
    if (first_slice) reinterpret_cast<T*>(a.out_state)[row] = from_f32<T>(0.0f);
    grid_dependency_wait();
    return;
  }
  const int32_t row_block = row_of / a.rows, r = row_of - row_block * a.rows;
  const int32_t begin = mine + (kv * a.row_blocks + row_block) * (a.whole_runs ? filled_up(tiles, chunk) : tiles);
  const int32_t first = begin / chunk, last = (begin + tiles - 1) / chunk;
  grid_dependency_wait();
  if (first == last) return;  // one block had all of it
  // a warp has every eighth part, a lane four columns
  const int32_t words = a.part_row - 4;
  const bool has = d0 + 4 * lane < words;
  float top = -INFINITY, all = 0.0f, st = 0.0f, seen = 0.0f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int32_t block = first + warp; block <= last; block += 4 * 8) {
    float4 v[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (block + 8 * i <= last) {
        // only in the first block it can be a part that began there
        const float* p = a.parts + (((int64_t(block) + 8 * i) * 2 + (begin < chunk * (block + 8 * i) ? 0 : 1)) * a.rows + r) * a.part_row;
        w[i] = *reinterpret_cast<const float4*>(p + words);
        if (has) v[i] = *reinterpret_cast<const float4*>(p + d0 + 4 * lane);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float higher = fmaxf(top, w[i].x);
      const bool none = higher == -INFINITY;
      const float f = none ? 1.0f : power2(top - higher), h = none ? 1.0f : power2(w[i].x - higher);
      all = fmaf(w[i].y, h, all * f);
      st = fmaf(w[i].z, h, st * f);
      seen = fmaxf(seen, w[i].w);
      x.x = fmaf(v[i].x, h, x.x * f), x.y = fmaf(v[i].y, h, x.y * f), x.z = fmaf(v[i].z, h, x.z * f), x.w = fmaf(v[i].w, h, x.w * f);
      top = higher;
    }
  }
  if (lane == 0) words_s[warp][0] = top, words_s[warp][1] = all, words_s[warp][2] = st, words_s[warp][3] = seen;
  *reinterpret_cast<float4*>(&columns[warp][4 * lane]) = x;
  __syncthreads();
  top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, words_s[w][0]);
  float y = 0.0f;
  all = st = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float ref = words_s[w][0], f = top == -INFINITY ? 1.0f : power2(ref - top);
    all = fmaf(words_s[w][1], f, all), st = fmaf(words_s[w][2], f, st);
    seen = fmaxf(seen, words_s[w][3]);
    if (tid < 128) y = fmaf(columns[w][tid], f, y);
  }
  float norm = std::is_same_v<T, __half> ? kSoftsignDown : 1.0f;
  if (a.compress != JK_SOFTSIGN) norm = top == -INFINITY ? NAN : 1.0f / all;
  const bool zero = t >= span.n || (top == -INFINITY && seen == 0.0f);
  if (tid < 128 && d0 + tid < a.dim) out[tid] = from_f32<T>(zero ? 0.0f : y * norm);
  if (first_slice) reinterpret_cast<T*>(a.out_state)[row] = from_f32<T>(zero ? 0.0f : st * norm);
}

// ---- host

struct Shape {
  int rows, dim;     // template arguments
  int row_blocks;
  int key_cols, query_row, key_bytes, stage_bytes, stages, ring_bytes;
  size_t shared;
  int per_sm;        // blocks of an SM
};

// Rows of a block and its shared memory, from sizes alone (the workspace's size depends on them).
inline Shape shape_of(int64_t unit_rows, int64_t rank, int64_t dim, int dtype, bool tiled) {
  Shape s;
  const bool wide = dtype == JK_F32;
  const int size = wide ? 4 : 2, column = 128 / size;
  s.dim = dim <= 64 && !wide ? 64 : dim <= 128 ? 128 : dim <= 256 ? 256 : 512;
  // (On the device, 32 sequences of 10240 f16 nodes, rank and dim 128, 32 heads on 8: 16 rows a
  // unit in blocks of 16 285 us, of 8 420; 32 rows in blocks of 32 432, of 16 554, of 8 830.) 128
  // registers of sums a thread at most (f32: 64, as it keeps a tile's values too); where rows are
  // copied in pieces the copies are what takes time, so blocks have fewer sizes
  if (wide) s.rows = unit_rows == 1 ? 1 : (tiled && unit_rows <= 4) || s.dim == 512 ? 4 : 8;
  else s.rows = !tiled || unit_rows <= 8 || s.dim == 512 ? 8 : unit_rows <= 16 || s.dim == 256 ? 16 : 32;
  s.row_blocks = static_cast<int>((unit_rows + s.rows - 1) / s.rows);
  // columns in the products' steps (two of 16, or 4); queries of 16-bit types an odd number of
  // 16-byte blocks apart, so that eight of them lie in different banks
  s.key_cols = static_cast<int>(wide ? (rank + 3) / 4 * 4 : (rank + 31) / 32 * 32);
  s.query_row = s.key_cols + 16 / size;
  s.key_bytes = static_cast<int>((rank + column - 1) / column) * kColumn;
  s.stage_bytes = s.key_bytes + static_cast<int>((dim + column - 1) / column) * kColumn;
  const int join = kWarps * s.rows * (s.dim + 4) * 4;
  // f32 reads a value's row up to DIM columns
  const int past = wide ? s.dim / column * kColumn - (s.stage_bytes - s.key_bytes) : 0;
  auto ring = [&](int stages) {
    const int bytes = kWarps * stages * s.stage_bytes + past;
    return bytes > join ? bytes : join;
  };
  const int rest = s.rows * s.query_row * size + kWarps * s.rows * (wide ? 2 * kKeys : kKeys + 1) * 4;
  auto blocks = [&](int stages) { return static_cast<int>(227 * 1024 / (1024 + ring(stages) + rest + 4 * 1024)); };
  const int most = s.rows * s.dim <= 1024 ? kMaxPerSm : 2;
  // Two stages a warp in as many blocks of an SM as fit (a third stage gained nothing in any of the
  // cases that are measured); where not even one block has room for two, one stage.
  s.stages = blocks(2) < 1 ? 1 : 2;
  s.per_sm = blocks(s.stages) < most ? blocks(s.stages) : most;
  s.ring_bytes = ring(s.stages);
  s.shared = 1024 + s.ring_bytes + rest;
  return s;
}

template <typename T, int ROWS, int DIM, int COMPRESS, bool TILED>
int launch_kernel(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream) {
  if (cudaFuncSetAttribute(cached_kernel<T, ROWS, DIM, COMPRESS, TILED>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(s.shared)) != cudaSuccess) {
    cudaGetLastError();
    return JK_ERR_LAUNCH;
  }
  cached_kernel<T, ROWS, DIM, COMPRESS, TILED><<<static_cast<unsigned>(a.split ? a.blocks : units), kThreads, s.shared, stream>>>(a, maps);
  if (int st = launch_status()) return st;
  if (!a.split) return JK_OK;
  launch_dependent(join_kernel<T>, static_cast<unsigned>(int64_t(a.batch) * a.heads * a.new_nodes * ((a.dim + 127) / 128)), 256, 0, stream, a);
  return launch_status();
}

template <typename T, int ROWS, int DIM, bool TILED = true>
int launch_one(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream) {
  if (a.compress == JK_SOFTMAX) return launch_kernel<T, ROWS, DIM, JK_SOFTMAX, TILED>(a, maps, s, units, stream);
  if (a.compress == JK_SOFTSIGN) return launch_kernel<T, ROWS, DIM, JK_SOFTSIGN, TILED>(a, maps, s, units, stream);
  return launch_kernel<T, ROWS, DIM, JK_SIGNED_ABS_SOFTMAX, TILED>(a, maps, s, units, stream);
}

// One launch, for at most kMaxBatch sequences; instantiated for each type in a unit of its own.
template <typename T>
int launch(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream) {
  if constexpr (std::is_same_v<T, float>) {
    if (!a.tiled) {
      if (s.rows == 1) {
        if (s.dim == 128) return launch_one<T, 1, 128, false>(a, maps, s, units, stream);
        if (s.dim == 256) return launch_one<T, 1, 256, false>(a, maps, s, units, stream);
        return launch_one<T, 1, 512, false>(a, maps, s, units, stream);
      }
      if (s.dim == 128) return launch_one<T, 8, 128, false>(a, maps, s, units, stream);
      if (s.dim == 256) return launch_one<T, 8, 256, false>(a, maps, s, units, stream);
      return launch_one<T, 4, 512, false>(a, maps, s, units, stream);
    }
    if (s.rows == 1) {
      if (s.dim == 128) return launch_one<T, 1, 128>(a, maps, s, units, stream);
      if (s.dim == 256) return launch_one<T, 1, 256>(a, maps, s, units, stream);
      return launch_one<T, 1, 512>(a, maps, s, units, stream);
    }
    if (s.rows == 4) {
      if (s.dim == 128) return launch_one<T, 4, 128>(a, maps, s, units, stream);
      if (s.dim == 256) return launch_one<T, 4, 256>(a, maps, s, units, stream);
      return launch_one<T, 4, 512>(a, maps, s, units, stream);
    }
    if (s.dim == 128) return launch_one<T, 8, 128>(a, maps, s, units, stream);
    return launch_one<T, 8, 256>(a, maps, s, units, stream);
  } else {
    if (!a.tiled) {
      if (s.dim == 64) return launch_one<T, 8, 64, false>(a, maps, s, units, stream);
      if (s.dim == 128) return launch_one<T, 8, 128, false>(a, maps, s, units, stream);
      if (s.dim == 256) return launch_one<T, 8, 256, false>(a, maps, s, units, stream);
      return launch_one<T, 8, 512, false>(a, maps, s, units, stream);
    }
    if (s.dim == 64) {
      if (s.rows == 8) return launch_one<T, 8, 64>(a, maps, s, units, stream);
      if (s.rows == 16) return launch_one<T, 16, 64>(a, maps, s, units, stream);
      return launch_one<T, 32, 64>(a, maps, s, units, stream);
    }
    if (s.dim == 128) {
      if (s.rows == 8) return launch_one<T, 8, 128>(a, maps, s, units, stream);
      if (s.rows == 16) return launch_one<T, 16, 128>(a, maps, s, units, stream);
      return launch_one<T, 32, 128>(a, maps, s, units, stream);
    }
    if (s.dim == 256) {
      if (s.rows == 8) return launch_one<T, 8, 256>(a, maps, s, units, stream);
      return launch_one<T, 16, 256>(a, maps, s, units, stream);
    }
    return launch_one<T, 8, 512>(a, maps, s, units, stream);
  }
}

int launch_f32(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream);
int launch_bf16(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream);
int launch_f16(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream);

}  // namespace cached
}  // namespace jk
