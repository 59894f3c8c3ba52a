// Host side of the propagation over a paged cache (jk_cached_propagation); the kernels are in
// jk_cached.cuh, instantiated by type in jk_cached_{f32,bf16,f16}.cu.
#include "jk_cached.cuh"

#include <cmath>
#include <limits>

namespace jk {
namespace cached {
namespace {

int64_t part_row(int64_t dim) { return (dim + 3) / 4 * 4 + 4; }

// Tiles that a unit can have: the places of a table's row, as far as they are seen.
int64_t tiles_at_most(int64_t page_size, int64_t columns, int64_t window, int64_t new_nodes) {
  const int64_t room = columns > (int64_t(1) << 31) / page_size ? int64_t(1) << 31 : columns * page_size;
  // (with a window tiles may begin up to 15 places before what is seen)
  const int64_t reach = window < 0 || window + new_nodes + kKeys - 1 > room ? room : window + new_nodes + kKeys - 1;
  return reach < 1 ? 1 : (reach + kTile - 1) / kTile;
}

int32_t window_of(int64_t window) { return window < 0 ? -1 : window > 0x7fffffff ? 0x7fffffff : static_cast<int32_t>(window); }

// Bytes of the pieces that rows can be copied in: what addresses, strides and the row's length allow.
int piece_of(const void* base, const int64_t (&stride)[3], int64_t row_bytes) {
  uint64_t odd = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(row_bytes);
  for (int64_t s : stride) odd |= static_cast<uint64_t>(s);
  return (odd & 15) == 0 ? 16 : (odd & 7) == 0 ? 8 : (odd & 3) == 0 ? 4 : 2;
}

// The map of [pages][heads][places][columns], of which a copy fetches 16 places x 128 bytes.
bool make_map(CUtensorMap* map, const void* base, int64_t columns, const int64_t (&stride)[3], int64_t pages, int64_t heads, int64_t page_size,
              int dtype) {
  const uint64_t dims[4] = {static_cast<uint64_t>(columns), static_cast<uint64_t>(page_size), static_cast<uint64_t>(heads), static_cast<uint64_t>(pages)};
  uint64_t strides[3] = {static_cast<uint64_t>(stride[2]), static_cast<uint64_t>(stride[1]), static_cast<uint64_t>(stride[0])};
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] == 1 && strides[i] == 0) strides[i] = 16;  // of a dim of one, any
    if (strides[i] == 0 || strides[i] >= (uint64_t(1) << 40)) return false;
  }
  return make_tmap_4d(map, base, dims, strides, static_cast<uint32_t>(128 / dtype_bytes(dtype)), kKeys, dtype) == JK_OK;
}

}  // namespace
}  // namespace cached
}  // namespace jk

extern "C" {

int64_t jk_cached_propagation_workspace(int64_t batch, int64_t new_nodes, int64_t heads, int64_t kv_heads, int64_t rank, int64_t dim,
                                        int64_t page_size, int64_t columns, int64_t window, int dtype) {
  using namespace jk;
  using namespace jk::cached;
  if (batch < 1 || new_nodes < 1 || heads < 1 || kv_heads < 1 || rank < 1 || dim < 1 || page_size < 1 || columns < 1) return 0;
  if (tiles_at_most(page_size, columns, window_of(window), new_nodes) <= kUnitTiles) return 0;
  int64_t most = 0;
  for (const bool tiled : {false, true}) {
    const Shape s = shape_of(heads / kv_heads * new_nodes, rank, dim, dtype, tiled);
    const int64_t bytes = int64_t(kSms) * s.per_sm * 2 * s.rows * part_row(dim) * 4;
    most = bytes > most ? bytes : most;
  }
  return most;
}

int jk_cached_propagation(const jk_cache_t* cache, const jk_nodes_t* q, float scale, float score_bias, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cached;
  if (cache == nullptr || q == nullptr) return JK_ERR_BAD_ARG;
  const int64_t batch = cache->batch, pages = cache->pages, page_size = cache->page_size, columns = cache->columns;
  const int64_t new_nodes = q->new_nodes, heads = q->heads, kv_heads = q->kv_heads, rank = q->rank, dim = q->dim;
  constexpr int64_t most = 0x7fffffff;
  if (batch < 0 || new_nodes < 0 || new_nodes > kMaxNew || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 65536 || rank < 1 ||
      rank > kMaxRank || dim < 1 || dim > kMaxDim || pages < 0 || pages > most || page_size < 1 || page_size > most || columns < 0 ||
      columns > most || cache->table_stride < 0)
    return JK_ERR_BAD_SHAPE;
  if (q->dtype < 0 || q->dtype > most || !float_dtype(static_cast<int>(q->dtype))) return JK_ERR_BAD_DTYPE;
  if (q->compress != JK_SOFTMAX && q->compress != JK_SOFTSIGN && q->compress != JK_SIGNED_ABS_SOFTMAX) return JK_ERR_UNSUPPORTED_KIND;
  const int dtype = static_cast<int>(q->dtype);
  if ((q->states == nullptr) != (q->out_state == nullptr)) return JK_ERR_BAD_ARG;
  const int32_t window = window_of(q->window);
  const int64_t unit_tiles = pages == 0 || columns == 0 ? 1 : tiles_at_most(page_size, columns, window, new_nodes);
  const bool split = unit_tiles > kUnitTiles;
  if (batch > 0 && new_nodes > 0) {
    if (q->query == nullptr || cache->lengths == nullptr || q->out_value == nullptr || (split && q->workspace == nullptr)) return JK_ERR_BAD_ARG;
    if (pages > 0 && columns > 0 && (q->keys == nullptr || q->values == nullptr || cache->table == nullptr)) return JK_ERR_BAD_ARG;
  }
  if (!aligned16(q->workspace)) return JK_ERR_ALIGNMENT;
  if (int st = check_device()) return st;
  if (batch == 0 || new_nodes == 0) return JK_OK;
  const int64_t size = dtype_bytes(dtype);
  Args a{};
  a.keys = static_cast<const char*>(q->keys), a.values = static_cast<const char*>(q->values), a.states = static_cast<const char*>(q->states);
  for (int i = 0; i < 3; ++i) {
    a.query_stride[i] = q->query_stride[i] * size, a.key_stride[i] = q->key_stride[i] * size;
    a.value_stride[i] = q->value_stride[i] * size, a.state_stride[i] = q->state_stride[i] * size;
  }
  a.table_stride = cache->table_stride, a.pages = pages, a.columns = pages == 0 ? 0 : columns;
  a.new_nodes = static_cast<int32_t>(new_nodes), a.heads = static_cast<int32_t>(heads), a.kv_heads = static_cast<int32_t>(kv_heads);
  a.group = static_cast<int32_t>(heads / kv_heads), a.rank = static_cast<int32_t>(rank), a.dim = static_cast<int32_t>(dim);
  a.page_size = static_cast<uint32_t>(page_size);
  a.window = window;
  a.compress = static_cast<int32_t>(q->compress);
  a.scale = a.compress == JK_SOFTMAX ? static_cast<float>(double(scale) * 1.4426950408889634) : scale;
  a.bias = score_bias;
  // (the softmax leaves a bias out, as it moves all scores together; with one that is no number or
  // infinite they are not apart)
  if (a.compress == JK_SOFTMAX && !std::isfinite(score_bias)) a.scale = std::numeric_limits<float>::quiet_NaN();
  a.key_piece = piece_of(q->keys, a.key_stride, rank * size), a.value_piece = piece_of(q->values, a.value_stride, dim * size);
  Maps maps{};
  Shape s = shape_of(heads / kv_heads * new_nodes, rank, dim, dtype, true);
  // tiled copies: pages of a multiple of 16 places, rows in 16-byte blocks, strides that a map can
  // hold, and a second stage
  a.tiled = a.key_piece == 16 && a.value_piece == 16 && page_size % kKeys == 0 && s.stages > 1 && pages > 0 && a.columns > 0 &&
            make_map(&maps.keys, q->keys, rank, a.key_stride, pages, kv_heads, page_size, dtype) &&
            make_map(&maps.values, q->values, dim, a.value_stride, pages, kv_heads, page_size, dtype);
  if (!a.tiled) s = shape_of(heads / kv_heads * new_nodes, rank, dim, dtype, false);
  a.rows = s.rows, a.row_blocks = s.row_blocks;
  a.key_cols = s.key_cols, a.query_row = s.query_row, a.key_bytes = s.key_bytes;
  a.stages = s.stages, a.stage_bytes = s.stage_bytes, a.ring_bytes = s.ring_bytes;
  a.part_row = static_cast<int32_t>(part_row(dim));
  a.parts = static_cast<float*>(q->workspace);
  a.split = split;
  const int64_t row_bytes = new_nodes * heads * size;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  // sequences of a launch: their tiles are counted in 32 bits
  const int64_t of_one = kv_heads * s.row_blocks * unit_tiles;
  if (of_one > (1 << 30)) return JK_ERR_BAD_SHAPE;
  const int64_t together = (1 << 30) / of_one < kMaxBatch ? (1 << 30) / of_one : kMaxBatch;
  for (int64_t b0 = 0; b0 < batch; b0 += together) {
    a.batch = static_cast<int32_t>(batch - b0 < together ? batch - b0 : together);
    a.query = static_cast<const char*>(q->query) + b0 * a.query_stride[0];
    a.table = cache->table == nullptr ? nullptr : cache->table + b0 * a.table_stride;
    a.lengths = cache->lengths + b0;
    a.counts = q->counts == nullptr ? nullptr : q->counts + b0;
    a.out_value = static_cast<char*>(q->out_value) + b0 * row_bytes * dim;
    a.out_state = q->out_state == nullptr ? nullptr : static_cast<char*>(q->out_state) + b0 * row_bytes;
    const int64_t units = int64_t(a.batch) * kv_heads * s.row_blocks;
    if (units > most || int64_t(a.batch) * heads * new_nodes * ((dim + 127) / 128) > most) return JK_ERR_BAD_SHAPE;
    const int64_t slots = int64_t(kSms) * s.per_sm;
    a.blocks = static_cast<int32_t>(units > slots / unit_tiles ? slots : units * unit_tiles);
    // A block whose run is of two units begins and ends twice, which takes as long as two or three
    // tiles; runs that end with their unit leave up to a run a unit empty, a quarter at most so.
    // (On the device: 4 units of 4097 places, dim 512, 13.4 us, 15.6 with runs of any; 32 units of
    // 2250 places in f32 27.0 and 29.8.)
    a.units = static_cast<int32_t>(units);
    a.whole_runs = a.blocks > 4 * units;
    int status;
    if (dtype == JK_F32) status = launch_f32(a, maps, s, units, st);
    else if (dtype == JK_BF16) status = launch_bf16(a, maps, s, units, st);
    else status = launch_f16(a, maps, s, units, st);
    if (status != JK_OK) return status;
  }
  return JK_OK;
}

}  // extern "C"
