// Host side of the propagation over a paged cache (jk_cached_propagation); the kernels are in
// jk_cached.cuh, instantiated by type in jk_cached_{f32,bf16,f16}.cu.
#include "jk_cached.cuh"

namespace jk {
namespace cached {
namespace {

int64_t part_row(int64_t dim) { return (dim + 3) / 4 * 4 + 4; }

int64_t plan_bytes(int64_t batch) { return ((batch < kMaxBatch ? batch : kMaxBatch) + 2 + 1) / 2 * 16; }

// Bytes of one asynchronous copy: the most that addresses, strides and the row's length allow.
int chunk_of(const void* base, const int64_t (&stride)[3], int64_t row_bytes) {
  uint64_t odd = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(row_bytes);
  for (int64_t s : stride) odd |= static_cast<uint64_t>(s);
  return (odd & 15) == 0 ? 16 : (odd & 7) == 0 ? 8 : (odd & 3) == 0 ? 4 : 0;
}

}  // namespace
}  // namespace cached
}  // namespace jk

extern "C" {

int64_t jk_cached_propagation_workspace(int64_t batch, int64_t new_nodes, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page_size,
                                        int64_t columns, int dtype) {
  using namespace jk;
  using namespace jk::cached;
  (void)page_size, (void)columns;
  if (batch < 1 || new_nodes < 1 || heads < 1 || kv_heads < 1 || dim < 1) return 16;
  const Shape s = shape_of(heads / kv_heads * new_nodes, 1, dim, dtype);
  return plan_bytes(batch) + int64_t(kSms) * 2 * 2 * s.rows * part_row(dim) * 4;
}

int jk_cached_propagation(const void* query, int64_t query_stride_b, int64_t query_stride_t, int64_t query_stride_h, const void* keys,
                          int64_t key_stride_p, int64_t key_stride_h, int64_t key_stride_n, const void* values, int64_t value_stride_p,
                          int64_t value_stride_h, int64_t value_stride_n, const void* states, int64_t state_stride_p, int64_t state_stride_h,
                          int64_t state_stride_n, const int32_t* table, int64_t table_stride, const int32_t* lengths, const int32_t* counts,
                          int64_t batch, int64_t new_nodes, int64_t heads, int64_t kv_heads, int64_t rank, int64_t dim, int64_t pages,
                          int64_t page_size, int64_t columns, int dtype, int64_t window, int compress, float scale, float score_bias,
                          void* out_value, void* out_state, void* workspace, jk_stream_t stream) {
  using namespace jk;
  using namespace jk::cached;
  if (batch < 0 || new_nodes < 0 || new_nodes > kMaxNew || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 65536 || rank < 1 ||
      rank > kMaxRank || dim < 1 || dim > kMaxDim || pages < 0 || pages > 0x7fffffff || page_size < 1 || page_size > 0x7fffffff || columns < 0 ||
      columns > 0x7fffffff || table_stride < 0)
    return JK_ERR_BAD_SHAPE;
  if (!float_dtype(dtype)) return JK_ERR_BAD_DTYPE;
  if (compress != JK_SOFTMAX && compress != JK_SOFTSIGN && compress != JK_SIGNED_ABS_SOFTMAX) return JK_ERR_UNSUPPORTED_KIND;
  if ((states == nullptr) != (out_state == nullptr)) return JK_ERR_BAD_ARG;
  if (batch > 0 && new_nodes > 0) {
    if (query == nullptr || lengths == nullptr || out_value == nullptr || workspace == nullptr) return JK_ERR_BAD_ARG;
    if (pages > 0 && columns > 0 && (keys == nullptr || values == nullptr || table == nullptr)) return JK_ERR_BAD_ARG;
  }
  if (!aligned16(workspace)) return JK_ERR_ALIGNMENT;
  if (int st = check_device()) return st;
  if (batch == 0 || new_nodes == 0) return JK_OK;
  const int64_t size = dtype_bytes(dtype);
  const Shape s = shape_of(heads / kv_heads * new_nodes, rank, dim, dtype);
  Args a{};
  a.keys = static_cast<const char*>(keys), a.values = static_cast<const char*>(values), a.states = static_cast<const char*>(states);
  const int64_t qs[3] = {query_stride_b, query_stride_t, query_stride_h}, ks[3] = {key_stride_p, key_stride_h, key_stride_n};
  const int64_t vs[3] = {value_stride_p, value_stride_h, value_stride_n}, ss[3] = {state_stride_p, state_stride_h, state_stride_n};
  for (int i = 0; i < 3; ++i)
    a.query_stride[i] = qs[i] * size, a.key_stride[i] = ks[i] * size, a.value_stride[i] = vs[i] * size, a.state_stride[i] = ss[i] * size;
  a.table_stride = table_stride, a.pages = pages, a.columns = pages == 0 ? 0 : columns;
  a.new_nodes = static_cast<int32_t>(new_nodes), a.heads = static_cast<int32_t>(heads), a.kv_heads = static_cast<int32_t>(kv_heads);
  a.group = static_cast<int32_t>(heads / kv_heads), a.rank = static_cast<int32_t>(rank), a.dim = static_cast<int32_t>(dim);
  a.page_size = static_cast<uint32_t>(page_size);
  a.window = window < 0 ? -1 : window > 0x7fffffff ? 0x7fffffff : static_cast<int32_t>(window);
  a.compress = compress;
  // the softmax's scores are compared and subtracted in units of log 2, and a bias moves them all
  a.scale = compress == JK_SOFTMAX ? static_cast<float>(double(scale) * 1.4426950408889634) : scale;
  a.bias = score_bias;
  a.rows = s.rows, a.row_blocks = s.row_blocks;
  a.key_chunk = chunk_of(keys, a.key_stride, rank * size), a.value_chunk = chunk_of(values, a.value_stride, dim * size);
  const bool wide = dtype == JK_F32;
  a.key_row = static_cast<int32_t>(wide ? (rank + 7) / 8 * 8 + 4 : (rank + 15) / 16 * 16 + 8);
  a.value_row = static_cast<int32_t>(wide ? (dim + 3) / 4 * 4 : (dim + 15) / 16 * 16 + 8);
  a.stages = s.stages, a.stage_bytes = s.stage_bytes;
  a.part_row = static_cast<int32_t>(part_row(dim));
  a.plan = static_cast<int64_t*>(workspace);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan_bytes(batch));
  // places that a sequence can have, as far as they are seen
  const int64_t room = a.columns > (int64_t(1) << 31) / page_size ? int64_t(1) << 31 : a.columns * page_size;
  const int64_t reach = a.window < 0 || a.window + new_nodes > room ? room : a.window + new_nodes;
  const int64_t unit_tiles = reach < 1 ? 1 : (reach + kTile - 1) / kTile;
  const int64_t row_bytes = new_nodes * heads * size;
  auto st = reinterpret_cast<cudaStream_t>(stream);
  for (int64_t b0 = 0; b0 < batch; b0 += kMaxBatch) {
    a.batch = static_cast<int32_t>(batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch);
    a.query = static_cast<const char*>(query) + b0 * a.query_stride[0];
    a.table = table == nullptr ? nullptr : table + b0 * table_stride;
    a.lengths = lengths + b0;
    a.counts = counts == nullptr ? nullptr : counts + b0;
    a.out_value = static_cast<char*>(out_value) + b0 * row_bytes * dim;
    a.out_state = out_state == nullptr ? nullptr : static_cast<char*>(out_state) + b0 * row_bytes;
    const int64_t units = int64_t(a.batch) * kv_heads * s.row_blocks;
    if (units > 0x7fffffff || int64_t(a.batch) * heads * new_nodes > 0x7fffffff) return JK_ERR_BAD_SHAPE;
    a.split = unit_tiles > kUnitTiles;
    const int64_t slots = int64_t(kSms) * s.per_sm;
    a.blocks = static_cast<int32_t>(units > slots / unit_tiles ? slots : units * unit_tiles);
    int status;
    if (dtype == JK_F32) status = launch_f32(a, s, units, st);
    else if (dtype == JK_BF16) status = launch_bf16(a, s, units, st);
    else status = launch_f16(a, s, units, st);
    if (status != JK_OK) return status;
  }
  return JK_OK;
}

}  // extern "C"
