// Scaled embedding lookup with dropout, and dropout of rows: out[i, c] = keep(i, c) * factor * row_i[c].
//
// A flat list of blocks of eight columns, rows one after the other, U of them to a thread: reads and writes of a warp are
// neighbours whatever the width, one row of one token is spread over the CTAs that it needs, and no lane idles but in the
// last CTA.  Bound by memory; with dropout of 16-bit values the generator takes about as long as the values' way.
#include "droprows.cuh"

namespace hb {
int* device_error_word();  // runtime.cu

namespace {

constexpr int kThreads = 256;

struct LookupArgs {
  const void* src;
  void* dst;
  const void* ids;      // null: row i of src for row i
  int64_t n, rows, src_stride, dst_stride;
  int64_t padding;
  uint32_t cols, blocks;  // of a row
  uint32_t magic;       // ceil(2^32 / blocks), 0 where it does not divide exactly
  int idx_bytes;
  int src_width, dst_width;
  Dropout drop;
  int* err;
};

__device__ __forceinline__ int64_t token_row(const LookupArgs& a, int64_t i) {
  if (!a.ids) return i;
  const int64_t id = a.idx_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
  if (id == a.padding) return -1;
  if (id < 0 || id >= a.rows) {
    atomicExch(a.err, HB_ERR_INVALID);
    return -1;
  }
  return id;
}

template <typename TI, typename TO, int U>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const LookupArgs a) {
  const uint64_t first = (uint64_t)blockIdx.x * (kThreads * U);
  const uint64_t row0 = first >> 32 ? first / a.blocks : (uint32_t)first / a.blocks;
  const uint32_t rest = (uint32_t)(first - row0 * a.blocks);
  int64_t row[U], from[U];
  uint32_t block[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t at = rest + u * kThreads + threadIdx.x;
    const uint32_t q = a.magic ? __umulhi(at, a.magic) : at / a.blocks;
    block[u] = at - q * a.blocks;
    row[u] = (int64_t)row0 + q;
    from[u] = row[u] < a.n ? token_row(a, row[u]) : -1;
  }
  Words<block_words<TI>()> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t c = block[u] * kBlockCols;
    if (from[u] >= 0)
      load_words(static_cast<const TI*>(a.src) + from[u] * a.src_stride + c, a.src_width, a.cols - c, in[u]);
  }
  PhiloxKey key = {};
  if (a.drop.drop_below) key = philox_key(a.drop);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row[u] >= a.n) continue;
    float x[kBlockCols];
    if (from[u] >= 0) {
      values_of<TI>(in[u], x);
      if (a.drop.drop_below) {
        drop_block(x, key, a.drop.drop_below, a.drop.factor, block[u], (uint32_t)row[u]);
      } else {
#pragma unroll
        for (int i = 0; i < kBlockCols; ++i) x[i] *= a.drop.factor;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kBlockCols; ++i) x[i] = 0.0f;
    }
    Words<block_words<TO>()> out;
    words_of<TO>(x, out);
    const uint32_t c = block[u] * kBlockCols;
    store_words(static_cast<TO*>(a.dst) + row[u] * a.dst_stride + c, a.dst_width, a.cols - c, out);
  }
}

int lookup(const char* who, LookupArgs a, int src_type, int dst_type, cudaStream_t st) {
  if (a.n == 0) return HB_OK;
  a.err = device_error_word();
  HB_CHECK_ARG(a.err != nullptr, "%s: no error word on this device", who);
  a.blocks = (a.cols + kBlockCols - 1) / kBlockCols;
  // at * (magic * blocks - 2^32) < 2^32 for every local index: exact
  const uint64_t top = (uint64_t)a.blocks + 4 * kThreads;
  a.magic = a.blocks > 1 && top * a.blocks < ((uint64_t)1 << 32) ? (uint32_t)((((uint64_t)1 << 32) + a.blocks - 1) / a.blocks) : 0;
  a.src_width = access_bytes(a.src, a.src_stride, src_type);
  a.dst_width = access_bytes(a.dst, a.dst_stride, dst_type);
  const int64_t items = a.n * a.blocks;
  const bool few = items <= (int64_t)sm_count() * kThreads * 8;
  const int64_t grid = ceil_div(items, (int64_t)kThreads * (few ? 1 : 4));
  HB_CHECK_ARG(grid < ((int64_t)1 << 31), "%s: more blocks than a launch holds", who);
  return with_type(src_type, [&](auto ti) {
    return with_type(dst_type, [&](auto to) -> int {
      using TI = decltype(ti);
      using TO = decltype(to);
      if (few) HB_LAUNCH((embedding_kernel<TI, TO, 1>), (int)grid, kThreads, 0, st, a);
      else HB_LAUNCH((embedding_kernel<TI, TO, 4>), (int)grid, kThreads, 0, st, a);
      return HB_OK;
    });
  });
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" {

int hb_embedding(const void* weight, int weight_type, int64_t weight_stride, int64_t num_rows, int64_t dim, const void* ids,
                 int idx_bytes, int64_t n, int64_t padding_idx, double scale, const hb_drop_t* drop, void* out, int out_type,
                 int64_t out_stride, hb_stream_t stream) {
  HB_CHECK_ARG(n >= 0 && n <= ((int64_t)1 << 32) && dim > 0 && dim < ((int64_t)1 << 24) && num_rows >= 0,
               "hb_embedding: bad sizes");
  HB_CHECK_ARG(type_known(weight_type) && type_known(out_type), "hb_embedding: unknown value type");
  HB_CHECK_ARG(idx_bytes == 4 || idx_bytes == 8, "hb_embedding: idx_bytes must be 4 or 8");
  HB_CHECK_ARG(n == 0 || (ids && out && (weight || num_rows == 0)), "hb_embedding: null argument");
  HB_CHECK_ARG(weight_stride >= 0, "hb_embedding: bad table stride");
  HB_CHECK_ARG(out_stride >= dim || n <= 1, "hb_embedding: output rows overlap");
  LookupArgs a = {};
  const int rc = dropout_of("hb_embedding", scale, drop, &a.drop);
  if (rc != HB_OK) return rc;
  HB_CHECK_ARG(!overlap(weight, weight_stride, weight_type, num_rows, out, out_stride, out_type, n, dim),
               "hb_embedding: the output lies in the table");
  a.src = weight;
  a.dst = out;
  a.ids = ids;
  a.n = n;
  a.rows = num_rows;
  a.src_stride = weight_stride;
  a.dst_stride = out_stride;
  a.padding = padding_idx;
  a.cols = (uint32_t)dim;
  a.idx_bytes = idx_bytes;
  return lookup("hb_embedding", a, weight_type, out_type, (cudaStream_t)stream);
}

int hb_dropout(const void* x, int x_type, int64_t x_stride, int64_t n, int64_t dim, double scale, const hb_drop_t* drop,
               void* y, int y_type, int64_t y_stride, hb_stream_t stream) {
  HB_CHECK_ARG(n >= 0 && n <= ((int64_t)1 << 32) && dim > 0 && dim < ((int64_t)1 << 24), "hb_dropout: bad sizes");
  HB_CHECK_ARG(type_known(x_type) && type_known(y_type), "hb_dropout: unknown value type");
  HB_CHECK_ARG(n == 0 || (x && y), "hb_dropout: null argument");
  HB_CHECK_ARG(x_stride >= 0 && (y_stride >= dim || n <= 1), "hb_dropout: output rows overlap");
  LookupArgs a = {};
  const int rc = dropout_of("hb_dropout", scale, drop, &a.drop);
  if (rc != HB_OK) return rc;
  const bool in_place = x == y && x_type == y_type && (x_stride == y_stride || n <= 1);
  HB_CHECK_ARG(in_place || !overlap(x, x_stride, x_type, n, y, y_stride, y_type, n, dim),
               "hb_dropout: the output is neither apart from the input nor the input itself");
  a.src = x;
  a.dst = y;
  a.n = a.rows = n;
  a.src_stride = x_stride;
  a.dst_stride = y_stride;
  a.cols = (uint32_t)dim;
  return lookup("hb_dropout", a, x_type, y_type, (cudaStream_t)stream);
}

}  // extern "C"
