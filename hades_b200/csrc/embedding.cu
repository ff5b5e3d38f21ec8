// Scaled embedding lookup with dropout, and dropout of rows: out[i, c] = keep(i, c) * factor * row_i[c].
//
// Rows whose blocks of eight columns can be moved at once (rows_kernel): a thread has one block of U rows that follow one
// another, so that U rows are on their way, the column's part of the generator's first rounds is computed once, and a warp
// moves 512 bytes or 1 KB of a row at a time.  Other rows (ragged_kernel): a flat list of blocks, 32 neighbours to a warp, in
// the largest pieces that the rows' starts and ends allow; single words leave through shared memory, halves in pairs that
// neighbouring lanes exchange.
//
// What bounds it: few rows the launch (2 us).  Many without dropout HBM (65,536 distinct tokens x 4,096 bf16: 1.07 GB in 166
// us), or, where rows come again and again, no unit alone (16,384 x 4,096 bf16 of 3,800 tokens 37 us, 32,768 x 2,048 fp32 to
// bf16 of 6,900 tokens 43: L1, L2 and HBM at 40 to 55 % of their peaks, 45 to 60 % of issue slots).  With dropout the
// generator's instructions (the same two 55 us and 55: 70 % of issue slots, 60 % of the ALU's and of the wide multipliers'
// cycles, L2 at 30 %; dropout alone of 65,536 x 4,096 bf16 182).  Ragged rows the issue of their pieces (10,007 x 1,001 fp16
// to fp32: 16 us at 75 % of all slots, 79 % of L1).
#include "droprows.cuh"

namespace hb {
int* device_error_word();  // runtime.cu

namespace {

constexpr int kThreads = 128;  // (us, dropout of 65,536 x 4,096 bf16: 512 threads 189, 256 181, 128 179)
constexpr int kRows = 4;       // of a thread (one 243 us, two 199, four 182, eight 183)
// Blocks of an SM up to which a thread has one (us, one a thread / kRows, or two of ragged rows: bf16 rows of 1,024 with
// dropout at 2,048 blocks an SM 8.2 / 9.7, at 4,096 12.3 / 10.3, at 8,192 16.5 / 14.3, without dropout 8.2 / 8.4, 10.3 / 10.3,
// 14.4 / 13.1; fp16 rows of 1,001 to fp32 10.2 / 11.7, 14.4 / 14.5, 20.6 / 22.5).
constexpr int64_t kFewBlocks = 2048;

struct LookupArgs {
  const void* src;
  void* dst;
  const void* ids;      // null: row i of src for row i
  int64_t first;        // row of the launch's first row
  int64_t rows, src_stride, dst_stride;
  int64_t padding;
  uint32_t n, cols;     // rows of the launch
  Divisor blocks;       // of a row
  int idx_bytes;
  int src_width, dst_width;
  bool dst_linear;      // a row of dst begins where the one before ends
  Dropout drop;
  int* err;
};

// Row of the source for row i of the output, -1: zeros.
__device__ __forceinline__ int64_t source_row(const LookupArgs& a, int64_t i) {
  if (!a.ids) return i;
  const int64_t id = a.idx_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
  if (id == a.padding) return -1;
  if (id < 0 || id >= a.rows) {
    atomicExch(a.err, HB_ERR_INVALID);
    return -1;
  }
  return id;
}

template <typename TI>
__device__ __forceinline__ void scaled_values(const LookupArgs& a, const Words<block_words<TI>()>& in, const PhiloxKey& key,
                                              uint32_t block, uint32_t row, float (&x)[kBlockCols]) {
  values_of<TI>(in, x);
  if (a.drop.drop_below) {
    drop_block(x, key, a.drop.drop_below, a.drop.factor, block, row);
  } else {
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) x[i] *= a.drop.factor;
  }
}

template <typename TI, typename TO, int U>
__global__ void __launch_bounds__(kThreads) rows_kernel(const LookupArgs a) {
  const uint32_t t = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t group = divide(t, a.blocks), block = t - group * a.blocks.by;
  const uint32_t row0 = group * U;
  if (row0 >= a.n) return;
  int64_t from[U];
#pragma unroll
  for (int u = 0; u < U; ++u) from[u] = row0 + u < a.n ? source_row(a, a.first + row0 + u) : -1;
  Words<block_words<TI>()> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (from[u] >= 0) {
      load_block(static_cast<const TI*>(a.src) + from[u] * a.src_stride + block * kBlockCols, in[u]);
    } else {
#pragma unroll
      for (int i = 0; i < block_words<TI>(); ++i) in[u].w[i] = 0u;
    }
  }
  PhiloxKey key = {};
  if (a.drop.drop_below) key = philox_key(a.drop);
  TO* to = static_cast<TO*>(a.dst) + (a.first + row0) * a.dst_stride + block * kBlockCols;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row0 + u >= a.n) break;
    float x[kBlockCols];
    scaled_values<TI>(a, in[u], key, block, (uint32_t)(a.first + row0 + u), x);
    if (from[u] < 0) {
#pragma unroll
      for (int i = 0; i < kBlockCols; ++i) x[i] = 0.0f;  // (not -0 of a negative scale)
    }
    Words<block_words<TO>()> out;
    words_of<TO>(x, out);
    store_block(to + u * a.dst_stride, out);
  }
}

__device__ __forceinline__ int staged_at(int e) { return e + (e >> 3); }

// A block of 16-bit values of rows that begin at any value, to words of memory: where those begin with a block's second
// value, its first goes with the last of the lane before, if that is of the same row.  The whole warp calls it.
__device__ __forceinline__ void store_halves(uint16_t* p, bool valid, bool first, bool last, int cols, const Words<4>& v) {
  const int lane = threadIdx.x & 31;
  const uint32_t before = __shfl_up_sync(0xffffffffu, v.w[3], 1);
  if (!valid) return;
  uint32_t* const even = reinterpret_cast<uint32_t*>(p);
  uint32_t* const odd = reinterpret_cast<uint32_t*>(p + 1);
  if (((uintptr_t)p & 2u) == 0) {
    if (cols == kBlockCols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) even[i] = v.w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (2 * i + 1 < cols) even[i] = v.w[i];
        else if (2 * i < cols) p[2 * i] = (uint16_t)v.w[i];
      }
    }
    return;
  }
  if (first || lane == 0) p[0] = (uint16_t)v.w[0];
  else odd[-1] = __funnelshift_r(before, v.w[0], 16);
  if (cols == kBlockCols) {
#pragma unroll
    for (int i = 0; i < 3; ++i) odd[i] = __funnelshift_r(v.w[i], v.w[i + 1], 16);
    if (last || lane == 31) p[7] = (uint16_t)(v.w[3] >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (2 * i + 2 < cols) odd[i] = __funnelshift_r(v.w[i], v.w[i + 1], 16);
      else if (2 * i + 1 < cols) p[2 * i + 1] = (uint16_t)(v.w[i] >> 16);
    }
  }
}

template <typename TI, typename TO, int U>
__global__ void __launch_bounds__(kThreads) ragged_kernel(const LookupArgs a) {
  __shared__ float s_row[sizeof(TO) == 4 ? kThreads / 32 : 1][32 * (kBlockCols + 1)];
  const int lane = threadIdx.x & 31;
  uint32_t row[U], block[U];
  int64_t from[U];
  Words<block_words<TI>()> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t t = (blockIdx.x * U + u) * kThreads + threadIdx.x;
    row[u] = divide(t, a.blocks);
    block[u] = t - row[u] * a.blocks.by;
    from[u] = row[u] < a.n ? source_row(a, a.first + row[u]) : -1;
  }
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
    const bool valid = row[u] < a.n;
    const uint32_t c = block[u] * kBlockCols;
    const int cols = a.cols - c < kBlockCols ? (int)(a.cols - c) : kBlockCols;
    const int64_t at = a.first + row[u];
    float x[kBlockCols];
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) x[i] = 0.0f;
    if (from[u] >= 0) scaled_values<TI>(a, in[u], key, block[u], (uint32_t)at, x);
    TO* to = static_cast<TO*>(a.dst) + at * a.dst_stride + c;
    if constexpr (sizeof(TO) == 2) {
      Words<4> out;
      words_of<TO>(x, out);
      if (a.dst_width == 2) store_halves(reinterpret_cast<uint16_t*>(to), valid, c == 0, c + kBlockCols >= a.cols, cols, out);
      else if (valid) store_words(to, a.dst_width, cols, out);
    } else if (a.dst_width > 8 || !a.dst_linear) {
      Words<8> out;
      words_of<TO>(x, out);
      if (valid) store_words(to, a.dst_width, cols, out);
    } else {
      // single words, eight apart, would take a store eight times as long: through shared memory they leave in order (the
      // warp's blocks are one stretch of memory: values [0, length) from `begin` on; 30,000 x 1,001: 77 us and 54, and pairs
      // of words still 29.7 and 26.7 for 60,000 x 250)
      float* staged = s_row[threadIdx.x >> 5];
      const int64_t place = at * a.cols + c;
      const int64_t begin = __shfl_sync(0xffffffffu, place, 0);
      const int length = __reduce_max_sync(0xffffffffu, valid ? (int)(place - begin) + cols : 0);
      __syncwarp();
      if (valid) {
#pragma unroll
        for (int i = 0; i < kBlockCols; ++i)
          if (i < cols) staged[staged_at((int)(place - begin) + i)] = x[i];
      }
      __syncwarp();
      for (int e = lane; e < length; e += 32) static_cast<float*>(a.dst)[begin + e] = staged[staged_at(e)];
    }
  }
}

int lookup(const char* who, LookupArgs a, int64_t n, int src_type, int dst_type, cudaStream_t st) {
  if (n == 0) return HB_OK;
  a.err = device_error_word();
  HB_CHECK_ARG(a.err != nullptr, "%s: no error word on this device", who);
  const uint32_t blocks = (a.cols + kBlockCols - 1) / kBlockCols;
  a.blocks = divisor(blocks);
  a.src_width = access_bytes(a.src, a.src_stride, src_type, a.cols);
  a.dst_width = access_bytes(a.dst, a.dst_stride, dst_type, a.cols);
  a.dst_linear = a.dst_stride == a.cols || n == 1;
  const bool whole = whole_blocks(a.src, a.src_stride, src_type, a.cols) && whole_blocks(a.dst, a.dst_stride, dst_type, a.cols);
  const bool few = n * blocks <= sm_count() * kFewBlocks;
  const int64_t most = (((int64_t)1 << 31) / blocks) & ~(int64_t)(kRows - 1);  // rows whose blocks count in 32 bits
  for (int64_t first = 0; first < n; first += most) {
    a.first = first;
    a.n = (uint32_t)(n - first < most ? n - first : most);
    const int rc = with_type(src_type, [&](auto ti) {
      return with_type(dst_type, [&](auto to) -> int {
        using TI = decltype(ti);
        using TO = decltype(to);
        auto grid = [&](int64_t items, int each) { return (int)ceil_div(items, (int64_t)kThreads * each); };
        if (whole && few) HB_LAUNCH((rows_kernel<TI, TO, 1>), grid((int64_t)a.n * blocks, 1), kThreads, 0, st, a);
        else if (whole) HB_LAUNCH((rows_kernel<TI, TO, kRows>), grid(ceil_div(a.n, kRows) * blocks, 1), kThreads, 0, st, a);
        else if (few) HB_LAUNCH((ragged_kernel<TI, TO, 1>), grid((int64_t)a.n * blocks, 1), kThreads, 0, st, a);
        else HB_LAUNCH((ragged_kernel<TI, TO, 2>), grid((int64_t)a.n * blocks, 2), kThreads, 0, st, a);
        return HB_OK;
      });
    });
    if (rc != HB_OK) return rc;
  }
  return HB_OK;
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
  HB_CHECK_ARG(aligned(ids, idx_bytes) && aligned(weight, type_bytes(weight_type)) && aligned(out, type_bytes(out_type)),
               "hb_embedding: ids, table or output not aligned to their values");
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
  a.rows = num_rows;
  a.src_stride = weight_stride;
  a.dst_stride = out_stride;
  a.padding = padding_idx;
  a.cols = (uint32_t)dim;
  a.idx_bytes = idx_bytes;
  return lookup("hb_embedding", a, n, weight_type, out_type, (cudaStream_t)stream);
}

int hb_dropout(const void* x, int x_type, int64_t x_stride, int64_t n, int64_t dim, double scale, const hb_drop_t* drop,
               void* y, int y_type, int64_t y_stride, hb_stream_t stream) {
  HB_CHECK_ARG(n >= 0 && n <= ((int64_t)1 << 32) && dim > 0 && dim < ((int64_t)1 << 24), "hb_dropout: bad sizes");
  HB_CHECK_ARG(type_known(x_type) && type_known(y_type), "hb_dropout: unknown value type");
  HB_CHECK_ARG(n == 0 || (x && y), "hb_dropout: null argument");
  HB_CHECK_ARG(aligned(x, type_bytes(x_type)) && aligned(y, type_bytes(y_type)),
               "hb_dropout: input or output not aligned to its values");
  HB_CHECK_ARG(x_stride >= 0 && (y_stride >= dim || n <= 1), "hb_dropout: output rows overlap");
  LookupArgs a = {};
  const int rc = dropout_of("hb_dropout", scale, drop, &a.drop);
  if (rc != HB_OK) return rc;
  const bool in_place = x == y && x_type == y_type && (x_stride == y_stride || n <= 1);
  HB_CHECK_ARG(in_place || !overlap(x, x_stride, x_type, n, y, y_stride, y_type, n, dim),
               "hb_dropout: the output is neither apart from the input nor the input itself");
  a.src = x;
  a.dst = y;
  a.rows = n;
  a.src_stride = x_stride;
  a.dst_stride = y_stride;
  a.cols = (uint32_t)dim;
  return lookup("hb_dropout", a, n, x_type, y_type, (cudaStream_t)stream);
}

}  // extern "C"
