// Gradient of an embedding table by sorted tokens: dW[v, c] = factor * (sum of the kept g[i, c] over the positions i of
// token v), every gradient row read once, no floating-point atomics.
//
// The tokens are sorted with their positions (runs.cu), and the sorted entries are cut into pieces of equal length, whatever
// token they hold: a token that is a tenth of all positions costs no warp more than another.  32 lanes take 256 columns of a
// piece, sums stay in registers, and a row leaves as soon as its token ends.  What of a token lies in two pieces or more is
// left as fp32 partial rows and added up by a second launch, in the order of the pieces, so that the result depends on
// the sizes of the call alone.
#include "droprows.cuh"
#include "runs.cuh"

namespace hb {
int* device_error_word();  // runtime.cu

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int64_t kNoRow = -1;

// ---- tokens as sort keys: what takes no part (padding, ids outside of the table) sorts last, as num_rows --------------
template <typename Id>
__global__ void __launch_bounds__(kThreads) token_keys_kernel(const Id* ids, int64_t n, int64_t padding, int64_t num_rows,
                                                              int64_t* keys, int* err) {
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int64_t id = ids[i];
    const bool inside = id >= 0 && id < num_rows;
    if (!inside && id != padding) atomicExch(err, HB_ERR_INVALID);
    keys[i] = inside && id != padding ? id : num_rows;
  }
}

// ---- sums ---------------------------------------------------------------------------------------------------------------
struct GradArgs {
  hb_runs_t runs;
  const void* grads;
  int64_t grad_stride;
  int grad_width;
  uint32_t cols, blocks, tiles;  // columns, blocks of eight, tiles of `lanes` blocks
  int lanes;                     // of a unit, a power of two
  int64_t per;                   // sorted entries of a piece, a multiple of 8
  int64_t pieces;
  float* parts;                  // [pieces][2][tiles * lanes * 8]: what the piece has of the token before, of the token behind
  Dropout drop;
  void* out;
  int64_t out_stride;
  int out_width;
  int64_t num_rows;
  bool by_run;                   // rows of the output are runs, not tokens
  bool accumulate;
  int64_t* num_unique;           // nullable
};

// Entries and runs that take part: the run of what does not is the last one.
__device__ __forceinline__ void taking_part(const GradArgs& a, int64_t& entries, int64_t& runs) {
  runs = *a.runs.num_runs;
  entries = runs_valid_entries(a.runs);
  if (runs > 0 && a.runs.uniq_ids[runs - 1] >= a.num_rows) entries = a.runs.run_start[--runs];
  if (runs <= 0) entries = 0;
}

__device__ __forceinline__ int64_t part_at(const GradArgs& a, int64_t piece, int behind, uint32_t block) {
  return ((piece * 2 + behind) * (int64_t)(a.tiles * a.lanes) + block) * kBlockCols;
}

template <typename TO>
__device__ __forceinline__ void put_row(const GradArgs& a, int64_t run, uint32_t block, float (&x)[kBlockCols]) {
  const int64_t row = a.by_run ? run : a.runs.uniq_ids[run];
  const uint32_t c = block * kBlockCols;
  TO* p = static_cast<TO*>(a.out) + row * a.out_stride + c;
  Words<block_words<TO>()> w;
  if (a.accumulate) {
    float y[kBlockCols];
    load_words(p, a.out_width, a.cols - c, w);
    values_of<TO>(w, y);
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) x[i] = fmaf(x[i], a.drop.factor, y[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) x[i] *= a.drop.factor;
  }
  words_of<TO>(x, w);
  store_words(p, a.out_width, a.cols - c, w);
}

template <typename TG, typename TO>
__global__ void __launch_bounds__(kThreads) grad_sum_kernel(const GradArgs a) {
  constexpr int kFly = sizeof(TG) == 4 ? 4 : 8;  // rows on their way at once
  const int64_t unit = (blockIdx.x * (int64_t)kThreads + threadIdx.x) / a.lanes;
  const int64_t piece = unit / a.tiles;
  const uint32_t block = (uint32_t)(unit - piece * a.tiles) * a.lanes + (threadIdx.x & (a.lanes - 1));
  int64_t entries, runs;
  taking_part(a, entries, runs);
  if (a.num_unique && blockIdx.x == 0 && threadIdx.x == 0) *a.num_unique = runs;
  const int64_t begin = piece * a.per, end = begin + a.per < entries ? begin + a.per : entries;
  if (begin >= end || block >= a.blocks) return;
  const uint32_t c = block * kBlockCols;
  PhiloxKey key = {};
  if (a.drop.drop_below) key = philox_key(a.drop);
  float sum[kBlockCols];
#pragma unroll
  for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
  int64_t run = a.runs.base8[begin >> 3] - 1;  // (of the entry before, which a head at `begin` ends)
  bool before = a.runs.head[begin] == 0;       // the sum belongs to a token that began before the piece
  bool any = before;
  for (int64_t j0 = begin; j0 < end; j0 += kFly) {
    uint32_t pos[kFly];
    uint8_t head[kFly];
    Words<block_words<TG>()> in[kFly];
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      const int64_t j = j0 + k < end ? j0 + k : end - 1;
      pos[k] = a.runs.perm[j];
      head[k] = a.runs.head[j];
    }
#pragma unroll
    for (int k = 0; k < kFly; ++k)
      load_words(static_cast<const TG*>(a.grads) + (int64_t)pos[k] * a.grad_stride + c, a.grad_width, a.cols - c, in[k]);
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (j0 + k >= end) break;
      if (head[k]) {
        if (any) {
          if (before) {
            float* p = a.parts + part_at(a, piece, 0, block);
            *reinterpret_cast<float4*>(p) = make_float4(sum[0], sum[1], sum[2], sum[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
          } else {
            put_row<TO>(a, run, block, sum);
          }
#pragma unroll
          for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
        }
        ++run;
        before = false;
        any = true;
      }
      float x[kBlockCols];
      values_of<TG>(in[k], x);
      if (a.drop.drop_below) drop_block(x, key, a.drop.drop_below, 1.0f, block, pos[k]);
#pragma unroll
      for (int i = 0; i < kBlockCols; ++i) sum[i] += x[i];
    }
  }
  const bool ends = end == entries || a.runs.head[end] != 0;  // its last token goes no further
  if (ends && !before) {
    put_row<TO>(a, run, block, sum);
  } else {
    float* p = a.parts + part_at(a, piece, before ? 0 : 1, block);
    *reinterpret_cast<float4*>(p) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
  }
}

// Tokens that begin in one piece and end in another: the piece that they begin in adds up what the pieces have.  The warps
// of a CTA take a stretch of the pieces each.
template <typename TO>
__global__ void __launch_bounds__(kThreads) grad_join_kernel(const GradArgs a) {
  __shared__ float s_sum[kWarps][32][kBlockCols];
  const int64_t piece = blockIdx.x / a.tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t block = (uint32_t)(blockIdx.x - piece * a.tiles) * a.lanes + lane;
  int64_t entries, runs;
  taking_part(a, entries, runs);
  const int64_t end = (piece + 1) * a.per;
  if (end >= entries || a.runs.head[end]) return;
  const int64_t run = a.runs.base8[end >> 3] - 1;
  if (a.runs.run_start[run] < piece * a.per) return;
  const int64_t stop = run + 1 < runs ? a.runs.run_start[run + 1] : entries;
  const int64_t last = (stop - 1) / a.per, count = last - piece;  // and so many pieces behind this one
  const int64_t share = (count + kWarps - 1) / kWarps;
  float sum[kBlockCols];
#pragma unroll
  for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
  const bool mine = lane < a.lanes && block < a.blocks;
  if (mine) {
    auto add = [&](const float* p) {
      const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
      sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
      sum[4] += y.x; sum[5] += y.y; sum[6] += y.z; sum[7] += y.w;
    };
    if (warp == 0) add(a.parts + part_at(a, piece, 1, block));
    int64_t from = piece + 1 + warp * share, to = from + share;
    if (to > last + 1) to = last + 1;
#pragma unroll 4
    for (int64_t q = from; q < to; ++q) add(a.parts + part_at(a, q, 0, block));
  }
  if (share * 1 < count) {  // (more than one warp had a part)
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) s_sum[warp][lane][i] = sum[i];
    __syncthreads();
    if (warp == 0)
      for (int w = 1; w < kWarps; ++w)
#pragma unroll
        for (int i = 0; i < kBlockCols; ++i) sum[i] += s_sum[w][lane][i];
  }
  if (warp == 0 && mine) put_row<TO>(a, run, block, sum);
}

struct GradPlan {
  int lanes;
  uint32_t blocks, tiles;
  int64_t per, pieces;
  int64_t* keys;
  float* parts;
  void* runs_ws;
  size_t runs_bytes, total;
};

GradPlan make_plan(void* ws, int64_t n, int64_t dim) {
  GradPlan p;
  const int64_t m = n > 0 ? n : 1;
  p.blocks = (uint32_t)ceil_div(dim, kBlockCols);
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes < (int)p.blocks) p.lanes *= 2;
  p.tiles = (uint32_t)ceil_div(p.blocks, p.lanes);
  const int64_t warps = (int64_t)sm_count() * 24;
  const int64_t units = warps * (32 / p.lanes);
  p.per = align_up((size_t)ceil_div(m * p.tiles, units), 8);
  if (p.per > 256) p.per = 256;
  p.pieces = ceil_div(m, p.per);
  Carver cv(ws ? ws : (void*)256);
  p.keys = cv.take<int64_t>(m);
  p.parts = cv.take<float>((size_t)p.pieces * 2 * p.tiles * p.lanes * kBlockCols);
  p.runs_bytes = align_up(hb_runs_workspace_bytes(m), 256);
  p.runs_ws = cv.take<char>(p.runs_bytes);
  p.total = cv.used() + 256;
  return p;
}

struct Call {
  const char* who;
  const void* ids;
  int idx_bytes;
  int64_t n, padding;
  const void* grads;
  int grad_type;
  int64_t grad_stride, dim;
  double scale;
  const hb_drop_t* drop;
  int64_t num_rows;
  void* out;
  int out_type;
  int64_t out_stride;
  bool by_run, accumulate;
  int64_t *uniq_ids, *num_unique;
  void* ws;
  size_t ws_bytes;
  cudaStream_t st;
};

int check_call(const Call& k) {
  HB_CHECK_ARG(k.n >= 0 && k.n < ((int64_t)1 << 31) && k.dim > 0 && k.dim < ((int64_t)1 << 24) && k.num_rows >= 0 &&
                   k.num_rows <= ((int64_t)1 << 60),
               "%s: bad sizes", k.who);
  HB_CHECK_ARG(type_known(k.grad_type) && type_known(k.out_type), "%s: unknown value type", k.who);
  HB_CHECK_ARG(k.idx_bytes == 4 || k.idx_bytes == 8, "%s: idx_bytes must be 4 or 8", k.who);
  HB_CHECK_ARG(k.n == 0 || (k.ids && k.grads), "%s: null argument", k.who);
  HB_CHECK_ARG(k.grad_stride >= 0, "%s: bad gradient stride", k.who);
  HB_CHECK_ARG(!k.out || !overlap(k.grads, k.grad_stride, k.grad_type, k.n, k.out, k.out_stride, k.out_type,
                                  k.by_run ? k.n : k.num_rows, k.dim),
               "%s: the output lies in the gradients", k.who);
  return HB_OK;
}

int grad(const Call& k) {
  GradArgs a = {};
  int rc = dropout_of(k.who, k.scale, k.drop, &a.drop);
  if (rc != HB_OK) return rc;
  const GradPlan p = make_plan(k.ws, k.n, k.dim);
  if (!k.ws || k.ws_bytes < p.total) {
    set_error("%s: workspace of %zu bytes needed, %zu given", k.who, p.total, k.ws_bytes);
    return HB_ERR_WORKSPACE;
  }
  int* err = device_error_word();
  HB_CHECK_ARG(err != nullptr, "%s: no error word on this device", k.who);
  if (!k.by_run && !k.accumulate && k.num_rows > 0) {
    const size_t e = (size_t)type_bytes(k.out_type);
    if (k.out_stride == k.dim || k.num_rows == 1)
      HB_CUDA(cudaMemsetAsync(k.out, 0, (size_t)k.num_rows * k.dim * e, k.st));
    else
      HB_CUDA(cudaMemset2DAsync(k.out, k.out_stride * e, 0, k.dim * e, k.num_rows, k.st));
  }
  if (k.n == 0) {
    if (k.num_unique) HB_CUDA(cudaMemsetAsync(k.num_unique, 0, sizeof(int64_t), k.st));
    return HB_OK;
  }
  const int64_t key_blocks = ceil_div(k.n, kThreads), cap = (int64_t)sm_count() * 8;
  const int key_grid = (int)(key_blocks < cap ? key_blocks : cap);
  if (k.idx_bytes == 8)
    HB_LAUNCH(token_keys_kernel<int64_t>, key_grid, kThreads, 0, k.st, static_cast<const int64_t*>(k.ids), k.n, k.padding,
              k.num_rows, p.keys, err);
  else
    HB_LAUNCH(token_keys_kernel<int32_t>, key_grid, kThreads, 0, k.st, static_cast<const int32_t*>(k.ids), k.n, k.padding,
              k.num_rows, p.keys, err);
  int bits = 1;
  while ((((int64_t)1 << bits) - 1) <= k.num_rows) ++bits;  // keys up to num_rows lie below the sort's sentinel
  rc = runs_build(p.keys, k.n, nullptr, nullptr, 0, bits, nullptr, 0, nullptr, nullptr, k.uniq_ids, nullptr, nullptr, 0,
                  p.runs_ws, p.runs_bytes, &a.runs, k.st);
  if (rc != HB_OK) return rc;
  a.grads = k.grads;
  a.grad_stride = k.grad_stride;
  a.grad_width = access_bytes(k.grads, k.grad_stride, k.grad_type);
  a.cols = (uint32_t)k.dim;
  a.blocks = p.blocks;
  a.tiles = p.tiles;
  a.lanes = p.lanes;
  a.per = p.per;
  a.pieces = p.pieces;
  a.parts = p.parts;
  a.out = k.out;
  a.out_stride = k.out_stride;
  a.out_width = access_bytes(k.out, k.out_stride, k.out_type);
  a.num_rows = k.num_rows;
  a.by_run = k.by_run;
  a.accumulate = k.accumulate;
  a.num_unique = k.num_unique;
  const int64_t sum_grid = ceil_div(p.pieces * p.tiles * p.lanes, kThreads), join_grid = (p.pieces - 1) * p.tiles;
  HB_CHECK_ARG(sum_grid < ((int64_t)1 << 31) && join_grid < ((int64_t)1 << 31), "%s: more blocks than a launch holds", k.who);
  rc = with_type(k.grad_type, [&](auto tg) {
    return with_type(k.out_type, [&](auto to) -> int {
      HB_LAUNCH((grad_sum_kernel<decltype(tg), decltype(to)>), (int)sum_grid, kThreads, 0, k.st, a);
      return HB_OK;
    });
  });
  if (rc != HB_OK || join_grid == 0) return rc;
  return with_type(k.out_type, [&](auto to) -> int {
    HB_LAUNCH(grad_join_kernel<decltype(to)>, (int)join_grid, kThreads, 0, k.st, a);
    return HB_OK;
  });
}

}  // namespace
}  // namespace hb

using namespace hb;

extern "C" {

size_t hb_embedding_grad_workspace_bytes(int64_t n, int64_t dim) {
  return n < 0 || n >= ((int64_t)1 << 31) || dim <= 0 || dim >= ((int64_t)1 << 24) ? 0 : make_plan(nullptr, n, dim).total;
}

int hb_embedding_grad(const void* ids, int idx_bytes, int64_t n, int64_t padding_idx, const void* grads, int grad_type,
                      int64_t grad_stride, int64_t dim, double scale, const hb_drop_t* drop, int64_t num_rows, void* out,
                      int out_type, int64_t out_stride, int accumulate, void* workspace, size_t workspace_bytes,
                      hb_stream_t stream) {
  const Call k{"hb_embedding_grad", ids, idx_bytes, n, padding_idx, grads, grad_type, grad_stride, dim, scale, drop,
               num_rows, out, out_type, out_stride, false, accumulate != 0, nullptr, nullptr, workspace, workspace_bytes,
               (cudaStream_t)stream};
  const int rc = check_call(k);
  if (rc != HB_OK) return rc;
  HB_CHECK_ARG(num_rows == 0 || out, "hb_embedding_grad: null output");
  HB_CHECK_ARG(out_stride >= dim || num_rows <= 1, "hb_embedding_grad: output rows overlap");
  return grad(k);
}

int hb_embedding_grad_rows(const void* ids, int idx_bytes, int64_t n, int64_t padding_idx, const void* grads, int grad_type,
                           int64_t grad_stride, int64_t dim, double scale, const hb_drop_t* drop, int64_t num_rows,
                           int64_t* uniq_ids, float* rows, int64_t* num_unique, void* workspace, size_t workspace_bytes,
                           hb_stream_t stream) {
  const Call k{"hb_embedding_grad_rows", ids, idx_bytes, n, padding_idx, grads, grad_type, grad_stride, dim, scale, drop,
               num_rows, rows, HB_TYPE_F32, dim, true, false, uniq_ids, num_unique, workspace, workspace_bytes,
               (cudaStream_t)stream};
  const int rc = check_call(k);
  if (rc != HB_OK) return rc;
  HB_CHECK_ARG(num_unique && (n == 0 || (uniq_ids && rows)), "hb_embedding_grad_rows: null output");
  return grad(k);
}

}  // extern "C"
