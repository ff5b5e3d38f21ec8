// Gradient of an embedding table by sorted tokens: dW[v, c] = factor * (sum of the kept g[i, c] over the positions i of
// token v), every gradient row read once, no floating-point atomics.
//
// The tokens are sorted with their positions (runs.cu), and the sorted entries are cut into pieces of equal length, whatever
// token they hold: a token that is a tenth of all positions costs no warp more than another.  32 lanes take 256 columns of a
// piece; rows come through a ring of asynchronous copies in shared memory (where rows begin at 16 bytes a lane copies and reads
// its own eight columns, so that nothing is waited for but the copy), sums stay in registers, and a row leaves as soon as its
// token ends.  What of a token lies in two pieces or more is left as fp32 partial rows, and whoever leaves the last of them adds
// them up, in the order of the pieces, so that the bits do not depend on who that is.
//
// What bounds it: for many wide rows HBM, at the 5 TB/s that rows read and written all over the place reach here (65,536 x
// 1,024 fp16 to fp32 rows: 214 MB in 40 us behind a sort of 27); for fewer the chain sort, look-up of the entries, first rows,
// joins (8,192 x 2,048 bf16: 14 + 2 + 6 + 5 us).  With dropout the generator's 78 instructions a block come on top of some 50.
#include "aside.cuh"
#include "embedding_grad.cuh"
#include "runs.cuh"

namespace hb {
int* device_error_word();  // runtime.cu

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;      // 32 entries each, that a warp looks up at once
constexpr int kGroup = 16;     // pieces whose parts of a token are added up first
constexpr int kWindow = 256;   // sorted entries of a warp
constexpr int kStages = 4;     // rows of a warp's ring (eight: as fast, and no room for the rows that sums are added to)
constexpr int kSumWarps = 4;   // of a CTA
// Warps of an SM that pieces are made for (us, 65,536 x 1,024 fp16: 20 warps 66.7, 24 65.3, 28 74.4; 8,192 x 2,048 bf16:
// 30.2, 30.2, 32.8; two micro-batches of 16,384 x 2,048, a quarter of it padding: 120.3, 121.4, 122.5).  Pieces are a multiple
// of 8 entries and counted over all positions, padding too, whose pieces are empty: of the 24 some 17 to 22 have work.  All
// run at once but for sums that are added to fp32 rows: fp32 gradients then take 45 KB a CTA, of which five, not six, fit an
// SM (without padding, 20 / 24 / 28 warps: fp32 16,384 x 2,048 99 / 118 / 100, 65,536 x 1,024 185 / 184 / 157, bf16 16,384 x
// 2,048 added to fp32 59 / 73 / 60, to bf16 44.5 / 46 / 44).
constexpr int kWarpsOfSm = 24;
constexpr uint32_t kHead = 0x80000000u;

// ---- tokens as sort keys: what takes no part (padding, ids outside of the table) sorts last, as num_rows --------------
struct Zeros {
  char* p;          // rows to zero in the same launch, null: none
  int64_t rows, row_bytes, stride_bytes;
  int width;        // bytes at a time, as all rows allow
};

template <typename Id>
__global__ void __launch_bounds__(kThreads) token_keys_kernel(const Id* ids, int64_t n, int64_t padding, int64_t num_rows,
                                                              int64_t* keys, int* err, Zeros z) {
  const int64_t at = blockIdx.x * (int64_t)kThreads + threadIdx.x, threads = (int64_t)gridDim.x * kThreads;
  for (int64_t i = at; i < n; i += threads) {
    const int64_t id = ids[i];
    const bool inside = id >= 0 && id < num_rows;
    if (!inside && id != padding) atomicExch(err, HB_ERR_INVALID);
    keys[i] = inside && id != padding ? id : num_rows;
  }
  if (!z.p) return;
  const int64_t per_row = z.row_bytes / z.width, items = z.rows * per_row;
  for (int64_t i = at; i < items; i += threads) {
    char* p = z.p + i / per_row * z.stride_bytes + i % per_row * z.width;
    if (z.width == 16) *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
    else if (z.width == 8) *reinterpret_cast<uint2*>(p) = make_uint2(0u, 0u);
    else if (z.width == 4) *reinterpret_cast<uint32_t*>(p) = 0u;
    else *reinterpret_cast<uint16_t*>(p) = 0;
  }
}

// ---- sums ---------------------------------------------------------------------------------------------------------------
struct GradArgs {
  hb_runs_t runs;
  const void* grads;
  uint32_t grad_step;            // bytes from one row to the next
  int align;                     // of the rows' starts, at most 16
  uint32_t cols, blocks, tiles;  // columns, blocks of eight, tiles of `lanes` blocks
  int lanes;                     // of a unit, a power of two; a warp holds 32 / lanes units, pieces that follow one another
  int per;                       // sorted entries of a piece, a multiple of 8
  int64_t pieces;
  float* parts;                  // [pieces][2][tiles * lanes * 8]: what a piece has of the token before, of the token behind
  unsigned* arrived;             // [pieces][3][tiles] parts that are there; zero before
  Dropout drop;
  OutRows out;
  int64_t num_rows;
  bool by_run;                   // rows of the output are runs, not tokens
  int64_t* num_unique;           // nullable
};

__device__ __forceinline__ float* part_at(const GradArgs& a, int64_t piece, int behind, uint32_t block) {
  return a.parts + ((piece * 2 + behind) * (int64_t)(a.tiles * a.lanes) + block) * kBlockCols;
}
__device__ __forceinline__ void put_part(float* p, const float (&x)[kBlockCols]) {
  __stcg(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  __stcg(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
}
__device__ __forceinline__ void add_part(const float* p, float (&sum)[kBlockCols]) {
  const float4 x = __ldcg(reinterpret_cast<const float4*>(p)), y = __ldcg(reinterpret_cast<const float4*>(p) + 1);
  sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
  sum[4] += y.x; sum[5] += y.y; sum[6] += y.z; sum[7] += y.w;
}

// The first and the last entry of the token of entry j, a multiple of 8 and not its first.
struct Extent { uint32_t first, last; };
__device__ __forceinline__ Extent token_at(const GradArgs& a, int64_t j) {
  const int64_t run = a.runs.base8[j >> 3] - 1;
  return {(uint32_t)a.runs.run_start[run], (uint32_t)(a.runs.run_start[run + 1] - 1)};
}

// A unit's part of a token that lies in several pieces, left in `parts`.  Whoever leaves the last one of kGroup pieces adds
// those up, and of the groups' sums whoever leaves the last: then `sum` is the token's.
struct Part {
  bool on;
  int64_t p0, p1;       // pieces that the token begins and ends in
  int64_t first, last;  // of the unit's group
  __device__ __forceinline__ Part(const GradArgs& a, bool on, const Extent& token, int64_t piece) : on(on) {
    const uint32_t per = (uint32_t)a.per;
    p0 = token.first / per;
    p1 = token.last / per;
    const int64_t from = piece / kGroup * kGroup;
    first = p0 > from ? p0 : from;
    last = p1 < from + kGroup - 1 ? p1 : from + kGroup - 1;
  }
  __device__ __forceinline__ unsigned* count(const GradArgs& a, uint32_t tile) const {
    return a.arrived + (first * 3 + (first == p0)) * a.tiles + tile;
  }
  // was: parts of the group that were there before the unit's
  __device__ __forceinline__ bool finish(const GradArgs& a, unsigned was, uint32_t block, unsigned mask, int leader,
                                         float (&sum)[kBlockCols]) const {
    if (was != (unsigned)(last - first)) return false;
    __threadfence();
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
#pragma unroll 8
    for (int64_t k = first; k <= last; ++k) add_part(part_at(a, k, k == p0, block), sum);
    const int64_t g0 = p0 / kGroup, g1 = p1 / kGroup;
    if (g0 == g1) return true;
    put_part(part_at(a, first, first == p0, block), sum);
    __threadfence();
    __syncwarp(mask);
    unsigned groups = 0;
    if ((int)(threadIdx.x & 31) == leader) groups = atomicAdd(a.arrived + (p0 * 3 + 2) * a.tiles + block / a.lanes, 1u);
    if (__shfl_sync(mask, groups, leader) != (unsigned)(g1 - g0)) return false;
    __threadfence();
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
#pragma unroll 8
    for (int64_t g = g0; g <= g1; ++g) add_part(part_at(a, g == g0 ? p0 : g * kGroup, g == g0, block), sum);
    return true;
  }
};

// ---- a unit's columns of a row through shared memory ----------------------------------------------------------------------
// WIDE: rows begin at 16 bytes; a lane copies and reads its own block, copy i of a stage at (i * 32 + lane) * 16.  Others: the
// unit copies the aligned 16 bytes that its columns lie in, as they are in memory, and a lane reads its block from where it is.
template <typename T, bool WIDE>
constexpr int stage_bytes() { return 32 * kBlockCols * (int)sizeof(T) + (WIDE ? 0 : 32 * 16); }
template <typename T> constexpr int added_bytes() { return 32 * kBlockCols * (int)sizeof(T); }

__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async_part(uint32_t to, const void* from, int bytes) {  // the rest of 16: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <typename T>
__device__ __forceinline__ void copy_block(uint32_t stage, const T* p, int lane) {
#pragma unroll
  for (int i = 0; i < block_words<T>() / 4; ++i) copy_async(stage + (i * 32 + lane) * 16, reinterpret_cast<const char*>(p) + i * 16);
}
template <typename T>
__device__ __forceinline__ void copied_block(const char* stage, int lane, Words<block_words<T>()>& v) {
#pragma unroll
  for (int i = 0; i < block_words<T>() / 4; ++i) {
    const uint4 t = reinterpret_cast<const uint4*>(stage)[i * 32 + lane];
    v.w[4 * i] = t.x; v.w[4 * i + 1] = t.y; v.w[4 * i + 2] = t.z; v.w[4 * i + 3] = t.w;
  }
}

// bytes: of the unit's columns, which begin at p; lane l of `lanes`.  (The first 16 may begin in the row before, or, as an
// allocation begins at 16 bytes, at least in the same allocation; the last are cut where the columns end.)
__device__ __forceinline__ void copy_span(uint32_t stage, const char* p, int bytes, int l, int lanes) {
  const int skew = (int)((uintptr_t)p & 15u), all = skew + bytes;
  for (int at = l * 16; at < all; at += lanes * 16) copy_async_part(stage + at, p - skew + at, all - at < 16 ? all - at : 16);
}
// align: of the rows' starts
template <typename T>
__device__ __forceinline__ void span_block(const char* stage, const char* p, int align, int l, Words<block_words<T>()>& v) {
  constexpr int W = block_words<T>();
  const int at = (int)((uintptr_t)p & 15u) + l * (kBlockCols * (int)sizeof(T));
  if (align >= 8) {
    const uint2* s = reinterpret_cast<const uint2*>(stage + at);
#pragma unroll
    for (int i = 0; i < W; i += 2) {
      const uint2 t = s[i / 2];
      v.w[i] = t.x; v.w[i + 1] = t.y;
    }
    return;
  }
  const uint32_t* s = reinterpret_cast<const uint32_t*>(stage + (at & ~3));
#pragma unroll
  for (int i = 0; i < W; ++i) v.w[i] = s[i];
  if constexpr (sizeof(T) == 2)
    if (at & 2) {
      const uint32_t last = s[W];
#pragma unroll
      for (int i = 0; i < W; ++i) v.w[i] = __funnelshift_r(v.w[i], i + 1 < W ? v.w[i + 1] : last, 16);
    }
}

// WIDE: blocks of the gradients and of the output can be moved at once.
template <typename TG, typename TO, bool WIDE>
__global__ void __launch_bounds__(kSumWarps * 32) grad_sum_kernel(const GradArgs a) {
  begin_after_previous();
  __shared__ alignas(16) char s_ring[kSumWarps][kStages][stage_bytes<TG, WIDE>()];
  extern __shared__ __align__(16) char s_dynamic[];  // WIDE: rows that sums are added to
  __shared__ int64_t s_to[kSumWarps][kWindow];                           // where its row of the output begins, in values
  __shared__ alignas(16) uint32_t s_entry[kSumWarps][kWindow + kStages];  // its position; kHead: a token begins
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t index = blockIdx.x * (int64_t)kSumWarps + warp;
  if (a.num_unique && blockIdx.x == 0 && threadIdx.x == 0) {  // (the run of what takes no part is the last one)
    const int64_t runs = *a.runs.num_runs;
    *a.num_unique = runs > 0 && a.runs.uniq_ids[runs - 1] >= a.num_rows ? runs - 1 : runs;
  }
  const int units = 32 / a.lanes, length = units * a.per;
  const int64_t first = index / a.tiles, begin = first * length;  // (one tile where a warp holds several units)
  if (begin >= a.runs.n) return;

  // the warp's entries, and the one behind them; entries that take no part count as heads, and lie behind all others
  const int64_t valid_entries = runs_valid_entries(a.runs);
  int valid = 0;
#pragma unroll 1
  for (int i0 = 0; i0 <= length; i0 += 32 * kBatch) {  // (loads of a kind on their way at once)
    uint32_t word[kBatch];
    int64_t run[kBatch], token[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int64_t i = i0 + q * 32 + lane, j = begin + i;
      const bool in = i <= length && j < valid_entries;
      word[q] = in ? a.runs.perm[j] | (a.runs.head[j] ? kHead : 0u) : 0u;
      run[q] = in ? a.runs.base8[j >> 3] - 1 : -1;
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int64_t i = i0 + q * 32 + lane, j = begin + i;
      const uint32_t octet = (__ballot_sync(0xffffffffu, word[q] >> 31) >> (lane & ~7)) & 0xffu;
      run[q] += __popc(octet & ((2u << (lane & 7)) - 1u));
      token[q] = i <= length && j < valid_entries ? a.runs.uniq_ids[run[q]] : INT64_MAX;
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int i = i0 + q * 32 + lane;
      const bool part = token[q] < a.num_rows;
      if (i <= length) s_entry[warp][i] = part ? word[q] : kHead;
      if (i < length) s_to[warp][i] = (a.by_run ? run[q] : token[q]) * a.out.stride;
      valid += __popc(__ballot_sync(0xffffffffu, part && i < length));
    }
  }
  __syncwarp();

  const int unit = lane / a.lanes;
  const int64_t piece = first * units + unit;
  const uint32_t block = (uint32_t)(index - first * a.tiles) * a.lanes + (lane & (a.lanes - 1));
  const uint32_t c = block * kBlockCols;
  const int from = unit * a.per, to = from + a.per < valid ? from + a.per : valid;
  if (from >= to || block >= a.blocks) return;
  const uint32_t tile_blocks = a.blocks - (block - (lane & (a.lanes - 1)));  // from the unit's first lane on
  const int leader = unit * a.lanes, unit_lanes = tile_blocks < (uint32_t)a.lanes ? (int)tile_blocks : a.lanes;
  const unsigned mask = (unit_lanes == 32 ? ~0u : (1u << unit_lanes) - 1u) << leader;
  const uint32_t* entry = s_entry[warp];
  constexpr int kStageBytes = stage_bytes<TG, WIDE>();
  const int l = lane & (a.lanes - 1);
  const int span_at = WIDE ? 0 : unit * (a.lanes * kBlockCols * (int)sizeof(TG) + 16);  // of the unit in a stage
  const char* stages = s_ring[warp][0] + span_at;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(stages);
  const uint32_t c0 = WIDE ? c : c - l * kBlockCols;  // the first column that the copies are about
  const char* grads = static_cast<const char*>(a.grads) + c0 * sizeof(TG);
  TO* const out = static_cast<TO*>(a.out.p) + c;
  const int span_cols = a.cols - c0 < (uint32_t)(a.lanes * kBlockCols) ? (int)(a.cols - c0) : a.lanes * kBlockCols;
  const int span_bytes = span_cols * (int)sizeof(TG);
  auto row_of = [&](uint32_t word) { return grads + (uint64_t)(word & ~kHead) * a.grad_step; };
  auto load_words4 = [&](int e, uint32_t (&w)[kStages]) {  // (what lies behind the unit's entries is not used)
#pragma unroll
    for (int k = 0; k < kStages; k += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(entry + e + k);
      w[k] = q.x; w[k + 1] = q.y; w[k + 2] = q.z; w[k + 3] = q.w;
    }
  };
  // the row of entry e, and where a token begins with it and the sum is added to what is there, that row
  const bool add = a.out.accumulate;
  constexpr int kAddedBytes = added_bytes<TO>();
  const char* s_added = s_dynamic + warp * kStages * kAddedBytes;
  const uint32_t added = (uint32_t)__cvta_generic_to_shared(s_added);
  auto issue = [&](int e, int k, uint32_t word) {
    if constexpr (WIDE) copy_block(ring + k * kStageBytes, reinterpret_cast<const TG*>(row_of(word)), lane);
    else copy_span(ring + k * kStageBytes, row_of(word), span_bytes, l, unit_lanes);
    if (add && (word & kHead)) {
      const TO* p = out + s_to[warp][e];
      if constexpr (WIDE) copy_block(added + k * kAddedBytes, p, lane);
      else asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    }
  };
  uint32_t now[kStages];
  load_words4(from, now);
#pragma unroll
  for (int k = 0; k < kStages; ++k) {
    if (from + k < to) issue(from + k, k, now[k]);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const bool leads = !(now[0] & kHead), ends = (entry[to] & kHead) != 0;  // (the last token goes no further)
  Extent lead{}, tail{};
  if (leads) lead = token_at(a, begin + from);
  if (!ends) tail = token_at(a, begin + to);
  PhiloxKey key = {};
  if (a.drop.drop_below) key = philox_key(a.drop);
  float sum[kBlockCols];
#pragma unroll
  for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
  bool before = leads;              // the sum belongs to a token that began before the piece
  Words<block_words<TO>()> there = {};  // of the row that the token's sum is added to
  for (int e0 = from; e0 < to; e0 += kStages) {
    uint32_t next[kStages];
    load_words4(e0 + kStages < to ? e0 + kStages : e0, next);
    uint4 draws[2] = {};
#pragma unroll
    for (int k = 0; k < kStages; ++k) {
      const int e = e0 + k;
      if (e >= to) break;
      const bool head = (now[k] & kHead) != 0;
      if (head && e > from) {  // the token before ends
        if (before) put_part(part_at(a, piece, 0, block), sum);
        else put_block<TO, WIDE>(a.out, out + s_to[warp][e - 1], c, sum, WIDE ? &there : nullptr);
#pragma unroll
        for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
        before = false;
      }
      if (k % 2 == 0 && a.drop.drop_below) {  // (of two rows at once, while they are on their way)
        draws[0] = draws_of(key, block, now[k] & ~kHead);
        draws[1] = draws_of(key, block, now[k + 1] & ~kHead);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      Words<block_words<TG>()> in;
      if constexpr (WIDE) {
        copied_block<TG>(stages + k * kStageBytes, lane, in);
        if (add && head) copied_block<TO>(s_added + k * kAddedBytes, lane, there);
      } else {
        __syncwarp(mask);  // (what the unit's other lanes have copied)
        span_block<TG>(stages + k * kStageBytes, row_of(now[k]), a.align, l, in);
        __syncwarp(mask);
      }
      if (a.drop.drop_below) add_kept<TG>(sum, in, draws[k % 2], a.drop.drop_below);
      else add_block<TG>(sum, in);
      if (e + kStages < to) issue(e + kStages, k, next[k]);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
#pragma unroll
    for (int k = 0; k < kStages; ++k) now[k] = next[k];
  }
  if (!before && ends) {
    put_block<TO, WIDE>(a.out, out + s_to[warp][to - 1], c, sum, WIDE ? &there : nullptr);
  } else {
    put_part(part_at(a, piece, !before, block), sum);
  }
  // the tokens that the piece begins and ends with, where they lie in others too.  (What a lane reads of other units was
  // written by lanes of the same columns: each fences its own writes, and the leader counts behind all of them.)
  const bool trails = !before && !ends;
  if (!leads && !trails) return;
  const Part of_lead(a, leads, lead, piece), of_tail(a, trails, tail, piece);
  __threadfence();
  __syncwarp(mask);
  unsigned lead_was = 0, tail_was = 0;
  if (lane == leader) {
    if (leads) lead_was = atomicAdd(of_lead.count(a, block / a.lanes), 1u);
    if (trails) tail_was = atomicAdd(of_tail.count(a, block / a.lanes), 1u);
  }
  lead_was = __shfl_sync(mask, lead_was, leader);
  tail_was = __shfl_sync(mask, tail_was, leader);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Part& part = which == 0 ? of_lead : of_tail;
    if (part.on && part.finish(a, which == 0 ? lead_was : tail_was, block, mask, leader, sum))
      put_block<TO, WIDE>(a.out, out + s_to[warp][which == 0 ? from : to - 1], c, sum);
  }
}

struct GradPlan {
  int lanes, per;
  uint32_t blocks, tiles;
  int64_t pieces;
  int64_t* keys;
  float* parts;
  unsigned *ticket, *arrived;
  int64_t counts;
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
  const int units = 32 / p.lanes;
  const int64_t warps = (int64_t)sm_count() * kWarpsOfSm;
  const int64_t per = (int64_t)align_up((size_t)ceil_div(m * p.tiles, warps * units), 8);
  p.per = (int)(per > kWindow / units ? kWindow / units : per);
  p.pieces = ceil_div(m, p.per);
  Carver cv(ws ? ws : (void*)256);
  p.keys = cv.take<int64_t>(m);
  p.parts = cv.take<float>((size_t)p.pieces * 2 * p.tiles * p.lanes * kBlockCols);
  p.counts = p.pieces * 3 * p.tiles;
  p.arrived = cv.take<unsigned>(p.counts);
  p.ticket = cv.take<unsigned>(1);
  p.runs_bytes = align_up(hb_runs_workspace_bytes(m), 256);
  p.runs_ws = cv.take<char>(p.runs_bytes);
  p.total = cv.used() + 256;
  return p;
}

int check_call(const GradCall& k) {
  HB_CHECK_ARG(k.n >= 0 && k.n < ((int64_t)1 << 31) && k.dim > 0 && k.dim < ((int64_t)1 << 24) && k.num_rows >= 0 &&
                   k.num_rows <= ((int64_t)1 << 60),
               "%s: bad sizes", k.who);
  HB_CHECK_ARG(type_known(k.grad_type) && type_known(k.out_type), "%s: unknown value type", k.who);
  HB_CHECK_ARG(k.idx_bytes == 4 || k.idx_bytes == 8, "%s: idx_bytes must be 4 or 8", k.who);
  HB_CHECK_ARG(k.n == 0 || (k.ids && k.grads), "%s: null argument", k.who);
  HB_CHECK_ARG(aligned(k.ids, k.idx_bytes) && aligned(k.grads, type_bytes(k.grad_type)) && aligned(k.out, type_bytes(k.out_type)) &&
                   aligned(k.uniq_ids, 8) && aligned(k.num_unique, 8) && aligned(k.ws, 16),
               "%s: ids, gradients or outputs not aligned to their values, or the workspace to 16 bytes", k.who);
  HB_CHECK_ARG(k.grad_stride >= 0 && k.grad_stride < ((int64_t)1 << 30), "%s: bad gradient stride", k.who);
  HB_CHECK_ARG(!k.out || !overlap(k.grads, k.grad_stride, k.grad_type, k.n, k.out, k.out_stride, k.out_type,
                                  k.by_run ? k.n : k.num_rows, k.dim),
               "%s: the output lies in the gradients", k.who);
  return HB_OK;
}

int grad(const GradCall& k) {
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
  if (grad_few_takes(k, a.drop.drop_below > 0)) return grad_few(k, a.drop, err);
  if (k.n == 0 && k.num_unique) HB_CUDA(cudaMemsetAsync(k.num_unique, 0, sizeof(int64_t), k.st));
  // Zeros in one stretch come beside the sort (1.07 GB for 8,192 tokens of 4,096 bf16: 218 us with them in front of it, 180
  // beside it; 8 MB 36.9 and 35.1), but for many beside a sort of the whole GPU: they would all leave from the few SMs that it
  // has not taken (262,144 tokens of 1,024 into 537 MB: 424 us beside it, 267 in front; 70,000 of 1,001 into 100 MB 141 and
  // 143, 100,000 of 256 into 26 MB 65 and 77).  Those of rows at a distance come with the tokens' keys.
  Zeros z = {};
  Aside aside;
  if (k.zeros()) {
    const int64_t e = type_bytes(k.out_type);
    if (k.num_rows == 1 || k.out_stride == k.dim) {
      const int64_t bytes = k.num_rows * k.dim * e;
      const bool beside = k.n > 0 && (k.n <= kSortClusterEntries || bytes <= (100 << 20)) && !stream_captures(k.st) &&
                          aside.fork(k.st);
      const cudaStream_t st = beside ? aside.stream() : k.st;
      HB_CUDA(cudaMemsetAsync(p.ticket, 0, sizeof(unsigned), st));
      HB_LAUNCH(zeros_kernel, sm_count(), 32, kZerosChunk, st, static_cast<char*>(k.out), bytes, p.ticket);
    } else {
      z = Zeros{static_cast<char*>(k.out), k.num_rows, k.dim * e, k.out_stride * e, 0};
      const uint64_t width = (uint64_t)(uintptr_t)z.p | (uint64_t)z.row_bytes | (uint64_t)z.stride_bytes | 16u;
      z.width = (int)(width & (~width + 1));
    }
  }
  if (k.n == 0 && !z.p) return HB_OK;
  int bits = 1;
  while ((((int64_t)1 << bits) - 1) <= k.num_rows) ++bits;  // keys up to num_rows lie below the sort's sentinel
  if (k.n > 0 && k.n <= kSortClusterEntries && !z.p) {
    rc = token_runs(k, bits, p.arrived, p.counts, p.runs_ws, &a.runs);
  } else {
    const int64_t items = z.p ? z.rows * (z.row_bytes / z.width) : 0;
    const int64_t key_blocks = ceil_div(k.n > items ? k.n : items, kThreads), cap = (int64_t)sm_count() * 8;
    const int key_grid = (int)(key_blocks < cap ? key_blocks : cap);
    if (k.idx_bytes == 8)
      HB_LAUNCH(token_keys_kernel<int64_t>, key_grid, kThreads, 0, k.st, static_cast<const int64_t*>(k.ids), k.n, k.padding,
                k.num_rows, p.keys, err, z);
    else
      HB_LAUNCH(token_keys_kernel<int32_t>, key_grid, kThreads, 0, k.st, static_cast<const int32_t*>(k.ids), k.n, k.padding,
                k.num_rows, p.keys, err, z);
    if (k.n == 0) return HB_OK;
    rc = runs_build(p.keys, k.n, nullptr, nullptr, 0, bits, nullptr, 0, nullptr, nullptr, k.uniq_ids, nullptr, p.arrived,
                    p.counts, p.runs_ws, p.runs_bytes, &a.runs, k.st);
  }
  if (rc != HB_OK) return rc;
  HB_CUDA(aside.join());
  a.grads = k.grads;
  a.grad_step = (uint32_t)(k.grad_stride * type_bytes(k.grad_type));
  const uint64_t starts = (uint64_t)(uintptr_t)k.grads | (uint64_t)a.grad_step | 16u;
  a.align = (int)(starts & (~starts + 1));
  a.cols = (uint32_t)k.dim;
  a.blocks = p.blocks;
  a.tiles = p.tiles;
  a.lanes = p.lanes;
  a.per = p.per;
  a.pieces = p.pieces;
  a.parts = p.parts;
  a.arrived = p.arrived;
  a.out = out_rows(k, a.drop);
  a.num_rows = k.num_rows;
  a.by_run = k.by_run;
  a.num_unique = k.num_unique;
  const bool wide = a.align == 16 && whole_blocks(k.out, k.out_stride, k.out_type, k.dim);
  const int64_t warps = ceil_div(p.pieces, 32 / p.lanes) * p.tiles, sum_grid = ceil_div(warps, kSumWarps);
  HB_CHECK_ARG(sum_grid < ((int64_t)1 << 31), "%s: more blocks than a launch holds", k.who);
  return with_type(k.grad_type, [&](auto tg) {
    return with_type(k.out_type, [&](auto to) -> int {
      using TG = decltype(tg);
      using TO = decltype(to);
      const size_t added = k.accumulate ? (size_t)kSumWarps * kStages * added_bytes<TO>() : 0;
      if (wide) HB_LAUNCH_NEXT((grad_sum_kernel<TG, TO, true>), (int)sum_grid, kSumWarps * 32, added, k.st, a);
      else HB_LAUNCH_NEXT((grad_sum_kernel<TG, TO, false>), (int)sum_grid, kSumWarps * 32, 0, k.st, a);
      return HB_OK;
    });
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
  const GradCall k{"hb_embedding_grad", ids, idx_bytes, n, padding_idx, grads, grad_type, grad_stride, dim, scale, drop,
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
  const GradCall k{"hb_embedding_grad_rows", ids, idx_bytes, n, padding_idx, grads, grad_type, grad_stride, dim, scale, drop,
               num_rows, rows, HB_TYPE_F32, dim, true, false, uniq_ids, num_unique, workspace, workspace_bytes,
               (cudaStream_t)stream};
  const int rc = check_call(k);
  if (rc != HB_OK) return rc;
  HB_CHECK_ARG(num_unique && (n == 0 || (uniq_ids && rows)), "hb_embedding_grad_rows: null output");
  return grad(k);
}

}  // extern "C"
