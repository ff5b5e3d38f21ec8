// The embedding gradient of few tokens in one launch.
//
// Every CTA sorts all tokens for itself (bitonic, of words of token and position, so that nothing compares equal; in
// registers, by shuffles, between warps through shared memory), and has its share of the distinct tokens, of the long ones
// among them with all of its warps, and of the rows that no token points to.  No CTA waits for another.  Bound by latency:
// the chain ids, sort, rows of the gradient, output (us, 512 / 2,048 tokens: ids 1.4 / 2.3, sort 1.4 / 2.9, runs 0.9 / 1.4, rows
// and zeros 6 / 11); and by code that runs once and is fetched as it runs, so that long and short tokens share it.
#include <climits>

#include "embedding_grad.cuh"

namespace hb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMost = 2048;    // (us, 1,024 bf16 columns into 8,000 rows: 17.0, in the other form 21.1)
// Positions of a token that a CTA adds up together, as the longest one that a warp has is what the others wait for (us, 8 / 16 /
// 32: 512 x 256 fp32 10.3 / 10.3 / 11.6, 2,048 x 1,024 bf16 19.0 / 17.0 / 16.9, 2,048 x 4,096 32.4 / 21.9 / 24.1).
constexpr int kLong = 16;
constexpr int kRows = 4096;    // of the output, whose zeros a CTA writes at a time

struct FewArgs {
  const void* ids;
  int idx_bytes;
  int n;
  int64_t padding;
  const void* grads;
  int64_t grad_stride;
  int grad_width;
  uint32_t cols, blocks, tiles;
  int lanes, per;             // of a unit; sorted entries of a piece
  Dropout drop;
  OutRows out;
  uint32_t num_rows;          // token and position fit in a word
  bool by_run, zeros, linear; // linear: a row of the output begins where the one before ends
  Divisor row_bytes;          // of the output
  Divisor zero_pieces;        // of zero_width bytes, of a row
  int zero_width;
  int64_t stride_bytes;
  int64_t *uniq_ids, *num_unique;  // nullable
  int* err;
};

// The word of entry threadIdx.x * E + r of kThreads * E, sorted.
template <int E>
__device__ __forceinline__ void sort_words(uint32_t (&w)[E], uint32_t* s_words) {
  const int t = threadIdx.x;
  auto keep = [](uint32_t mine, uint32_t other, bool low) { return low ? min(mine, other) : max(mine, other); };
#pragma unroll
  for (int k = 2; k <= kThreads * E; k *= 2) {
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      if (j >= 32 * E) {
        __syncthreads();
#pragma unroll
        for (int r = 0; r < E; ++r) s_words[r * kThreads + t] = w[r];
        __syncthreads();
        const bool low = ((t * E & k) == 0) == ((t * E & j) == 0);
#pragma unroll
        for (int r = 0; r < E; ++r) w[r] = keep(w[r], s_words[r * kThreads + (t ^ (j / E))], low);
      } else if (j >= E) {
        const bool low = ((t * E & k) == 0) == ((t * E & j) == 0);
#pragma unroll
        for (int r = 0; r < E; ++r) w[r] = keep(w[r], __shfl_xor_sync(0xffffffffu, w[r], j / E), low);
      } else {
#pragma unroll
        for (int r = 0; r < E; ++r)
          if ((r & j) == 0) {
            const bool up = ((t * E + r) & k) == 0;
            const uint32_t lo = min(w[r], w[r | j]), hi = max(w[r], w[r | j]);
            w[r] = up ? lo : hi;
            w[r | j] = up ? hi : lo;
          }
      }
    }
  }
  __syncthreads();
}

// WHOLE: blocks of the gradients and of the output can be moved at once.
template <typename TG, typename TO, int E, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 1) grad_few_kernel(const FewArgs a) {
  constexpr int kSize = kThreads * E, kBits = E == 1 ? 9 : E == 2 ? 10 : 11;
  __shared__ uint32_t s_words[kSize + 1];             // token and position, sorted
  __shared__ uint16_t s_run[kSize], s_start[kSize + 1], s_found[kSize / kLong], s_long[kSize / kLong];
  __shared__ int s_warp[kWarps], s_longs, s_ticket;
  __shared__ float s_sum[kWarps][32][kBlockCols + 1];
  __shared__ uint32_t s_there[kRows / 32];            // rows of the output, from v0 on, that a token points to
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  uint32_t word[E];
#pragma unroll
  for (int r = 0; r < E; ++r) {
    const int i = r * kThreads + t;
    word[r] = 0xffffffffu;
    if (i < a.n) {
      const int64_t id = a.idx_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
      const bool inside = id >= 0 && id < a.num_rows;
      if (!inside && id != a.padding && blockIdx.x == 0) atomicExch(a.err, HB_ERR_INVALID);
      word[r] = (inside && id != a.padding ? (uint32_t)id : a.num_rows) << kBits | (uint32_t)i;
    }
  }
  if (t == 0) s_longs = 0;
  for (int i = t; i < kRows / 32; i += kThreads) s_there[i] = 0u;
  sort_words<E>(word, s_words);
  // runs of equal tokens; what takes no part lies last and is none
#pragma unroll
  for (int r = 0; r < E; ++r) s_words[t * E + r] = word[r];
  __syncthreads();
  int heads = 0, parts = 0;
  uint32_t token_before = t == 0 ? 0xffffffffu : s_words[t * E - 1] >> kBits;
#pragma unroll
  for (int r = 0; r < E; ++r) {
    const uint32_t token = word[r] >> kBits;
    const bool part = token < a.num_rows;
    parts += part;
    if (part && token != token_before) heads |= 1 << r;
    token_before = token;
  }
  const int own = __popc(heads);
  int ahead = own | parts << 16;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, ahead, d);
    if (lane >= d) ahead += other;
  }
  if (lane == 31) s_warp[warp] = ahead;
  __syncthreads();
  int total = 0, at = (ahead & 0xffff) - own;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) at += s_warp[w] & 0xffff;
    total += s_warp[w];
  }
  const int runs = total & 0xffff, valid = total >> 16;
  // the CTA's rows whose zeros it writes
  const int64_t row_share = ((int64_t)a.num_rows + gridDim.x - 1) / gridDim.x;
  const int64_t row_begin = blockIdx.x * row_share;
  const int64_t row_end = row_begin + row_share < a.num_rows ? row_begin + row_share : a.num_rows;
  auto note = [&](uint32_t token, int64_t v0) {
    const int64_t v = (int64_t)token - v0;
    if (v >= 0 && v < kRows) atomicOr(&s_there[v >> 5], 1u << (v & 31));
  };
#pragma unroll
  for (int r = 0; r < E; ++r) {
    if (heads >> r & 1) {
      s_start[at++] = (uint16_t)(t * E + r);
      if (a.uniq_ids && blockIdx.x == 0) a.uniq_ids[at - 1] = word[r] >> kBits;
      if (a.zeros) note(word[r] >> kBits, row_begin);
    }
    s_run[t * E + r] = (uint16_t)(at - 1);
  }
  if (t == 0) {
    s_start[runs] = (uint16_t)valid;
    s_ticket = 0;
    if (a.num_unique && blockIdx.x == 0) {
      *a.num_unique = runs;
      if (runs == 0) a.uniq_ids[0] = a.num_rows;  // (as after the sort of more tokens; -1 there: it gave up)
    }
  }
  __syncthreads();
  for (int r = t; r < runs; r += kThreads)
    if (s_start[r + 1] - s_start[r] >= kLong) s_found[atomicAdd(&s_longs, 1)] = (uint16_t)r;
  __syncthreads();
  const int longs = s_longs;
  if (longs) {
    if (t < longs) {  // in one order for all CTAs
      int before = 0;
      for (int o = 0; o < longs; ++o) before += s_found[o] < s_found[t];
      s_long[before] = s_found[t];
    }
    __syncthreads();
  }

  PhiloxKey key = {};
  if (a.drop.drop_below) key = philox_key(a.drop);
  constexpr int kFly = sizeof(TG) == 4 || !WHOLE ? 4 : 8;  // rows on their way at once
  const int units = 32 / a.lanes, l = t & (a.lanes - 1), group = t / a.lanes, groups = kThreads / a.lanes;
  auto row_out = [&](int run) {
    return static_cast<TO*>(a.out.p) + (a.by_run ? (int64_t)run : (int64_t)(s_words[s_start[run]] >> kBits)) * a.out.stride;
  };
  // the last CTAs, at most a third, have the long tokens, the others the short ones
  const int long_jobs = longs * (int)a.tiles, third = ((int)gridDim.x + 2) / 3;
  const int long_ctas = long_jobs < third ? long_jobs : third, short_ctas = gridDim.x == 1 ? 1 : (int)gridDim.x - long_ctas;
  int job = (int)gridDim.x - 1 - (int)blockIdx.x;
  bool is_long = job < long_ctas;
  const int short_job = (int)blockIdx.x < short_ctas ? (int)blockIdx.x * groups + group : INT_MAX;
  if (!is_long) job = short_job;
  const int short_jobs = (valid + a.per - 1) / a.per * (int)a.tiles;
  for (;;) {
    // a long token's share of a group of lanes, or the short tokens that begin in the piece of a unit
    uint32_t block;
    int run, last, e = 0, end = 0;
    if (is_long) {
      run = last = s_long[job / (int)a.tiles];
      block = (uint32_t)(job % (int)a.tiles) * a.lanes + l;
      const int from = s_start[run], to = s_start[run + 1], share = (to - from + groups - 1) / groups;
      e = from + group * share;
      end = e + share < to ? e + share : to;
      if (e >= end) last = -1;
    } else {
      if (job >= short_jobs) break;
      const int first = job / (int)a.tiles * a.per;
      block = (uint32_t)(job % (int)a.tiles) * a.lanes + l;
      run = first == 0 ? 0 : s_run[first - 1] + 1;
      last = s_run[(first + a.per < valid ? first + a.per : valid) - 1];
    }
    if (block >= a.blocks) last = -1;
    auto settle = [&] {  // at the first entry of the run, or of the next one that is short
      for (; run <= last; ++run) {
        e = s_start[run];
        end = s_start[run + 1];
        if (end - e < kLong) return;
      }
    };
    if (!is_long) settle();
    const uint32_t c = block * kBlockCols;
    float sum[kBlockCols];
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
    while (run <= last) {
      int entry[kFly], of[kFly];  // of: its run where it is the last entry of one, else -1
      Words<block_words<TG>()> in[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        entry[k] = of[k] = -1;
        if (run <= last) {
          entry[k] = (int)(s_words[e++] & (kSize - 1));
          if (e == end) {
            if (!is_long) of[k] = run;
            ++run;
            if (!is_long) settle();
          }
          const TG* p = static_cast<const TG*>(a.grads) + (int64_t)entry[k] * a.grad_stride + c;
          if constexpr (WHOLE) load_block(p, in[k]);
          else load_words(p, a.grad_width, a.cols - c, in[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        if (entry[k] < 0) break;
        if (a.drop.drop_below) add_kept<TG>(sum, in[k], draws_of(key, block, entry[k]), a.drop.drop_below);
        else add_block<TG>(sum, in[k]);
        if (of[k] < 0) continue;
        put_block<TO, WHOLE>(a.out, row_out(of[k]) + c, c, sum);
#pragma unroll
        for (int i = 0; i < kBlockCols; ++i) sum[i] = 0.0f;
      }
    }
    if (!is_long) {
      job += short_ctas * groups;
      continue;
    }
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) s_sum[warp][lane][i] = sum[i];
    __syncthreads();
    const int the = s_long[job / (int)a.tiles];
    if (group == 0 && block < a.blocks) {
      const int length = s_start[the + 1] - s_start[the], share = (length + groups - 1) / groups;
      for (int g = 1; g * share < length; ++g) {
        const int other = g * a.lanes + l;
#pragma unroll
        for (int i = 0; i < kBlockCols; ++i) sum[i] += s_sum[other >> 5][other & 31][i];
      }
      put_block<TO, WHOLE>(a.out, row_out(the) + c, c, sum);
    }
    __syncthreads();
    job += long_ctas;
    is_long = job < long_jobs;
    if (!is_long) job = short_job;
  }
  if (!a.zeros) return;
  // zeros to the rows that no token points to, kRows at a time, a stretch at a time to the warp that comes for it
  for (int64_t v0 = row_begin; v0 < row_end; v0 += kRows) {
    if (v0 != row_begin) {
      __syncthreads();
      for (int i = t; i < kRows / 32; i += kThreads) s_there[i] = 0u;
      if (t == 0) s_ticket = 0;
      __syncthreads();
      for (int r = t; r < runs; r += kThreads) note(s_words[s_start[r]] >> kBits, v0);
      __syncthreads();
    }
    const int rows = (int)(row_end - v0 < kRows ? row_end - v0 : kRows);
    char* base = static_cast<char*>(a.out.p) + v0 * a.stride_bytes;
    // rows that follow one another are a stretch of memory, and its pieces of 32 bytes may lie in two rows or more
    const uint32_t skew = a.linear ? (uint32_t)((uintptr_t)base & 31u) : 0u, size = (uint32_t)rows * a.row_bytes.by;
    const uint32_t items = a.linear ? (size + skew + 31u) / 32u : (uint32_t)rows * a.zero_pieces.by;
    auto there = [&](uint32_t v) { return (s_there[v >> 5] >> (v & 31) & 1u) != 0u; };
    for (;;) {
      constexpr uint32_t kStretch = 256;
      uint32_t i0 = lane == 0 ? (uint32_t)atomicAdd(&s_ticket, 1) * kStretch : 0u;
      i0 = __shfl_sync(0xffffffffu, i0, 0);
      if (i0 >= items) break;
      if (a.linear) {
        for (uint32_t i = i0 + lane; i < i0 + kStretch && i < items; i += 32) {
          const int from = (int)(i * 32u) - (int)skew, first = from < 0 ? 0 : from;
          const int last = from + 31 < (int)size ? from + 31 : (int)size - 1;
          const uint32_t v = divide(first, a.row_bytes), w = divide(last, a.row_bytes);
          const bool none = !there(v) && !there(w);
          if (v + 1 >= w && none && last - first == 31) {
            store_block(base + from, Words<8>{});
          } else if (v + 1 < w || !there(v) || !there(w)) {
            for (int b = first; b <= last; b += (int)sizeof(TO))
              if (!there(divide(b, a.row_bytes))) *reinterpret_cast<std::conditional_t<sizeof(TO) == 4, uint32_t, uint16_t>*>(base + b) = 0;
          }
        }
        continue;
      }
#pragma unroll 4
      for (uint32_t i = i0 + lane; i < i0 + kStretch; i += 32) {
        if (i >= items) break;
        const uint32_t v = divide(i, a.zero_pieces);
        if (there(v)) continue;
        char* p = base + v * a.stride_bytes + (i - v * a.zero_pieces.by) * a.zero_width;
        if (a.zero_width == 16) *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
        else if (a.zero_width == 8) *reinterpret_cast<uint2*>(p) = make_uint2(0u, 0u);
        else if (a.zero_width == 4) *reinterpret_cast<uint32_t*>(p) = 0u;
        else *reinterpret_cast<uint16_t*>(p) = 0;
      }
    }
  }
}

int entries_each(const GradCall& k) { return k.n <= kThreads ? 1 : k.n <= 2 * kThreads ? 2 : 4; }
// Bytes of zeros at a time, as all rows at a distance allow.
int zero_width(const GradCall& k) {
  const int64_t e = type_bytes(k.out_type);
  const uint64_t bits = (uint64_t)(uintptr_t)k.out | (uint64_t)(k.dim * e) | (uint64_t)(k.out_stride * e) | 16u;
  return (int)(bits & (~bits + 1));
}

bool whole_rows(const GradCall& k) {
  return whole_blocks(k.grads, k.grad_stride, k.grad_type, k.dim) && whole_blocks(k.out, k.out_stride, k.out_type, k.dim);
}

}  // namespace

// Where the launches that this form spares weigh more than the sums, which the other form's ring of copies feeds better, and
// than the zeros, which it writes beside its sort (us, this form and the other; 2,048 tokens, bf16: 4,096 columns 23.2 and
// 27.3, 6,144 26.6 and 27.0, 8,192 31.5 and 26.0; with dropout 2,048 19.9 and 23.4, 4,096 27.8 and 25.3; ragged 1,001 20.9 and
// 23.2, 2,001 26.0 and 24.4, 500 tokens of 8,001 25.3 and 21.7; 1,024 of 4,096 into 131 MB 36.2 and 37.1, 262 MB 54.8 and
// 55.0, 1.07 GB 181 and 161).  What is held to fit: token and position a word, bytes of kRows rows of zeros 31 bits.
bool grad_few_takes(const GradCall& k, bool dropout) {
  const int64_t row_bytes = k.dim * type_bytes(k.out_type);
  if (k.n <= 0 || k.n > kMost || k.num_rows >= ((int64_t)1 << 32) / (kThreads * entries_each(k)) - 1) return false;
  if (k.n * k.dim * (whole_rows(k) ? 1 : 3) * (dropout ? 2 : 1) > (8 << 20)) return false;
  return !k.zeros() || (row_bytes < (1 << 19) && k.num_rows * row_bytes <= (192 << 20));
}

int grad_few(const GradCall& k, const Dropout& drop, int* err) {
  FewArgs f = {};
  f.ids = k.ids;
  f.idx_bytes = k.idx_bytes;
  f.n = (int)k.n;
  f.padding = k.padding;
  f.grads = k.grads;
  f.grad_stride = k.grad_stride;
  f.grad_width = access_bytes(k.grads, k.grad_stride, k.grad_type, k.dim);
  f.cols = (uint32_t)k.dim;
  f.blocks = (uint32_t)ceil_div(k.dim, kBlockCols);
  f.lanes = 1;
  while (f.lanes < 32 && f.lanes < (int)f.blocks) f.lanes *= 2;
  f.tiles = (uint32_t)ceil_div(f.blocks, f.lanes);
  f.drop = drop;
  f.out = out_rows(k, drop);
  f.num_rows = (uint32_t)k.num_rows;
  f.by_run = k.by_run;
  f.zeros = k.zeros();
  f.uniq_ids = k.uniq_ids;
  f.num_unique = k.num_unique;
  f.err = err;
  const int64_t units = kWarps * (32 / f.lanes), row_bytes = k.dim * type_bytes(k.out_type);
  f.per = (int)ceil_div(k.n * f.tiles, sm_count() * units);
  int64_t grid = 2 * ceil_div(ceil_div(k.n, f.per) * f.tiles, units);  // (room for the long tokens)
  if (f.zeros) {
    f.stride_bytes = k.out_stride * type_bytes(k.out_type);
    f.zero_width = zero_width(k);
    f.zero_pieces = divisor((uint32_t)(row_bytes / f.zero_width));
    f.row_bytes = divisor((uint32_t)row_bytes);
    f.linear = k.num_rows == 1 || k.out_stride == k.dim;
    if (ceil_div(k.num_rows * row_bytes, 8192) > grid) grid = ceil_div(k.num_rows * row_bytes, 8192);
  }
  if (grid > sm_count()) grid = sm_count();
  const bool whole = whole_rows(k);
  return with_type(k.grad_type, [&](auto tg) {
    return with_type(k.out_type, [&](auto to) -> int {
      using TG = decltype(tg);
      using TO = decltype(to);
      auto launch = [&](auto each) -> int {
        constexpr int E = decltype(each)::value;
        if (whole) HB_LAUNCH((grad_few_kernel<TG, TO, E, true>), (int)grid, kThreads, 0, k.st, f);
        else HB_LAUNCH((grad_few_kernel<TG, TO, E, false>), (int)grid, kThreads, 0, k.st, f);
        return HB_OK;
      };
      const int each = entries_each(k);
      if (each == 1) return launch(std::integral_constant<int, 1>{});
      return each == 2 ? launch(std::integral_constant<int, 2>{}) : launch(std::integral_constant<int, 4>{});
    });
  });
}

}  // namespace hb
