// The finish of a sort of ids that leaves the runs of equal ids (hb_runs_t): the batch's ids (runs.cu) and the tokens of a
// language model's embedding (tokenruns.cu).
#pragma once

#include <type_traits>

#include "runs.cuh"
#include "sortcore.cuh"

namespace hb {

// what stands for an entry without a valid id: above every other
static int64_t runs_sentinel(int id_bits) { return id_bits >= 63 ? INT64_MAX : (((int64_t)1 << id_bits) - 1); }

#ifdef __CUDACC__

// Runs of equal ids in the sorted order, numbered over all runs and inside the class of their id.  RESOLVE: each
// is looked up where it is written.
template <bool RESOLVE>
struct RunsFinish {
  static constexpr bool kOneEach = RESOLVE;
  const int8_t* table;   // nullable: no classes
  int64_t table_len;
  uint32_t* perm;        // [n]
  uint8_t* head;
  int64_t* uniq;
  int64_t* uniq2;        // nullable second copy (the caller's buffer)
  int64_t* run_start;
  int8_t* dclass;
  int32_t* dpos;
  int64_t* out_ids[3];
  int64_t* num_runs;
  int64_t* num_runs2;    // nullable second copy
  int64_t* class_counts;
  int64_t* class_counts2;
  int32_t* base8;        // [ceil(n / 8)] runs that start before entry 8k
  int64_t* n_valid;      // number of valid entries (read where the input is segmented or large)
  unsigned* zero;        // nullable: words that `resolve` or the next launch needs at zero
  int zero_words;
  struct Nothing {};
  std::conditional_t<RESOLVE, RunsResolve, Nothing> resolve;

  // No runs and no entries: what works on the runs has nothing to do.  The sums go by the entries and do not
  // wait for a device count where the caller has none: they find one run of all entries and no id.
  template <class Ctx, class Src>
  __device__ __forceinline__ void give_up(Ctx& ctx, const Src& src) const {
    for (int k = threadIdx.x; k < zero_words; k += Ctx::kThreads) zero[k] = 0u;
    for (uint32_t j = ctx.chunk_begin() + threadIdx.x; j < ctx.chunk_end(); j += Ctx::kThreads) {
      perm[j] = j;
      head[j] = j == 0;
      if ((j & 7u) == 0u) base8[j >> 3] = j != 0;
    }
    if (threadIdx.x != 0) return;  // (every CTA writes the same)
    *num_runs = *n_valid = run_start[0] = 0;
    run_start[1] = ctx.count;
    uniq[0] = src.sentinel;
    if (uniq2) uniq2[0] = -1;  // (no id is: entries that all take no part leave the sentinel there)
    if (table) {
      dclass[0] = -1;
      dpos[0] = 0;
    }
    if (num_runs2) *num_runs2 = 0;
    for (int c = 0; c < 4; ++c) class_counts[c] = 0;
    for (int c = 0; class_counts2 && c < 3; ++c) class_counts2[c] = 0;
  }

  template <class Ctx, class Src>
  __device__ __forceinline__ void run(Ctx& ctx, const Src& src) const {
    constexpr int T = Ctx::kThreads, W = T / 32;
    __shared__ int4 s_sum[2 * W + 1];
    __shared__ unsigned long long s_valid;
    const int lane = threadIdx.x & 31;
    for (int k = ctx.rank * T + threadIdx.x; k < zero_words; k += ctx.ctas * T) zero[k] = 0u;
    int ne = ctx.count;
    if (src.seg_counts) {
      // valid entries are scattered over the segments; their number becomes the device count
      if (threadIdx.x == 0) s_valid = 0ull;
      __syncthreads();
      unsigned long long t = 0;
      for (int64_t k = threadIdx.x; k < src.n / src.seg_cap; k += T) {
        const int64_t c = src.seg_counts[k];
        t += (unsigned long long)(c < 0 ? 0 : (c > (int64_t)src.seg_cap ? (int64_t)src.seg_cap : c));
      }
      if (t) atomicAdd(&s_valid, t);
      __syncthreads();
      ne = (int)s_valid;
    }
    const uint32_t begin = ctx.chunk_begin(), end = ctx.chunk_end();
    // id of an entry of the narrow kind (entries that sort last: the sentinel)
    auto narrow_id = [&](uint32_t key) -> int64_t {
      return key == kSortNone && ctx.none ? src.sentinel : (int64_t)key;
    };
    auto wide_id = [&](uint32_t pos) -> int64_t {
      unsigned long long key;
      return sort_load(src, pos, key) ? (int64_t)key : src.sentinel;
    };
    // A thread takes 8 consecutive entries (whole vectors of positions and head flags to
    // write, one entry of base8, no votes), the CTA 8 * T in a strip.
    uint32_t at[8];      // their positions
    uint32_t code = 0u;  // per entry 3 bits: 4 | class (3: none) where a run starts, else 0
    auto classify = [&](uint32_t j0) -> int4 {
      int4 c = make_int4(0, 0, 0, 0);
      code = 0u;
      uint2 e[8];
      e[7] = make_uint2(0u, 0u);
      if (j0 < end) ctx.get8(j0, e);
      uint32_t before = __shfl_up_sync(0xffffffffu, e[7].x, 1);
      if (j0 >= end) return c;
      if (lane == 0 && j0 > 0) before = ctx.get(j0 - 1).x;
      unsigned heads = 0u;
      if (!ctx.wide) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          heads |= (unsigned)(j0 + x < (uint32_t)ne && (j0 + x == 0 || e[x].x != before)) << x;
          before = e[x].x;
        }
      } else {
        int64_t was = j0 > 0 ? wide_id(ctx.get(j0 - 1).y) : -1;
#pragma unroll 1
        for (int x = 0; x < 8 && j0 + x < end; ++x) {
          const int64_t id = wide_id(ctx.get(j0 + x).y);
          heads |= (unsigned)(j0 + x < (uint32_t)ne && id != was) << x;
          was = id;
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) at[x] = e[x].y;
      if (!table) {
#pragma unroll
        for (int x = 0; x < 8; ++x) code |= ((heads >> x) & 1u) << (3 * x + 2);
        c.x = __popc(heads);
        return c;
      }
      int8_t cls[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        cls[x] = 3;
        if ((heads >> x) & 1u) {
          const int64_t id = ctx.wide ? wide_id(e[x].y) : narrow_id(e[x].x);
          if (id < table_len) cls[x] = Ctx::kBehindAll ? load_settled(table + id) : table[id];
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if (!((heads >> x) & 1u)) continue;
        const int k = cls[x] >= 0 && cls[x] <= 2 ? cls[x] : 3;
        code |= (4u | k) << (3 * x);
        c.x += k == 0;
        c.y += k == 1;
        c.z += k == 2;
        c.w += k == 3;
      }
      return c;
    };
    auto put_entries = [&](uint32_t j0) {
      if (j0 >= end) return;
      if (j0 + 8 <= end) {
        uint4* p = reinterpret_cast<uint4*>(perm + j0);
        p[0] = make_uint4(at[0], at[1], at[2], at[3]);
        p[1] = make_uint4(at[4], at[5], at[6], at[7]);
      } else {
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (j0 + x < end) perm[j0 + x] = at[x];
      }
      // one byte per entry (the allocation holds whole groups of 8)
      auto flag = [&](int x) -> uint32_t { return (code >> (3 * x + 2)) & 1u; };
      const uint32_t lo = flag(0) | (flag(1) << 8) | (flag(2) << 16) | (flag(3) << 24);
      const uint32_t hi = flag(4) | (flag(5) << 8) | (flag(6) << 16) | (flag(7) << 24);
      *reinterpret_cast<uint2*>(head + j0) = make_uint2(lo, hi);
    };
    // a thread's counts -> those of the threads ahead in its warp and of the whole warp
    auto scan_warp = [&](const int4& c, int4& total) -> int4 {
      const unsigned long long v = (unsigned long long)(uint32_t)(c.x | (c.y << 16)) | ((unsigned long long)(uint32_t)(c.z | (c.w << 16)) << 32);
      unsigned long long inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const unsigned long long t = __shfl_sync(0xffffffffu, inc, 31);
      total = make_int4((int)(t & 0xffff), (int)((t >> 16) & 0xffff), (int)((t >> 32) & 0xffff), (int)(t >> 48));
      inc -= v;
      return make_int4((int)(inc & 0xffff), (int)((inc >> 16) & 0xffff), (int)((inc >> 32) & 0xffff), (int)(inc >> 48));
    };
    uint32_t kept = 0u;  // the codes of the first of two strips
    // (stores ahead of the barrier are what it waits for; that a kernel has them behind it, and then one strip, is known
    // when it is compiled: 512 ids with their classes 10.8 -> 10.3 us, 8,192 17.3 -> 16.8)
    constexpr bool late = Ctx::kStoresLate;
    const int strips = late ? (int)(end > begin) : (int)((end - begin + 8 * T - 1) / (8 * T));
    int4 mine = make_int4(0, 0, 0, 0), lanes = mine, warps, cta, ahead, all;
#pragma unroll 1
    for (int q = 0; q < strips; ++q) {
      const uint32_t j0 = begin + q * (8 * T) + threadIdx.x * 8;
      const int4 c = classify(j0);
      if (!late) put_entries(j0);
      int4 total;
      lanes = scan_warp(c, total);
      mine.x += total.x; mine.y += total.y; mine.z += total.z; mine.w += total.w;
      if (q == 0) kept = code;
    }
    sort_warp_sums<W>(mine, s_sum, warps, cta);
    if (!ctx.prefix(cta, ahead, all)) return give_up(ctx, src);
    if (late) put_entries(begin + threadIdx.x * 8);
#pragma unroll 1
    for (int q = 0; q < strips; ++q) {
      const uint32_t strip = begin + q * (8 * T);
      const uint32_t j0 = strip + threadIdx.x * 8;
      if (strips > 1) {
        int4 total, c = make_int4(0, 0, 0, 0);
        if (strips > 2) {
          c = classify(j0);
        } else {
          const uint32_t last = code;  // strip 1 was classified last: its codes stay for the next turn
          if (q == 0) code = kept;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const uint32_t v = (code >> (3 * x)) & 7u;
            c.x += v == 4u;
            c.y += v == 5u;
            c.z += v == 6u;
            c.w += v == 7u;
          }
          if (q == 0) kept = last;
        }
        lanes = scan_warp(c, total);
        __syncthreads();
        sort_warp_sums<W>(total, s_sum, warps, cta);
      }
      // The runs of the strip as a list in shared memory, so that what is written per run leaves in
      // whole sectors: 13 bits place in the strip, 2 class, 14 number inside the class and strip.
      int4 run = make_int4(warps.x + lanes.x, warps.y + lanes.y, warps.z + lanes.z, warps.w + lanes.w);
      const int before = ahead.x + ahead.y + ahead.z + ahead.w;
      if (j0 < end) base8[j0 >> 3] = before + run.x + run.y + run.z + run.w;
      if (code) {
        int at = run.x + run.y + run.z + run.w;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t c = (code >> (3 * x)) & 7u;
          if (!c) continue;
          const uint32_t k = c & 3u;
          const int pos = k == 0 ? run.x : (k == 1 ? run.y : (k == 2 ? run.z : run.w));
          ctx.scratch[at++] = (threadIdx.x * 8 + x) | (k << 13) | ((uint32_t)pos << 15);
          run.x += k == 0;
          run.y += k == 1;
          run.z += k == 2;
          run.w += k == 3;
        }
      }
      __syncthreads();
      const int runs = cta.x + cta.y + cta.z + cta.w;
      auto put = [&](int r, int64_t& id, bool& cold) {
        const uint32_t w = ctx.scratch[r];
        const uint32_t j = strip + (w & 8191u);
        const uint2 e = ctx.get(j);
        id = ctx.wide ? wide_id(e.y) : narrow_id(e.x);
        const int u = before + r;
        uniq[u] = id;
        if (uniq2) uniq2[u] = id;
        run_start[u] = j;
        if (table) {
          const int k = (int)(w >> 13) & 3;
          const int pos = (int)(w >> 15) + (k == 0 ? ahead.x : (k == 1 ? ahead.y : (k == 2 ? ahead.z : ahead.w)));
          dclass[u] = k < 3 ? (int8_t)k : (int8_t)-1;
          dpos[u] = pos;
          int64_t* to = k == 0 ? out_ids[0] : (k == 1 ? out_ids[1] : (k == 2 ? out_ids[2] : nullptr));
          if (to) to[pos] = id;
          cold = k == 2;
        }
      };
      if constexpr (RESOLVE) {
#pragma unroll 1
        for (int r = threadIdx.x; r - lane < runs; r += T) {  // whole warps
          int64_t id = -1;
          bool cold = false;
          if (r < runs) put(r, id, cold);
          resolve_run(resolve, before + r, r < runs, id, cold);
        }
      } else {
#pragma unroll 2
        for (int r = threadIdx.x; r < runs; r += T) {
          int64_t id;
          bool cold;
          put(r, id, cold);
        }
      }
      if (strips > 1) __syncthreads();
      if (strips == 2) code = kept;
      ahead.x += cta.x; ahead.y += cta.y; ahead.z += cta.z; ahead.w += cta.w;
    }
    if (ctx.rank == 0 && threadIdx.x == 0) {
      const int64_t u = (int64_t)all.x + all.y + all.z + all.w;
      *num_runs = u;
      if (num_runs2) *num_runs2 = u;
      run_start[u] = ne;
      *n_valid = ne;
      class_counts[0] = all.x; class_counts[1] = all.y; class_counts[2] = all.z; class_counts[3] = all.w;
      if (class_counts2) { class_counts2[0] = all.x; class_counts2[1] = all.y; class_counts2[2] = all.z; }
    }
  }
};

#endif  // __CUDACC__

}  // namespace hb
