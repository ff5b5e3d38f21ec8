// Runs of equal tokens of a batch of up to kSortClusterMax positions: hb_runs_build's sort straight from the tokens as a
// caller has them (32 or 64 bits, padding and ids outside of the table among them), without a launch that makes ids of them.
#include <cstring>

#include "embedding_grad.cuh"
#include "runsfinish.cuh"

namespace hb {
int* device_error_word();  // runtime.cu

namespace {

struct TokenSource {
  static constexpr bool kSkips = false;
  static constexpr const int64_t* seg_counts = nullptr;  // (no segments)
  static constexpr uint32_t seg_cap = 1;
  const void* ids;
  int idx_bytes;
  int64_t n, padding, num_rows;
  int64_t sentinel;  // at least num_rows
  int* err;
  int bits;
  __host__ __device__ int known_bits() const { return bits; }
  __device__ __forceinline__ int64_t count() const { return n; }
  __device__ __forceinline__ bool fetch(int64_t i, int64_t& id) const {
    id = idx_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
    return true;
  }
  __device__ __forceinline__ bool accept(int64_t id, unsigned long long& key) const {
    if (id == padding) return false;
    if (id < 0 || id >= num_rows) {
      atomicExch(err, HB_ERR_INVALID);
      return false;
    }
    key = (unsigned long long)id;
    return true;
  }
};

}  // namespace

int token_runs(const GradCall& k, int bits, unsigned* zero, int64_t zero_words, void* workspace, hb_runs_t* out) {
  const RunsPlan s = make_runs_plan(workspace, k.n, false);
  memset(out, 0, sizeof(*out));
  out->n = k.n;
  out->perm = s.perm;
  out->num_runs = s.num_runs;
  out->run_start = s.run_start;
  out->head = s.head;
  out->uniq_ids = s.uniq;
  out->base8 = s.base8;
  const TokenSource src{k.ids, k.idx_bytes, k.n, k.padding, k.num_rows, runs_sentinel(bits), device_error_word(), bits};
  RunsFinish<false> fin = {};
  fin.perm = s.perm;
  fin.head = s.head;
  fin.uniq = s.uniq;
  fin.uniq2 = k.uniq_ids;
  fin.run_start = s.run_start;
  fin.num_runs = s.num_runs;
  fin.class_counts = s.class_counts;
  fin.base8 = s.base8;
  fin.n_valid = s.n_valid;
  fin.zero = zero;
  fin.zero_words = (int)zero_words;
  return sort_run_cluster(src, fin, k.n, k.st);
}

}  // namespace hb
