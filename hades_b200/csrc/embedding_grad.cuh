// What the forms of the embedding gradient share: the call, and a finished row on its way out.
#pragma once

#include "droprows.cuh"

namespace hb {

// hb_embedding_grad and hb_embedding_grad_rows, checked
struct GradCall {
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
  bool by_run, accumulate;  // by_run: rows of the output are distinct tokens
  int64_t *uniq_ids, *num_unique;
  void* ws;
  size_t ws_bytes;
  cudaStream_t st;

  bool zeros() const { return !by_run && !accumulate && num_rows > 0; }  // rows of other tokens are written
};

// Few tokens, in one launch (embedding_grad_few.cu).
bool grad_few_takes(const GradCall& k, bool dropout);
int grad_few(const GradCall& k, const Dropout& drop, int* err);

// Runs of the tokens in one launch (tokenruns.cu), up to kSortClusterMax of them; bits: num_rows < 2^bits.
int token_runs(const GradCall& k, int bits, unsigned* zero, int64_t zero_words, void* workspace, hb_runs_t* out);

struct OutRows {
  void* p;
  int64_t stride;
  int width;        // access_bytes
  uint32_t cols;
  bool accumulate;  // add to what is there
  float factor;
};
static inline OutRows out_rows(const GradCall& k, const Dropout& drop) {
  return {k.out, k.out_stride, access_bytes(k.out, k.out_stride, k.out_type, k.dim), (uint32_t)k.dim, k.accumulate, drop.factor};
}

#ifdef __CUDACC__

// A block of a finished sum, from column c on, times the factor, rounded once, to p.  WHOLE: its blocks can be moved at once.
// there: what is added to, where the caller has loaded it.
template <typename TO, bool WHOLE>
__device__ __forceinline__ void put_block(const OutRows& o, TO* p, uint32_t c, float (&x)[kBlockCols],
                                          const Words<block_words<TO>()>* there = nullptr) {
  Words<block_words<TO>()> w;
  if (o.accumulate) {
    float y[kBlockCols];
    if (there) w = *there;
    else if constexpr (WHOLE) load_block(p, w);
    else load_words(p, o.width, o.cols - c, w);
    values_of<TO>(w, y);
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) x[i] = fmaf(x[i], o.factor, y[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i) x[i] *= o.factor;
  }
  words_of<TO>(x, w);
  if constexpr (WHOLE) store_block(p, w);
  else store_words(p, o.width, o.cols - c, w);
}

#endif  // __CUDACC__

}  // namespace hb
