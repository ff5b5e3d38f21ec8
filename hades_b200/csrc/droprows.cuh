// Rows of fp32, fp16 or bf16 values in blocks of eight columns, and the dropout of such rows: what the embedding lookup,
// its gradient and the dropout of rows that exist already share.
//
// Dropout: value (row, column) is kept where the 16 bits that the generator gives its place are at least T; T of 65536
// values are dropped, and what is kept is multiplied by 65536 / (65536 - T).  The generator is Philox4x32 with ten rounds
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): counter (column / 8, row, offset's
// low and high word), key the seed.  A call's 128 bits are the draws of eight neighbouring columns, so that a place needs
// no state and no mask in memory, and forward and backward passes agree whatever kernel or layout they use.  Ten rounds and
// the eight selections are 78 of the 138 instructions that a block of bf16 values takes (65,536 x 4,096: 162 us without, 182
// with dropout, at 62 % of the ALU's and of the wide multipliers' cycles; 195 to 200 where L2 is full of lines that have yet
// to be written); 32 bits a value would need twice the rounds.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "launch.cuh"

namespace hb {

constexpr int kBlockCols = 8;  // columns of a block: a thread's, and a call's of the generator

struct Dropout {
  uint32_t drop_below;  // T; 0: nothing is dropped
  float factor;         // of what is kept: scale * 65536 / (65536 - T), rounded once
  uint64_t seed, offset;
  const int64_t* rng;   // nullable, device: seed and offset as they are when the kernel runs
};

// The checks and the numbers of a call's (scale, dropout); drop nullable.
static inline int dropout_of(const char* who, double scale, const hb_drop_t* drop, Dropout* out) {
  HB_CHECK_ARG(!drop || (drop->p >= 0.0 && drop->p <= 1.0), "%s: the dropout probability must be in [0, 1]", who);
  const double t = drop ? std::floor(drop->p * 65536.0 + 0.5) : 0.0;
  const double f = t < 65536.0 ? scale * 65536.0 / (65536.0 - t) : 0.0;
  HB_CHECK_ARG(!drop || ((uintptr_t)drop->rng & 7) == 0, "%s: seed and offset are not aligned", who);
  HB_CHECK_ARG(std::isfinite(scale) && std::isfinite((float)f), "%s: the scale must be finite", who);
  out->drop_below = (uint32_t)t;
  out->factor = (float)f;
  out->seed = drop ? drop->seed : 0;
  out->offset = drop ? drop->offset : 0;
  out->rng = drop && t > 0.0 ? drop->rng : nullptr;
  return HB_OK;
}

static inline int type_bytes(int type) { return type == HB_TYPE_F32 ? 4 : 2; }
static inline bool type_known(int type) { return type == HB_TYPE_F32 || type == HB_TYPE_F16 || type == HB_TYPE_BF16; }

// Whether what lies at p begins where its values of so many bytes can.
static inline bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// Whether matrices of rows of dim values share memory (as ranges of addresses).
static inline bool overlap(const void* a, int64_t a_stride, int a_type, int64_t a_rows, const void* b, int64_t b_stride,
                           int b_type, int64_t b_rows, int64_t dim) {
  if (a_rows <= 0 || b_rows <= 0) return false;
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  const uintptr_t a1 = a0 + (uintptr_t)(((a_rows - 1) * a_stride + dim) * type_bytes(a_type));
  const uintptr_t b1 = b0 + (uintptr_t)(((b_rows - 1) * b_stride + dim) * type_bytes(b_type));
  return a0 < b1 && b0 < a1;
}

// Bytes that a thread can move at once of every block of a matrix: as many as its rows' starts and ends allow, at most a
// block (32 of fp32, 16 of the others).
static inline int access_bytes(const void* base, int64_t stride, int type, int64_t dim) {
  const int64_t e = type_bytes(type);
  const uint64_t bits = (uint64_t)(uintptr_t)base | (uint64_t)(stride * e) | (uint64_t)(dim * e) | (uint64_t)(kBlockCols * e);
  return (int)(bits & (~bits + 1));
}
static inline bool whole_blocks(const void* base, int64_t stride, int type, int64_t dim) {
  return access_bytes(base, stride, type, dim) == kBlockCols * type_bytes(type);
}

// Division of 32-bit numbers by one that a launch does not change (Granlund and Montgomery, "Division by invariant
// integers using multiplication", PLDI 1994).
struct Divisor {
  uint32_t by, magic, shift1, shift2;
};
static inline Divisor divisor(uint32_t d) {
  int l = 0;
  while (l < 32 && ((uint64_t)1 << l) < d) ++l;
  const uint64_t m = ((((uint64_t)1 << l) - d) << 32) / d + 1;
  return {d, (uint32_t)m, (uint32_t)(l < 1 ? l : 1), (uint32_t)(l > 1 ? l - 1 : 0)};
}

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) {
  const uint32_t t = __umulhi(d.magic, n);
  return (t + ((n - t) >> d.shift1)) >> d.shift2;
}

struct PhiloxKey { uint32_t k0, k1, offset_lo, offset_hi; };

__device__ __forceinline__ PhiloxKey philox_key(const Dropout& d) {
  const uint64_t seed = d.rng ? (uint64_t)d.rng[0] : d.seed, offset = d.rng ? (uint64_t)d.rng[1] : d.offset;
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
}

__device__ __forceinline__ uint4 philox(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1, (uint32_t)a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// The draws of a block of a row: column 2 j in the low half of word j, 2 j + 1 in the high one.
__device__ __forceinline__ uint4 draws_of(const PhiloxKey& k, uint32_t block, uint32_t row) {
  return philox(make_uint4(block, row, k.offset_lo, k.offset_hi), k.k0, k.k1);
}

// Multiplies a block by the factor; zeros where values are dropped, whatever they were.
__device__ __forceinline__ void drop_block(float (&x)[kBlockCols], const PhiloxKey& k, uint32_t drop_below, float factor,
                                           uint32_t block, uint32_t row) {
  const uint4 w = draws_of(k, block, row);
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
  if (drop_below > 0xffffu) {  // all of them
#pragma unroll
    for (int j = 0; j < kBlockCols; ++j) x[j] = 0.0f;
    return;
  }
  const uint32_t top = drop_below << 16;  // halves are compared where they lie high in a word
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = (word[j] << 16) >= top ? x[2 * j] * factor : 0.0f;
    x[2 * j + 1] = word[j] >= top ? x[2 * j + 1] * factor : 0.0f;
  }
}

// ---- a block in memory: eight values as the words that they take -------------------------------------------------------
template <typename T> constexpr int block_words() { return kBlockCols * (int)sizeof(T) / 4; }

template <int W> struct Words { uint32_t w[W]; };

// Whole blocks that begin where a block can be moved at once.
__device__ __forceinline__ void load_block(const void* p, Words<4>& v) {
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]) : "l"(p));
}
__device__ __forceinline__ void load_block(const void* p, Words<8>& v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p));
}
__device__ __forceinline__ void store_block(void* p, const Words<4>& v) {
  *static_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
__device__ __forceinline__ void store_block(void* p, const Words<8>& v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]),
               "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
               : "memory");
}

// Loads of what no other thread of the launch writes (an in-place call reads a value before it writes it, in one thread).
// width: access_bytes of the matrix; cols: columns of the row from the block on.  What lies behind the row's end is not read,
// and undefined in `v`.
template <typename T>
__device__ __forceinline__ void load_words(const T* p, int width, int cols, Words<block_words<T>()>& v) {
  constexpr int W = block_words<T>(), per = 4 / (int)sizeof(T);  // values of a word
  const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
  if (width >= 16) {
#pragma unroll
    for (int i = 0; i < W; i += 4)
      if (i == 0 || i * per < cols) {
        const uint4 t = *reinterpret_cast<const uint4*>(q + i);
        v.w[i] = t.x; v.w[i + 1] = t.y; v.w[i + 2] = t.z; v.w[i + 3] = t.w;
      }
  } else if (width == 8) {
#pragma unroll
    for (int i = 0; i < W; i += 2)
      if (i == 0 || i * per < cols) {
        const uint2 t = *reinterpret_cast<const uint2*>(q + i);
        v.w[i] = t.x; v.w[i + 1] = t.y;
      }
  } else if (width == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i == 0 || i * per < cols) v.w[i] = q[i];
  } else if constexpr (sizeof(T) == 2) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    if (cols < kBlockCols) {
#pragma unroll
      for (int i = 0; i < kBlockCols; ++i)
        if (i < cols) v.w[i / 2] = i & 1 ? v.w[i / 2] | (uint32_t)h[i] << 16 : h[i];
    } else if ((uintptr_t)p & 2u) {  // the first value, three words, the last value
      const uint32_t* m = reinterpret_cast<const uint32_t*>(h + 1);
      const uint32_t first = h[0], m0 = m[0], m1 = m[1], m2 = m[2], last = h[7];
      v.w[0] = first | m0 << 16;
      v.w[1] = __funnelshift_r(m0, m1, 16);
      v.w[2] = __funnelshift_r(m1, m2, 16);
      v.w[3] = m2 >> 16 | last << 16;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) v.w[i] = q[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_words(T* p, int width, int cols, const Words<block_words<T>()>& v) {
  constexpr int W = block_words<T>(), per = 4 / (int)sizeof(T);
  uint32_t* q = reinterpret_cast<uint32_t*>(p);
  if (width >= 16) {
#pragma unroll
    for (int i = 0; i < W; i += 4)
      if (i == 0 || i * per < cols) *reinterpret_cast<uint4*>(q + i) = make_uint4(v.w[i], v.w[i + 1], v.w[i + 2], v.w[i + 3]);
  } else if (width == 8) {
#pragma unroll
    for (int i = 0; i < W; i += 2)
      if (i == 0 || i * per < cols) *reinterpret_cast<uint2*>(q + i) = make_uint2(v.w[i], v.w[i + 1]);
  } else if (width == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i == 0 || i * per < cols) q[i] = v.w[i];
  } else if constexpr (sizeof(T) == 2) {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < kBlockCols; ++i)
      if (i < cols) h[i] = (uint16_t)(v.w[i / 2] >> (16 * (i & 1)));
  }
}

// ---- words and values: everything between a load and a store is fp32, and rounded once ----------------------------------
template <typename T>
__device__ __forceinline__ void values_of(const Words<block_words<T>()>& v, float (&x)[kBlockCols]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f;
      if constexpr (std::is_same_v<T, __half>) f = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
      else f = make_float2(__uint_as_float(v.w[i] << 16), __uint_as_float(v.w[i] & 0xffff0000u));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void words_of(const float (&x)[kBlockCols], Words<block_words<T>()>& v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
}

// sum += value j of a word of two, or of a word of one (j = 0), in one instruction
template <typename T>
__device__ __forceinline__ void add_value(float& sum, uint32_t w, int j) {
  if constexpr (sizeof(T) == 4) {
    sum += __uint_as_float(w);
  } else if constexpr (std::is_same_v<T, __half>) {
    if (j == 0) asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; add.rn.f32.f16 %0, l, %0;}" : "+f"(sum) : "r"(w));
    else asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; add.rn.f32.f16 %0, h, %0;}" : "+f"(sum) : "r"(w));
  } else {
    if (j == 0) asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; add.rn.f32.bf16 %0, l, %0;}" : "+f"(sum) : "r"(w));
    else asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; add.rn.f32.bf16 %0, h, %0;}" : "+f"(sum) : "r"(w));
  }
}
// Adds a block to a sum: all of it, or what is kept of it.
template <typename T>
__device__ __forceinline__ void add_block(float (&sum)[kBlockCols], const Words<block_words<T>()>& v) {
  constexpr int per = 4 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < kBlockCols; ++i) add_value<T>(sum[i], v.w[i / per], i % per);
}
template <typename T>
__device__ __forceinline__ void add_kept(float (&sum)[kBlockCols], const Words<block_words<T>()>& v, const uint4& d,
                                         uint32_t drop_below) {
  constexpr int per = 4 / (int)sizeof(T);
  if (drop_below > 0xffffu) return;  // none of it
  const uint32_t word[4] = {d.x, d.y, d.z, d.w}, top = drop_below << 16;
#pragma unroll
  for (int i = 0; i < kBlockCols; ++i)
    if ((i & 1 ? word[i / 2] : word[i / 2] << 16) >= top) add_value<T>(sum[i], v.w[i / per], i % per);
}

#endif  // __CUDACC__

// f(T{}) for the value type of a matrix
template <typename F>
int with_type(int type, F f) {
  if (type == HB_TYPE_F32) return f(float{});
  if (type == HB_TYPE_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace hb
