// Work that needs nothing of a call's first kernels and runs beside them: zeros for an output.
//
// A warp on every SM does it through the bulk-copy engine, so that whatever runs meanwhile finds its room on the SMs: a
// cluster of CTAs that sorts, most of all.  Zeros leave from 32 KB of shared memory, and the warps take the stretches of the
// output by a ticket: writes that advance in step are what HBM likes (1 GB in 147 us, 7.3 TB/s; a fixed share of the
// stretches to every warp 171 us, plain stores 155 to 180, one short-lived CTA per 16 KB 145, which leaves no room).
// (Rows that will be read, brought into L2 meanwhile, gained nothing: the sums behind are not bound by HBM.)
#pragma once

#include "bulk.cuh"
#include "launch.cuh"

namespace hb {

// A stream of this thread on the current device that forks from a stream of the caller's and joins it again.
class Aside {
 public:
  // After everything that `main` holds so far; false: no stream (then nothing is to be launched on it).  Not for captures:
  // the stream would belong to two of them where a thread captures two graphs in turns.
  bool fork(cudaStream_t main) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return false;
    Lane& l = lanes().of[dev];
    if (!l.ready) {
      if (cudaStreamCreateWithFlags(&l.stream, cudaStreamNonBlocking) != cudaSuccess ||
          cudaEventCreateWithFlags(&l.forked, cudaEventDisableTiming) != cudaSuccess ||
          cudaEventCreateWithFlags(&l.done, cudaEventDisableTiming) != cudaSuccess) {
        cudaGetLastError();
        return false;
      }
      l.ready = true;
    }
    if (cudaEventRecord(l.forked, main) != cudaSuccess || cudaStreamWaitEvent(l.stream, l.forked, 0) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    lane_ = &l;
    main_ = main;
    return true;
  }
  bool forked() const { return lane_ != nullptr; }
  cudaStream_t stream() const { return lane_->stream; }
  // What comes next on the caller's stream comes behind what was launched on this one.
  cudaError_t join() {
    if (!lane_) return cudaSuccess;
    Lane* l = lane_;
    lane_ = nullptr;
    const cudaError_t e = cudaEventRecord(l->done, l->stream);
    return e != cudaSuccess ? e : cudaStreamWaitEvent(main_, l->done, 0);
  }
  ~Aside() { join(); }  // (a call that failed half way)

 private:
  static constexpr int kDevices = 64;
  struct Lane {
    cudaStream_t stream = nullptr;
    cudaEvent_t forked = nullptr, done = nullptr;
    bool ready = false;
  };
  struct Lanes {
    Lane of[kDevices];
    ~Lanes() {  // the end of the thread; fails harmlessly where the runtime is gone
      for (Lane& l : of)
        if (l.ready) {
          cudaEventDestroy(l.forked);
          cudaEventDestroy(l.done);
          cudaStreamDestroy(l.stream);
        }
    }
  };
  static Lanes& lanes() {
    static thread_local Lanes t;
    return t;
  }
  Lane* lane_ = nullptr;
  cudaStream_t main_ = nullptr;
};

constexpr int kZerosChunk = 32768;

#ifdef __CUDACC__
// [zeros, zeros + bytes), whole values of two bytes; ticket: zero before.  kZerosChunk bytes of shared memory.
static __global__ void __launch_bounds__(32) zeros_kernel(char* zeros, int64_t bytes, unsigned* ticket) {
  extern __shared__ __align__(128) char s_zeros[];
  for (int i = threadIdx.x * 16; i < kZerosChunk; i += 32 * 16) *reinterpret_cast<uint4*>(s_zeros + i) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
  char *const end = zeros + bytes, *from = reinterpret_cast<char*>(((uintptr_t)zeros + 15) & ~(uintptr_t)15);
  if (from > end) from = end;
  char* const to = from + ((end - from) & ~(int64_t)15);
  if (blockIdx.x == 0 && threadIdx.x < 8) {  // the ends that bulk copies do not reach
    if (zeros + 2 * threadIdx.x < from) reinterpret_cast<uint16_t*>(zeros)[threadIdx.x] = 0;
    if (to + 2 * threadIdx.x < end) reinterpret_cast<uint16_t*>(to)[threadIdx.x] = 0;
  }
  if (threadIdx.x != 0) return;
  for (;;) {
    char* p = from + (int64_t)atomicAdd(ticket, 1u) * kZerosChunk;
    if (p >= to) break;
    bulk_s2g(p, s_zeros, (uint32_t)(to - p < kZerosChunk ? to - p : kZerosChunk));
    bulk_commit();
    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
  }
  bulk_wait_all();
}
#endif

}  // namespace hb
