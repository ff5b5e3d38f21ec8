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

// A stream that forks from a stream of the caller's and joins it again.  Each stream of a caller's has one of its own for
// every thread that calls: of a stream that two of them shared, the second call's work would wait for all that came in front
// of the first, and two streams that are to run side by side would run one after the other, or wait for one another.
class Aside {
 public:
  // After everything that `main` holds so far; false: no stream (then nothing is to be launched on it).  Not for captures:
  // the stream would belong to two of them where a thread captures two graphs in turns.
  bool fork(cudaStream_t main) {
    Lane* l = lane_of(main);
    if (!l) return false;
    if (cudaEventRecord(l->forked, main) != cudaSuccess || cudaStreamWaitEvent(l->stream, l->forked, 0) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    lane_ = l;
    main_ = main;
    return true;
  }
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
  static constexpr int kLanes = 64;  // of a thread: streams of callers that come behind those have none
  struct Lane {
    int device = -1;
    unsigned long long caller = 0;  // of the caller's stream, which no later stream has (a handle may come again)
    cudaStream_t stream = nullptr;
    cudaEvent_t forked = nullptr, done = nullptr;
    bool make() {
      // (a capture that another thread has begun allows it too)
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaThreadExchangeStreamCaptureMode(&mode);
      const bool made = cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking) == cudaSuccess &&
                        cudaEventCreateWithFlags(&forked, cudaEventDisableTiming) == cudaSuccess &&
                        cudaEventCreateWithFlags(&done, cudaEventDisableTiming) == cudaSuccess;
      if (!made) {
        cudaGetLastError();
        drop();
      }
      cudaThreadExchangeStreamCaptureMode(&mode);
      return made;
    }
    void drop() {
      if (done) cudaEventDestroy(done);
      if (forked) cudaEventDestroy(forked);
      if (stream) cudaStreamDestroy(stream);
      *this = Lane();
    }
  };
  struct Lanes {
    Lane of[kLanes];
    int made = 0;
    ~Lanes() {  // the end of the thread; fails harmlessly where the runtime is gone
      for (int k = 0; k < made; ++k) of[k].drop();
    }
  };
  static Lanes& lanes() {
    static thread_local Lanes t;
    return t;
  }
  static Lane* lane_of(cudaStream_t main) {
    int dev = 0;
    unsigned long long caller = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaStreamGetId(main, &caller) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    Lanes& t = lanes();
    for (int k = 0; k < t.made; ++k)
      if (t.of[k].caller == caller && t.of[k].device == dev) return &t.of[k];
    if (t.made == kLanes || !t.of[t.made].make()) return nullptr;
    Lane& l = t.of[t.made++];
    l.device = dev;
    l.caller = caller;
    return &l;
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
