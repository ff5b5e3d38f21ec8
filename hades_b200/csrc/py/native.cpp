// The host half of the calls that a training or serving loop makes per batch: argument checks, the
// tensors they return, the launches of libhades_b200, in one native call instead of some thirty
// Python and ctypes operations.  A small batch is bound by exactly that: 1,000 looked-up rows cost
// 6 us on the GPU and 19 us in Python.
//
// Nothing is kept between calls except, per thread, one pinned word through which a kernel hands the
// host a number (how many ids are distinct) while later kernels of the call still run.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <atomic>
#include <cstring>
#include <stdexcept>
#include <string>

#include "hades_b200.h"

namespace {

PyObject* g_error = nullptr;  // hades_b200._lib.HadesError

struct Status {};  // a library call failed; the Python error is set
struct LibraryError : std::runtime_error {  // the same where the interpreter's lock is not held
  using std::runtime_error::runtime_error;
};

void check(int rc) {
  if (rc == HB_OK) return;
  PyErr_Format(g_error ? g_error : PyExc_RuntimeError, "libhades_b200 status %d: %s", rc, hb_last_error());
  throw Status();
}

void require(bool ok, const char* what) {
  if (ok) return;
  PyErr_Format(PyExc_RuntimeError, "Check failed: %s", what);
  throw Status();
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: a tensor is expected", what);
    throw Status();
  }
  return THPVariable_Unpack(o);
}

bool none(PyObject* o) { return o == Py_None; }

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Status();
  return v;
}
void* pointer(PyObject* o) { return reinterpret_cast<void*>(static_cast<uintptr_t>(integer(o))); }

at::Tensor cuda_empty(at::IntArrayRef size, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(size, type, dev, std::nullopt);
}

void* stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

int64_t row_bytes(const at::Tensor& t) { return (t.dim() == 1 ? 1 : t.size(1)) * (int64_t)t.element_size(); }

void ids_ok(const at::Tensor& ids) {
  require(ids.is_cuda() && ids.scalar_type() == at::kLong, "ids is a CUDA int64 tensor");
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Status&) {
  } catch (const LibraryError& e) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

void arity(Py_ssize_t n, Py_ssize_t want, const char* name) {
  if (n == want) return;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
  throw Status();
}

PyObject* pack(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New((Py_ssize_t)items.size());
  Py_ssize_t k = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(t, k++, o);
  return t;
}
PyObject* wrap_or_none(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// A few words of pinned memory per thread that kernels of any device can write.
struct HostWord {
  volatile int64_t* word = nullptr;  // 8 of them
  ~HostWord() {
    if (word) cudaFreeHost(const_cast<int64_t*>(word));  // fails harmlessly when the runtime is gone
  }
  int64_t* arm() {
    if (!word) {
      void* p = nullptr;
      if (cudaHostAlloc(&p, 64, cudaHostAllocPortable) != cudaSuccess) {
        PyErr_SetString(PyExc_RuntimeError, "cudaHostAlloc of 64 bytes failed");
        throw Status();
      }
      word = static_cast<int64_t*>(p);
    }
    for (int k = 0; k < 8; ++k) word[k] = -1;
    return const_cast<int64_t*>(word);
  }
  // Waits until a kernel on `stream` has written the word.  The stream is asked now and then whether
  // it still runs, so that a launch that failed ends the wait with its error.
  int64_t wait(cudaStream_t stream, int which = 0) {
    volatile int64_t* word = this->word + which;
    int64_t v = -1;
    cudaError_t e = cudaSuccess;
    Py_BEGIN_ALLOW_THREADS;
    for (unsigned spins = 1; (v = *word) < 0; ++spins) {
      if ((spins & 0x3fff) == 0) {
        e = cudaStreamQuery(stream);
        if (e != cudaErrorNotReady) {
          v = *word;
          break;
        }
      }
#if defined(__x86_64__)
      __builtin_ia32_pause();
#endif
    }
    Py_END_ALLOW_THREADS;
    if (v < 0) {
      PyErr_Format(PyExc_RuntimeError, "no count arrived from the device: %s", cudaGetErrorString(e));
      throw Status();
    }
    return v;
  }
};
thread_local HostWord t_word;

// lookup_fetch(index, ids, cache_rows, cache_ptr, backing_ptr, out_rows | None, mode, mover, want_locs)
PyObject* lookup_fetch(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 9, "lookup_fetch");
    const at::Tensor& given = tensor(a[1], "ids");
    ids_ok(given);
    const at::Tensor ids = given.contiguous();
    const at::Tensor& rows = tensor(a[2], "cache_rows");
    const at::Device dev = ids.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t n = ids.numel();
    at::Tensor out = none(a[5]) ? cuda_empty({n, rows.size(1)}, rows.scalar_type(), dev) : tensor(a[5], "out_rows");
    require(out.size(1) == rows.size(1), "out_rows.size(1) == cache_rows.size(1)");
    at::Tensor locs, found = cuda_empty({n}, at::kBool, dev);
    if (PyObject_IsTrue(a[8])) locs = cuda_empty({n}, at::kLong, dev);
    check(hb_lookup_fetch(static_cast<hb_index_t*>(pointer(a[0])), ids.data_ptr<int64_t>(), n, pointer(a[3]), pointer(a[4]),
                          row_bytes(rows), out.data_ptr(), locs.defined() ? locs.data_ptr<int64_t>() : nullptr,
                          static_cast<uint8_t*>(found.data_ptr()), (int)integer(a[6]), (int)integer(a[7]), stream_of(dev)));
    return pack({THPVariable_Wrap(out), wrap_or_none(locs), THPVariable_Wrap(found)});
  });
}

// unique_segsum(ids, grads, cnt | None, mean, id_bits) -> (unique ids, rows, counts), cut to the number
// of distinct ids, which is awaited while the rows are still being added up
PyObject* unique_segsum(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 5, "unique_segsum");
    const at::Tensor ids = tensor(a[0], "ids").contiguous();
    const at::Tensor grads = tensor(a[1], "grads").contiguous();
    const at::Device dev = ids.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t n = ids.numel(), dim = grads.size(1);
    at::Tensor cnt;
    if (!none(a[2])) cnt = tensor(a[2], "cnt").contiguous();
    at::Tensor uniq = cuda_empty({n}, at::kLong, dev), counts = cuda_empty({n}, at::kLong, dev);
    at::Tensor sums = cuda_empty({n, dim}, at::kFloat, dev);
    const size_t need = hb_unique_segsum_workspace_bytes(n, dim);
    const at::Tensor ws = cuda_empty({(int64_t)need}, at::kByte, dev);
    void* st = stream_of(dev);
    int64_t* num = t_word.arm();
    check(hb_unique_segsum_f32(ids.data_ptr<int64_t>(), grads.data_ptr<float>(), cnt.defined() ? cnt.data_ptr<int64_t>() : nullptr,
                               n, nullptr, nullptr, 0, dim, (int)integer(a[4]), PyObject_IsTrue(a[3]),
                               uniq.data_ptr<int64_t>(), sums.data_ptr<float>(), counts.data_ptr<int64_t>(), num, nullptr,
                               nullptr, ws.data_ptr(), need, st));
    const int64_t u = t_word.wait(static_cast<cudaStream_t>(st));
    if (u == 0) throw std::runtime_error("the sort of the ids gave up waiting (hb_device_status)");
    return pack({THPVariable_Wrap(uniq.narrow(0, 0, u)), THPVariable_Wrap(sums.narrow(0, 0, u)),
                 THPVariable_Wrap(counts.narrow(0, 0, u))});
  });
}

// unique_update(ids, grads, cnt | None, n_dev | None, seg_counts | None, seg_cap, id_bits, optimiser, mean):
// optimiser: address of an hb_optim_t
PyObject* unique_update(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 9, "unique_update");
    const at::Tensor &ids = tensor(a[0], "idx"), &grads = tensor(a[1], "grad");
    const at::Device dev = ids.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t n = ids.numel(), dim = grads.size(1);
    const hb_optim_t* opt = static_cast<const hb_optim_t*>(pointer(a[7]));
    auto i64 = [&](PyObject* o) -> const int64_t* { return none(o) ? nullptr : tensor(o, "count").data_ptr<int64_t>(); };
    const size_t need = hb_unique_update_workspace_bytes(n, dim, grads.data_ptr<float>(), opt);
    const at::Tensor ws = cuda_empty({(int64_t)need}, at::kByte, dev);
    check(hb_unique_update_f32(ids.data_ptr<int64_t>(), grads.data_ptr<float>(), i64(a[2]), n, i64(a[3]), i64(a[4]),
                               integer(a[5]), dim, (int)integer(a[6]), PyObject_IsTrue(a[8]),
                               opt, ws.data_ptr(), need, stream_of(dev)));
    Py_RETURN_NONE;
  });
}

// Kernels of a call read and write pinned buffers of that call: one that fails half way waits for them, and
// leaves no batch open.
struct InFlight {
  cudaStream_t stream;
  hb_index_t* index = nullptr;
  const int64_t* locs = nullptr;
  int64_t looked_up = 0;
  bool ended = false;
  ~InFlight() {
    if (ended) return;
    if (looked_up) hb_index_lookup_touch_end(index, locs, looked_up, stream);
    cudaStreamSynchronize(stream);
  }
};

// n ids as signed 32-bit numbers; false: some do not fit, found out within 512 ids of the first that does not, or at
// once from the last (sorted ids).  (Ids beyond 32 bits, 32,768 / 65,536: 48 / 79 us, 54 / 87 where all of a part was
// narrowed first, 47 / 78 without narrowing; one such id amid others near the end of a part still 54 / 71.)
__attribute__((optimize("O3"))) bool narrow(const int64_t* __restrict__ from, int32_t* __restrict__ to, int64_t n) {
  if (from[n - 1] != (int32_t)from[n - 1]) return false;
  for (int64_t at = 0; at < n; at += 512) {
    const int64_t end = n - at < 512 ? n : at + 512;
    uint64_t off = 0;  // (an id that fits lies in [0, 2^32) from -2^31 on)
    for (int64_t i = at; i < end; ++i) {
      off |= ((uint64_t)from[i] + 0x80000000ull) >> 32;
      to[i] = (int32_t)from[i];
    }
    if (off) return false;
  }
  return true;
}
__attribute__((optimize("O3"))) void widen(const int32_t* __restrict__ from, int64_t* __restrict__ to, int64_t n) {
  for (int64_t i = 0; i < n; ++i) to[i] = from[i];
}

at::Tensor pinned_empty(int64_t n) {
  return at::empty({n}, at::TensorOptions().dtype(at::kLong).pinned_memory(true));
}

// index_lookup(index, ids in host memory, device, mode, address of two words shared with other processes | 0) ->
// slots in host memory.  Ids and slots pass through two pinned buffers each, a part of the batch at a time: while
// the GPU looks one part up the host copies the next in and the one before out, and the ageing runs under the last
// copies and after.  Calls on the index from other streams wait for it; where another process has opened the index
// (words[0]), which can only be ordered by the host, the call does.  A process that opens it later finds in words[1]
// how many lookups to wait for: that is written before words[0] is read, so that one of the two waits.
// 500 ids: 25 us (two pageable copies: 70), 65,536: 65 (183; 85 with ids and slots in 64 bits on their way).
PyObject* index_lookup(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 5, "index_lookup");
    hb_index_t* h = static_cast<hb_index_t*>(pointer(a[0]));
    const at::Tensor ids = tensor(a[1], "ids").contiguous();
    const at::Device dev(at::kCUDA, (c10::DeviceIndex)integer(a[2]));
    const int mode = (int)integer(a[3]);
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t st = static_cast<cudaStream_t>(stream_of(dev));
    const int64_t n = ids.numel();
    at::Tensor out = at::empty_like(ids);
    // as few parts as 32,768 ids each allow, all of one size: a part costs the GPU some 10 us of trips over
    // PCIe whatever its size (65,536 ids in parts of 11,000: 109 us, 16,384: 87, 22,000: 74, 32,768: 65, 65,536: 70)
    constexpr int64_t kPart = 32768;
    const int64_t parts = (n + kPart - 1) / kPart, part = (n + parts - 1) / parts;
    const at::Tensor in = pinned_empty(2 * part), back = pinned_empty(2 * part);
    const at::Tensor locs = cuda_empty({n}, at::kLong, dev);
    const int64_t* src = ids.data_ptr<int64_t>();
    int64_t *to = out.data_ptr<int64_t>(), *pin = in.data_ptr<int64_t>(), *pback = back.data_ptr<int64_t>();
    volatile int64_t* words = t_word.arm();
    InFlight in_flight{st, h, locs.data_ptr<int64_t>()};
    auto length = [&](int64_t k) { return (k + 1) * part < n ? part : n - k * part; };
    bool narrowed[2] = {false, false};
    auto collect = [&](int64_t k) {
      t_word.wait(st, (int)(k & 1));
      words[k & 1] = -1;
      const int64_t* slots = pback + (k & 1) * part;
      if (narrowed[k & 1]) widen(reinterpret_cast<const int32_t*>(slots), to + k * part, length(k));
      else memcpy(to + k * part, slots, length(k) * sizeof(int64_t));
    };
    for (int64_t k = 0; k < parts; ++k) {
      if (k >= 2) collect(k - 2);
      int64_t *ids_in = pin + (k & 1) * part, *slots = pback + (k & 1) * part;
      int64_t* word = const_cast<int64_t*>(words + (k & 1));
      int32_t* ids32 = reinterpret_cast<int32_t*>(ids_in);
      narrowed[k & 1] = narrow(src + k * part, ids32, length(k));
      if (narrowed[k & 1]) {
        check(hb_index_lookup_touch_part32(h, ids32, length(k), locs.data_ptr<int64_t>(), k * part,
                                           reinterpret_cast<int32_t*>(slots), word, mode, st));
      } else {
        memcpy(ids_in, src + k * part, length(k) * sizeof(int64_t));
        check(hb_index_lookup_touch_part(h, ids_in, length(k), locs.data_ptr<int64_t>(), k * part, slots, word, mode, st));
      }
      in_flight.looked_up = k * part + length(k);
    }
    check(hb_index_lookup_touch_end(h, locs.data_ptr<int64_t>(), n, st));
    in_flight.looked_up = 0;
    for (int64_t k = parts < 2 ? 0 : parts - 2; k < parts; ++k) collect(k);
    volatile uint64_t* shared = static_cast<volatile uint64_t*>(pointer(a[4]));
    if (shared) {
      shared[1] = hb_index_lookups(h);
      std::atomic_thread_fence(std::memory_order_seq_cst);
    }
    if (shared && shared[0]) {
      cudaError_t e;
      Py_BEGIN_ALLOW_THREADS;
      e = cudaStreamSynchronize(st);
      Py_END_ALLOW_THREADS;
      if (e != cudaSuccess) throw std::runtime_error(cudaGetErrorString(e));
    }
    in_flight.ended = true;  // (what still runs uses device memory only)
    return THPVariable_Wrap(out);
  });
}

// index_add(index, ids in host memory, device) -> slots in host memory
PyObject* index_add(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 3, "index_add");
    hb_index_t* h = static_cast<hb_index_t*>(pointer(a[0]));
    const at::Tensor ids = tensor(a[1], "ids").contiguous();
    const at::Device dev(at::kCUDA, (c10::DeviceIndex)integer(a[2]));
    c10::cuda::CUDAGuard guard(dev);
    cudaStream_t st = static_cast<cudaStream_t>(stream_of(dev));
    const int64_t n = ids.numel();
    const size_t bytes = (size_t)n * sizeof(int64_t);
    at::Tensor out = at::empty_like(ids);
    const at::Tensor in = pinned_empty(n), back = pinned_empty(n);
    // up to here the walk writes its slots, one word at a time, to the pinned buffer (2,000 ids: 31 us, 41
    // with a copy); 50,000 ids: 125 us so, 93 with a copy
    const bool direct = n <= 16384;
    const at::Tensor dids = cuda_empty({n}, at::kLong, dev), locs = direct ? back : cuda_empty({n}, at::kLong, dev);
    const size_t need = hb_index_add_workspace_bytes(n);
    const at::Tensor ws = cuda_empty({(int64_t)need}, at::kByte, dev);
    memcpy(in.data_ptr(), ids.data_ptr(), bytes);
    InFlight in_flight{st};
    if (cudaMemcpyAsync(dids.data_ptr(), in.data_ptr(), bytes, cudaMemcpyHostToDevice, st) != cudaSuccess)
      throw std::runtime_error("copy of the ids to the device failed");
    check(hb_index_add(h, dids.data_ptr<int64_t>(), n, locs.data_ptr<int64_t>(), nullptr, ws.data_ptr(), need, st));
    cudaError_t e = cudaSuccess;
    Py_BEGIN_ALLOW_THREADS;
    if (!direct) e = cudaMemcpyAsync(back.data_ptr(), locs.data_ptr(), bytes, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    Py_END_ALLOW_THREADS;
    if (e != cudaSuccess) throw std::runtime_error(cudaGetErrorString(e));
    in_flight.ended = true;
    memcpy(out.data_ptr(), back.data_ptr(), bytes);
    return THPVariable_Wrap(out);
  });
}

// staging_flush(index | None, address of the hb_staging_t, cnt_threshold, rows the output holds, device) for
// one client -> (ids, rows, cnt, counts, number of stale rows); the number is read while the rows move
PyObject* staging_flush(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 5, "staging_flush");
    hb_index_t* h = none(a[0]) ? nullptr : static_cast<hb_index_t*>(pointer(a[0]));
    const hb_staging_t* s = static_cast<const hb_staging_t*>(pointer(a[1]));
    const int64_t cap = integer(a[3]);
    const at::Device dev(at::kCUDA, (c10::DeviceIndex)integer(a[4]));
    c10::cuda::CUDAGuard guard(dev);
    at::Tensor ids = cuda_empty({cap}, at::kLong, dev), rows = cuda_empty({cap, s->dim}, at::kFloat, dev);
    at::Tensor cnt = cuda_empty({cap}, at::kLong, dev), counts = cuda_empty({1}, at::kLong, dev);
    const size_t need = hb_staging_flush_workspace_bytes(s->slots, 1);
    const at::Tensor ws = cuda_empty({(int64_t)need}, at::kByte, dev);
    void* st = stream_of(dev);
    int64_t* num = t_word.arm();
    check(hb_staging_flush_counted(h, s, (int32_t)integer(a[2]), 1, cap, ids.data_ptr<int64_t>(), rows.data_ptr<float>(),
                                   cnt.data_ptr<int64_t>(), counts.data_ptr<int64_t>(), num, ws.data_ptr(), need, st));
    const int64_t stale = t_word.wait(static_cast<cudaStream_t>(st)), u = stale < cap ? stale : cap;
    return pack({THPVariable_Wrap(ids.narrow(0, 0, u)), THPVariable_Wrap(rows.narrow(0, 0, u)),
                 THPVariable_Wrap(cnt.narrow(0, 0, u)), THPVariable_Wrap(counts), PyLong_FromLongLong(stale)});
  });
}

// step_forward(step, desc, ids, dim, row dtype tensor, out_rows | None, want_locs, aside, ws | None)
// -> (rows, locs | None, found, counters, ws)
PyObject* step_forward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 9, "step_forward");
    const at::Tensor& ids = tensor(a[2], "ids");
    ids_ok(ids);
    require(ids.is_contiguous(), "ids is contiguous");
    const at::Device dev = ids.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t n = ids.numel(), dim = integer(a[3]);
    at::Tensor out = none(a[5]) ? cuda_empty({n, dim}, tensor(a[4], "rows").scalar_type(), dev) : tensor(a[5], "out_rows");
    require(out.size(1) == dim, "out_rows.size(1) == cache_rows.size(1)");
    require(out.is_contiguous(), "out_rows is contiguous");
    at::Tensor locs, found = cuda_empty({n}, at::kBool, dev), counters = cuda_empty({4}, at::kLong, dev);
    if (PyObject_IsTrue(a[6])) locs = cuda_empty({n}, at::kLong, dev);
    const size_t need = hb_step_workspace_bytes(n, dim);
    at::Tensor ws;
    if (!none(a[8])) ws = tensor(a[8], "ws");
    if (!ws.defined() || ws.numel() < (int64_t)need) ws = cuda_empty({(int64_t)(need + need / 4)}, at::kByte, dev);
    check(hb_step_forward(static_cast<hb_step_t*>(pointer(a[0])), static_cast<const hb_step_desc_t*>(pointer(a[1])),
                          ids.data_ptr<int64_t>(), n, out.data_ptr(), locs.defined() ? locs.data_ptr<int64_t>() : nullptr,
                          static_cast<uint8_t*>(found.data_ptr()), counters.data_ptr<int64_t>(), PyObject_IsTrue(a[7]),
                          ws.data_ptr(), (size_t)ws.numel(), stream_of(dev)));
    return pack({THPVariable_Wrap(out), wrap_or_none(locs), THPVariable_Wrap(found), THPVariable_Wrap(counters),
                 THPVariable_Wrap(ws)});
  });
}

// step_backward(step, desc, ids | None, n, grads, counters, ws)
PyObject* step_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 7, "step_backward");
    const at::Tensor& grads = tensor(a[4], "grads");
    const at::Tensor& ws = tensor(a[6], "ws");
    const at::Device dev = grads.device();
    c10::cuda::CUDAGuard guard(dev);
    const int64_t n = integer(a[3]);
    const int64_t* ids = none(a[2]) ? nullptr : tensor(a[2], "ids").data_ptr<int64_t>();
    check(hb_step_backward(static_cast<hb_step_t*>(pointer(a[0])), static_cast<const hb_step_desc_t*>(pointer(a[1])), ids, n,
                           grads.data_ptr<float>(), tensor(a[5], "counters").data_ptr<int64_t>(), ws.data_ptr(),
                           (size_t)ws.numel(), stream_of(dev)));
    Py_RETURN_NONE;
  });
}

// ---- token embeddings ---------------------------------------------------------------------------------------------------
// What runs in a backward pass is on a thread of the autograd engine, without the interpreter's lock: errors of these
// functions are C++ exceptions, which `guarded` and the engine turn into Python's.
void need(bool ok, const char* what) {
  if (!ok) throw std::runtime_error(std::string("Check failed: ") + what);
}
void succeed(int rc) {
  if (rc != HB_OK) throw LibraryError("libhades_b200 status " + std::to_string(rc) + ": " + hb_last_error());
}

int value_type(at::ScalarType t, const char* what) {
  if (t == at::kFloat) return HB_TYPE_F32;
  if (t == at::kHalf) return HB_TYPE_F16;
  if (t == at::kBFloat16) return HB_TYPE_BF16;
  throw std::runtime_error(std::string("Check failed: ") + what + " is fp32, fp16 or bf16");
}
at::ScalarType type_or(PyObject* o, at::ScalarType other) {
  if (none(o)) return other;
  if (!THPDtype_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "dtype: a torch.dtype is expected");
    throw Status();
  }
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
// The type of a result: that of `out` where it is given (and of dtype, if that is given too).
at::ScalarType result_type(PyObject* dtype, const at::Tensor& out, at::ScalarType other) {
  if (!out.defined()) return type_or(dtype, other);
  need(type_or(dtype, out.scalar_type()) == out.scalar_type(), "out.dtype == dtype");
  return out.scalar_type();
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Status();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Status();
  return v != 0;
}
uint64_t word64(PyObject* o) {  // OverflowError outside of [0, 2^64)
  const unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == (unsigned long long)-1 && PyErr_Occurred()) throw Status();
  return v;
}
at::Tensor optional_tensor(PyObject* o, const char* what) { return none(o) ? at::Tensor() : tensor(o, what); }
int64_t padding_of(PyObject* o) { return none(o) ? HB_NO_PADDING : integer(o); }

// p, seed, offset, rng | None
struct Mask {
  double p;
  uint64_t seed, offset;
  at::Tensor rng;
  explicit Mask(PyObject* const* a) : p(number(a[0])), seed(word64(a[1])), offset(word64(a[2])), rng(optional_tensor(a[3], "rng")) {}
  hb_drop_t on(const at::Device& dev) const {
    hb_drop_t d{p, seed, offset, nullptr};
    if (rng.defined()) {
      need(rng.device() == dev && rng.scalar_type() == at::kLong && rng.numel() == 2 && rng.is_contiguous(),
           "rng is an int64 tensor of two (seed, offset) on the device of the call");
      d.rng = rng.data_ptr<int64_t>();
    }
    return d;
  }
};

// [rows, dim] of a tensor whose last dimension is dim: the distance of its rows, or -1 where they are not evenly spaced.
int64_t row_stride(const at::Tensor& t) {
  const int64_t k = t.dim();
  if (k > 0 && t.numel() == 0) return t.size(k - 1);  // no rows
  if (k == 0 || (t.size(k - 1) > 1 && t.stride(k - 1) != 1)) return -1;
  int64_t stride = 0, rows = 1;  // rows of the inner dimensions so far
  for (int64_t d = k - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (rows == 1) stride = t.stride(d);
    else if (t.stride(d) != stride * rows) return -1;
    rows *= t.size(d);
  }
  return rows == 1 ? t.size(k - 1) : stride;
}
// A matrix to read: itself, or a contiguous copy where its rows are not evenly spaced (or gigabytes apart).
at::Tensor readable(const at::Tensor& t, int64_t& stride) {
  stride = row_stride(t);
  if (stride >= 0 && stride < ((int64_t)1 << 30)) return t;
  stride = t.size(t.dim() - 1);
  return t.contiguous();
}
at::Tensor token_ids(const at::Tensor& t, const at::Device& dev) {
  need(t.is_cuda() && t.device() == dev, "ids lie on the device of the rows");
  need(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, "ID can only be int32 or int64");
  return t.contiguous();
}
// A result: new, or the caller's, whose rows may lie at a distance.
at::Tensor result(const at::Tensor& out, at::IntArrayRef size, at::ScalarType type, const at::Device& dev, int64_t& stride) {
  stride = size[size.size() - 1];
  if (!out.defined()) return cuda_empty(size, type, dev);
  need(out.device() == dev && out.sizes() == size, "out has the shape of the result and lies on its device");
  stride = row_stride(out);
  need(stride >= 0, "the rows of out are contiguous and evenly spaced");
  out.unsafeGetTensorImpl()->bump_version();  // (a graph that has saved it notices)
  return out;
}

at::Tensor run_embedding(const at::Tensor& weight, const at::Tensor& given, double scale, int64_t padding, const Mask& mask,
                         at::ScalarType type, const at::Tensor& given_out) {
  need(given.is_cuda(), "ids is a CUDA tensor");
  const at::Device dev = given.device();
  need(weight.dim() == 2 && weight.size(1) > 0, "weight is [rows, dim]");
  need(weight.is_cuda() ? weight.device() == dev : weight.is_pinned(),
       "weight lies on the device of the ids, or in pinned host memory");
  need(weight.size(1) == 1 || weight.stride(1) == 1, "the rows of weight are contiguous");
  const int wt = value_type(weight.scalar_type(), "weight"), ot = value_type(type, "out");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor ids = token_ids(given, dev);
  const hb_drop_t drop = mask.on(dev);
  const int64_t dim = weight.size(1);
  c10::SmallVector<int64_t, 5> size(given.sizes().begin(), given.sizes().end());
  size.push_back(dim);
  int64_t stride;
  at::Tensor out = result(given_out, size, type, dev, stride);
  succeed(hb_embedding(weight.data_ptr(), wt, weight.stride(0), weight.size(0), dim, ids.data_ptr(), (int)ids.element_size(),
                       ids.numel(), padding, scale, &drop, out.data_ptr(), ot, stride, stream_of(dev)));
  return out;
}

at::Tensor run_dropout(const at::Tensor& given, double scale, const Mask& mask, at::ScalarType type, const at::Tensor& given_out) {
  need(given.is_cuda() && given.dim() >= 1 && given.size(given.dim() - 1) > 0, "x is a CUDA tensor [..., dim]");
  const at::Device dev = given.device();
  const int xt = value_type(given.scalar_type(), "x"), ot = value_type(type, "out");
  c10::cuda::CUDAGuard guard(dev);
  int64_t x_stride, stride;
  const at::Tensor x = readable(given, x_stride);
  const hb_drop_t drop = mask.on(dev);
  const int64_t dim = x.size(x.dim() - 1);
  at::Tensor out = result(given_out, x.sizes(), type, dev, stride);
  succeed(hb_dropout(x.data_ptr(), xt, x_stride, x.numel() / dim, dim, scale, &drop, out.data_ptr(), ot, stride, stream_of(dev)));
  return out;
}

// What both forms of the gradient take.
struct GradInputs {
  at::Device dev = at::kCPU;
  at::Tensor ids, grads;
  int type;
  int64_t n, dim, stride, rows;
  GradInputs(const at::Tensor& t, const at::Tensor& g, int64_t num_rows) : rows(num_rows) {
    need(g.is_cuda() && g.dim() >= 1 && g.size(g.dim() - 1) > 0, "grad is a CUDA tensor [..., dim]");
    dev = g.device();
    type = value_type(g.scalar_type(), "grad");
    dim = g.size(g.dim() - 1);
    need(g.numel() / dim == t.numel(), "grad has a row for every id");
    need(rows >= 0, "num_embeddings >= 0");
    c10::cuda::CUDAGuard guard(dev);
    ids = token_ids(t, dev);
    grads = readable(g, stride);
    n = ids.numel();
  }
  at::Tensor workspace(size_t& bytes) const {
    bytes = hb_embedding_grad_workspace_bytes(n, dim);
    return cuda_empty({(int64_t)bytes}, at::kByte, dev);
  }
};

at::Tensor run_embedding_grad(const GradInputs& in, double scale, int64_t padding, const Mask& mask, at::ScalarType type,
                              const at::Tensor& given_out, bool accumulate) {
  const int ot = value_type(type, "out");
  c10::cuda::CUDAGuard guard(in.dev);
  const hb_drop_t drop = mask.on(in.dev);
  int64_t stride;
  at::Tensor out = result(given_out, {in.rows, in.dim}, type, in.dev, stride);
  size_t bytes;
  const at::Tensor ws = in.workspace(bytes);
  succeed(hb_embedding_grad(in.ids.data_ptr(), (int)in.ids.element_size(), in.n, padding, in.grads.data_ptr(), in.type, in.stride,
                            in.dim, scale, &drop, in.rows, out.data_ptr(), ot, stride, accumulate, ws.data_ptr(), bytes,
                            stream_of(in.dev)));
  return out;
}

// embedding(weight, ids, scale, padding | None, p, seed, offset, rng | None, dtype | None, out | None)
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 10, "embedding");
    const at::Tensor& weight = tensor(a[0], "weight");
    const at::Tensor out = optional_tensor(a[9], "out");
    return THPVariable_Wrap(run_embedding(weight, tensor(a[1], "ids"), number(a[2]), padding_of(a[3]), Mask(a + 4),
                                          result_type(a[8], out, weight.scalar_type()), out));
  });
}

// dropout(x, scale, p, seed, offset, rng | None, dtype | None, out | None)
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 8, "dropout");
    const at::Tensor& x = tensor(a[0], "x");
    const at::Tensor out = optional_tensor(a[7], "out");
    return THPVariable_Wrap(run_dropout(x, number(a[1]), Mask(a + 2), result_type(a[6], out, x.scalar_type()), out));
  });
}

// embedding_grad(ids, grads, num_rows, scale, padding | None, p, seed, offset, rng | None, dtype | None, out | None, accumulate)
PyObject* embedding_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 12, "embedding_grad");
    const GradInputs in(tensor(a[0], "ids"), tensor(a[1], "grad"), integer(a[2]));
    const bool accumulate = truth(a[11]);
    need(!accumulate || !none(a[10]), "accumulate adds to a given out");
    const at::Tensor out = optional_tensor(a[10], "out");
    return THPVariable_Wrap(run_embedding_grad(in, number(a[3]), padding_of(a[4]), Mask(a + 5),
                                               result_type(a[9], out, in.grads.scalar_type()), out, accumulate));
  });
}

// embedding_grad_rows(ids, grads, num_rows, scale, padding | None, p, seed, offset, rng | None, sync) -> (tokens, rows), cut to
// the number of distinct tokens, which is awaited while the rows are being added up; sync false: (tokens, rows, number)
PyObject* embedding_grad_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 10, "embedding_grad_rows");
    const GradInputs in(tensor(a[0], "ids"), tensor(a[1], "grad"), integer(a[2]));
    const bool sync = truth(a[9]);
    c10::cuda::CUDAGuard guard(in.dev);
    void* st = stream_of(in.dev);
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (sync && cudaStreamIsCapturing(static_cast<cudaStream_t>(st), &capturing) == cudaSuccess)
      need(capturing == cudaStreamCaptureStatusNone, "sync=False in a captured graph (the number is not read on the host)");
    const hb_drop_t drop = Mask(a + 5).on(in.dev);
    at::Tensor uniq = cuda_empty({in.n}, at::kLong, in.dev), rows = cuda_empty({in.n, in.dim}, at::kFloat, in.dev);
    size_t bytes;
    const at::Tensor ws = in.workspace(bytes);
    at::Tensor count;
    if (!sync) count = cuda_empty({1}, at::kLong, in.dev);
    if (sync && in.n == 0) return pack({THPVariable_Wrap(uniq), THPVariable_Wrap(rows)});
    int64_t* num = sync ? t_word.arm() : count.data_ptr<int64_t>();
    succeed(hb_embedding_grad_rows(in.ids.data_ptr(), (int)in.ids.element_size(), in.n, padding_of(a[4]), in.grads.data_ptr(),
                                   in.type, in.stride, in.dim, number(a[3]), &drop, in.rows, uniq.data_ptr<int64_t>(),
                                   rows.data_ptr<float>(), num, ws.data_ptr(), bytes, st));
    if (!sync) return pack({THPVariable_Wrap(uniq), THPVariable_Wrap(rows), THPVariable_Wrap(count)});
    const int64_t u = t_word.wait(static_cast<cudaStream_t>(st));
    // (none: all of it padding, or nothing to go by)
    if (u == 0 && uniq.narrow(0, 0, 1).item<int64_t>() < 0)
      throw std::runtime_error("the sort of the tokens gave up waiting (hb_device_status)");
    return pack({THPVariable_Wrap(uniq.narrow(0, 0, u)), THPVariable_Wrap(rows.narrow(0, 0, u))});
  });
}

// ---- autograd: nodes of the engine's own kind (a training step of a few tokens 84 us on the host with Python's functions) --
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

bool captures(const at::Device& dev) {
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(static_cast<cudaStream_t>(stream_of(dev)), &s) == cudaSuccess && s != cudaStreamCaptureStatusNone;
}

// In a capture: a graph of the same leaf that was built on another stream still lives, and with it what adds up the leaf's
// gradient, on a stream that the capture's backward pass would have to wait for.
void refuse_foreign_graphs(const at::Tensor& leaf, const at::Device& dev) {
  if (!captures(dev)) return;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!accumulator) return;
  const auto stream = accumulator->stream();
  need(stream.has_value() && *stream == c10::cuda::getCurrentCUDAStream(dev.index()).unwrap(),
       "a graph of the same leaf that was built outside of this capture still lives (drop its outputs first)");
}

// Derivatives in forward mode are not carried: a result without one would count as a derivative of zero.
void refuse_tangents(const at::Tensor& t) { need(!t._fw_grad(/*level=*/0).defined(), "no derivatives in forward mode"); }

// A trace would have the result as a constant: it records what goes through torch's dispatcher.
void refuse_tracing() {
  need(!torch::jit::tracer::isTracing() &&
           !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
       "a trace does not record this call");
}

struct TokenNode : public Node {
  SavedVariable ids, rng;
  bool has_ids, captured;
  double scale;
  int64_t padding, rows;
  Mask mask;
  at::ScalarType type;
  TokenNode(const Mask& m, double scale, const at::Tensor& of, const at::Device& dev)
      : has_ids(false), captured(captures(dev)), scale(scale), padding(HB_NO_PADDING), rows(0), mask(m), type(of.scalar_type()) {
    if (mask.rng.defined()) rng = SavedVariable(mask.rng, false);
    mask.rng = at::Tensor();
    set_next_edges(torch::autograd::collect_next_edges(of));
  }
  std::string name() const override { return has_ids ? "TokenEmbeddingBackward" : "TokenDropoutBackward"; }
  void release_variables() override {
    ids.reset_data();
    rng.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    const at::Tensor& g = grads[0];
    if (!g.defined()) return {at::Tensor()};
    need(!(at::GradMode::is_enabled() && g.requires_grad()), "the backward pass is not differentiated again");
    refuse_tangents(g);
    need(captured || !captures(g.device()), "the forward pass belongs to the capture that its backward pass is in");
    at::AutoGradMode none(false);
    Mask m = mask;
    m.rng = rng.unpack();
    if (!has_ids) return {run_dropout(g, scale, m, type, at::Tensor())};
    return {run_embedding_grad(GradInputs(ids.unpack(), g, rows), scale, padding, m, type, at::Tensor(), false)};
  }
};

at::Tensor with_history(at::Tensor out, const std::shared_ptr<TokenNode>& node) {
  torch::autograd::set_history(out, node);
  return out;
}

// embedding_autograd(weight, ids, scale, padding | None, p, seed, offset, rng | None, dtype | None)
PyObject* embedding_autograd(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 9, "embedding_autograd");
    const at::Tensor &weight = tensor(a[0], "weight"), &ids = tensor(a[1], "ids");
    const Mask mask(a + 4);
    const double scale = number(a[2]);
    const int64_t padding = padding_of(a[3]);
    const at::ScalarType type = type_or(a[8], weight.scalar_type());
    refuse_tracing();
    refuse_tangents(weight);
    const bool track = at::GradMode::is_enabled() && weight.requires_grad();
    if (track && ids.is_cuda()) refuse_foreign_graphs(weight, ids.device());
    at::Tensor out;
    {
      at::AutoGradMode none(false);
      out = run_embedding(weight, ids, scale, padding, mask, type, at::Tensor());
    }
    if (!track) return THPVariable_Wrap(out);
    need(weight.is_cuda(), "a weight with a gradient lies on the GPU");
    std::shared_ptr<TokenNode> node(new TokenNode(mask, scale, weight, ids.device()), torch::autograd::deleteNode);
    node->has_ids = true;
    node->ids = SavedVariable(ids, false);
    node->padding = padding;
    node->rows = weight.size(0);
    return THPVariable_Wrap(with_history(out, node));
  });
}

// dropout_autograd(x, scale, p, seed, offset, rng | None, dtype | None)
PyObject* dropout_autograd(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    arity(n_args, 7, "dropout_autograd");
    const at::Tensor& x = tensor(a[0], "x");
    const Mask mask(a + 2);
    const double scale = number(a[1]);
    refuse_tracing();
    refuse_tangents(x);
    const bool track = at::GradMode::is_enabled() && x.requires_grad();
    if (track && x.is_cuda()) refuse_foreign_graphs(x, x.device());
    at::Tensor out;
    {
      at::AutoGradMode none(false);
      out = run_dropout(x, scale, mask, type_or(a[6], x.scalar_type()), at::Tensor());
    }
    if (!track) return THPVariable_Wrap(out);
    std::shared_ptr<TokenNode> node(new TokenNode(mask, scale, x, x.device()), torch::autograd::deleteNode);
    return THPVariable_Wrap(with_history(out, node));
  });
}

PyObject* set_error_class(PyObject*, PyObject* cls) {
  Py_XINCREF(cls);
  Py_XSETREF(g_error, cls);
  Py_RETURN_NONE;
}

#define HB_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef g_methods[] = {
    {"lookup_fetch", HB_FAST(lookup_fetch), nullptr},
    {"unique_segsum", HB_FAST(unique_segsum), nullptr},
    {"unique_update", HB_FAST(unique_update), nullptr},
    {"index_lookup", HB_FAST(index_lookup), nullptr},
    {"index_add", HB_FAST(index_add), nullptr},
    {"staging_flush", HB_FAST(staging_flush), nullptr},
    {"step_forward", HB_FAST(step_forward), nullptr},
    {"step_backward", HB_FAST(step_backward), nullptr},
    {"embedding", HB_FAST(embedding), nullptr},
    {"dropout", HB_FAST(dropout), nullptr},
    {"embedding_grad", HB_FAST(embedding_grad), nullptr},
    {"embedding_grad_rows", HB_FAST(embedding_grad_rows), nullptr},
    {"embedding_autograd", HB_FAST(embedding_autograd), nullptr},
    {"dropout_autograd", HB_FAST(dropout_autograd), nullptr},
    {"set_error_class", set_error_class, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&g_module); }
