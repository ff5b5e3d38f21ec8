"""The streams that work beside a call runs on (csrc/aside.cuh), compiled for the host over a runtime that writes down which
piece of work waits for which: calls on different streams of a caller's never wait for one another."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include <utility>
#include "aside.cuh"

// A stream or an event: the pieces of work that what comes next on it, or what waits for it, comes behind.
struct Behind { std::set<int> work; unsigned long long id = 0; };
static int g_device = 0, g_streams = 0, g_destroyed = 0;
static unsigned long long g_ids = 100;
static bool g_no_streams = false, g_relaxed = true;
static cudaStreamCaptureMode g_mode = cudaStreamCaptureModeGlobal;
static Behind* at(void* p) { return static_cast<Behind*>(p); }

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = g_device; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaStreamGetId(cudaStream_t s, unsigned long long* id) { *id = at(s)->id; return cudaSuccess; }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) {
  if (g_no_streams) return cudaErrorUnknown;
  g_relaxed &= g_mode == cudaStreamCaptureModeRelaxed;
  ++g_streams;
  Behind* b = new Behind;
  b->id = ++g_ids;
  *s = reinterpret_cast<cudaStream_t>(b);
  return cudaSuccess;
}
cudaError_t cudaStreamDestroy(cudaStream_t s) { ++g_destroyed; delete at(s); return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { *e = reinterpret_cast<cudaEvent_t>(new Behind); return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t e) { delete at(e); return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { at(e)->work = at(s)->work; return cudaSuccess; }
cudaError_t cudaStreamWaitEvent(cudaStream_t s, cudaEvent_t e, unsigned) {
  at(s)->work.insert(at(e)->work.begin(), at(e)->work.end());
  return cudaSuccess;
}
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) { std::swap(*m, g_mode); return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* c) { *c = cudaStreamCaptureStatusNone; return cudaSuccess; }
}

static int g_work = 0;
static int launch(cudaStream_t s) { at(s)->work.insert(++g_work); return g_work; }

// A call: something on the caller's stream, zeros beside it, something behind both.
struct Call { bool beside; int front, zeros, back; };
static Call call(cudaStream_t s) {
  Call c{};
  hb::Aside aside;
  c.front = launch(s);
  c.beside = aside.fork(s);
  if (c.beside) c.zeros = launch(aside.stream());
  aside.join();
  if (c.beside && !at(s)->work.count(c.zeros)) std::printf("joined too early\n"), std::exit(1);
  c.back = launch(s);
  return c;
}
static cudaStream_t stream() {
  Behind* b = new Behind;
  b->id = ++g_ids;
  return reinterpret_cast<cudaStream_t>(b);
}
#define EXPECT(x) do { if (!(x)) { std::printf("%d: " #x "\n", __LINE__); return 1; } } while (0)

int main() {
  g_no_streams = true;
  cudaStream_t a = stream(), b = stream();
  EXPECT(!call(a).beside && g_mode == cudaStreamCaptureModeGlobal);
  g_no_streams = false;
  // two streams in turns: none of one's work comes behind the other's
  std::set<int> of_a, of_b;
  for (int turn = 0; turn < 3; ++turn) {
    Call c = call(a), d = call(b);
    EXPECT(c.beside && d.beside);
    of_a.insert({c.front, c.zeros, c.back});
    of_b.insert({d.front, d.zeros, d.back});
  }
  for (int w : of_b) EXPECT(!at(a)->work.count(w));
  for (int w : of_a) EXPECT(!at(b)->work.count(w));
  EXPECT(g_streams == 2);
  // the same handle on another device, and as another stream's that was created later
  g_device = 1;
  EXPECT(call(a).beside && g_streams == 3);
  g_device = 0;
  at(a)->id = ++g_ids;
  at(a)->work.clear();
  EXPECT(call(a).beside && g_streams == 4);
  for (int w : of_a) EXPECT(!at(a)->work.count(w));
  // more streams than a thread keeps any for
  int without = 0;
  for (int k = 0; k < 100; ++k) without += !call(stream()).beside;
  EXPECT(without == 100 - (g_streams - 4) && g_streams == 64 && call(b).beside && g_streams == 64);
  // streams are made in a mode that no other thread's capture minds
  EXPECT(g_relaxed && g_mode == cudaStreamCaptureModeGlobal && g_destroyed == 0);
  return 0;
}
"""


def test_calls_on_two_streams_do_not_wait_for_one_another(tmp_path):
    (tmp_path / "aside.cpp").write_text(PROGRAM)
    exe = tmp_path / "aside"
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", str(ROOT / "include"), "-I", str(ROOT / "hades_b200" / "csrc"),
                    "-I", "/usr/local/cuda/include", str(tmp_path / "aside.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
