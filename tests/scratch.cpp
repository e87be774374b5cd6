// Runs scratch.cuh against a stand-in for the CUDA runtime: addresses without memory behind them, a limit, and streams that can be
// capturing.  One scenario per run; exit status 0: it held.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>
#include <thread>

#include "../ruai_b200/csrc/scratch.cuh"

#define CHECK(c)                                                     \
  do {                                                               \
    if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); std::exit(1); } \
  } while (0)

namespace fake {
std::mutex lock;
std::map<char*, size_t> memory;  // what the driver has handed out
std::map<char*, size_t> zeroed;
size_t limit = ~(size_t)0, used = 0;
bool capturing = false;
std::atomic<int> device_waits{0};
char* next = (char*)0x1000000;
bool has(const void* p, size_t bytes) {
  auto it = memory.find((char*)p);
  return it != memory.end() && it->second >= bytes;
}
}  // namespace fake

extern "C" {
cudaError_t cudaMalloc(void** out, size_t bytes) {
  std::lock_guard<std::mutex> g(fake::lock);
  if (fake::used + bytes > fake::limit) return cudaErrorMemoryAllocation;
  fake::memory[fake::next] = bytes;
  fake::used += bytes;
  *out = fake::next;
  fake::next += (bytes + 4095) / 4096 * 4096;
  return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
  std::lock_guard<std::mutex> g(fake::lock);
  if (!p) return cudaSuccess;
  auto it = fake::memory.find((char*)p);
  if (it == fake::memory.end()) { std::printf("freed twice\n"); std::exit(1); }
  fake::used -= it->second;
  fake::memory.erase(it);
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* p, int, size_t bytes, cudaStream_t) {
  if (!fake::has(p, bytes)) { std::printf("cleared what is not allocated\n"); std::exit(1); }
  fake::zeroed[(char*)p] = bytes;
  return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t) { return fake::capturing ? cudaErrorStreamCaptureUnsupported : cudaSuccess; }
cudaError_t cudaDeviceSynchronize(void) { ++fake::device_waits; return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* st) {
  *st = fake::capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
}

constexpr size_t MB = 1 << 20;
cudaStream_t const kStream = (cudaStream_t)16;

struct Held : Scratch {  // a context's
  Held() { CHECK(scratch::grow(*this, kStream, 10 * MB, 4096) == cudaSuccess); }
  ~Held() { scratch::release(*this); }
  bool sound() const { return fake::has(partial, partial_bytes) && fake::has(counters, counters_n * sizeof(unsigned)) && partial_bytes >= 10 * MB && counters_n >= 4096; }
};

int main(int argc, char** argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  {
    Held s;
    CHECK(s.sound());
    float* const p = s.partial;
    unsigned* const n = s.counters;
    const unsigned long long epoch = s.scratch_epoch;
    if (what == "grows") {
      CHECK(scratch::grow(s, kStream, 10 * MB, 4096) == cudaSuccess && s.partial == p && s.scratch_epoch == epoch);
      CHECK(scratch::grow(s, kStream, 30 * MB, 9000) == cudaSuccess && s.sound() && s.partial_bytes >= 30 * MB && s.counters_n >= 9000);
      CHECK(s.scratch_epoch > epoch && !fake::has(p, 1) && !fake::has(n, 1) && fake::zeroed[(char*)s.counters] == s.counters_n * sizeof(unsigned));
    } else if (what == "out of memory") {
      fake::limit = fake::used + 5 * MB;  // neither both blocks nor the new one by itself
      CHECK(scratch::grow(s, kStream, 40 * MB, 0) == cudaErrorMemoryAllocation);
      CHECK(s.sound() && s.partial_bytes == 10 * MB);
      CHECK(scratch::grow(s, kStream, 8 * MB, 4096) == cudaSuccess && s.sound());
    } else if (what == "out of memory for both") {
      fake::limit = fake::used + 5 * MB;
      CHECK(scratch::grow(s, kStream, 14 * MB, 0) == cudaSuccess && s.sound() && s.partial_bytes == 14 * MB && s.scratch_epoch > epoch);
    } else if (what == "out of memory and kept for a graph") {
      s.partial_in_graph = true;
      fake::limit = fake::used + 5 * MB;
      CHECK(scratch::grow(s, kStream, 14 * MB, 0) == cudaErrorMemoryAllocation && s.sound() && s.partial == p && s.scratch_epoch == epoch);
    } else if (what == "out of memory for counters") {
      fake::limit = fake::used;
      CHECK(scratch::grow(s, kStream, 0, 1 << 20) == cudaErrorMemoryAllocation && s.sound() && s.counters == n && s.scratch_epoch == epoch);
    } else if (what == "in a capture") {
      fake::capturing = true;
      CHECK(scratch::grow(s, kStream, 10 * MB, 4096) == cudaSuccess);  // nothing to do
      CHECK(scratch::grow(s, kStream, 11 * MB, 0) != cudaSuccess && scratch::grow(s, kStream, 0, 5000) != cudaSuccess);
      CHECK(s.sound() && s.partial == p && s.counters == n && s.scratch_epoch == epoch);
      fake::capturing = false;
    } else if (what == "kept for a graph") {
      s.partial_in_graph = s.counters_in_graph = true;
      CHECK(scratch::grow(s, kStream, 30 * MB, 9000) == cudaSuccess && s.sound() && s.partial != p && s.counters != n);
      CHECK(fake::has(p, 10 * MB) && fake::has(n, 4096 * sizeof(unsigned)));
      fake::zeroed.clear();
      scratch::clear_counters(s, kStream);
      CHECK(fake::zeroed.size() == 2 && fake::zeroed[(char*)n] == 4096 * sizeof(unsigned) && fake::zeroed[(char*)s.counters] == s.counters_n * sizeof(unsigned));
    } else if (what == "kept only if captured") {
      s.partial_in_graph = s.counters_in_graph = true;
      CHECK(scratch::grow(s, kStream, 30 * MB, 9000) == cudaSuccess);
      float* const p2 = s.partial;  // no graph has seen these two
      unsigned* const n2 = s.counters;
      CHECK(scratch::grow(s, kStream, 90 * MB, 30000) == cudaSuccess && s.sound());
      CHECK(fake::has(p, 10 * MB) && fake::has(n, 4096 * sizeof(unsigned)) && !fake::has(p2, 1) && !fake::has(n2, 1));
    } else if (what == "rising little by little") {
      size_t most = 0;
      for (size_t want = 11 * MB; want < 300 * MB; want += MB) {
        s.partial_in_graph = s.counters_in_graph = true;  // captured every time
        CHECK(scratch::grow(s, kStream, want, want / 4096) == cudaSuccess && s.sound() && s.partial_bytes >= want);
        most = s.partial_bytes;
      }
      CHECK(most <= 450 * MB && s.scratch_epoch - epoch <= 25 && fake::used <= 3 * most + 2 * MB);
    } else if (what == "half as much again does not fit") {
      fake::limit = fake::used + 12 * MB;
      CHECK(scratch::grow(s, kStream, 11 * MB, 0) == cudaSuccess && s.sound() && s.partial_bytes == 11 * MB);
    } else if (what == "held by another thread") {
      std::thread other;
      {
        const ScratchLock held(s.scratch_lock);
        CHECK(scratch::grow(s, kStream, 12 * MB, 0) == cudaSuccess);  // by the one that holds it, at once
        float* const p2 = s.partial;
        other = std::thread([&] { CHECK(scratch::grow(s, kStream, 60 * MB, 9000) == cudaSuccess); });
        std::this_thread::sleep_for(std::chrono::milliseconds(100));
        CHECK(s.partial == p2 && s.counters == n && fake::has(p2, 12 * MB) && s.sound());
      }
      other.join();
      CHECK(s.sound() && s.partial_bytes >= 60 * MB && s.counters_n >= 9000);
    } else if (what == "no wait for the device during a capture") {
      CHECK(block_pool::attach(&s, 0, kStream));
      void* q = nullptr;
      CHECK(block_pool::allocate(0, 5000, &q) == cudaSuccess && block_pool::give_back(0, kStream, q) == cudaSuccess && fake::device_waits == 0);
      std::thread other;
      {
        const std::lock_guard<std::recursive_mutex> captures(block_pool::of(0).device_wide);
        other = std::thread([] { CHECK(block_pool::settle(block_pool::of(0))); });
        std::this_thread::sleep_for(std::chrono::milliseconds(100));
        CHECK(fake::device_waits == 0);
      }
      other.join();
      CHECK(fake::device_waits == 1);
      block_pool::detach(&s, 0);
    } else {
      std::printf("no such scenario: %s\n", what.c_str());
      return 1;
    }
  }
  CHECK(fake::used == 0);  // all of it went with the context
  return 0;
}
