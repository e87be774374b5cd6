// A context's scratch: what a launch leaves for the next one or for its own last CTAs (partial sums, pieces of operands, parts of outputs), and
// arrival counters, zero between launches.  Host code that needs nothing but the CUDA runtime's interface, so that it can be run against
// a stand-in for it.
#pragma once
#include <cuda_runtime_api.h>

#include <cstddef>
#include <mutex>
#include <new>

#include "block_pool.cuh"

struct Scratch {
  // Held from the reading of an address (or the growth) to the last launch that uses what it found: threads that step models of one
  // context share its stream too, and neither a block that goes nor another thread's launches may come between.  Taken before block_pool's locks.
  std::recursive_mutex scratch_lock;
  float* partial = nullptr;
  size_t partial_bytes = 0;
  unsigned* counters = nullptr;
  size_t counters_n = 0;
  unsigned long long scratch_epoch = 0;  // counts the changes of address: captured graphs hold them
  bool partial_in_graph = false, counters_in_graph = false;  // a caller's graph may hold the block's address: it is kept when it is outgrown
  struct Kept { void* p; size_t counter_bytes; Kept* next; }* kept_scratch = nullptr;
};

using ScratchLock = std::lock_guard<std::recursive_mutex>;

namespace scratch {

// What the scratch has outgrown, nothing on the stream uses it: freed, or kept for the graphs that write to it.  (Out of host memory it is
// left to the process's end.)
inline void outgrown(Scratch& s, void* p, size_t counter_bytes, bool in_graph) {
  if (!p) return;
  if (!in_graph) {
    (void)cudaFree(p);
    return;
  }
  if (Scratch::Kept* k = new (std::nothrow) Scratch::Kept{p, counter_bytes, s.kept_scratch}) s.kept_scratch = k;
}

// At least these; more by half than before, as long as memory holds it, since a new block is a wait for the stream, and a new capture of
// every model's decoding step: a caller whose sizes rise little by little (a long prompt in chunks) has a few of them, and what graphs keep
// of outgrown blocks is no more than three times the last.  After an error the scratch is as it was: the new block is there before the old one goes, and where memory holds
// them one at a time only, the old one comes back.
inline cudaError_t grow(Scratch& s, cudaStream_t stream, size_t partial_bytes, size_t counters) {
  const ScratchLock held(s.scratch_lock);
  if (partial_bytes <= s.partial_bytes && counters <= s.counters_n) return cudaSuccess;
  cudaError_t e = cudaStreamSynchronize(stream);  // fails in a capture, where nothing may be allocated
  if (e != cudaSuccess) return e;
  if (partial_bytes > s.partial_bytes) {
    void* p = nullptr;
    size_t got = s.partial_bytes + s.partial_bytes / 2;
    if (got < partial_bytes) got = partial_bytes;
    e = block_pool::device_malloc(&p, got);
    if (e == cudaErrorMemoryAllocation && got > partial_bytes) {
      (void)cudaGetLastError();
      e = cudaMalloc(&p, got = partial_bytes);
    }
    if (e == cudaErrorMemoryAllocation && s.partial && !s.partial_in_graph) {
      (void)cudaGetLastError();
      (void)cudaFree(s.partial);
      s.partial = nullptr;
      s.scratch_epoch++;
      e = cudaMalloc(&p, got = partial_bytes);
      if (e != cudaSuccess) {
        (void)cudaGetLastError();
        got = cudaMalloc(&p, s.partial_bytes) == cudaSuccess ? s.partial_bytes : 0;
        if (!got) p = nullptr;
      }
      s.partial = static_cast<float*>(p);
      s.partial_bytes = got;
      if (e != cudaSuccess) return e;
    } else if (e != cudaSuccess) {
      return e;
    } else {
      outgrown(s, s.partial, 0, s.partial_in_graph);
      s.partial = static_cast<float*>(p);
      s.partial_bytes = got;
      s.partial_in_graph = false;
      s.scratch_epoch++;
    }
  }
  if (counters > s.counters_n) {
    void* p = nullptr;
    if (counters < s.counters_n + s.counters_n / 2) counters = s.counters_n + s.counters_n / 2;
    e = cudaMalloc(&p, counters * sizeof(unsigned));
    if (e != cudaSuccess) return e;
    e = cudaMemsetAsync(p, 0, counters * sizeof(unsigned), stream);
    if (e != cudaSuccess) {
      (void)cudaFree(p);
      return e;
    }
    outgrown(s, s.counters, s.counters_n * sizeof(unsigned), s.counters_in_graph);
    s.counters = static_cast<unsigned*>(p);
    s.counters_n = counters;
    s.counters_in_graph = false;
    s.scratch_epoch++;
  }
  return cudaSuccess;
}

// A launch that gave up may have left some counted.
inline void clear_counters(Scratch& s, cudaStream_t stream) {
  const ScratchLock held(s.scratch_lock);
  if (s.counters) (void)cudaMemsetAsync(s.counters, 0, s.counters_n * sizeof(unsigned), stream);
  for (Scratch::Kept* k = s.kept_scratch; k; k = k->next)
    if (k->counter_bytes) (void)cudaMemsetAsync(k->p, 0, k->counter_bytes, stream);
}

inline void release(Scratch& s) {
  (void)cudaFree(s.partial);
  (void)cudaFree(s.counters);
  while (Scratch::Kept* k = s.kept_scratch) {
    s.kept_scratch = k->next;
    (void)cudaFree(k->p);
    delete k;
  }
  s.partial = nullptr;
  s.counters = nullptr;
  s.partial_bytes = s.counters_n = 0;
}

}  // namespace scratch
