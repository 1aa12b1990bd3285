// Scratch memory of the training and serving operators.
#include <stdio.h>

#include "b200_elem.cuh"
#include "b200_tiers.h"

namespace b200 {
namespace {
std::mutex g_mu;  // guards the block, and the launches of the call that uses it
uint8_t* g_block = nullptr;
size_t g_bytes = 0;
}  // namespace

uint8_t* OpScratch::reserve(size_t bytes, cudaStream_t st) {
  if (bytes == 0) bytes = 16;
  hold_ = std::unique_lock<std::mutex>(g_mu);
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &status) != cudaSuccess || status == cudaStreamCaptureStatusInvalidated) {
    fprintf(stderr, "[eshkol-b200] the library stream cannot be used: %s\n", cudaGetErrorString(cudaGetLastError()));
    return nullptr;
  }
  if (status == cudaStreamCaptureStatusActive) {
    // an allocation node and, in release(), its free node: memory of the captured graph itself
    if (cudaMallocAsync(&captured_, bytes, st) != cudaSuccess) {
      captured_ = nullptr;
      fprintf(stderr, "[eshkol-b200] captured scratch of %zu bytes failed: %s\n", bytes,
              cudaGetErrorString(cudaGetLastError()));
      return nullptr;
    }
    st_ = st;
    return static_cast<uint8_t*>(captured_);
  }
  if (bytes > g_bytes) {
    // the block may still be in use by kernels of the library's stream
    if (cudaStreamSynchronize(st) != cudaSuccess) {
      fprintf(stderr, "[eshkol-b200] stream failed: %s\n", cudaGetErrorString(cudaGetLastError()));
      return nullptr;
    }
    if (g_block) eshkol_b200_mem_free(0, g_block);
    g_block = nullptr;
    g_bytes = 0;
    void* p = nullptr;
    if (eshkol_b200_mem_alloc(0, bytes, &p) != 0) {
      fprintf(stderr, "[eshkol-b200] scratch allocation of %zu bytes failed\n", bytes);
      return nullptr;
    }
    g_block = static_cast<uint8_t*>(p);
    g_bytes = bytes;
  }
  return g_block;
}

int OpScratch::release() {
  if (!captured_) return 0;
  void* p = captured_;
  captured_ = nullptr;
  if (cudaFreeAsync(p, st_) != cudaSuccess) {
    fprintf(stderr, "[eshkol-b200] captured scratch was not freed: %s\n", cudaGetErrorString(cudaGetLastError()));
    return -1;
  }
  return 0;
}

size_t op_scratch_bytes() {
  const std::lock_guard<std::mutex> lock(g_mu);
  return g_bytes;
}

void op_scratch_shutdown() {
  const std::lock_guard<std::mutex> lock(g_mu);
  if (g_block) cudaFree(g_block);
  g_block = nullptr;
  g_bytes = 0;
}

}  // namespace b200
