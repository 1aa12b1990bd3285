// Element types of the training and serving operators: storage types f64, f32, f16 and bf16 (the
// dispatcher's dtype tags), the type their sums are held in (f64 for f64, else f32), and vectors of
// 16 bytes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

template <typename T> struct Elem;
template <> struct Elem<double> {
  using Acc = double;
  static __device__ __forceinline__ double widen(double v) { return v; }
  static __device__ __forceinline__ double narrow(double v) { return v; }
};
template <> struct Elem<float> {
  using Acc = float;
  static __device__ __forceinline__ float widen(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <> struct Elem<__half> {
  using Acc = float;
  static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
  using Acc = float;
  static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
};

// kV consecutive elements as they lie in memory (kV = 1, or 16 bytes' worth)
template <typename T, int kV> struct alignas(sizeof(T) * kV) Pack {
  T v[kV];
};

template <typename T> constexpr int kVec16 = 16 / static_cast<int>(sizeof(T));

// elements between p and the 16-byte boundary at or before it
template <typename T> __host__ __device__ __forceinline__ int elems_past_boundary(const T* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

__device__ __forceinline__ float sum_rsqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double sum_rsqrt(double v) { return 1.0 / sqrt(v); }

// every lane gets the sum over the warp (the same tree on every lane)
template <typename A> __device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// every thread of the block gets both sums; sm holds 2 * 32 values and may be reused after the
// next barrier
template <typename A> __device__ __forceinline__ void block_sum2(A& a, A& b, A* sm, int warps) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (warps == 1) return;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) { sm[w] = a; sm[32 + w] = b; }
  __syncthreads();
  // the partial sums are added by shuffles, the same tree in every warp
  a = warp_sum(lane < warps ? sm[lane] : A(0));
  b = warp_sum(lane < warps ? sm[32 + lane] : A(0));
}

// A device pointer's alignment and a row pitch both a multiple of 16 bytes
template <typename T> inline bool rows_on_16_bytes(const void* p, long long ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * static_cast<long long>(sizeof(T))) % 16 == 0;
}

// Makes the library's device current for one call and puts the caller's back.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess) return;
    if (now == device) { ok_ = true; return; }
    ok_ = cudaSetDevice(device) == cudaSuccess;
    if (ok_) back_ = now;
  }
  ~DeviceScope() { if (back_ >= 0) cudaSetDevice(back_); }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  bool ok() const { return ok_; }

 private:
  int back_ = -1;
  bool ok_ = false;
};

// Scratch of one operator call (b200_scratch.cu).  Outside a capture: a grow-only block of the
// library, ordered by the library's stream.  While the library's stream is captured: stream-ordered
// allocation nodes, so every graph owns its scratch and two graphs never share any.
class OpScratch {
 public:
  ~OpScratch() { release(); }
  uint8_t* reserve(size_t bytes, cudaStream_t st);  // nullptr on failure (a message is printed)
  int release();                                    // ends the use; -1 when the free node failed

 private:
  void* captured_ = nullptr;
  cudaStream_t st_ = nullptr;
};
void op_scratch_shutdown();

}  // namespace b200
