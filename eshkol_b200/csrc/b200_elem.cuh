// Element types of the training and serving operators: storage types f64, f32, f16 and bf16 (the
// dispatcher's dtype tags), the type their sums are held in (f64 for f64, else f32), and vectors of
// 16 bytes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

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

// ------------------------------------------------------------------ two values at a time
// f32 pairs go through the packed f32x2 instructions (one issue slot for two additions, products or fused
// multiply-adds, each rounded as its scalar form); f64 pairs are two scalars.
template <typename A> struct Duo;
template <> struct Duo<float> {
  unsigned long long v;
  static __device__ __forceinline__ Duo of(float x, float y) {
    Duo r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
  }
  __device__ __forceinline__ float lo() const {
    float x;
    asm("mov.b64 {%0, _}, %1;" : "=f"(x) : "l"(v));
    return x;
  }
  __device__ __forceinline__ float hi() const {
    float y;
    asm("mov.b64 {_, %0}, %1;" : "=f"(y) : "l"(v));
    return y;
  }
};
template <> struct Duo<double> {
  double x, y;
  static __device__ __forceinline__ Duo of(double a, double b) { return Duo{a, b}; }
  __device__ __forceinline__ double lo() const { return x; }
  __device__ __forceinline__ double hi() const { return y; }
};
template <typename A> __device__ __forceinline__ Duo<A> both(A x) { return Duo<A>::of(x, x); }
__device__ __forceinline__ Duo<float> operator+(Duo<float> a, Duo<float> b) {
  Duo<float> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Duo<float> operator*(Duo<float> a, Duo<float> b) {
  Duo<float> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Duo<float> fma2(Duo<float> a, Duo<float> b, Duo<float> c) {
  Duo<float> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Duo<double> operator+(Duo<double> a, Duo<double> b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Duo<double> operator*(Duo<double> a, Duo<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Duo<double> fma2(Duo<double> a, Duo<double> b, Duo<double> c) {
  return {fma(a.x, b.x, c.x), fma(a.y, b.y, c.y)};
}
template <typename A> __device__ __forceinline__ A total(Duo<A> a) { return a.lo() + a.hi(); }

// sixteen bytes as pairs in the stat type, and back with one rounding
template <typename T> using Word = Pack<T, kVec16<T>>;
template <typename T> constexpr int kDuos = kVec16<T> / 2;
__device__ __forceinline__ void widen_word(const Word<double>& p, Duo<double> (&d)[1]) { d[0] = {p.v[0], p.v[1]}; }
__device__ __forceinline__ void widen_word(const Word<float>& p, Duo<float> (&d)[2]) {
  d[0] = Duo<float>::of(p.v[0], p.v[1]);
  d[1] = Duo<float>::of(p.v[2], p.v[3]);
}
__device__ __forceinline__ void widen_word(const Word<__half>& p, Duo<float> (&d)[4]) {
  const __half2* h = reinterpret_cast<const __half2*>(&p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    d[i] = Duo<float>::of(f.x, f.y);
  }
}
__device__ __forceinline__ void widen_word(const Word<__nv_bfloat16>& p, Duo<float> (&d)[4]) {
  const uint4 w = *reinterpret_cast<const uint4*>(&p);  // a bf16 is the upper half of its f32
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = Duo<float>::of(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
__device__ __forceinline__ Word<double> narrow_word(const Duo<double> (&d)[1]) {
  Word<double> p;
  p.v[0] = d[0].x; p.v[1] = d[0].y;
  return p;
}
__device__ __forceinline__ Word<float> narrow_word(const Duo<float> (&d)[2]) {
  Word<float> p;
  p.v[0] = d[0].lo(); p.v[1] = d[0].hi(); p.v[2] = d[1].lo(); p.v[3] = d[1].hi();
  return p;
}
template <typename T> __device__ __forceinline__ Word<T> narrow_word(const Duo<float> (&d)[4]) {
  Word<T> p;
  if constexpr (sizeof(T) == 2) {
    uint32_t* u = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(d[i].hi()), "f"(d[i].lo()));
      else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(d[i].hi()), "f"(d[i].lo()));
    }
  }
  return p;
}
template <typename T, int kD> __device__ __forceinline__ Word<T> to_word(const Duo<typename Elem<T>::Acc> (&d)[kD]) {
  if constexpr (sizeof(T) == 2) return narrow_word<T>(d);
  else return narrow_word(d);
}

// How the rows of a matrix may be accessed: in words of 16 bytes, (16-bit types) in pairs, one by one
enum Access : int { kSingly = 0, kInPairs = 1, kInWords = 2 };

// Sixteen bytes' worth of a row of n elements from element c, `otherwise` outside.  A word that does not lie
// whole in the row goes element by element; pairs imply an even n.
template <typename T> __device__ __forceinline__ Word<T> read_word(const T* row, int c, int n, int access, T otherwise) {
  constexpr int kV = kVec16<T>;
  if (access == kInWords && c + kV <= n) return *reinterpret_cast<const Word<T>*>(row + c);
  Word<T> p;
  if (sizeof(T) == 2 && access == kInPairs) {
#pragma unroll
    for (int j = 0; j < kV; j += 2) {
      Pack<T, 2> q;
      q.v[0] = q.v[1] = otherwise;
      if (c + j < n) q = *reinterpret_cast<const Pack<T, 2>*>(row + c + j);
      p.v[j] = q.v[0];
      p.v[j + 1] = q.v[1];
    }
    return p;
  }
#pragma unroll
  for (int j = 0; j < kV; ++j) p.v[j] = c + j < n ? row[c + j] : otherwise;
  return p;
}
template <typename T> __device__ __forceinline__ void write_word(T* row, int c, int n, int access, const Word<T>& p) {
  constexpr int kV = kVec16<T>;
  if (access == kInWords && c + kV <= n) {
    *reinterpret_cast<Word<T>*>(row + c) = p;
    return;
  }
  if (sizeof(T) == 2 && access == kInPairs) {
#pragma unroll
    for (int j = 0; j < kV; j += 2)
      if (c + j < n) {
        Pack<T, 2> q;
        q.v[0] = p.v[j];
        q.v[1] = p.v[j + 1];
        *reinterpret_cast<Pack<T, 2>*>(row + c + j) = q;
      }
    return;
  }
#pragma unroll
  for (int j = 0; j < kV; ++j)
    if (c + j < n) row[c + j] = p.v[j];
}

// elements between p and the 16-byte boundary at or before it
template <typename T> __host__ __device__ __forceinline__ int elems_past_boundary(const T* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
}

__device__ __forceinline__ float inverse_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return rsqrt(v); }

// every lane gets the sum over the warp (the same tree on every lane)
template <typename A> __device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Every thread of the block gets the sum, or both sums.  sm (32 or 64 values) may be written again by a
// reduction that has another block-wide reduction or barrier between itself and this one: callers
// alternate between two arrays, which leaves one barrier per reduction.
template <typename A> __device__ __forceinline__ A block_sum(A a, A* sm, int warps) {
  a = warp_sum(a);
  if (warps == 1) return a;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sm[w] = a;
  __syncthreads();
  return warp_sum(lane < warps ? sm[lane] : A(0));
}
template <typename A> __device__ __forceinline__ void block_sum2(A& a, A& b, A* sm, int warps) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, at = lane & 15;
  // the lower half of the warp goes on with a, the upper half with b: half the shuffles
  A v = (half ? b : a) + __shfl_xor_sync(0xffffffffu, half ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps > 1) {
    if (at == 0) sm[half * 32 + w] = v;
    __syncthreads();
    v = (at < warps ? sm[half * 32 + at] : A(0)) + (at + 16 < warps ? sm[half * 32 + at + 16] : A(0));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  a = __shfl_sync(0xffffffffu, v, 0);
  b = __shfl_sync(0xffffffffu, v, 16);
}

// Copies from global to shared memory that a thread waits for by itself (cp.async): 16 bytes, or one
// element of 4 or 8
__device__ __forceinline__ void copy_async16(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(shared))), "l"(global) : "memory");
}
template <int kBytes> __device__ __forceinline__ void copy_async_small(void* shared, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(shared))), "l"(global), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void wait_async() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Launches of one operator that follow one another (launch_after): the next kernel's blocks may come to the
// SMs as soon as all blocks of the one before have called let_next_start, and wait in after_previous, before
// they touch global memory, until that kernel is complete and its writes are visible.  That hides the start of the
// launch, 1 to 2 us.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
inline cudaLaunchAttribute after_attribute() {
  cudaLaunchAttribute a;
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}
template <typename... Params, typename... Args>
inline cudaError_t launch_after(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t shared, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cudaLaunchAttribute attr = after_attribute();
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// How a row's words get from memory to the threads that work on them, some rows ahead: in registers, or
// through shared memory in copies of words or of elements (16-bit ones in pairs: an asynchronous copy moves
// four bytes at least, so their rows must be even in length and lie on 4-byte boundaries)
enum Ahead : int { kInRegisters = 0, kByWords = 1, kByElements = 2 };
template <typename T> inline bool rows_by_elements(const void* p, long long ld, long long n) {
  return sizeof(T) >= 4 || ((reinterpret_cast<uintptr_t>(p) & 3u) == 0 && ld % 2 == 0 && n % 2 == 0);
}
// starts the copy of the word at element c < n of a row into this thread's place
template <typename T, int kHow> __device__ __forceinline__ void copy_word(Word<T>* place, const T* row, int c, int n) {
  if constexpr (kHow == kByWords) {
    copy_async16(place, row + c);
  } else {
    constexpr int kStep = sizeof(T) >= 4 ? 1 : 2;
#pragma unroll
    for (int j = 0; j < kVec16<T>; j += kStep)
      if (c + j < n) copy_async_small<sizeof(T) * kStep>(&place->v[j], row + c + j);
  }
}
// the copied word, `zero` behind the row
template <typename T, int kHow> __device__ __forceinline__ Word<T> take_word(const Word<T>* place, int c, int n, T zero) {
  Word<T> p;
  if (kHow == kByWords ? c < n : c + kVec16<T> <= n) return *place;
#pragma unroll
  for (int j = 0; j < kVec16<T>; ++j) p.v[j] = (kHow == kByElements && c + j < n) ? place->v[j] : zero;
  return p;
}
// read_word and write_word where kByWords promises that every word is aligned and whole, c < n
template <typename T, int kHow> __device__ __forceinline__ Word<T> get_word(const T* row, int c, int n, int access, T otherwise) {
  if constexpr (kHow == kByWords) return *reinterpret_cast<const Word<T>*>(row + c);
  else return read_word(row, c, n, access, otherwise);
}
template <typename T, int kHow> __device__ __forceinline__ void put_word(T* row, int c, int n, int access, const Word<T>& p) {
  if constexpr (kHow == kByWords) *reinterpret_cast<Word<T>*>(row + c) = p;
  else write_word(row, c, n, access, p);
}

// A device pointer's alignment and a row pitch both a multiple of 16 bytes
template <typename T> inline bool rows_on_16_bytes(const void* p, long long ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * static_cast<long long>(sizeof(T))) % 16 == 0;
}

template <typename T> inline int row_access(const void* p, long long ld, long long n) {
  return rows_on_16_bytes<T>(p, ld) ? kInWords : sizeof(T) == 2 && rows_by_elements<T>(p, ld, n) ? kInPairs : kSingly;
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
// The order of the stream protects the block only if one call's launches follow one another, and the block
// may be replaced by a larger one: from reserve() to the end of its call an OpScratch holds a lock, and
// calls of other host threads that need scratch wait for it (a few launches long).
class OpScratch {
 public:
  ~OpScratch() { release(); }
  uint8_t* reserve(size_t bytes, cudaStream_t st);  // nullptr on failure (a message is printed)
  int release();                                    // ends the use; -1 when the free node failed

 private:
  std::unique_lock<std::mutex> hold_;  // until destruction, after the call's last launch
  void* captured_ = nullptr;
  cudaStream_t st_ = nullptr;
};
void op_scratch_shutdown();
size_t op_scratch_bytes();

}  // namespace b200
