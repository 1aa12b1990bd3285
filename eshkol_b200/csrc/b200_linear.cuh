// What the linear layer's kernels share: activations and their slopes, and the epilogue of a sum.
#pragma once
#include "b200_elem.cuh"

namespace b200 {

// What becomes of a product's sums
struct LinEpilogue {
  const void *bias, *residual;
  void *out, *pre;
  long long ldo, ld_res, ld_pre;
  int M, N, act;
  int words;              // 1: out, pre and residual rows lie on 16-byte boundaries
  int pairs;              // 1: N is even and those rows lie on 4-byte boundaries (16-bit types)
};

// ------------------------------------------------------------------ activations
// Roundings are written out (no contraction left to the compiler), so that a forward result does not depend
// on which other results a call asks for.  (Which gradients are asked for decides how reductions are cut.)
template <bool kExact> __device__ __forceinline__ float logistic(float v) {
  if (kExact) return __fdiv_rn(1.f, __fadd_rn(1.f, expf(-v)));
  // a few 2^-22: below half a step of the 16-bit results
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(v, -1.4426950408889634f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.f, e)));
  return r;
}
constexpr float kGeluA = 0.7978845608028654f, kGeluB = 0.044715f;
// 2 u(z) = 2 A (z + B z^3)
__device__ __forceinline__ float gelu_argument(float z) {
  return __fmul_rn(z, __fmaf_rn(2.f * kGeluA * kGeluB, __fmul_rn(z, z), 2.f * kGeluA));
}
// 0 none, 1 ReLU, 2 the tanh form of GELU: z (1 + tanh u) / 2 = z logistic(2 u)
template <bool kExact> __device__ __forceinline__ float activate(float z, int act) {
  if (act == 1) return z > 0.f ? z : 0.f;
  if (act == 2) return __fmul_rn(z, logistic<kExact>(gelu_argument(z)));
  return z;
}
// kV elements of a row: bias, activation, residual, the two results
template <typename T, int kV>
__device__ __forceinline__ void finish_elements(const LinEpilogue& e, const float (&acc)[kV], const float (&bias)[kV],
                                                const Pack<T, kV>& res, Pack<T, kV>& y, Pack<T, kV>& pre) {
  constexpr bool kExact = sizeof(T) == 4;
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const float z = __fadd_rn(acc[j], bias[j]);
    float a = activate<kExact>(z, e.act);
    if (e.residual) a = __fadd_rn(a, Elem<T>::widen(res.v[j]));
    pre.v[j] = Elem<T>::narrow(z);
    y.v[j] = Elem<T>::narrow(a);
  }
}
template <typename T> __device__ __forceinline__ float bias_at(const LinEpilogue& e, int c) {
  return (e.bias && c < e.N) ? Elem<T>::widen(static_cast<const T*>(e.bias)[c]) : 0.f;
}

// act'(z) of a pair.  GELU, with s the logistic function of 2 u(z): s + s (1 - s) z 2 u'(z); z^2 is capped at
// 10^6, where s is 0 or 1 for long, so that nothing overflows on the way.
template <bool kExact> __device__ __forceinline__ Duo<float> slope_pair(Duo<float> z, int act) {
  if (act == 1) return Duo<float>::of(z.lo() > 0.f ? 1.f : 0.f, z.hi() > 0.f ? 1.f : 0.f);
  Duo<float> z2 = z * z;
  z2 = Duo<float>::of(fminf(z2.lo(), 1e6f), fminf(z2.hi(), 1e6f));
  const Duo<float> arg = z * fma2(both(2.f * kGeluA * kGeluB), z2, both(2.f * kGeluA));
  const Duo<float> du = fma2(both(6.f * kGeluA * kGeluB), z2, both(2.f * kGeluA));
  const Duo<float> s = Duo<float>::of(logistic<kExact>(arg.lo()), logistic<kExact>(arg.hi()));
  const Duo<float> t = fma2(s * both(-1.f), s, s);  // s (1 - s)
  return fma2(t * z, du, s);
}

// ------------------------------------------------------------------ few rows (b200_linear_small.cu)
// out[r][n] = sum over k of a[r][k] W(k, n) for a few rows, with the epilogue e; a is multiplied by the
// activation's slope at `pre` where `slope` names one.
struct SmallRows {
  LinEpilogue e;
  const void *a, *pre, *w;
  long long lda, ld_pre, ldw, K;
  int k_contiguous;  // 1: W is stored [N][K], 0: [K][N]
  int slope;
};
template <typename T> constexpr int kSmallRows = sizeof(T) == 4 ? 16 : 8;
// Rows up to which this beats the tensor cores, measured on 134 MB of weights.  f32, whose weights would be
// split first: 65 us (K-contiguous: 112) at 16 rows against 105.  16-bit: 39 us at 4 rows (53) against 41,
// but on rows off the 16-byte boundaries, which would be packed first, 68 us (113) at 8 rows against 86.
template <typename T> inline bool few_rows(long long rows, const void* w, long long ldw, bool k_contiguous) {
  if (sizeof(T) == 4) return rows <= (k_contiguous ? 12 : 16);
  if (rows_on_16_bytes<T>(w, ldw)) return rows <= (k_contiguous ? 2 : 4);
  return rows <= (k_contiguous ? 4 : 8);
}
template <typename T> int launch_small_rows(const SmallRows& q, cudaStream_t st);  // launches, or -1
cudaError_t linear_small_set_attributes();

}  // namespace b200
