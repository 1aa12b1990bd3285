// Layer normalisation with weight vectors, and its three gradients, on f64, f32, f16 and bf16 tensors.
//
//   y = (x - mean) r gamma + beta,  mean = sum x / D,  r = 1 / sqrt(sum (x - mean)^2 / D + epsilon)
//   with xhat = (x - mean) r and u = grad_out gamma:
//   grad_in    = r (u - sum u / D - xhat sum(u xhat) / D)
//   grad_gamma = sum over samples of grad_out xhat,   grad_beta = sum over samples of grad_out
//
// 2 (forward) or 3 (gradients) tensors cross HBM once: a row is held in registers from its one read to its
// one write, so the statistics are the two-pass ones (the mean first, then the deviations, with the
// deviations' own sum as a correction) at the traffic of one pass.  What bounds the kernels is instruction
// issue and the latency of a row's reductions: 8192 x 4096 bf16 takes 39 us (3.4 TB/s, 0.53 of the measured
// copy rate), its gradients at 16384 x 4096 87 us (4.6 TB/s, 0.71).  Sums, statistics and the weights'
// gradients are f32 (f64 for f64 tensors); a result is rounded to the storage type once.  Sums are combined in
// a fixed order: results do not depend on timing.
#include <math.h>
#include <stdio.h>

#include <cooperative_groups.h>

#include "b200_elem.cuh"
#include "b200_tiers.h"

namespace b200 {
namespace {
namespace cg = cooperative_groups;

// What the deviations are taken from, the pivot: the first places of the mean, at least 10 bits of it.  x minus
// it is exact for x up to 2^13 times it; from the whole mean all x of one binade would share a rounding, and
// with it the correction by the deviations' own sum (rows around zero: their mean off by 10^-6 instead of 10^-7).
// Where the mean is more than some 10^3 deviations the correction is larger than these, and taking its square from
// the mean square would cancel: such a row (off_too_far) takes its deviations once more, from the corrected mean,
// which they are so close to that the differences are exact again.
__device__ __forceinline__ float leading_bits(float v) { return __uint_as_float(__float_as_uint(v) & 0xffffe000u); }
__device__ __forceinline__ double leading_bits(double v) {
  return __longlong_as_double(__double_as_longlong(v) & ~0x3ffffffffffll);
}
template <typename A> __device__ __forceinline__ bool off_too_far(A off, A var) { return off * off > var; }
// The mean itself is the pivot and the correction, except where it is far below the deviations: the first sum,
// of entries of few bits, is then the more exact one (18000 f16 entries, mean of 2^-8 deviations: 10^-7 of the
// mean against 10^-6).
template <typename A> __device__ __forceinline__ A better_mean(A first, A corrected, A var) {
  return first * first * A(256) < var ? first : corrected;
}

struct NormArgs {
  const void *x, *gamma, *beta;
  void *y, *mean, *inv_std;
  long long rows, ldx, ldy;
  int n;
  int x_access, y_access, gamma_access, beta_access;
  double epsilon;
};

// ------------------------------------------------------------------ forward
// A row belongs to a warp, or to a block, whose threads hold kN words of 16 bytes each.  What a thread does
// once per row (its share of the reductions, the root, addresses) is some 150 instructions, an element of a
// bf16 row 21 in all (packed f32 arithmetic), so a thread gets four words where rows are many.  The next kAhead
// rows are on their way in shared memory: every thread copies the words that it will read itself.  Measured at
// 8192 x 4096 bf16: 128 threads with four words 39 us, 64 with eight 46, a warp with sixteen 53.
template <int kThreads, int kHow> constexpr int kNormAhead = kHow == kInRegisters ? 1 : kThreads == 1024 ? 2 : 4;

template <typename T, int kN, bool kWarp, int kThreads, int kHow>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 6 : kThreads == 256 ? 3 : 1) layernorm_kernel(const NormArgs a) {  // x and y may be the same
  using A = typename Elem<T>::Acc;
  using D = Duo<A>;
  constexpr int kV = kVec16<T>, kD = kDuos<T>, kAhead = kNormAhead<kThreads, kHow>;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ A sm1[32], sm2[64], sm3[64];
  constexpr int width = kWarp ? 32 : kThreads, warps = kWarp ? 1 : kThreads / 32, per_block = kWarp ? kThreads / 32 : 1;
  constexpr int kWritten = sizeof(T) == 8 ? 2 : 1;
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x, group = kWarp ? threadIdx.x >> 5 : 0;
  const int n = a.n;
  const T *gamma = static_cast<const T*>(a.gamma), *beta = static_cast<const T*>(a.beta);
  const A inv_n = A(1) / A(n), epsilon = static_cast<A>(a.epsilon);
  const T zero = Elem<T>::narrow(0), one = Elem<T>::narrow(1);
  const long long first = static_cast<long long>(blockIdx.x) * per_block + group;
  const long long step = static_cast<long long>(gridDim.x) * per_block;
  const T* in = static_cast<const T*>(a.x) + first * a.ldx;  // the next row to come
  T* out = static_cast<T*>(a.y) + first * a.ldy;
  const long long in_step = step * a.ldx, out_step = step * a.ldy;
  long long coming = first;
  Word<T>* ring = reinterpret_cast<Word<T>*>(dyn) + threadIdx.x;  // [stage][word of the row][thread]
  const auto fetch = [&](int stage) {
    if constexpr (kHow != kInRegisters) {
      if (coming < a.rows) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const int c = (t + i * width) * kV;
          if (c < n) copy_word<T, kHow>(ring + (stage * kN + i) * kThreads, in, c, n);
        }
      }
      commit_async();
      coming += step;
      in += in_step;
    }
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s) fetch(s);
  int stage = 0;
  for (long long r = first; r < a.rows; r += step) {
    D d[kN][kD];
    if constexpr (kHow != kInRegisters) {
      wait_async<kAhead - 1>();
#pragma unroll
      for (int i = 0; i < kN; ++i)
        widen_word(take_word<T, kHow>(ring + (stage * kN + i) * kThreads, (t + i * width) * kV, n, zero), d[i]);
      fetch(stage);
      stage = stage + 1 == kAhead ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) widen_word(read_word(in, (t + i * width) * kV, n, a.x_access, zero), d[i]);
      in += in_step;
    }
    D sum2[kD];
#pragma unroll
    for (int j = 0; j < kD; ++j) sum2[j] = d[0][j];
#pragma unroll
    for (int i = 1; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < kD; ++j) sum2[j] = sum2[j] + d[i][j];  // places behind the row hold zero
#pragma unroll
    for (int j = 1; j < kD; ++j) sum2[0] = sum2[0] + sum2[j];
    const A first_mean = block_sum(total(sum2[0]), sm1, warps) * inv_n;
    A off, var, mean = A(0), by = leading_bits(first_mean);
    // Once, or twice; the same for the whole row.  Written out twice for f64 alone: 60000 x 500 takes 100 us so
    // and 104 as a loop, but 8192 x 4096 bf16 in pairs 64 so, 53 as a loop (and 59 without a second time).
#pragma unroll kWritten
    for (A* sm = sm2;; sm = sm3) {
      D ds2[kD], sq2[kD];
#pragma unroll
      for (int j = 0; j < kD; ++j) ds2[j] = sq2[j] = both(A(0));
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int c = (t + i * width) * kV;
        if (c >= n) break;
#pragma unroll
        for (int j = 0; j < kD; ++j) {
          d[i][j] = d[i][j] + both(-by);
          if constexpr (kHow != kByWords)  // the row may end inside a word: what is behind it deviates by nothing
            d[i][j] = D::of(c + 2 * j < n ? d[i][j].lo() : A(0), c + 2 * j + 1 < n ? d[i][j].hi() : A(0));
          ds2[j] = ds2[j] + d[i][j];
          sq2[j] = fma2(d[i][j], d[i][j], sq2[j]);
        }
      }
#pragma unroll
      for (int j = 1; j < kD; ++j) {
        ds2[0] = ds2[0] + ds2[j];
        sq2[0] = sq2[0] + sq2[j];
      }
      A ds = total(ds2[0]), sq = total(sq2[0]);
      block_sum2(ds, sq, sm, warps);
      off = ds * inv_n;
      var = sq * inv_n - off * off;
      mean += by;
      if (sm == sm3 || !off_too_far(off, var)) break;
      by = off;
    }
    const A r_std = inverse_root((var > A(0) ? var : var * A(0)) + epsilon);  // a NaN stays one
    if (t == 0) {
      if (a.mean) static_cast<A*>(a.mean)[r] = better_mean(first_mean, mean + off, var);
      if (a.inv_std) static_cast<A*>(a.inv_std)[r] = r_std;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = (t + i * width) * kV;
      if (c >= n) break;
      D g[kD], b[kD];
      if (gamma) widen_word(get_word<T, kHow>(gamma, c, n, a.gamma_access, one), g);
      if (beta) widen_word(get_word<T, kHow>(beta, c, n, a.beta_access, zero), b);
#pragma unroll
      for (int j = 0; j < kD; ++j) {
        const D scale = gamma ? g[j] * both(r_std) : both(r_std), centred = d[i][j] + both(-off);
        d[i][j] = beta ? fma2(centred, scale, b[j]) : centred * scale;
      }
      put_word<T, kHow>(out, c, n, a.y_access, to_word<T>(d[i]));
    }
    out += out_step;
  }
  if constexpr (kHow != kInRegisters) wait_async<0>();
}

// rows longer than a block's registers hold: the row is read three times, the second and third from L2
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_long_kernel(
    const T* x, const T* __restrict__ gamma, const T* __restrict__ beta, T* y,
    typename Elem<T>::Acc* __restrict__ mean_out, typename Elem<T>::Acc* __restrict__ inv_std_out, long long rows,
    int n, long long ldx, long long ldy, typename Elem<T>::Acc epsilon) {
  using A = typename Elem<T>::Acc;
  __shared__ A sm1[32], sm2[64], sm3[64];
  const int warps = blockDim.x >> 5;
  const A inv_n = A(1) / A(n);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* in = x + r * ldx;
    T* out = y + r * ldy;
    A sum = 0;
    for (int c = threadIdx.x; c < n; c += blockDim.x) sum += Elem<T>::widen(in[c]);
    const A first_mean = block_sum(sum, sm1, warps) * inv_n, mean0 = leading_bits(first_mean);
    const auto deviations = [&](A more, A& ds, A& sq, A* sm) {
      ds = sq = 0;
      for (int c = threadIdx.x; c < n; c += blockDim.x) {
        const A d = (Elem<T>::widen(in[c]) - mean0) - more;
        ds += d;
        sq += d * d;
      }
      block_sum2(ds, sq, sm, warps);
    };
    A ds, sq, far = 0;  // far: from the pivot to where the deviations are taken from
    deviations(far, ds, sq, sm2);
    A off = ds * inv_n, mean = mean0 + off;
    A var = sq * inv_n - off * off;
    if (off_too_far(off, var)) {  // the same for the whole row
      far = off;
      deviations(far, ds, sq, sm3);
      off = ds * inv_n;
      mean += off;
      var = sq * inv_n - off * off;
    }
    const A r_std = inverse_root((var > A(0) ? var : var * A(0)) + epsilon);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = better_mean(first_mean, mean, var);
      if (inv_std_out) inv_std_out[r] = r_std;
    }
    const auto results = [&](auto centred) {
      for (int c = threadIdx.x; c < n; c += blockDim.x) {
        const A xhat = centred(Elem<T>::widen(in[c])) * r_std;
        out[c] = Elem<T>::narrow(xhat * (gamma ? Elem<T>::widen(gamma[c]) : A(1)) + (beta ? Elem<T>::widen(beta[c]) : A(0)));
      }
    };
    if (far == A(0)) results([&](A v) { return (v - mean0) - off; });
    else results([&](A v) { return ((v - mean0) - far) - off; });
  }
}

// ------------------------------------------------------------------ gradients
struct NormGradArgs {
  const void *grad_out, *x, *mean, *inv_std, *gamma;
  void *grad_in, *grad_gamma, *grad_beta, *partial;
  long long rows, ldg, ldx, ldi;
  int n;
  int g_access, x_access, i_access, gamma_access;
};

// A row belongs to a warp, to a block, or to the blocks of a cluster, each with a contiguous part of the
// columns.  A thread keeps its columns (kN words of 16 bytes) over all rows of its group, and with them
// its share of grad_gamma and grad_beta in registers; a block's share goes to partial[group][2][n].  Many
// elements a thread and few warps a row, because what a thread does once per row costs as much as ten
// elements.  The next rows are on their way in shared memory, kAhead of them (every thread copies the words
// that it will read itself, so no barrier is involved), or, where the rows are not on 16-byte boundaries, one
// in registers.
// words a thread holds in a row of a block: 16 elements, or 8 of f64
template <typename T> constexpr int kGradWords = sizeof(T) == 2 ? 2 : 4;
template <int kN, int kHow> constexpr int kRowsAhead = kHow == kInRegisters ? 1 : 4;

template <typename T, int kN, bool kWarp, int kThreads, int kHow>
__global__ void __launch_bounds__(kThreads, kWarp ? 3 : 512 / kThreads) layernorm_gradients_kernel(const NormGradArgs a) {
  using A = typename Elem<T>::Acc;
  using D = Duo<A>;
  let_next_start();
  constexpr int kV = kVec16<T>, kD = kDuos<T>, kAhead = kRowsAhead<kN, kHow>;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ A sm[2][64];
  __shared__ A of_blocks[2][2][8];  // the cluster's blocks' sums of two rows in turn
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = kWarp ? 1 : static_cast<int>(cluster.num_blocks());
  const int part = kWarp ? 0 : static_cast<int>(cluster.block_rank());
  constexpr int width = kWarp ? 32 : kThreads, warps = kWarp ? 1 : kThreads / 32, per_block = kWarp ? kThreads / 32 : 1;
  const int t = (kWarp ? threadIdx.x & 31 : threadIdx.x) + part * kN * width;  // word of the first pass
  const int local = kWarp ? threadIdx.x >> 5 : 0;
  const long long group = static_cast<long long>(blockIdx.x / parts) * per_block + local;
  const long long groups = static_cast<long long>(gridDim.x / parts) * per_block;
  const int n = a.n;
  const A inv_n = A(1) / A(n);
  const T zero = Elem<T>::narrow(0);
  // the next row to come, and the next to go
  const T *x = static_cast<const T*>(a.x) + group * a.ldx, *grad_out = static_cast<const T*>(a.grad_out) + group * a.ldg;
  const A *mean = static_cast<const A*>(a.mean) + group, *inv_std = static_cast<const A*>(a.inv_std) + group;
  T* out = static_cast<T*>(a.grad_in) + group * a.ldi;
  const long long x_step = groups * a.ldx, g_step = groups * a.ldg, i_step = groups * a.ldi;
  long long coming = group;
  D sum_g[kN][kD], sum_gx[kN][kD];
  Word<T> w[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    w[i] = read_word(static_cast<const T*>(a.gamma), (t + i * width) * kV, a.gamma ? n : 0, a.gamma_access, Elem<T>::narrow(1));
#pragma unroll
    for (int j = 0; j < kD; ++j) sum_g[i][j] = sum_gx[i][j] = both(A(0));
  }
  Word<T>* ring = reinterpret_cast<Word<T>*>(dyn);  // [stage][x or grad_out][word of the pass][thread]
  const auto place = [&](int stage, int which, int i) {
    return ring + ((stage * 2 + which) * kN + i) * kThreads + threadIdx.x;
  };
  Word<T> px[kN], pg[kN];
  A next_m[kAhead], next_s[kAhead];
  const auto fetch = [&](int stage) {  // stage is a constant wherever this is inlined
    if (coming < a.rows) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int c = (t + i * width) * kV;
        if constexpr (kHow != kInRegisters) {
          if (c < n) {
            copy_word<T, kHow>(place(stage, 0, i), x, c, n);
            copy_word<T, kHow>(place(stage, 1, i), grad_out, c, n);
          }
        } else {
          px[i] = read_word(x, c, n, a.x_access, zero);
          pg[i] = read_word(grad_out, c, n, a.g_access, zero);
        }
      }
      next_m[stage] = *mean;
      next_s[stage] = *inv_std;
      x += x_step;
      grad_out += g_step;
      mean += groups;
      inv_std += groups;
      coming += groups;
    }
    if constexpr (kHow != kInRegisters) commit_async();
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s) fetch(s);
  int turn = 0;
  if (!kWarp && parts > 1) cluster.sync();  // every block has started before any writes to another
  for (long long r0 = group; r0 < a.rows; r0 += kAhead * groups) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const long long r = r0 + s * groups;
      if (r >= a.rows) break;  // the same for the whole group
      if constexpr (kHow != kInRegisters) wait_async<kAhead - 1>();
      const A m = next_m[s], rs = next_s[s];
      D xhat[kN][kD], u[kN][kD];
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int c = (t + i * width) * kV;
        Word<T> cx, cg_;
        if constexpr (kHow != kInRegisters) {
          cx = take_word<T, kHow>(place(s, 0, i), c, n, zero);
          cg_ = take_word<T, kHow>(place(s, 1, i), c, n, zero);
        } else {
          cx = px[i];
          cg_ = pg[i];
        }
        widen_word(cx, xhat[i]);
        widen_word(cg_, u[i]);
      }
      fetch(s);
      D su2 = both(A(0)), sux2 = both(A(0));
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        D wi[kD];
        widen_word(w[i], wi);
#pragma unroll
        for (int j = 0; j < kD; ++j) {  // behind the row grad_out is zero and nothing is added
          xhat[i][j] = (xhat[i][j] + both(-m)) * both(rs);
          sum_g[i][j] = sum_g[i][j] + u[i][j];
          sum_gx[i][j] = fma2(u[i][j], xhat[i][j], sum_gx[i][j]);
          u[i][j] = u[i][j] * wi[j];
          su2 = su2 + u[i][j];
          sux2 = fma2(u[i][j], xhat[i][j], sux2);
        }
      }
      A su = total(su2), sux = total(sux2);
      block_sum2(su, sux, sm[turn], warps);
      if (!kWarp && parts > 1) {
        // every block writes its sums into all blocks of the cluster; two places in turn, because a
        // block may be one row ahead of another, but no more
        if (threadIdx.x < parts) {
          *cluster.map_shared_rank(&of_blocks[turn][0][part], threadIdx.x) = su;
          *cluster.map_shared_rank(&of_blocks[turn][1][part], threadIdx.x) = sux;
        }
        cluster.sync();
        su = sux = A(0);
        for (int b = 0; b < parts; ++b) {
          su += of_blocks[turn][0][b];
          sux += of_blocks[turn][1][b];
        }
      }
      turn ^= 1;
      const D level = both(-su * inv_n * rs), along = both(-sux * inv_n);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int c = (t + i * width) * kV;
        if (c >= n) break;
#pragma unroll
        for (int j = 0; j < kD; ++j) u[i][j] = fma2(fma2(xhat[i][j], along, u[i][j]), both(rs), level);
        put_word<T, kHow>(out, c, n, a.i_access, to_word<T>(u[i]));
      }
      out += i_step;
    }
  }
  if constexpr (kHow != kInRegisters) wait_async<0>();
  if (!kWarp && parts > 1) cluster.sync();  // no block leaves while another may still write to it
  if (!a.partial) return;
  A* mine = static_cast<A*>(a.partial) + static_cast<long long>(blockIdx.x / parts) * 2 * n;
  if constexpr (kWarp) {
    // the block's warps hold the same columns: summed in order through shared memory, one of the two sums
    // after the other
    A* add = reinterpret_cast<A*>(dyn);  // [warp][word][element][lane]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kN; ++i)
#pragma unroll
        for (int j = 0; j < kD; ++j) {
          const D v = which ? sum_g[i][j] : sum_gx[i][j];
          add[((local * kN + i) * kV + 2 * j) * 32 + t] = v.lo();
          add[((local * kN + i) * kV + 2 * j + 1) * 32 + t] = v.hi();
        }
      __syncthreads();
      for (int e = threadIdx.x; e < kN * kV * 32; e += kThreads) {
        A v = add[e];
        for (int b = 1; b < per_block; ++b) v += add[b * kN * kV * 32 + e];
        const int lane = e & 31, j = (e >> 5) % kV, i = (e >> 5) / kV, c = (lane + 32 * i) * kV + j;
        if (c < n) mine[which * n + c] = v;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < kD; ++j) {
        const int c = (t + i * width) * kV + 2 * j;
        if (c < n) { mine[c] = sum_gx[i][j].lo(); mine[n + c] = sum_g[i][j].lo(); }
        if (c + 1 < n) { mine[c + 1] = sum_gx[i][j].hi(); mine[n + c + 1] = sum_g[i][j].hi(); }
      }
  }
}

// rows longer than a block's registers hold, first half: the two sums of every row
template <typename T>
__global__ void __launch_bounds__(512) layernorm_row_sums_kernel(
    const T* __restrict__ grad_out, const T* __restrict__ x, const typename Elem<T>::Acc* __restrict__ mean,
    const typename Elem<T>::Acc* __restrict__ inv_std, const T* __restrict__ gamma,
    typename Elem<T>::Acc* __restrict__ row_sums, long long rows, int n, long long ldg, long long ldx) {
  using A = typename Elem<T>::Acc;
  __shared__ A sm[2][64];
  int turn = 0;
  const A inv_n = A(1) / A(n);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const A m = mean[r], s = inv_std[r];
    A su = 0, sux = 0;
    for (int c = threadIdx.x; c < n; c += 512) {
      const A u = Elem<T>::widen(grad_out[r * ldg + c]) * (gamma ? Elem<T>::widen(gamma[c]) : A(1));
      su += u;
      sux += u * ((Elem<T>::widen(x[r * ldx + c]) - m) * s);
    }
    block_sum2(su, sux, sm[turn], 16);
    turn ^= 1;
    if (threadIdx.x == 0) {
      row_sums[2 * r] = su * inv_n;
      row_sums[2 * r + 1] = sux * inv_n;
    }
  }
}
// second half: a thread per column over a share of the rows (blockIdx.y)
template <typename T>
__global__ void __launch_bounds__(256) layernorm_columns_kernel(
    const T* grad_out, const T* __restrict__ x, const typename Elem<T>::Acc* __restrict__ mean,
    const typename Elem<T>::Acc* __restrict__ inv_std, const T* __restrict__ gamma,
    const typename Elem<T>::Acc* __restrict__ row_sums, T* grad_in, typename Elem<T>::Acc* __restrict__ partial,
    long long rows, int n, long long ldg, long long ldx, long long ldi) {
  using A = typename Elem<T>::Acc;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  const A w = gamma ? Elem<T>::widen(gamma[c]) : A(1);
  A sg = 0, sgx = 0;
#pragma unroll 4
  for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
    const A g = Elem<T>::widen(grad_out[r * ldg + c]), s = inv_std[r];
    const A xhat = (Elem<T>::widen(x[r * ldx + c]) - mean[r]) * s;
    grad_in[r * ldi + c] = Elem<T>::narrow(s * (g * w - row_sums[2 * r] - xhat * row_sums[2 * r + 1]));
    sg += g;
    sgx += g * xhat;
  }
  if (!partial) return;
  A* mine = partial + static_cast<long long>(blockIdx.y) * 2 * n;
  mine[c] = sgx;
  mine[n + c] = sg;
}

// grad_gamma and grad_beta: the groups' shares added in a fixed order, 32 columns of the 2 n per block,
// 32 threads per column
template <typename A>
__global__ void __launch_bounds__(1024) layernorm_join_kernel(const A* __restrict__ partial, int groups, int n,
                                                              A* __restrict__ grad_gamma, A* __restrict__ grad_beta) {
  __shared__ A sm[32][33];
  after_previous();
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const long long c = static_cast<long long>(blockIdx.x) * 32 + col, width = 2LL * n;
  A s = 0;
  if (c < width) {
#pragma unroll 8
    for (int g = lane; g < groups; g += 32) s += partial[g * width + c];
  }
  sm[lane][col] = s;
  __syncthreads();
  // transposed: a warp now holds the 32 shares of one column
  s = warp_sum(sm[col][lane]);
  const long long cc = static_cast<long long>(blockIdx.x) * 32 + lane;
  if (col != 0 || cc >= width) return;
  if (cc < n) { if (grad_gamma) grad_gamma[cc] = s; }
  else if (grad_beta) grad_beta[cc - n] = s;
}

unsigned grid_of(long long want, long long cap) {
  return static_cast<unsigned>(want < 1 ? 1 : (want < cap ? want : cap));
}

// more dynamic shared memory than a kernel gets unasked
template <typename F> bool allow_shared(F kernel, size_t bytes) {
  return bytes <= 32 * 1024 ||  // static shared memory counts towards the 48 KB that need no asking
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) == cudaSuccess;
}

template <typename T, int kN, bool kWarp, int kThreads, int kHow>
void launch_forward_as(const NormArgs& a, cudaStream_t st) {
  constexpr size_t smem = kHow == kInRegisters ? 0 : static_cast<size_t>(kNormAhead<kThreads, kHow>) * kN * kThreads * 16;
  const auto kernel = layernorm_kernel<T, kN, kWarp, kThreads, kHow>;
  if (!allow_shared(kernel, smem)) return;  // the error is read after the launch
  // blocks that an SM holds, by registers (the launch bounds) and by shared memory
  constexpr long long by_registers = kThreads <= 256 ? 768 / kThreads : 1, by_shared = 220 * 1024 / (smem + 1024);
  const long long want = kWarp ? (a.rows + kThreads / 32 - 1) / (kThreads / 32) : a.rows;
  kernel<<<grid_of(want, lib_num_sms() * (by_registers < by_shared ? by_registers : by_shared)), kThreads, smem, st>>>(a);
}

// rows in many: a warp each while four words a thread hold it, then a block
template <typename T, int kHow> void launch_forward_many(const NormArgs& a, int words, cudaStream_t st) {
  if (words <= 32) launch_forward_as<T, 1, true, 128, kHow>(a, st);
  else if (words <= 64) launch_forward_as<T, 2, true, 128, kHow>(a, st);
  else if (words <= 128) launch_forward_as<T, 4, true, 128, kHow>(a, st);
  else if (words <= 256) launch_forward_as<T, 2, false, 128, kHow>(a, st);
  else if (words <= 512) launch_forward_as<T, 4, false, 128, kHow>(a, st);
  else if (words <= 1024) launch_forward_as<T, 4, false, 256, kHow>(a, st);
  else if (words <= 2048) launch_forward_as<T, 4, false, 512, kHow>(a, st);
  else launch_forward_as<T, 4, false, 1024, kHow>(a, st);
}

template <typename T> int launch_forward(NormArgs a, cudaStream_t st) {
  using A = typename Elem<T>::Acc;
  a.x_access = row_access<T>(a.x, a.ldx, a.n);
  a.y_access = row_access<T>(a.y, a.ldy, a.n);
  a.gamma_access = row_access<T>(a.gamma, 0, a.n);
  a.beta_access = row_access<T>(a.beta, 0, a.n);
  const int words = (a.n + kVec16<T> - 1) / kVec16<T>;
  const long long sms = lib_num_sms();
  if (words > 4096) {  // over four words for each of 1024 threads
    layernorm_long_kernel<T><<<grid_of(a.rows, sms * 2), 1024, 0, st>>>(
        static_cast<const T*>(a.x), static_cast<const T*>(a.gamma), static_cast<const T*>(a.beta), static_cast<T*>(a.y),
        static_cast<A*>(a.mean), static_cast<A*>(a.inv_std), a.rows, a.n, a.ldx, a.ldy, static_cast<A>(a.epsilon));
  } else if (a.rows < 4 * sms && words > 32) {
    // few rows: the latency of one counts, so it gets as many threads as it has words, and nothing comes after it
    if (words <= 128) launch_forward_as<T, 1, false, 128, kInRegisters>(a, st);
    else if (words <= 512) launch_forward_as<T, 1, false, 512, kInRegisters>(a, st);
    else if (words <= 1024) launch_forward_as<T, 1, false, 1024, kInRegisters>(a, st);
    else launch_forward_as<T, 4, false, 1024, kInRegisters>(a, st);
  } else if (a.x_access == kInWords && a.y_access == kInWords && a.gamma_access == kInWords && a.beta_access == kInWords &&
             a.n % kVec16<T> == 0) {
    launch_forward_many<T, kByWords>(a, words, st);
  } else {
    if (rows_by_elements<T>(a.x, a.ldx, a.n)) launch_forward_many<T, kByElements>(a, words, st);
    else launch_forward_many<T, kInRegisters>(a, words, st);
  }
  return 1;
}

// How a row is dealt out: a warp per row (threads 0), or `parts` blocks of `threads`; groups: rows at once.
// parts 0: the row does not fit.
struct GradShape { int per, threads, parts; long long groups; };

template <typename T> GradShape gradients_shape(const NormGradArgs& a) {
  constexpr int kV = kVec16<T>, kN = kGradWords<T>;
  const long long sms = lib_num_sms();
  const int words = (a.n + kV - 1) / kV;
  if (words <= 32 * kN) return {words <= 32 ? 1 : words <= 64 ? 2 : 4, 0, 1, grid_of((a.rows + 3) / 4, sms * 3)};
  // a block takes up to 256 threads' words; a wider row takes more blocks, at most eight
  int threads = 64, parts = 1;
  while (threads < 256 && words > threads * kN) threads *= 2;
  while (parts < 8 && words > threads * kN * parts) parts *= 2;
  if (words > threads * kN * parts) return {0, 0, 0, 0};
  return {kN, threads, parts, grid_of(a.rows, sms * (512 / threads) / parts)};
}

template <typename T, int kN, bool kWarp, int kThreads, int kHow>
cudaError_t launch_gradients_as(const NormGradArgs& a, const GradShape& q, cudaStream_t st) {
  size_t smem = kHow != kInRegisters ? static_cast<size_t>(kRowsAhead<kN, kHow>) * 2 * kN * kThreads * 16 : 0;
  if (kWarp) {  // the warps' shares are summed there at the end
    const size_t add = static_cast<size_t>(kThreads) * kN * kVec16<T> * sizeof(typename Elem<T>::Acc);
    if (add > smem) smem = add;
  }
  const auto kernel = layernorm_gradients_kernel<T, kN, kWarp, kThreads, kHow>;
  if (!allow_shared(kernel, smem)) return cudaGetLastError();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(q.groups * q.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(q.parts);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int kHow>
cudaError_t launch_gradients_shaped(const NormGradArgs& a, const GradShape& q, cudaStream_t st) {
  constexpr int kN = kGradWords<T>;
  if (q.threads == 0) {
    if (q.per == 1) return launch_gradients_as<T, 1, true, 128, kHow>(a, q, st);
    if (q.per == 2) return launch_gradients_as<T, 2, true, 128, kHow>(a, q, st);
    return launch_gradients_as<T, kN, true, 128, kHow>(a, q, st);
  }
  if (q.threads == 64) return launch_gradients_as<T, kN, false, 64, kHow>(a, q, st);
  if (q.threads == 128) return launch_gradients_as<T, kN, false, 128, kHow>(a, q, st);
  return launch_gradients_as<T, kN, false, 256, kHow>(a, q, st);
}
template <typename T> cudaError_t launch_gradients_any(const NormGradArgs& a, const GradShape& q, cudaStream_t st) {
  if (a.g_access == kInWords && a.x_access == kInWords && a.i_access == kInWords && a.n % kVec16<T> == 0)
    return launch_gradients_shaped<T, kByWords>(a, q, st);
  if (rows_by_elements<T>(a.grad_out, a.ldg, a.n) && rows_by_elements<T>(a.x, a.ldx, a.n))
    return launch_gradients_shaped<T, kByElements>(a, q, st);
  if constexpr (sizeof(T) >= 4) return cudaErrorInvalidValue;  // any such row can be copied
  else return launch_gradients_shaped<T, kInRegisters>(a, q, st);
}

template <typename T>
int launch_gradients(NormGradArgs a, OpScratch& scratch, cudaStream_t st) {
  using A = typename Elem<T>::Acc;
  a.g_access = row_access<T>(a.grad_out, a.ldg, a.n);
  a.x_access = row_access<T>(a.x, a.ldx, a.n);
  a.i_access = row_access<T>(a.grad_in, a.ldi, a.n);
  a.gamma_access = row_access<T>(a.gamma, 0, a.n);
  const GradShape q = gradients_shape<T>(a);
  const bool weights = a.grad_gamma || a.grad_beta;
  const size_t row_of_sums = 2 * static_cast<size_t>(a.n) * sizeof(A);
  int groups = 0, launches = 1;
  if (q.parts) {
    groups = static_cast<int>(q.groups);
    if (weights) {
      a.partial = scratch.reserve(groups * row_of_sums, st);
      if (!a.partial) return -1;
    }
    const cudaError_t e = launch_gradients_any<T>(a, q, st);
    if (e != cudaSuccess) {
      fprintf(stderr, "[eshkol-b200] layer norm launch failed: %s\n", cudaGetErrorString(e));
      cudaGetLastError();
      return -1;
    }
  } else {
    const long long sms = lib_num_sms();
    const unsigned col_blocks = static_cast<unsigned>((a.n + 255) / 256);
    groups = static_cast<int>(grid_of(a.rows, sms * 8 / col_blocks < 1 ? 1 : sms * 8 / col_blocks));
    const size_t head = (static_cast<size_t>(a.rows) * 2 * sizeof(A) + 255) & ~static_cast<size_t>(255);
    uint8_t* base = scratch.reserve(head + (weights ? groups * row_of_sums : 0), st);
    if (!base) return -1;
    A* sums = reinterpret_cast<A*>(base);
    if (weights) a.partial = base + head;
    layernorm_row_sums_kernel<T><<<grid_of(a.rows, sms * 4), 512, 0, st>>>(
        static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), static_cast<const A*>(a.mean),
        static_cast<const A*>(a.inv_std), static_cast<const T*>(a.gamma), sums, a.rows, a.n, a.ldg, a.ldx);
    layernorm_columns_kernel<T><<<dim3(col_blocks, static_cast<unsigned>(groups)), 256, 0, st>>>(
        static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), static_cast<const A*>(a.mean),
        static_cast<const A*>(a.inv_std), static_cast<const T*>(a.gamma), sums, static_cast<T*>(a.grad_in),
        static_cast<A*>(a.partial), a.rows, a.n, a.ldg, a.ldx, a.ldi);
    launches = 2;
  }
  if (weights) {
    const cudaError_t e = launch_after(layernorm_join_kernel<A>, static_cast<unsigned>((2LL * a.n + 31) / 32), 1024, 0, st,
                                       static_cast<const A*>(a.partial), groups, a.n, static_cast<A*>(a.grad_gamma),
                                       static_cast<A*>(a.grad_beta));
    if (e != cudaSuccess) {
      fprintf(stderr, "[eshkol-b200] layer norm launch failed: %s\n", cudaGetErrorString(e));
      cudaGetLastError();
      return -1;
    }
    ++launches;
  }
  return launches;
}

int finish(int launches) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    fprintf(stderr, "[eshkol-b200] layer norm launch failed: %s\n", cudaGetErrorString(e));
    return -1;
  }
  count_launches(launches);
  return 0;
}

bool shape_ok(uint64_t samples, uint64_t features, int dtype) {
  return samples <= (1ull << 40) && features >= 1 && features <= (1ull << 28) && dtype >= ESHKOL_B200_F64 &&
         dtype <= ESHKOL_B200_BF16;
}
// a row pitch: 0 stands for dense rows, anything shorter than a row is refused
bool pitch_ok(uint64_t ld, uint64_t features) { return (ld == 0 || ld >= features) && ld <= (1ull << 40); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int eshkol_b200_layernorm_forward_device(const void* x, const void* gamma, const void* beta, void* y, void* mean,
                                         void* inv_std, uint64_t samples, uint64_t features, uint64_t ldx, uint64_t ldy,
                                         double epsilon, int dtype) {
  if (lib_device() < 0 || !shape_ok(samples, features, dtype) || !pitch_ok(ldx, features) || !pitch_ok(ldy, features) ||
      !(epsilon >= 0.0))
    return -1;
  if (samples == 0) return 0;
  if (!x || !y || (x == y && (ldx ? ldx : features) != (ldy ? ldy : features))) return -1;
  DeviceScope scope(lib_device());
  if (!scope.ok()) return -1;
  NormArgs a;
  a.x = x; a.gamma = gamma; a.beta = beta; a.y = y; a.mean = mean; a.inv_std = inv_std;
  a.rows = static_cast<long long>(samples); a.n = static_cast<int>(features);
  a.ldx = static_cast<long long>(ldx ? ldx : features); a.ldy = static_cast<long long>(ldy ? ldy : features);
  a.epsilon = epsilon;
  cudaStream_t st = lib_stream();
  switch (dtype) {
    case ESHKOL_B200_F64: return finish(launch_forward<double>(a, st));
    case ESHKOL_B200_F32: return finish(launch_forward<float>(a, st));
    case ESHKOL_B200_F16: return finish(launch_forward<__half>(a, st));
    default: return finish(launch_forward<__nv_bfloat16>(a, st));
  }
}

int eshkol_b200_layernorm_gradients_device(const void* grad_out, const void* x, const void* mean, const void* inv_std,
                                           const void* gamma, void* grad_in, void* grad_gamma, void* grad_beta,
                                           uint64_t samples, uint64_t features, uint64_t ld_grad_out, uint64_t ldx,
                                           uint64_t ld_grad_in, int dtype) {
  if (lib_device() < 0 || !shape_ok(samples, features, dtype) || !pitch_ok(ld_grad_out, features) ||
      !pitch_ok(ldx, features) || !pitch_ok(ld_grad_in, features))
    return -1;
  DeviceScope scope(lib_device());
  if (!scope.ok()) return -1;
  cudaStream_t st = lib_stream();
  if (samples == 0) {  // sums over no samples
    const size_t bytes = static_cast<size_t>(features) * (dtype == ESHKOL_B200_F64 ? 8 : 4);
    if (grad_gamma && cudaMemsetAsync(grad_gamma, 0, bytes, st) != cudaSuccess) return finish(0);
    if (grad_beta && cudaMemsetAsync(grad_beta, 0, bytes, st) != cudaSuccess) return finish(0);
    return 0;
  }
  NormGradArgs a;
  a.ldg = static_cast<long long>(ld_grad_out ? ld_grad_out : features);
  a.ldx = static_cast<long long>(ldx ? ldx : features);
  a.ldi = static_cast<long long>(ld_grad_in ? ld_grad_in : features);
  if (!grad_out || !x || !mean || !inv_std || !grad_in || (grad_in == grad_out && a.ldi != a.ldg) || grad_in == x) return -1;
  a.grad_out = grad_out; a.x = x; a.mean = mean; a.inv_std = inv_std; a.gamma = gamma;
  a.grad_in = grad_in; a.grad_gamma = grad_gamma; a.grad_beta = grad_beta; a.partial = nullptr;
  a.rows = static_cast<long long>(samples); a.n = static_cast<int>(features);
  OpScratch scratch;
  int launches;
  switch (dtype) {
    case ESHKOL_B200_F64: launches = launch_gradients<double>(a, scratch, st); break;
    case ESHKOL_B200_F32: launches = launch_gradients<float>(a, scratch, st); break;
    case ESHKOL_B200_F16: launches = launch_gradients<__half>(a, scratch, st); break;
    default: launches = launch_gradients<__nv_bfloat16>(a, scratch, st); break;
  }
  if (launches < 0) return -1;
  if (finish(launches) != 0) return -1;
  return scratch.release();
}

}  // extern "C"
