// Layer normalisation with weight vectors, and its three gradients, on f64, f32, f16 and bf16 tensors.
//
//   y = (x - mean) r gamma + beta,  mean = sum x / D,  r = 1 / sqrt(sum (x - mean)^2 / D + epsilon)
//   with xhat = (x - mean) r and u = grad_out gamma:
//   grad_in    = r (u - sum u / D - xhat sum(u xhat) / D)
//   grad_gamma = sum over samples of grad_out xhat,   grad_beta = sum over samples of grad_out
//
// Both directions are bound by HBM: 2 (forward) or 3 (gradients) tensors cross it once.  A row is held
// in registers from its one read to its one write, so the statistics are the two-pass ones (the mean
// first, then the deviations, with the deviations' own sum as a correction) at the traffic of one
// pass.  Sums, statistics and the weights' gradients are f32 (f64 for f64 tensors); a result is rounded
// to the storage type once.  Sums are combined in a fixed order: results do not depend on timing.
#include <math.h>
#include <stdio.h>

#include "b200_elem.cuh"
#include "b200_tiers.h"

namespace b200 {
namespace {

template <typename T, int kV, int kN>
__device__ __forceinline__ void load_row(const T* row, int n, int first, int stride, Pack<T, kV> (&p)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int c = (first + i * stride) * kV;
    if (c + kV <= n) {
      p[i] = *reinterpret_cast<const Pack<T, kV>*>(row + c);
    } else {
#pragma unroll
      for (int j = 0; j < kV; ++j) p[i].v[j] = (c + j < n) ? row[c + j] : Elem<T>::narrow(0);
    }
  }
}

template <typename T, int kV>
__device__ __forceinline__ void store_pack(T* row, int n, int c, const Pack<T, kV>& p) {
  if (c + kV <= n) {
    *reinterpret_cast<Pack<T, kV>*>(row + c) = p;
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j)
      if (c + j < n) row[c + j] = p.v[j];
  }
}

template <typename T, int kV>
__device__ __forceinline__ Pack<T, kV> load_weights(const T* w, int n, int c, float otherwise) {
  Pack<T, kV> p;
  if (w && c + kV <= n) return *reinterpret_cast<const Pack<T, kV>*>(w + c);
#pragma unroll
  for (int j = 0; j < kV; ++j) p.v[j] = (w && c + j < n) ? w[c + j] : Elem<T>::narrow(otherwise);
  return p;
}

// ------------------------------------------------------------------ forward
// A row is shared by `width` threads (a warp, or the block), each holding kN packs of kV elements.
template <typename T, int kV, int kN, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : 1024) layernorm_kernel(
    const T* x, const T* __restrict__ gamma, const T* __restrict__ beta, T* y,  // x and y may be the same
    typename Elem<T>::Acc* __restrict__ mean_out, typename Elem<T>::Acc* __restrict__ inv_std_out, long long rows,
    int n, long long ldx, long long ldy, typename Elem<T>::Acc epsilon) {
  using A = typename Elem<T>::Acc;
  __shared__ A sm[64];
  const int width = kWarp ? 32 : blockDim.x, warps = kWarp ? 1 : blockDim.x >> 5;
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int per_block = kWarp ? blockDim.x >> 5 : 1, group = kWarp ? threadIdx.x >> 5 : 0;
  const A inv_n = A(1) / A(n);
  for (long long r = static_cast<long long>(blockIdx.x) * per_block + group; r < rows;
       r += static_cast<long long>(gridDim.x) * per_block) {
    Pack<T, kV> p[kN];
    load_row<T, kV, kN>(x + r * ldx, n, t, width, p);
    A sum = 0, none = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < kV; ++j) sum += Elem<T>::widen(p[i].v[j]);  // places behind the row hold zero
    block_sum2(sum, none, sm, warps);
    const A mean0 = sum * inv_n;
    A ds = 0, sq = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const A d = ((t + i * width) * kV + j < n) ? Elem<T>::widen(p[i].v[j]) - mean0 : A(0);
        ds += d;
        sq += d * d;
      }
    block_sum2(ds, sq, sm, warps);
    // mean0 carries the rounding of a long sum; the deviations' own mean is what it is off by
    const A off = ds * inv_n;
    const A var = sq * inv_n - off * off;
    const A r_std = sum_rsqrt((var > A(0) ? var : var * A(0)) + epsilon);  // a NaN stays one
    if (t == 0) {
      if (mean_out) mean_out[r] = mean0 + off;
      if (inv_std_out) inv_std_out[r] = r_std;
    }
    T* out = y + r * ldy;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = (t + i * width) * kV;
      if (c >= n) break;
      const Pack<T, kV> g = load_weights<T, kV>(gamma, n, c, 1.f), b = load_weights<T, kV>(beta, n, c, 0.f);
      Pack<T, kV> o;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const A xhat = ((Elem<T>::widen(p[i].v[j]) - mean0) - off) * r_std;
        o.v[j] = Elem<T>::narrow(xhat * Elem<T>::widen(g.v[j]) + Elem<T>::widen(b.v[j]));
      }
      store_pack<T, kV>(out, n, c, o);
    }
  }
}

// rows longer than a block's registers hold: the row is read three times, the second and third from L2
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_long_kernel(
    const T* x, const T* __restrict__ gamma, const T* __restrict__ beta, T* y,
    typename Elem<T>::Acc* __restrict__ mean_out, typename Elem<T>::Acc* __restrict__ inv_std_out, long long rows,
    int n, long long ldx, long long ldy, typename Elem<T>::Acc epsilon) {
  using A = typename Elem<T>::Acc;
  __shared__ A sm[64];
  const int warps = blockDim.x >> 5;
  const A inv_n = A(1) / A(n);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* in = x + r * ldx;
    T* out = y + r * ldy;
    A sum = 0, none = 0;
    for (int c = threadIdx.x; c < n; c += blockDim.x) sum += Elem<T>::widen(in[c]);
    block_sum2(sum, none, sm, warps);
    const A mean0 = sum * inv_n;
    A ds = 0, sq = 0;
    for (int c = threadIdx.x; c < n; c += blockDim.x) {
      const A d = Elem<T>::widen(in[c]) - mean0;
      ds += d;
      sq += d * d;
    }
    block_sum2(ds, sq, sm, warps);
    const A off = ds * inv_n;
    const A var = sq * inv_n - off * off;
    const A r_std = sum_rsqrt((var > A(0) ? var : var * A(0)) + epsilon);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean0 + off;
      if (inv_std_out) inv_std_out[r] = r_std;
    }
    for (int c = threadIdx.x; c < n; c += blockDim.x) {
      const A xhat = ((Elem<T>::widen(in[c]) - mean0) - off) * r_std;
      out[c] = Elem<T>::narrow(xhat * (gamma ? Elem<T>::widen(gamma[c]) : A(1)) + (beta ? Elem<T>::widen(beta[c]) : A(0)));
    }
  }
}

// ------------------------------------------------------------------ gradients
// A row is shared by `width` threads (a warp of a block of eight, or the block); every thread keeps its
// columns over all the rows of its group, and with them its share of grad_gamma and grad_beta in
// registers.  A group's shares go to partial[group][2][n].
template <typename T, int kV, int kN, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 256 : 512) layernorm_gradients_kernel(
    const T* grad_out, const T* __restrict__ x, const typename Elem<T>::Acc* __restrict__ mean,
    const typename Elem<T>::Acc* __restrict__ inv_std, const T* __restrict__ gamma, T* grad_in,
    typename Elem<T>::Acc* __restrict__ partial, long long rows, int n, long long ldg, long long ldx, long long ldi) {
  using A = typename Elem<T>::Acc;
  __shared__ A sm[64];
  const int width = kWarp ? 32 : blockDim.x, warps = kWarp ? 1 : blockDim.x >> 5;
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int per_block = kWarp ? blockDim.x >> 5 : 1, local = kWarp ? threadIdx.x >> 5 : 0;
  const long long group = static_cast<long long>(blockIdx.x) * per_block + local;
  const long long groups = static_cast<long long>(gridDim.x) * per_block;
  const A inv_n = A(1) / A(n);
  A sum_g[kN][kV], sum_gx[kN][kV];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kV; ++j) sum_g[i][j] = sum_gx[i][j] = A(0);
  Pack<T, kV> w[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) w[i] = load_weights<T, kV>(gamma, n, (t + i * width) * kV, 1.f);
  Pack<T, kV> px[kN], pg[kN];
  A mu = 0, rs = 0;
  if (group < rows) {
    load_row<T, kV, kN>(x + group * ldx, n, t, width, px);
    load_row<T, kV, kN>(grad_out + group * ldg, n, t, width, pg);
    mu = mean[group];
    rs = inv_std[group];
  }
  for (long long r = group; r < rows; r += groups) {
    Pack<T, kV> cx[kN], cg[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) { cx[i] = px[i]; cg[i] = pg[i]; }
    const A m = mu, s = rs;
    const long long next = r + groups;  // the next row is on its way while this one is worked on
    if (next < rows) {
      load_row<T, kV, kN>(x + next * ldx, n, t, width, px);
      load_row<T, kV, kN>(grad_out + next * ldg, n, t, width, pg);
      mu = mean[next];
      rs = inv_std[next];
    }
    A su = 0, sux = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const A g = Elem<T>::widen(cg[i].v[j]);  // zero behind the row
        const A xhat = (Elem<T>::widen(cx[i].v[j]) - m) * s;
        const A u = g * Elem<T>::widen(w[i].v[j]);
        if ((t + i * width) * kV + j < n) {
          su += u;
          sux += u * xhat;
          sum_g[i][j] += g;
          sum_gx[i][j] += g * xhat;
        }
      }
    block_sum2(su, sux, sm, warps);
    const A level = su * inv_n, along = sux * inv_n;
    T* out = grad_in + r * ldi;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int c = (t + i * width) * kV;
      if (c >= n) break;
      Pack<T, kV> o;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const A xhat = (Elem<T>::widen(cx[i].v[j]) - m) * s;
        const A u = Elem<T>::widen(cg[i].v[j]) * Elem<T>::widen(w[i].v[j]);
        o.v[j] = Elem<T>::narrow(s * (u - level - xhat * along));
      }
      store_pack<T, kV>(out, n, c, o);
    }
  }
  if (!partial) return;
  A* mine = partial + group * 2 * n;
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const int c = (t + i * width) * kV + j;
      if (c < n) {
        mine[c] = sum_gx[i][j];
        mine[n + c] = sum_g[i][j];
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
  __shared__ A sm[64];
  const A inv_n = A(1) / A(n);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const A m = mean[r], s = inv_std[r];
    A su = 0, sux = 0;
    for (int c = threadIdx.x; c < n; c += 512) {
      const A u = Elem<T>::widen(grad_out[r * ldg + c]) * (gamma ? Elem<T>::widen(gamma[c]) : A(1));
      su += u;
      sux += u * ((Elem<T>::widen(x[r * ldx + c]) - m) * s);
    }
    block_sum2(su, sux, sm, 16);
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
// eight threads per column
template <typename A>
__global__ void __launch_bounds__(256) layernorm_join_kernel(const A* __restrict__ partial, int groups, int n,
                                                             A* __restrict__ grad_gamma, A* __restrict__ grad_beta) {
  __shared__ A sm[8][32];
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const long long c = static_cast<long long>(blockIdx.x) * 32 + col, width = 2LL * n;
  A s = 0;
  if (c < width) {
#pragma unroll 8
    for (int g = lane; g < groups; g += 8) s += partial[g * width + c];
  }
  sm[lane][col] = s;
  __syncthreads();
  if (lane != 0 || c >= width) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += sm[i][col];
  if (c < n) { if (grad_gamma) grad_gamma[c] = s; }
  else if (grad_beta) grad_beta[c - n] = s;
}

struct NormArgs {
  const void *x, *gamma, *beta;
  void *y, *mean, *inv_std;
  long long rows, ldx, ldy;
  int n;
  double epsilon;
};

template <typename T, int kV, int kN, bool kWarp>
void launch_forward_as(const NormArgs& a, unsigned grid, int threads, cudaStream_t st) {
  using A = typename Elem<T>::Acc;
  layernorm_kernel<T, kV, kN, kWarp><<<grid, threads, 0, st>>>(
      static_cast<const T*>(a.x), static_cast<const T*>(a.gamma), static_cast<const T*>(a.beta), static_cast<T*>(a.y),
      static_cast<A*>(a.mean), static_cast<A*>(a.inv_std), a.rows, a.n, a.ldx, a.ldy, static_cast<A>(a.epsilon));
}

unsigned grid_of(long long want, long long cap) {
  return static_cast<unsigned>(want < 1 ? 1 : (want < cap ? want : cap));
}

template <typename T, int kV>
bool launch_forward_packed(const NormArgs& a, cudaStream_t st) {
  const long long sms = lib_num_sms();
  const int packs = (a.n + kV - 1) / kV;
  if (packs <= 32 * 4) {
    const unsigned grid = grid_of((a.rows + 7) / 8, sms * 8);
    if (packs <= 32) launch_forward_as<T, kV, 1, true>(a, grid, 256, st);
    else if (packs <= 64) launch_forward_as<T, kV, 2, true>(a, grid, 256, st);
    else launch_forward_as<T, kV, 4, true>(a, grid, 256, st);
    return true;
  }
  // few rows: as many threads as packs, one pack each; many rows: four packs a thread
  const bool few = a.rows < 2 * sms;
  const auto threads_for = [&](int per) { return ((packs + per - 1) / per + 31) / 32 * 32; };
  int per = few ? 1 : 4;
  while (threads_for(per) > 1024) per *= 2;
  if (per > 8) return false;
  const int threads = threads_for(per);
  const unsigned grid = grid_of(a.rows, sms * (2048 / threads));
  if (per == 1) launch_forward_as<T, kV, 1, false>(a, grid, threads, st);
  else if (per == 2) launch_forward_as<T, kV, 2, false>(a, grid, threads, st);
  else if (per == 4) launch_forward_as<T, kV, 4, false>(a, grid, threads, st);
  else launch_forward_as<T, kV, 8, false>(a, grid, threads, st);
  return true;
}

template <typename T>
int launch_forward(const NormArgs& a, cudaStream_t st) {
  using A = typename Elem<T>::Acc;
  constexpr int kV = kVec16<T>;
  const bool packed = rows_on_16_bytes<T>(a.x, a.ldx) && rows_on_16_bytes<T>(a.y, a.ldy) &&
                      rows_on_16_bytes<T>(a.gamma, 0) && rows_on_16_bytes<T>(a.beta, 0);
  if (packed ? launch_forward_packed<T, kV>(a, st) : launch_forward_packed<T, 1>(a, st)) return 1;
  layernorm_long_kernel<T><<<grid_of(a.rows, static_cast<long long>(lib_num_sms()) * 2), 1024, 0, st>>>(
      static_cast<const T*>(a.x), static_cast<const T*>(a.gamma), static_cast<const T*>(a.beta), static_cast<T*>(a.y),
      static_cast<A*>(a.mean), static_cast<A*>(a.inv_std), a.rows, a.n, a.ldx, a.ldy, static_cast<A>(a.epsilon));
  return 1;
}

struct NormGradArgs {
  const void *grad_out, *x, *mean, *inv_std, *gamma;
  void *grad_in, *grad_gamma, *grad_beta;
  long long rows, ldg, ldx, ldi;
  int n;
};

// threads of a row, packs a thread holds and blocks, for rows that fit into registers; kN = 0: they do not
struct GradShape { int per, threads; bool warp; unsigned grid; };

template <typename T, int kV> GradShape gradients_shape(const NormGradArgs& a) {
  const long long sms = lib_num_sms();
  const int packs = (a.n + kV - 1) / kV;
  // registers of a pack: the row and the next row (twice two), the weights, two sums of kV
  constexpr int kMost = 4;
  if (packs <= 32 * 2) {
    const int per = packs <= 32 ? 1 : 2;
    return {per, 256, true, grid_of((a.rows + 7) / 8, sms * 4)};
  }
  const auto threads_for = [&](int per) { return ((packs + per - 1) / per + 31) / 32 * 32; };
  int per = 2;
  while (threads_for(per) > 512 && per < kMost) per *= 2;
  if (threads_for(per) > 512) return {0, 0, false, 0};
  const int threads = threads_for(per);
  return {per, threads, false, grid_of(a.rows, sms * (threads <= 128 ? 6 : threads <= 256 ? 3 : 1))};
}

template <typename T, int kV, int kN, bool kWarp>
void launch_gradients_as(const NormGradArgs& a, const GradShape& q, void* partial, cudaStream_t st) {
  using A = typename Elem<T>::Acc;
  layernorm_gradients_kernel<T, kV, kN, kWarp><<<q.grid, q.threads, 0, st>>>(
      static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), static_cast<const A*>(a.mean),
      static_cast<const A*>(a.inv_std), static_cast<const T*>(a.gamma), static_cast<T*>(a.grad_in),
      static_cast<A*>(partial), a.rows, a.n, a.ldg, a.ldx, a.ldi);
}

template <typename T, int kV>
void launch_gradients_packed(const NormGradArgs& a, const GradShape& q, void* partial, cudaStream_t st) {
  if (q.warp) {
    if (q.per == 1) launch_gradients_as<T, kV, 1, true>(a, q, partial, st);
    else launch_gradients_as<T, kV, 2, true>(a, q, partial, st);
  } else if (q.per == 2) {
    launch_gradients_as<T, kV, 2, false>(a, q, partial, st);
  } else {
    launch_gradients_as<T, kV, 4, false>(a, q, partial, st);
  }
}

template <typename T>
int launch_gradients(const NormGradArgs& a, OpScratch& scratch, cudaStream_t st) {
  using A = typename Elem<T>::Acc;
  constexpr int kV = kVec16<T>;
  const bool packed = rows_on_16_bytes<T>(a.grad_out, a.ldg) && rows_on_16_bytes<T>(a.x, a.ldx) &&
                      rows_on_16_bytes<T>(a.grad_in, a.ldi) && rows_on_16_bytes<T>(a.gamma, 0);
  const GradShape q = packed ? gradients_shape<T, kV>(a) : gradients_shape<T, 1>(a);
  const bool weights = a.grad_gamma || a.grad_beta;
  const size_t row_of_sums = 2 * static_cast<size_t>(a.n) * sizeof(A);
  int groups = 0, launches = 1;
  A* partial = nullptr;
  if (q.per) {
    groups = static_cast<int>(q.grid) * (q.warp ? q.threads / 32 : 1);
    if (weights) {
      partial = reinterpret_cast<A*>(scratch.reserve(groups * row_of_sums, st));
      if (!partial) return -1;
    }
    if (packed) launch_gradients_packed<T, kV>(a, q, partial, st);
    else launch_gradients_packed<T, 1>(a, q, partial, st);
  } else {
    const long long sms = lib_num_sms();
    const unsigned col_blocks = static_cast<unsigned>((a.n + 255) / 256);
    groups = static_cast<int>(grid_of(a.rows, sms * 8 / col_blocks < 1 ? 1 : sms * 8 / col_blocks));
    const size_t head = (static_cast<size_t>(a.rows) * 2 * sizeof(A) + 255) & ~static_cast<size_t>(255);
    uint8_t* base = scratch.reserve(head + (weights ? groups * row_of_sums : 0), st);
    if (!base) return -1;
    A* sums = reinterpret_cast<A*>(base);
    if (weights) partial = reinterpret_cast<A*>(base + head);
    layernorm_row_sums_kernel<T><<<grid_of(a.rows, sms * 4), 512, 0, st>>>(
        static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), static_cast<const A*>(a.mean),
        static_cast<const A*>(a.inv_std), static_cast<const T*>(a.gamma), sums, a.rows, a.n, a.ldg, a.ldx);
    layernorm_columns_kernel<T><<<dim3(col_blocks, static_cast<unsigned>(groups)), 256, 0, st>>>(
        static_cast<const T*>(a.grad_out), static_cast<const T*>(a.x), static_cast<const A*>(a.mean),
        static_cast<const A*>(a.inv_std), static_cast<const T*>(a.gamma), sums, static_cast<T*>(a.grad_in), partial, a.rows,
        a.n, a.ldg, a.ldx, a.ldi);
    launches = 2;
  }
  if (weights) {
    layernorm_join_kernel<A><<<static_cast<unsigned>((2LL * a.n + 31) / 32), 256, 0, st>>>(
        partial, groups, a.n, static_cast<A*>(a.grad_gamma), static_cast<A*>(a.grad_beta));
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
  a.grad_in = grad_in; a.grad_gamma = grad_gamma; a.grad_beta = grad_beta;
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
