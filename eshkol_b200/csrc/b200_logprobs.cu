// Log probabilities of given tokens with entropy and top alternatives, and the gradient of the logits,
// on f64, f32, f16 and bf16 logits.
//
//   lse = log sum_j exp x_j,   logprob = x_token - lse,   entropy = -sum_j p_j log p_j,   p_j = exp(x_j - lse)
//   grad_j = g ([j = token] - p_j) - h p_j (log p_j + entropy)     (g, h: gradients of logprob and entropy)
//
// Forward: one pass over a row with a running reference m, s = sum exp(x - m) and t = sum exp(x - m) (x - m);
// lse = m + log s and entropy = log s - t / s.  A row is read once from HBM, by one block or, when the
// rows are few, by a cluster of blocks that join their m, s, t and alternatives through distributed
// shared memory, so there is no workspace and no second launch.
//
// Top alternatives cost the pass nothing but the threads' own maxima: the n-th largest of them bounds
// the n-th largest logit from below, so every alternative lies in the places of a thread whose maximum
// reaches the bound, and only those threads' places (about n of them) are read again.  Order: larger
// logit first, equal logits by index, kept exactly by comparing (logit, index) as one key.
//
// Entries of minus infinity have probability zero and add nothing.  A row of nothing else has lse minus
// infinity, entropy zero and a zero gradient.  NaN or plus infinity makes the row's outputs NaN.
#include <math.h>
#include <stdio.h>

#include <cooperative_groups.h>

#include "b200_elem.cuh"
#include "b200_tiers.h"

namespace b200 {
namespace {
namespace cg = cooperative_groups;

constexpr int kMaxTop = 32;  // one alternative per lane

// ------------------------------------------------------------------ order keys
// value keys order like the numbers, -0 beside +0 as equal, every number above zero's place; 0 stands
// for "nothing" and for NaN
template <typename T> struct KeyOf { using type = uint32_t; };
template <> struct KeyOf<double> { using type = unsigned long long; };

__device__ __forceinline__ uint32_t value_key(float v) {
  if (!(v == v)) return 0u;
  const uint32_t b = __float_as_uint(v + 0.f);  // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long value_key(double v) {
  if (!(v == v)) return 0ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ double key_value(unsigned long long k) {
  return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}

// (value key, 2^32 - 1 - index): the larger one is the better alternative; {0, 0} is none
template <typename K> struct Entry {
  K key;
  uint32_t rank;
};
template <typename K> __device__ __forceinline__ bool better(const Entry<K>& a, const Entry<K>& b) {
  return a.key > b.key || (a.key == b.key && a.rank > b.rank);
}
template <typename K> __device__ __forceinline__ Entry<K> best_of(const Entry<K>& a, const Entry<K>& b, bool want_better) {
  return (better(a, b) == want_better) ? a : b;
}
template <typename K> __device__ __forceinline__ Entry<K> shfl_xor(const Entry<K>& a, int o) {
  Entry<K> r;
  r.key = __shfl_xor_sync(0xffffffffu, a.key, o);
  r.rank = __shfl_xor_sync(0xffffffffu, a.rank, o);
  return r;
}
// plain keys go through the same networks
__device__ __forceinline__ uint32_t best_of(uint32_t a, uint32_t b, bool want) { return ((a > b) == want) ? a : b; }
__device__ __forceinline__ unsigned long long best_of(unsigned long long a, unsigned long long b, bool want) {
  return ((a > b) == want) ? a : b;
}
__device__ __forceinline__ uint32_t shfl_xor(uint32_t a, int o) { return __shfl_xor_sync(0xffffffffu, a, o); }
__device__ __forceinline__ unsigned long long shfl_xor(unsigned long long a, int o) {
  return __shfl_xor_sync(0xffffffffu, a, o);
}

// the last five steps of a bitonic sort: lanes hold a bitonic sequence, afterwards the largest is in lane 0
template <typename E> __device__ __forceinline__ E merge_down(E e) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) e = best_of(e, shfl_xor(e, o), (lane & o) == 0);
  return e;
}
// 32 values over the lanes, largest first
template <typename E> __device__ __forceinline__ E sort_down(E e) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 16; size <<= 1) {
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1)
      e = best_of(e, shfl_xor(e, o), ((lane & o) == 0) == ((lane & size) == 0));
  }
  return merge_down(e);
}
// the 32 best of a sorted list over the lanes and another whose places are given backwards
template <typename E> __device__ __forceinline__ E merge_lists(E list, E other_backwards) {
  return merge_down(best_of(list, other_backwards, true));
}

// ------------------------------------------------------------------ running sums
__device__ __forceinline__ float exp_of(float v) {  // results below 2^-126 are zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }
// v, or the bound when v is below it; NaN stays
__device__ __forceinline__ float floor_at(float v, float bound) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(bound));
  return r;
}
__device__ __forceinline__ double floor_at(double v, double bound) { return v < bound ? bound : v; }
template <typename A> constexpr A kFar = A(-1e30);  // exp of it is zero, a product with it finite
template <typename A> __device__ __forceinline__ A lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -3.402823466e38f; }
template <> __device__ __forceinline__ double lowest<double>() { return -1.7976931348623157e308; }
template <typename A> constexpr A kSlack = A(4);  // how far a value may pass the reference before it moves

// s and t relative to the finite reference m
template <typename A> struct Sums {
  A m, s, t;
};
template <typename A> __device__ __forceinline__ void move_reference(Sums<A>& a, A m) {
  const A d = floor_at(a.m - m, kFar<A>);
  const A f = exp_of(d);
  a.t = (a.t + d * a.s) * f;
  a.s *= f;
  a.m = m;
}
template <typename A> __device__ __forceinline__ Sums<A> joined(Sums<A> a, Sums<A> b) {
  const A m = a.m > b.m ? a.m : b.m;
  move_reference(a, m);
  move_reference(b, m);
  a.s += b.s;
  a.t += b.t;
  return a;
}
template <typename A> __device__ __forceinline__ Sums<A> warp_joined(Sums<A> a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums<A> b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
    a = joined(a, b);
  }
  return a;
}

// ------------------------------------------------------------------ a row on the 16-byte grid
// Place v of a row holds the elements v*kV - shift + (0 .. kV-1), kV of them in one aligned 16-byte
// word; the first and last place may reach beyond the row and are read element by element.
template <typename T> struct RowGrid {
  static constexpr int kV = kVec16<T>;
  const T* row;
  int n, shift, places;
  __device__ __forceinline__ RowGrid(const T* r, int len) : row(r), n(len) {
    shift = elems_past_boundary(r);
    places = (len + shift + kV - 1) / kV;
  }
  __device__ __forceinline__ int first(int place) const { return place * kV - shift; }
  // whole in the row
  __device__ __forceinline__ bool inside(int place) const { return first(place) >= 0 && first(place) + kV <= n; }
  __device__ __forceinline__ Pack<T, kV> load(int place, T otherwise) const {
    const int c = first(place);
    if (c >= 0 && c + kV <= n) return *reinterpret_cast<const Pack<T, kV>*>(row + c);
    Pack<T, kV> p;
#pragma unroll
    for (int j = 0; j < kV; ++j) p.v[j] = (c + j >= 0 && c + j < n) ? row[c + j] : otherwise;
    return p;
  }
};

template <typename T> __device__ __forceinline__ T minus_infinity();
template <> __device__ __forceinline__ double minus_infinity<double>() { return -INFINITY; }
template <> __device__ __forceinline__ float minus_infinity<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __half minus_infinity<__half>() { return __ushort_as_half(0xfc00u); }
template <> __device__ __forceinline__ __nv_bfloat16 minus_infinity<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80u); }

struct LogprobArgs {
  const void* logits;
  const int64_t* tokens;
  void *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_index;
  long long ld;
  int vocab, top;
};

template <typename T, int kThreads> struct LogprobShared {
  using A = typename Elem<T>::Acc;
  using K = typename KeyOf<T>::type;
  static constexpr int kWarps = kThreads / 32;
  Sums<A> sums[kWarps];
  Sums<A> block;             // this block's, read by the cluster's first block
  K maxima[kWarps][32];      // the threads' maxima, sorted within their warp
  K bound;
  int n_again;
  uint16_t again[kThreads];  // threads whose places are read again
  Entry<K> lists[kWarps][32];
  Entry<K> found[kWarps][32 * kVec16<T>];
  Entry<K> best[32];         // this block's alternatives, read by the cluster's first block
};

// One row per cluster; the cluster's blocks take contiguous shares of the row's places.
template <typename T, int kThreads, bool kTop>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const LogprobArgs a) {
  using A = typename Elem<T>::Acc;
  using K = typename KeyOf<T>::type;
  constexpr int kV = kVec16<T>, kWarps = kThreads / 32, kAhead = 4;
  __shared__ LogprobShared<T, kThreads> sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const long long r = blockIdx.x / parts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const RowGrid<T> grid(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
  const int share = (grid.places + parts - 1) / parts;
  const int lo = min(part * share, grid.places), hi = min(lo + share, grid.places);
  const T nothing = minus_infinity<T>();

  Sums<A> q{lowest<A>(), A(0), A(0)};
  A mine = minus_infinity<A>();  // this thread's maximum
  for (int v0 = lo + tid; v0 < hi; v0 += kAhead * kThreads) {
    Pack<T, kV> p[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = v0 + u * kThreads;
      if (v < hi) {
        p[u] = grid.load(v, nothing);
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j) p[u].v[j] = nothing;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      A x[kV], most = minus_infinity<A>();
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        x[j] = Elem<T>::widen(p[u].v[j]);
        most = most < x[j] ? x[j] : most;  // a NaN is passed over
      }
      mine = mine < most ? most : mine;
      // exp(x - m) may grow to exp(4): as exact as below one, and the reference seldom moves
      if (most > q.m + kSlack<A>) move_reference(q, most);
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const A d = floor_at(x[j] - q.m, kFar<A>);
        const A e = exp_of(d);
        q.s += e;
        q.t += e * d;
      }
    }
  }
  q = warp_joined(q);
  if (lane == 0) sm.sums[warp] = q;
  __syncthreads();
  if (warp == 0) {
    Sums<A> b = lane < kWarps ? sm.sums[lane] : Sums<A>{lowest<A>(), A(0), A(0)};
    b = warp_joined(b);
    if (lane == 0) sm.block = b;
  }

  if (kTop) {
    // the bound: the top-th largest of the threads' maxima (nothing, if fewer threads saw any logit)
    const bool saw = lo + tid < hi;
    const K own = saw ? value_key(mine) : K(0);
    sm.maxima[warp][lane] = sort_down(own);
    if (tid == 0) sm.n_again = 0;
    __syncthreads();
    if (warp == 0) {
      K list = sm.maxima[0][lane];
#pragma unroll 1
      for (int w = 1; w < kWarps; ++w) list = merge_lists(list, sm.maxima[w][31 - lane]);
      const K b = __shfl_sync(0xffffffffu, list, a.top - 1);
      if (lane == 0) sm.bound = b;
    }
    __syncthreads();
    const K bound = sm.bound;
    if (saw && own >= bound) sm.again[atomicAdd(&sm.n_again, 1)] = static_cast<uint16_t>(tid);
    __syncthreads();
    const int n_again = sm.n_again;  // their order does not matter: entries are ordered by key and index
    Entry<K> list{K(0), 0u};
    for (int i = warp; i < n_again; i += kWarps) {
      const int who = sm.again[i];
      for (int v0 = lo + who; v0 < hi; v0 += 32 * kThreads) {
        const int v = v0 + lane * kThreads;
        const K worst = __shfl_sync(0xffffffffu, list.key, 31);
        const uint32_t worst_rank = __shfl_sync(0xffffffffu, list.rank, 31);
        const Entry<K> last{worst, worst_rank};
        Entry<K> e[kV];
        unsigned take = 0;
        if (v < hi) {
          const Pack<T, kV> p = grid.load(v, nothing);
          const int c = grid.first(v);
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            e[j].key = value_key(Elem<T>::widen(p.v[j]));
            e[j].rank = 0xffffffffu - static_cast<uint32_t>(c + j);
            // NaN has key 0 and is no alternative; neither are places beyond the row
            if (e[j].key != K(0) && e[j].key >= bound && c + j >= 0 && c + j < a.vocab && better(e[j], last)) take |= 1u << j;
          }
        }
        const int count = __popc(take);
        int at = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += up;
        }
        const int total = __shfl_sync(0xffffffffu, at, 31);
        if (total == 0) continue;
        at -= count;
#pragma unroll
        for (int j = 0; j < kV; ++j)
          if (take & (1u << j)) sm.found[warp][at++] = e[j];
        __syncwarp();
        for (int b = 0; b < total; b += 32) {
          const Entry<K> c = sort_down(b + lane < total ? sm.found[warp][b + lane] : Entry<K>{K(0), 0u});
          Entry<K> back;
          back.key = __shfl_sync(0xffffffffu, c.key, 31 - lane);
          back.rank = __shfl_sync(0xffffffffu, c.rank, 31 - lane);
          list = merge_lists(list, back);
        }
        __syncwarp();
      }
    }
    sm.lists[warp][lane] = list;
    __syncthreads();
    if (warp == 0) {
      const int used = min(n_again, kWarps);
#pragma unroll 1
      for (int w = 1; w < used; ++w) list = merge_lists(list, sm.lists[w][31 - lane]);
      sm.best[lane] = list;
    }
  }

  // the cluster's first block joins the others' sums and alternatives
  if (parts > 1) cluster.sync();
  else __syncthreads();
  if (part == 0 && warp == 0) {
    Sums<A> all{lowest<A>(), A(0), A(0)};
    if (lane < parts) all = *cluster.map_shared_rank(&sm.block, lane);
    all = warp_joined(all);
    const bool empty = all.s == A(0);
    const A log_s = log_of(all.s);
    const A lse = empty ? minus_infinity<A>() : all.m + log_s;
    if (lane == 0) {
      if (a.lse) static_cast<A*>(a.lse)[r] = lse;
      if (a.entropy) static_cast<A*>(a.entropy)[r] = empty ? A(0) : log_s - all.t / all.s;
      if (a.logprob) {
        const int64_t token = a.tokens[r];
        A lp = A(0);  // no token was given
        if (token >= a.vocab) {
          lp = A(NAN);
        } else if (token >= 0) {
          const A x = Elem<T>::widen(grid.row[token]);
          // x - lse, by way of the reference: x - m is exact for a likely token where lse is rounded
          lp = (x == minus_infinity<A>() && lse == lse) ? x : (x - all.m) - log_s;
        }
        static_cast<A*>(a.logprob)[r] = lp;
      }
    }
    if (kTop) {
      Entry<K> list = sm.best[lane];
#pragma unroll 1
      for (int b = 1; b < parts; ++b) list = merge_lists(list, *cluster.map_shared_rank(&sm.best[31 - lane], b));
      if (lane < a.top) {
        const bool none = list.key == K(0);
        const A x = none ? A(NAN) : static_cast<A>(key_value(list.key));
        if (a.top_index) a.top_index[r * a.top + lane] = none ? -1 : static_cast<int64_t>(0xffffffffu - list.rank);
        if (a.top_logprob)
          static_cast<A*>(a.top_logprob)[r * a.top + lane] =
              (x == minus_infinity<A>() && lse == lse) ? x : (x - all.m) - log_s;
      }
    }
  }
  if (parts > 1) cluster.sync();  // no block leaves while its shared memory may still be read
}

// ------------------------------------------------------------------ gradient
struct LogprobGradArgs {
  const void* logits;
  const int64_t* tokens;
  const void *lse, *entropy, *grad_logprob, *grad_entropy;
  void* grad_logits;
  long long ld, ldg;
  int vocab, parts;
};

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_gradient_kernel(const LogprobGradArgs a) {
  using A = typename Elem<T>::Acc;
  constexpr int kV = kVec16<T>, kAhead = 4;
  const long long r = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x - r * a.parts);
  const T* in = static_cast<const T*>(a.logits) + r * a.ld;
  T* out = static_cast<T*>(a.grad_logits) + r * a.ldg;
  // places on the output's 16-byte grid; the input is read in words too where it lies the same way
  const RowGrid<T> to(out, a.vocab);
  const RowGrid<T> from(in, a.vocab);
  const bool same = to.shift == from.shift;
  const int share = (to.places + a.parts - 1) / a.parts;
  const int lo = min(part * share, to.places), hi = min(lo + share, to.places);
  const int64_t token = a.tokens ? a.tokens[r] : -1;
  const A lse = static_cast<const A*>(a.lse)[r];
  A g = (a.grad_logprob && token >= 0) ? static_cast<const A*>(a.grad_logprob)[r] : A(0);
  const A h = a.grad_entropy ? static_cast<const A*>(a.grad_entropy)[r] : A(0);
  const A ent = a.grad_entropy ? static_cast<const A*>(a.entropy)[r] : A(0);
  if (token >= a.vocab) g = A(NAN);  // a token that does not exist: the row says so
  const A level = g + h * ent;
  const bool empty = lse == minus_infinity<A>();
  const T nothing = minus_infinity<T>();
  for (int v0 = lo + static_cast<int>(threadIdx.x); v0 < hi; v0 += kAhead * 256) {
    Pack<T, kV> p[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = v0 + u * 256;
      if (v >= hi) continue;
      if (same) {
        p[u] = from.load(v, nothing);
      } else {
        const int c = to.first(v);
#pragma unroll
        for (int j = 0; j < kV; ++j) p[u].v[j] = (c + j >= 0 && c + j < a.vocab) ? in[c + j] : nothing;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = v0 + u * 256;
      if (v >= hi) continue;
      const int c = to.first(v);
      Pack<T, kV> o;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const A x = Elem<T>::widen(p[u].v[j]);
        const A lp = floor_at(x - lse, kFar<A>);
        const A prob = empty ? A(0) : exp_of(lp);
        A d = -prob * (h * (empty ? A(0) : lp) + level);
        if (c + j == token) d += g;
        o.v[j] = Elem<T>::narrow(d);
      }
      if (to.inside(v)) {
        *reinterpret_cast<Pack<T, kV>*>(out + c) = o;
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j)
          if (c + j >= 0 && c + j < a.vocab) out[c + j] = o.v[j];
      }
    }
  }
}

int finish(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError(); else cudaGetLastError();
  if (e != cudaSuccess) {
    fprintf(stderr, "[eshkol-b200] token log probabilities: launch failed: %s\n", cudaGetErrorString(e));
    return -1;
  }
  count_launches(1);
  return 0;
}

template <typename T, int kThreads, bool kTop>
cudaError_t launch_parts(const LogprobArgs& a, long long rows, int parts, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(parts);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, kThreads, kTop>, a);
}

template <typename T> int launch_forward(const LogprobArgs& a, long long rows, cudaStream_t st) {
  // blocks of a row: as many as give every SM four, while each still has 2048 elements
  const long long want = (4LL * lib_num_sms() + rows - 1) / rows;
  int parts = 1;
  while (parts < 8 && parts * 2 <= want && a.vocab / (parts * 2) >= 2048) parts *= 2;
  return finish(a.top ? launch_parts<T, 256, true>(a, rows, parts, st) : launch_parts<T, 256, false>(a, rows, parts, st));
}

template <typename T> int launch_gradient(LogprobGradArgs a, long long rows, cudaStream_t st) {
  const long long want = (8LL * lib_num_sms() + rows - 1) / rows;
  int parts = 1;
  while (parts < 64 && parts * 2 <= want && a.vocab / (parts * 2) >= 1024) parts *= 2;
  a.parts = parts;
  token_logprobs_gradient_kernel<T><<<static_cast<unsigned>(rows * parts), 256, 0, st>>>(a);
  return finish(cudaSuccess);
}

bool shape_ok(uint64_t rows, uint64_t vocab, int dtype) {
  return rows <= (1ull << 24) && vocab >= 1 && vocab <= (1ull << 30) && dtype >= ESHKOL_B200_F64 && dtype <= ESHKOL_B200_BF16;
}
bool pitch_ok(uint64_t ld, uint64_t n) { return (ld == 0 || ld >= n) && ld <= (1ull << 40); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int eshkol_b200_token_logprobs_device(const void* logits, const int64_t* tokens, void* logprob, void* entropy, void* lse,
                                      void* top_logprob, int64_t* top_index, uint64_t rows, uint64_t vocab, uint64_t ld,
                                      uint64_t n_top, int dtype) {
  if (lib_device() < 0 || !shape_ok(rows, vocab, dtype) || !pitch_ok(ld, vocab)) return -1;
  if (n_top > static_cast<uint64_t>(kMaxTop) || n_top > vocab || (n_top == 0) != (!top_logprob && !top_index)) return -1;
  if ((logprob && !tokens) || (!logprob && !entropy && !lse && n_top == 0)) return -1;
  if (rows == 0) return 0;
  if (!logits) return -1;
  DeviceScope scope(lib_device());
  if (!scope.ok()) return -1;
  LogprobArgs a;
  a.logits = logits; a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.lse = lse;
  a.top_logprob = top_logprob; a.top_index = top_index;
  a.ld = static_cast<long long>(ld ? ld : vocab); a.vocab = static_cast<int>(vocab); a.top = static_cast<int>(n_top);
  const long long n = static_cast<long long>(rows);
  switch (dtype) {
    case ESHKOL_B200_F64: return launch_forward<double>(a, n, lib_stream());
    case ESHKOL_B200_F32: return launch_forward<float>(a, n, lib_stream());
    case ESHKOL_B200_F16: return launch_forward<__half>(a, n, lib_stream());
    default: return launch_forward<__nv_bfloat16>(a, n, lib_stream());
  }
}

int eshkol_b200_token_logprobs_gradient_device(const void* logits, const int64_t* tokens, const void* lse,
                                               const void* entropy, const void* grad_logprob, const void* grad_entropy,
                                               void* grad_logits, uint64_t rows, uint64_t vocab, uint64_t ld,
                                               uint64_t ld_grad, int dtype) {
  if (lib_device() < 0 || !shape_ok(rows, vocab, dtype) || !pitch_ok(ld, vocab) || !pitch_ok(ld_grad, vocab)) return -1;
  if ((grad_logprob && !tokens) || (grad_entropy && !entropy) || (!grad_logprob && !grad_entropy)) return -1;
  if (rows == 0) return 0;
  LogprobGradArgs a;
  a.ld = static_cast<long long>(ld ? ld : vocab);
  a.ldg = static_cast<long long>(ld_grad ? ld_grad : vocab);
  if (!logits || !lse || !grad_logits || (grad_logits == logits && a.ld != a.ldg)) return -1;
  DeviceScope scope(lib_device());
  if (!scope.ok()) return -1;
  a.logits = logits; a.tokens = grad_logprob ? tokens : nullptr; a.lse = lse; a.entropy = entropy;
  a.grad_logprob = grad_logprob; a.grad_entropy = grad_entropy; a.grad_logits = grad_logits;
  a.vocab = static_cast<int>(vocab); a.parts = 1;
  const long long n = static_cast<long long>(rows);
  switch (dtype) {
    case ESHKOL_B200_F64: return launch_gradient<double>(a, n, lib_stream());
    case ESHKOL_B200_F32: return launch_gradient<float>(a, n, lib_stream());
    case ESHKOL_B200_F16: return launch_gradient<__half>(a, n, lib_stream());
    default: return launch_gradient<__nv_bfloat16>(a, n, lib_stream());
  }
}

}  // extern "C"
