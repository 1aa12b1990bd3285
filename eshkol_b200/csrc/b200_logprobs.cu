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
// Top alternatives cost the pass nothing but the threads' own maxima: the n-th largest of the largest 64 or
// so of them bounds the n-th largest logit from below, so every alternative lies in the words of a thread
// whose maximum reaches the bound, and only those threads' words (about n of them) are read again.  Order:
// larger logit first, equal logits by index, kept exactly by comparing (logit, index) as one key; a
// candidate's rank is the number of better candidates.
//
// 4096 x 50257 bf16 with 8 alternatives takes 108 us (3.8 TB/s, 0.58 of the measured copy rate; without them
// 88), bound by instruction issue and the exponential unit, one exponential an element: 46 us by itself.  The
// gradient takes 134 us (6.1 TB/s, 0.94).
//
// Entries of minus infinity have probability zero and add nothing.  A row of nothing else has lse minus
// infinity, entropy zero and, for a gradient, g at the token and zeros.  NaN or plus infinity makes the row's
// outputs NaN.
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
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
    if (other > k) k = other;
  }
  return k;
}

// the warp's largest key, taken out of one lane that holds it
template <typename K> __device__ __forceinline__ K take_largest(K& left) {
  const K m = warp_max(left);
  const unsigned have = __ballot_sync(0xffffffffu, left == m);
  if (static_cast<int>(threadIdx.x & 31) == __ffs(have) - 1) left = K(0);
  return m;
}
template <typename K> __device__ __forceinline__ K exchange(K k, int o, bool larger) {
  const K other = __shfl_xor_sync(0xffffffffu, k, o);
  return (k > other) == larger ? k : other;
}
// the last steps of a bitonic sort: a bitonic sequence over the lanes becomes one with the largest first
template <typename K> __device__ __forceinline__ K merge_down(K k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = exchange(k, o, (lane & o) == 0);
  return k;
}
template <typename K> __device__ __forceinline__ K sort_down(K k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 16; size <<= 1) {
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) k = exchange(k, o, ((lane & o) == 0) == ((lane & size) == 0));
  }
  return merge_down(k);
}
// the 32 largest of a sorted list over the lanes and another one, given backwards
template <typename K> __device__ __forceinline__ K merge_lists(K list, K backwards) {
  return merge_down(list > backwards ? list : backwards);
}

// ------------------------------------------------------------------ running sums
__device__ __forceinline__ float exp_of(float v) {  // results below 2^-126 are zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ Duo<float> exp2_both(Duo<float> w) {
  float x, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(w.lo()));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(w.hi()));
  return Duo<float>::of(x, y);
}
__device__ __forceinline__ Duo<float> exp_both(Duo<float> d) { return exp2_both(d * both(kLog2e)); }
__device__ __forceinline__ Duo<double> exp_both(Duo<double> d) { return {exp(d.x), exp(d.y)}; }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }
// v, or the bound when v is below it; NaN stays
__device__ __forceinline__ float floor_at(float v, float bound) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(bound));
  return r;
}
__device__ __forceinline__ double floor_at(double v, double bound) { return v < bound ? bound : v; }
// Where differences end: exp of it is zero in f32 and f64, and so is a sum's or a gradient's part with it, while
// its product with a factor as large as 10^35 (f32) is still finite: zero times infinity would be NaN.
template <typename A> constexpr A kFar = A(-1e3);
template <typename A> __device__ __forceinline__ A lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -3.402823466e38f; }
template <> __device__ __forceinline__ double lowest<double>() { return -1.7976931348623157e308; }
constexpr float kNear = 64.f;  // references up to here may be multiplied by log2 e before the subtraction
template <typename A> constexpr A kSlack = A(4);  // how far a value may pass the reference before it moves

// s and t relative to the finite reference m
template <typename A> struct Sums {
  A m, s, t;
};
template <typename A> __device__ __forceinline__ Sums<A> nothing_yet() { return {lowest<A>(), A(0), A(0)}; }
// the sums of the warp's lanes on every lane: the largest reference first, then plain sums
template <typename A> __device__ __forceinline__ Sums<A> warp_joined(Sums<A> a) {
  A m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const A other = __shfl_xor_sync(0xffffffffu, m, o);
    m = m < other ? other : m;
  }
  const A d = floor_at(a.m - m, kFar<A>), f = exp_of(d);
  a.t = (a.t + d * a.s) * f;
  a.s *= f;
  block_sum2(a.s, a.t, static_cast<A*>(nullptr), 1);
  a.m = m;
  return a;
}

// ------------------------------------------------------------------ a row on the 16-byte grid
// Place v of a row holds the elements v*kV - shift + (0 .. kV-1), kV of them in one aligned 16-byte
// word.  The first and the last place may reach beyond the row; those between lie whole in it.
template <typename T> struct RowGrid {
  static constexpr int kV = kVec16<T>;
  const T* row;
  int n, shift, places;
  __device__ __forceinline__ RowGrid(const T* r, int len) : row(r), n(len) {
    shift = elems_past_boundary(r);
    places = (len + shift + kV - 1) / kV;
  }
  __device__ __forceinline__ int first(int place) const { return place * kV - shift; }
  __device__ __forceinline__ bool inside(int place) const { return first(place) >= 0 && first(place) + kV <= n; }
  __device__ __forceinline__ Word<T> whole(int place) const { return *reinterpret_cast<const Word<T>*>(row + first(place)); }
  __device__ __forceinline__ Word<T> load(int place, T otherwise) const {
    const int c = first(place);
    if (c >= 0 && c + kV <= n) return whole(place);
    Word<T> p;
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

// ------------------------------------------------------------------ a thread's share of a row
// What the packed pass cannot take is left to the plain one, element by element: for 16-bit logits the
// pass replaces minus infinity by a very low value (one packed instruction for two elements), which is
// right while the reference is far above it and differences stay finite.
template <typename T> struct Range { static constexpr float kLow = -1e38f, kHigh = 1e36f; };
template <> struct Range<__half> { static constexpr float kLow = -60000.f, kHigh = 65504.f; };

// the largest of kWords words, NaN passed over
template <typename T, int kWords> __device__ __forceinline__ typename Elem<T>::Acc largest(const Word<T> (&p)[kWords]) {
  using A = typename Elem<T>::Acc;
  if constexpr (std::is_same<T, __half>::value) {
    __half2 m = *reinterpret_cast<const __half2*>(&p[0]);
#pragma unroll
    for (int u = 0; u < kWords; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2(m, reinterpret_cast<const __half2*>(&p[u])[i]);
    return fmaxf(__low2float(m), __high2float(m));
  } else if constexpr (sizeof(T) == 2) {
    __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&p[0]);
#pragma unroll
    for (int u = 0; u < kWords; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2(m, reinterpret_cast<const __nv_bfloat162*>(&p[u])[i]);
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    A m = minus_infinity<A>();
#pragma unroll
    for (int u = 0; u < kWords; ++u)
#pragma unroll
      for (int j = 0; j < kVec16<T>; ++j) m = m < p[u].v[j] ? static_cast<A>(p[u].v[j]) : m;
    return m;
  }
}
// minus infinity replaced by the lowest finite value (bf16: what is below -1.99e38 by that), NaN kept
__device__ __forceinline__ Word<__half> without_infinity(Word<__half> p) {
  __half2* h = reinterpret_cast<__half2*>(&p);
  const __half2 low = __half2half2(__ushort_as_half(0xfbffu));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
  return p;
}
__device__ __forceinline__ Word<__nv_bfloat16> without_infinity(Word<__nv_bfloat16> p) {
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&p);
  const __nv_bfloat162 low = __bfloat162bfloat162(__ushort_as_bfloat16(0xff16u));  // -1.99e38: log2 e times it is finite
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
  return p;
}

template <typename T> struct Running {
  using A = typename Elem<T>::Acc;
  A m, most;        // the reference, the maximum so far
  Duo<A> s, t;
  __device__ __forceinline__ void start() {
    m = lowest<A>();
    most = minus_infinity<A>();
    s = t = both(A(0));
  }
  __device__ __forceinline__ void move(A to) {
    const A d = floor_at(m - to, kFar<A>), f = exp_of(d);
    t = fma2(s, both(d), t) * both(f);
    s = s * both(f);
    m = to;
  }
  __device__ __forceinline__ void plainly(const Word<T>& p) {
#pragma unroll
    for (int j = 0; j < kVec16<T>; ++j) {
      const A x = Elem<T>::widen(p.v[j]);
      most = most < x ? x : most;
      if (x > m) move(x);
      const A d = floor_at(x - m, kFar<A>), e = exp_of(d);
      s = s + Duo<A>::of(e, A(0));
      t = t + Duo<A>::of(e * d, A(0));
    }
  }
  template <int kWords> __device__ __forceinline__ void add(const Word<T> (&p)[kWords]) {
    const A top = largest<T, kWords>(p);
    most = most < top ? top : most;
    if constexpr (sizeof(T) == 2) {
      if (!(top >= Range<T>::kLow) || most > Range<T>::kHigh) {
#pragma unroll
        for (int u = 0; u < kWords; ++u) plainly(p[u]);
        return;
      }
    }
    // exp(x - m) may grow to exp(4): as exact as below one, and the reference seldom moves
    if (top > m + kSlack<A>) move(top);
    if constexpr (sizeof(T) == 2) {
      // (x - m) log2 e; t in units of log 2
      const Duo<A> scale = both(kLog2e);
      Duo<A> t2 = both(A(0));
      const auto sums = [&](auto exponent) {
#pragma unroll
        for (int u = 0; u < kWords; ++u) {
          Duo<A> x[kDuos<T>];
          widen_word(without_infinity(p[u]), x);
#pragma unroll
          for (int j = 0; j < kDuos<T>; ++j) {
            const Duo<A> d = exponent(x[j]), e = exp2_both(d);
            s = s + e;
            t2 = fma2(e, d, t2);
          }
        }
      };
      if (fabsf(m) <= kNear) {
        // one instruction: the roundings of log2 e and of m log2 e, 2^-26 + 2^-25 of m, shift all of the
        // thread's exponents alike, by less than 3e-6
        const Duo<A> minus = both(-m * kLog2e);
        sums([&](Duo<A> x) { return fma2(x, scale, minus); });
      } else {
        const Duo<A> minus = both(-m);
        sums([&](Duo<A> x) { return (x + minus) * scale; });
      }
      t = fma2(t2, both(kLn2), t);
    } else {
      const Duo<A> minus = both(-m);
#pragma unroll
      for (int u = 0; u < kWords; ++u) {
        Duo<A> x[kDuos<T>];
        widen_word(p[u], x);
#pragma unroll
        for (int j = 0; j < kDuos<T>; ++j) {
          Duo<A> d = x[j] + minus;
          d = Duo<A>::of(floor_at(d.lo(), kFar<A>), floor_at(d.hi(), kFar<A>));
          const Duo<A> e = exp_both(d);
          s = s + e;
          t = fma2(e, d, t);
        }
      }
    }
  }
};

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
  static constexpr int kCandidates = kThreads == 32 ? 256 : 512;
  Sums<A> sums[kWarps];
  Sums<A> block;             // this block's, read by the cluster's first block
  K largest[64];             // 64 / kWarps of the largest of each warp's maxima
  int n_again, n_found;
  uint16_t again[kThreads];  // threads whose words are read again
  Entry<K> found[kCandidates + kMaxTop];
  Entry<K> best[kMaxTop];    // this block's alternatives, read by the cluster's first block
};

// best[0 .. top) from the n candidates in `found`: an entry's place is the number of better ones, counted by
// a warp.  Between barriers; ends with one.
template <typename T, int kThreads>
__device__ __forceinline__ void select_best(LogprobShared<T, kThreads>& sm, int n, int top) {
  using K = typename KeyOf<T>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < n; i += kThreads / 32) {
    const Entry<K> mine = sm.found[i];
    int place = 0;
    for (int j = lane; j < n + lane; j += 32)  // as many turns for every lane
      place += __popc(__ballot_sync(0xffffffffu, j < n && better(sm.found[j < n ? j : 0], mine)));
    if (lane == 0 && place < top) sm.best[place] = mine;
  }
  if (static_cast<int>(threadIdx.x) >= n && static_cast<int>(threadIdx.x) < top) sm.best[threadIdx.x] = Entry<K>{K(0), 0u};
  __syncthreads();
}

// The words of 16 bytes that one thread takes from a row, kGroup at a time and kGroups groups ahead in its
// places of shared memory (cp.async: no registers, no barrier)
template <typename T, int kThreads, int kGroup, int kGroups> struct WordStream {
  const Word<T>* from;   // word 0 of this thread; the next are kThreads words further each
  Word<T>* places;       // [kGroups][kGroup][kThreads] of the block, this thread's column
  int count, asked;
  __device__ __forceinline__ void start(const Word<T>* first, int n, Word<T>* shared) {
    from = first;
    count = n;
    places = shared + threadIdx.x;
    asked = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) ask(g);
  }
  __device__ __forceinline__ void ask(int slot) {
#pragma unroll
    for (int u = 0; u < kGroup; ++u)
      if (asked + u < count) copy_async16(places + (slot * kGroup + u) * kThreads, from + static_cast<long long>(asked + u) * kThreads);
    asked += kGroup;
    commit_async();
  }
  // the words of the group that was asked for first; its slot is asked again afterwards
  __device__ __forceinline__ void take(int slot, Word<T> (&p)[kGroup]) {
    wait_async<kGroups - 1>();
#pragma unroll
    for (int u = 0; u < kGroup; ++u) p[u] = places[(slot * kGroup + u) * kThreads];
    ask(slot);
  }
};

// One row per cluster; the cluster's blocks take contiguous shares of the row's places.
template <typename T, int kThreads, bool kTop>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) token_logprobs_kernel(const LogprobArgs a) {
  using A = typename Elem<T>::Acc;
  using K = typename KeyOf<T>::type;
  constexpr int kV = kVec16<T>, kWarps = kThreads / 32, kGroup = 4, kGroups = 3;
  constexpr int kCandidates = LogprobShared<T, kThreads>::kCandidates;
  __shared__ LogprobShared<T, kThreads> sm;
  extern __shared__ __align__(16) unsigned char dyn[];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const long long r = blockIdx.x / parts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const RowGrid<T> grid(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);
  const int share = (grid.places + parts - 1) / parts;
  const int lo = min(part * share, grid.places), hi = min(lo + share, grid.places);
  // the row's ends, where a place is not whole, go to two threads; the whole places to all
  const bool end0 = lo < hi && !grid.inside(lo), end1 = hi - 1 > lo && !grid.inside(hi - 1);
  const int wlo = lo + (end0 ? 1 : 0), whi = hi - (end1 ? 1 : 0);
  const T nothing = minus_infinity<T>();
  // the token's logit is on its way while the row is read
  int64_t token = -1;
  T picked = nothing;
  if (part == 0 && tid == 0 && a.logprob) {
    token = a.tokens[r];
    if (token >= 0 && token < a.vocab) picked = grid.row[token];
  }

  Running<T> q;
  q.start();
  const int count = whi - wlo > tid ? (whi - wlo - tid + kThreads - 1) / kThreads : 0;
  WordStream<T, kThreads, kGroup, kGroups> words;
  words.start(reinterpret_cast<const Word<T>*>(grid.row + grid.first(wlo + tid)), count, reinterpret_cast<Word<T>*>(dyn));
  int slot = 0;
  for (int k = 0; k < count; k += kGroup) {
    Word<T> p[kGroup];
    words.take(slot, p);
    slot = slot + 1 == kGroups ? 0 : slot + 1;
    if (k + kGroup > count) {  // the last group: minus infinity adds nothing
#pragma unroll
      for (int u = 0; u < kGroup; ++u)
        if (k + u >= count) {
#pragma unroll
          for (int j = 0; j < kV; ++j) p[u].v[j] = nothing;
        }
    }
    q.template add<kGroup>(p);
  }
  wait_async<0>();
  const A mine = q.most;  // over the whole places
  constexpr int kSecond = kThreads > 32 ? 32 : 0;  // the thread of the other end
  if (tid == 0 && end0) q.plainly(grid.load(lo, nothing));
  if (tid == kSecond && end1) q.plainly(grid.load(hi - 1, nothing));
  {
    const Sums<A> w = warp_joined(Sums<A>{q.m, total(q.s), total(q.t)});
    if (lane == 0) sm.sums[warp] = w;
  }

  if (kTop) {
    // the bound: at least `top` threads' maxima reach it (zero when there are not so many among the 32)
    const bool saw = count > 0;
    const K own = saw ? value_key(mine) : K(0);
    constexpr int kOfWarp = kWarps > 1 ? 64 / kWarps : 32;
    const int of_warp = min(a.top, kOfWarp);
    if (kWarps > 1) {
      if (a.top <= 8) {
        K left = own;
#pragma unroll 1
        for (int i = 0; i < of_warp; ++i) {
          const K m = take_largest(left);
          if (lane == 0) sm.largest[warp * of_warp + i] = m;
        }
      } else {
        const K sorted = sort_down(own);
        if (lane < of_warp) sm.largest[warp * of_warp + lane] = sorted;
      }
    }
    if (tid == 0) sm.n_again = sm.n_found = 0;
    __syncthreads();
    K bound = K(0);
    if (kWarps == 1) {
      bound = __shfl_sync(0xffffffffu, sort_down(own), a.top - 1);
    } else {
      const int have = kWarps * of_warp;
      K first = lane < have ? sm.largest[lane] : K(0);
      const K second = lane + 32 < have ? sm.largest[lane + 32] : K(0);
      if (a.top <= 8 && have <= 32) {
#pragma unroll 1
        for (int i = 0; i < a.top; ++i) bound = take_largest(first);
      } else {
        bound = __shfl_sync(0xffffffffu, merge_lists(sort_down(first), __shfl_sync(0xffffffffu, sort_down(second), 31 - lane)), a.top - 1);
      }
    }
    if (saw && own >= bound) sm.again[atomicAdd(&sm.n_again, 1)] = static_cast<uint16_t>(tid);
    __syncthreads();
    // their words again, a thread's by a warp at a time; candidates in any order.  NaN fails the comparison.
    const A bound_value = bound == K(0) ? minus_infinity<A>() : static_cast<A>(key_value(bound));
    const auto consider = [&](A x, int index, const Entry<K>& worst) {
      if (x >= bound_value) {
        const Entry<K> e{value_key(x), 0xffffffffu - static_cast<uint32_t>(index)};
        if (better(e, worst)) {
          const int at = atomicAdd(&sm.n_found, 1);
          if (at < kCandidates) sm.found[at] = e;
        }
      }
    };
    const auto collect = [&](int place, const Entry<K>& worst) {  // any place
      const Word<T> p = grid.load(place, nothing);
      const int c = grid.first(place);
#pragma unroll
      for (int j = 0; j < kV; ++j)
        if (c + j >= 0 && c + j < a.vocab) consider(Elem<T>::widen(p.v[j]), c + j, worst);
    };
    const Entry<K> none{K(0), 0u};
    const int n_again = sm.n_again;
    for (int i = warp; i < n_again; i += kWarps)
      for (int place = wlo + sm.again[i] + lane * kThreads; place < whi; place += 32 * kThreads) {
        const Word<T> p[1] = {grid.whole(place)};
        if (largest<T, 1>(p) >= bound_value) {
#pragma unroll
          for (int j = 0; j < kV; ++j) consider(Elem<T>::widen(p[0].v[j]), grid.first(place) + j, none);
        }
      }
    if (tid == 0 && end0) collect(lo, none);
    if (tid == kSecond && end1) collect(hi - 1, none);
    __syncthreads();
    int n = sm.n_found;
    __syncthreads();  // all have read it before it is used again
    if (n <= kCandidates) {
      select_best<T, kThreads>(sm, n, a.top);
    } else {
      // more logits reach the bound than there is room for (many equal ones): the places in order, as many
      // at a time as there is room for, each time against the worst alternative so far
      constexpr int kPlaces = kCandidates / kV < kThreads ? kCandidates / kV : kThreads;
      if (tid < kMaxTop) sm.best[tid] = none;
      if (tid == 0) sm.n_found = 0;
      __syncthreads();
      for (int v0 = lo; v0 < hi; v0 += kPlaces) {
        const Entry<K> worst = sm.best[a.top - 1];
        if (tid < kPlaces && v0 + tid < hi) collect(v0 + tid, worst);
        __syncthreads();
        n = sm.n_found;  // at most kCandidates
        __syncthreads();
        if (n) {  // the same for all
          if (tid < a.top) sm.found[n + tid] = sm.best[tid];
          __syncthreads();
          if (tid == 0) sm.n_found = 0;
          select_best<T, kThreads>(sm, n + a.top, a.top);
        }
      }
    }
  } else {
    __syncthreads();
  }
  Sums<A> all = nothing_yet<A>();
  if (warp == 0) {
    if (kWarps == 1) {
      all = sm.sums[0];
    } else {
      if (lane < kWarps) all = sm.sums[lane];
      all = warp_joined(all);
    }
    if (parts > 1 && lane == 0) sm.block = all;
  }

  // the cluster's first block joins the others' sums and alternatives
  if (parts > 1) cluster.sync();
  if (part == 0) {
    if (kTop && parts > 1) {
      for (int i = tid; i < parts * a.top; i += kThreads)
        sm.found[i] = *cluster.map_shared_rank(&sm.best[i % a.top], i / a.top);
      __syncthreads();
      // empty entries equal one another and would take one place: the index makes them differ, and keeps
      // them behind every logit
      for (int i = tid; i < parts * a.top; i += kThreads)
        if (sm.found[i].key == K(0)) sm.found[i].rank = static_cast<uint32_t>(i);
      __syncthreads();
      select_best<T, kThreads>(sm, parts * a.top, a.top);
    }
    if (warp == 0) {
      if (parts > 1) {
        all = nothing_yet<A>();
        if (lane < parts) all = *cluster.map_shared_rank(&sm.block, lane);
        all = warp_joined(all);
      }
      const bool empty = all.s == A(0);
      const A log_s = log_of(all.s);
      const A lse = empty ? minus_infinity<A>() : all.m + log_s;
      if (lane == 0) {
        if (a.lse) static_cast<A*>(a.lse)[r] = lse;
        if (a.entropy) static_cast<A*>(a.entropy)[r] = empty ? A(0) : log_s - all.t / all.s;
        if (a.logprob) {
          A lp = A(0);  // no token was given
          if (token >= a.vocab) {
            lp = A(NAN);
          } else if (token >= 0) {
            const A x = Elem<T>::widen(picked);
            // x - lse, by way of the reference: x - m is exact for a likely token where lse is rounded
            lp = (x == minus_infinity<A>() && lse == lse) ? x : (x - all.m) - log_s;
          }
          static_cast<A*>(a.logprob)[r] = lp;
        }
      }
      if (kTop && lane < a.top) {
        const Entry<K> e = sm.best[lane];
        const bool none = e.key == K(0);
        const A x = none ? A(NAN) : static_cast<A>(key_value(e.key));
        if (a.top_index) a.top_index[r * a.top + lane] = none ? -1 : static_cast<int64_t>(0xffffffffu - e.rank);
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
__global__ void __launch_bounds__(256, 4) token_logprobs_gradient_kernel(const LogprobGradArgs a) {
  using A = typename Elem<T>::Acc;
  using D = Duo<A>;
  constexpr int kV = kVec16<T>, kD = kDuos<T>, kGroup = 2, kGroups = 4;
  extern __shared__ __align__(16) unsigned char dyn[];
  const long long r = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x - r * a.parts), tid = threadIdx.x;
  const T* in = static_cast<const T*>(a.logits) + r * a.ld;
  T* out = static_cast<T*>(a.grad_logits) + r * a.ldg;
  // places on the output's 16-byte grid; the input is read in words too where it lies the same way
  const RowGrid<T> to(out, a.vocab);
  const bool same = to.shift == elems_past_boundary(in);
  const int share = (to.places + a.parts - 1) / a.parts;
  const int lo = min(part * share, to.places), hi = min(lo + share, to.places);
  const bool end0 = lo < hi && !to.inside(lo), end1 = hi - 1 > lo && !to.inside(hi - 1);
  const int wlo = lo + (end0 ? 1 : 0), whi = hi - (end1 ? 1 : 0);
  const int count = whi - wlo > tid ? (whi - wlo - tid + 255) / 256 : 0;
  const int64_t token = a.tokens ? a.tokens[r] : -1;
  const A lse = static_cast<const A*>(a.lse)[r];
  A g = (a.grad_logprob && token >= 0) ? static_cast<const A*>(a.grad_logprob)[r] : A(0);
  const A h = a.grad_entropy ? static_cast<const A*>(a.grad_entropy)[r] : A(0);
  const A ent = a.grad_entropy ? static_cast<const A*>(a.entropy)[r] : A(0);
  if (token >= a.vocab) g = A(NAN);  // a token that does not exist: the row says so
  const bool empty = lse == minus_infinity<A>();  // then every logit is, and every probability zero
  const D minus_lse = both(empty ? A(0) : -lse), minus_h = both(-h), minus_level = both(-(g + h * ent));
  // -p (g + h (log p + entropy)) for a pair
  const auto slope = [&](D x) {
    D lp = x + minus_lse;
    lp = D::of(floor_at(lp.lo(), kFar<A>), floor_at(lp.hi(), kFar<A>));
    return exp_both(lp) * fma2(minus_h, lp, minus_level);
  };
  const auto single = [&](T x) { return slope(both(Elem<T>::widen(x))).lo(); };
  // the token's own element gets g more, with one rounding: by the thread that writes its place, which
  // keeps the logit in case the result goes over it
  const int where = (token >= 0 && token < a.vocab) ? static_cast<int>(token) : -1;
  const int place = where >= 0 ? (where + to.shift) / kV : -1;
  const bool mine = place >= lo && place < hi &&
                    tid == (place < wlo ? 0 : place >= whi ? 32 : (place - wlo) & 255);
  const A peak = mine ? single(in[where]) + g : A(0);

  if (same) {
    WordStream<T, 256, kGroup, kGroups> words;
    words.start(reinterpret_cast<const Word<T>*>(in + to.first(wlo + tid)), count, reinterpret_cast<Word<T>*>(dyn));
    Word<T>* at = reinterpret_cast<Word<T>*>(out + to.first(wlo + tid));
    int slot = 0;
    for (int k = 0; k < count; k += kGroup) {
      Word<T> p[kGroup];
      words.take(slot, p);
      slot = slot + 1 == kGroups ? 0 : slot + 1;
#pragma unroll
      for (int u = 0; u < kGroup; ++u) {
        if (k + u >= count) break;
        D x[kD];
        widen_word(p[u], x);
#pragma unroll
        for (int j = 0; j < kD; ++j) x[j] = slope(x[j]);
        at[static_cast<long long>(k + u) * 256] = to_word<T>(x);
      }
    }
    wait_async<0>();
  } else {
    for (int k = 0; k < count; ++k) {
      const int c = to.first(wlo + tid + k * 256);
      Word<T> p;
#pragma unroll
      for (int j = 0; j < kV; ++j) p.v[j] = in[c + j];
      D x[kD];
      widen_word(p, x);
#pragma unroll
      for (int j = 0; j < kD; ++j) x[j] = slope(x[j]);
      *reinterpret_cast<Word<T>*>(out + c) = to_word<T>(x);
    }
  }
  const auto finish_end = [&](int v) {  // a place that is not whole in the row
    const int c = to.first(v);
    for (int j = max(0, -c); j < kV && c + j < a.vocab; ++j) out[c + j] = Elem<T>::narrow(single(in[c + j]));
  };
  if (tid == 0 && end0) finish_end(lo);
  if (tid == 32 && end1) finish_end(hi - 1);
  if (mine) out[where] = Elem<T>::narrow(peak);
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
  cfg.dynamicSmemBytes = kThreads * 12 * 16;  // three groups of four words a thread
  cfg.stream = st;
  if (kThreads * 12 * 16 > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(token_logprobs_kernel<T, kThreads, kTop>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kThreads * 12 * 16);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(parts);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, kThreads, kTop>, a);
}

template <typename T, int kThreads> int launch_with(const LogprobArgs& a, long long rows, int parts, cudaStream_t st) {
  return finish(a.top ? launch_parts<T, kThreads, true>(a, rows, parts, st) : launch_parts<T, kThreads, false>(a, rows, parts, st));
}
template <typename T> int launch_forward(const LogprobArgs& a, long long rows, cudaStream_t st) {
  // A row costs a block some microseconds beside its bytes, the more the wider the block: rows that fill
  // the SMs go to a warp each up to 256 words and to four warps beyond; fewer rows to clusters of up to
  // eight large blocks, as many as give every SM two of them, while each still has 4096 elements
  const long long sms = lib_num_sms();
  const int words = a.vocab / kVec16<T>;
  if (a.top <= 8 && (words <= 64 || (words <= 256 && rows >= 4 * sms))) return launch_with<T, 32>(a, rows, 1, st);
  if (rows >= 4 * sms || a.vocab < 8192) return launch_with<T, 128>(a, rows, 1, st);
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2 * sms && a.vocab / (parts * 2) >= 4096) parts *= 2;
  return launch_with<T, 512>(a, rows, parts, st);
}

template <typename T> int launch_gradient(LogprobGradArgs a, long long rows, cudaStream_t st) {
  const long long want = (8LL * lib_num_sms() + rows - 1) / rows;
  int parts = 1;
  while (parts < 64 && parts * 2 <= want && a.vocab / (parts * 2) >= 1024) parts *= 2;
  a.parts = parts;
  token_logprobs_gradient_kernel<T><<<static_cast<unsigned>(rows * parts), 256, 256 * 8 * 16, st>>>(a);  // four groups of two words a thread
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
