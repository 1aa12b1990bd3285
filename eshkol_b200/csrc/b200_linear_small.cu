// The linear layer for a few rows (one decoded token, a handful of sequences), forward and gradient of x:
//
//   out[r][n] = sum over k of a[r][k] W(k, n)
//
// Every weight is read once and used `rows` times, so HBM bounds it: the tensor cores would only add the
// packing of what they cannot read in place and the loading of empty rows.  f32 arithmetic on the CUDA
// cores (packed pairs), W in either orientation and at any alignment.  A block takes a tile of columns, and
// where the tiles are few the blocks of a cluster share the reduction and add their sums up through
// distributed shared memory, in the order of the blocks: no scratch, one launch.
#include <cooperative_groups.h>
#include <stdio.h>

#include "b200_linear.cuh"
#include "b200_tiers.h"

namespace b200 {
namespace {
namespace cg = cooperative_groups;

constexpr int kChunk = 512;  // k values of a staged at a time
constexpr int kGroups = 4;   // groups of weights on their way per thread
// columns of a block: a word's worth per lane and 32 lanes, or four per warp
template <typename T> constexpr int kWideTile = 32 * kVec16<T>;
constexpr int kDeepTile = 32;
constexpr size_t kRingBytes = static_cast<size_t>(kGroups) * 4 * 256 * 16;

template <typename T, int R, bool kDeep> constexpr size_t small_shared() {
  const size_t work = kRingBytes + static_cast<size_t>(kChunk) * R * 4, sums = static_cast<size_t>(R) * kWideTile<T> * 4 * 9;
  return kDeep ? work + static_cast<size_t>(R) * kDeepTile * 4 : (work > sums ? work : sums);
}

// A thread's words of the weights, four at a time and kGroups groups ahead in its places of shared memory
// (cp.async), or read directly where that cannot be (16-bit rows off the 16-byte boundaries)
template <typename T, int kHow> struct Weights {
  Word<T>* places;
  int slot;
  __device__ __forceinline__ explicit Weights(unsigned char* shared) : places(reinterpret_cast<Word<T>*>(shared) + threadIdx.x), slot(0) {}
  // word u of the group now asked for: element c of a row of n, nothing where row is null
  __device__ __forceinline__ void ask(int group, int u, const T* row, long long c, long long n) const {
    if constexpr (kHow != kInRegisters) {
      Word<T>* to = places + ((group % kGroups) * 4 + u) * 256;
      if (row && c < n) copy_word<T, kHow>(to, row + c, 0, n - c < kVec16<T> ? static_cast<int>(n - c) : kVec16<T>);
    }
  }
  __device__ __forceinline__ Word<T> take(int group, int u, const T* row, long long c, long long n) const {
    const T zero = Elem<T>::narrow(0);
    const int left = !row || c >= n ? 0 : (n - c < kVec16<T> ? static_cast<int>(n - c) : kVec16<T>);
    Word<T> p;
    if constexpr (kHow != kInRegisters) {
      const Word<T>* from = places + ((group % kGroups) * 4 + u) * 256;
      if (left == kVec16<T>) return *from;
#pragma unroll
      for (int j = 0; j < kVec16<T>; ++j) p.v[j] = j < left ? from->v[j] : zero;
    } else {
#pragma unroll
      for (int j = 0; j < kVec16<T>; ++j) p.v[j] = j < left ? row[c + j] : zero;
    }
    return p;
  }
};

// a[r][k] with the slope, zero outside
template <typename T> __device__ __forceinline__ float activation_in(const SmallRows& q, int r, long long k, long long k_end) {
  if (r >= q.e.M || k >= k_end) return 0.f;
  float f = Elem<T>::widen(static_cast<const T*>(q.a)[r * q.lda + k]);
  if (q.slope) {
    const float z = Elem<T>::widen(static_cast<const T*>(q.pre)[r * q.ld_pre + k]);
    f *= slope_pair<sizeof(T) == 4>(both(z), q.slope).lo();
  }
  return f;
}

// the cluster's sums of a tile [R][columns], each block its share of them, and the epilogue
template <typename T, int R>
__device__ __forceinline__ void finish_tile(const SmallRows& q, cg::cluster_group& cluster, float* mine, int columns, long long n0) {
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  if (parts > 1) cluster.sync();
  else __syncthreads();
  for (int i = part * 256 + threadIdx.x; i < R * columns; i += parts * 256) {
    const int r = i / columns, c = i - r * columns;
    const long long n = n0 + c;
    if (r >= q.e.M || n >= q.e.N) continue;
    float acc[1] = {0.f};
    for (int b = 0; b < parts; ++b) acc[0] += *cluster.map_shared_rank(mine + i, b);
    const float bias[1] = {bias_at<T>(q.e, static_cast<int>(n))};
    Pack<T, 1> res, y, z;
    res.v[0] = q.e.residual ? static_cast<const T*>(q.e.residual)[r * q.e.ld_res + n] : Elem<T>::narrow(0);
    finish_elements<T, 1>(q.e, acc, bias, res, y, z);
    static_cast<T*>(q.e.out)[r * q.e.ldo + n] = y.v[0];
    if (q.e.pre) static_cast<T*>(q.e.pre)[r * q.e.ld_pre + n] = z.v[0];
  }
  if (parts > 1) cluster.sync();  // no block leaves while its sums may still be read
}

// R values next to each other in shared memory
template <int R> __device__ __forceinline__ void load_staged(const float* at, float (&f)[R]) {
  if constexpr (R >= 4) {
#pragma unroll
    for (int r = 0; r < R; r += 4) {
      const float4 v = *reinterpret_cast<const float4*>(at + r);
      f[r] = v.x; f[r + 1] = v.y; f[r + 2] = v.z; f[r + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) f[r] = at[r];
  }
}

// W stored [K][N]: a lane keeps a word's columns, the warps take the k values in turn
template <typename T, int R, int kHow>
__global__ void __launch_bounds__(256, R <= 8 ? 2 : 1) small_rows_wide_kernel(const __grid_constant__ SmallRows q) {
  constexpr int kV = kVec16<T>, kD = kDuos<T>, kTile = kWideTile<T>;
  extern __shared__ __align__(16) unsigned char dyn_small[];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long n0 = static_cast<long long>(blockIdx.x / parts) * kTile, c = n0 + lane * kV;
  const long long share = (q.K + parts - 1) / parts, k0 = min(part * share, q.K), k1 = min(k0 + share, q.K);
  float* stage = reinterpret_cast<float*>(dyn_small + kRingBytes);  // [k][R]
  Duo<float> acc[R][kD];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kD; ++j) acc[r][j] = both(0.f);
  // group g of this warp: the rows k0 + 32 g + warp + (0, 8, 16, 24)
  const Weights<T, kHow> weights(dyn_small);
  const T* w = static_cast<const T*>(q.w);
  const int groups = static_cast<int>((k1 - k0 + 31) / 32);
  const auto row_of = [&](int g, int u) -> const T* {
    const long long k = k0 + 32LL * g + warp + 8 * u;
    return k < k1 ? w + k * q.ldw : nullptr;
  };
  const auto ask = [&](int g) {
    if (g < groups) {
#pragma unroll
      for (int u = 0; u < 4; ++u) weights.ask(g, u, row_of(g, u), c, q.e.N);
    }
    if constexpr (kHow != kInRegisters) commit_async();
  };
#pragma unroll
  for (int g = 0; g < kGroups; ++g) ask(g);
  for (int g0 = 0; g0 < groups; g0 += kChunk / 32) {
    __syncthreads();  // the chunk before has been used
    for (int i = threadIdx.x; i < kChunk * R; i += 256) {
      const int r = i / kChunk, k = i - r * kChunk;  // neighbours read neighbours
      stage[k * R + r] = activation_in<T>(q, r, k0 + 32LL * g0 + k, k1);
    }
    __syncthreads();
    const int g1 = min(g0 + kChunk / 32, groups);
    for (int g = g0; g < g1; ++g) {
      if constexpr (kHow != kInRegisters) wait_async<kGroups - 1>();
      Word<T> p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = weights.take(g, u, row_of(g, u), c, q.e.N);
      ask(g + kGroups);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        Duo<float> d[kD];
        widen_word(p[u], d);
        float f[R];
        load_staged<R>(stage + ((g - g0) * 32 + warp + 8 * u) * R, f);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < kD; ++j) acc[r][j] = fma2(both(f[r]), d[j], acc[r][j]);
      }
    }
  }
  if constexpr (kHow != kInRegisters) wait_async<0>();
  // the warps' sums over what was the ring: [warp][R][columns], then their total behind them
  __syncthreads();
  float* sums = reinterpret_cast<float*>(dyn_small);
  float* mine = sums + 8 * R * kTile;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kD; ++j) {
      float* at = sums + (warp * R + r) * kTile + lane * kV + 2 * j;
      at[0] = acc[r][j].lo();
      at[1] = acc[r][j].hi();
    }
  __syncthreads();
  for (int i = threadIdx.x; i < R * kTile; i += 256) {
    float s = sums[i];
#pragma unroll
    for (int b = 1; b < 8; ++b) s += sums[b * R * kTile + i];
    mine[i] = s;
  }
  finish_tile<T, R>(q, cluster, mine, kTile, n0);
}

// W stored [N][K]: a warp keeps four columns, its lanes take a word of k values each
template <typename T, int R, int kHow>
__global__ void __launch_bounds__(256, R <= 8 ? 2 : 1) small_rows_deep_kernel(const __grid_constant__ SmallRows q) {
  constexpr int kV = kVec16<T>, kD = kDuos<T>, kTurn = 32 * kV;  // k values of a warp's group
  extern __shared__ __align__(16) unsigned char dyn_small[];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long n0 = static_cast<long long>(blockIdx.x / parts) * kDeepTile, n = n0 + warp * 4;
  // shares on whole groups of eight, so that aligned rows stay aligned
  const long long share = ((q.K + parts - 1) / parts + 7) / 8 * 8, k0 = min(part * share, q.K), k1 = min(k0 + share, q.K);
  float* stage = reinterpret_cast<float*>(dyn_small + kRingBytes);  // [R][k]
  float* mine = stage + kChunk * R;
  Duo<float> acc[4][R];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[i][r] = both(0.f);
  const Weights<T, kHow> weights(dyn_small);
  const T* w = static_cast<const T*>(q.w) + n * q.ldw;
  const int groups = static_cast<int>((k1 - k0 + kTurn - 1) / kTurn);
  const auto ask = [&](int g) {
    if (g < groups) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        weights.ask(g, i, n + i < q.e.N ? w + i * q.ldw : nullptr, k0 + static_cast<long long>(g) * kTurn + lane * kV, k1);
    }
    if constexpr (kHow != kInRegisters) commit_async();
  };
#pragma unroll
  for (int g = 0; g < kGroups; ++g) ask(g);
  for (int g0 = 0; g0 < groups; g0 += kChunk / kTurn) {
    __syncthreads();
    for (int i = threadIdx.x; i < kChunk * R; i += 256) {
      const int r = i / kChunk, k = i - r * kChunk;
      stage[i] = activation_in<T>(q, r, k0 + static_cast<long long>(g0) * kTurn + k, k1);
    }
    __syncthreads();
    const int g1 = min(g0 + kChunk / kTurn, groups);
    for (int g = g0; g < g1; ++g) {
      if constexpr (kHow != kInRegisters) wait_async<kGroups - 1>();
      Duo<float> d[4][kD];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        widen_word(weights.take(g, i, n + i < q.e.N ? w + i * q.ldw : nullptr, k0 + static_cast<long long>(g) * kTurn + lane * kV, k1), d[i]);
      ask(g + kGroups);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float* at = stage + r * kChunk + (g - g0) * kTurn + lane * kV;
        float f[kV];
        load_staged<kV>(at, f);
#pragma unroll
        for (int j = 0; j < kD; ++j) {
          const Duo<float> x = Duo<float>::of(f[2 * j], f[2 * j + 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i][r] = fma2(x, d[i][j], acc[i][r]);
        }
      }
    }
  }
  if constexpr (kHow != kInRegisters) wait_async<0>();
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float s = warp_sum(total(acc[i][r]));
      if (lane == 0) mine[r * kDeepTile + warp * 4 + i] = s;
    }
  finish_tile<T, R>(q, cluster, mine, kDeepTile, n0);
}

template <typename T, int R, int kHow> cudaError_t launch_kernel(const cudaLaunchConfig_t& base, const SmallRows& q) {
  cudaLaunchConfig_t cfg = base;
  if (q.k_contiguous) {
    cfg.dynamicSmemBytes = small_shared<T, R, true>();
    return cudaLaunchKernelEx(&cfg, small_rows_deep_kernel<T, R, kHow>, q);
  }
  cfg.dynamicSmemBytes = small_shared<T, R, false>();
  return cudaLaunchKernelEx(&cfg, small_rows_wide_kernel<T, R, kHow>, q);
}
template <typename T> constexpr int kUnaligned = sizeof(T) >= 4 ? kByElements : kInRegisters;

template <typename T, int R> int launch_rows(const SmallRows& q, cudaStream_t st) {
  const int tile = q.k_contiguous ? kDeepTile : kWideTile<T>;
  const long long tiles = (static_cast<long long>(q.e.N) + tile - 1) / tile, sms = lib_num_sms();
  // blocks per tile: as many as the SMs hold at once, while each still has 256 k values (a second wave of
  // blocks costs more than longer blocks: 512 blocks where 444 fit took 34 us, 384 take 27)
  const long long room = sms * (R <= 2 ? 3 : R <= 8 ? 2 : 1) / tiles, deep = q.K / 256;
  long long parts = room < deep ? room : deep;
  parts = parts < 1 ? 1 : parts > 8 ? 8 : parts;
  if (tiles * parts > 0x7fffffffLL) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * parts));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(parts);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  // whole words: rows on 16-byte boundaries whose ends are, too
  const bool words = rows_on_16_bytes<T>(q.w, q.ldw) && (q.k_contiguous ? q.K : q.e.N) % kVec16<T> == 0;
  const cudaError_t e = words ? launch_kernel<T, R, kByWords>(cfg, q) : launch_kernel<T, R, kUnaligned<T>>(cfg, q);
  if (e != cudaSuccess) {
    fprintf(stderr, "[eshkol-b200] linear layer launch failed: %s\n", cudaGetErrorString(e));
    cudaGetLastError();
    return -1;
  }
  return 1;
}

template <typename T, int R, int kHow> cudaError_t set_attributes_how() {
  const cudaError_t e = cudaFuncSetAttribute(small_rows_wide_kernel<T, R, kHow>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(small_shared<T, R, false>()));
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(small_rows_deep_kernel<T, R, kHow>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(small_shared<T, R, true>()));
}
template <typename T, int R> cudaError_t set_attributes() {
  const cudaError_t e = set_attributes_how<T, R, kByWords>();
  return e != cudaSuccess ? e : set_attributes_how<T, R, kUnaligned<T>>();
}
template <typename T> cudaError_t set_attributes_of() {
  cudaError_t e = set_attributes<T, 1>();
  if (e == cudaSuccess) e = set_attributes<T, 2>();
  if (e == cudaSuccess) e = set_attributes<T, 4>();
  if (e == cudaSuccess) e = set_attributes<T, 8>();
  if constexpr (kSmallRows<T> > 8) {
    if (e == cudaSuccess) e = set_attributes<T, 16>();
  }
  return e;
}

}  // namespace

template <typename T> int launch_small_rows(const SmallRows& q, cudaStream_t st) {
  if (q.e.M <= 1) return launch_rows<T, 1>(q, st);
  if (q.e.M <= 2) return launch_rows<T, 2>(q, st);
  if (q.e.M <= 4) return launch_rows<T, 4>(q, st);
  if constexpr (kSmallRows<T> > 8) {
    if (q.e.M > 8) return launch_rows<T, 16>(q, st);
  }
  return launch_rows<T, 8>(q, st);
}
template int launch_small_rows<float>(const SmallRows&, cudaStream_t);
template int launch_small_rows<__half>(const SmallRows&, cudaStream_t);
template int launch_small_rows<__nv_bfloat16>(const SmallRows&, cudaStream_t);

cudaError_t linear_small_set_attributes() {
  cudaError_t e = set_attributes_of<float>();
  if (e == cudaSuccess) e = set_attributes_of<__half>();
  if (e == cudaSuccess) e = set_attributes_of<__nv_bfloat16>();
  return e;
}

}  // namespace b200
