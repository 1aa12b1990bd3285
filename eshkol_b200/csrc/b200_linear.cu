// The linear layer of 16-bit and f32 tensors on the tensor cores, forward with bias, activation and
// residual in the epilogue, and its gradients:
//
//   y = act(x W + b) + residual                 pre = x W + b
//   dz = grad_out act'(pre),  grad_x = dz W^T,  grad_w = x^T dz,  grad_b = sum over rows of dz
//
// One persistent kernel multiplies: warp 0 loads operand tiles by TMA into a ring of shared-memory
// stages, warp 1 issues tcgen05.mma into one of two TMEM accumulators, warps 2-5 drain the other one.
// Each operand is read as it lies, with the reduction axis along its rows ("K-major") or across them
// ("MN-major"): the matrix descriptors take both, so no product needs a transposed copy.  Sums are f32 in
// TMEM; a result is rounded to the storage type once.
//
// f32 tensors: every value is split into three bf16 numbers (8 + 8 + 8 bits of its significand, exact
// but for the last rounding, relative 2^-27), and six of the nine products of the parts, the smallest
// first, make the result; the three left out are below 2^-26 of the terms.
//
// Few output tiles and a long reduction: the reduction is split over blocks, their f32 sums go to scratch
// and a second kernel adds them in order and applies the epilogue.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

#include "b200_common.cuh"
#include "b200_elem.cuh"
#include "b200_internal.h"
#include "b200_tiers.h"

namespace b200 {
namespace {

constexpr int kLinThreads = 192;
constexpr int kLinBM = 128;
constexpr int kLinBK = 64;          // 16-bit elements per k-block: one 128-byte swizzle row
constexpr int kLinUmmaK = 16;
constexpr uint32_t kABytes = kLinBM * 128;
constexpr int kStagePitch = 36;     // f32 per row of a warp's 32 x 32 exchange tile: 16-byte accesses without conflicts
constexpr uint32_t kExchangeBytes = 4 * 32 * kStagePitch * 4;

template <int BN> struct LinShape {
  static constexpr uint32_t kBBytes = BN * 128;
  static constexpr int kStages = 196608 / (kABytes + kBBytes);
  static constexpr uint32_t kTmem = 2 * BN;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * (kABytes + kBBytes) + kExchangeBytes + 1024;
};

constexpr int kMaxSegs = 6;

// One product C[M x N] = sum over segments of A_plane B_plane, and what becomes of it.
struct LinProduct {
  int M, N;
  int kb;                 // k-blocks of a segment
  int n_seg;
  int seg_a[kMaxSegs], seg_b[kMaxSegs];
  int a_mn, b_mn;         // 1: the operand is MN-major
  int tiles_m, tiles_n, splits, kb_per_split;  // k-blocks over all segments, dealt out to the splits
  int first_work;         // of this product among the launch's work items
  float* partial;         // with splits > 1: [splits][M][ldp]
  long long ldp;
  // the epilogue (without splits)
  const void *bias, *residual;
  void *out, *pre;
  long long ldo, ld_res, ld_pre;
  int act;
  int words;              // 1: out, pre and residual rows lie on 16-byte boundaries
};

struct LinParams {
  LinProduct p[2];
  int n_products, total_work;
  uint32_t formats;       // operand type bits of the instruction descriptor
  int* status;
  unsigned long long wait_ns;
  int withhold;
};

struct LinMaps {
  CUtensorMap a[2], b[2];
};

struct LinWork {
  int which, tm, tn, split, kb0, kb1;
};
__device__ __forceinline__ LinWork decode(const LinParams& prm, int w) {
  LinWork it;
  it.which = (prm.n_products > 1 && w >= prm.p[1].first_work) ? 1 : 0;
  const LinProduct& q = prm.p[it.which];
  int t = w - q.first_work;
  const int tiles = q.tiles_m * q.tiles_n;
  it.split = t / tiles;
  t -= it.split * tiles;
  // groups of 16 tiles along M share the operand B's tiles while they are in L2
  const int per_group = 16 * q.tiles_n;
  const int g = t / per_group, r = t - g * per_group;
  const int gm = min(16, q.tiles_m - g * 16);
  it.tn = r / gm;
  it.tm = g * 16 + (r - it.tn * gm);
  it.kb0 = it.split * q.kb_per_split;
  it.kb1 = min(it.kb0 + q.kb_per_split, q.kb * q.n_seg);
  return it;
}

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: rows of 128 bytes, groups of eight rows
// 1024 bytes apart.  MN-major: one row holds 64 elements of the M or N axis at one k; eight such rows are
// 1024 bytes apart (stride offset), the next 64 elements of the axis one box of 64 rows further (leading
// offset).
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, int mn) {
  uint64_t d = umma_desc_k128(saddr);
  if (mn) d |= static_cast<uint64_t>((64u * 128u) >> 4) << 16;
  return d;
}

// ------------------------------------------------------------------ activations
template <bool kExact> __device__ __forceinline__ float logistic(float v) {
  if (kExact) return 1.f / (1.f + expf(-v));
  return __fdividef(1.f, 1.f + __expf(-v));  // a few 2^-22: below half a step of the 16-bit results
}
constexpr float kGeluA = 0.7978845608028654f, kGeluB = 0.044715f;

// 0 none, 1 ReLU, 2 the tanh form of GELU: z (1 + tanh u) / 2 = z logistic(2 u)
template <bool kExact> __device__ __forceinline__ float activate(float z, int act) {
  if (act == 1) return z > 0.f ? z : 0.f;
  if (act == 2) return z * logistic<kExact>(2.f * kGeluA * (z + kGeluB * z * z * z));
  return z;
}
template <bool kExact> __device__ __forceinline__ float activate_slope(float z, int act) {
  if (act == 1) return z > 0.f ? 1.f : 0.f;
  if (act == 2) {
    const float x = z > 20.f ? 20.f : (z < -20.f ? -20.f : z);  // the slope is 1 or 0 beyond; no overflow of x^3
    const float s = logistic<kExact>(2.f * kGeluA * (x + kGeluB * x * x * x));
    return s + x * s * (1.f - s) * 2.f * kGeluA * (1.f + 3.f * kGeluB * x * x);
  }
  return 1.f;
}

// kV elements of row `row` from column c: bias, activation, residual, the two results
template <typename T, int kV>
__device__ __forceinline__ void finish_row(const LinProduct& q, long long row, int c, const float (&acc)[kV],
                                           const float (&bias)[kV], const Pack<T, kV>& res) {
  constexpr bool kExact = sizeof(T) == 4;
  Pack<T, kV> z, y;
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const float v = acc[j] + bias[j];
    z.v[j] = Elem<T>::narrow(v);
    float a = activate<kExact>(v, q.act);
    if (q.residual) a += Elem<T>::widen(res.v[j]);
    y.v[j] = Elem<T>::narrow(a);
  }
  T* out = static_cast<T*>(q.out) + row * q.ldo + c;
  T* pre = q.pre ? static_cast<T*>(q.pre) + row * q.ld_pre + c : nullptr;
  if (c + kV <= q.N) {
    *reinterpret_cast<Pack<T, kV>*>(out) = y;
    if (pre) *reinterpret_cast<Pack<T, kV>*>(pre) = z;
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j)
      if (c + j < q.N) {
        out[j] = y.v[j];
        if (pre) pre[j] = z.v[j];
      }
  }
}
template <typename T, int kV>
__device__ __forceinline__ Pack<T, kV> load_residual(const LinProduct& q, long long row, int c) {
  Pack<T, kV> p;
  const T* r = static_cast<const T*>(q.residual) + row * q.ld_res + c;
  if (c + kV <= q.N) return *reinterpret_cast<const Pack<T, kV>*>(r);
#pragma unroll
  for (int j = 0; j < kV; ++j) p.v[j] = (c + j < q.N) ? r[j] : Elem<T>::narrow(0);
  return p;
}
template <typename T, int kV>
__device__ __forceinline__ void load_bias(const LinProduct& q, int c, float (&b)[kV]) {
#pragma unroll
  for (int j = 0; j < kV; ++j)
    b[j] = (q.bias && c + j < q.N) ? Elem<T>::widen(static_cast<const T*>(q.bias)[c + j]) : 0.f;
}

// a 32 x 32 block of the accumulator, one row per lane in v, from row0 and column c0 of the result
template <typename T, int kV>
__device__ __forceinline__ void finish_block(const LinProduct& q, float* tile, const uint32_t (&v)[32], long long row0, int c0) {
  const int lane = threadIdx.x & 31;
  constexpr int kLanesPerRow = 32 / kV, kRows = 32 / kLanesPerRow, kSteps = 32 / kRows;
  const int c = c0 + (lane % kLanesPerRow) * kV, r = lane / kLanesPerRow;
  constexpr int kGroup = kSteps < 8 ? kSteps : 8;  // residual words on their way at a time
  float bias[kV];
  load_bias<T, kV>(q, c, bias);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(tile + lane * kStagePitch + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
#pragma unroll
  for (int s0 = 0; s0 < kSteps; s0 += kGroup) {
    Pack<T, kV> res[kGroup];
    if (q.residual) {
#pragma unroll
      for (int s = 0; s < kGroup; ++s) {
        const long long row = row0 + r + (s0 + s) * kRows;
        if (row < q.M && c < q.N) res[s] = load_residual<T, kV>(q, row, c);
      }
    }
#pragma unroll
    for (int s = 0; s < kGroup; ++s) {
      const int in_tile = r + (s0 + s) * kRows;
      const long long row = row0 + in_tile;
      float acc[kV];
      if (kV >= 4) {
#pragma unroll
        for (int j = 0; j < kV; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(tile + in_tile * kStagePitch + (lane % kLanesPerRow) * kV + j);
          acc[j] = f.x; acc[j + 1] = f.y; acc[j + 2] = f.z; acc[j + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j) acc[j] = tile[in_tile * kStagePitch + (lane % kLanesPerRow) * kV + j];
      }
      if (row < q.M && c < q.N) finish_row<T, kV>(q, row, c, acc, bias, res[s]);
    }
  }
}

// a block of a split reduction's partial sums
__device__ __forceinline__ void store_partial(const LinProduct& q, float* tile, const uint32_t (&v)[32], int split,
                                              long long row0, int c0) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(tile + lane * kStagePitch + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  const int c = c0 + (lane & 7) * 4;
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int in_tile = (lane >> 3) + 4 * s;
    const long long row = row0 + in_tile;
    if (row < q.M && c < q.ldp)  // ldp is N rounded up to 4: whole words
      *reinterpret_cast<float4*>(q.partial + (static_cast<long long>(split) * q.M + row) * q.ldp + c) =
          *reinterpret_cast<const float4*>(tile + in_tile * kStagePitch + (lane & 7) * 4);
  }
}

template <int BN, typename T>
__global__ void __launch_bounds__(kLinThreads, 1)
linear_kernel(const __grid_constant__ LinMaps maps, const __grid_constant__ LinParams prm) {
  using Shape = LinShape<BN>;
  constexpr int kStages = Shape::kStages;
  constexpr uint32_t kBBytes = Shape::kBBytes;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t dyn_addr = smem_u32(smem_dyn);
  const uint32_t tile_base = (dyn_addr + 1023u) & ~1023u;
  uint8_t* tiles = smem_dyn + (tile_base - dyn_addr);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 128); }
    abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, Shape::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, last_parity = 0;
      bool ok = true;
      int withhold = prm.withhold && blockIdx.x == 0;
      for (int w = blockIdx.x; w < prm.total_work && ok; w += gridDim.x) {
        const LinWork it = decode(prm, w);
        const LinProduct& q = prm.p[it.which];
        const CUtensorMap* ma = &maps.a[it.which];
        const CUtensorMap* mb = &maps.b[it.which];
        int seg = it.kb0 / q.kb, kb = it.kb0 - seg * q.kb;
        for (int i = it.kb0; i < it.kb1; ++i) {
          if (!mbar_wait<false>(&empty_bar[stage], phase ^ 1u, &abort_flag, prm.wait_ns)) {
            atomicCAS(prm.status, kStatusOk, kStatusProducerTimeout);
            abort_flag = 1;
            ok = false;
            break;
          }
          if (withhold) {  // tests only: this stage never arrives and the waits behind it run out
            withhold = 0;
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
            if (++kb == q.kb) { kb = 0; ++seg; }
            continue;
          }
          mbar_arrive_expect_tx(&full_bar[stage], kABytes + kBBytes);
          uint8_t* sa = tiles + stage * kABytes;
          uint8_t* sb = tiles + kStages * kABytes + stage * kBBytes;
          const int k0 = kb * kLinBK, m0 = it.tm * kLinBM, n0 = it.tn * BN, pa = q.seg_a[seg], pb = q.seg_b[seg];
          if (q.a_mn) {
#pragma unroll
            for (int j = 0; j < kLinBM / 64; ++j) tma_load_3d(sa + j * 8192, ma, &full_bar[stage], m0 + 64 * j, k0, pa);
          } else {
            tma_load_3d(sa, ma, &full_bar[stage], k0, m0, pa);
          }
          if (q.b_mn) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) tma_load_3d(sb + j * 8192, mb, &full_bar[stage], n0 + 64 * j, k0, pb);
          } else {
            tma_load_3d(sb, mb, &full_bar[stage], k0, n0, pb);
          }
          issued |= 1u << stage;
          last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
          if (++kb == q.kb) { kb = 0; ++seg; }
        }
      }
      if (!ok || abort_flag) {  // leaving early: the copies in flight land first
        int none = 0;
        for (int s = 0; s < kStages; ++s)
          if (issued & (1u << s)) mbar_wait<true>(&full_bar[s], (last_parity >> s) & 1u, &none, prm.wait_ns);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, unit = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < prm.total_work && ok; w += gridDim.x) {
        const LinWork it = decode(prm, w);
        const LinProduct& q = prm.p[it.which];
        const uint32_t idesc = umma_idesc_f16(kLinBM, BN) | prm.formats | (static_cast<uint32_t>(q.a_mn) << 15) |
                               (static_cast<uint32_t>(q.b_mn) << 16);
        // an instruction's 16 steps of k: 32 bytes along a K-major row, 16 rows of an MN-major box
        const uint32_t step_a = q.a_mn ? (16u * 128u) >> 4 : 2u, step_b = q.b_mn ? (16u * 128u) >> 4 : 2u;
        const uint32_t buf = unit & 1u, aphase = (unit >> 1) & 1u;
        if (!mbar_wait<false>(&acc_empty[buf], aphase ^ 1u, &abort_flag, prm.wait_ns)) {
          atomicCAS(prm.status, kStatusOk, kStatusMmaTimeout);
          abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int i = it.kb0; i < it.kb1; ++i) {
          if (!mbar_wait<false>(&full_bar[stage], phase, &abort_flag, prm.wait_ns)) {
            atomicCAS(prm.status, kStatusOk, kStatusMmaTimeout);
            abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = operand_desc(tile_base + stage * kABytes, q.a_mn);
          const uint64_t db = operand_desc(tile_base + kStages * kABytes + stage * kBBytes, q.b_mn);
#pragma unroll
          for (int k = 0; k < kLinBK / kLinUmmaK; ++k)
            umma_f16(d_tmem, da + step_a * k, db + step_b * k, idesc, (i > it.kb0 || k > 0) ? 1u : 0u);
          umma_commit(&empty_bar[stage]);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (ok) umma_commit(&acc_full[buf]);
        ++unit;
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    float* tile = reinterpret_cast<float*>(tiles + static_cast<size_t>(kStages) * (kABytes + kBBytes)) +
                  quarter * 32 * kStagePitch;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t unit = 0;
    for (int w = blockIdx.x; w < prm.total_work; w += gridDim.x) {
      const LinWork it = decode(prm, w);
      const LinProduct& q = prm.p[it.which];
      const uint32_t buf = unit & 1u, aphase = (unit >> 1) & 1u;
      if (!mbar_wait<true>(&acc_full[buf], aphase, &abort_flag, prm.wait_ns)) {
        atomicCAS(prm.status, kStatusOk, kStatusEpilogueTimeout);
        abort_flag = 1;
        break;
      }
      tc_fence_after();
      const long long row0 = static_cast<long long>(it.tm) * kLinBM + quarter * 32;
      const int n0 = it.tn * BN;
#pragma unroll 1
      for (int cc = 0; cc < BN / 32; ++cc) {
        const int c0 = n0 + cc * 32;
        if (row0 >= q.M || c0 >= q.N) break;  // the same for the whole warp
        uint32_t v[32];
        tmem_ld32(tmem_base + lane_addr + buf * BN + cc * 32, v);
        tmem_ld_wait();
        if (q.splits > 1) store_partial(q, tile, v, it.split, row0, c0);
        else if (q.words) finish_block<T, kVec16<T>>(q, tile, v, row0, c0);
        else finish_block<T, 1>(q, tile, v, row0, c0);
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[buf]);
      ++unit;
    }
  }

  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Shape::kTmem);
  }
}

// the partial sums of a split reduction, added in order, and the epilogue
template <typename T>
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ LinProduct q) {
  const long long words = q.ldp / 4, total = q.M * words;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / words;
    const int c = static_cast<int>(i - row * words) * 4;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < q.splits; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(q.partial + (static_cast<long long>(s) * q.M + row) * q.ldp + c);
      acc[0] += f.x; acc[1] += f.y; acc[2] += f.z; acc[3] += f.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c + j >= q.N) break;
      float b[1], a[1] = {acc[j]};
      load_bias<T, 1>(q, c + j, b);
      Pack<T, 1> res;
      res.v[0] = Elem<T>::narrow(0);
      if (q.residual) res = load_residual<T, 1>(q, row, c + j);
      finish_row<T, 1>(q, row, c + j, a, b, res);
    }
  }
}

// ------------------------------------------------------------------ operand preparation
// value -> the operand's 16-bit planes
__device__ __forceinline__ void split3(float v, __nv_bfloat16& a, __nv_bfloat16& b, __nv_bfloat16& c) {
  a = __float2bfloat16_rn(v);
  const float r = v - __bfloat162float(a);
  b = __float2bfloat16_rn(r);
  c = __float2bfloat16_rn(r - __bfloat162float(b));
}
template <typename T> struct Plane { using type = T; static constexpr int kCount = 1; };
template <> struct Plane<float> { using type = __nv_bfloat16; static constexpr int kCount = 3; };

// eight consecutive results into the operand's planes
template <typename T>
__device__ __forceinline__ void store_planes(typename Plane<T>::type* dst, long long plane_stride, const float (&f)[8]) {
  using P = typename Plane<T>::type;
  Pack<P, 8> p[Plane<T>::kCount];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (Plane<T>::kCount == 3) split3(f[j], p[0].v[j], p[1].v[j], p[2].v[j]);
    else p[0].v[j] = Elem<T>::narrow(f[j]);
  }
#pragma unroll
  for (int i = 0; i < Plane<T>::kCount; ++i) *reinterpret_cast<Pack<P, 8>*>(dst + i * plane_stride) = p[i];
}

template <typename T, bool kWords>
__device__ __forceinline__ void load8(const T* row, int c, int n, float (&f)[8]) {
  if (kWords && c + 8 <= n) {
    constexpr int kV = kVec16<T>;
#pragma unroll
    for (int i = 0; i < 8; i += kV) {
      const Pack<T, kV> p = *reinterpret_cast<const Pack<T, kV>*>(row + c + i);
#pragma unroll
      for (int j = 0; j < kV; ++j) f[i + j] = Elem<T>::widen(p.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (c + j < n) ? Elem<T>::widen(row[c + j]) : 0.f;
  }
}

struct PackJob {
  const void* src;
  void* dst;
  long long rows, lds, ldd, plane_stride;
  int cols;
  int words;  // the source's rows lie on 16-byte boundaries
  long long first;  // of this job among the launch's groups of eight elements
};
struct PackJobs {
  PackJob j[2];
  int n;
  long long total;
};
template <typename T>
__global__ void __launch_bounds__(256) linear_pack_kernel(const __grid_constant__ PackJobs jobs) {
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < jobs.total;
       i += static_cast<long long>(gridDim.x) * 256) {
    const PackJob& q = jobs.j[(jobs.n > 1 && i >= jobs.j[1].first) ? 1 : 0];
    const long long per_row = q.ldd / 8, at = i - q.first, row = at / per_row;
    const int c = static_cast<int>(at - row * per_row) * 8;
    float f[8];
    const T* src = static_cast<const T*>(q.src) + row * q.lds;
    if (q.words) load8<T, true>(src, c, q.cols, f);
    else load8<T, false>(src, c, q.cols, f);
    store_planes<T>(static_cast<typename Plane<T>::type*>(q.dst) + row * q.ldd + c, q.plane_stride, f);
  }
}

struct SlopeArgs {
  const void *grad_out, *pre;
  void* dz;                  // NULL: only the column sums are wanted
  float* partial;            // [gridDim.y][cols], or NULL
  long long rows, ldg, ld_pre, ldd, plane_stride;
  int cols, act, words;
};
// dz = grad_out act'(pre), rounded into the products' operand, and its column sums from the f32 values:
// 256 columns per block, eight per lane; eight warps share the block's rows
template <typename T>
__global__ void __launch_bounds__(256) linear_slope_kernel(const __grid_constant__ SlopeArgs a) {
  constexpr bool kExact = sizeof(T) == 4;
  __shared__ float sm[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 256 + lane * 8;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < a.cols) {
    for (long long r = static_cast<long long>(blockIdx.y) * 8 + warp; r < a.rows; r += static_cast<long long>(gridDim.y) * 8) {
      float g[8], z[8];
      const T* gr = static_cast<const T*>(a.grad_out) + r * a.ldg;
      if (a.words) load8<T, true>(gr, c, a.cols, g);
      else load8<T, false>(gr, c, a.cols, g);
      if (a.act) {
        const T* zr = static_cast<const T*>(a.pre) + r * a.ld_pre;
        if (a.words) load8<T, true>(zr, c, a.cols, z);
        else load8<T, false>(zr, c, a.cols, z);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] *= activate_slope<kExact>(z[j], a.act);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += g[j];
      if (a.dz) store_planes<T>(static_cast<typename Plane<T>::type*>(a.dz) + r * a.ldd + c, a.plane_stride, g);
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sm[warp][lane * 8 + j] = sum[j];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += sm[w][threadIdx.x];
  if (col < a.cols) a.partial[static_cast<long long>(blockIdx.y) * a.cols + col] = s;
}
__global__ void __launch_bounds__(256) linear_bias_join_kernel(const float* __restrict__ partial, int parts, int cols,
                                                               float* __restrict__ out) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
#pragma unroll 8
  for (int p = 0; p < parts; ++p) s += partial[static_cast<long long>(p) * cols + c];
  out[c] = s;
}

// ------------------------------------------------------------------ host side
long long round8(long long v) { return (v + 7) / 8 * 8; }

// A stored matrix as an operand of the products: `inner` elements in a row, `outer` rows
struct Stored {
  const void* p;
  long long inner, outer, ld, plane_stride;
  int planes;
};

int operand_map(CUtensorMap* map, const Stored& s, bool mn, int tile) {
  return make_matrix_map16(map, s.p, s.inner, s.outer, s.ld, s.planes, s.plane_stride, mn ? 64 : tile);
}

bool tma_ready(const void* p, long long ld) { return rows_on_16_bytes<uint16_t>(p, ld); }

struct ProductSpec {
  Stored a, b;
  bool a_mn, b_mn;
  long long M, N, K;
};

template <int BN, typename T> int launch_products(const LinMaps& maps, const LinParams& prm, cudaStream_t st) {
  const int sms = lib_num_sms();
  linear_kernel<BN, T><<<prm.total_work < sms ? prm.total_work : sms, kLinThreads, LinShape<BN>::kSmem, st>>>(maps, prm);
  return 1;
}

struct Plan {
  int bn, splits[2], kb_per_split[2];
  size_t partial_bytes[2];
};

// Tile width and splits: the estimate of a launch in units of one k-block of a 128 x 256 tile.  An item
// costs its k-blocks (a narrower tile's cost by the bytes it loads) and its epilogue; items run in rounds
// over the SMs; a split product pays for its partial sums and the second launch.
Plan plan_products(const ProductSpec* s, int n, int n_seg) {
  const double sms = lib_num_sms();
  Plan best = {};
  double best_cost = 1e300;
  const int widths[3] = {256, 128, 64};
  for (int bn : widths) {
    const double per_kb = bn == 256 ? 1.0 : bn == 128 ? 0.62 : 0.46, per_tile = 4.0 * bn / 256 + 2.0;
    Plan q = {};
    q.bn = bn;
    double items = 0, longest = 0, work = 0, extra = 0;
    for (int i = 0; i < n; ++i) {
      const double tiles = static_cast<double>((s[i].M + 127) / 128) * static_cast<double>((s[i].N + bn - 1) / bn);
      const int kb = static_cast<int>((s[i].K + kLinBK - 1) / kLinBK) * n_seg;
      int split = 1;
      // enough items for the SMs, at least eight k-blocks in each
      while (tiles * split < sms && kb / (split * 2) >= 8 && split < 64) split *= 2;
      q.kb_per_split[i] = (kb + split - 1) / split;
      q.splits[i] = (kb + q.kb_per_split[i] - 1) / q.kb_per_split[i];
      const double cost = q.kb_per_split[i] * per_kb + per_tile;
      items += tiles * q.splits[i];
      work += tiles * q.splits[i] * cost;
      if (cost > longest) longest = cost;
      q.partial_bytes[i] = 0;
      if (q.splits[i] > 1) {
        q.partial_bytes[i] = (static_cast<size_t>(q.splits[i]) * s[i].M * ((s[i].N + 3) / 4 * 4) * 4 + 1023) & ~size_t(1023);
        extra += 8.0 + q.partial_bytes[i] * 2.0 / 1.2e6;  // a k-block takes about 0.3 us
      }
    }
    const double rounds = ceil(items / sms);
    const double cost = fmax(work / sms, fmax(longest, rounds * work / items)) + extra;
    if (cost < best_cost) { best_cost = cost; best = q; }
  }
  return best;
}

// Multiplies one or two independent products in one launch, and joins those whose reduction was split.
// epi[i] carries the epilogue of product i; scratch_at: room for the partial sums (plan.partial_bytes).
template <typename T>
int run_products(const ProductSpec* s, LinProduct* epi, int n, const Plan& plan, uint8_t* scratch_at, cudaStream_t st) {
  LinMaps maps;
  LinParams prm;
  memset(&prm, 0, sizeof(prm));
  static const int seg_a[6] = {2, 0, 1, 1, 0, 0}, seg_b[6] = {0, 2, 1, 0, 1, 0};
  const int n_seg = Plane<T>::kCount == 3 ? 6 : 1;
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    LinProduct& q = epi[i];
    q.M = static_cast<int>(s[i].M);
    q.N = static_cast<int>(s[i].N);
    q.kb = static_cast<int>((s[i].K + kLinBK - 1) / kLinBK);
    q.n_seg = n_seg;
    for (int k = 0; k < n_seg; ++k) {
      q.seg_a[k] = n_seg == 6 ? seg_a[k] : 0;
      q.seg_b[k] = n_seg == 6 ? seg_b[k] : 0;
    }
    q.a_mn = s[i].a_mn; q.b_mn = s[i].b_mn;
    q.tiles_m = (q.M + kLinBM - 1) / kLinBM;
    q.tiles_n = (q.N + plan.bn - 1) / plan.bn;
    q.splits = plan.splits[i];
    q.kb_per_split = plan.kb_per_split[i];
    q.first_work = static_cast<int>(total);
    total += static_cast<long long>(q.tiles_m) * q.tiles_n * q.splits;
    if (total > 0x7fffffffLL) return -1;
    q.ldp = (q.N + 3) / 4 * 4;
    q.partial = nullptr;
    if (q.splits > 1) {
      q.partial = reinterpret_cast<float*>(scratch_at);
      scratch_at += plan.partial_bytes[i];
    }
    q.words = rows_on_16_bytes<T>(q.out, q.ldo) && (!q.pre || rows_on_16_bytes<T>(q.pre, q.ld_pre)) &&
              (!q.residual || rows_on_16_bytes<T>(q.residual, q.ld_res));
    if (operand_map(&maps.a[i], s[i].a, s[i].a_mn, kLinBM) || operand_map(&maps.b[i], s[i].b, s[i].b_mn, plan.bn)) return -1;
    prm.p[i] = q;
  }
  if (n == 1) { maps.a[1] = maps.a[0]; maps.b[1] = maps.b[0]; }
  prm.n_products = n;
  prm.total_work = static_cast<int>(total);
  prm.formats = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value ? 0u : (1u << 7) | (1u << 10);
  prm.status = lib_status_word();
  prm.wait_ns = lib_wait_limit_ns();
  prm.withhold = lib_take_withhold();
  int launches = plan.bn == 256 ? launch_products<256, T>(maps, prm, st)
                 : plan.bn == 128 ? launch_products<128, T>(maps, prm, st) : launch_products<64, T>(maps, prm, st);
  for (int i = 0; i < n; ++i) {
    if (epi[i].splits == 1) continue;
    const long long words = epi[i].ldp / 4 * epi[i].M, cap = static_cast<long long>(lib_num_sms()) * 8;
    const long long blocks = (words + 255) / 256;
    linear_join_kernel<T><<<static_cast<unsigned>(blocks < cap ? blocks : cap), 256, 0, st>>>(epi[i]);
    ++launches;
  }
  return launches;
}

int finish(int launches) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    fprintf(stderr, "[eshkol-b200] linear layer launch failed: %s\n", cudaGetErrorString(e));
    return -1;
  }
  count_launches(launches);
  return 0;
}

struct Carver {
  size_t off = 0;
  size_t take(size_t bytes) {
    const size_t o = off;
    off += (bytes + 1023) & ~static_cast<size_t>(1023);
    return o;
  }
};

// A matrix that the products can read: the tensor itself, or a packed (f32: split) copy in scratch
template <typename T> struct Operand {
  Stored s;
  bool copy;
  size_t at;
  Operand(const void* p, long long rows, long long cols, long long ld, bool force, Carver& cv) {
    copy = force || Plane<T>::kCount > 1 || !tma_ready(p, ld);
    s.p = p; s.inner = cols; s.outer = rows; s.ld = ld; s.planes = 1; s.plane_stride = rows * ld;
    at = 0;
    if (copy) {
      s.ld = round8(cols);
      s.planes = Plane<T>::kCount;
      s.plane_stride = rows * s.ld;
      at = cv.take(static_cast<size_t>(s.plane_stride) * s.planes * 2);
    }
  }
  void bind(uint8_t* base) { if (copy) s.p = base + at; }
};

template <typename T> void add_pack(PackJobs& jobs, const void* src, long long lds, const Operand<T>& o) {
  if (!o.copy) return;
  PackJob& j = jobs.j[jobs.n];
  j.src = src; j.dst = const_cast<void*>(o.s.p);
  j.rows = o.s.outer; j.cols = static_cast<int>(o.s.inner); j.lds = lds; j.ldd = o.s.ld; j.plane_stride = o.s.plane_stride;
  j.words = rows_on_16_bytes<T>(src, lds);
  j.first = jobs.total;
  jobs.total += j.rows * (j.ldd / 8);
  ++jobs.n;
}
template <typename T> int launch_pack(const PackJobs& jobs, cudaStream_t st) {
  if (jobs.n == 0) return 0;
  const long long blocks = (jobs.total + 255) / 256, cap = static_cast<long long>(lib_num_sms()) * 16;
  linear_pack_kernel<T><<<static_cast<unsigned>(blocks < cap ? blocks : cap), 256, 0, st>>>(jobs);
  return 1;
}

struct LinearArgs {
  const void *x, *w;
  long long rows, d_in, d_out, ldx, ldw, ldy, ld_res, ld_pre;
  EshkolB200LinearOpts o;
};

template <typename T> int linear_forward(const LinearArgs& a, void* y, OpScratch& scratch, cudaStream_t st) {
  const bool tw = a.o.trans_w != 0;
  Carver cv;
  Operand<T> x(a.x, a.rows, a.d_in, a.ldx, false, cv);
  Operand<T> w(a.w, tw ? a.d_out : a.d_in, tw ? a.d_in : a.d_out, a.ldw, false, cv);
  ProductSpec s = {x.s, w.s, false, !tw, a.rows, a.d_out, a.d_in};
  const Plan plan = plan_products(&s, 1, Plane<T>::kCount == 3 ? 6 : 1);
  const size_t parts = cv.take(plan.partial_bytes[0]);
  uint8_t* base = scratch.reserve(cv.off, st);
  if (!base) return -1;
  x.bind(base);
  w.bind(base);
  s.a = x.s; s.b = w.s;
  PackJobs jobs = {};
  add_pack<T>(jobs, a.x, a.ldx, x);
  add_pack<T>(jobs, a.w, a.ldw, w);
  const int packs = launch_pack<T>(jobs, st);
  LinProduct epi;
  memset(&epi, 0, sizeof(epi));
  epi.bias = a.o.bias; epi.residual = a.o.residual; epi.out = y; epi.pre = a.o.pre;
  epi.ldo = a.ldy; epi.ld_res = a.ld_res; epi.ld_pre = a.ld_pre; epi.act = a.o.activation;
  const int n = run_products<T>(&s, &epi, 1, plan, base + parts, st);
  return n < 0 ? -1 : packs + n;
}

template <typename T>
int linear_gradients(const LinearArgs& a, const void* grad_out, void* grad_x, void* grad_w, void* grad_bias,
                     OpScratch& scratch, cudaStream_t st) {
  const bool tw = a.o.trans_w != 0, products = grad_x || grad_w;
  Carver cv;
  // dz: grad_out itself when there is no activation and the products can read it
  Operand<T> dz(grad_out, a.rows, a.d_out, a.ldy, a.o.activation != 0, cv);
  Operand<T> x(a.x, a.rows, a.d_in, a.ldx, false, cv);
  Operand<T> w(a.w, tw ? a.d_out : a.d_in, tw ? a.d_in : a.d_out, a.ldw, false, cv);
  ProductSpec s[2];
  LinProduct epi[2];
  memset(epi, 0, sizeof(epi));
  int n = 0;
  const auto describe = [&]() {
    n = 0;
    if (grad_x) {
      s[n] = {dz.s, w.s, false, tw, a.rows, a.d_in, a.d_out};
      epi[n].out = grad_x; epi[n].ldo = a.ldx;
      ++n;
    }
    if (grad_w) {
      if (tw) s[n] = {dz.s, x.s, true, true, a.d_out, a.d_in, a.rows};
      else s[n] = {x.s, dz.s, true, true, a.d_in, a.d_out, a.rows};
      epi[n].out = grad_w; epi[n].ldo = a.ldw;
      ++n;
    }
  };
  describe();
  Plan plan = {};
  if (n) plan = plan_products(s, n, Plane<T>::kCount == 3 ? 6 : 1);
  const size_t parts = cv.take(plan.partial_bytes[0] + plan.partial_bytes[1]);
  // blocks of the column sums: the SMs several times over, at least 16 rows a block
  const long long col_blocks = (a.d_out + 255) / 256;
  long long row_blocks = static_cast<long long>(lib_num_sms()) * 6 / col_blocks;
  if (row_blocks > (a.rows + 15) / 16) row_blocks = (a.rows + 15) / 16;
  if (row_blocks < 1) row_blocks = 1;
  const size_t sums = cv.take(grad_bias ? static_cast<size_t>(row_blocks) * a.d_out * 4 : 0);
  uint8_t* base = scratch.reserve(cv.off, st);
  if (!base) return -1;
  dz.bind(base); x.bind(base); w.bind(base);
  describe();
  int launches = 0;
  if ((products && dz.copy) || grad_bias) {
    SlopeArgs q;
    q.grad_out = grad_out; q.pre = a.o.pre; q.dz = (products && dz.copy) ? const_cast<void*>(dz.s.p) : nullptr;
    q.partial = grad_bias ? reinterpret_cast<float*>(base + sums) : nullptr;
    q.rows = a.rows; q.ldg = a.ldy; q.ld_pre = a.ld_pre; q.ldd = dz.s.ld; q.plane_stride = dz.s.plane_stride;
    q.cols = static_cast<int>(a.d_out); q.act = a.o.activation;
    q.words = rows_on_16_bytes<T>(grad_out, a.ldy) && (!q.act || rows_on_16_bytes<T>(q.pre, a.ld_pre));
    linear_slope_kernel<T><<<dim3(static_cast<unsigned>(col_blocks), static_cast<unsigned>(row_blocks)), 256, 0, st>>>(q);
    ++launches;
    if (grad_bias) {
      linear_bias_join_kernel<<<static_cast<unsigned>(col_blocks), 256, 0, st>>>(
          q.partial, static_cast<int>(row_blocks), q.cols, static_cast<float*>(grad_bias));
      ++launches;
    }
  }
  if (!products) return launches;
  PackJobs jobs = {};
  if (grad_w) add_pack<T>(jobs, a.x, a.ldx, x);
  if (grad_x) add_pack<T>(jobs, a.w, a.ldw, w);
  launches += launch_pack<T>(jobs, st);
  const int m = run_products<T>(s, epi, n, plan, base + parts, st);
  return m < 0 ? -1 : launches + m;
}

bool pitch_ok(int64_t ld, uint64_t n) { return ld == 0 || (ld >= static_cast<int64_t>(n) && ld <= (1ll << 36)); }

// what both directions check; fills the pitches
int check(const EshkolB200LinearOpts* opts, uint64_t rows, uint64_t d_in, uint64_t d_out, LinearArgs& a) {
  if (lib_device() < 0 || !opts) return -1;
  a.o = *opts;
  if (a.o.dtype == ESHKOL_B200_F64) {
    fprintf(stderr, "[eshkol-b200] linear layer: f64 tensors go through eshkol_b200_gemm_f64_device or _feed_forward_f64_device\n");
    return -1;
  }
  if (a.o.dtype < ESHKOL_B200_F32 || a.o.dtype > ESHKOL_B200_BF16 || a.o.activation < 0 || a.o.activation > 2) return -1;
  const uint64_t most = 1ull << 30;
  if (rows > most || d_in == 0 || d_in > most || d_out == 0 || d_out > most) return -1;
  const uint64_t w_row = a.o.trans_w ? d_in : d_out;
  if (!pitch_ok(a.o.ldx, d_in) || !pitch_ok(a.o.ldw, w_row) || !pitch_ok(a.o.ldy, d_out) ||
      !pitch_ok(a.o.ld_residual, d_out) || !pitch_ok(a.o.ld_pre, d_out))
    return -1;
  a.rows = static_cast<long long>(rows); a.d_in = static_cast<long long>(d_in); a.d_out = static_cast<long long>(d_out);
  a.ldx = a.o.ldx ? a.o.ldx : a.d_in;
  a.ldw = a.o.ldw ? a.o.ldw : static_cast<long long>(w_row);
  a.ldy = a.o.ldy ? a.o.ldy : a.d_out;
  a.ld_res = a.o.ld_residual ? a.o.ld_residual : a.d_out;
  a.ld_pre = a.o.ld_pre ? a.o.ld_pre : a.d_out;
  return 0;
}

template <int BN, typename T> cudaError_t set_attribute() {
  return cudaFuncSetAttribute(linear_kernel<BN, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(LinShape<BN>::kSmem));
}
template <typename T> cudaError_t set_attributes_of() {
  cudaError_t e = set_attribute<256, T>();
  if (e == cudaSuccess) e = set_attribute<128, T>();
  if (e == cudaSuccess) e = set_attribute<64, T>();
  return e;
}

}  // namespace

cudaError_t linear_set_attributes() {
  cudaError_t e = set_attributes_of<float>();
  if (e == cudaSuccess) e = set_attributes_of<__half>();
  if (e == cudaSuccess) e = set_attributes_of<__nv_bfloat16>();
  return e;
}

}  // namespace b200

using namespace b200;

extern "C" {

int eshkol_b200_linear_forward_device(const void* x, const void* w, void* y, uint64_t rows, uint64_t d_in, uint64_t d_out,
                                      const EshkolB200LinearOpts* opts) {
  LinearArgs a;
  if (check(opts, rows, d_in, d_out, a) != 0) return -1;
  if (rows == 0) return 0;
  if (!x || !w || !y || y == x || y == a.o.pre || (y == a.o.residual && a.ldy != a.ld_res)) return -1;
  DeviceScope scope(lib_device());
  if (!scope.ok()) return -1;
  a.x = x; a.w = w;
  OpScratch scratch;
  cudaStream_t st = lib_stream();
  const int n = a.o.dtype == ESHKOL_B200_F32   ? linear_forward<float>(a, y, scratch, st)
                : a.o.dtype == ESHKOL_B200_F16 ? linear_forward<__half>(a, y, scratch, st)
                                               : linear_forward<__nv_bfloat16>(a, y, scratch, st);
  if (n < 0 || finish(n) != 0) return -1;
  return scratch.release();
}

int eshkol_b200_linear_gradients_device(const void* grad_out, const void* x, const void* w, void* grad_x, void* grad_w,
                                        void* grad_bias, uint64_t rows, uint64_t d_in, uint64_t d_out,
                                        const EshkolB200LinearOpts* opts) {
  LinearArgs a;
  if (check(opts, rows, d_in, d_out, a) != 0) return -1;
  if (!grad_x && !grad_w && !grad_bias) return -1;
  DeviceScope scope(lib_device());
  if (!scope.ok()) return -1;
  cudaStream_t st = lib_stream();
  if (rows == 0) {  // sums over no rows
    const size_t size = a.o.dtype == ESHKOL_B200_F32 ? 4 : 2;
    const size_t w_rows = a.o.trans_w ? d_out : d_in, w_cols = a.o.trans_w ? d_in : d_out;
    if (grad_w && cudaMemset2DAsync(grad_w, a.ldw * size, 0, w_cols * size, w_rows, st) != cudaSuccess) return finish(0);
    if (grad_bias && cudaMemsetAsync(grad_bias, 0, d_out * 4, st) != cudaSuccess) return finish(0);
    return 0;
  }
  if (!grad_out || (grad_x && !w) || (grad_w && !x) || (a.o.activation && !a.o.pre)) return -1;
  if (grad_x == grad_out || (grad_x && (grad_x == w || grad_x == x)) || (grad_w && (grad_w == w || grad_w == x))) return -1;
  a.x = x; a.w = w;
  OpScratch scratch;
  const int n = a.o.dtype == ESHKOL_B200_F32   ? linear_gradients<float>(a, grad_out, grad_x, grad_w, grad_bias, scratch, st)
                : a.o.dtype == ESHKOL_B200_F16 ? linear_gradients<__half>(a, grad_out, grad_x, grad_w, grad_bias, scratch, st)
                                               : linear_gradients<__nv_bfloat16>(a, grad_out, grad_x, grad_w, grad_bias, scratch, st);
  if (n < 0 || finish(n) != 0) return -1;
  return scratch.release();
}

}  // extern "C"
