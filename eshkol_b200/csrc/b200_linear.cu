// The linear layer of 16-bit and f32 tensors on the tensor cores, forward with bias, activation and
// residual in the epilogue, and its gradients:
//
//   y = act(x W + b) + residual                 pre = x W + b
//   dz = grad_out act'(pre),  grad_x = dz W^T,  grad_w = x^T dz,  grad_b = sum over rows of dz
//
// One persistent kernel multiplies: warp 0 loads operand tiles by TMA into a ring of shared-memory
// stages, warp 1 issues tcgen05.mma into one of two TMEM accumulators, warps 2-9 drain the other one.
// Each operand is read as it lies, with the reduction axis along its rows ("K-major") or across them
// ("MN-major"): the matrix descriptors take both, so no product needs a transposed copy.  Sums are f32 in
// TMEM; a result is rounded to the storage type once.
//
// f32 tensors: every value is split into three bf16 numbers (8 + 8 + 8 bits of its significand, exact for
// magnitudes from 2^-103, whose parts are all normal numbers), and six of the nine products of the parts make
// the result; the three left out are at most 2^-24 of the terms.
//
// Bound by the tensor pipe (active 94 % of the time on pairs of SMs): 8192 x 16384 x 4096 bf16 takes 725 us in
// a burst, 1517 TFLOP/s, and 850 under the power cap; all gradients at 4096 x 4096 x 16384 755 us in a burst.
//
// A few rows: b200_linear_small.cu.  Few output tiles and a long reduction: the reduction is split over
// blocks, their f32 sums go to scratch and a second kernel adds them in order and applies the epilogue.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

#include "b200_common.cuh"
#include "b200_elem.cuh"
#include "b200_internal.h"
#include "b200_linear.cuh"
#include "b200_tiers.h"

namespace b200 {
namespace {

constexpr int kLinThreads = 320;    // warps 0 and 1 load and issue, eight warps drain
constexpr int kLinBM = 128;
constexpr int kLinUmmaK = 16;
constexpr int kStagePitch = 36;     // f32 per row of a warp's 16 x 32 exchange tile: 16-byte accesses without conflicts
constexpr int kExchange = 16 * kStagePitch + 128;  // f32 of an epilogue warp: the exchange tile, its columns' bias
constexpr uint32_t kExchangeBytes = 8 * kExchange * 4;

// 16-bit operands as they are, f32 as three bf16 planes
template <typename T> struct Plane { using type = T; static constexpr int kCount = 1; };
template <> struct Plane<float> { using type = __nv_bfloat16; static constexpr int kCount = 3; };

// The kernel's shape: tiles of 128 x BN, or of 256 x BN by a pair of SMs (cta_group::2), each of which loads
// 128 rows of A and half of B's columns: per SM a third less to load than a 128 x 256 tile by itself.
// f32: k-blocks of 32, the three planes of both operands in a stage, so that their six products cost the
// loads of three; two accumulators, the product of the leading parts in one and the rest, 2^-8 of it, in
// the other, handed over every kDrain k-blocks and added up in registers: the tensor core truncates its
// sums, and 16 truncations in a row are as many as the result's accuracy bears (measured at K = 2001: 126 in
// a row left 2e-6 of the norm, 16 leave 2.3e-7, a plain f32 product 7.7e-7).
template <int BN, typename T, bool kPair> struct LinShape {
  static constexpr int kPlanes = Plane<T>::kCount;
  static constexpr int kBK = kPlanes == 3 ? 32 : 64;       // elements per k-block: 64- or 128-byte swizzle rows
  static constexpr int kDrain = kPlanes == 3 ? 8 : 1 << 28;
  static constexpr int kAccs = kPlanes == 3 ? 2 : 1;
  static constexpr int kBRows = kPair ? BN / 2 : BN;       // columns of B that this SM loads
  static constexpr uint32_t kABytes = kLinBM * kBK * 2, kBBytes = kBRows * kBK * 2;
  static constexpr uint32_t kStageBytes = kPlanes * (kABytes + kBBytes);
  static constexpr int kStages = 196608 / kStageBytes;
  static constexpr uint32_t kTmem = 2 * kAccs * BN;
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes + kExchangeBytes + 1024;
};

// One product C[M x N] = A B
struct LinProduct {
  LinEpilogue e;
  int kb;                 // k-blocks
  int a_mn, b_mn;         // 1: the operand is MN-major
  int tiles_m, tiles_n, splits, kb_per_split, items;
  float* partial;         // with splits > 1: [splits][M][ldp]
  long long ldp;
};

// The workers (SMs, or pairs) take the first product's items in turn, then the second's.  Where the first
// product leaves some workers, the first `late` of them, with one item more, the others take `head` items of
// the second product meanwhile.  In every round the workers are at neighbouring tiles, whose operands L2
// then serves to many.
struct LinParams {
  LinProduct p[2];
  int n_products, workers, late, head;
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
// a worker's way through its items, the same for all its warps
struct LinSchedule {
  int at0, step, worker, round1;
  __device__ __forceinline__ LinSchedule(const LinParams& prm, int w) : at0(w), step(prm.workers), worker(w), round1(0) {}
  __device__ __forceinline__ bool next(const LinParams& prm, LinWork& it) {
    int t;
    if (at0 < prm.p[0].items) {
      it.which = 0;
      t = at0;
      at0 += step;
    } else if (prm.n_products > 1) {
      const int early = step - prm.late, ahead = prm.head * early;
      if (worker < prm.late) t = ahead + round1 * step + worker;
      else if (round1 < prm.head) t = round1 * early + worker - prm.late;
      else t = ahead + (round1 - prm.head) * step + worker;
      ++round1;
      if (t >= prm.p[1].items) return false;
      it.which = 1;
    } else {
      return false;
    }
    const LinProduct& q = prm.p[it.which];
    const int tiles = q.tiles_m * q.tiles_n;
    it.split = t / tiles;
    t -= it.split * tiles;
    // groups of 8 tiles along M share the operand B's tiles while they are in L2
    const int per_group = 8 * q.tiles_n;
    const int g = t / per_group, r = t - g * per_group;
    const int gm = min(8, q.tiles_m - g * 8);
    it.tn = r / gm;
    it.tm = g * 8 + (r - it.tn * gm);
    it.kb0 = it.split * q.kb_per_split;
    it.kb1 = min(it.kb0 + q.kb_per_split, q.kb);
    return true;
  }
};

// Shared-memory matrix descriptor.  K-major: rows of kBK elements in 128- or 64-byte swizzle rows, groups of
// eight rows apart by eight times that.  MN-major (128-byte swizzle): one row holds 64 elements of the M or
// N axis at one k; eight such rows are 1024 bytes apart (stride offset), the next 64 elements of the axis one
// box of kBK rows further (leading offset).
template <int kBK> __device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, int mn) {
  const bool narrow = kBK == 32 && !mn;
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  if (mn) d |= static_cast<uint64_t>((kBK * 128u) >> 4) << 16;
  d |= static_cast<uint64_t>((narrow ? 512u : 1024u) >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(narrow ? 4 : 2) << 61;
  return d;
}

// ------------------------------------------------------------------ pairs of SMs
__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t leader_address(uint32_t saddr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(saddr));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// the same instruction for one SM and for a pair
template <bool kPair> struct Tensor;
template <> struct Tensor<false> {
  static __device__ __forceinline__ void alloc(uint32_t* slot, uint32_t n) { tmem_alloc(slot, n); tmem_relinquish(); }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) { tmem_dealloc(t, n); }
  static __device__ __forceinline__ void load(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
    tma_load_3d(dst, m, bar, c0, c1, c2);
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    umma_f16(d, a, b, idesc, acc);
  }
  static __device__ __forceinline__ void commit(uint64_t* bar) { umma_commit(bar); }
  static __device__ __forceinline__ void arrive_leader(uint64_t* bar) { mbar_arrive(bar); }
};
template <> struct Tensor<true> {
  static __device__ __forceinline__ void alloc(uint32_t* slot, uint32_t n) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(n) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  static __device__ __forceinline__ void dealloc(uint32_t t, uint32_t n) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(n) : "memory");
  }
  // into this SM's shared memory, counted on the leader's barrier
  static __device__ __forceinline__ void load(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        :
        : "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(leader_address(smem_u32(bar))), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
  // arrives on the barrier of both SMs (a commit, not a load)
  static __device__ __forceinline__ void commit(uint64_t* bar) {
    const uint16_t both_sms = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"(both_sms)
        : "memory");
  }
  static __device__ __forceinline__ void arrive_leader(uint64_t* bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_address(smem_u32(bar))) : "memory");
  }
};

// A 32 x 32 block of sums, one row per lane in v.  Where rows lie on 16-byte boundaries a lane writes its own
// row's 64 (f32: 128) bytes: whole sectors, and nothing to exchange.
template <typename T> constexpr int kRowWords = 32 / kVec16<T>;
template <typename T>
__device__ __forceinline__ void load_residual(const LinEpilogue& e, long long row, int c0, Word<T> (&res)[kRowWords<T>]) {
  if (!e.residual || row >= e.M || c0 + 32 > e.N) return;
  const Word<T>* from = reinterpret_cast<const Word<T>*>(static_cast<const T*>(e.residual) + row * e.ld_res + c0);
#pragma unroll
  for (int w = 0; w < kRowWords<T>; ++w) res[w] = from[w];
}
template <typename T>
__device__ __forceinline__ void finish_words(const LinEpilogue& e, const float* bias, const uint32_t (&v)[32], long long row, int c0,
                                             const Word<T> (&res)[kRowWords<T>]) {
  constexpr int kV = kVec16<T>;
  Word<T>* out = reinterpret_cast<Word<T>*>(static_cast<T*>(e.out) + row * e.ldo + c0);
  Word<T>* pre = reinterpret_cast<Word<T>*>(static_cast<T*>(e.pre) + row * e.ld_pre + c0);
#pragma unroll
  for (int w = 0; w < kRowWords<T>; ++w) {
    float acc[kV], b[kV];
    Word<T> y, z;
#pragma unroll
    for (int j = 0; j < kV; j += 4) {  // the same for all lanes
      const float4 f = *reinterpret_cast<const float4*>(bias + w * kV + j);
      b[j] = f.x; b[j + 1] = f.y; b[j + 2] = f.z; b[j + 3] = f.w;
    }
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] = __uint_as_float(v[w * kV + j]);
    finish_elements<T, kV>(e, acc, b, res[w], y, z);
    if (row < e.M) {
      out[w] = y;
      if (e.pre) pre[w] = z;
    }
  }
}
// Any other block goes through the warp's exchange tile, so that lanes next to each other write elements, or
// pairs of 16-bit ones where rows lie on 4-byte boundaries, next to each other.
template <typename T, int kV>
__device__ __forceinline__ void finish_through_tile(const LinEpilogue& e, float* tile, const float* bias, const uint32_t (&v)[32],
                                                    long long row0, int c0) {
  constexpr int kAcross = 32 / kV, kSteps = 16 / kV;  // lanes of a row, steps of kV rows in half a block
  const int lane = threadIdx.x & 31, at = (lane % kAcross) * kV, c = c0 + at, r = lane / kAcross;
  const T* res_at = static_cast<const T*>(e.residual) + (row0 + r) * e.ld_res + c;
  T* out_at = static_cast<T*>(e.out) + (row0 + r) * e.ldo + c;
  T* pre_at = static_cast<T*>(e.pre) + (row0 + r) * e.ld_pre + c;
  float b[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) b[j] = bias[at + j];
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    __syncwarp();
    if ((lane >> 4) == half) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<uint4*>(tile + (lane & 15) * kStagePitch + 4 * j) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    }
    __syncwarp();
    const long long left = e.M - row0 - 16 * half;
    const int rows = left < 16 ? static_cast<int>(left) : 16;
    if (c < e.N) {  // pairs: N is even
#pragma unroll 1
      for (int s0 = 0; s0 < kSteps; s0 += 8) {  // eight steps on their way at a time
        Pack<T, kV> res[8];
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (e.residual && r + (s0 + s) * kV < rows)
            res[s] = *reinterpret_cast<const Pack<T, kV>*>(res_at + (16 * half + (s0 + s) * kV) * e.ld_res);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const int row = r + (s0 + s) * kV;
          if (row >= rows) break;
          float acc[kV];
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] = tile[row * kStagePitch + at + j];
          Pack<T, kV> y, z;
          finish_elements<T, kV>(e, acc, b, res[s], y, z);
          *reinterpret_cast<Pack<T, kV>*>(out_at + (16 * half + (s0 + s) * kV) * e.ldo) = y;
          if (e.pre) *reinterpret_cast<Pack<T, kV>*>(pre_at + (16 * half + (s0 + s) * kV) * e.ld_pre) = z;
        }
      }
    }
  }
}

// a block of a split reduction's partial sums: whole words, ldp is N rounded up to 4
__device__ __forceinline__ void store_partial(const LinProduct& q, const uint32_t (&v)[32], int split, long long row, int c0) {
  if (row >= q.e.M) return;
  float* to = q.partial + (static_cast<long long>(split) * q.e.M + row) * q.ldp + c0;
#pragma unroll
  for (int j = 0; j < 32; j += 4)
    if (c0 + j < q.ldp) *reinterpret_cast<uint4*>(to + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
}

template <int BN, typename T, bool kPair>
__global__ void __launch_bounds__(kLinThreads, 1)
linear_kernel(const __grid_constant__ LinMaps maps, const __grid_constant__ LinParams prm) {
  using Shape = LinShape<BN, T, kPair>;
  using Tc = Tensor<kPair>;
  constexpr int kStages = Shape::kStages, kBK = Shape::kBK, kPlanes = Shape::kPlanes, kAccs = Shape::kAccs;
  constexpr uint32_t kABytes = Shape::kABytes, kBBytes = Shape::kBBytes, kStageBytes = Shape::kStageBytes;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint64_t full_bar[kStages];   // the pair's leader: all loads of a stage landed
  __shared__ uint64_t empty_bar[kStages];  // the products that read a stage are done
  __shared__ uint64_t acc_full[2];         // an accumulator is complete
  __shared__ uint64_t acc_empty[2];        // the pair's leader: an accumulator was drained
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // the same for the whole warp, and known to be
  const uint32_t rank = kPair ? pair_rank() : 0u;
  const int worker = kPair ? blockIdx.x >> 1 : blockIdx.x;
  const uint32_t dyn_addr = smem_u32(smem_dyn);
  const uint32_t tile_base = (dyn_addr + 1023u) & ~1023u;
  uint8_t* tiles = smem_dyn + (tile_base - dyn_addr);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], kPair ? 512 : 256); }
    abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 1) Tc::alloc(&tmem_slot, Shape::kTmem);
  tc_fence_before();
  __syncthreads();
  if (kPair) pair_sync();  // the other SM's barriers exist before anything is signalled on them
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  after_previous();  // operands may come from the kernel before
  let_next_start();
  LinSchedule schedule(prm, worker);
  LinWork it;

  // The loading and the issuing warp go through their loops as whole warps, and one elected lane issues:
  // descriptors and addresses then live in uniform registers.  With the loops inside one lane's branch they
  // had to be moved there for every instruction, and the tensor pipe waited a third of the time.
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    int stage = 0;
    uint32_t phase = 0, issued = 0, last_parity = 0;
    bool ok = true;
    int withhold = prm.withhold && blockIdx.x == 0;
    while (ok && schedule.next(prm, it)) {
      const LinProduct& q = prm.p[it.which];
      const CUtensorMap* ma = &maps.a[it.which];
      const CUtensorMap* mb = &maps.b[it.which];
      const bool a_mn = q.a_mn != 0, b_mn = q.b_mn != 0;
      const int m0 = (kPair ? 2 * it.tm + static_cast<int>(rank) : it.tm) * kLinBM;
      const int n0 = it.tn * BN + static_cast<int>(rank) * Shape::kBRows;
      for (int i = it.kb0; i < it.kb1; ++i) {
        const bool come = mbar_wait<false>(&empty_bar[stage], phase ^ 1u, &abort_flag, prm.wait_ns);
        if (!__all_sync(0xffffffffu, come)) {
          atomicCAS(prm.status, kStatusOk, kStatusProducerTimeout);
          abort_flag = 1;
          ok = false;
          break;
        }
        if (withhold) {  // tests only: this stage never arrives and the waits behind it run out
          withhold = 0;
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
          continue;
        }
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], (kPair ? 2u : 1u) * kStageBytes);
          uint8_t* sa = tiles + stage * kStageBytes;
          uint8_t* sb = sa + kPlanes * kABytes;
          const int k0 = i * kBK;
#pragma unroll
          for (int pl = 0; pl < kPlanes; ++pl) {
            if (a_mn) {
#pragma unroll
              for (int j = 0; j < kLinBM / 64; ++j)
                Tc::load(sa + pl * kABytes + j * (kBK * 128), ma, &full_bar[stage], m0 + 64 * j, k0, pl);
            } else {
              Tc::load(sa + pl * kABytes, ma, &full_bar[stage], k0, m0, pl);
            }
            if (b_mn) {
#pragma unroll
              for (int j = 0; j < Shape::kBRows / 64; ++j)
                Tc::load(sb + pl * kBBytes + j * (kBK * 128), mb, &full_bar[stage], n0 + 64 * j, k0, pl);
            } else {
              Tc::load(sb + pl * kBBytes, mb, &full_bar[stage], k0, n0, pl);
            }
          }
        }
        __syncwarp();
        issued |= 1u << stage;
        last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    if ((!ok || abort_flag) && rank == 0) {
      // leaving early: the copies in flight land first (a pair's all count on the leader's barriers, and
      // the other SM cannot leave before the leader does)
      int none = 0;
      for (int s = 0; s < kStages; ++s)
        if (issued & (1u << s)) mbar_wait<true>(&full_bar[s], (last_parity >> s) & 1u, &none, prm.wait_ns);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (of a pair: the leader's)
    if (rank == 0) {
      int stage = 0;
      uint32_t phase = 0, unit = 0;
      bool ok = true;
      while (ok && schedule.next(prm, it)) {
        const LinProduct& q = prm.p[it.which];
        const int a_mn = q.a_mn, b_mn = q.b_mn;
        const uint32_t idesc = umma_idesc_f16(kPair ? 256 : kLinBM, BN) | prm.formats | (static_cast<uint32_t>(a_mn) << 15) |
                               (static_cast<uint32_t>(b_mn) << 16);
        // an instruction's 16 steps of k: 32 bytes along a K-major row, 16 rows of an MN-major box
        const uint32_t step_a = a_mn ? (16u * 128u) >> 4 : 2u, step_b = b_mn ? (16u * 128u) >> 4 : 2u;
        const uint64_t desc_a = operand_desc<kBK>(tile_base, a_mn), desc_b = operand_desc<kBK>(tile_base + kPlanes * kABytes, b_mn);
        for (int i0 = it.kb0; i0 < it.kb1 && ok; i0 += Shape::kDrain) {
          const int i1 = it.kb1 - i0 > Shape::kDrain ? i0 + Shape::kDrain : it.kb1;
          const uint32_t buf = unit & 1u, aphase = (unit >> 1) & 1u;
          bool come = mbar_wait<false>(&acc_empty[buf], aphase ^ 1u, &abort_flag, prm.wait_ns);
          if (!__all_sync(0xffffffffu, come)) {
            atomicCAS(prm.status, kStatusOk, kStatusMmaTimeout);
            abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + buf * kAccs * BN;
          for (int i = i0; i < i1; ++i) {
            come = mbar_wait<false>(&full_bar[stage], phase, &abort_flag, prm.wait_ns);
            if (!__all_sync(0xffffffffu, come)) {
              atomicCAS(prm.status, kStatusOk, kStatusMmaTimeout);
              abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t da = desc_a + stage * (kStageBytes >> 4), db = desc_b + stage * (kStageBytes >> 4);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kBK / kLinUmmaK; ++k) {
                const uint32_t on = (i > i0 || k > 0) ? 1u : 0u;
                if constexpr (kPlanes == 1) {
                  Tc::mma(d_tmem, da + step_a * k, db + step_b * k, idesc, on);
                } else {
                  // the parts' products: the five small ones beside the large one
                  constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
                  for (int s = 0; s < 6; ++s)
                    Tc::mma(d_tmem + (s < 5 ? BN : 0), da + pa[s] * (kABytes >> 4) + step_a * k,
                            db + pb[s] * (kBBytes >> 4) + step_b * k, idesc, (s == 0 || s == 5) ? on : 1u);
                }
              }
              Tc::commit(&empty_bar[stage]);
              if (i + 1 == i1) Tc::commit(&acc_full[buf]);
            }
            __syncwarp();
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
          }
          ++unit;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    // a warp reads the quarter of the accumulator's rows that its number allows; two warps share the columns
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    constexpr int kBlocks = BN / 64;  // of 32 columns, for each of them
    const int lane = threadIdx.x & 31;
    float* tile = reinterpret_cast<float*>(tiles + static_cast<size_t>(kStages) * kStageBytes) + (warp - 2) * kExchange;
    float* bias = tile + 16 * kStagePitch;  // of the tile's columns, as f32
    const uint32_t lane_addr = (static_cast<uint32_t>(quarter * 32) << 16) + part * (BN / 2);
    uint32_t unit = 0;
    bool ok = true;
    const auto wait_full = [&]() {
      if (mbar_wait<true>(&acc_full[unit & 1u], (unit >> 1) & 1u, &abort_flag, prm.wait_ns)) {
        tc_fence_after();
        return true;
      }
      atomicCAS(prm.status, kStatusOk, kStatusEpilogueTimeout);
      abort_flag = 1;
      return false;
    };
    while (ok && schedule.next(prm, it)) {
      const LinProduct& q = prm.p[it.which];
      const LinEpilogue e = q.e;
      const long long row0 = static_cast<long long>(kPair ? 2 * it.tm + static_cast<int>(rank) : it.tm) * kLinBM + quarter * 32;
      const long long row = row0 + lane;
      const int n0 = it.tn * BN + part * (BN / 2);
      const bool whole = q.splits == 1;
      // what the tile needs beside its sums is fetched while they are still being made
      Word<T> res[kRowWords<T>];
      if (whole) {
        __syncwarp();
#pragma unroll
        for (int c = 0; c < BN / 2; c += 32) bias[c + lane] = bias_at<T>(e, n0 + c + lane);
        __syncwarp();
        if (e.words) load_residual<T>(e, row, n0, res);
      }
      const auto store = [&](const uint32_t (&v)[32], int cc) {
        const int c0 = n0 + cc * 32;
        if (!whole) {
          store_partial(q, v, it.split, row, c0);
        } else if (e.words && c0 + 32 <= e.N) {
          Word<T> now[kRowWords<T>];
#pragma unroll
          for (int w = 0; w < kRowWords<T>; ++w) now[w] = res[w];
          if (cc + 1 < kBlocks) load_residual<T>(e, row, c0 + 32, res);  // the next block's
          finish_words<T>(e, bias + cc * 32, v, row, c0, now);
        } else {
          if (sizeof(T) == 2 && e.pairs) finish_through_tile<T, sizeof(T) == 2 ? 2 : 1>(e, tile, bias + cc * 32, v, row0, c0);
          else finish_through_tile<T, 1>(e, tile, bias + cc * 32, v, row0, c0);
        }
      };
      if constexpr (kPlanes == 1) {
        if (!(ok = wait_full())) break;
#pragma unroll 1
        for (int cc = 0; cc < kBlocks; ++cc) {
          if (row0 >= e.M || n0 + cc * 32 >= e.N) break;  // the same for the whole warp
          uint32_t v[32];
          tmem_ld32(tmem_base + lane_addr + (unit & 1u) * BN + cc * 32, v);
          tmem_ld_wait();
          store(v, cc);
        }
        tc_fence_before();
        Tc::arrive_leader(&acc_empty[unit & 1u]);
        ++unit;
      } else {
        float acc[kBlocks][32];
#pragma unroll
        for (int cc = 0; cc < kBlocks; ++cc)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[cc][j] = 0.f;
        for (int i0 = it.kb0; i0 < it.kb1; i0 += Shape::kDrain) {
          if (!(ok = wait_full())) break;
#pragma unroll
          for (int cc = 0; cc < kBlocks; ++cc) {
            uint32_t v[32];
            tmem_ld32(tmem_base + lane_addr + (unit & 1u) * 2 * BN + BN + cc * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[cc][j] += __uint_as_float(v[j]);
            tmem_ld32(tmem_base + lane_addr + (unit & 1u) * 2 * BN + cc * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[cc][j] += __uint_as_float(v[j]);
          }
          tc_fence_before();
          Tc::arrive_leader(&acc_empty[unit & 1u]);
          ++unit;
        }
        if (!ok) break;
#pragma unroll
        for (int cc = 0; cc < kBlocks; ++cc) {
          if (row0 < e.M && n0 + cc * 32 < e.N) {
            uint32_t v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(acc[cc][j]);
            store(v, cc);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (kPair) pair_sync();  // neither SM leaves while the other may still signal or read it
  if (warp == 1) {
    tc_fence_after();
    Tc::dealloc(tmem_base, Shape::kTmem);
  }
}

// the partial sums of a split reduction, added in order, and the epilogue
template <typename T>
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ LinProduct q) {
  after_previous();
  let_next_start();
  const LinEpilogue e = q.e;
  const long long words = q.ldp / 4, total = e.M * words, slab = e.M * q.ldp;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * 256) {
    const long long row = i / words;
    const int c = static_cast<int>(i - row * words) * 4;
    const float* from = q.partial + row * q.ldp + c;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < q.splits; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(from + s * slab);
      acc[0] += f.x; acc[1] += f.y; acc[2] += f.z; acc[3] += f.w;
    }
    T* out = static_cast<T*>(e.out) + row * e.ldo + c;
    T* pre = static_cast<T*>(e.pre) + row * e.ld_pre + c;
    const T* from_res = static_cast<const T*>(e.residual) + row * e.ld_res + c;
    const float bias[4] = {bias_at<T>(e, c), bias_at<T>(e, c + 1), bias_at<T>(e, c + 2), bias_at<T>(e, c + 3)};
    Pack<T, 4> res, y, z;
    const bool together = e.words && c + 4 <= e.N;  // four elements lie on a multiple of their size
    if (e.residual) {
      if (together) {
        res = *reinterpret_cast<const Pack<T, 4>*>(from_res);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) res.v[j] = c + j < e.N ? from_res[j] : Elem<T>::narrow(0);
      }
    }
    finish_elements<T, 4>(e, acc, bias, res, y, z);
    if (together) {
      *reinterpret_cast<Pack<T, 4>*>(out) = y;
      if (e.pre) *reinterpret_cast<Pack<T, 4>*>(pre) = z;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c + j >= e.N) break;
        out[j] = y.v[j];
        if (e.pre) pre[j] = z.v[j];
      }
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
// eight consecutive results into the operand's planes
template <typename T>
__device__ __forceinline__ void store_planes(typename Plane<T>::type* dst, long long plane_stride, const float (&f)[8]) {
  using P = typename Plane<T>::type;
  if constexpr (Plane<T>::kCount == 3) {
    Pack<P, 8> p[3];
#pragma unroll
    for (int j = 0; j < 8; ++j) split3(f[j], p[0].v[j], p[1].v[j], p[2].v[j]);
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<Pack<P, 8>*>(dst + i * plane_stride) = p[i];
  } else {
    const Duo<float> d[4] = {Duo<float>::of(f[0], f[1]), Duo<float>::of(f[2], f[3]), Duo<float>::of(f[4], f[5]),
                             Duo<float>::of(f[6], f[7])};
    *reinterpret_cast<Word<P>*>(dst) = to_word<P>(d);
  }
}

template <typename T, bool kWords>
__device__ __forceinline__ void load8(const T* row, int c, int n, float (&f)[8]) {
  if (kWords && c + 8 <= n) {
    constexpr int kV = kVec16<T>;
#pragma unroll
    for (int i = 0; i < 8; i += kV) {
      Duo<float> d[kDuos<T>];
      widen_word(*reinterpret_cast<const Word<T>*>(row + c + i), d);
#pragma unroll
      for (int j = 0; j < kDuos<T>; ++j) { f[i + 2 * j] = d[j].lo(); f[i + 2 * j + 1] = d[j].hi(); }
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
  after_previous();
  let_next_start();
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
// 256 columns per block, eight per lane; eight warps share the block's rows, the next kDepth of each on their
// way in shared memory
constexpr int kSlopeDepth = 4;
template <typename T, int kHow>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) linear_slope_kernel(const __grid_constant__ SlopeArgs a) {
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kV = kVec16<T>, kD = kDuos<T>, kWords = 8 / kV;
  let_next_start();
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ float sm[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 256 + lane * 8;
  const T zero = Elem<T>::narrow(0);
  Duo<float> sum[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] = both(0.f);
  if (c < a.cols) {
    const long long step = static_cast<long long>(gridDim.y) * 8, first = static_cast<long long>(blockIdx.y) * 8 + warp;
    const T* gr = static_cast<const T*>(a.grad_out) + first * a.ldg;
    const T* zr = a.act ? static_cast<const T*>(a.pre) + first * a.ld_pre : nullptr;
    typename Plane<T>::type* out = static_cast<typename Plane<T>::type*>(a.dz) + first * a.ldd + c;
    const long long g_step = step * a.ldg, z_step = step * a.ld_pre, out_step = step * a.ldd;
    long long coming = first;
    Word<T>* ring = reinterpret_cast<Word<T>*>(dyn) + threadIdx.x;  // [stage][grad_out or pre][word][thread]
    const auto fetch = [&](int stage) {
      if constexpr (kHow != kInRegisters) {
        if (coming < a.rows) {
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            if (kHow == kByWords || c + w * kV < a.cols) {
              copy_word<T, kHow>(ring + ((stage * 2) * kWords + w) * 256, gr, c + w * kV, a.cols);
              if (a.act) copy_word<T, kHow>(ring + ((stage * 2 + 1) * kWords + w) * 256, zr, c + w * kV, a.cols);
            }
          }
        }
        commit_async();
        coming += step;
        gr += g_step;
        zr += z_step;
      }
    };
#pragma unroll
    for (int s = 0; s < kSlopeDepth; ++s) fetch(s);
    int stage = 0;
    for (long long r = first; r < a.rows; r += step) {
      Word<T> g[kWords], z[kWords];
      if constexpr (kHow != kInRegisters) {
        wait_async<kSlopeDepth - 1>();
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          g[w] = take_word<T, kHow>(ring + ((stage * 2) * kWords + w) * 256, c + w * kV, a.cols, zero);
          if (a.act) z[w] = take_word<T, kHow>(ring + ((stage * 2 + 1) * kWords + w) * 256, c + w * kV, a.cols, zero);
        }
        fetch(stage);
        stage = stage + 1 == kSlopeDepth ? 0 : stage + 1;
      } else {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          g[w] = read_word(gr, c + w * kV, a.cols, kSingly, zero);
          if (a.act) z[w] = read_word(zr, c + w * kV, a.cols, kSingly, zero);
        }
        gr += g_step;
        zr += z_step;
      }
      Duo<float> d[4];
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        Duo<float> gw[kD], zw[kD];
        widen_word(g[w], gw);
        if (a.act) widen_word(z[w], zw);
#pragma unroll
        for (int j = 0; j < kD; ++j) d[w * kD + j] = a.act ? gw[j] * slope_pair<kExact>(zw[j], a.act) : gw[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = sum[j] + d[j];
      if (a.dz) {
        const float f[8] = {d[0].lo(), d[0].hi(), d[1].lo(), d[1].hi(), d[2].lo(), d[2].hi(), d[3].lo(), d[3].hi()};
        store_planes<T>(out, a.plane_stride, f);
      }
      out += out_step;
    }
    if constexpr (kHow != kInRegisters) wait_async<0>();
  }
  if (!a.partial) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sm[warp][lane * 8 + 2 * j] = sum[j].lo();
    sm[warp][lane * 8 + 2 * j + 1] = sum[j].hi();
  }
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += sm[w][threadIdx.x];
  if (col < a.cols) a.partial[static_cast<long long>(blockIdx.y) * a.cols + col] = s;
}
// the blocks' column sums added in a fixed order: 32 columns per block, 32 threads per column
__global__ void __launch_bounds__(1024) linear_bias_join_kernel(const float* __restrict__ partial, int parts, int cols,
                                                                float* __restrict__ out) {
  __shared__ float sm[32][33];
  after_previous();
  let_next_start();
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int p = lane; p < parts; p += 32) s += partial[static_cast<long long>(p) * cols + c];
  }
  sm[lane][col] = s;
  __syncthreads();
  s = warp_sum(sm[col][lane]);  // a warp now holds the 32 shares of one column
  if (col == 0 && blockIdx.x * 32 + lane < cols) out[blockIdx.x * 32 + lane] = s;
}

// ------------------------------------------------------------------ host side
long long round8(long long v) { return (v + 7) / 8 * 8; }

// A stored matrix as an operand of the products: `inner` elements in a row, `outer` rows
struct Stored {
  const void* p;
  long long inner, outer, ld, plane_stride;
  int planes;
};

bool tma_ready(const void* p, long long ld) { return rows_on_16_bytes<uint16_t>(p, ld); }

struct ProductSpec {
  Stored a, b;
  bool a_mn, b_mn;
  long long M, N, K;
};

template <int BN, typename T, bool kPair>
int launch_products(const ProductSpec* s, LinProduct* p, int n, LinParams& prm, bool follows, cudaStream_t st) {
  using Shape = LinShape<BN, T, kPair>;
  LinMaps maps;
  for (int i = 0; i < n; ++i) {
    // K-major: a box of one k-block and the tile's rows; MN-major: 64 elements of the axis and one k-block
    const Stored &a = s[i].a, &b = s[i].b;
    if (make_matrix_map16(&maps.a[i], a.p, a.inner, a.outer, a.ld, a.planes, a.plane_stride, s[i].a_mn ? 64 : Shape::kBK,
                          s[i].a_mn ? Shape::kBK : kLinBM) ||
        make_matrix_map16(&maps.b[i], b.p, b.inner, b.outer, b.ld, b.planes, b.plane_stride, s[i].b_mn ? 64 : Shape::kBK,
                          s[i].b_mn ? Shape::kBK : Shape::kBRows))
      return -1;
    prm.p[i] = p[i];
  }
  if (n == 1) { maps.a[1] = maps.a[0]; maps.b[1] = maps.b[0]; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(prm.workers) * (kPair ? 2u : 1u));
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = Shape::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPair ? 2 : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1] = after_attribute();
  cfg.attrs = attr;
  cfg.numAttrs = follows ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_kernel<BN, T, kPair>, maps, prm);
  if (e != cudaSuccess) {
    fprintf(stderr, "[eshkol-b200] linear layer launch failed: %s\n", cudaGetErrorString(e));
    cudaGetLastError();
    return -1;
  }
  return 1;
}

int failed() {
  fprintf(stderr, "[eshkol-b200] linear layer launch failed: %s\n", cudaGetErrorString(cudaGetLastError()));
  return -1;
}

struct Plan {
  int bn;
  bool pair;
  int splits[2], kb_per_split[2];
  size_t partial_bytes[2];
  double item_cost[2];
};

// Tile shape and splits, by an estimate in units of one k-block (64 elements) of a 128 x 256 tile, 0.28 us.
// An item costs its k-blocks, the narrower its tile the more by what it loads, and a hand-over by its rows;
// one product's items run in whole rounds over the workers, two products even each other out; a split
// product pays for its partial sums and a second launch.  Measured at 8192 x 16384 x 4096 bf16: pairs of SMs
// 725 us, single ones 778.
template <typename T> Plan plan_products(const ProductSpec* s, int n) {
  constexpr bool kSplit3 = Plane<T>::kCount == 3;
  const int sms = lib_num_sms(), kbk = kSplit3 ? 32 : 64;
  Plan best = {};
  double best_cost = 1e300;
  // pairs on 256 x 256, single SMs on 128 x 256, 128 x 128, 128 x 64; f32: pairs on 256 x 128, then 128 x 128 and 128 x 64
  for (int shape = 0; shape < 4; ++shape) {
    if (kSplit3 && shape == 1) continue;
    const int bn = kSplit3 ? (shape == 3 ? 64 : 128) : shape <= 1 ? 256 : shape == 2 ? 128 : 64;
    Plan q = {};
    q.bn = bn;
    q.pair = shape == 0;
    const int workers = q.pair ? sms / 2 : sms, bm = q.pair ? 256 : 128;
    const double per_kb = kSplit3 ? (shape == 0 ? 2.3 : shape == 2 ? 2.9 : 1.8) : shape == 0 ? 0.93 : shape == 1 ? 1.0 : shape == 2 ? 0.6 : 0.42;
    double longest = 0, work = 0, extra = 0, alone = 0;
    for (int i = 0; i < n; ++i) {
      const double tiles = static_cast<double>((s[i].M + bm - 1) / bm) * static_cast<double>((s[i].N + bn - 1) / bn);
      const int kb = static_cast<int>((s[i].K + kbk - 1) / kbk);
      const double rows = s[i].M < bm ? static_cast<double>(s[i].M) : bm;
      const double hand_over = 2.0 + 8.0 * bn / 256 * rows / bm;
      double least = 1e300;
      for (int split = 1; split <= 64 && (split == 1 || kb / split >= 2) && (split == 1 || tiles * (split - 1) < 8.0 * workers); ++split) {
        int per = (kb + split - 1) / split;
        if (kSplit3) per = (per + 7) / 8 * 8;  // whole hand-overs
        const int parts = (kb + per - 1) / per;
        const double item = (per < kb ? per : kb) * per_kb + hand_over;
        const size_t bytes = parts > 1 ? (static_cast<size_t>(parts) * s[i].M * ((s[i].N + 3) / 4 * 4) * 4 + 1023) & ~size_t(1023) : 0;
        const double join = parts > 1 ? 14.0 + bytes * 2.0 / 1.2e6 : 0.0;
        const double cost = ceil(tiles * parts / workers) * item + join;
        if (cost < least) {
          least = cost;
          q.kb_per_split[i] = per;
          q.splits[i] = parts;
          q.item_cost[i] = item;
          q.partial_bytes[i] = bytes;
          if (i == 0) { work = tiles * parts * item; longest = item; extra = join; alone = cost; }
          else { alone = cost; }
        }
      }
      if (i == 1) {
        work += tiles * q.splits[1] * q.item_cost[1];
        extra += q.partial_bytes[1] ? 14.0 + q.partial_bytes[1] * 2.0 / 1.2e6 : 0.0;
        if (q.item_cost[1] > longest) longest = q.item_cost[1];
      }
    }
    const double cost = n == 1 ? alone : fmax(work / workers, longest) + extra;
    if (cost < best_cost) { best_cost = cost; best = q; }
  }
  return best;
}

// Multiplies one or two independent products in one launch, and joins those whose reduction was split.
// p[i].e carries the epilogue of product i; scratch_at: room for the partial sums (plan.partial_bytes); follows:
// a kernel of this call went before.
template <typename T>
int run_products(const ProductSpec* s, LinProduct* p, int n, const Plan& plan, uint8_t* scratch_at, bool follows,
                 cudaStream_t st) {
  constexpr int kBK = Plane<T>::kCount == 3 ? 32 : 64;
  LinParams prm;
  memset(&prm, 0, sizeof(prm));
  const int bm = plan.pair ? 256 : kLinBM;
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    LinProduct& q = p[i];
    q.e.M = static_cast<int>(s[i].M);
    q.e.N = static_cast<int>(s[i].N);
    q.kb = static_cast<int>((s[i].K + kBK - 1) / kBK);
    q.a_mn = s[i].a_mn; q.b_mn = s[i].b_mn;
    q.tiles_m = (q.e.M + bm - 1) / bm;
    q.tiles_n = (q.e.N + plan.bn - 1) / plan.bn;
    q.splits = plan.splits[i];
    q.kb_per_split = plan.kb_per_split[i];
    const long long items = static_cast<long long>(q.tiles_m) * q.tiles_n * q.splits;
    total += items;
    if (total > 0x3fffffffLL) return -1;
    q.items = static_cast<int>(items);
    q.ldp = (q.e.N + 3) / 4 * 4;
    q.partial = nullptr;
    if (q.splits > 1) {
      q.partial = reinterpret_cast<float*>(scratch_at);
      scratch_at += plan.partial_bytes[i];
    }
    q.e.words = rows_on_16_bytes<T>(q.e.out, q.e.ldo) && (!q.e.pre || rows_on_16_bytes<T>(q.e.pre, q.e.ld_pre)) &&
                (!q.e.residual || rows_on_16_bytes<T>(q.e.residual, q.e.ld_res));
    q.e.pairs = rows_by_elements<T>(q.e.out, q.e.ldo, q.e.N) && (!q.e.pre || rows_by_elements<T>(q.e.pre, q.e.ld_pre, q.e.N)) &&
                (!q.e.residual || rows_by_elements<T>(q.e.residual, q.e.ld_res, q.e.N));
  }
  int workers = lib_num_sms();
  if (plan.pair) workers /= 2;
  if (total < workers) workers = static_cast<int>(total);
  prm.n_products = n;
  prm.workers = workers;
  if (n == 2) {
    prm.late = p[0].items % workers;
    prm.head = prm.late ? static_cast<int>(floor(plan.item_cost[0] / plan.item_cost[1] + 0.5)) : 0;
    // no more ahead than there are
    while (prm.head > 0 && static_cast<long long>(prm.head) * (workers - prm.late) > p[1].items) --prm.head;
  }
  prm.formats = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
  prm.status = lib_status_word();
  prm.wait_ns = lib_wait_limit_ns();
  prm.withhold = lib_take_withhold();
  int launches = -1;
  if constexpr (Plane<T>::kCount == 3) {
    launches = plan.pair       ? launch_products<128, T, true>(s, p, n, prm, follows, st)
               : plan.bn == 128 ? launch_products<128, T, false>(s, p, n, prm, follows, st)
                                : launch_products<64, T, false>(s, p, n, prm, follows, st);
  } else {
    launches = plan.pair        ? launch_products<256, T, true>(s, p, n, prm, follows, st)
               : plan.bn == 256 ? launch_products<256, T, false>(s, p, n, prm, follows, st)
               : plan.bn == 128 ? launch_products<128, T, false>(s, p, n, prm, follows, st)
                                : launch_products<64, T, false>(s, p, n, prm, follows, st);
  }
  if (launches < 0) return -1;
  for (int i = 0; i < n; ++i) {
    if (p[i].splits == 1) continue;
    const long long words = p[i].ldp / 4 * p[i].e.M, cap = static_cast<long long>(lib_num_sms()) * 8;
    const long long blocks = (words + 255) / 256;
    if (launch_after(linear_join_kernel<T>, static_cast<unsigned>(blocks < cap ? blocks : cap), 256, 0, st, p[i]) != cudaSuccess)
      return failed();
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
template <typename T> int launch_pack(const PackJobs& jobs, bool follows, cudaStream_t st) {
  if (jobs.n == 0) return 0;
  const long long blocks = (jobs.total + 255) / 256, cap = static_cast<long long>(lib_num_sms()) * 16;
  const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
  if (!follows) linear_pack_kernel<T><<<grid, 256, 0, st>>>(jobs);
  else if (launch_after(linear_pack_kernel<T>, grid, 256, 0, st, jobs) != cudaSuccess) return failed();
  return 1;
}

struct LinearArgs {
  const void *x, *w;
  long long rows, d_in, d_out, ldx, ldw, ldy, ld_res, ld_pre;
  EshkolB200LinearOpts o;
};

template <typename T> int linear_forward(const LinearArgs& a, void* y, OpScratch& scratch, cudaStream_t st) {
  const bool tw = a.o.trans_w != 0;
  LinProduct epi;
  memset(&epi, 0, sizeof(epi));
  epi.e.bias = a.o.bias; epi.e.residual = a.o.residual; epi.e.out = y; epi.e.pre = a.o.pre;
  epi.e.ldo = a.ldy; epi.e.ld_res = a.ld_res; epi.e.ld_pre = a.ld_pre; epi.e.act = a.o.activation;
  if (few_rows<T>(a.rows, a.w, a.ldw, tw)) {
    SmallRows q;
    memset(&q, 0, sizeof(q));
    q.e = epi.e;
    q.e.M = static_cast<int>(a.rows); q.e.N = static_cast<int>(a.d_out);
    q.a = a.x; q.lda = a.ldx; q.w = a.w; q.ldw = a.ldw; q.K = a.d_in; q.k_contiguous = tw;
    return launch_small_rows<T>(q, st);
  }
  Carver cv;
  Operand<T> x(a.x, a.rows, a.d_in, a.ldx, false, cv);
  Operand<T> w(a.w, tw ? a.d_out : a.d_in, tw ? a.d_in : a.d_out, a.ldw, false, cv);
  ProductSpec s = {x.s, w.s, false, !tw, a.rows, a.d_out, a.d_in};
  const Plan plan = plan_products<T>(&s, 1);
  const size_t parts = cv.take(plan.partial_bytes[0]);
  uint8_t* base = scratch.reserve(cv.off, st);
  if (!base) return -1;
  x.bind(base);
  w.bind(base);
  s.a = x.s; s.b = w.s;
  PackJobs jobs = {};
  add_pack<T>(jobs, a.x, a.ldx, x);
  add_pack<T>(jobs, a.w, a.ldw, w);
  const int packs = launch_pack<T>(jobs, false, st);
  const int n = run_products<T>(&s, &epi, 1, plan, base + parts, packs > 0, st);
  return n < 0 ? -1 : packs + n;
}

template <typename T>
int linear_gradients(const LinearArgs& a, const void* grad_out, void* grad_x, void* grad_w, void* grad_bias,
                     OpScratch& scratch, cudaStream_t st) {
  const bool tw = a.o.trans_w != 0;
  int launches = 0;
  if (grad_x && few_rows<T>(a.rows, a.w, a.ldw, !tw)) {  // dz as it is needed, from grad_out and pre
    SmallRows q;
    memset(&q, 0, sizeof(q));
    q.e.out = grad_x; q.e.ldo = a.ldx;
    q.e.M = static_cast<int>(a.rows); q.e.N = static_cast<int>(a.d_in);
    q.a = grad_out; q.lda = a.ldy; q.pre = a.o.pre; q.ld_pre = a.ld_pre; q.slope = a.o.activation;
    q.w = a.w; q.ldw = a.ldw; q.K = a.d_out; q.k_contiguous = !tw;
    launches = launch_small_rows<T>(q, st);
    if (launches < 0) return -1;
    grad_x = nullptr;
    if (!grad_w && !grad_bias) return launches;
  }
  const bool products = grad_x || grad_w;
  Carver cv, none;  // an operand that no product reads takes no scratch
  // dz: grad_out itself when there is no activation and the products can read it
  Operand<T> dz(grad_out, a.rows, a.d_out, a.ldy, a.o.activation != 0, products ? cv : none);
  Operand<T> x(a.x, a.rows, a.d_in, a.ldx, false, grad_w ? cv : none);
  Operand<T> w(a.w, tw ? a.d_out : a.d_in, tw ? a.d_in : a.d_out, a.ldw, false, grad_x ? cv : none);
  ProductSpec s[2];
  LinProduct epi[2];
  memset(epi, 0, sizeof(epi));
  int n = 0;
  const auto describe = [&]() {
    n = 0;
    if (grad_x) {
      s[n] = {dz.s, w.s, false, tw, a.rows, a.d_in, a.d_out};
      epi[n].e.out = grad_x; epi[n].e.ldo = a.ldx;
      ++n;
    }
    if (grad_w) {
      if (tw) s[n] = {dz.s, x.s, true, true, a.d_out, a.d_in, a.rows};
      else s[n] = {x.s, dz.s, true, true, a.d_in, a.d_out, a.rows};
      epi[n].e.out = grad_w; epi[n].e.ldo = a.ldw;
      ++n;
    }
  };
  describe();
  Plan plan = {};
  if (n) plan = plan_products<T>(s, n);
  const size_t parts = cv.take(plan.partial_bytes[0] + plan.partial_bytes[1]);
  // blocks: as many as the SMs hold at once, at least 16 rows in each
  const long long col_blocks = (a.d_out + 255) / 256;
  long long row_blocks = static_cast<long long>(lib_num_sms()) * (sizeof(T) == 2 ? 4 : 3) / col_blocks;
  if (row_blocks > (a.rows + 15) / 16) row_blocks = (a.rows + 15) / 16;
  if (row_blocks < 1) row_blocks = 1;
  const size_t sums = cv.take(grad_bias ? static_cast<size_t>(row_blocks) * a.d_out * 4 : 0);
  uint8_t* base = scratch.reserve(cv.off, st);
  if (!base) return -1;
  dz.bind(base); x.bind(base); w.bind(base);
  describe();
  if ((products && dz.copy) || grad_bias) {
    SlopeArgs q;
    q.grad_out = grad_out; q.pre = a.o.pre; q.dz = (products && dz.copy) ? const_cast<void*>(dz.s.p) : nullptr;
    q.partial = grad_bias ? reinterpret_cast<float*>(base + sums) : nullptr;
    q.rows = a.rows; q.ldg = a.ldy; q.ld_pre = a.ld_pre; q.ldd = dz.s.ld; q.plane_stride = dz.s.plane_stride;
    q.cols = static_cast<int>(a.d_out); q.act = a.o.activation;
    q.words = rows_on_16_bytes<T>(grad_out, a.ldy) && (!q.act || rows_on_16_bytes<T>(q.pre, a.ld_pre));
    const dim3 grid(static_cast<unsigned>(col_blocks), static_cast<unsigned>(row_blocks));
    constexpr size_t smem = static_cast<size_t>(kSlopeDepth) * 2 * (8 / kVec16<T>) * 256 * 16;
    if (q.words && a.d_out % 8 == 0) linear_slope_kernel<T, kByWords><<<grid, 256, smem, st>>>(q);
    else if (rows_by_elements<T>(grad_out, a.ldy, a.d_out) && (!q.act || rows_by_elements<T>(q.pre, a.ld_pre, a.d_out)))
      linear_slope_kernel<T, kByElements><<<grid, 256, smem, st>>>(q);
    else linear_slope_kernel<T, kInRegisters><<<grid, 256, 0, st>>>(q);
    ++launches;
    if (grad_bias) {
      if (launch_after(linear_bias_join_kernel, static_cast<unsigned>((a.d_out + 31) / 32), 1024, 0, st,
                       static_cast<const float*>(q.partial), static_cast<int>(row_blocks), q.cols,
                       static_cast<float*>(grad_bias)) != cudaSuccess)
        return failed();
      ++launches;
    }
  }
  if (!products) return launches;
  PackJobs jobs = {};
  if (grad_w) add_pack<T>(jobs, a.x, a.ldx, x);
  if (grad_x) add_pack<T>(jobs, a.w, a.ldw, w);
  const bool sloped = (products && dz.copy) || grad_bias;
  const int packs = launch_pack<T>(jobs, sloped, st);
  if (packs < 0) return -1;
  const int m = run_products<T>(s, epi, n, plan, base + parts, sloped || packs > 0, st);
  return m < 0 ? -1 : launches + packs + m;
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

template <int BN, typename T, bool kPair> cudaError_t set_attribute() {
  return cudaFuncSetAttribute(linear_kernel<BN, T, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(LinShape<BN, T, kPair>::kSmem));
}
template <typename T> cudaError_t set_attributes_of() {
  constexpr int kSlopeBytes = kSlopeDepth * 2 * (8 / kVec16<T>) * 256 * 16;
  cudaError_t e = cudaFuncSetAttribute(linear_slope_kernel<T, kByWords>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlopeBytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(linear_slope_kernel<T, kByElements>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlopeBytes);
  if (e == cudaSuccess) e = set_attribute<128, T, false>();
  if (e == cudaSuccess) e = set_attribute<64, T, false>();
  if constexpr (Plane<T>::kCount == 1) {
    if (e == cudaSuccess) e = set_attribute<256, T, false>();
    if (e == cudaSuccess) e = set_attribute<256, T, true>();
  } else {
    if (e == cudaSuccess) e = set_attribute<128, T, true>();
  }
  return e;
}

}  // namespace

cudaError_t linear_set_attributes() {
  cudaError_t e = linear_small_set_attributes();
  if (e == cudaSuccess) e = set_attributes_of<float>();
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
