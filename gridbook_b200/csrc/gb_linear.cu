// 16-bit linears with their epilogue, and the products of their backward pass.
//
//     z = X W^T + bias,   Y = act(z) + R        X [M, K], W [N, K], bias [N], R and Y [M, N], bf16 or fp16, sums in fp32
//     dz = dY act'(z),  dX = dz W,  dW = dz^T X,  dbias = sum over rows of dz,  dR = dY
//
// Everything behind the product happens on the accumulators in fp32 before the one rounding to the output's type.  For the backward
// pass the forward pass also stores z, rounded to the output's type: act' is taken at the rounded z, which moves dz by half a step of z
// times |act'' dY|, an absolute bound (left of zero, where the smooth slopes are small, more than dz's own rounding).  Of dz's rounding, which
// the tensor cores need, and this together the gradients are off by 2.4e-3 of their norm in bf16 (4096 x 8192 x 5120, gelu), the output's
// rounding alone by 1.7e-3.
//
// Three kernels, which of them by an estimate of their times (route_of):
//   linear_pair_kernel   tiles of 256 rows x 128 to 256 columns on CTA pairs (cta_group::2), two accumulators, so that a tile's epilogue
//                        runs under the next tile's MMAs; the residual comes through registers meanwhile.
//   linear_rows_kernel   128 weight rows times up to 256 activation rows on one CTA, K sliced over a cluster: few rows, narrow layers.
//   linear_few_kernel    one to four rows of small layers on the plain units.
// linear_sign_kernel follows where a relu's z is kept, and settles the sign of values near zero, in z and Y alike.
// Bound by the tensor cores at the clock that the power cap leaves where tiles fill the GPU (8192 x 34816 x 5120: 2.1 ms, 1.4 PFLOP/s, what a
// plain library product sustains), by HBM at a few rows (16 x 34816 x 5120: 58 us, 92% of the copy rate), by launch, first fetches and the
// last tile's epilogue in between.
// The backward products read the same matrices where they lie, along their other axis: an operand whose rows run along the
// contraction is the tensor core's MN-major form, tiles of 64 columns x 64 rows with the 128-byte swizzle, so that nothing
// is transposed in memory.  dW's contraction runs over M: where its tiles are fewer than the pairs, M is split and the slices' fp32 sums
// are added by a second launch in their order.
#include "gb_blocks.cuh"

#include <cuda.h>
#include <algorithm>
#include <atomic>
#include <mutex>

namespace {

using namespace gb_blocks;

constexpr int kSlab = 64;                            // contraction elements of a stage: 128 bytes
constexpr int kSlabBytes = 128;
constexpr int kBM = 128;                             // rows of D that a CTA has
constexpr int kEpiWarps = 8;
constexpr uint32_t kTmemCols = 512;

// ------------------------------------------------------------------------------------------------ waits, loads, MMAs
template <bool kOfPair>
GB_DEVINL bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  if (kOfPair)
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// A bounded wait that remembers a timeout for the rest of the CTA: later waits return at once.
template <bool kOfPair>
__device__ __noinline__ void wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  uint64_t t0 = 0;
  for (uint32_t spin = 0; !*abort_flag; ++spin) {
    if (try_wait<kOfPair>(bar, parity)) return;
    if ((spin & 255u) == 255u) {
      const uint64_t now = gb_globaltimer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > 2000000000ull) { *abort_flag = 1; atomicExch(status, code); }
    }
  }
}
// By a whole warp that goes on together; false: given up.
template <bool kOfPair = false>
GB_DEVINL bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, try_wait<kOfPair>(bar, parity))) return true;
  wait_slow<kOfPair>(bar, parity, abort_flag, status, code);
  return !__any_sync(0xffffffffu, *abort_flag != 0);
}
GB_DEVINL int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
GB_DEVINL void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
GB_DEVINL void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
GB_DEVINL uint32_t of_rank(uint32_t addr, uint32_t rank) {       // the same place in the shared memory of another CTA of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// What the pair of arrive and wait hands over is tensor memory alone, ordered by its own fences: the arrive may be relaxed.
GB_DEVINL void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
GB_DEVINL void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
// Into this CTA's shared memory, reported to a barrier of the pair.
GB_DEVINL void tma_load_pair(uint32_t dst, uint64_t map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
GB_DEVINL void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(src) : "memory");
}
// An operand in shared memory, 128-byte swizzle.  K-major: rows of 128 bytes along the contraction, sixteen elements of it 32 bytes on.
// MN-major: 64 x 64 tiles of 8 KiB, their rows along M or N; sixteen rows of the contraction 2048 bytes on.
template <bool kMn>
GB_DEVINL uint64_t desc_of(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (kMn ? (uint64_t)(8192u >> 4) << 16 : 0ull) | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <bool kMn>
constexpr uint64_t kStep = kMn ? 2048 >> 4 : 32 >> 4;
template <int kCtas>
GB_DEVINL void mma_16bit(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, bool accumulate) {
  if (kCtas == 2)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
template <int kCtas>
GB_DEVINL void commit_to(uint32_t bar) {
  if (kCtas == 2) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
GB_DEVINL void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
GB_DEVINL void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(taddr));
}

// ------------------------------------------------------------------------------------------------ elements
GB_DEVINL float to_f(uint32_t half_word, int fp16) {
  return fp16 ? __half2float(__ushort_as_half((uint16_t)half_word)) : gb_bf16_bits_to_f32(half_word & 0xFFFFu);
}
GB_DEVINL uint32_t pack2(float a, float b, int fp16) {
  if (!fp16) return gb_pack_bf16x2(a, b);
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
GB_DEVINL uint16_t pack1(float a, int fp16) { return fp16 ? __half_as_ushort(__float2half_rn(a)) : (uint16_t)gb_f32_to_bf16_bits(a); }
// v / (1 + e^-t): sigmoid-weighted; both functions are off by a few units in the last place of fp32, far below the output's.
GB_DEVINL float weighted(float v, float t) { return __fdividef(v, 1.0f + __expf(-t)); }
constexpr float kTanhA = 1.5957691216057308f, kTanhB = 0.044715f;      // 2 sqrt(2 / pi): (1 + tanh(u)) / 2 is the sigmoid of 2 u

// 1 + erf(z / sqrt 2), and e^(-z^2 / 2) on the way: Abramowitz and Stegun's rational approximation 7.1.26 of erf, off by 1.5e-7 at most, a third
// of erff's instructions, and the exponential is what the slope needs too.  gelu is off by 2.1e-7 at most (at z = -3.1), a value of its tail, which
// goes to zero, by a growing part of itself: 5e-5 at -3, 5e-4 at -4 (half a step of fp16 there), 1.6e-3 at -5, 1e-2 at -8 (past half a step of
// bf16 from -5.3 on, where gelu is below 4e-7).
GB_DEVINL float one_plus_erf(float z, float& bell) {
  const float x = fabsf(z) * 0.70710678118654752f, t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f));
  bell = __expf(-0.5f * z * z);
  const float tail = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f) * bell;
  return z < 0.0f ? tail : 2.0f - tail;                    // a NaN stays one
}

template <int kN>
GB_DEVINL void activate(float (&v)[kN], int act) {
  switch (act) {
    case GB_EPI_RELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
      break;
    case GB_EPI_GELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        float bell;
        v[i] = 0.5f * v[i] * one_plus_erf(v[i], bell);
      }
      break;
    case GB_EPI_GELU_TANH:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = weighted(v[i], kTanhA * fmaf(kTanhB * v[i] * v[i], v[i], v[i]));
      break;
    case GB_EPI_SILU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = weighted(v[i], v[i]);
      break;
    default: break;
  }
}
// act' in place of its arguments.
template <int kN>
GB_DEVINL void slopes(float (&v)[kN], int act) {
  switch (act) {
    case GB_EPI_RELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = v[i] > 0.0f ? 1.0f : 0.0f;
      break;
    case GB_EPI_GELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        float bell;
        const float phi = 0.5f * one_plus_erf(v[i], bell);
        v[i] = fabsf(v[i]) > 16.0f ? phi : fmaf(v[i] * 0.39894228040143268f, bell, phi);      // (an infinity times none)
      }
      break;
    case GB_EPI_GELU_TANH:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float z = v[i], c = fminf(fmaxf(z, -16.0f), 16.0f), s = weighted(1.0f, kTanhA * fmaf(kTanhB * c * c, c, c));   // constant past these
        v[i] = z != z ? z : fmaf(kTanhA * c * s * (1.0f - s), fmaf(3.0f * kTanhB * c, c, 1.0f), s);
      }
      break;
    case GB_EPI_SILU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float s = weighted(1.0f, v[i]), c = fminf(fmaxf(v[i], -128.0f), 128.0f);     // s is 0 or 1 past these (z kept in fp16 may be infinite)
        v[i] = s * fmaf(c, 1.0f - s, 1.0f);
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = 1.0f;
  }
}

// ------------------------------------------------------------------------------------------------ CTA pairs
enum Major { kForward = 0, kRowsGrad = 1, kWeightGrad = 2 };   // which operands are MN-major: none, B, both
enum Epilogue { kPlain = 0, kResidual = 1, kKeepZ = 2, kBoth = 3 };   // kKeepZ: z is stored too

constexpr int kPairM = 256;
constexpr int kChunk = 2048;                         // 32 rows x 32 columns on their way out
constexpr int kGroupM = 16;                          // row tiles walked together before the next columns

constexpr int kOutBytes = kEpiWarps * 2 * kChunk, kPairFixed = 1024 + 512;        // alignment, barriers
template <Major kMajor, int kBN>
struct Shape {
  static constexpr bool kAmn = kMajor == kWeightGrad, kBmn = kMajor != kForward;
  static constexpr int kABytes = kBM * kSlabBytes, kBBytes = kBmn ? (kBN + 127) / 128 * 8192 : kBN / 2 * kSlabBytes, kStageBytes = kABytes + kBBytes;
  static constexpr int kFit = (227 * 1024 - kPairFixed - kOutBytes) / kStageBytes, kStages = kFit < 8 ? kFit : 8;
  static constexpr int kSmem = kStages * kStageBytes + kOutBytes + kPairFixed;
};

struct LinearParams {
  int64_t M, N;                // of D
  int k_tiles, m_tiles, n_tiles, slices, per_slice;
  uint32_t idesc;
  int fp16, act, tma;          // tma: rows of D, z and the residual come in whole 16-byte pieces
  const uint16_t *bias, *r;
  int64_t r_ld;
  uint16_t *d, *z;
  float* sums;                 // [slice][M][N] where slices > 1
  int* status;
  // few rows
  int rows_per_pass, box_rows, stages;
  // one to four rows
  const uint16_t *x, *w;
  int64_t x_ld;
  int K;
};

GB_DEVINL void tile_at(const LinearParams& p, int tile, int& mt, int& nt) {
  const int per = kGroupM * p.n_tiles, g = tile / per, in = tile - g * per;
  const int rows = min(kGroupM, p.m_tiles - g * kGroupM);
  mt = g * kGroupM + in % rows;
  nt = in / rows;
}

constexpr int kPairThreads = 32 * (kEpiWarps + 2);

template <Major kMajor, int kBN, int kEpi>
__global__ void __launch_bounds__(kPairThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_d,
                   const __grid_constant__ CUtensorMap map_z, const __grid_constant__ LinearParams p) {
  using S = Shape<kMajor, kBN>;
  constexpr bool kAmn = S::kAmn, kBmn = S::kBmn;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (gb_smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in both CTAs
  uint8_t* ring_ptr = smem_raw + (ring - gb_smem_u32(smem_raw));
  const uint32_t out_ring = ring + kStages * S::kStageBytes;            // two chunks per epilogue warp
  const uint32_t full_bar = out_ring + kOutBytes;                     // leader: both CTAs' operand tiles have landed
  const uint32_t empty_bar = full_bar + 8 * kStages;                     // the MMAs that read the stage are done
  const uint32_t acc_full = empty_bar + 8 * kStages;                     // [2] accumulator complete
  const uint32_t acc_empty = acc_full + 16;                              // [2] leader: drained by both CTAs
  const uint32_t slot = acc_empty + 16;
  volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(ring_ptr + (slot - ring));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot_ptr + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  gb_pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      bar_init(full_bar + 8 * s, 1);
      bar_init(empty_bar + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(acc_full + 8 * b, 1);
      bar_init(acc_empty + 8 * b, 2 * kEpiWarps);
    }
    *abort_flag = 0;
    gb_fence_barrier_init();
  }
  if (warp == kEpiWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  gb_cluster_sync();                                                     // both CTAs' barriers exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *slot_ptr;
  gb_pdl_wait();

  const int k_tiles = p.k_tiles, per_slice = p.per_slice;
  const int per_tile = p.m_tiles * p.n_tiles, total_tiles = per_tile * p.slices;
  const int stride = (int)(gridDim.x >> 1), first = (int)(blockIdx.x >> 1);

  if (warp == kEpiWarps) {
    // ------------------------------- producer (each CTA) -------------------------------
    // What its loop and the issuer's need lies in registers or is known to the compiler: a stage costs each of them a wait, a vote and a
    // copy or MMA issued at a time, and with widths, stages and addresses taken from the parameters the narrow tiles waited for them
    // (512 x 4096 x 4096 in tiles of 128: 17.5 us, 18.5 so; stages of two slabs, fewer of them, 21.9).
    const uint32_t full_pair = (uint32_t)uniform((int)of_rank(full_bar, 0));
    const int me = uniform((int)rank);
    const bool one = gb_elect_one();
    const uint64_t ma = reinterpret_cast<uint64_t>(&map_a), mb = reinterpret_cast<uint64_t>(&map_b);
    uint32_t at = 0, bar = 0, ph = 1;                        // the stage's place in the ring, its barriers'
    bool ok = true;
    for (int tile = first; ok && tile < total_tiles; tile += stride) {
      const int slice = tile / per_tile;
      int mt, nt;
      tile_at(p, tile - slice * per_tile, mt, nt);
      const int m0 = uniform(mt * kPairM) + me * kBM, n0 = uniform(nt * kBN) + me * (kBN / 2);
      const int k_end = uniform(min(k_tiles, (slice + 1) * per_slice)) * kSlab;
      for (int k = uniform(slice * per_slice) * kSlab; k < k_end; k += kSlab) {
        ok = warp_wait<true>(empty_bar + bar, ph, abort_flag, p.status, 101);
        if (!ok) break;
        if (one) {
          const uint32_t sa = ring + at, sb = sa + S::kABytes, full = full_pair + bar;
          if (me == 0) expect_tx(full_bar + bar, 2 * S::kStageBytes);
          if (kAmn) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i) tma_load_pair(sa + 8192 * i, ma, m0 + 64 * i, k, full);
          } else {
            tma_load_pair(sa, ma, k, m0, full);
          }
          if (kBmn) {
#pragma unroll
            for (int i = 0; i < S::kBBytes / 8192; ++i) tma_load_pair(sb + 8192 * i, mb, n0 + 64 * i, k, full);
          } else {
            tma_load_pair(sb, mb, k, n0, full);
          }
        }
        __syncwarp();
        at += S::kStageBytes;
        bar += 8;
        if (bar == 8 * kStages) { at = bar = 0; ph ^= 1; }
      }
    }
  } else if (warp == kEpiWarps + 1) {
    // --------------------------- MMA issuer (the leader's) ------------------------------
    if (uniform((int)rank) == 0) {
      const uint32_t to_peer = (uint32_t)uniform((int)(of_rank(full_bar, 1) - full_bar));   // distance of the peer's barriers
      const uint32_t tmem = (uint32_t)uniform((int)tmem_base), idesc = p.idesc;
      const bool one = gb_elect_one();
      int it = 0;
      uint32_t at = 0, bar = 0, ph = 0;
      bool ok = true;
      for (int tile = first; ok && tile < total_tiles; tile += stride, ++it) {
        const int buf = it & 1, slice = tile / per_tile, stages = uniform(min(k_tiles, (slice + 1) * per_slice) - slice * per_slice);
        ok = warp_wait<true>(acc_empty + 8 * buf, ((uint32_t)(it >> 1) & 1) ^ 1, abort_flag, p.status, 102);   // its last tile is drained
        if (!ok) break;
        const uint32_t acc = tmem + (buf ? 256u : 0u);
        for (int kt = 0; kt < stages; ++kt) {
          ok = warp_wait(full_bar + bar, ph, abort_flag, p.status, 103);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (one) {
            const uint64_t da = desc_of<kAmn>(ring + at), db = desc_of<kBmn>(ring + at + S::kABytes);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma_16bit<2>(acc, da + kStep<kAmn> * i, db + kStep<kBmn> * i, idesc, kt > 0 || i > 0);
            commit_to<2>(empty_bar + bar);
            commit_to<2>(empty_bar + to_peer + bar);
          }
          __syncwarp();
          at += S::kStageBytes;
          bar += 8;
          if (bar == 8 * kStages) { at = bar = 0; ph ^= 1; }
        }
        if (ok && one) {
          commit_to<2>(acc_full + 8 * buf);
          commit_to<2>(acc_full + to_peer + 8 * buf);
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------- epilogue (each CTA) --------------------------------
    // Lane = row, 32 columns at a time, out through shared memory (64-byte swizzle), a TMA store each; the next columns' sums and
    // residuals are on their way meanwhile.  (Residuals by TMA into the buffers of the output, and buffers of z's own, took one or two
    // of the six stages: 4096 x 8192 x 5120 with residual 263 us, keeping z 301.)
    constexpr bool kRes = (kEpi & kResidual) != 0, kZ = (kEpi & kKeepZ) != 0;
    const uint32_t acc_empty_pair = of_rank(acc_empty, 0);
    constexpr int kChunks = kBN / 32, kHalf = (kChunks + 1) / 2;
    const int mine = warp < 4 ? kHalf : kChunks - kHalf;                 // of the warp's columns
    const int quarter = warp & 3, c_lo = warp < 4 ? 0 : 32 * kHalf;
    const uint32_t out = out_ring + (uint32_t)warp * 2 * kChunk;
    const uint32_t row_at = (uint32_t)lane * 64u, swz = (uint32_t)((lane >> 1) & 3);
    const bool staged = p.tma && p.slices == 1;
    int it = 0, flip = 0;
    for (int tile = first; tile < total_tiles; tile += stride, ++it) {
      const int slice = tile / per_tile, buf = it & 1;
      int mt, nt;
      tile_at(p, tile - slice * per_tile, mt, nt);
      const int n0 = nt * kBN + c_lo, row0 = mt * kPairM + (int)rank * kBM + quarter * 32, row = row0 + lane;
      uint32_t bias[2];                                      // of columns 64 i + 2 lane and the next, zeros past the last
      if (kMajor == kForward) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = n0 + 64 * i + 2 * lane;
          bias[i] = (p.bias && c < p.N ? (uint32_t)__ldg(p.bias + c) : 0u) | (p.bias && c + 1 < p.N ? (uint32_t)__ldg(p.bias + c + 1) << 16 : 0u);
        }
      }
      uint4 rr[4];                                           // the row's residual, 32 columns
      const auto fetch_residual = [&](int c) {
        const uint16_t* from = p.r + (int64_t)row * p.r_ld + n0 + 32 * c;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          rr[q] = staged && row < p.M && n0 + 32 * c + 8 * q < p.N ? __ldg(reinterpret_cast<const uint4*>(from) + q) : make_uint4(0u, 0u, 0u, 0u);
      };
      if (kRes) fetch_residual(0);
      if (!warp_wait<true>(acc_full + 8 * buf, (uint32_t)(it >> 1) & 1, abort_flag, p.status, 104)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + (buf ? 256u : 0u) + (uint32_t)c_lo;
      uint32_t raw[32];
      tmem_ld32(at, raw);
#pragma unroll
      for (int c = 0; c < kHalf; ++c) {
        if (c >= mine) break;
        float v[32];
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]);
        if (c == mine - 1) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_cluster(acc_empty_pair + 8 * buf);
        } else {
          tmem_ld32(at + 32u * (c + 1), raw);
        }
        const int col = n0 + 32 * c;
        if (kMajor != kForward && p.slices > 1) {
          float* to = p.sums + ((int64_t)slice * p.M + row) * p.N + col;
          if (row < p.M) {
            if (p.N % 4 == 0) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                if (col + i < p.N) *reinterpret_cast<float4*>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i < p.N) to[i] = v[i];
            }
          }
          continue;
        }
        if (kMajor == kForward) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint32_t b = __shfl_sync(0xffffffffu, bias[c / 2], 16 * (c & 1) + i / 2);
            v[i] += to_f(b & 0xFFFFu, p.fp16);
            v[i + 1] += to_f(b >> 16, p.fp16);
          }
        }
        const auto put = [&](uint32_t dst) {                 // v as it is now; eight rows touch eight bank groups
#pragma unroll
          for (int q = 0; q < 4; ++q)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(dst + row_at + (((uint32_t)q ^ swz) * 16u)), "r"(pack2(v[8 * q], v[8 * q + 1], p.fp16)),
                           "r"(pack2(v[8 * q + 2], v[8 * q + 3], p.fp16)), "r"(pack2(v[8 * q + 4], v[8 * q + 5], p.fp16)),
                           "r"(pack2(v[8 * q + 6], v[8 * q + 7], p.fp16)) : "memory");
        };
        const auto send = [&](const CUtensorMap* map) {
          const uint32_t dst = out + (uint32_t)flip * kChunk;            // in turn: the chunk before last has left its buffer
          flip ^= 1;
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
          put(dst);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && row0 < p.M && col < p.N) tma_store_2d(map, col, row0, dst);   // what sticks out is not written
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        };
        // Rows that TMA does not take go through the buffers too, a row at a time with the lanes along its columns: of 32 rows at once a
        // store touches 32 sectors (4096 x 5001 x 2048 with residual 368 us).
        const int inside = min(32, (int)min((int64_t)32, p.M - row0));
        const bool column = col + lane < p.N;
        const auto cell = [&](uint32_t dst, int r) { return dst + (uint32_t)r * 64u + ((((uint32_t)lane >> 3) ^ ((uint32_t)(r >> 1) & 3u)) * 16u) + ((uint32_t)lane & 7u) * 2u; };
        const auto rows_out = [&](uint16_t* to) {
          __syncwarp();
          put(out);
          __syncwarp();
          uint16_t* at_row = to + (int64_t)row0 * p.N + col + lane;
#pragma unroll 8
          for (int r = 0; r < inside; ++r) {
            uint16_t w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(cell(out, r)));
            if (column) at_row[(int64_t)r * p.N] = w;
          }
        };
        const auto residual_in = [&]() {
          const uint16_t* from = p.r + (int64_t)row0 * p.r_ld + col + lane;
          __syncwarp();
#pragma unroll 8
          for (int r = 0; r < inside; ++r) {
            const uint16_t w = column ? __ldg(from + (int64_t)r * p.r_ld) : (uint16_t)0;
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(cell(out + kChunk, r)), "h"(w) : "memory");
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(rr[q].x), "=r"(rr[q].y), "=r"(rr[q].z), "=r"(rr[q].w) : "r"(out + kChunk + row_at + (((uint32_t)q ^ swz) * 16u)));
        };
        const auto add_residual = [&]() {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w[4] = {rr[q].x, rr[q].y, rr[q].z, rr[q].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              v[8 * q + 2 * j] += to_f(w[j] & 0xFFFFu, p.fp16);
              v[8 * q + 2 * j + 1] += to_f(w[j] >> 16, p.fp16);
            }
          }
        };
        if (staged) {
          if (kZ) send(&map_z);
          activate(v, p.act);
          if (kRes) {
            add_residual();
            if (c + 1 < mine) fetch_residual(c + 1);
          }
          send(&map_d);
        } else {
          if (kZ) rows_out(p.z);
          activate(v, p.act);
          if (kRes) {
            residual_in();
            add_residual();
          }
          rows_out(p.d);
        }
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag) __nanosleep(1000000);                   // loads and MMAs still in flight end before the memory goes
  gb_cluster_sync();                                       // the peer may still signal barriers here
  if (warp == kEpiWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
}

// ------------------------------------------------------------------------------------------------ few rows
// D[m, n] = sum over k of X[m, k] W[n, k]; kWmn: W's rows run along n (the rows' gradient, whose contraction is over the layer's
// outputs).
constexpr int kMaxRows = 256, kMaxStages = 8, kMaxSlices = 8;
constexpr int kRowsSmem = 224 * 1024;
constexpr int kRowsThreads = 32 * (kEpiWarps + 2);

// The epilogue of four neighbouring outputs of a row; `left` of them and what lies behind them are inside.
GB_DEVINL void finish4(const LinearParams& p, float (&v)[4], const float (&bias)[4], int64_t m, int n, int left) {
  const int64_t at = m * p.N + n;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] += bias[i];
  if (p.tma) {
    if (p.z) *reinterpret_cast<uint2*>(p.z + at) = make_uint2(pack2(v[0], v[1], p.fp16), pack2(v[2], v[3], p.fp16));
    activate(v, p.act);
    if (p.r) {
      const uint2 w = *reinterpret_cast<const uint2*>(p.r + m * p.r_ld + n);
      v[0] += to_f(w.x & 0xFFFFu, p.fp16); v[1] += to_f(w.x >> 16, p.fp16);
      v[2] += to_f(w.y & 0xFFFFu, p.fp16); v[3] += to_f(w.y >> 16, p.fp16);
    }
    *reinterpret_cast<uint2*>(p.d + at) = make_uint2(pack2(v[0], v[1], p.fp16), pack2(v[2], v[3], p.fp16));
  } else {
    if (p.z) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) p.z[at + i] = pack1(v[i], p.fp16);
    }
    activate(v, p.act);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p.d[at + i] = pack1(p.r ? v[i] + to_f(p.r[m * p.r_ld + n + i], p.fp16) : v[i], p.fp16);
  }
}

template <bool kWmn>
__global__ void __launch_bounds__(kRowsThreads, 1)
linear_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_s[kMaxStages], empty_s[kMaxStages], acc_s;
  __shared__ uint32_t slot_s;
  __shared__ volatile int abort_s;
  const uint32_t ring = (gb_smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in every CTA of a cluster
  const uint32_t full_bar = gb_smem_u32(full_s), empty_bar = gb_smem_u32(empty_s), acc_bar = gb_smem_u32(&acc_s);
  const uint32_t x_bytes = (uint32_t)p.box_rows * kSlabBytes, stage_bytes = kBM * kSlabBytes + x_bytes;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int pass = (int)blockIdx.x / p.n_tiles, tile = (int)blockIdx.x - pass * p.n_tiles, slice = (int)blockIdx.y;
  const int n0 = tile * kBM, m0 = pass * p.rows_per_pass;
  const int rows = (int)min((int64_t)p.rows_per_pass, p.M - m0), cols = (rows + 15) / 16 * 16;
  const int k_begin = slice * p.per_slice, k_end = min(p.k_tiles, k_begin + p.per_slice);

  gb_pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      gb_mbar_init(&full_s[s], 1);
      gb_mbar_init(&empty_s[s], 1);
    }
    gb_mbar_init(&acc_s, 1);
    abort_s = 0;
    gb_fence_barrier_init();
  }
  if (warp == kEpiWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gb_smem_u32(&slot_s)), "r"(kTmemCols / 2) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, slot_s, 0);
  gb_pdl_wait();

  if (warp == kEpiWarps) {
    // ------------------------------- producer -----------------------------------
    const bool one = gb_elect_one();
    int s = 0;
    uint32_t ph = 1;
    for (int kt = k_begin; kt < k_end; ++kt) {
      if (!warp_wait(empty_bar + 8 * s, ph, &abort_s, p.status, 111)) break;
      if (one) {
        const uint32_t st = ring + (uint32_t)s * stage_bytes, bar = full_bar + 8 * s;
        expect_tx(bar, stage_bytes);
        if (kWmn) {
#pragma unroll
          for (int i = 0; i < kBM / 64; ++i) tma_load_2d(st + 8192 * i, &map_w, n0 + 64 * i, kt * kSlab, bar);
        } else {
          tma_load_2d(st, &map_w, kt * kSlab, n0, bar);
        }
        tma_load_2d(st + kBM * kSlabBytes, &map_x, kt * kSlab, m0, bar);
      }
      __syncwarp();
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
  } else if (warp == kEpiWarps + 1) {
    // ------------------------------- MMA issuer ---------------------------------
    const bool one = gb_elect_one();
    const uint32_t idesc = p.idesc | (uint32_t)(cols >> 3) << 17 | (uint32_t)(kBM >> 4) << 24;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int kt = k_begin; kt < k_end; ++kt) {
      ok = warp_wait(full_bar + 8 * s, ph, &abort_s, p.status, 112);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (one) {
        const uint32_t st = ring + (uint32_t)s * stage_bytes;
        const uint64_t dw = desc_of<kWmn>(st), dx = desc_of<false>(st + kBM * kSlabBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_16bit<1>(tmem, dw + kStep<kWmn> * k, dx + kStep<false> * k, idesc, kt > k_begin || k > 0);
        commit_to<1>(empty_bar + 8 * s);
      }
      __syncwarp();
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
    if (ok && one) commit_to<1>(acc_bar);
    __syncwarp();
  } else {
    if (!warp_wait(acc_bar, 0, &abort_s, p.status, 113)) abort_s = 1;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // All eight warps see the same flag behind it: the wait may run out in one and end in another, and they meet at barriers below.
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
  }

  // Sums into the shared memory of the CTA that owns the activation row, [slice][own row][feature], over the operand ring: every CTA of
  // the cluster has finished its MMAs, and with them its loads.  Rows are owned in sixteens.
  const bool live = warp < kEpiWarps && !abort_s;
  const int quarter = warp & 3, feature = quarter * 32 + lane;
  const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
  const int own = (cols / 16 + p.slices - 1) / p.slices * 16;
  if (p.slices > 1) gb_cluster_sync();
  if (live) {
    for (int c = (warp >> 2) * 16; c < cols; c += 32) {
      uint32_t v[16];
      tmem_ld16(acc + (uint32_t)c, v);
      const int to = c / own, at = c - to * own;
      uint32_t dst = ring + (uint32_t)((slice * own + at) * kBM + feature) * 4u;
      if (p.slices > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(dst), "r"(to));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (p.slices > 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i)                         // rows past the last are sums of zeros
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + (uint32_t)i * kBM * 4u), "r"(v[i]) : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + (uint32_t)i * kBM * 4u), "r"(v[i]) : "memory");
      }
    }
  }
  if (p.slices > 1) gb_cluster_sync();                       // the last access to another CTA's memory lies in front of it
  else __syncthreads();
  if (live) {
    const int f = lane * 4, left = (int)min((int64_t)kBM, p.N - n0) - f;
    float bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = p.bias && i < left ? to_f(p.bias[n0 + f + i], p.fp16) : 0.0f;
    const int last = min(own, rows - slice * own);
    for (int r = warp; r < last; r += kEpiWarps) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 0.0f;
#pragma unroll 4
      for (int q = 0; q < p.slices; ++q) {
        float u[4];
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(u[0]), "=f"(u[1]), "=f"(u[2]), "=f"(u[3]) : "r"(ring + (uint32_t)((q * own + r) * kBM + f) * 4u));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += u[i];
      }
      if (left <= 0) continue;
      finish4(p, v, bias, (int64_t)m0 + slice * own + r, n0 + f, left);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (abort_s) __nanosleep(1000000);                       // loads and MMAs still in flight end before the memory goes
  if (warp == kEpiWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols / 2) : "memory");
}

// ------------------------------------------------------------------------------------------------ one to four rows
// A layer's weights are read once and multiplied on the plain fp32 units: a warp, or two to eight of them, takes a row of W, eight 16-byte
// pieces a lane on their way at a time; the activations lie in shared memory in fp32.  It needs no clusters, tensor memory or barriers,
// which are a third of a small layer's time in the few-rows kernel; that one is as fast or faster where a layer is larger, or has more
// rows (its / this one's time, us, launches back to back, weights from HBM): one row of 128 x 2048 4.4 / 2.3, 128 x 7168 6.1 / 3.6, 2048 x 2048 6.0 / 4.0,
// 4096 x 4096 9.3 / 9.9, 5120 x 17408 30.5 / 39; two rows of 1000 x 2048 5.5 / 3.9, 4096 x 4096 9.3 / 12.1; four of 256 x 2048 4.4 / 3.7.
constexpr int kFewThreads = 256, kFewRows = 4, kFewSmem = 100 * 1024;
constexpr int64_t kFewProducts = 1 << 22;                    // rows x weights up to which it is taken

template <int kM>
__global__ void __launch_bounds__(kFewThreads, 2)
linear_few_kernel(const __grid_constant__ LinearParams p) {
  extern __shared__ float4 x_s[];                            // [row][half of eight values][piece]
  __shared__ float red[kFewThreads / 32][kM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pieces = p.K / 8, split = p.slices;
  const int per_block = kFewThreads / 32 / split, mine = warp / split, part = warp - mine * split;
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  constexpr int kU = 8;
  uint4 w[kU];
  const auto fetch = [&](int n, int i0) {
    const uint4* row = reinterpret_cast<const uint4*>(p.w + (int64_t)n * p.K);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + u * 32 * split;
      w[u] = n < p.N && i < pieces ? __ldg(row + i) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  int n0 = (int)blockIdx.x * per_block;
  const int first = part * 32 + lane;
  fetch(n0 + mine, first);
  for (int i = threadIdx.x; i < kM * pieces; i += kFewThreads) {
    const int m = i / pieces, at = i - m * pieces;
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p.x + (int64_t)m * p.x_ld) + at);
    x_s[(2 * m) * pieces + at] = make_float4(to_f(q.x & 0xFFFFu, p.fp16), to_f(q.x >> 16, p.fp16), to_f(q.y & 0xFFFFu, p.fp16), to_f(q.y >> 16, p.fp16));
    x_s[(2 * m + 1) * pieces + at] = make_float4(to_f(q.z & 0xFFFFu, p.fp16), to_f(q.z >> 16, p.fp16), to_f(q.w & 0xFFFFu, p.fp16), to_f(q.w >> 16, p.fp16));
  }
  __syncthreads();
  for (; n0 < p.N; n0 += (int)gridDim.x * per_block) {
    const int n = n0 + mine;
    float acc[kM][2];
#pragma unroll
    for (int m = 0; m < kM; ++m) acc[m][0] = acc[m][1] = 0.0f;
    for (int i0 = first; i0 < pieces; i0 += kU * 32 * split) {
      if (i0 != first) fetch(n, i0);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int i = i0 + u * 32 * split;
        if (i >= pieces) break;
        const float f[8] = {to_f(w[u].x & 0xFFFFu, p.fp16), to_f(w[u].x >> 16, p.fp16), to_f(w[u].y & 0xFFFFu, p.fp16), to_f(w[u].y >> 16, p.fp16),
                            to_f(w[u].z & 0xFFFFu, p.fp16), to_f(w[u].z >> 16, p.fp16), to_f(w[u].w & 0xFFFFu, p.fp16), to_f(w[u].w >> 16, p.fp16)};
#pragma unroll
        for (int m = 0; m < kM; ++m) {
          const float4 a = x_s[(2 * m) * pieces + i], b = x_s[(2 * m + 1) * pieces + i];
          acc[m][0] = fmaf(f[0], a.x, acc[m][0]); acc[m][1] = fmaf(f[1], a.y, acc[m][1]);
          acc[m][0] = fmaf(f[2], a.z, acc[m][0]); acc[m][1] = fmaf(f[3], a.w, acc[m][1]);
          acc[m][0] = fmaf(f[4], b.x, acc[m][0]); acc[m][1] = fmaf(f[5], b.y, acc[m][1]);
          acc[m][0] = fmaf(f[6], b.z, acc[m][0]); acc[m][1] = fmaf(f[7], b.w, acc[m][1]);
        }
      }
    }
    fetch(n + (int)gridDim.x * per_block, first);            // the next row's, past the sums
    float sum[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      sum[m] = acc[m][0] + acc[m][1];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], o);
    }
    if (split > 1) {
      __syncthreads();
      if (lane == 0) {
#pragma unroll
        for (int m = 0; m < kM; ++m) red[warp][m] = sum[m];
      }
      __syncthreads();
    }
    float v[1] = {0.0f};
#pragma unroll
    for (int m = 0; m < kM; ++m)
      if (lane == m) v[0] = sum[m];
    if (part == 0 && lane < kM && n < p.N) {                 // lane m finishes row m
      if (split > 1) {
        v[0] = 0.0f;
        for (int q = 0; q < split; ++q) v[0] += red[warp + q][lane];
      }
      const int64_t at = (int64_t)lane * p.N + n;
      if (p.bias) v[0] += to_f(p.bias[n], p.fp16);
      if (p.z) p.z[at] = pack1(v[0], p.fp16);
      activate(v, p.act);
      p.d[at] = pack1(p.r ? v[0] + to_f(p.r[(int64_t)lane * p.r_ld + n], p.fp16) : v[0], p.fp16);
    }
  }
}

// ------------------------------------------------------------------------------------------------ elementwise parts of the backward pass
struct DzParams {
  const uint16_t *dy, *z;
  uint16_t* dz;               // or null: only the column sums
  int64_t M, N, dy_ld, dz_ld;
  int fp16, act;
  float* part;                // [blocks along M][N] column sums, or null
};
constexpr int kDzThreads = 256, kDzCols = 256, kDzRows = 4;

// A warp takes four rows of 256 columns at a time, a lane eight columns; a block's warps add their column sums up in their order.
template <bool kVec>
__global__ void __launch_bounds__(kDzThreads)
linear_dz_kernel(const __grid_constant__ DzParams p) {
  __shared__ float s[kDzThreads / 32][kDzCols];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * kDzCols + lane * 8;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  const int64_t step = (int64_t)gridDim.y * (kDzThreads / 32) * kDzRows;
  for (int64_t m0 = ((int64_t)blockIdx.y * (kDzThreads / 32) + warp) * kDzRows; m0 < p.M; m0 += step) {
    uint32_t g[kDzRows][4], w[kDzRows][4];                  // every row's bytes are on their way before the first is looked at
#pragma unroll
    for (int r = 0; r < kDzRows; ++r) {
      const int64_t m = m0 + r;
      const uint16_t *dy = p.dy + m * p.dy_ld + c, *z = p.z + m * p.N + c;
#pragma unroll
      for (int i = 0; i < 4; ++i) g[r][i] = w[r][i] = 0u;
      if (m >= p.M) continue;
      if (kVec) {
        if (c < p.N) {
          const uint4 a = __ldg(reinterpret_cast<const uint4*>(dy));
          g[r][0] = a.x; g[r][1] = a.y; g[r][2] = a.z; g[r][3] = a.w;
          if (p.z) { const uint4 b = __ldg(reinterpret_cast<const uint4*>(z)); w[r][0] = b.x; w[r][1] = b.y; w[r][2] = b.z; w[r][3] = b.w; }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.N) {
            g[r][i >> 1] |= (uint32_t)dy[i] << (16 * (i & 1));
            if (p.z) w[r][i >> 1] |= (uint32_t)z[i] << (16 * (i & 1));
          }
      }
    }
#pragma unroll
    for (int r = 0; r < kDzRows; ++r) {
      if (m0 + r >= p.M) break;
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = to_f(g[r][i >> 1] >> (16 * (i & 1)) & 0xFFFFu, p.fp16);
      if (p.z) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f(w[r][i >> 1] >> (16 * (i & 1)) & 0xFFFFu, p.fp16);
        slopes(f, p.act);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= f[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += d[i];
      if (p.dz) {
        uint16_t* to = p.dz + (m0 + r) * p.dz_ld + c;
        if (kVec) {
          if (c < p.N)
            *reinterpret_cast<uint4*>(to) = make_uint4(pack2(d[0], d[1], p.fp16), pack2(d[2], d[3], p.fp16), pack2(d[4], d[5], p.fp16), pack2(d[6], d[7], p.fp16));
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < p.N) to[i] = pack1(d[i], p.fp16);
        }
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[warp][lane * 8 + i] = acc[i];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * kDzCols + threadIdx.x;
  if (col >= p.N) return;
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kDzThreads / 32; ++w) sum += s[w][threadIdx.x];
  p.part[(int64_t)blockIdx.y * p.N + col] = sum;
}

// The relu's gradient has a step at zero, so that the sign of z there matters as its value elsewhere does not.  The tensor cores' sums
// drop the bits behind the accumulator at every one of their K/16 steps and are off by about 5e-6 of a row's usual value at K = 7232, which turns
// the sign of three values in 1.5 million: few, but each is a whole value of the gradient (2e-3 of an fp16 gradient's norm, ten times
// its rounding).  So where z is kept for the backward pass, the values that such an error can carry across zero are summed up again in fp32
// on the plain units, one in 15000 of them.  How large z is otherwise is read off its own row (a warp's 256 columns) and its own column
// (the four rows), so that a row or a weight that is small as a whole counts as that; exact zeros stand.  Y is written again from the same
// sum, so that a value has a gradient where it is above zero and nowhere else.
// Bound by the read of z and the few rows that are summed up: 30 us for 4096 x 8192 values with K = 5120 (10 for the read alone), 6 for 411 x 3648 with K = 7232.
// Magnitudes are compared as pairs of integers (as floats 46 us).  No more than kMostAgain of 1024 values are summed up again, which bounds the time for values of any other spread.
struct SignParams {
  const uint16_t *x, *w, *bias, *r;
  uint16_t *z, *y;
  int64_t M, N, K, x_ld, r_ld;
  int fp16;
  float reach;
};
constexpr int kMostAgain = 4;

template <bool kVec>
__global__ void __launch_bounds__(kDzThreads)
linear_sign_kernel(const __grid_constant__ SignParams p) {
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = (int64_t)blockIdx.x * kDzCols, c = c0 + lane * 8;
  const int64_t step = (int64_t)gridDim.y * (kDzThreads / 32) * kDzRows;
  for (int64_t m0 = ((int64_t)blockIdx.y * (kDzThreads / 32) + warp) * kDzRows; m0 < p.M; m0 += step) {
    uint32_t a[kDzRows][4], row[kDzRows], col[4];            // magnitudes in pairs, as integers: they order as the numbers do
#pragma unroll
    for (int r = 0; r < kDzRows; ++r) {
      const uint16_t* z = p.z + (m0 + r) * p.N + c;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[r][i] = 0u;
      if (m0 + r >= p.M) continue;
      if (kVec) {
        if (c < p.N) { const uint4 v = *reinterpret_cast<const uint4*>(z); a[r][0] = v.x; a[r][1] = v.y; a[r][2] = v.z; a[r][3] = v.w; }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.N) a[r][i >> 1] |= (uint32_t)z[i] << (16 * (i & 1));
      }
    }
#pragma unroll
    for (int r = 0; r < kDzRows; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[r][i] &= 0x7FFF7FFFu;
      const uint32_t top = __vmaxu2(__vmaxu2(a[r][0], a[r][1]), __vmaxu2(a[r][2], a[r][3]));
      const float most = p.reach * to_f(__reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16)), p.fp16);
      row[r] = pack2(most, most, p.fp16) & 0x7FFF7FFFu;
    }
    const bool whole = m0 + kDzRows <= p.M;                  // fewer rows say nothing of a column
    uint32_t any = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t top = __vmaxu2(__vmaxu2(a[0][i], a[1][i]), __vmaxu2(a[2][i], a[3][i]));
      col[i] = whole ? pack2(p.reach * to_f(top & 0xFFFFu, p.fp16), p.reach * to_f(top >> 16, p.fp16), p.fp16) & 0x7FFF7FFFu : 0x7FFF7FFFu;
#pragma unroll
      for (int r = 0; r < kDzRows; ++r) any |= __vcmpltu2(a[r][i], __vminu2(row[r], col[i]));
    }
    if (!__any_sync(0xffffffffu, any != 0u)) continue;
    uint32_t near = 0u;
#pragma unroll
    for (int r = 0; r < kDzRows; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t is = __vcmpltu2(a[r][i], __vminu2(row[r], col[i])) & __vcmpgtu2(a[r][i], 0u);
        near |= ((is & 1u) | (is >> 16 & 1u) << 1) << (r * 8 + 2 * i);
      }
    for (int left = kMostAgain; left > 0; --left) {
      const uint32_t who = __ballot_sync(0xffffffffu, near != 0u);
      if (who == 0u) break;
      const int src = __ffs(who) - 1, bit = __ffs(__shfl_sync(0xffffffffu, near, src)) - 1;
      if (lane == src) near &= near - 1u;
      const int64_t m = m0 + (bit >> 3), n = c0 + src * 8 + (bit & 7);
      const uint4 *xs = reinterpret_cast<const uint4*>(p.x + m * p.x_ld), *ws = reinterpret_cast<const uint4*>(p.w + n * p.K);
      float s0 = 0.0f, s1 = 0.0f;
      constexpr int kU = 8;                                  // pieces of both rows on their way at once
      for (int64_t k0 = lane; k0 < p.K / 8; k0 += 32 * kU) {
        uint4 f[kU], g[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          f[u] = g[u] = make_uint4(0u, 0u, 0u, 0u);
          if (k0 + u * 32 < p.K / 8) { f[u] = __ldg(xs + k0 + u * 32); g[u] = __ldg(ws + k0 + u * 32); }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const uint32_t fs[4] = {f[u].x, f[u].y, f[u].z, f[u].w}, gs[4] = {g[u].x, g[u].y, g[u].z, g[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s0 = fmaf(to_f(fs[i] & 0xFFFFu, p.fp16), to_f(gs[i] & 0xFFFFu, p.fp16), s0);
            s1 = fmaf(to_f(fs[i] >> 16, p.fp16), to_f(gs[i] >> 16, p.fp16), s1);
          }
        }
      }
      float s = s0 + s1;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) {
        if (p.bias) s += to_f(p.bias[n], p.fp16);
        const float y = s < 0.0f ? 0.0f : s;
        p.z[m * p.N + n] = pack1(s, p.fp16);
        p.y[m * p.N + n] = pack1(p.r ? y + to_f(p.r[m * p.r_ld + n], p.fp16) : y, p.fp16);
      }
    }
  }
}

// The slices' sums, in their order, and the epilogue behind them; a thread has four neighbours of a row.
__global__ void __launch_bounds__(256)
linear_join_kernel(const __grid_constant__ LinearParams p) {
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, m = blockIdx.y, at = m * p.N + n, values = p.M * p.N;
  if (n >= p.N) return;
  const int left = (int)min((int64_t)4, p.N - n);
  float v[4] = {}, bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = p.bias && i < left ? to_f(p.bias[n + i], p.fp16) : 0.0f;
  for (int s = 0; s < p.slices; ++s) {
    if (p.N % 4 == 0) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p.sums + s * values + at));
      v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) v[i] += p.sums[s * values + at + i];
    }
  }
  finish4(p, v, bias, m, (int)n, left);
}

// ------------------------------------------------------------------------------------------------ host
std::mutex g_mutex;
int g_pairs[64];                                             // pairs that run at once, per device (0: not asked)
std::atomic<bool> g_ready[64];
GbClusters g_clusters;

int set_limits() {
#define GB_ATTR(k, bytes) GB_CUDA_OK(cudaFuncSetAttribute((const void*)k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
#define GB_PAIR(M, N, E) GB_ATTR((linear_pair_kernel<M, N, E>), (Shape<M, N>::kSmem))
#define GB_FORWARD(N) GB_PAIR(kForward, N, kPlain); GB_PAIR(kForward, N, kResidual); GB_PAIR(kForward, N, kKeepZ); GB_PAIR(kForward, N, kBoth)
  GB_FORWARD(256);
  GB_FORWARD(224);
  GB_FORWARD(192);
  GB_FORWARD(160);
  GB_FORWARD(128);
  GB_PAIR(kRowsGrad, 256, kPlain);
  GB_PAIR(kRowsGrad, 192, kPlain);
  GB_PAIR(kRowsGrad, 128, kPlain);
  GB_PAIR(kWeightGrad, 256, kPlain);
  GB_PAIR(kWeightGrad, 192, kPlain);
  GB_PAIR(kWeightGrad, 128, kPlain);
#undef GB_FORWARD
  GB_ATTR(linear_few_kernel<1>, kFewSmem);
  GB_ATTR(linear_few_kernel<2>, kFewSmem);
  GB_ATTR(linear_few_kernel<3>, kFewSmem);
  GB_ATTR(linear_few_kernel<4>, kFewSmem);
  GB_ATTR(linear_rows_kernel<false>, kRowsSmem);
  GB_ATTR(linear_rows_kernel<true>, kRowsSmem);
#undef GB_PAIR
#undef GB_ATTR
  return GB_OK;
}

// Once per device: the kernels' shared memory, and how many pairs run at once.
int ready(int* pairs) {
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  GB_REQUIRE(dev >= 0 && dev < 64, "device %d out of range", dev);
  if (!g_ready[dev].load(std::memory_order_acquire)) {
    if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
    std::lock_guard<std::mutex> lock(g_mutex);
    const int rc = set_limits();
    if (rc != GB_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * 256);
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = Shape<kForward, 256>::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    GB_CUDA_OK(cudaOccupancyMaxActiveClusters(&n, linear_pair_kernel<kForward, 256, kPlain>, &cfg));
    GB_REQUIRE(n > 0, "no CTA pair runs on this device");
    g_pairs[dev] = n;
    g_ready[dev].store(true, std::memory_order_release);
  }
  *pairs = g_pairs[dev];
  return GB_OK;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Operand maps: K-major [rows, contraction] in boxes of 64 x box_rows, MN-major [contraction, columns] in boxes of 64 x 64.
int operand(CUtensorMap* map, const void* base, int64_t rows, int64_t inner, int64_t ld, int box_rows) {
  return gb_tensor_map_rows16(map, base, inner, rows, ld, kSlab, box_rows, 128);
}
int tile_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld) { return gb_tensor_map_rows16(map, base, cols, rows, ld, 32, 32, 64); }

struct Mats {
  const void *a, *b;
  int64_t a_ld, b_ld, K;       // K: the contraction
};

template <Major kMajor, int kBN, int kEpi>
int run_pair(const Mats& m, LinearParams p, int pairs, cudaStream_t stream) {
  using S = Shape<kMajor, kBN>;
  p.k_tiles = (int)ceil_div(m.K, kSlab);
  p.m_tiles = (int)ceil_div(p.M, kPairM);
  p.n_tiles = (int)ceil_div(p.N, kBN);
  p.per_slice = (int)ceil_div(p.k_tiles, p.slices);
  p.slices = (int)ceil_div(p.k_tiles, p.per_slice);
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles * p.slices;
  GB_REQUIRE(tiles < (1ll << 30), "too many output tiles");
  p.idesc |= ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kPairM >> 4) << 24) | (S::kAmn ? 1u << 15 : 0u) | (S::kBmn ? 1u << 16 : 0u);
  CUtensorMap map_a, map_b, map_d = {}, map_z = {};
  int rc = S::kAmn ? operand(&map_a, m.a, m.K, p.M, m.a_ld, kSlab) : operand(&map_a, m.a, p.M, m.K, m.a_ld, kBM);
  if (rc != GB_OK) return rc;
  rc = S::kBmn ? operand(&map_b, m.b, m.K, p.N, m.b_ld, kSlab) : operand(&map_b, m.b, p.N, m.K, m.b_ld, kBN / 2);
  if (rc != GB_OK) return rc;
  if (p.tma && p.slices == 1) {
    rc = tile_map(&map_d, p.d, p.M, p.N, p.N);
    if (rc == GB_OK && (kEpi & kKeepZ)) rc = tile_map(&map_z, p.z, p.M, p.N, p.N);
    if (rc != GB_OK) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs)));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = gb_pdl_enabled() ? 2 : 1;
  gb_count_launch();
  GB_CUDA_OK(cudaLaunchKernelEx(&cfg, linear_pair_kernel<kMajor, kBN, kEpi>, map_a, map_b, map_d, map_z, p));
  return GB_OK;
}

// Rows of a pass: all of them, else 192 or 256, whichever leaves fewer passes, then fewer empty rows.
int pass_rows(int64_t M) {
  if (M <= kMaxRows) return (int)M;
  return ceil_div(M, 192) == ceil_div(M, 256) ? 192 : 256;
}
struct Split { int rows, slices, per_slice; int64_t tiles; };
// K slices of the few-rows kernel: as many as the SMs take, at least four slabs each, no more than four past 64 rows.
Split split_of(int64_t M, int64_t N, int64_t k_tiles) {
  Split s;
  s.rows = pass_rows(M);
  s.tiles = ceil_div(N, kBM) * ceil_div(M, s.rows);
  const int64_t sms = gb_sm_count();
  int want = 1;
  for (int n = 2; n <= (s.rows <= 64 ? kMaxSlices : 4) && s.tiles * n <= sms && n * 4 <= k_tiles; ++n)
    if (s.tiles <= g_clusters.ask((const void*)linear_rows_kernel<false>, kRowsThreads, kRowsSmem, n)) want = n;
  s.per_slice = (int)ceil_div(k_tiles, want);
  s.slices = (int)ceil_div(k_tiles, s.per_slice);
  return s;
}
int run_join(const LinearParams& p, cudaStream_t stream) {
  GB_REQUIRE(p.M <= 65535, "too many rows of sliced sums");
  GB_CUDA_OK(gb_launch(linear_join_kernel, dim3((unsigned)ceil_div(p.N, 1024), (unsigned)p.M), dim3(256), 0, stream, p));
  return GB_OK;
}

template <bool kWmn>
int run_rows(const Mats& m, LinearParams p, cudaStream_t stream) {   // a: activation rows, b: weights
  p.k_tiles = (int)ceil_div(m.K, kSlab);
  const Split split = split_of(p.M, p.N, p.k_tiles);
  GB_REQUIRE(split.tiles < (1ll << 31), "too many output tiles");
  p.rows_per_pass = split.rows;
  p.box_rows = (int)ceil_div(split.rows, 16) * 16;
  p.n_tiles = (int)ceil_div(p.N, kBM);
  p.per_slice = split.per_slice;
  p.slices = split.slices;
  p.idesc |= kWmn ? 1u << 15 : 0u;
  const int stage = kBM * kSlabBytes + p.box_rows * kSlabBytes;
  p.stages = (kRowsSmem - 1024) / stage;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  int bytes = p.stages * stage;
  const int sums = (int)ceil_div(p.box_rows / 16, p.slices) * 16 * p.slices * kBM * 4;
  if (bytes < sums) bytes = sums;
  CUtensorMap map_w, map_x;
  int rc = kWmn ? operand(&map_w, m.b, m.K, p.N, m.b_ld, kSlab) : operand(&map_w, m.b, p.N, m.K, m.b_ld, kBM);
  if (rc != GB_OK) return rc;
  rc = operand(&map_x, m.a, p.M, m.K, m.a_ld, p.box_rows);
  if (rc != GB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)split.tiles, (unsigned)p.slices);
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = (size_t)bytes + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (gb_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.slices > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1; attr[n].val.clusterDim.y = (unsigned)p.slices; attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  gb_count_launch();
  GB_CUDA_OK(cudaLaunchKernelEx(&cfg, linear_rows_kernel<kWmn>, map_w, map_x, p));
  return GB_OK;
}

// Warps a row of W: more than one where the rows are fewer than sixteen warps an SM and long enough.
int run_few(const Mats& m, LinearParams p, cudaStream_t stream) {
  p.x = static_cast<const uint16_t*>(m.a);
  p.w = static_cast<const uint16_t*>(m.b);
  p.x_ld = m.a_ld;
  p.K = (int)m.K;
  const int64_t sms = gb_sm_count();
  p.slices = 1;
  while (p.slices < 8 && p.N * p.slices < sms * 16 && m.K >= p.slices * 2 * 2048) p.slices *= 2;
  const size_t smem = (size_t)p.M * (size_t)m.K * 4;
  const int64_t blocks = ceil_div(p.N * p.slices, kFewThreads / 32), fit = std::max<int64_t>(1, std::min<int64_t>(4, (int64_t)(220 * 1024 / (smem + 1024))));
  const dim3 grid((unsigned)std::min(blocks, sms * fit));
  switch (p.M) {
    case 1: GB_CUDA_OK(gb_launch(linear_few_kernel<1>, grid, dim3(kFewThreads), smem, stream, p)); break;
    case 2: GB_CUDA_OK(gb_launch(linear_few_kernel<2>, grid, dim3(kFewThreads), smem, stream, p)); break;
    case 3: GB_CUDA_OK(gb_launch(linear_few_kernel<3>, grid, dim3(kFewThreads), smem, stream, p)); break;
    default: GB_CUDA_OK(gb_launch(linear_few_kernel<4>, grid, dim3(kFewThreads), smem, stream, p)); break;
  }
  return GB_OK;
}

LinearParams params_of(int64_t M, int64_t N, int dtype, void* d) {
  LinearParams p = {};
  p.M = M; p.N = N;
  p.slices = 1;
  p.fp16 = dtype == GB_DTYPE_FP16;
  p.idesc = (1u << 4) | (p.fp16 ? 0u : (1u << 7) | (1u << 10));
  p.tma = N % 8 == 0;
  p.d = static_cast<uint16_t*>(d);
  p.status = gb_status_word();
  return p;
}

// Which kernel a product takes, and how wide a pair's tiles are: what this estimate, in us, is least for.  A slab of a tile costs what its
// MMAs take, 30% more than at full rate, or what the fetches of all CTAs that run with it take out of L2 at 14 TB/s; in front and
// behind are the launch, the first fetches and the last tile's epilogue, and the slices' sums on their way to each other.  Measured (estimated), us, weights
// from HBM, tiles of 128 / 160 / 192 / 256 columns / few-rows kernel:
//   128 x 4096 x 4096    17.8 (17.8) / 20.3 / 22.5 / 27.5 (28.4) / 13.8 (13.3)
//   256 x 4096 x 4096    17.8 / 20.2 / 22.4 / 27.6 / 19.0 (17.3)
//   512 x 4096 x 4096    18.5 (19.4) / 20.3 / 23.5 / 28.5 (28.4) / 23.4
//   1000 x 2048 x 2048   12.4 (12.2) / 14.2 / 15.5 / 18.1 (17.2) / 17.8
//   333 x 5120 x 17408   97 / 65 (65) / 72 (77) / 92 (101) / 81 (77)
//   700 x 4096 x 4096    29.3 / 32.4 / 23.7 / 29.9 / 36.5
//   4096 x 8192 x 5120   273 / 254 / 249 / 225
double slab_us(int64_t ctas, double bytes, double columns) { return std::max(columns * 2.0 / 1900.0 * 1.3, (double)ctas * bytes / 14e6); }
double pair_us(int64_t M, int64_t N, int64_t k_tiles, int width, int64_t pairs) {
  const int64_t tiles = ceil_div(M, kPairM) * ceil_div(N, width), full = tiles / pairs, rest = tiles - full * pairs;
  const double bytes = kBM * kSlabBytes + width / 2 * kSlabBytes;
  return 4.0 + width / 128.0 + (double)k_tiles * ((double)full * slab_us(2 * pairs, bytes, width) + (rest ? slab_us(2 * rest, bytes, width) : 0.0));
}
double rows_us(int64_t M, int64_t N, int64_t k_tiles) {
  const Split s = split_of(M, N, k_tiles);
  const int64_t sms = gb_sm_count(), ctas = s.tiles * s.slices, box = ceil_div(s.rows, 16) * 16;
  return 4.5 + (s.slices > 1 ? 1.0 + 0.02 * s.rows : 0.01 * s.rows) +
         (double)(ceil_div(ctas, sms) * s.per_slice) * slab_us(std::min(ctas, sms), kBM * kSlabBytes + (double)box * kSlabBytes, (double)box);
}
constexpr int kWidths[] = {256, 224, 192, 160, 128}, kGradWidths[] = {256, 192, 128};
template <int kN>
int width_of(const int (&widths)[kN], int64_t M, int64_t N, int64_t k_tiles, int64_t pairs, double* us = nullptr) {
  int best = 0;
  double least = 0.0;
  for (int w : widths) {
    const double t = pair_us(M, N, k_tiles, w, pairs);
    if (best == 0 || t < least) { least = t; best = w; }
  }
  if (us) *us = least;
  return best;
}
// Width of a pair's tiles; 0: the few-rows kernel.
template <int kN>
int route_of(const int (&widths)[kN], int64_t M, int64_t N, int64_t K, int pairs) {
  const int64_t k_tiles = ceil_div(K, kSlab);
  double us;
  const int width = width_of(widths, M, N, k_tiles, pairs, &us);
  return M <= 1024 && rows_us(M, N, k_tiles) < us ? 0 : width;
}
template <int kEpi>
int run_forward(int width, const Mats& m, const LinearParams& p, int pairs, cudaStream_t st) {
  switch (width) {
    case 224: return run_pair<kForward, 224, kEpi>(m, p, pairs, st);
    case 192: return run_pair<kForward, 192, kEpi>(m, p, pairs, st);
    case 160: return run_pair<kForward, 160, kEpi>(m, p, pairs, st);
    case 128: return run_pair<kForward, 128, kEpi>(m, p, pairs, st);
    default: return run_pair<kForward, 256, kEpi>(m, p, pairs, st);
  }
}
template <Major kMajor>
int run_grad(int width, const Mats& m, const LinearParams& p, int pairs, cudaStream_t st) {
  switch (width) {
    case 192: return run_pair<kMajor, 192, kPlain>(m, p, pairs, st);
    case 128: return run_pair<kMajor, 128, kPlain>(m, p, pairs, st);
    default: return run_pair<kMajor, 256, kPlain>(m, p, pairs, st);
  }
}

int check_shape(int64_t M, int64_t N, int64_t K, int dtype) {
  GB_REQUIRE(dtype == GB_DTYPE_BF16 || dtype == GB_DTYPE_FP16, "bf16 or fp16 expected");
  GB_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31), "bad shape M=%lld N=%lld K=%lld", (long long)M,
             (long long)N, (long long)K);
  GB_REQUIRE(K % 8 == 0, "K=%lld: rows are fetched in 16-byte pieces, a multiple of 8 is needed", (long long)K);
  return GB_OK;
}
bool aligned(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// The backward pass's plan: where the pieces of the workspace lie, and over how many slices dW's contraction is split.
struct GradPlan {
  bool own_dz;                 // dz is a matrix of its own
  int64_t dz_ld, dz_at, part_at, sums_at, bytes;
  int part_rows, slices, rows_width, width;                  // slices of dW, widths of dX's and dW's tiles
};
GradPlan grad_plan(int64_t M, int64_t N, int64_t K, int act, bool rows_too, bool weight, bool bias, bool dy_whole, int pairs) {
  const bool products = rows_too || weight;
  GradPlan g = {};
  auto up = [](int64_t v) { return (v + 255) & ~(int64_t)255; };
  g.dz_ld = ceil_div(N, 8) * 8;
  g.own_dz = products && (act != GB_EPI_NONE || N % 8 != 0 || !dy_whole);
  int64_t at = 0;
  g.dz_at = at;
  if (g.own_dz) at += up(M * g.dz_ld * 2);
  const int64_t sms = gb_sm_count() > 0 ? gb_sm_count() : 148;
  // about eight blocks an SM; a block's warps take four rows each at least
  int64_t rows = ceil_div(sms * 8, ceil_div(N, kDzCols));
  if (rows > ceil_div(M, 32)) rows = ceil_div(M, 32);
  g.part_rows = (int)(rows < 1 ? 1 : rows > 512 ? 512 : rows);
  g.part_at = at;
  if (bias) at += up((int64_t)g.part_rows * N * 4);
  g.sums_at = at;
  g.slices = 1;
  if (rows_too) g.rows_width = route_of(kGradWidths, M, K, N, pairs);
  if (weight) {
    const int64_t k_tiles = ceil_div(M, kSlab);
    g.width = width_of(kGradWidths, N, K, k_tiles, pairs);
    const int64_t tiles = ceil_div(N, kPairM) * ceil_div(K, g.width);
    // as many slices as the pairs take at once, of at least eight slabs
    while (g.slices < 16 && tiles * (g.slices + 1) <= pairs && (g.slices + 1) * 8 <= k_tiles) ++g.slices;
    if (g.slices > 1) at += up((int64_t)g.slices * N * K * 4);
  }
  g.bytes = at;
  return g;
}

int run_signs(const Mats& m, const LinearParams& p, cudaStream_t st) {
  SignParams s = {};
  s.x = static_cast<const uint16_t*>(m.a);
  s.w = static_cast<const uint16_t*>(m.b);
  s.bias = p.bias;
  s.r = p.r;
  s.z = p.z;
  s.y = p.d;
  s.M = p.M; s.N = p.N; s.K = m.K; s.x_ld = m.a_ld; s.r_ld = p.r_ld;
  s.fp16 = p.fp16;
  s.reach = (float)ceil_div(m.K, 16) * 0x1p-24f;
  const int64_t cols = ceil_div(p.N, kDzCols), rows = std::min<int64_t>(ceil_div(p.M, kDzThreads / 32 * kDzRows), std::max<int64_t>(1, (int64_t)gb_sm_count() * 16 / cols));
  const dim3 grid((unsigned)cols, (unsigned)std::min<int64_t>(rows, 65535));
  if (p.N % 8 == 0) GB_CUDA_OK(gb_launch(linear_sign_kernel<true>, grid, dim3(kDzThreads), 0, st, s));
  else GB_CUDA_OK(gb_launch(linear_sign_kernel<false>, grid, dim3(kDzThreads), 0, st, s));
  return GB_OK;
}

}  // namespace

extern "C" {

int gb_linear_act(const void* x, int64_t x_ld, const void* w, const void* bias, const void* r, int64_t r_ld, int dtype, int64_t M, int64_t N, int64_t K, int act,
                  void* y, void* z, void* stream) {
  int rc = check_shape(M, N, K, dtype);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(x && w && y, "null pointer argument");
  GB_REQUIRE(act >= GB_EPI_NONE && act <= GB_EPI_SILU, "unknown activation %d", act);
  GB_REQUIRE(aligned(x) && aligned(w) && aligned(y) && aligned(z) && x_ld >= K && x_ld % 8 == 0, "operands must be rows of whole 16-byte pieces");
  GB_REQUIRE(!r || r_ld >= N, "residual rows that do not overlap expected");
  GB_REQUIRE(!r || r != y || !z || act != GB_EPI_RELU, "a relu whose z is kept adds its residual twice: it lies elsewhere than the result");
  int pairs = 0;
  rc = ready(&pairs);
  if (rc != GB_OK) return rc;
  LinearParams p = params_of(M, N, dtype, y);
  p.act = act;
  p.bias = static_cast<const uint16_t*>(bias);
  p.r = static_cast<const uint16_t*>(r);
  p.r_ld = r_ld;
  p.z = static_cast<uint16_t*>(z);
  if (r && (!aligned(r) || r_ld % 8 != 0)) p.tma = 0;
  const Mats m = {x, w, x_ld, K, K};
  const cudaStream_t st = (cudaStream_t)stream;
  if (M <= kFewRows && M * N * K <= kFewProducts && M * K * 4 <= kFewSmem) return run_few(m, p, st);
  const int width = route_of(kWidths, M, N, K, pairs);
  if (width == 0) rc = run_rows<false>(m, p, st);
  else if (z) rc = r ? run_forward<kBoth>(width, m, p, pairs, st) : run_forward<kKeepZ>(width, m, p, pairs, st);
  else rc = r ? run_forward<kResidual>(width, m, p, pairs, st) : run_forward<kPlain>(width, m, p, pairs, st);
  return rc == GB_OK && z && act == GB_EPI_RELU ? run_signs(m, p, st) : rc;
}

int64_t gb_linear_act_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int act, int rows, int weight, int bias, int dy_whole) {
  int pairs = 0;
  return M < 1 || N < 1 || K < 1 || ready(&pairs) != GB_OK ? 0 : grad_plan(M, N, K, act, rows != 0, weight != 0, bias != 0, dy_whole != 0, pairs).bytes;
}

int gb_linear_act_grad(const void* dy, int64_t dy_ld, const void* z, const void* x, int64_t x_ld, const void* w, int dtype, int64_t M, int64_t N, int64_t K, int act,
                       void* dx, void* dw, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_shape(M, N, K, dtype);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(act >= GB_EPI_NONE && act <= GB_EPI_SILU, "unknown activation %d", act);
  GB_REQUIRE(dy && (act == GB_EPI_NONE || z) && (!dx || w) && (!dw || x), "null pointer argument");
  GB_REQUIRE(dy_ld >= N && (!dw || (x_ld >= K && x_ld % 8 == 0)), "rows that do not overlap expected");
  GB_REQUIRE(aligned(w) && aligned(x) && aligned(z) && aligned(dx) && aligned(dw), "operands must be rows of whole 16-byte pieces");
  int pairs = 0;
  rc = ready(&pairs);
  if (rc != GB_OK) return rc;
  const bool dy_whole = aligned(dy) && dy_ld % 8 == 0;
  const GradPlan g = grad_plan(M, N, K, act, dx != nullptr, dw != nullptr, dbias != nullptr, dy_whole, pairs);
  if (workspace_bytes < g.bytes || (g.bytes > 0 && !workspace))
    return gb_fail(GB_EWORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)g.bytes);
  GB_REQUIRE(aligned(workspace), "the workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const cudaStream_t st = (cudaStream_t)stream;
  const void* dz = dy;
  int64_t dz_ld = dy_ld;
  if (g.own_dz || dbias) {
    DzParams d = {};
    d.dy = static_cast<const uint16_t*>(dy);
    d.z = act == GB_EPI_NONE ? nullptr : static_cast<const uint16_t*>(z);
    d.dz = g.own_dz ? reinterpret_cast<uint16_t*>(ws + g.dz_at) : nullptr;
    d.M = M; d.N = N; d.dy_ld = dy_ld; d.dz_ld = g.dz_ld;
    d.fp16 = dtype == GB_DTYPE_FP16; d.act = act;
    d.part = dbias ? reinterpret_cast<float*>(ws + g.part_at) : nullptr;
    const dim3 grid((unsigned)ceil_div(N, kDzCols), (unsigned)g.part_rows);
    if (N % 8 == 0 && dy_whole) GB_CUDA_OK(gb_launch(linear_dz_kernel<true>, grid, dim3(kDzThreads), 0, st, d));
    else GB_CUDA_OK(gb_launch(linear_dz_kernel<false>, grid, dim3(kDzThreads), 0, st, d));
    if (g.own_dz) { dz = ws + g.dz_at; dz_ld = g.dz_ld; }
    if (dbias) {
      rc = gb_join_columns(d.part, g.part_rows, N, dbias, dtype, st);
      if (rc != GB_OK) return rc;
    }
  }
  if (dx) {                                                  // [M, K], the contraction over N
    const LinearParams p = params_of(M, K, dtype, dx);
    const Mats m = {dz, w, dz_ld, K, N};
    rc = g.rows_width == 0 ? run_rows<true>(m, p, st) : run_grad<kRowsGrad>(g.rows_width, m, p, pairs, st);
    if (rc != GB_OK) return rc;
  }
  if (dw) {                                                  // [N, K], the contraction over M
    LinearParams p = params_of(N, K, dtype, dw);
    const Mats m = {dz, x, dz_ld, x_ld, M};
    const int64_t k_tiles = ceil_div(M, kSlab);
    p.slices = (int)ceil_div(k_tiles, ceil_div(k_tiles, g.slices));      // none of them empty
    p.sums = reinterpret_cast<float*>(ws + g.sums_at);
    rc = run_grad<kWeightGrad>(g.width, m, p, pairs, st);
    if (rc == GB_OK && p.slices > 1) rc = run_join(p, st);
    if (rc != GB_OK) return rc;
  }
  return GB_OK;
}

}  // extern "C"
