// GEMMs of block-scaled E4M3: D[m, n] = sum over blocks b of 128 columns of
//     a_scale[m, b] * b_scale[n / 128, b] * sum over k in b of A[m, k] W[n, k],
// dense, or grouped over expert segments (rows seg[e] .. seg[e + 1] of A times expert e's weights).
//
// The scales differ from block to block, so a sum on the tensor cores goes over one block only (four instructions of
// kind::f8f6f4) and the blocks are added in fp32 registers: every block has an accumulator of its own in tensor memory, a ring
// of them, and the read-out warps turn each into one multiply-add per element while the next blocks are multiplied.
//
// Two kernels.  gemm_blocks_tile_kernel: activations on the M side, so that a thread holds one row and its scale is one number per
// block; tiles of 128 rows x 256 features on single CTAs (K sliced over a thread-block cluster where there are fewer tiles
// than SMs; grouped), or of 256 x 256 on CTA pairs (cta_group::2).  gemm_blocks_rows_kernel: few rows; the WEIGHTS are the M side
// (128 features a CTA, one scale per block for the whole tile), the rows the N side in steps of sixteen, K sliced alike.
//
// What bounds them.  Tiles: the tensor cores take 392 ns a slab of 256 x 256 x 128 with nothing to wait for (3.1 PFLOP/s); the
// multiply-adds of the read-out (two warps of a scheduler, 256 clocks of its 700 a slab) and the power cap leave 2.4 in a graph and 2.1 over seconds.  Rows: the
// bytes of the weights, up to some 64 rows; from there on the shared memory, through which every warp gets the rows' scales
// at 128 bytes a clock beside the operands.
#include "gb_blocks.cuh"
#include "gb_row_ring.cuh"

#include <cuda.h>
#include <atomic>
#include <mutex>

namespace {

constexpr int kSlab = 128;                           // columns of a block = bytes of K of a stage (one swizzle span)
constexpr int kBM = 128;                             // rows of an operand tile of a CTA on the M side
constexpr int kMaxGroups = 1024;                     // experts of one grouped launch
constexpr int kMaxSlices = 8;                        // of K, over a thread-block cluster
constexpr int kSegBytes = 2 * (kMaxGroups + 1) * 4 + 8;

struct BlocksParams {
  int64_t M, N;              // rows of A (grouped: all of them), features (grouped: of an expert)
  int kb, nb;                // blocks along K, along the features (of an expert)
  int m_tiles, n_tiles;
  const float* a_scale;      // [M][kb]
  const float* b_scale;      // [E][nb][kb]
  void* D;
  int out;                   // GB_DTYPE_*
  int vec4;                  // rows of both scales are whole aligned 16-byte pieces
  int out_tma, out16;        // 16-bit rows of D that TMA takes; rows of D are whole 16-byte pieces
  const int32_t* seg;        // [E + 1], or null
  int E;
  int most_row_tiles;        // grouped: of offsets that rise
  int beside;                // W, its scales and seg are not written by the launch ahead: read before it has finished
  uint32_t idesc;            // without M and N
  int* status;
  // rows kernel
  int rows_per_pass, passes, per_slice, slices, stages;
  int overlay, sums_at;      // sums of a sliced K lie over the ring, or that far behind its start
  int pitch;                 // rows of a slice's sums in a CTA
  // rows quantised by the kernel itself: M of them, ld elements apart
  const void* x;
  int64_t ld, K;
  int scale_rule;
};

// ---- waits, copies, MMAs -------------------------------------------------------------------------------------
// What a wait hands over: this CTA's writes or copies; those of either CTA of the pair; tensor memory alone, which the
// tcgen05 fences on both sides order, so that the wait itself may be relaxed (an acquire at cluster scope took 150 clocks
// with the barrier already complete).
enum Scope { kOfCta, kOfPair, kTensorMemory };
template <Scope kScope>
GB_DEVINL bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  if (kScope == kOfPair)
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  else if (kScope == kTensorMemory)
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// A bounded wait that remembers a timeout for the rest of the CTA: later waits return at once.
template <Scope kScope>
GB_DEVINL void wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  uint64_t t0 = 0;
  for (uint32_t spin = 0; !*abort_flag; ++spin) {
    if (try_wait<kScope>(bar, parity)) return;
    if ((spin & 255u) == 255u) {
      const uint64_t now = gb_globaltimer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > 2000000000ull) { *abort_flag = 1; atomicExch(status, code); }
    }
  }
}
// By a whole warp that goes on together; false: given up.
template <Scope kScope = kOfCta>
GB_DEVINL bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, try_wait<kScope>(bar, parity))) return true;
  wait_slow<kScope>(bar, parity, abort_flag, status, code);
  return !__any_sync(0xffffffffu, *abort_flag != 0);
}
GB_DEVINL int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
GB_DEVINL void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
GB_DEVINL void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
GB_DEVINL void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Hands tensor memory from read-out warps of both CTAs to the leader's MMA issuer: ordered by the tensor-memory fences on
// both sides, so the arrive itself may be relaxed (one that released would wait for the output stores in flight).
GB_DEVINL void arrive_cluster(uint32_t addr, bool mine) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %1, 0;\n@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n}\n" ::"r"(addr), "r"((uint32_t)mine) : "memory");
}
GB_DEVINL uint32_t leader_addr(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
GB_DEVINL void tma_load_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
GB_DEVINL void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
// K-major operand tile stored as rows of 128 bytes with the 128-byte swizzle.
GB_DEVINL uint64_t desc_sw128(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <int kGroup>
GB_DEVINL void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, bool accumulate) {
  if (kGroup == 2)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
template <int kGroup>
GB_DEVINL void commit_to(uint32_t bar) {
  if (kGroup == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// To the barrier of every CTA that works on the tile.
template <int kCtas>
GB_DEVINL void commit_all(uint32_t bar, uint32_t to_peer) {
  commit_to<kCtas>(bar);
  if (kCtas == 2) commit_to<2>(bar + to_peer);
}
template <int kCtas>
GB_DEVINL void tmem_alloc(uint32_t slot, uint32_t cols) {
  if (kCtas == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
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
template <int kRegs>
GB_DEVINL void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
GB_DEVINL void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
// The loads issued so far have arrived; `v`, loaded by them, is read behind this only.
GB_DEVINL void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]),
                 "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31]) ::"memory");
}
GB_DEVINL void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
GB_DEVINL void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
GB_DEVINL void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Scales of four consecutive blocks, kt .. kt + 3, of a row of `kb`; zeros past its end and for a null row.  The loads are
// volatile so that they stay where they are issued, four blocks ahead: free to move, they were sunk to their use, and every
// fourth block waited some 1900 clocks for them (333 rows of 5120 x 17408: 78 us, 65 with them in flight).
GB_DEVINL float load1(const float* at) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(at));
  return v;
}
GB_DEVINL float4 scales4(const float* row, int kt, int kb, bool vec4) {
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (row == nullptr) return v;
  if (vec4 && (kt & 3) == 0) {                             // kb is a multiple of four
    asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(row + kt));
    return v;
  }
  if (kt < kb) v.x = load1(row + kt);
  if (kt + 1 < kb) v.y = load1(row + kt + 1);
  if (kt + 2 < kb) v.z = load1(row + kt + 2);
  if (kt + 3 < kb) v.w = load1(row + kt + 3);
  return v;
}
GB_DEVINL float pick(const float4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

GB_DEVINL uint32_t pack2(float a, float b, int out) {
  if (out == GB_DTYPE_BF16) return gb_pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
GB_DEVINL void store1(void* D, int64_t at, float v, int out) {
  if (out == GB_DTYPE_FP32) static_cast<float*>(D)[at] = v;
  else if (out == GB_DTYPE_BF16) static_cast<uint16_t*>(D)[at] = (uint16_t)gb_f32_to_bf16_bits(v);
  else static_cast<uint16_t*>(D)[at] = __half_as_ushort(__float2half_rn(v));
}

// 32 rows of 64 bytes, the first `cols` columns of which count, from a warp's 2 KB of shared memory (64-byte swizzle) to D from
// (row0, f0) on: lanes along the columns, in pieces as large as rows of D allow.  (A row a lane, as the sums lie in the registers, 7098 rows
// of 7834 x 512 took 572 us for 76, 32768 of 128 experts of 1534 x 2048 659 for 167.)
GB_DEVINL void store_chunk(const BlocksParams& p, uint32_t chunk, int row0, int rows, int f0, int cols) {
  const int lane = threadIdx.x & 31, bytes = p.out == GB_DTYPE_FP32 ? 4 : 2;
  uint8_t* D = static_cast<uint8_t*>(p.D) + ((int64_t)row0 * p.N + f0) * bytes;
  const int64_t pitch = p.N * bytes;
  if (p.out16) {
    const int q = lane & 3;
#pragma unroll 1
    for (int r = lane >> 2; r < rows; r += 8) {
      uint4 v;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(chunk + (uint32_t)(r * 64 + (q ^ ((r >> 1) & 3)) * 16)) : "memory");
      if (q * 16 < cols * bytes) *reinterpret_cast<uint4*>(D + r * pitch + q * 16) = v;
    }
  } else if (bytes == 4 || p.N % 2 == 0) {
    const int w = lane & 15;
#pragma unroll 1
    for (int r = lane >> 4; r < rows; r += 2) {
      uint32_t v;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(chunk + (uint32_t)(r * 64 + ((w >> 2) ^ ((r >> 1) & 3)) * 16 + (w & 3) * 4)) : "memory");
      if (w * 4 < cols * bytes) *reinterpret_cast<uint32_t*>(D + r * pitch + w * 4) = v;
    }
  } else {
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(chunk + (uint32_t)(r * 64 + ((lane >> 3) ^ ((r >> 1) & 3)) * 16 + (lane & 7) * 2)) : "memory");
      if (lane < cols) *reinterpret_cast<uint16_t*>(D + r * pitch + lane * 2) = v;
    }
  }
}
// A lane's row of such a chunk: piece q of its four.
GB_DEVINL void stage_piece(uint32_t chunk, int q, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const int lane = threadIdx.x & 31;
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(chunk + (uint32_t)(lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16))), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Segment starts and the number of row tiles in front of each expert, into shared memory, by one warp: a lane takes consecutive
// experts, so that their loads are in flight together.  Offsets that fall and rise again make segments that overlap and more tiles: a lane's
// stop at kManyTiles, which rising offsets never have, so that the sum fits, and row_tiles takes no more than those can have.
constexpr int kManyTiles = 1 << 25;
GB_DEVINL void load_segments(const BlocksParams& p, int tile_rows, int* seg_s, int* base_s) {
  const int lane = threadIdx.x & 31, per = (p.E + 31) / 32, e0 = lane * per, e1 = min(p.E, e0 + per);
  int tiles = 0;
#pragma unroll 8
  for (int e = e0; e < e1; ++e) {
    // within the rows there are, whatever the offsets say
    const int lo = min(max(p.seg[e], 0), (int)p.M), hi = min(max(p.seg[e + 1], lo), (int)p.M);
    seg_s[e] = lo;
    base_s[e] = tiles;
    tiles += (hi - lo + tile_rows - 1) / tile_rows;        // below 2^28: 32 experts of fewer than 2^30 rows in tiles of 128, or of a few rows in smaller ones
    if (e == p.E - 1) seg_s[p.E] = hi;
  }
  tiles = min(tiles, kManyTiles);
  int incl = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  for (int e = e0; e < e1; ++e) base_s[e] += incl - tiles;
  if (lane == 31) base_s[p.E] = incl;
}
GB_DEVINL int row_tiles(const BlocksParams& p, const int* base_s) { return min(base_s[p.E], p.most_row_tiles); }

// The expert whose row tiles hold tile `gp`: e or a later one; those without rows are stepped over, 32 at a time.  By a whole warp. (One
// at a time, a load from shared memory each: 12.4 us instead of 10.0 for one token of eight of 128 experts, 39 instead of 12.4 of 1024.)
GB_DEVINL int expert_of(const int* base_s, int E, int gp, int e) {
  if (base_s[e + 1] > gp) return e;
  for (int at = e + 1; at < E; at += 32) {
    const int i = at + (int)(threadIdx.x & 31);
    const unsigned past = __ballot_sync(0xffffffffu, i >= E || base_s[i + 1] > gp);
    if (past) return min(at + __ffs(past) - 1, E - 1);
  }
  return E - 1;
}

// ======================================== CTA pairs, and single CTAs ========================================================
constexpr int kEpiWarps = 8;                         // two per lane quarter, half of the columns each
constexpr int kOutChunk = 2048;                      // 32 rows x 32 16-bit columns on their way out
constexpr int kPairThreads = 32 * (kEpiWarps + 4);     // three warpgroups, the last two warps idle
// A thread of the read-out holds 128 sums and has 64 more on their way; 168 registers a thread at launch.
// (What spills is a scale on its way, and the wait for it: 333 rows of 5120 x 17408 in single CTAs 45 us with 224 of them.)
template <int kCtas>
struct Registers {
  static constexpr int kRead = kCtas == 2 ? 224 : 232, kOther = kCtas == 2 ? 56 : 40;
  static_assert(256 * kRead + 128 * kOther <= 384 * 168, "a register split draws on what the block was launched with");
};
constexpr int kTmemCols = 512;
constexpr int kBN = 256, kPart = 128, kParts = 2;    // features of a tile, of a part: one block of features, an accumulator
constexpr int kAccs = kTmemCols / kPart;
constexpr int kGroupM = 16;                          // row tiles walked together before the next columns (see gb_gemm_pair.cu)

template <int kCtas, bool kGrouped>
struct Tile {
  static constexpr int kM = kBM * kCtas;               // rows of a tile
  static constexpr int kABytes = kBM * kSlab, kBBytes = kBN / kCtas * kSlab, kStageBytes = kABytes + kBBytes;
  static constexpr int kChunks = kGrouped ? 1 : 2;     // on their way out, of a warp
  static constexpr int kOutBytes = kEpiWarps * kChunks * kOutChunk + (kGrouped ? kSegBytes : 0);
  // an even number: each of the two MMA issuers meets every phase of the stages that it waits for
  static constexpr int kStages = (227 * 1024 - 2048 - kOutBytes) / kStageBytes / 2 * 2;
  static constexpr int kSmem = kStages * kStageBytes + kOutBytes + 2048;
  static_assert(kStages >= 4, "the sums of a sliced K lie over four stages");
};

// The tiles of a pair or CTA: first, first + stride, ...
template <int kM, bool kGrouped>
struct TileWalk {
  int tile, stride, e = 0;
  int m0 = 0, n0 = 0, w0 = 0, end = 0;               // first row, first feature, first weight row, end of the rows that count
  GB_DEVINL TileWalk(int first, int stride_) : tile(first - stride_), stride(stride_) {}
  GB_DEVINL bool next(const BlocksParams& p, int total, const int* seg_s, const int* base_s) {
    tile += stride;
    if (tile >= total) return false;
    if (kGrouped) {                                  // features fastest: a row tile's columns run together
      const int gp = tile / p.n_tiles, nt = tile - gp * p.n_tiles;
      e = expert_of(base_s, p.E, gp, e);
      m0 = seg_s[e] + (gp - base_s[e]) * kM;
      end = seg_s[e + 1];
      n0 = nt * kBN;
      w0 = e * (int)p.N + n0;
    } else {
      const int per = kGroupM * p.n_tiles, g = tile / per, in = tile - g * per;
      const int rows = min(kGroupM, p.m_tiles - g * kGroupM);
      m0 = (g * kGroupM + in % rows) * kM;
      n0 = in / rows * kBN;
      w0 = n0;
      end = (int)p.M;
    }
    return true;
  }
};

// fmaf, kept where it stands between the loads and the waits.
GB_DEVINL void add_scaled(float& acc, uint32_t v, float scale) {
  asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(acc) : "f"(__uint_as_float(v)), "f"(scale));
}
GB_DEVINL void read64(uint32_t at, uint32_t (&v)[2][32]) {
  tmem_ld32(at, v[0]);
  tmem_ld32(at + 32u, v[1]);
  tmem_wait_ld(v[0]);
  tmem_wait_ld(v[1]);
}

template <int kCtas, bool kGrouped>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_blocks_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_d,
                        const __grid_constant__ BlocksParams p) {
  using S = Tile<kCtas, kGrouped>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (gb_smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in both CTAs
  uint8_t* ring_ptr = smem_raw + (ring - gb_smem_u32(smem_raw));
  const uint32_t out_ring = ring + kStages * S::kStageBytes;             // one or two chunks per read-out warp
  const uint32_t full_bar = out_ring + (S::kOutBytes + 7) / 8 * 8;       // leader: both CTAs' operand tiles have landed
  const uint32_t empty_bar = full_bar + 8 * kStages;                     // the MMAs that read the stage are done
  const uint32_t acc_full = empty_bar + 8 * kStages;                     // [kAccs] a block's sums are complete
  const uint32_t acc_empty = acc_full + 8 * kAccs;                       // [kAccs] leader: read out by both CTAs
  const uint32_t slot = acc_empty + 8 * kAccs;
  volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(ring_ptr + (slot - ring));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot_ptr + 1);
  int* seg_s = reinterpret_cast<int*>(ring_ptr + (out_ring - ring) + kEpiWarps * S::kChunks * kOutChunk);
  int* base_s = seg_s + kMaxGroups + 1;

  const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  uint32_t rank = 0;                                       // of the pair
  if constexpr (kCtas == 2) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  gb_pdl_launch_dependents();
  {                                                        // a barrier of each kind per thread
    const uint32_t i = threadIdx.x;
    if (i < kStages) {
      bar_init(full_bar + 8 * i, 1);
      bar_init(empty_bar + 8 * i, 1);
    }
    if (i < kAccs) {
      bar_init(acc_full + 8 * i, 1);
      bar_init(acc_empty + 8 * i, 4 * kCtas);
    }
    if (i == 0) *abort_flag = 0;
    gb_fence_barrier_init();
  }
  if (warp == kEpiWarps + 1) tmem_alloc<kCtas>(slot, kTmemCols);
  gb_pdl_wait();
  if (kGrouped && warp == kEpiWarps) load_segments(p, S::kM, seg_s, base_s);
  tmem_fence_before();
  __syncthreads();
  if constexpr (kCtas == 2) gb_cluster_sync();                           // both CTAs' barriers exist
  tmem_fence_after();
  const uint32_t tmem_base = *slot_ptr;
  const int total = kGrouped ? row_tiles(p, base_s) * p.n_tiles : p.m_tiles * p.n_tiles;
  const int stride = (int)gridDim.x / kCtas, first = (int)blockIdx.x / kCtas;
  // K slices, of single CTAs: a tile for every cluster along y
  const int slice = kCtas == 1 ? (int)blockIdx.y : 0, k_begin = kCtas == 1 ? slice * p.per_slice : 0;
  const int k_end = kCtas == 1 ? min(p.kb, k_begin + p.per_slice) : p.kb;

  if (warp == kEpiWarps) {
    // ------------------------------- producer (each CTA) -------------------------------
    fewer_registers<Registers<kCtas>::kOther>();
    const uint32_t full_pair = kCtas == 2 ? (uint32_t)uniform((int)leader_addr(full_bar)) : full_bar;
    const int me = uniform((int)rank);
    const bool one = gb_elect_one();
    int s = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (TileWalk<S::kM, kGrouped> T(first, stride); ok && T.next(p, total, seg_s, base_s);) {
      const int m0 = uniform(T.m0) + me * kBM, w0 = uniform(T.w0) + me * (kPart / 2);
      for (int kt = k_begin; kt < k_end; ++kt) {
        ok = warp_wait<kTensorMemory>(empty_bar + 8 * s, ph, abort_flag, p.status, 91);
        if (!ok) break;
        if (one) {
          const uint32_t st = ring + (uint32_t)s * S::kStageBytes;
          if (me == 0) expect_tx(full_bar + 8 * s, kCtas * S::kStageBytes);
          if constexpr (kCtas == 2) {
            tma_load_pair(st, &map_a, kt * kSlab, m0, full_pair + 8 * s);
            tma_load_pair(st + S::kABytes, &map_b, kt * kSlab, w0, full_pair + 8 * s);                            // half of a part's
            tma_load_pair(st + S::kABytes + S::kBBytes / 2, &map_b, kt * kSlab, w0 + kPart, full_pair + 8 * s);    // features each
          } else {
            tma_load_2d(st, &map_a, kt * kSlab, m0, full_pair + 8 * s);
            tma_load_2d(st + S::kABytes, &map_b, kt * kSlab, w0, full_pair + 8 * s);
            tma_load_2d(st + S::kABytes + S::kBBytes / 2, &map_b, kt * kSlab, w0 + kPart, full_pair + 8 * s);
          }
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == kEpiWarps + 1 || warp == kEpiWarps + 2) {
    // ------ MMA issuers (the leader's): the waits, MMAs and commits of a slab take one some 700 clocks, so two share the slabs
    // in turn; every slab has accumulators of its own, so that their order does not matter ------
    fewer_registers<Registers<kCtas>::kOther>();
    if (uniform((int)rank) == 0) {
      uint32_t to_peer = 0;                                  // distance of the peer's barriers
      if constexpr (kCtas == 2) {
        asm volatile("mapa.shared::cluster.u32 %0, %1, 1;" : "=r"(to_peer) : "r"(full_bar));
        to_peer = (uint32_t)uniform((int)(to_peer - full_bar));
      }
      const uint32_t tmem = (uint32_t)uniform((int)tmem_base);
      const int tiles = uniform(total > first ? (total - first + stride - 1) / stride : 0), turn = warp - kEpiWarps - 1;
      const int64_t slabs = (int64_t)tiles * (k_end - k_begin);
      const bool one = gb_elect_one();
      int s = turn % kStages;
      uint32_t ph = turn >= kStages ? 1 : 0, acc_ph = 1;
      bool ok = true;
      for (int64_t slab = turn; ok && slab < slabs; slab += 2) {
        ok = warp_wait(full_bar + 8 * s, ph, abort_flag, p.status, 93);
        if (!ok) break;
        const uint32_t st = ring + (uint32_t)s * S::kStageBytes;
        const uint64_t da = desc_sw128(st);
        // A pair's halves of the features are multiplied one after the other, so that each is read out while the other is at work (in one
        // instruction of 256 columns 8192 rows of 34816 x 5120 took 1455 us for 1424).  A single CTA, which reads all features itself, takes both at once and
        // A's rows from shared memory once: the same time, and with less power (333 rows of 5120 x 17408 over seconds 48.2 -> 46.2).
        constexpr int kAtOnce = kCtas == 1 ? kParts : 1;
#pragma unroll
        for (int h = 0; h < kParts; h += kAtOnce) {
          const int buf = turn * kParts + h;
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) ok = ok && warp_wait<kTensorMemory>(acc_empty + 8 * (buf + i), acc_ph, abort_flag, p.status, 92);
          if (!ok) break;
          tmem_fence_after();
          const uint64_t db = desc_sw128(st + S::kABytes + (uint32_t)h * (S::kBBytes / 2));
          if (one) {
#pragma unroll
            for (int k = 0; k < 4; ++k)                      // 32 columns of K per instruction
              mma<kCtas>(tmem + (uint32_t)(buf * kPart), da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), p.idesc, k > 0);
            commit_all<kCtas>(acc_full + 8 * buf, to_peer);
            if (h + kAtOnce == kParts) commit_all<kCtas>(empty_bar + 8 * s, to_peer);
          }
          __syncwarp();
        }
        acc_ph ^= 1;
        s += 2;
        if (s >= kStages) { s -= kStages; ph ^= 1; }
      }
    }
  } else if (warp < kEpiWarps) {
    // ------------------------------- read-out (each CTA) --------------------------------
    more_registers<Registers<kCtas>::kRead>();
    const uint32_t acc_empty_pair = kCtas == 2 ? leader_addr(acc_empty) : acc_empty;
    // Four warps for each part, one per lane quarter: while one of a scheduler's two adds, the other waits or loads.  (All
    // eight on half of every part wait together and then add together.)
    constexpr int kOuts = kPart / 32;
    const int quarter = warp & 3, part = warp >> 2, c_lo = part * kPart;
    const uint32_t out = out_ring + (uint32_t)warp * S::kChunks * kOutChunk;
    const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16);
    int buf = part, flip = 0;
    uint32_t ph = 0;
    bool ok = true;
    TileWalk<S::kM, kGrouped> T(first, stride);
    const float *as = nullptr, *bs = nullptr;
    float4 as4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), bs4 = as4;
    auto begin = [&] {                                       // a tile's scales, the first four blocks' on their way
      const int row = T.m0 + (int)rank * kBM + quarter * 32 + lane;
      as = row < T.end ? p.a_scale + (int64_t)row * p.kb : nullptr;
      // a part is one block of features; one past the last is not stored
      bs = p.b_scale + ((int64_t)(kGrouped ? T.e : 0) * p.nb + min((T.n0 + c_lo) / kSlab, p.nb - 1)) * p.kb;
      as4 = scales4(as, k_begin, p.kb, p.vec4);
      bs4 = scales4(bs, k_begin, p.kb, p.vec4);
    };
    bool more = T.next(p, total, seg_s, base_s);
    if (more) begin();
    while (ok && more) {
      const int row0 = T.m0 + (int)rank * kBM + quarter * 32, row = row0 + lane, n0 = T.n0 + c_lo, end = T.end;
      const bool row_ok = row < end;
      float acc[kPart];
#pragma unroll
      for (int c = 0; c < kPart; ++c) acc[c] = 0.0f;
      for (int kt0 = k_begin; ok && kt0 < k_end; kt0 += 4) {
        const float4 sc = make_float4(as4.x * bs4.x, as4.y * bs4.y, as4.z * bs4.z, as4.w * bs4.w);
        if (kt0 + 4 < k_end) {                               // the next four blocks' while these are added
          as4 = scales4(as, kt0 + 4, p.kb, p.vec4);
          bs4 = scales4(bs, kt0 + 4, p.kb, p.vec4);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!ok || kt0 + j >= k_end) break;
          const float scale = pick(sc, j);
          ok = warp_wait<kTensorMemory>(acc_full + 8 * (kCtas == 1 ? buf - part : buf), ph, abort_flag, p.status, 94);
          if (!ok) break;
          tmem_fence_after();
          uint32_t v[2][32];
          read64(at + (uint32_t)(buf * kPart), v);
#pragma unroll
          for (int c = 0; c < 64; ++c) add_scaled(acc[c], v[c >> 5][c & 31], scale);
          read64(at + (uint32_t)(buf * kPart + 64), v);
          tmem_fence_before();
          __syncwarp();
          if constexpr (kCtas == 2) arrive_cluster(acc_empty_pair + 8 * buf, lane == 0);
          else if (lane == 0) arrive(acc_empty_pair + 8 * buf);
          buf += kParts;
          if (buf >= kAccs) { buf -= kAccs; ph ^= 1; }
#pragma unroll
          for (int c = 0; c < 64; ++c) add_scaled(acc[64 + c], v[c >> 5][c & 31], scale);
        }
      }
      if constexpr (kCtas == 1 && !kGrouped) {
        if (p.slices > 1) {
          // Every CTA of the cluster has finished its MMAs, and with them its loads: the sums go into the shared memory of the CTA
          // that owns the features, [slice][own feature][row], over the ring, and it adds them in the order of K.
          asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
          const bool live = !*abort_flag;
          const int own = (16 + p.slices - 1) / p.slices, r = quarter * 32 + lane;       // sixteens of features
          gb_cluster_sync();
          if (live) {
#pragma unroll
            for (int i = 0; i < kPart / 16; ++i) {
              const int c0 = part * (kPart / 16) + i, to = c0 / own;
              uint32_t dst;
              asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                           : "=r"(dst) : "r"(ring + (uint32_t)((slice * own + c0 - to * own) * 16 * kBM + r) * 4u), "r"(to));
#pragma unroll
              for (int c = 0; c < 16; ++c)
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + (uint32_t)c * kBM * 4u), "f"(acc[16 * i + c]) : "memory");
            }
          }
          gb_cluster_sync();                                 // the last access to another CTA's memory lies in front of it
          if (live) {
            for (int i = part; i < own && slice * own + i < 16; i += 2) {
              float sum[16] = {};
              for (int q = 0; q < p.slices; ++q) {
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                  float v;
                  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(ring + (uint32_t)(((q * own + i) * 16 + c) * kBM + r) * 4u) : "memory");
                  sum[c] += v;
                }
              }
              const int f = T.n0 + (slice * own + i) * 16;
              const int64_t d = (int64_t)row * p.N + f;
              if (f >= p.N) continue;
              if (p.out16 && p.out != GB_DTYPE_FP32) {
#pragma unroll
                for (int c = 0; c < 16; c += 8)
                  if (row_ok && f + c < p.N)
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.D) + d + c) =
                        make_uint4(pack2(sum[c], sum[c + 1], p.out), pack2(sum[c + 2], sum[c + 3], p.out), pack2(sum[c + 4], sum[c + 5], p.out),
                                   pack2(sum[c + 6], sum[c + 7], p.out));
              } else {
                __syncwarp();                                // the last chunk has left
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  if (p.out == GB_DTYPE_FP32)
                    stage_piece(out, q, __float_as_uint(sum[4 * q]), __float_as_uint(sum[4 * q + 1]), __float_as_uint(sum[4 * q + 2]), __float_as_uint(sum[4 * q + 3]));
                  else if (q < 2)
                    stage_piece(out, q, pack2(sum[8 * q], sum[8 * q + 1], p.out), pack2(sum[8 * q + 2], sum[8 * q + 3], p.out),
                                pack2(sum[8 * q + 4], sum[8 * q + 5], p.out), pack2(sum[8 * q + 6], sum[8 * q + 7], p.out));
                }
                __syncwarp();
                store_chunk(p, out, row0, min(32, end - row0), f, (int)min((int64_t)16, p.N - f));
              }
            }
          }
          break;                                             // one tile a cluster
        }
      }
      if (!ok) break;
      more = T.next(p, total, seg_s, base_s);
      if (more) begin();                                     // while this tile is stored
      if (p.out_tma && (!kGrouped || row0 + 32 <= end)) {  // dense: what sticks out is not written
#pragma unroll
        for (int c = 0; c < kOuts; ++c) {
          const uint32_t dst = out + (uint32_t)flip * kOutChunk;
          if (S::kChunks == 2) flip ^= 1;
          asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(S::kChunks - 1) : "memory");     // the buffer's last chunk has left it
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {                      // 64-byte swizzle: eight rows touch eight bank groups
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack2(acc[32 * c + 8 * q + 2 * i], acc[32 * c + 8 * q + 2 * i + 1], p.out);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(dst + (uint32_t)lane * 64u + (uint32_t)((q ^ ((lane >> 1) & 3)) * 16)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && row0 < end && n0 + 32 * c < p.N)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                         ::"l"(reinterpret_cast<uint64_t>(&map_d)), "r"(n0 + 32 * c), "r"(row0), "r"(dst) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else if (row0 < end) {
        const int rows = min(32, end - row0), cols = (int)min((int64_t)kPart, p.N - n0);
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");       // an earlier tile's chunks have left
        if (p.out == GB_DTYPE_FP32) {
#pragma unroll
          for (int c = 0; c < kPart / 16; ++c) {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q)
              stage_piece(out, q, __float_as_uint(acc[16 * c + 4 * q]), __float_as_uint(acc[16 * c + 4 * q + 1]), __float_as_uint(acc[16 * c + 4 * q + 2]),
                          __float_as_uint(acc[16 * c + 4 * q + 3]));
            __syncwarp();
            store_chunk(p, out, row0, rows, n0 + 16 * c, min(16, cols - 16 * c));
          }
        } else {
#pragma unroll
          for (int c = 0; c < kOuts; ++c) {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float* v = acc + 32 * c + 8 * q;
              stage_piece(out, q, pack2(v[0], v[1], p.out), pack2(v[2], v[3], p.out), pack2(v[4], v[5], p.out), pack2(v[6], v[7], p.out));
            }
            __syncwarp();
            store_chunk(p, out, row0, rows, n0 + 32 * c, min(32, cols - 32 * c));
          }
        }
        __syncwarp();
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
    fewer_registers<Registers<kCtas>::kOther>();
  }
  if (kCtas == 1 && !kGrouped && p.slices > 1 && warp >= kEpiWarps) {       // the read-out's meetings with the other slices
    gb_cluster_sync();
    gb_cluster_sync();
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (*abort_flag) __nanosleep(1000000);                   // loads and MMAs still in flight end before the memory goes
  if constexpr (kCtas == 2) gb_cluster_sync();             // the peer may still signal barriers here
  if (warp == kEpiWarps + 1) {
    if constexpr (kCtas == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kTmemCols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kTmemCols) : "memory");
  }
}

// ======================================== few rows =========================================================
constexpr int kMaxStages = 12;
constexpr int kFewStages = 8;                        // of CTAs with one tile and up to sixteen rows
static_assert(kFewStages % 2 == 0 && gb_row_ring::kStages % 2 == 0, "each of the two MMA issuers meets every phase of its stages");
constexpr int kScaleSlots = 4;                       // groups of four blocks whose scales are there ahead of their sums
constexpr int kQuantWarps = 4, kQuantMaxRows = 4, kScaleRing = 32;    // rows quantised here: warps that do, most rows, blocks whose scales are kept
static_assert(gb_row_ring::kSlabsAStep * kQuantMaxRows <= 4 * kQuantWarps, "a group of eight lanes for each block of a step");
static_assert(kScaleRing >= gb_row_ring::kStages + 8 + 4, "see the read-out: stages and accumulators, and some");

// In: the type of rows that the kernel quantises itself, or void: A is E4M3 with its scales.
template <int kR, typename In = void>
struct Rows {
  static constexpr bool kQuantize = !std::is_void<In>::value;
  static constexpr int kRead = kR == 16 ? 4 : 8;     // read-out warps: two per lane quarter where there are columns for both
  static constexpr int kThreads = 32 * (kRead + 3 + (kQuantize ? kQuantWarps : 1));
  static constexpr int kBox = kR < 32 ? kR : 32;     // rows of a copy of A
  static constexpr int kMine = kR / 16 / (kRead / 4);          // chunks of sixteen columns of a warp
  static constexpr int kAccs = kR <= 64 ? 8 : 512 / kR;
  static constexpr uint32_t kTmem = kAccs * kR < 32 ? 32 : kAccs * kR;
  static constexpr int kStageBytes = kBM * kSlab + kR * kSlab;
};
constexpr int kSmemMax = 217 * 1024;                 // with the static arrays within the 227 KB of a CTA

template <int kR, bool kGrouped, typename In>
__global__ void __launch_bounds__(Rows<kR, In>::kThreads, 1)
gemm_blocks_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ BlocksParams p) {
  using S = Rows<kR, In>;
  constexpr bool kQuantize = S::kQuantize;
  constexpr int kScaleBars = kQuantize ? kScaleRing : kScaleSlots, kScaleRows = kQuantize ? kScaleRing : 4 * kScaleSlots;
  constexpr int kRead = S::kRead, kAccs = S::kAccs, kMine = S::kMine;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_s[kMaxStages], empty_s[kMaxStages], acc_full_s[kAccs], acc_empty_s[kAccs], sc_full_s[kScaleBars], sc_empty_s[kScaleSlots];
  __shared__ __align__(16) uint8_t out_s[kRead * 1024];
  __shared__ uint32_t slot_s;
  __shared__ volatile int abort_s;
  const uint32_t ring = (gb_smem_u32(smem_raw) + 1023u) & ~1023u;        // the same offset in every CTA of a cluster
  uint8_t* ring_ptr = smem_raw + (ring - gb_smem_u32(smem_raw));
  float* scale_s = reinterpret_cast<float*>(ring_ptr + p.stages * S::kStageBytes);      // [slot][4][kR], or [block % kScaleRing][kR]
  int* seg_s = reinterpret_cast<int*>(scale_s + kScaleRows * kR);
  int* base_s = seg_s + kMaxGroups + 1;
  const uint32_t full_bar = gb_smem_u32(full_s), empty_bar = gb_smem_u32(empty_s), acc_full = gb_smem_u32(acc_full_s),
                 acc_empty = gb_smem_u32(acc_empty_s), sc_full = gb_smem_u32(sc_full_s), sc_empty = gb_smem_u32(sc_empty_s);

  const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  gb_pdl_launch_dependents();
  {                                                        // a barrier of each kind per thread: one thread took 600 clocks
    const int i = (int)threadIdx.x;
    if (i < p.stages) {
      gb_mbar_init(&full_s[i], kQuantize ? 1 + (uint32_t)p.M : 1);       // and every row's block
      gb_mbar_init(&empty_s[i], 1);
    }
    if (i < kAccs) {
      gb_mbar_init(&acc_full_s[i], 1);
      gb_mbar_init(&acc_empty_s[i], kRead);
    }
    if (i < kScaleBars) gb_mbar_init(&sc_full_s[i], kQuantize ? (uint32_t)p.M : 1);
    if (i < kScaleSlots) gb_mbar_init(&sc_empty_s[i], kRead);
    if (i == 0) abort_s = 0;
    gb_fence_barrier_init();
  }
  if (warp == kRead + 1) {
    tmem_alloc<1>(gb_smem_u32(&slot_s), S::kTmem);
  }
  // the sums of a sliced K have a place of their own: that the others have started is all that a CTA has to know, by the end
  if (p.slices > 1 && !p.overlay) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  if (!p.beside) gb_pdl_wait();
  if (kGrouped && warp == kRead) load_segments(p, kR, seg_s, base_s);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = (uint32_t)uniform((int)slot_s);
  // sliced: one item per cluster; otherwise the CTA walks items
  const int total = kGrouped ? row_tiles(p, base_s) * p.n_tiles : p.passes * p.n_tiles;
  const int slice = (int)blockIdx.y, k_begin = slice * p.per_slice, k_end = min(p.kb, k_begin + p.per_slice), k_n = k_end - k_begin;
  const int first = (int)blockIdx.x, stride = (int)gridDim.x;

  // What an item is: rows [m0, m0 + rows) of A, features [n0, n0 + 128), weight row of the first.
  struct Item { int m0, rows, n0, w0, e; };
  auto item_at = [&](int item, int e) {
    Item t;
    if (kGrouped) {
      const int gp = item / p.n_tiles;
      e = expert_of(base_s, p.E, gp, e);
      t.m0 = seg_s[e] + (gp - base_s[e]) * kR;
      t.rows = min(kR, seg_s[e + 1] - t.m0);
      t.n0 = (item - gp * p.n_tiles) * kBM;
      t.e = e;
      t.w0 = e * (int)p.N + t.n0;
    } else {
      const int tile = item / p.passes, pass = item - tile * p.passes;
      t.m0 = pass * p.rows_per_pass;
      t.rows = (int)min((int64_t)p.rows_per_pass, p.M - t.m0);
      t.n0 = t.w0 = tile * kBM;
      t.e = 0;
    }
    return t;
  };

  float acc[kMine][16];
  Item last{};
  if (warp == kRead) {
    // ------------------------------- producer -----------------------------------
    const bool one = gb_elect_one();
    int s = 0, e = 0;
    uint32_t ph = 1;
    bool ok = true, waited = !p.beside;
    for (int item = first; ok && item < total; item += stride) {
      const Item t = item_at(item, e);
      e = t.e;
      const int m0 = uniform(t.m0), w0 = uniform(t.w0), boxes = kQuantize ? 0 : (uniform(t.rows) + S::kBox - 1) / S::kBox;
      const uint32_t bytes = kBM * kSlab + (uint32_t)boxes * (S::kBox * kSlab);
      int ahead = 0;                                       // slabs whose weights are on their way already
      if (!waited) {
        // the launch ahead still writes the rows: the weights of the first stages need not wait for it
        for (; ok && ahead < min(p.stages, k_n); ++ahead) {
          ok = warp_wait(empty_bar + 8 * ahead, 1, &abort_s, p.status, 95);
          if (ok && one) {
            expect_tx(full_bar + 8 * ahead, bytes);
            tma_load_2d(ring + (uint32_t)ahead * S::kStageBytes, &map_w, (k_begin + ahead) * kSlab, w0, full_bar + 8 * ahead);
          }
          __syncwarp();
        }
        gb_pdl_wait();
        waited = true;
      }
      for (int kt = 0; ok && kt < k_n; ++kt) {
        if (kt >= ahead) ok = warp_wait(empty_bar + 8 * s, ph, &abort_s, p.status, 95);
        if (!ok) break;
        if (one) {
          const uint32_t st = ring + (uint32_t)s * S::kStageBytes, bar = full_bar + 8 * s;
          if (kt >= ahead) {
            expect_tx(bar, bytes);
            tma_load_2d(st, &map_w, (k_begin + kt) * kSlab, w0, bar);
          }
          for (int i = 0; i < boxes; ++i)
            tma_load_2d(st + kBM * kSlab + (uint32_t)i * (S::kBox * kSlab), &map_x, (k_begin + kt) * kSlab, m0 + i * S::kBox, bar);
        }
        __syncwarp();
        if (++s == p.stages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == kRead + 1 || warp == kRead + 2) {
    // ------ MMA issuers: the waits, MMAs and commits of a slab take one some 450 clocks, so two share the slabs in turn; every
    // slab has an accumulator of its own.  Stages and accumulators are even in number: each issuer meets all phases of its ones. ------
    const bool one = gb_elect_one();
    const int mine = warp - kRead - 1;
    int s = mine, buf = mine, e = 0, kt = mine;
    uint32_t ph = 0, acc_ph = 1;
    bool ok = true;
    for (int item = first; ok && item < total; item += stride, kt -= k_n) {
      const Item t = item_at(item, e);
      e = t.e;
      const uint32_t idesc = p.idesc | (uint32_t)((uniform(t.rows) + 15) / 16 * 2) << 17 | (uint32_t)(kBM >> 4) << 24;
      for (; kt < k_n; kt += 2) {
        ok = warp_wait<kTensorMemory>(acc_empty + 8 * buf, acc_ph, &abort_s, p.status, 96);
        if (!ok) break;
        ok = warp_wait(full_bar + 8 * s, ph, &abort_s, p.status, 97);
        if (!ok) break;
        tmem_fence_after();
        if (one) {
          const uint32_t st = ring + (uint32_t)s * S::kStageBytes;
          const uint64_t dw = desc_sw128(st), dx = desc_sw128(st + kBM * kSlab);
#pragma unroll
          for (int k = 0; k < 4; ++k)                      // 32 columns of K per instruction
            mma<1>(tmem + (uint32_t)(buf * kR), dw + (uint64_t)(2 * k), dx + (uint64_t)(2 * k), idesc, k > 0);
          commit_to<1>(acc_full + 8 * buf);
          commit_to<1>(empty_bar + 8 * s);
        }
        __syncwarp();
        s += 2;
        if (s >= p.stages) { s -= p.stages; ph ^= 1; }
        buf += 2;
        if (buf >= kAccs) { buf -= kAccs; acc_ph ^= 1; }
      }
    }
  } else if (kQuantize && warp >= kRead + 3) {
    // ------- rows -> E4M3 in the operand's place, their scales times the tile's: eight lanes take a row's block, sixteen columns
    // each, four slabs a step, loaded two steps ahead, over the ends of tiles too -------
    if constexpr (kQuantize) {
      constexpr int kPieces = sizeof(typename In::word);       // of sixteen bytes, in sixteen columns
      const int group = (warp - kRead - 3) * 4 + (lane >> 3), c = lane & 7, rows = (int)p.M;
      const int row = gb_row_ring::row(group, rows), slabs = (total > first ? (total - first + stride - 1) / stride : 0) * k_n;
      const typename In::word* x = static_cast<const typename In::word*>(p.x) + row * p.ld + (int64_t)k_begin * kSlab + c * 16;
      const int64_t width = p.K - (int64_t)k_begin * kSlab - c * 16;
      struct Raw { uint4 v[kPieces]; float bs; };
      // where the loads are: a slab, the tile of features that it belongs to (there is one pass of rows), its block within the tile
      int ahead = gb_row_ring::works(group, rows) ? gb_row_ring::first_slab(group, rows) : slabs, item = first, kt = ahead;
      auto load = [&](Raw& r) {
        const bool live = ahead < slabs;
        if (live)
          for (; kt >= k_n; kt -= k_n) item += stride;
        const uint4* at = reinterpret_cast<const uint4*>(x + (int64_t)kt * kSlab);
#pragma unroll
        for (int q = 0; q < kPieces; ++q) r.v[q] = live && (int64_t)kt * kSlab < width ? at[q] : make_uint4(0u, 0u, 0u, 0u);
        r.bs = live ? p.b_scale[(int64_t)item * p.kb + k_begin + kt] : 0.0f;
        if (live) {
          ahead += gb_row_ring::kSlabsAStep;
          kt += gb_row_ring::kSlabsAStep;
        }
      };
      int n = ahead;                                         // the slab that is written
      Raw cur, next;
      load(cur);
      load(next);
      bool ok = true;
      for (int n0 = 0; n0 < slabs; n0 += gb_row_ring::kSlabsAStep, n += gb_row_ring::kSlabsAStep) {
        Raw after;
        load(after);
        float v[16], scale;
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) gb_blocks::unpack16<In>(cur.v[k], v + k * (16 / kPieces));
        gb_blocks::quantize_block<16, 8>(v, p.scale_rule, scale, q);
        const bool live = n < slabs;
        const int s = n % gb_row_ring::kStages;
        // The stage is free once the MMAs that read it last are done; this group has waited for every phase of the stage before.
        const uint32_t parity = (uint32_t)(n / gb_row_ring::kStages & 1) ^ 1u;
        const bool there = !live || try_wait<kOfCta>(empty_bar + 8 * s, parity);
        if (!__all_sync(0xffffffffu, there)) {
          if (!there) wait_slow<kOfCta>(empty_bar + 8 * s, parity, &abort_s, p.status, 98);
          ok = !__any_sync(0xffffffffu, abort_s != 0);
          if (!ok) break;
        }
        if (live) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                       ::"r"(ring + (uint32_t)s * S::kStageBytes + kBM * kSlab + (uint32_t)(row * kSlab + ((c ^ (row & 7)) * 16))), "r"(q[0]), "r"(q[1]),
                         "r"(q[2]), "r"(q[3]) : "memory");
          if (c == 0) scale_s[(n % kScaleRing) * kR + row] = scale * cur.bs;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (live && c == 0) {
          arrive(full_bar + 8 * s);
          arrive(sc_full + 8 * (n % kScaleRing));
        }
        cur = next;
        next = after;
      }
    }
  } else if (warp == kRead + 3) {
    // ------------------- scales of the rows times the tile's, four blocks at a time --------------------
    if (p.beside) gb_pdl_wait();
    int slot = 0, e = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int item = first; ok && item < total; item += stride) {
      const Item t = item_at(item, e);
      e = t.e;
      const float* bs = p.b_scale + ((int64_t)t.e * p.nb + t.n0 / kSlab) * p.kb;
      for (int kt = k_begin; kt < k_end; kt += 4) {
        const float4 b = scales4(bs, kt, p.kb, p.vec4);
        float4 a[(kR + 31) / 32];
#pragma unroll
        for (int i = 0; i < (kR + 31) / 32; ++i) {
          const int r = i * 32 + lane;
          a[i] = scales4(r < t.rows ? p.a_scale + (int64_t)(t.m0 + r) * p.kb : nullptr, kt, p.kb, p.vec4);
        }
        ok = warp_wait(sc_empty + 8 * slot, ph, &abort_s, p.status, 98);
        if (!ok) break;
        float* to = scale_s + slot * 4 * kR;
#pragma unroll
        for (int i = 0; i < (kR + 31) / 32; ++i) {
          const int r = i * 32 + lane;
          if (r < kR) {
            to[r] = a[i].x * b.x;
            to[kR + r] = a[i].y * b.y;
            to[2 * kR + r] = a[i].z * b.z;
            to[3 * kR + r] = a[i].w * b.w;
          }
        }
        __syncwarp();
        if (lane == 0) arrive(sc_full + 8 * slot);
        if (++slot == kScaleSlots) { slot = 0; ph ^= 1; }
      }
    }
  } else {
    // ------------------------------- read-out -----------------------------------
    if (p.beside) gb_pdl_wait();                           // nothing is written before the launch ahead has finished
    const int quarter = warp & 3, group = warp >> 2;
    const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16);
    int buf = 0, slot = 0, e = 0;
    uint32_t ph = 0, sc_ph = 0;
    bool ok = true;
    for (int item = first; ok && item < total; item += stride) {
      const Item t = item_at(item, e);
      e = t.e;
      const int cols = (t.rows + 15) / 16;                 // sixteens that hold rows
#pragma unroll
      for (int i = 0; i < kMine; ++i)
#pragma unroll
        for (int c = 0; c < 16; ++c) acc[i][c] = 0.0f;
      for (int kt = 0; ok && kt < k_n; ++kt) {
        if (kQuantize || (kt & 3) == 0) {
          ok = warp_wait(sc_full + 8 * slot, sc_ph, &abort_s, p.status, 99);
          if (!ok) break;
        }
        ok = warp_wait<kTensorMemory>(acc_full + 8 * buf, ph, &abort_s, p.status, 100);
        if (!ok) break;
        tmem_fence_after();
        const float* sc = scale_s + (kQuantize ? slot : slot * 4 + (kt & 3)) * kR;
        uint32_t v[kMine][16];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (kMine == 1 || i * (kRead / 4) + group < cols) tmem_ld16(at + (uint32_t)(buf * kR + (i * (kRead / 4) + group) * 16), v[i]);
        tmem_wait_ld();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) arrive(acc_empty + 8 * buf);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          if (kMine > 1 && i * (kRead / 4) + group >= cols) break;
          const float4* s4 = reinterpret_cast<const float4*>(sc + (i * (kRead / 4) + group) * 16);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float4 f = s4[c];
            acc[i][4 * c] = fmaf(__uint_as_float(v[i][4 * c]), f.x, acc[i][4 * c]);
            acc[i][4 * c + 1] = fmaf(__uint_as_float(v[i][4 * c + 1]), f.y, acc[i][4 * c + 1]);
            acc[i][4 * c + 2] = fmaf(__uint_as_float(v[i][4 * c + 2]), f.z, acc[i][4 * c + 2]);
            acc[i][4 * c + 3] = fmaf(__uint_as_float(v[i][4 * c + 3]), f.w, acc[i][4 * c + 3]);
          }
        }
        if (++buf == kAccs) { buf = 0; ph ^= 1; }
        if (kQuantize) {
          // no arrival: an entry is written again 32 slabs on, behind a stage that was freed by MMAs whose accumulators this
          // warp had released long after (stages + accumulators = 16 slabs)
          if (++slot == kScaleRing) { slot = 0; sc_ph ^= 1; }
        } else if ((kt & 3) == 3 || kt + 1 == k_n) {
          __syncwarp();
          if (lane == 0) arrive(sc_empty + 8 * slot);
          if (++slot == kScaleSlots) { slot = 0; sc_ph ^= 1; }
        }
      }
      if (!ok) break;
      last = t;
      if (p.slices == 1) {
        // lane = feature; out through a KB of shared memory per warp, so that four lanes store 64 contiguous bytes of a row
        // (one value a lane and store: 7400 clocks for 128 features of 70 rows, more than half of what their sums took)
        const uint32_t out = gb_smem_u32(out_s) + (uint32_t)warp * 1024u;
        const int f0 = t.n0 + quarter * 32;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int r0 = (i * (kRead / 4) + group) * 16;
          if (r0 >= t.rows) break;
          if (p.out16 && p.out != GB_DTYPE_FP32) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(out + (uint32_t)(c * 64 + lane * 2)), "h"((uint16_t)pack2(acc[i][c], 0.0f, p.out)) : "memory");
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = h * 8 + (lane >> 2), f = f0 + (lane & 3) * 8;
              uint4 q;
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(out + (uint32_t)(h * 512 + lane * 16)) : "memory");
              if (r0 + r < t.rows && f < p.N) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.D) + (int64_t)(t.m0 + r0 + r) * p.N + f) = q;
            }
            __syncwarp();
          } else if (p.out16) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
              for (int c = 0; c < 8; ++c)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(out + (uint32_t)(c * 128 + lane * 4)), "f"(acc[i][half * 8 + c]) : "memory");
              __syncwarp();
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int r = half * 8 + h * 4 + (lane >> 3), f = f0 + (lane & 7) * 4;
                uint4 q;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(out + (uint32_t)(h * 512 + lane * 16)) : "memory");
                if (r0 + r < t.rows && f < p.N) *reinterpret_cast<uint4*>(static_cast<float*>(p.D) + (int64_t)(t.m0 + r0 + r) * p.N + f) = q;
              }
              __syncwarp();
            }
          } else if (f0 + lane < p.N) {                    // rows of D that are no multiple of 16 bytes
            for (int c = 0; c < 16; ++c)
              if (r0 + c < t.rows) {
                float v = acc[i][0];
#pragma unroll
                for (int k = 1; k < 16; ++k) v = c == k ? acc[i][k] : v;
                store1(p.D, (int64_t)(t.m0 + r0 + c) * p.N + f0 + lane, v, p.out);
              }
          }
        }
      }
    }
    if (p.slices > 1) asm volatile("bar.sync 1, %0;" ::"n"(32 * kRead) : "memory");     // all of them see the same flag behind it
  }

  if (p.slices > 1) {
    // Sums into the shared memory of the CTA that owns the row, [slice][own row][feature] (never more than the product's rows); where that lies over the operand
    // ring, every CTA of the cluster has finished its MMAs first, and with them its loads.  Rows are owned in sixteens.
    const bool live = warp < kRead && !abort_s && first < total;
    const int rows = live ? last.rows : 0, cols = (rows + 15) / 16 * 16;
    const int own = (cols / 16 + p.slices - 1) / p.slices * 16;
    const int quarter = warp & 3, group = warp >> 2, feature = quarter * 32 + lane;
    const uint32_t sums = p.overlay ? ring : ring + (uint32_t)p.sums_at;
    if (p.overlay) {
      gb_cluster_sync();
    } else {
      __syncwarp();
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int r0 = (i * (kRead / 4) + group) * 16;
        if (r0 >= cols) continue;
        const int to = r0 / own, off = r0 - to * own;
        uint32_t dst;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                     : "=r"(dst) : "r"(sums + (uint32_t)((slice * p.pitch + off) * kBM + feature) * 4u), "r"(to));
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (r0 + c < rows)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + (uint32_t)c * kBM * 4u), "r"(__float_as_uint(acc[i][c])) : "memory");
      }
    }
    gb_cluster_sync();                                     // the last access to another CTA's memory lies in front of it
    if (live) {
      const int f = lane * 4, left = (int)min((int64_t)kBM, p.N - last.n0) - f, end = min(own, rows - slice * own);
      for (int r = warp; r < end; r += kRead) {
        float sum[4] = {};
#pragma unroll 4
        for (int q = 0; q < p.slices; ++q) {
          float v[4];
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(sums + (uint32_t)((q * p.pitch + r) * kBM + f) * 4u));
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] += v[i];
        }
        const int64_t d = (int64_t)(last.m0 + slice * own + r) * p.N + last.n0 + f;
        if (p.out16 && left > 0 && p.out != GB_DTYPE_FP32) {
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.D) + d) = make_uint2(pack2(sum[0], sum[1], p.out), pack2(sum[2], sum[3], p.out));
        } else if (p.out16 && left > 0) {
          *reinterpret_cast<float4*>(static_cast<float*>(p.D) + d) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < left) store1(p.D, d + i, sum[i], p.out);
        }
      }
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (abort_s) __nanosleep(1000000);                       // loads and MMAs still in flight end before the memory goes
  if (warp == kRead + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmem) : "memory");
}

// ======================================== host =============================================================
std::mutex g_mutex;
int g_pairs[64];                                           // pairs that run at once, per device (0: not asked)
std::atomic<bool> g_ready[64];                             // shared-memory limits of the device's kernels are set

int set_limits() {
#define GB_ATTR(k, bytes) GB_CUDA_OK(cudaFuncSetAttribute((const void*)k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
  GB_ATTR((gemm_blocks_tile_kernel<2, false>), (Tile<2, false>::kSmem));
  GB_ATTR((gemm_blocks_tile_kernel<1, false>), (Tile<1, false>::kSmem));
  GB_ATTR((gemm_blocks_tile_kernel<1, true>), (Tile<1, true>::kSmem));
  GB_ATTR((gemm_blocks_rows_kernel<16, false, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<32, false, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<64, false, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<128, false, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<16, true, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<32, true, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<64, true, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<128, true, void>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<16, false, gb_blocks::Bf16>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<16, false, gb_blocks::Fp16>), kSmemMax);
  GB_ATTR((gemm_blocks_rows_kernel<16, false, gb_blocks::Fp32>), kSmemMax);
#undef GB_ATTR
  return GB_OK;
}

// The limits of the current device, once; callers need not have gone through gb_prepare.
int ready() {
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  GB_REQUIRE(dev >= 0 && dev < 64, "device %d out of range", dev);
  if (g_ready[dev].load(std::memory_order_acquire)) return GB_OK;
  std::lock_guard<std::mutex> lock(g_mutex);
  const int rc = set_limits();
  if (rc == GB_OK) g_ready[dev].store(true, std::memory_order_release);
  return rc;
}

int resident_pairs() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(g_mutex);
  int& n = g_pairs[dev];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * 256);
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = Tile<2, false>::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, gemm_blocks_tile_kernel<2, false>, &cfg) != cudaSuccess) { n = 0; cudaGetLastError(); }
  }
  return n;
}

// Slices of K of a single CTA's tiles: as many as the SMs take, at least eight blocks each; slices start at multiples of four blocks
// where rows of the scales are whole 16-byte pieces.
struct Slices { int n, per; };
Slices slices_of(int64_t tiles, int kb) {
  static GbClusters clusters;
  int want = 1;
  for (int n = 2; n <= kMaxSlices && tiles * n <= gb_sm_count() && n * 8 <= kb; ++n)
    if (tiles <= clusters.ask((const void*)gemm_blocks_tile_kernel<1, false>, kPairThreads, Tile<1, false>::kSmem, n)) want = n;
  int per = (kb + want - 1) / want;
  if (kb % 4 == 0) per = (per + 3) / 4 * 4;
  return {(kb + per - 1) / per, per};
}

template <int kCtas, bool kGrouped>
int run_tiles(const void* A, const void* W, int64_t K, BlocksParams p, cudaStream_t stream) {
  using S = Tile<kCtas, kGrouped>;
  const int most = kCtas == 2 ? resident_pairs() : gb_sm_count();
  if (most <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  p.n_tiles = (int)((p.N + kBN - 1) / kBN);
  p.m_tiles = (int)((p.M + S::kM - 1) / S::kM);
  p.idesc = (1u << 4) | ((uint32_t)((kCtas == 1 ? kBN : kPart) >> 3) << 17) | ((uint32_t)(S::kM >> 4) << 24);
  p.out_tma = p.N % 8 == 0 && p.out != GB_DTYPE_FP32;
  CUtensorMap map_a, map_b, map_d = {};
  int rc = gb_tensor_map_operand(&map_a, A, p.M, K, 1, kBM);
  if (rc != GB_OK) return rc;
  rc = gb_tensor_map_operand(&map_b, W, (kGrouped ? p.E : 1) * p.N, K, 1, kPart / kCtas);
  if (rc != GB_OK) return rc;
  if (p.out_tma) {
    rc = gb_tensor_map_out(&map_d, p.D, p.M, p.N);
    if (rc != GB_OK) return rc;
  }
  p.most_row_tiles = (int)(p.M / S::kM + (p.M < p.E ? p.M : p.E));
  const int64_t tiles = (int64_t)(kGrouped ? p.most_row_tiles : p.m_tiles) * p.n_tiles;
  GB_REQUIRE(tiles < (1ll << 31), "too many output tiles");
  Slices slices = {1, p.kb};
  if (kCtas == 1 && !kGrouped) slices = slices_of(tiles, p.kb);
  p.slices = slices.n;
  p.per_slice = slices.per;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(kCtas * (tiles < most ? tiles : most)), (unsigned)p.slices);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (kCtas == 2 || p.slices > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = kCtas; attr[n].val.clusterDim.y = (unsigned)p.slices; attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (gb_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  gb_count_launch();
  GB_CUDA_OK(cudaLaunchKernelEx(&cfg, gemm_blocks_tile_kernel<kCtas, kGrouped>, map_a, map_b, map_d, p));
  return GB_OK;
}

template <int kR, bool kGrouped, typename In = void>
int run_rows(const void* A, const void* W, int64_t K, BlocksParams p, cudaStream_t stream) {
  using S = Rows<kR, In>;
  const int64_t sms = gb_sm_count();
  if (sms <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  p.n_tiles = (int)((p.N + kBM - 1) / kBM);
  int64_t most;                                            // items there can be
  if (kGrouped) {
    p.most_row_tiles = (int)(p.M / kR + (p.M < p.E ? p.M : p.E));
    most = (int64_t)p.most_row_tiles * p.n_tiles;
  } else {
    p.passes = (int)((p.M + kR - 1) / kR);
    p.rows_per_pass = (int)(((p.M + p.passes - 1) / p.passes + 15) / 16 * 16);
    p.passes = (int)((p.M + p.rows_per_pass - 1) / p.rows_per_pass);
    most = (int64_t)p.passes * p.n_tiles;
  }
  GB_REQUIRE(most < (1ll << 31), "too many output tiles");
  // K slices: as many as the SMs take, at least four blocks each
  static GbClusters clusters;
  int want = 1;
  for (int n = 2; n <= (kR <= 64 ? kMaxSlices : 4) && most * n <= sms && n * 4 <= p.kb; ++n)
    if (most <= clusters.ask((const void*)gemm_blocks_rows_kernel<kR, kGrouped, In>, S::kThreads, kSmemMax, n)) want = n;
  p.per_slice = (p.kb + want - 1) / want;
  p.slices = (p.kb + p.per_slice - 1) / p.per_slice;
  constexpr int kFixed = 1024 + (S::kQuantize ? kScaleRing : 4 * kScaleSlots) * kR * 4 + (kGrouped ? kSegBytes : 0);
  // the sums take up to 64 KB: of their own where that leaves enough stages
  constexpr int kLeast = 8;
  const int own = (kR / 16 + p.slices - 1) / p.slices * 16;
  p.pitch = p.M < own ? (int)p.M : own;
  const int sums = p.slices > 1 ? p.slices * p.pitch * kBM * 4 : 0;
  p.overlay = (kSmemMax - kFixed - sums) / S::kStageBytes < kLeast;
  p.stages = (kSmemMax - kFixed - (p.overlay ? 0 : sums)) / S::kStageBytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.stages &= ~1;
  // One tile a CTA and few rows: eight stages do, and more in flight at the start cost (one row of 5120 x 8192 10.5 us with ten, 9.9 with
  // eight, 10.6 with twelve and 11.8 with four; 16 rows 10.9 and 10.7).
  if (kR == 16 && !kGrouped && (p.slices > 1 || most <= sms) && p.stages > kFewStages) p.stages = kFewStages;
  if (S::kQuantize) p.stages = gb_row_ring::kStages;
  static_assert(!S::kQuantize || (kSmemMax - kFixed - kMaxSlices * kQuantMaxRows * kBM * 4) / S::kStageBytes >= gb_row_ring::kStages,
                "so many stages, and the sums of a sliced K beside them");
  p.sums_at = kFixed - 1024 + p.stages * S::kStageBytes;
  p.idesc = 1u << 4;
  CUtensorMap map_w, map_x = {};
  int rc = gb_tensor_map_operand(&map_w, W, (kGrouped ? p.E : 1) * p.N, K, 1, kBM);
  if (rc != GB_OK) return rc;
  if (!S::kQuantize) {
    rc = gb_tensor_map_operand(&map_x, A, p.M, K, 1, S::kBox);
    if (rc != GB_OK) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.slices > 1 || most < sms ? most : sms), (unsigned)p.slices);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = kFixed + p.stages * S::kStageBytes + (p.overlay ? 0 : sums);
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
  GB_CUDA_OK(cudaLaunchKernelEx(&cfg, gemm_blocks_rows_kernel<kR, kGrouped, In>, map_w, map_x, p));
  return GB_OK;
}

template <bool kGrouped>
int run_few(const void* A, const void* W, int64_t K, const BlocksParams& p, int64_t rows, cudaStream_t stream) {
  if (rows <= 16) return run_rows<16, kGrouped>(A, W, K, p, stream);
  if (rows <= 32) return run_rows<32, kGrouped>(A, W, K, p, stream);
  if (rows <= 64) return run_rows<64, kGrouped>(A, W, K, p, stream);
  return run_rows<128, kGrouped>(A, W, K, p, stream);
}

int check_blocks(const void* A, const float* as, const void* W, const float* bs, const void* D, int out, int64_t M, int64_t N, int64_t K, int64_t E) {
  GB_REQUIRE(out >= GB_DTYPE_BF16 && out <= GB_DTYPE_FP32, "unknown dtype %d", out);
  GB_REQUIRE(M >= 0 && N > 0 && K > 0, "bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  GB_REQUIRE(K % 16 == 0, "K=%lld must be a multiple of 16: rows of both operands are fetched in 16-byte pieces", (long long)K);
  GB_REQUIRE(M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30) && E * N < (1ll << 31), "dimension too large");
  if (M == 0) return GB_OK;
  GB_REQUIRE(A && as && W && bs && D, "null pointer argument");
  GB_REQUIRE(((uintptr_t)A & 15u) == 0 && ((uintptr_t)W & 15u) == 0, "operands must be 16-byte aligned");
  GB_REQUIRE(((uintptr_t)D & 15u) == 0, "the output must be 16-byte aligned");
  GB_REQUIRE((((uintptr_t)as | (uintptr_t)bs) & 3u) == 0, "misaligned scales");
  return ready();
}

BlocksParams params(const float* as, const float* bs, void* D, int out, int64_t M, int64_t N, int64_t K, int beside) {
  BlocksParams p = {};
  p.M = M; p.N = N;
  p.kb = (int)((K + kSlab - 1) / kSlab);
  p.nb = (int)((N + kSlab - 1) / kSlab);
  p.a_scale = as; p.b_scale = bs;
  p.D = D; p.out = out;
  p.vec4 = p.kb % 4 == 0 && (((uintptr_t)as | (uintptr_t)bs) & 15u) == 0;
  p.out16 = N * (out == GB_DTYPE_FP32 ? 4 : 2) % 16 == 0;
  p.beside = beside;
  p.status = gb_status_word();
  return p;
}

// Which kernel a dense product takes; us.
//   rows kernel / single CTAs: 64 rows of 5120 x 17408 23.0 / 28.7, 100 of 4096 x 4096 12.3 / 12.9, 128 of 34816 x 5120 42.0 / 36.9, 160 of 2048 x 8192
//     14.4 / 18.5 (eight slices of K, whose sums cost more the larger the tiles), of 5120 x 17408 49.2 / 34.9, 333 of 2048 x 5120 16.4 / 16.4,
//     of 5120 x 17408 59.4 / 43.0.
//   pairs / single CTAs: 333 rows of 5120 x 17408 62.8 / 43.0, 512 of 5120 x 5120 24.4 / 24.6, 700 of 4096 x 4096 21.7 / 20.9, 256 of 34816 x 5120 49.6 / 52,
//     8192 of 34816 x 5120 over two seconds, where the power cap rules, 1407 / 1465: a pair fetches its features once for both.
enum Route { kRowsRoute, kCtaRoute, kPairRoute };
Route route_of(int64_t M, int64_t N) {
  const int64_t sms = gb_sm_count(), n_tiles = (N + kBN - 1) / kBN, tiles = (M + kBM - 1) / kBM * n_tiles;
  if (M <= 64 || (M <= kBM && 2 * n_tiles < sms) || 6 * tiles < sms) return kRowsRoute;
  return tiles <= sms ? kCtaRoute : kPairRoute;
}

}  // namespace

extern "C" {

int gb_gemm_fp8_blocks(const void* A, const float* a_scale, const void* W, const float* w_scale, void* D, int out, int64_t M, int64_t N, int64_t K,
                       int beside, void* stream) {
  const int rc = check_blocks(A, a_scale, W, w_scale, D, out, M, N, K, 1);
  if (rc != GB_OK || M == 0) return rc;
  const BlocksParams p = params(a_scale, w_scale, D, out, M, N, K, beside);
  const Route route = route_of(M, N);
  if (route == kRowsRoute) return run_few<false>(A, W, K, p, M, (cudaStream_t)stream);
  return route == kCtaRoute ? run_tiles<1, false>(A, W, K, p, (cudaStream_t)stream) : run_tiles<2, false>(A, W, K, p, (cudaStream_t)stream);
}

// The kernel that gb_gemm_fp8_blocks launches, and its slices of K where those are told.
int gb_gemm_fp8_blocks_kernel(int64_t M, int64_t N, int64_t K, int32_t* slices) {
  if (slices) *slices = 1;
  const Route route = route_of(M, N);
  if (route == kCtaRoute && slices && ready() == GB_OK)
    *slices = slices_of((M + kBM - 1) / kBM * ((N + kBN - 1) / kBN), (int)((K + kSlab - 1) / kSlab)).n;
  return route;
}

// us in a graph of many layers, two launches / one: 1 row of 34816 x 5120 30.8 / 28.9, 4 rows 30.7 / 29.1; 1 row of 4096 x 4096 7.9 / 6.1, 4 rows
// 8.1 / 6.2.  Not more rows: every CTA quantises all of them (when one launch took them, 8 rows of 34816 x 5120 36.7 / 43.0, 16 rows of 4096 x 4096
// 10.3 / 12.3).

int gb_linear_fp8_blocks(const void* x, int dtype, int64_t ld, int scale_rule, const void* W, const float* w_scale, void* D, int out, int64_t M, int64_t N,
                         int64_t K, void* stream) {
  GB_REQUIRE(dtype >= GB_DTYPE_BF16 && dtype <= GB_DTYPE_FP32, "unknown dtype %d", dtype);
  GB_REQUIRE(scale_rule == GB_SCALE_RULE_RECIP || scale_rule == GB_SCALE_RULE_DIV, "unknown scale rule %d", scale_rule);
  const int eb = dtype == GB_DTYPE_FP32 ? 4 : 2;
  GB_REQUIRE(ld >= K || M <= 1, "row stride %lld is shorter than the row", (long long)ld);
  if (M > kQuantMaxRows || ((uintptr_t)x & 15u) != 0 || (M > 1 && ld * eb % 16 != 0))
    return gb_fail(GB_EUNSUPPORTED, "more than 4 rows, or rows off the 16-byte alignment: quantise them first");
  const int rc = check_blocks(W, w_scale, W, w_scale, D, out, M, N, K, 1);
  if (rc != GB_OK || M == 0) return rc;
  GB_REQUIRE(x != nullptr, "null pointer argument");
  BlocksParams p = params(w_scale, w_scale, D, out, M, N, K, 0);
  p.x = x; p.ld = ld; p.K = K; p.scale_rule = scale_rule;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == GB_DTYPE_BF16) return run_rows<16, false, gb_blocks::Bf16>(nullptr, W, K, p, st);
  if (dtype == GB_DTYPE_FP16) return run_rows<16, false, gb_blocks::Fp16>(nullptr, W, K, p, st);
  return run_rows<16, false, gb_blocks::Fp32>(nullptr, W, K, p, st);
}

int gb_gemm_fp8_blocks_grouped(const void* A, const float* a_scale, const void* W, const float* w_scale, const int32_t* seg_offsets, int64_t E, void* D,
                               int out, int64_t P, int64_t N, int64_t K, int beside, void* stream) {
  GB_REQUIRE(E > 0 && E <= kMaxGroups, "expert count %lld outside [1, %d]", (long long)E, kMaxGroups);
  const int rc = check_blocks(A, a_scale, W, w_scale, D, out, P, N, K, E);
  if (rc != GB_OK || P == 0) return rc;
  GB_REQUIRE(seg_offsets != nullptr, "null pointer argument");
  BlocksParams p = params(a_scale, w_scale, D, out, P, N, K, beside);
  p.seg = seg_offsets;
  p.E = (int)E;
  // us, rows kernel / tiles of 128 rows, 128 experts of 1536 x 2048: 32 rows an expert on average 71.7 / 79.5, 64 77.9 / 83.4, 96 90.4 / 86.5,
  // 128 122 / 100, 256 198 / 148 (pairs' tiles of 256 rows 116, 119 and 164); 32 of 4096 x 7168: 100 185 / 173.  A pass of the
  // rows kernel holds twice the average where that is at most 128.
  const int64_t mean = P / E;
  if (mean <= 72) return run_few<true>(A, W, K, p, 2 * mean, (cudaStream_t)stream);
  return run_tiles<1, true>(A, W, K, p, (cudaStream_t)stream);
}

}  // extern "C"
