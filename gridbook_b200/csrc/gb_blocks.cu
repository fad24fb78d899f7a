// Rows of block-scaled E4M3 and the routed layer's tokens sorted by expert and back.
//
// Quantiser: a block is 128 consecutive columns of a row (the last one may be short).  With amax the block's largest
// magnitude (at least 1e-10, so that a block of zeros gets a scale that divides),
//     scale = amax / 448 (a product with the fp32 reciprocal, or a true division),  q = e4m3(x / scale),
// the quotient rounded once to fp32 and once to E4M3, ties to even.  A NaN or an infinity spreads over its block.
// Three sources of the rows: as they lie; a token's row written once for each of its experts; silu(gate) * up in fp32.
//
// Sixteen lanes take a block, eight columns each: the maximum is four shuffles away, a warp reads 512 contiguous bytes of
// 16-bit rows and writes 256 of the result.
#include "gb_blocks.cuh"

namespace {

using namespace gb_blocks;

constexpr int kThreads = 256, kHalfWarps = kThreads / 16;

enum Source { kRows = 0, kSorted = 1, kSwiglu = 2 };

// Eight consecutive columns as they lie in memory, zeros past the row's end.  kVec: rows of whole 16-byte pieces, K a multiple
// of 8.
template <typename T, bool kVec>
struct Eight {
  static constexpr int kPieces = sizeof(typename T::word) / 2;
  using word = typename T::word;
  uint4 v[kVec ? kPieces : 1];
  word w[kVec ? 1 : 8];
  GB_DEVINL void load(const word* row, int64_t c, int64_t K) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) v[i] = c < K ? __ldg(reinterpret_cast<const uint4*>(row + c) + i) : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = c + i < K ? row[c + i] : word(0);
    }
  }
  GB_DEVINL void clear() {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = word(0);
    }
  }
  GB_DEVINL void unpack(float (&f)[8]) const {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) unpack16<T>(v[i], f + i * (8 / kPieces));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(w[i]);
    }
  }
};

// gate / (1 + exp(-gate)): the reciprocal is off by a unit at most, the exponential by 2 + 1.2 |gate|; a gate far below zero
// gives zero, whose exponential is infinite.
GB_DEVINL float silu(float gate) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-gate)));
  return gate * r;
}
template <bool kVec>
GB_DEVINL void store8(uint8_t* row, int64_t c, int64_t K, uint2 q) {
  if constexpr (kVec) {
    if (c < K) *reinterpret_cast<uint2*>(row + c) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) row[c + i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

GB_DEVINL bool in_rows(int64_t at, int64_t rows) { return (uint64_t)at < (uint64_t)rows; }

struct QuantizeParams {
  const void* x;
  int64_t ld, rows, K;        // of the result; a swiglu row is [gate | up]
  uint32_t blocks;            // of a row
  uint32_t step_rows, step_blocks;      // sixteen blocks further on
  int64_t units;              // rows * blocks
  int scale_rule;
  uint8_t* q;
  float* scale;
  const int32_t* place;       // sorted: row of a (token, slot) pair, -1 where it is dropped
  const int32_t* live;        // sorted: rows that a pair has; swiglu: rows that count (null: all)
  int topk;
};

// kPer blocks for each half warp, their loads in flight together.
template <typename T, Source kSource, bool kVec, int kPer>
__global__ void __launch_bounds__(kThreads)
quantize_blocks_kernel(const __grid_constant__ QuantizeParams p) {
  gb_pdl_wait();
  gb_pdl_launch_dependents();              // behind the wait: a product behind this launch may read its weights at once
  const int half = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const typename T::word* x = static_cast<const typename T::word*>(p.x);
  int64_t rows = p.rows;
  if (kSource == kSwiglu && p.live) rows = min(rows, (int64_t)*p.live);
  // every block's bytes are on their way before the first is looked at
  Eight<T, kVec> raw[kPer], up[kSource == kSwiglu ? kPer : 1];
  int64_t row[kPer];
  uint32_t block[kPer];
  const int64_t unit = (int64_t)blockIdx.x * (kPer * kHalfWarps) + half;
  row[0] = (uint32_t)unit / p.blocks;
  block[0] = (uint32_t)unit - (uint32_t)row[0] * p.blocks;
#pragma unroll
  for (int i = 1; i < kPer; ++i) {         // sixteen blocks on
    row[i] = row[i - 1] + p.step_rows;
    block[i] = block[i - 1] + p.step_blocks;
    if (block[i] >= p.blocks) { block[i] -= p.blocks; ++row[i]; }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t c = (int64_t)block[i] * kBlock + lane * 8;
    if (row[i] < rows) {
      raw[i].load(x + row[i] * p.ld, c, p.K);
      if constexpr (kSource == kSwiglu) up[i].load(x + row[i] * p.ld + p.K, c, p.K);
    } else {
      raw[i].clear();
      if constexpr (kSource == kSwiglu) up[i].clear();
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t c = (int64_t)block[i] * kBlock + lane * 8;
    int to_lane = -1;
    if (kSource == kSorted && row[i] < rows && lane < p.topk) to_lane = p.place[row[i] * p.topk + lane];
    float v[8], scale;
    raw[i].unpack(v);
    if constexpr (kSource == kSwiglu) {    // zeros past the row's end stay zeros
      float u[8];
      up[i].unpack(u);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = silu(v[k]) * u[k];
    }
    uint32_t w[2];
    quantize_block<8, 16>(v, p.scale_rule, scale, w);
    const uint2 q = make_uint2(w[0], w[1]);
    if constexpr (kSource == kSorted) {
      for (int s = 0; s < p.topk; ++s) {   // the same for all sixteen lanes
        int64_t to = __shfl_sync(0xffffffffu, to_lane, s & 15, 16);
        if (s >= 16) to = row[i] < rows ? p.place[row[i] * p.topk + s] : -1;
        if (!in_rows(to, p.rows * p.topk)) continue;
        store8<kVec>(p.q + to * p.K, c, p.K, q);
        if (lane == 0) p.scale[to * p.blocks + block[i]] = scale;
      }
    } else if (row[i] < rows) {
      store8<kVec>(p.q + row[i] * p.K, c, p.K, q);
      if (lane == 0) p.scale[row[i] * p.blocks + block[i]] = scale;
    }
  }
  if constexpr (kSource == kSorted) {      // rows that no pair has read zero
    const int64_t pairs = p.rows * p.topk, first = max(*p.live, 0), left = (pairs - first) * p.blocks;
    for (int64_t u = (int64_t)blockIdx.x * kHalfWarps + half; u < left; u += (int64_t)gridDim.x * kHalfWarps) {
      const int64_t to = first + u / p.blocks, b = u % p.blocks;
      store8<kVec>(p.q + to * p.K, b * kBlock + lane * 8, p.K, make_uint2(0u, 0u));
      if (lane == 0) p.scale[to * p.blocks + b] = 0.0f;
    }
  }
}

template <typename T, Source kSource>
int launch_quantize(const QuantizeParams& p, bool vec, cudaStream_t stream) {
  // one block each for less than a wave of them, two from there on (8192 rows of 5120 bf16: 32.3 us, 31.2, four 32.9); where every
  // block is written several times, from two waves on (one, two, four: 512 tokens x 8 of 7168 columns 10.8 us, 11.6, 13.6; 4096 of
  // 2048 21.4, 20.5, 22.2; 2048 of 7168 35.4, 33.9, 37.8)
  const int64_t few = (kSource == kSorted ? 16ll : 8ll) * gb_sm_count() * kHalfWarps;
  const int per = p.units > few ? 2 : 1;
  const dim3 grid((unsigned)((p.units + per * kHalfWarps - 1) / (per * kHalfWarps)));
#define GB_Q(v, n) GB_CUDA_OK(gb_launch(quantize_blocks_kernel<T, kSource, v, n>, grid, dim3(kThreads), 0, stream, p))
  if (vec) { if (per == 2) GB_Q(true, 2); else GB_Q(true, 1); }
  else { if (per == 2) GB_Q(false, 2); else GB_Q(false, 1); }
#undef GB_Q
  return GB_OK;
}

int elem_bytes(int dtype) { return dtype == GB_DTYPE_FP32 ? 4 : 2; }

template <Source kSource>
int quantize(QuantizeParams p, int dtype, cudaStream_t stream) {
  GB_REQUIRE(dtype >= GB_DTYPE_BF16 && dtype <= GB_DTYPE_FP32, "unknown dtype %d", dtype);
  GB_REQUIRE(p.scale_rule == GB_SCALE_RULE_RECIP || p.scale_rule == GB_SCALE_RULE_DIV, "unknown scale rule %d", p.scale_rule);
  GB_REQUIRE(p.rows >= 0 && p.K > 0 && p.K < (1ll << 31), "bad shape rows=%lld K=%lld", (long long)p.rows, (long long)p.K);
  GB_REQUIRE(p.ld >= p.K * (kSource == kSwiglu ? 2 : 1), "row stride %lld is shorter than the row", (long long)p.ld);
  if (p.rows == 0) return GB_OK;
  GB_REQUIRE(p.x && p.q && p.scale, "null pointer argument");
  GB_REQUIRE(((uintptr_t)p.scale & 3u) == 0 && (uintptr_t)p.x % elem_bytes(dtype) == 0, "misaligned pointer");
  p.blocks = (uint32_t)((p.K + kBlock - 1) / kBlock);
  p.step_rows = kHalfWarps / p.blocks;
  p.step_blocks = kHalfWarps % p.blocks;
  p.units = p.rows * p.blocks;
  GB_REQUIRE(p.units < (1ll << 31), "too many blocks");
  const int eb = elem_bytes(dtype);
  const bool vec = p.K % 8 == 0 && p.ld * eb % 16 == 0 && ((uintptr_t)p.x & 15u) == 0 && ((uintptr_t)p.q & 7u) == 0;
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  if (dtype == GB_DTYPE_BF16) return launch_quantize<Bf16, kSource>(p, vec, stream);
  if (dtype == GB_DTYPE_FP16) return launch_quantize<Fp16, kSource>(p, vec, stream);
  return launch_quantize<Fp32, kSource>(p, vec, stream);
}

// ---- the sort itself -------------------------------------------------------------------------------------------
// Pairs by expert, stable, in ONE launch: a cluster of up to eight CTAs, a warp 32 kPer consecutive pairs.  A pair's place =
// the expert's segment start + its pairs in earlier CTAs + in earlier warps + in earlier steps of its warp + its rank among
// the step's lanes.  Every CTA counts its own pairs; the counts of the others are read through the cluster's shared memory.
// The same order as gb_moe_route's, which takes three launches from 4096 pairs on.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortExperts = 1024, kSortMostCtas = 8, kSortMostPer = 8;

GB_DEVINL int load_cluster(uint32_t addr, int rank) {
  uint32_t from, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
  return (int)v;
}
// Exclusive prefix of v over the CTA's threads, and the sum, by shuffles within the warps and one warp over them.
GB_DEVINL int prefix_sum(int v, int* warp_sums, int& sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += n;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int others = warp_sums[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, others, d);
    if (lane >= d) others += n;
  }
  sum = __shfl_sync(0xffffffffu, others, 31);
  const int before = __shfl_sync(0xffffffffu, others, (warp + 31) & 31);
  return incl - v + (warp ? before : 0);
}

template <typename Id, int kPer>
__global__ void __launch_bounds__(kSortThreads)
sort_pairs_kernel(const Id* __restrict__ ids, int P, int E, int64_t first_expert, int per_cta, int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                  int32_t* __restrict__ order, int32_t* __restrict__ place) {
  extern __shared__ int32_t sh[];          // [warp][E] counts, then starts; [E] the CTA's counts; [E] starts of its pairs
  __shared__ int32_t warp_sums[32];
  int32_t* mine = sh + (threadIdx.x >> 5) * E;
  int32_t *total = sh + kSortWarps * E, *start = total + E;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int rank, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  gb_pdl_launch_dependents();
  for (int k = tid; k < E * kSortWarps; k += kSortThreads) sh[k] = 0;
  gb_pdl_wait();
  const int base = rank * per_cta, end = min(P, base + per_cta), first = base + warp * 32 * kPer + lane;
  int id[kPer], at[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = first + 32 * j;
    const int64_t e = i < end ? (int64_t)ids[i] - first_expert : -1;
    id[j] = e >= 0 && e < E ? (int)e : -1;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const unsigned same = __match_any_sync(0xffffffffu, id[j]);
    const int before = id[j] >= 0 ? mine[id[j]] : 0;
    at[j] = before + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (id[j] >= 0 && (same & ((1u << lane) - 1u)) == 0) mine[id[j]] = before + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  const int warps = min(kSortWarps, (end - base + 32 * kPer - 1) / (32 * kPer));       // the others hold no pair
  for (int e = tid; e < E; e += kSortThreads) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < warps; ++w) {
      const int v = sh[w * E + e];
      sh[w * E + e] = run;
      run += v;
    }
    total[e] = run;
  }
  gb_cluster_sync();                       // E is at most the CTA's threads: one expert each from here on
  int all = 0, before = 0;
  if (tid < E)
    for (int r = 0; r < ctas; ++r) {
      const int v = load_cluster(gb_smem_u32(total + tid), r);
      before += r < rank ? v : 0;
      all += v;
    }
  int live;
  const int off = prefix_sum(all, warp_sums, live);
  if (tid < E) {
    start[tid] = off + before;
    if (rank == 0) {
      counts[tid] = all;
      offsets[tid] = off;
    }
  }
  if (rank == 0 && tid == 0) offsets[E] = live;
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");       // nothing of another CTA is read behind this
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = first + 32 * j;
    if (id[j] >= 0) {
      const int to = start[id[j]] + mine[id[j]] + at[j];
      order[to] = i;
      place[i] = to;
    } else if (i < end) {
      place[i] = -1;
    }
  }
  for (int i = live + rank * kSortThreads + tid; i < P; i += ctas * kSortThreads) order[i] = 0;     // dropped pairs
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

template <typename Id>
int launch_sort(const void* ids, int P, int E, int64_t base, int32_t* counts, int32_t* offsets, int32_t* order, int32_t* place, cudaStream_t stream) {
  // CTAs while each has at least 512 pairs, then pairs per thread
  int ctas = 1, per = 1;
  while (ctas < kSortMostCtas && P > ctas * 512) ctas *= 2;
  while (P > ctas * per * kSortThreads) per *= 2;
  const int per_cta = (P + ctas - 1) / ctas;
  const size_t smem = (size_t)(kSortWarps + 2) * E * sizeof(int32_t);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = gb_pdl_enabled() ? 2 : 1;
  gb_count_launch();
#define GB_SORT(n)                                                                                                                          \
  do {                                                                                                                                      \
    if (smem > 48 * 1024)                                                                                                                   \
      GB_CUDA_OK(cudaFuncSetAttribute((const void*)sort_pairs_kernel<Id, n>, cudaFuncAttributeMaxDynamicSharedMemorySize,                  \
                                      (int)((kSortWarps + 2) * kSortExperts * sizeof(int32_t))));                                          \
    GB_CUDA_OK(cudaLaunchKernelEx(&cfg, sort_pairs_kernel<Id, n>, (const Id*)ids, P, E, base, per_cta, counts, offsets, order, place));     \
  } while (0)
  if (per == 1) GB_SORT(1);
  else if (per == 2) GB_SORT(2);
  else if (per == 4) GB_SORT(4);
  else GB_SORT(8);
#undef GB_SORT
  return GB_OK;
}

// ---- tokens into expert order and back ---------------------------------------------------------------------
// A CTA holds blockDim.y tokens, blockDim.x lanes walk a row in vectors of V.  All three are bound by memory.

// Places and counts come from a sort of the same pairs; whatever they say, no row outside of [0, pairs) is touched.

// rows[place[t, s]] = x[t]: a token's row is read once and written for each of its experts; rows that no pair has
// become zero.
template <typename V>
__global__ void __launch_bounds__(256)
permute_kernel(const uint8_t* __restrict__ x, int64_t pitch, const int32_t* __restrict__ place, const int32_t* __restrict__ live, int64_t T,
               int topk, int vecs, uint8_t* __restrict__ rows) {
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int64_t row_bytes = (int64_t)vecs * sizeof(V), t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t < T) {
    const V* from = reinterpret_cast<const V*>(x + t * pitch);
    for (int c = threadIdx.x; c < vecs; c += blockDim.x) {
      const V v = from[c];
      for (int s = 0; s < topk; ++s) {
        const int64_t to = place[t * topk + s];
        if (in_rows(to, T * topk)) reinterpret_cast<V*>(rows + to * row_bytes)[c] = v;
      }
    }
  }
  for (int64_t j = max(*live, 0) + t; j < T * topk; j += (int64_t)gridDim.x * blockDim.y) {
    V* to = reinterpret_cast<V*>(rows + j * row_bytes);
    for (int c = threadIdx.x; c < vecs; c += blockDim.x) to[c] = V{};
  }
}

// One vector of a row as fp32, and back: sixteen bytes, or one value where the rows are not whole aligned vectors.
template <typename T, bool kVec>
struct Piece {
  static constexpr int n = kVec ? 16 / (int)sizeof(typename T::word) : 1;
  using raw = typename std::conditional<kVec, uint4, typename T::word>::type;
  static GB_DEVINL void unpack(const raw& r, float (&v)[n]) {
    if constexpr (kVec) unpack16<T>(r, v);
    else v[0] = to_f32<T>(r);
  }
  static GB_DEVINL raw pack(const float (&v)[n]) {
    if constexpr (kVec) return pack16<T>(v);
    else return from_f32<T>(v[0]);
  }
};

// out[t] = sum over the token's slots of w[t, s] * y[place[t, s]] (w null: ones), in slot order, fp32, rounded once.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256)
unpermute_kernel(const typename T::word* __restrict__ y, const int32_t* __restrict__ place, const float* __restrict__ w, int64_t tokens,
                 int topk, int vecs, typename T::word* __restrict__ out) {
  using P = Piece<T, kVec>;
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int64_t H = (int64_t)vecs * P::n, t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= tokens) return;
  constexpr int kInFlight = 4;           // eight: 37 us instead of 29 for 4096 tokens x 8 x 2048 columns, fewer CTAs being resident
  for (int c = threadIdx.x; c < vecs; c += blockDim.x) {
    float acc[P::n] = {};
    for (int s0 = 0; s0 < topk; s0 += kInFlight) {
      typename P::raw r[kInFlight];
      int at[kInFlight];
      float weight[kInFlight];
#pragma unroll
      for (int j = 0; j < kInFlight; ++j) {
        at[j] = s0 + j < topk ? place[t * topk + s0 + j] : -1;
        if (!in_rows(at[j], tokens * topk)) at[j] = -1;
        weight[j] = w && s0 + j < topk ? w[t * topk + s0 + j] : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < kInFlight; ++j)
        if (at[j] >= 0) r[j] = reinterpret_cast<const typename P::raw*>(y + at[j] * H)[c];
#pragma unroll
      for (int j = 0; j < kInFlight; ++j) {
        if (at[j] < 0) continue;
        float v[P::n];
        P::unpack(r[j], v);
#pragma unroll
        for (int i = 0; i < P::n; ++i) acc[i] = fmaf(weight[j], v[i], acc[i]);
      }
    }
    reinterpret_cast<typename P::raw*>(out + t * H)[c] = P::pack(acc);
  }
}

// The weighted sum's gradients, with g = d_out[t]: d_y[place[t, s]] = w[t, s] * g, d_w[t, s] = <y[place[t, s]], g>; a dropped
// pair's weight gets zero, rows of d_y that no pair has become zero.  A token's lanes are whole warps of one CTA: sums by
// shuffles, then over the warps in order.  kSlots of a token's slots at a time: the gradient's row comes out of L1 again for the
// next ones, which costs less than the registers of more (4096 tokens x 8 x 2048 columns: 59 us with eight, 53 with four).
template <typename T, bool kVec, int kSlots>
__global__ void __launch_bounds__(128)
unpermute_grad_kernel(const typename T::word* __restrict__ d_out, const typename T::word* __restrict__ y, const int32_t* __restrict__ place,
                      const int32_t* __restrict__ live, const float* __restrict__ w, int64_t tokens, int topk, int vecs,
                      typename T::word* __restrict__ d_y, float* __restrict__ d_w) {
  using P = Piece<T, kVec>;
  __shared__ float part[4][kSlots];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int64_t H = (int64_t)vecs * P::n, t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, first_warp = threadIdx.y * warps;
  const bool mine = t < tokens;
  for (int s0 = 0; s0 < topk; s0 += kSlots) {
    int64_t at[kSlots];
    float weight[kSlots], dot[kSlots];
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      at[j] = mine && s0 + j < topk ? (int64_t)place[t * topk + s0 + j] : -1;
      if (!in_rows(at[j], tokens * topk)) at[j] = -1;
      weight[j] = at[j] >= 0 ? w[t * topk + s0 + j] : 0.0f;
      dot[j] = 0.0f;
    }
    for (int c = threadIdx.x; mine && c < vecs; c += blockDim.x) {
      float g[P::n];
      P::unpack(reinterpret_cast<const typename P::raw*>(d_out + t * H)[c], g);
      typename P::raw r[kSlots];
      if (d_w) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
          if (at[j] >= 0) r[j] = reinterpret_cast<const typename P::raw*>(y + at[j] * H)[c];
      }
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (at[j] < 0) continue;
        float v[P::n];
        if (d_w) {
          P::unpack(r[j], v);
#pragma unroll
          for (int i = 0; i < P::n; ++i) dot[j] = fmaf(v[i], g[i], dot[j]);
        }
        if (d_y) {
#pragma unroll
          for (int i = 0; i < P::n; ++i) v[i] = weight[j] * g[i];
          reinterpret_cast<typename P::raw*>(d_y + at[j] * H)[c] = P::pack(v);
        }
      }
    }
    if (d_w) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
        if (lane == 0) part[first_warp + (threadIdx.x >> 5)][j] = dot[j];
      }
      __syncthreads();
      if (mine && threadIdx.x < kSlots && s0 + (int)threadIdx.x < topk) {
        float sum = 0.0f;
        for (int k = 0; k < warps; ++k) sum += part[first_warp + k][threadIdx.x];
        d_w[t * topk + s0 + threadIdx.x] = sum;
      }
      __syncthreads();
    }
  }
  if (d_y) {
    for (int64_t j = max(*live, 0) + t; j < tokens * topk; j += (int64_t)gridDim.x * blockDim.y) {
      typename P::raw* to = reinterpret_cast<typename P::raw*>(d_y + j * H);
      for (int c = threadIdx.x; c < vecs; c += blockDim.x) to[c] = typename P::raw{};
    }
  }
}

// Lanes of a token: whole warps, no more than the row has vectors, up to all `threads` of a CTA.
dim3 token_block(int vecs, unsigned threads) {
  unsigned x = 32;
  while (x < threads && x < (unsigned)vecs) x *= 2;
  return dim3(x, threads / x);
}

int check_sorted(const void* place, int64_t T, int64_t topk, int64_t H) {
  GB_REQUIRE(T >= 0 && topk >= 1 && topk <= 4096 && H > 0 && H < (1ll << 29), "bad shape T=%lld topk=%lld H=%lld", (long long)T, (long long)topk,
             (long long)H);
  GB_REQUIRE(T * topk < (1ll << 30), "too many routed pairs");
  GB_REQUIRE(T == 0 || place, "null pointer argument");
  return GB_OK;
}

}  // namespace

extern "C" {

int gb_fp8_quantize_blocks(const void* x, int dtype, int64_t ld, int64_t M, int64_t K, int scale_rule, void* q, float* scale, void* stream) {
  QuantizeParams p = {};
  p.x = x; p.ld = ld; p.rows = M; p.K = K; p.scale_rule = scale_rule; p.q = (uint8_t*)q; p.scale = scale;
  return quantize<kRows>(p, dtype, (cudaStream_t)stream);
}

int gb_moe_swiglu_fp8(const void* h, int dtype, int64_t ld, const int32_t* live, int64_t P, int64_t inter, int scale_rule, void* q, float* scale,
                      void* stream) {
  QuantizeParams p = {};
  p.x = h; p.ld = ld; p.rows = P; p.K = inter; p.scale_rule = scale_rule; p.q = (uint8_t*)q; p.scale = scale; p.live = live;
  return quantize<kSwiglu>(p, dtype, (cudaStream_t)stream);
}

int gb_moe_permute_fp8(const void* x, int dtype, int64_t ld, const int32_t* place, const int32_t* live, int64_t T, int64_t topk, int64_t K,
                       int scale_rule, void* q, float* scale, void* stream) {
  const int rc = check_sorted(place, T, topk, K);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(T == 0 || live, "null pointer argument");
  QuantizeParams p = {};
  p.x = x; p.ld = ld; p.rows = T; p.K = K; p.scale_rule = scale_rule; p.q = (uint8_t*)q; p.scale = scale;
  p.place = place; p.live = live; p.topk = (int)topk;
  return quantize<kSorted>(p, dtype, (cudaStream_t)stream);
}

int gb_moe_sort_applies(int64_t P, int64_t E) { return P >= 1 && P <= (int64_t)kSortMostCtas * kSortThreads * kSortMostPer && E >= 1 && E <= kSortExperts; }

int gb_moe_sort(const void* ids, int id_bytes, int64_t P, int64_t E, int64_t expert_base, int32_t* counts, int32_t* offsets, int32_t* order,
                int32_t* place, void* stream) {
  GB_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids of %d bytes", id_bytes);
  if (!gb_moe_sort_applies(P, E)) return gb_fail(GB_EUNSUPPORTED, "%lld pairs of %lld experts: gb_moe_route_inv sorts them", (long long)P, (long long)E);
  GB_REQUIRE(ids && counts && offsets && order && place, "null pointer argument");
  if (id_bytes == 8) return launch_sort<int64_t>(ids, (int)P, (int)E, expert_base, counts, offsets, order, place, (cudaStream_t)stream);
  return launch_sort<int32_t>(ids, (int)P, (int)E, expert_base, counts, offsets, order, place, (cudaStream_t)stream);
}

int gb_moe_permute(const void* x, int64_t elem_bytes, int64_t ld, const int32_t* place, const int32_t* live, int64_t T, int64_t topk, int64_t H,
                   void* rows, void* stream) {
  const int rc = check_sorted(place, T, topk, H);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(elem_bytes == 2 || elem_bytes == 4, "elements of %lld bytes", (long long)elem_bytes);
  GB_REQUIRE(ld >= H || T <= 1, "row stride %lld is shorter than the row", (long long)ld);
  if (T == 0) return GB_OK;
  GB_REQUIRE(x && live && rows, "null pointer argument");
  const int64_t bytes = H * elem_bytes, pitch = ld * elem_bytes;
  const uintptr_t all = (uintptr_t)x | (uintptr_t)rows | (uintptr_t)bytes | (uintptr_t)pitch;
  GB_REQUIRE(all % elem_bytes == 0, "misaligned pointer");
#define GB_PERMUTE(V)                                                                                                                \
  do {                                                                                                                               \
    const dim3 block = token_block((int)(bytes / (int64_t)sizeof(V)), 256);                                                               \
    GB_CUDA_OK(gb_launch(permute_kernel<V>, dim3((unsigned)((T + block.y - 1) / block.y)), block, 0, (cudaStream_t)stream,           \
                         (const uint8_t*)x, pitch, place, live, T, (int)topk, (int)(bytes / (int64_t)sizeof(V)), (uint8_t*)rows));   \
  } while (0)
  if (all % 16 == 0) GB_PERMUTE(uint4);
  else if (all % 4 == 0) GB_PERMUTE(uint32_t);
  else GB_PERMUTE(uint16_t);
#undef GB_PERMUTE
  return GB_OK;
}

int gb_moe_unpermute(const void* y, int dtype, const int32_t* place, const float* weights, int64_t T, int64_t topk, int64_t H, void* out,
                     void* stream) {
  const int rc = check_sorted(place, T, topk, H);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(dtype >= GB_DTYPE_BF16 && dtype <= GB_DTYPE_FP32, "unknown dtype %d", dtype);
  if (T == 0) return GB_OK;
  GB_REQUIRE(y && out, "null pointer argument");
  const int eb = elem_bytes(dtype), per = 16 / eb;
  const uintptr_t all = (uintptr_t)y | (uintptr_t)out;
  GB_REQUIRE(all % eb == 0, "misaligned pointer");
  const bool vec = H % per == 0 && all % 16 == 0;
  const int vecs = (int)(vec ? H / per : H);
  const dim3 block = token_block(vecs, 256), grid((unsigned)((T + block.y - 1) / block.y));
#define GB_UNPERMUTE(D, V)                                                                                                         \
  GB_CUDA_OK(gb_launch(unpermute_kernel<D, V>, grid, block, 0, (cudaStream_t)stream, (const D::word*)y, place, weights, T, (int)topk, vecs, \
                       (D::word*)out))
  if (dtype == GB_DTYPE_BF16) { if (vec) GB_UNPERMUTE(Bf16, true); else GB_UNPERMUTE(Bf16, false); }
  else if (dtype == GB_DTYPE_FP16) { if (vec) GB_UNPERMUTE(Fp16, true); else GB_UNPERMUTE(Fp16, false); }
  else { if (vec) GB_UNPERMUTE(Fp32, true); else GB_UNPERMUTE(Fp32, false); }
#undef GB_UNPERMUTE
  return GB_OK;
}

int gb_moe_unpermute_grad(const void* d_out, const void* y, int dtype, const int32_t* place, const int32_t* live, const float* weights, int64_t T,
                          int64_t topk, int64_t H, void* d_y, float* d_w, void* stream) {
  const int rc = check_sorted(place, T, topk, H);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(dtype >= GB_DTYPE_BF16 && dtype <= GB_DTYPE_FP32, "unknown dtype %d", dtype);
  if (T == 0 || (!d_y && !d_w)) return GB_OK;
  GB_REQUIRE(d_out && live && weights && (y || !d_w), "null pointer argument");
  const int eb = elem_bytes(dtype), per = 16 / eb;
  const uintptr_t all = (uintptr_t)d_out | (uintptr_t)(d_w ? y : nullptr) | (uintptr_t)d_y;
  GB_REQUIRE(all % eb == 0, "misaligned pointer");
  const bool vec = H % per == 0 && all % 16 == 0;
  const int vecs = (int)(vec ? H / per : H);
  const dim3 block = token_block(vecs, 128), grid((unsigned)((T + block.y - 1) / block.y));
#define GB_GRAD(D, V, S)                                                                                                                    \
  GB_CUDA_OK(gb_launch(unpermute_grad_kernel<D, V, S>, grid, block, 0, (cudaStream_t)stream, (const D::word*)d_out, (const D::word*)y, place, live, \
                       weights, T, (int)topk, vecs, (D::word*)d_y, d_w))
#define GB_GRAD_SLOTS(D, V) do { if (topk > 2) GB_GRAD(D, V, 4); else GB_GRAD(D, V, 2); } while (0)
  if (dtype == GB_DTYPE_BF16) { if (vec) GB_GRAD_SLOTS(Bf16, true); else GB_GRAD_SLOTS(Bf16, false); }
  else if (dtype == GB_DTYPE_FP16) { if (vec) GB_GRAD_SLOTS(Fp16, true); else GB_GRAD_SLOTS(Fp16, false); }
  else { if (vec) GB_GRAD_SLOTS(Fp32, true); else GB_GRAD_SLOTS(Fp32, false); }
#undef GB_GRAD_SLOTS
#undef GB_GRAD
  return GB_OK;
}

}  // extern "C"
