// The router of a routed layer: its choice of experts with the weights' gradient, and the loss that balances the experts with their
// counts and its gradient.
//
// Choice.  Of the row of logits l, the topk largest, ties to the lowest expert, NaN above all; an expert at -inf is never chosen, and slots
// without an expert get id -1 and weight 0, which is what the sort by expert drops.  Scores c are softmax(l) or sigmoid(l), both
// rising in l, so that the logits are compared as they are given and no rounding of an exponential decides between two experts.
//     w_j = scale c_j / sum over the chosen of c   (or scale c_j)
//     softmax, renormalised:  q = w / scale;   dl_j = scale q_j (dw_j - sum q dw)
//     softmax:                dl_e = c_e (scale dw_e - sum over the chosen of scale dw c),  dw_e = 0 for the others
//     sigmoid, renormalised:  q = w / scale;   dl_j = scale q_j (dw_j - sum q dw) (1 - c_j)
//     sigmoid:                dl_j = scale dw_j c_j (1 - c_j)
// Balance.  Over the n tokens that count (the mask's, and with a logit above -inf), p = softmax(l) and z = log sum exp l,
//     f_e = counts_e / (n topk),  P_e = sum p_e / n,   loss = coef E sum f P + z_coef sum z^2 / n
//     dl_te = d_loss / n p_te (coef E (f_e - sum f p_t) + 2 z_coef z_t)
//
// A warp takes a token, its logits in registers; for the loss a block takes one past 1024 experts, the choice and its gradient keep to a warp
// with up to 128 logits a lane.  Sums over tokens are fp32: a lane's own,
// then the block's warps, then the blocks, each in a fixed order; counts are whole numbers, added in any order.
//
// The loss is bound by instructions (one exponential and some ten others a logit) and by waits for the row, the choice by the chain of its reductions, one
// expert behind the other, neither by memory.  256 experts, measured in a stream of calls: the choice of 8192 fp32
// rows 9.3 us and its gradient 4.0 (2.7 for the bytes of both); the loss of 65536 bf16 rows 28 with the join (22 and 10, overlapping), its gradient 21 (10.6); cold,
// under the profiler, 31, 14 and 28, issue slots 56 to 63 % taken; one token's choice 5.5 from the caller's side, which is the launch.  Choices of 4096 bf16 rows, top-8: of 2048
// experts 52, of 4096 57 (as softmax without renormalising 76 and 86), their gradients 6 to 11 (34 and 37).
#include "gb_blocks.cuh"

namespace {

using namespace gb_blocks;

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kMostExperts = 4096, kMostTopk = 32;

GB_DEVINL float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
GB_DEVINL float warp_max(float v) {                        // a NaN wins
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kAll));
  return r;
}
// Two sums at once: after the first exchange the lower half warp adds up the one and the upper half the other.
GB_DEVINL void warp_sums(float& a, float& b) {
  const bool up = threadIdx.x & 16;
  float v = (up ? b : a) + __shfl_xor_sync(kAll, up ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  a = __shfl_sync(kAll, v, 0);
  b = __shfl_sync(kAll, v, 16);
}
// e^(v - top), two roundings of the exponent and two units of the function; results below 2^-126 are zero, next to the largest term's one.  The difference
// comes first: top log2 e rounded by itself is off by as much as the exponents are for logits far from zero, and passes fp32 for those
// at the end of its range.  (expf's ten instructions for each expert were half of the loss's.)
constexpr float kLog2e = 1.4426950408889634f;
GB_DEVINL float exp_from(float v, float top) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((v - top) * kLog2e));
  return r;
}

// Whole numbers in the order of the logits, zeros alike; 0: no expert or one at -inf, NaN on top.
GB_DEVINL uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return kAll;
  return b == 0xFF800000u ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}
GB_DEVINL float of_key(uint32_t k) {
  if (k == 0u) return -__int_as_float(0x7F800000);
  return k == kAll ? __int_as_float(0x7FC00000) : __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k);
}

// A row's values over kGroup threads, kPer each: pieces of kV neighbours (16 bytes, or what kPer takes) where kVec, else single ones.
template <typename T, int kPer, bool kVec, int kGroup = 32>
struct Row {
  using word = typename T::word;
  static constexpr int kMostV = 16 / (int)sizeof(word), kV = !kVec ? 1 : kPer < kMostV ? kPer : kMostV;
  static GB_DEVINL int expert(int i, int lane) { return ((i / kV) * kGroup + lane) * kV + i % kV; }
  static GB_DEVINL void load(const word* row, int E, int lane, float (&v)[kPer], float otherwise) {
#pragma unroll
    for (int i = 0; i < kPer; i += kV) {
      const int e = expert(i, lane);
      alignas(16) word w[kV];
      if constexpr (kV == 1) {
        if (e < E) w[0] = row[e];
      } else if (e < E) {
        if constexpr (kV * sizeof(word) == 16) *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(row + e));
        else *reinterpret_cast<uint2*>(w) = __ldg(reinterpret_cast<const uint2*>(row + e));
      }
#pragma unroll
      for (int j = 0; j < kV; ++j) v[i + j] = e < E ? to_f32<T>(w[j]) : otherwise;
    }
  }
  // The same in two steps: on their way, and as fp32.
  struct Raw { alignas(16) word w[kPer]; };
  static GB_DEVINL Raw fetch(const word* row, int E, int lane) {
    Raw r;
#pragma unroll
    for (int i = 0; i < kPer; i += kV) {
      const int e = expert(i, lane);
      if (e >= E) continue;
      if constexpr (kV == 1) r.w[i] = row[e];
      else if constexpr (kV * sizeof(word) == 16) *reinterpret_cast<uint4*>(r.w + i) = __ldg(reinterpret_cast<const uint4*>(row + e));
      else *reinterpret_cast<uint2*>(r.w + i) = __ldg(reinterpret_cast<const uint2*>(row + e));
    }
    return r;
  }
  static GB_DEVINL void unpack(const Raw& r, int E, int lane, float (&v)[kPer], float otherwise) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = expert(i, lane) < E ? to_f32<T>(r.w[i]) : otherwise;
  }
  static GB_DEVINL void store(word* row, int E, int lane, const float (&v)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; i += kV) {
      const int e = expert(i, lane);
      if (e >= E) continue;
      alignas(16) word w[kV];
      if constexpr (kV > 1 && std::is_same_v<T, Bf16>) {
#pragma unroll
        for (int j = 0; j < kV; j += 2) *reinterpret_cast<uint32_t*>(w + j) = gb_pack_bf16x2(v[i + j], v[i + j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j) w[j] = from_f32<T>(v[i + j]);
      }
      if constexpr (kV == 1) row[e] = w[0];
      else if constexpr (kV * sizeof(word) == 16) *reinterpret_cast<uint4*>(row + e) = *reinterpret_cast<uint4*>(w);
      else *reinterpret_cast<uint2*>(row + e) = *reinterpret_cast<uint2*>(w);
    }
  }
};

// ------------------------------------------------------------------------------------------------ choice
struct TopkParams {
  const void* logits;
  int64_t ld, T;
  int E, topk, sigmoid, renormalize;
  float scale;
  float* weights;
  int32_t* ids;
  const float* d_weights;
  void* d_logits;
};

constexpr int kTopkThreads = 128;

template <typename T, int kPer, bool kVec>
__global__ void __launch_bounds__(kTopkThreads)
topk_kernel(const __grid_constant__ TopkParams p) {
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * (kTopkThreads / 32) + (threadIdx.x >> 5);
  if (t >= p.T) return;
  using R = Row<T, kPer, kVec>;
  uint32_t key[kPer];
  {
    float v[kPer];
    R::load(static_cast<const typename T::word*>(p.logits) + t * p.ld, p.E, lane, v, -__int_as_float(0x7F800000));
#pragma unroll
    for (int i = 0; i < kPer; ++i) key[i] = key_of(v[i]);
  }
  uint32_t best = 0u;
  int at = 0;
  auto rank = [&]() {                                      // the lane's largest, the first of equals
    best = 0u;
    at = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
  };
  rank();
  const float top = of_key(__reduce_max_sync(kAll, best));
  float total = 0.0f;
  if (!p.sigmoid && !p.renormalize) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) total += key[i] ? expf(of_key(key[i]) - top) : 0.0f;
    total = warp_sum(total);
  }
  uint32_t mine = 0u;                                      // lane j: the j-th choice
  int id = -1;
  for (int j = 0; j < p.topk; ++j) {
    const uint32_t m = __reduce_max_sync(kAll, best);
    if (m == 0u) break;
    const int e = R::expert(at, lane), first = __reduce_min_sync(kAll, best == m ? e : 0x7FFFFFFF);
    if (lane == j) { mine = m; id = first; }
    if (best == m && e == first) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == at) key[i] = 0u;
      rank();
    }
  }
  const float l = of_key(mine);
  float c = 0.0f;
  if (id >= 0) c = p.sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - top);
  if (p.renormalize) total = warp_sum(c);
  else if (p.sigmoid) total = 1.0f;
  if (lane < p.topk) {
    p.ids[t * p.topk + lane] = id;
    p.weights[t * p.topk + lane] = id < 0 || total == 0.0f ? 0.0f : c / total * p.scale;
  }
}

template <typename T, int kPer, bool kVec>
__global__ void __launch_bounds__(kTopkThreads)
topk_grad_kernel(const __grid_constant__ TopkParams p) {
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * (kTopkThreads / 32) + (threadIdx.x >> 5);
  if (t >= p.T) return;
  using R = Row<T, kPer, kVec>;
  using word = typename T::word;
  const word* logits = static_cast<const word*>(p.logits) + t * p.ld;
  word* out = static_cast<word*>(p.d_logits) + t * p.E;
  int id = lane < p.topk ? p.ids[t * p.topk + lane] : -1;
  if (id >= p.E) id = -1;
  const float dw = id >= 0 ? p.d_weights[t * p.topk + lane] * p.scale : 0.0f;
  const float l = id >= 0 ? to_f32<T>(logits[id]) : 0.0f;
  float dense[kPer], mine = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) dense[i] = 0.0f;
  if (p.sigmoid) {
    const float c = id >= 0 ? 1.0f / (1.0f + expf(-l)) : 0.0f, rest = 1.0f / (1.0f + expf(l));
    if (p.renormalize) {                                   // shares first: dw over a sum of small scores may pass fp32, and is multiplied by them again
      const float total = warp_sum(c), q = total == 0.0f ? 0.0f : c / total, dot = warp_sum(q * dw);
      mine = q * (dw - dot) * rest;
    } else {
      mine = dw * c * rest;
    }
  } else {
    const float top = warp_max(id >= 0 ? l : -__int_as_float(0x7F800000));
    const float e = id >= 0 ? expf(l - top) : 0.0f;
    if (p.renormalize) {
      const float total = warp_sum(e), q = total == 0.0f ? 0.0f : e / total, dot = warp_sum(q * dw);
      mine = q * (dw - dot);
    } else {
      float v[kPer], total = 0.0f;
      R::load(logits, p.E, lane, v, -__int_as_float(0x7F800000));
      const bool none = top == -__int_as_float(0x7F800000);      // no expert was chosen: no logit above -inf
#pragma unroll
      for (int i = 0; i < kPer; ++i) { v[i] = none ? 0.0f : expf(v[i] - top); total += v[i]; }
      total = warp_sum(total);
      const float r = none ? 0.0f : 1.0f / total, q = e * r, dot = warp_sum(q * dw);
#pragma unroll
      for (int i = 0; i < kPer; ++i) dense[i] = -(v[i] * r) * dot;
      mine = q * (dw - dot);
    }
  }
  R::store(out, p.E, lane, dense);
  __syncwarp();                                            // the chosen experts' values go on top
  if (id >= 0) out[id] = from_f32<T>(mine);
}

// ------------------------------------------------------------------------------------------------ balance
struct BalanceParams {
  const void* logits;
  int64_t ld, T;
  int E, topk, id_bytes;
  const void* ids;
  const uint8_t* mask;
  float coef, z_coef;
  float* loss;
  int32_t* counts;
  float* stats;               // [E + 1]: the experts' shares f, then how many tokens count
  int blocks;
  float* part_p;              // [blocks][E] sums of p
  int32_t* part_c;            // [blocks][E] counts
  float* part_z;              // [blocks] sums of z^2
  int32_t* part_n;            // [blocks] tokens that count
  const float* d_loss;
  void* d_logits;
};

template <int kPer>
struct Balance { static constexpr int kThreads = kPer > 16 ? 512 : 1024; };

// Maximum or sum over a token's threads: a warp, or the whole block (every thread calls it).
template <int kGroup, bool kMax>
GB_DEVINL float over_token(float v, float* s) {
  v = kMax ? warp_max(v) : warp_sum(v);
  if constexpr (kGroup > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) s[warp] = v;
    __syncthreads();
    v = lane < kGroup / 32 ? s[lane] : kMax ? -__int_as_float(0x7F800000) : 0.0f;
    v = kMax ? warp_max(v) : warp_sum(v);
  }
  return v;
}

template <typename T, int kPer, bool kVec, int kGroup>
__global__ void __launch_bounds__((kGroup > 32 ? kGroup : Balance<kPer>::kThreads), 1)
balance_kernel(const __grid_constant__ BalanceParams p) {
  constexpr int kThreads = kGroup > 32 ? kGroup : Balance<kPer>::kThreads, kGroups = kThreads / kGroup;
  extern __shared__ float smem[];                          // [E] counts, then [min(groups, 8)][E] sums
  __shared__ float s_red[32], s_z[kGroups];
  __shared__ int s_n[kGroups];
  int* s_counts = reinterpret_cast<int*>(smem);
  float* s_p = smem + p.E;
  gb_pdl_launch_dependents();
  for (int e = threadIdx.x; e < p.E; e += kThreads) s_counts[e] = 0;
  gb_pdl_wait();
  __syncthreads();
  using R = Row<T, kPer, kVec, kGroup>;
  const int group = threadIdx.x / kGroup, lane = threadIdx.x % kGroup;
  const float inf = __int_as_float(0x7F800000);
  float acc[kPer], z2 = 0.0f;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.0f;
  // the next token's logits and ids are on their way while this one's are looked at
  const int64_t step = (int64_t)p.blocks * kGroups;
  const auto row = [&](int64_t t) { return static_cast<const typename T::word*>(p.logits) + t * p.ld; };
  const auto live = [&](int64_t t) { return t < p.T && (!p.mask || p.mask[t]); };
  const auto id_of = [&](int64_t t, int j) -> int64_t {
    return p.id_bytes == 8 ? static_cast<const int64_t*>(p.ids)[t * p.topk + j] : static_cast<const int32_t*>(p.ids)[t * p.topk + j];
  };
  int64_t t = (int64_t)blockIdx.x * kGroups + group;
  bool on = live(t);
  typename R::Raw next = {};
  int64_t next_id = -1;
  if (on) {
    next = R::fetch(row(t), p.E, lane);
    if (lane < p.topk) next_id = id_of(t, lane);
  }
  for (; t < p.T; t += step) {
    float v[kPer], top = -inf, total = 0.0f;
    const bool counts = on;
    const int64_t id = next_id;
    R::unpack(next, p.E, lane, v, -inf);
    on = live(t + step);
    if (on) {
      next = R::fetch(row(t + step), p.E, lane);
      if (lane < p.topk) next_id = id_of(t + step, lane);
    }
    if (!counts) continue;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = max_nan(top, v[i]);
    top = over_token<kGroup, true>(top, s_red);
    if (top == -inf) continue;                             // nothing to choose from
#pragma unroll
    for (int i = 0; i < kPer; ++i) { v[i] = exp_from(v[i], top); total += v[i]; }
    total = over_token<kGroup, false>(total, s_red);
    const float r = 1.0f / total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = fmaf(v[i], r, acc[i]);
    if (p.z_coef != 0.0f) {                                // without a z-loss no square of it, which may pass fp32
      const float z = top + logf(total);
      z2 = fmaf(z, z, z2);
    }
    ++n;
    if (lane < p.topk && (uint64_t)id < (uint64_t)p.E) atomicAdd(&s_counts[id], 1);
    for (int j = lane + kGroup; j < p.topk; j += kGroup) {
      const int64_t e = id_of(t, j);
      if ((uint64_t)e < (uint64_t)p.E) atomicAdd(&s_counts[e], 1);
    }
  }
  if (lane == 0) { s_z[group] = z2; s_n[group] = n; }
  // the groups' sums, eight groups at a time, in their order
  for (int g0 = 0; g0 < kGroups; g0 += 8) {
    if (group >= g0 && group < g0 + 8) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = R::expert(i, lane);
        if (e < p.E) s_p[(group - g0) * p.E + e] = acc[i];
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += kThreads) {
      float s = g0 == 0 ? 0.0f : p.part_p[(int64_t)blockIdx.x * p.E + e];
      for (int g = 0; g < min(8, kGroups - g0); ++g) s += s_p[g * p.E + e];
      p.part_p[(int64_t)blockIdx.x * p.E + e] = s;
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < p.E; e += kThreads) p.part_c[(int64_t)blockIdx.x * p.E + e] = s_counts[e];
  if (threadIdx.x == 0) {
    float z = 0.0f;
    int m = 0;
    for (int g = 0; g < kGroups; ++g) { z += s_z[g]; m += s_n[g]; }
    p.part_z[blockIdx.x] = z;
    p.part_n[blockIdx.x] = m;
  }
}

constexpr int kJoinThreads = 1024;

// The blocks' sums in one block: thread (g, e) adds every kJoinThreads / E-th block's.
__global__ void __launch_bounds__(kJoinThreads, 1)
balance_join_kernel(const __grid_constant__ BalanceParams p) {
  __shared__ float s_p[kJoinThreads], s_red[32];
  __shared__ int s_c[kJoinThreads], s_n[32];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float z = 0.0f;
  int n = 0;
  for (int b = tid; b < p.blocks; b += kJoinThreads) { z += p.part_z[b]; n += p.part_n[b]; }
  z = warp_sum(z);
  n = __reduce_add_sync(kAll, n);
  if (lane == 0) { s_red[warp] = z; s_n[warp] = n; }
  __syncthreads();
  z = warp_sum(s_red[lane]);
  n = __reduce_add_sync(kAll, s_n[lane]);
  __syncthreads();
  const float tokens = (float)max(n, 1), share = 1.0f / (tokens * (float)p.topk);
  const int wide = min(p.E, kJoinThreads), groups = kJoinThreads / wide, g = tid / wide;
  float fp = 0.0f;
  for (int e0 = 0; e0 < p.E; e0 += wide) {
    const int e = e0 + tid % wide;
    float s = 0.0f;
    int c = 0;
    if (g < groups && e < p.E)
      for (int b = g; b < p.blocks; b += groups) {
        s += p.part_p[(int64_t)b * p.E + e];
        c += p.part_c[(int64_t)b * p.E + e];
      }
    s_p[tid] = s;
    s_c[tid] = c;
    __syncthreads();
    if (g == 0 && e < p.E) {
      for (int i = 1; i < groups; ++i) { s += s_p[i * wide + tid]; c += s_c[i * wide + tid]; }
      const float f = (float)c * share;
      p.counts[e] = c;
      p.stats[e] = f;
      fp = fmaf(f, s / tokens, fp);
    }
    __syncthreads();
  }
  fp = warp_sum(fp);
  if (lane == 0) s_red[warp] = fp;
  __syncthreads();
  if (warp == 0) {
    fp = warp_sum(s_red[lane]);
    if (lane == 0) {
      p.stats[p.E] = (float)n;
      *p.loss = n == 0 ? 0.0f : p.coef * (float)p.E * fp + p.z_coef * (z / tokens);
    }
  }
}

// A group of threads takes one token behind the other, the next one's logits on their way; the experts' shares stay in its registers.
template <typename T, int kPer, bool kVec, int kGroup>
__global__ void __launch_bounds__(256)
balance_grad_kernel(const __grid_constant__ BalanceParams p) {
  constexpr int kGroups = 256 / kGroup;
  __shared__ float s_red[32];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  using R = Row<T, kPer, kVec, kGroup>;
  using word = typename T::word;
  const int group = threadIdx.x / kGroup, lane = threadIdx.x % kGroup;
  const float inf = __int_as_float(0x7F800000);
  const int64_t step = (int64_t)gridDim.x * kGroups;
  const auto live = [&](int64_t t) { return t < p.T && (!p.mask || p.mask[t]); };
  const auto row = [&](int64_t t) { return static_cast<const word*>(p.logits) + t * p.ld; };
  int64_t t = (int64_t)blockIdx.x * kGroups + group;
  bool on = live(t);
  typename R::Raw next = {};
  if (on) next = R::fetch(row(t), p.E, lane);
  float f[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = R::expert(i, lane);
    f[i] = e < p.E ? __ldg(p.stats + e) : 0.0f;
  }
  const float scale = *p.d_loss / fmaxf(__ldg(p.stats + p.E), 1.0f), b = p.coef * (float)p.E;
  for (; t < p.T; t += step) {
    float v[kPer], top = -inf, total = 0.0f, dot = 0.0f;
    const bool counts = on;
    R::unpack(next, p.E, lane, v, -inf);
    on = live(t + step);
    if (on) next = R::fetch(row(t + step), p.E, lane);
    if (counts) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) top = max_nan(top, v[i]);
      top = over_token<kGroup, true>(top, s_red);
    }
    if (top == -inf) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) { v[i] = exp_from(v[i], top); total += v[i]; dot = fmaf(v[i], f[i], dot); }
      if constexpr (kGroup == 32) {
        warp_sums(total, dot);
      } else {
        total = over_token<kGroup, false>(total, s_red);
        dot = over_token<kGroup, false>(dot, s_red);
      }
      const float r = 1.0f / total, z = top + logf(total), a = scale * r;
      dot *= r;
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] = a * v[i] * fmaf(b, f[i] - dot, 2.0f * p.z_coef * z);
    }
    R::store(static_cast<word*>(p.d_logits) + t * p.E, p.E, lane, v);
  }
}

// ------------------------------------------------------------------------------------------------ host
bool pieces(const void* a, int64_t ld, int64_t E, int size, int bytes) {   // rows of whole pieces of `bytes`
  return ((uintptr_t)a % bytes) == 0 && (ld * size) % bytes == 0 && (E * size) % bytes == 0;
}

// Calls go(T, values a thread, whether rows come in whole pieces) for a row type and a number of experts.
template <int kGroupPast, typename Go>
int dispatch(int dtype, int64_t E, const void* a, int64_t lda, const void* b, int64_t ldb, Go go) {
  const int size = dtype == GB_DTYPE_FP32 ? 4 : 2, per = E <= 128 ? 4 : 8;
  const int bytes = per * size < 16 ? per * size : 16;
  const bool vec = pieces(a, lda, E, size, bytes) && (!b || pieces(b, ldb, E, size, bytes));
  auto of_type = [&](auto t) {
    auto of_vec = [&](auto v) {
      if (E <= 128) return go(t, std::integral_constant<int, 4>(), v, std::integral_constant<int, 32>());
      if (E <= 256) return go(t, std::integral_constant<int, 8>(), v, std::integral_constant<int, 32>());
      if (E <= 512) return go(t, std::integral_constant<int, 16>(), v, std::integral_constant<int, 32>());
      if (E <= 1024) return go(t, std::integral_constant<int, 32>(), v, std::integral_constant<int, 32>());
      return go(t, std::integral_constant<int, kMostExperts / kGroupPast>(), v, std::integral_constant<int, kGroupPast>());
    };
    return vec ? of_vec(std::true_type()) : of_vec(std::false_type());
  };
  if (dtype == GB_DTYPE_BF16) return of_type(Bf16());
  if (dtype == GB_DTYPE_FP16) return of_type(Fp16());
  return of_type(Fp32());
}

int check_logits(const void* logits, int dtype, int64_t ld, int64_t T, int64_t E) {
  GB_REQUIRE(dtype >= GB_DTYPE_BF16 && dtype <= GB_DTYPE_FP32, "unknown element type %d", dtype);
  GB_REQUIRE(E >= 1 && E <= kMostExperts, "%lld experts: 1 to %d expected", (long long)E, kMostExperts);
  GB_REQUIRE(T >= 0 && T < (1ll << 31), "%lld tokens: fewer than 2^31 expected", (long long)T);
  GB_REQUIRE(T == 0 || (logits && ld >= E), "rows of logits that do not overlap expected");
  GB_REQUIRE(((uintptr_t)logits % (dtype == GB_DTYPE_FP32 ? 4 : 2)) == 0, "logits: an address of whole elements expected");
  return GB_OK;
}

int balance_blocks(int64_t T, int64_t E) {
  const int64_t sms = gb_sm_count(), tokens = E > 1024 ? 1 : E > 512 ? 16 : 32;
  const int64_t want = (T + tokens - 1) / tokens;
  return (int)(want < 1 ? 1 : want < sms ? want : sms);
}

struct BalanceSpace { int64_t c, z, n, bytes; };
BalanceSpace balance_space(int blocks, int64_t E) {
  auto up = [](int64_t v) { return (v + 255) & ~(int64_t)255; };
  BalanceSpace s;
  s.c = up(blocks * E * 4);
  s.z = s.c + up(blocks * E * 4);
  s.n = s.z + up(blocks * 4);
  s.bytes = s.n + up(blocks * 4);
  return s;
}

}  // namespace

extern "C" {

int gb_moe_topk(const void* logits, int dtype, int64_t ld, int64_t T, int64_t E, int64_t topk, int sigmoid, int renormalize, float scale, float* weights,
                int32_t* ids, void* stream) {
  const int rc = check_logits(logits, dtype, ld, T, E);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(topk >= 1 && topk <= kMostTopk && topk <= E, "top-%lld of %lld experts: 1 to %d, and no more than there are, expected", (long long)topk,
             (long long)E, kMostTopk);
  if (T == 0) return GB_OK;
  GB_REQUIRE(weights && ids, "null pointer argument");
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  TopkParams p = {};
  p.logits = logits; p.ld = ld; p.T = T; p.E = (int)E; p.topk = (int)topk;
  p.sigmoid = sigmoid; p.renormalize = renormalize; p.scale = scale;
  p.weights = weights; p.ids = ids;
  return dispatch<32>(dtype, E, logits, ld, nullptr, 0, [&](auto t, auto per, auto vec, auto) -> int {
    const unsigned blocks = (unsigned)((T + kTopkThreads / 32 - 1) / (kTopkThreads / 32));
    GB_CUDA_OK(gb_launch(topk_kernel<decltype(t), decltype(per)::value, decltype(vec)::value>, dim3(blocks), dim3(kTopkThreads), 0, (cudaStream_t)stream, p));
    return GB_OK;
  });
}

int gb_moe_topk_grad(const void* logits, int dtype, int64_t ld, const int32_t* ids, const float* d_weights, int64_t T, int64_t E, int64_t topk, int sigmoid,
                     int renormalize, float scale, void* d_logits, void* stream) {
  const int rc = check_logits(logits, dtype, ld, T, E);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(topk >= 1 && topk <= kMostTopk && topk <= E, "top-%lld of %lld experts: 1 to %d, and no more than there are, expected", (long long)topk,
             (long long)E, kMostTopk);
  if (T == 0) return GB_OK;
  GB_REQUIRE(ids && d_weights && d_logits, "null pointer argument");
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  TopkParams p = {};
  p.logits = logits; p.ld = ld; p.T = T; p.E = (int)E; p.topk = (int)topk;
  p.sigmoid = sigmoid; p.renormalize = renormalize; p.scale = scale;
  p.ids = const_cast<int32_t*>(ids); p.d_weights = d_weights; p.d_logits = d_logits;
  return dispatch<32>(dtype, E, logits, ld, d_logits, E, [&](auto t, auto per, auto vec, auto) -> int {
    const unsigned blocks = (unsigned)((T + kTopkThreads / 32 - 1) / (kTopkThreads / 32));
    GB_CUDA_OK(gb_launch(topk_grad_kernel<decltype(t), decltype(per)::value, decltype(vec)::value>, dim3(blocks), dim3(kTopkThreads), 0, (cudaStream_t)stream, p));
    return GB_OK;
  });
}

int64_t gb_moe_balance_workspace_bytes(int64_t T, int64_t E) {
  return T < 1 || E < 1 || E > kMostExperts ? 0 : balance_space(balance_blocks(T, E), E).bytes;
}

int gb_moe_balance(const void* logits, int dtype, int64_t ld, const void* ids, int id_bytes, const uint8_t* mask, int64_t T, int64_t E, int64_t topk, float coef,
                   float z_coef, float* loss, int32_t* counts, float* stats, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_logits(logits, dtype, ld, T, E);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(id_bytes == 4 || id_bytes == 8, "ids of 4 or 8 bytes expected");
  GB_REQUIRE(topk >= 1 && T >= 1 && topk < (1ll << 31) && T * topk < (1ll << 31), "at least one token and one choice, and fewer than 2^31 pairs, expected");
  GB_REQUIRE(ids && loss && counts && stats && workspace, "null pointer argument");
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  BalanceParams p = {};
  p.blocks = balance_blocks(T, E);
  const BalanceSpace space = balance_space(p.blocks, E);
  if (workspace_bytes < space.bytes) return gb_fail(GB_EWORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)space.bytes);
  p.logits = logits; p.ld = ld; p.T = T; p.E = (int)E; p.topk = (int)topk;
  p.ids = ids; p.id_bytes = id_bytes; p.mask = mask;
  p.coef = coef; p.z_coef = z_coef;
  p.loss = loss; p.counts = counts; p.stats = stats;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.part_p = reinterpret_cast<float*>(w);
  p.part_c = reinterpret_cast<int32_t*>(w + space.c);
  p.part_z = reinterpret_cast<float*>(w + space.z);
  p.part_n = reinterpret_cast<int32_t*>(w + space.n);
  return dispatch<256>(dtype, E, logits, ld, nullptr, 0, [&](auto t, auto per, auto vec, auto group) -> int {
    constexpr int kPer = decltype(per)::value, kGroup = decltype(group)::value, kThreads = kGroup > 32 ? kGroup : Balance<kPer>::kThreads;
    constexpr int kSums = kThreads / kGroup < 8 ? kThreads / kGroup : 8;
    const size_t smem = (size_t)(1 + kSums) * (size_t)E * 4;             // at most 36 KB
    GB_CUDA_OK(gb_launch(balance_kernel<decltype(t), kPer, decltype(vec)::value, kGroup>, dim3((unsigned)p.blocks), dim3(kThreads), smem, (cudaStream_t)stream, p));
    GB_CUDA_OK(gb_launch(balance_join_kernel, dim3(1), dim3(kJoinThreads), 0, (cudaStream_t)stream, p));
    return GB_OK;
  });
}

int gb_moe_balance_grad(const void* logits, int dtype, int64_t ld, const uint8_t* mask, const float* stats, const float* d_loss, int64_t T, int64_t E, float coef,
                        float z_coef, void* d_logits, void* stream) {
  const int rc = check_logits(logits, dtype, ld, T, E);
  if (rc != GB_OK) return rc;
  if (T == 0) return GB_OK;
  GB_REQUIRE(stats && d_loss && d_logits, "null pointer argument");
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  BalanceParams p = {};
  p.logits = logits; p.ld = ld; p.T = T; p.E = (int)E;
  p.mask = mask; p.stats = const_cast<float*>(stats);
  p.coef = coef; p.z_coef = z_coef; p.d_loss = d_loss; p.d_logits = d_logits;
  return dispatch<256>(dtype, E, logits, ld, d_logits, E, [&](auto t, auto per, auto vec, auto group) -> int {
    constexpr int kGroup = decltype(group)::value, kGroups = 256 / kGroup;
    const int64_t blocks = (T + kGroups - 1) / kGroups, most = (int64_t)gb_sm_count() * 6;       // about what runs at once
    GB_CUDA_OK(gb_launch(balance_grad_kernel<decltype(t), decltype(per)::value, decltype(vec)::value, kGroup>, dim3((unsigned)(blocks < most ? blocks : most)),
                         dim3(256), 0, (cudaStream_t)stream, p));
    return GB_OK;
  });
}

}  // extern "C"
