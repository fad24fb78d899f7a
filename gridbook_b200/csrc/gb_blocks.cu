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
#include "gb_common.cuh"

namespace {

constexpr int kBlock = 128, kThreads = 256, kHalfWarps = kThreads / 16;
constexpr float kAmaxFloor = 1e-10f;

enum Source { kRows = 0, kSorted = 1, kSwiglu = 2 };

struct Bf16 { using word = uint16_t; };
struct Fp16 { using word = uint16_t; };
struct Fp32 { using word = uint32_t; };

template <typename T>
GB_DEVINL float to_f32(typename T::word w);
template <> GB_DEVINL float to_f32<Bf16>(uint16_t w) { return gb_bf16_bits_to_f32(w); }
template <> GB_DEVINL float to_f32<Fp16>(uint16_t w) { return __half2float(__ushort_as_half(w)); }
template <> GB_DEVINL float to_f32<Fp32>(uint32_t w) { return __uint_as_float(w); }
template <typename T>
GB_DEVINL typename T::word from_f32(float v);
template <> GB_DEVINL uint16_t from_f32<Bf16>(float v) { return (uint16_t)gb_f32_to_bf16_bits(v); }
template <> GB_DEVINL uint16_t from_f32<Fp16>(float v) { return __half_as_ushort(__float2half_rn(v)); }
template <> GB_DEVINL uint32_t from_f32<Fp32>(float v) { return __float_as_uint(v); }

// Sixteen bytes of a row as fp32.
template <typename T>
GB_DEVINL void unpack16(const uint4& q, float* v) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(typename T::word) == 2) {
      v[2 * i] = to_f32<T>((uint16_t)(w[i] & 0xFFFFu));
      v[2 * i + 1] = to_f32<T>((uint16_t)(w[i] >> 16));
    } else {
      v[i] = to_f32<T>(w[i]);
    }
  }
}
template <typename T>
GB_DEVINL uint4 pack16(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(typename T::word) == 2)
      w[i] = (uint32_t)from_f32<T>(v[2 * i]) | (uint32_t)from_f32<T>(v[2 * i + 1]) << 16;
    else
      w[i] = from_f32<T>(v[i]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight consecutive columns from `c` of a row of `K`, zeros past its end.  kVec: rows of whole 16-byte pieces, K a multiple of 8.
template <typename T, bool kVec>
GB_DEVINL void load8(const typename T::word* row, int64_t c, int64_t K, float (&v)[8]) {
  if constexpr (kVec) {
    if (c < K) {
      if constexpr (sizeof(typename T::word) == 2) {
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(row + c)), v);
      } else {
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(row + c)), v);
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(row + c + 4)), v + 4);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f32<T>(row[c + i]) : 0.0f;
  }
}

GB_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The eight values' E4M3 bytes and the block's scale; the sixteen lanes of the block call it together.
GB_DEVINL uint2 quantize8(const float (&v)[8], int scale_rule, float& scale) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  amax = max_nan(amax, kAmaxFloor);
  scale = scale_rule == GB_SCALE_RULE_DIV ? __fdiv_rn(amax, 448.0f) : __fmul_rn(amax, 1.0f / 448.0f);
  uint32_t q[4];
  if (gb_plain_division(scale)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = gb_cvt_e4m3x2(__fdiv_rn(v[2 * i], scale), __fdiv_rn(v[2 * i + 1], scale));
  } else {
    const float rinv = __frcp_rn(scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = gb_cvt_e4m3x2(gb_div(v[2 * i], scale, rinv), gb_div(v[2 * i + 1], scale, rinv));
  }
  return make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
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

struct QuantizeParams {
  const void* x;
  int64_t ld, rows, K;        // of the result; a swiglu row is [gate | up]
  uint32_t blocks;            // of a row
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
  float v[kPer][8];
  int64_t row[kPer];
  uint32_t block[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t unit = ((int64_t)blockIdx.x * kPer + i) * kHalfWarps + half;
    row[i] = unit < p.units ? (int64_t)((uint32_t)unit / p.blocks) : p.rows;
    block[i] = (uint32_t)unit - (uint32_t)row[i] * p.blocks;
    const int64_t c = (int64_t)block[i] * kBlock + lane * 8;
    if (row[i] < rows) {
      const typename T::word* at = x + row[i] * p.ld;
      load8<T, kVec>(at, c, p.K, v[i]);
      if constexpr (kSource == kSwiglu) {
        float up[8];
        load8<T, kVec>(at + p.K, c, p.K, up);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = c + k < p.K ? gb_silu(v[i][k]) * up[k] : 0.0f;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t c = (int64_t)block[i] * kBlock + lane * 8;
    float scale;
    const uint2 q = quantize8(v[i], p.scale_rule, scale);
    if (row[i] >= rows) continue;
    if constexpr (kSource == kSorted) {
      for (int s = 0; s < p.topk; ++s) {
        const int64_t to = p.place[row[i] * p.topk + s];
        if (to < 0) continue;
        store8<kVec>(p.q + to * p.K, c, p.K, q);
        if (lane == 0) p.scale[to * p.blocks + block[i]] = scale;
      }
    } else {
      store8<kVec>(p.q + row[i] * p.K, c, p.K, q);
      if (lane == 0) p.scale[row[i] * p.blocks + block[i]] = scale;
    }
  }
  if constexpr (kSource == kSorted) {      // rows that no pair has read zero
    const int64_t pairs = p.rows * p.topk, first = *p.live, left = (pairs - first) * p.blocks;
    for (int64_t u = (int64_t)blockIdx.x * kHalfWarps + half; u < left; u += (int64_t)gridDim.x * kHalfWarps) {
      const int64_t to = first + u / p.blocks, b = u % p.blocks;
      store8<kVec>(p.q + to * p.K, b * kBlock + lane * 8, p.K, make_uint2(0u, 0u));
      if (lane == 0) p.scale[to * p.blocks + b] = 0.0f;
    }
  }
}

template <typename T, Source kSource>
int launch_quantize(const QuantizeParams& p, bool vec, cudaStream_t stream) {
  // one block each while that leaves SMs idle, four from some waves on
  const int64_t few = 8ll * gb_sm_count() * kHalfWarps;
  const int per = p.units > few ? 4 : 1;
  const dim3 grid((unsigned)((p.units + per * kHalfWarps - 1) / (per * kHalfWarps)));
#define GB_Q(v, n) GB_CUDA_OK(gb_launch(quantize_blocks_kernel<T, kSource, v, n>, grid, dim3(kThreads), 0, stream, p))
  if (vec) { if (per == 4) GB_Q(true, 4); else GB_Q(true, 1); }
  else { if (per == 4) GB_Q(false, 4); else GB_Q(false, 1); }
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
  p.units = p.rows * p.blocks;
  GB_REQUIRE(p.units < (1ll << 31), "too many blocks");
  const int eb = elem_bytes(dtype);
  const bool vec = p.K % 8 == 0 && p.ld * eb % 16 == 0 && ((uintptr_t)p.x & 15u) == 0 && ((uintptr_t)p.q & 7u) == 0;
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  if (dtype == GB_DTYPE_BF16) return launch_quantize<Bf16, kSource>(p, vec, stream);
  if (dtype == GB_DTYPE_FP16) return launch_quantize<Fp16, kSource>(p, vec, stream);
  return launch_quantize<Fp32, kSource>(p, vec, stream);
}

// ---- tokens into expert order and back ---------------------------------------------------------------------
// A CTA holds blockDim.y tokens, blockDim.x lanes walk a row in vectors of V.  All three are bound by memory.

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
        if (to >= 0) reinterpret_cast<V*>(rows + to * row_bytes)[c] = v;
      }
    }
  }
  for (int64_t j = *live + t; j < T * topk; j += (int64_t)gridDim.x * blockDim.y) {
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
  constexpr int kInFlight = 4;
  for (int c = threadIdx.x; c < vecs; c += blockDim.x) {
    float acc[P::n] = {};
    for (int s0 = 0; s0 < topk; s0 += kInFlight) {
      typename P::raw r[kInFlight];
      int64_t at[kInFlight];
#pragma unroll
      for (int j = 0; j < kInFlight; ++j) {
        at[j] = s0 + j < topk ? (int64_t)place[t * topk + s0 + j] : -1;
        if (at[j] >= 0) r[j] = reinterpret_cast<const typename P::raw*>(y + at[j] * H)[c];
      }
#pragma unroll
      for (int j = 0; j < kInFlight; ++j) {
        if (at[j] < 0) continue;
        const float weight = w ? w[t * topk + s0 + j] : 1.0f;
        float v[P::n];
        P::unpack(r[j], v);
#pragma unroll
        for (int i = 0; i < P::n; ++i) acc[i] = fmaf(weight, v[i], acc[i]);
      }
    }
    reinterpret_cast<typename P::raw*>(out + t * H)[c] = P::pack(acc);
  }
}

// The weighted sum's gradients, with g = d_out[t]: d_y[place[t, s]] = w[t, s] * g, d_w[t, s] = <y[place[t, s]], g>; a dropped
// pair's weight gets zero, rows of d_y that no pair has become zero.  A token's lanes are whole warps of one CTA: sums by
// shuffles, then over the warps in order.  kSlots of a token's slots at a time.
template <typename T, bool kVec, int kSlots>
__global__ void __launch_bounds__(256)
unpermute_grad_kernel(const typename T::word* __restrict__ d_out, const typename T::word* __restrict__ y, const int32_t* __restrict__ place,
                      const int32_t* __restrict__ live, const float* __restrict__ w, int64_t tokens, int topk, int vecs,
                      typename T::word* __restrict__ d_y, float* __restrict__ d_w) {
  using P = Piece<T, kVec>;
  __shared__ float part[8][kSlots];
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
    for (int64_t j = *live + t; j < tokens * topk; j += (int64_t)gridDim.x * blockDim.y) {
      typename P::raw* to = reinterpret_cast<typename P::raw*>(d_y + j * H);
      for (int c = threadIdx.x; c < vecs; c += blockDim.x) to[c] = typename P::raw{};
    }
  }
}

// Lanes of a token: whole warps, no more than the row has vectors; 256 threads a CTA.
dim3 token_block(int vecs) {
  unsigned x = 32;
  while (x < 256 && x < (unsigned)vecs) x *= 2;
  return dim3(x, 256 / x);
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
    const dim3 block = token_block((int)(bytes / (int64_t)sizeof(V)));                                                               \
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
  const dim3 block = token_block(vecs), grid((unsigned)((T + block.y - 1) / block.y));
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
  const dim3 block = token_block(vecs), grid((unsigned)((T + block.y - 1) / block.y));
#define GB_GRAD(D, V, S)                                                                                                                    \
  GB_CUDA_OK(gb_launch(unpermute_grad_kernel<D, V, S>, grid, block, 0, (cudaStream_t)stream, (const D::word*)d_out, (const D::word*)y, place, live, \
                       weights, T, (int)topk, vecs, (D::word*)d_y, d_w))
#define GB_GRAD_SLOTS(D, V) do { if (topk > 4) GB_GRAD(D, V, 8); else GB_GRAD(D, V, 4); } while (0)
  if (dtype == GB_DTYPE_BF16) { if (vec) GB_GRAD_SLOTS(Bf16, true); else GB_GRAD_SLOTS(Bf16, false); }
  else if (dtype == GB_DTYPE_FP16) { if (vec) GB_GRAD_SLOTS(Fp16, true); else GB_GRAD_SLOTS(Fp16, false); }
  else { if (vec) GB_GRAD_SLOTS(Fp32, true); else GB_GRAD_SLOTS(Fp32, false); }
#undef GB_GRAD_SLOTS
#undef GB_GRAD
  return GB_OK;
}

}  // extern "C"
