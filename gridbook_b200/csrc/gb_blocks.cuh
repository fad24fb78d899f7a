// Elements of the block-scaled E4M3 kernels: the row types as fp32, pairs of fp32, and the quantisation of a block whose columns lie
// in a group of lanes.
#pragma once

#include "gb_common.cuh"

#include <type_traits>

namespace gb_blocks {

constexpr int kBlock = 128;                // columns of a block, rows of a weight's
constexpr float kAmaxFloor = 1e-10f;       // a block of zeros gets a scale that divides

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

// Two fp32 in a register pair, each product or sum rounded as a single one's.
GB_DEVINL uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
GB_DEVINL uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
GB_DEVINL uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// The sum rounded down, and so -0 where it is exactly zero.
GB_DEVINL uint64_t fma_down_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rm.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

GB_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The E4M3 bytes of a lane's `kN` values, four to a word, and the block's scale; the block is kLanes neighbouring lanes, which call
// it together with the rest of their warp.
template <int kN, int kLanes>
GB_DEVINL void quantize_block(const float (&v)[kN], int scale_rule, float& scale, uint32_t (&q)[kN / 4]) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kN; ++i) amax = max_nan(amax, fabsf(v[i]));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  amax = max_nan(amax, kAmaxFloor);
  scale = scale_rule == GB_SCALE_RULE_DIV ? __fdiv_rn(amax, 448.0f) : __fmul_rn(amax, 1.0f / 448.0f);
  uint32_t h[kN / 2];
  if (gb_plain_division(scale)) {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) h[i] = gb_cvt_e4m3x2(__fdiv_rn(v[2 * i], scale), __fdiv_rn(v[2 * i + 1], scale));
  } else {
    // gb_div of two values at a time.  The remainder is exact, so that its rounding says one thing only, the sign of a remainder of zero: with
    // -0 the correction leaves a quotient of -0 what it is, where +0 would make it +0.  (It is not exact next to the least fp32
    // values, whose quotients are far below E4M3's least.)
    const float rinv = __frcp_rn(scale);
    const uint64_t r2 = pack_f32x2(rinv, rinv), d2 = pack_f32x2(-scale, -scale);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const uint64_t v2 = pack_f32x2(v[2 * i], v[2 * i + 1]);
      uint64_t t = mul_f32x2(v2, r2);
      t = fma_f32x2(fma_down_f32x2(t, d2, v2), r2, t);
      float lo, hi;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(t));
      h[i] = gb_cvt_e4m3x2(lo, hi);
    }
  }
#pragma unroll
  for (int i = 0; i < kN / 4; ++i) q[i] = h[2 * i] | h[2 * i + 1] << 16;
}

}  // namespace gb_blocks
