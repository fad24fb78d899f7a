// The norms behind and in front of a block, with the block's gate and the residual stream between them, and their gradients.
//
// For a row y that a block gives and the row r of the stream, H values each,
//     u = y, or y_hat (o + pw) with y_hat = y / sqrt(mean y^2 + eps)         the norm behind the block
//     x = a r + b g u                                                        the stream, stored in its own type
//     h = x_hat (o + w)        with x_hat = x / sqrt(mean x^2 + eps)         the norm in front of the next block
// g a gate for each channel, row or group of rows, or 1; o 0, or 1 for weights kept around zero.  h is taken from x as it is stored,
// so that it is the norm of what is returned; in E4M3 blocks (one scale per 128 columns) from x before its rounding.
// With gradients dh and ds of h and x,
//     dx = ds + (dh (o + w) - x_hat mean(dh (o + w) x_hat)) / rms x,      dr = a dx,      dw = sum over rows of dh x_hat
//     du = b g dx,   dg = sum over its rows of b u dx,   dpw = sum over rows of du y_hat
//     dy = du, or (du (o + pw) - y_hat mean(du (o + pw) y_hat)) / rms y
//
// A row is read and written once, and used in registers and shared memory in between.  Blocks stay and walk the
// rows; whole rows come by bulk copies into a ring that is some rows ahead, so that loads go on through the sums over a row.
// A thread has the same eight (or sixteen) columns of every row: the weights' gradients add up in its registers, and a second launch
// adds the blocks' sums, in their order.  Rows that are no whole 16-byte pieces, and very long ones, go value by value; backward also
// fp32 rows of 7571 to 8192 values with both weights and a gate for each channel, which leave no room for the weights beside one row.
//
// Measured, bf16, with both weights: 8192 x 5120 forward 59 us (51 at the copy rate), backward 98 and 7 for the join (77); 4096 x 7168 into E4M3
// blocks 42 (31.5); one row 3.7, launch included.  Cold, DRAM is 67, 59 and 47 % busy, issue slots 58 to 63 %, with a third of the warps that an SM
// holds: no single pipe is full; what is left are the waits at the row's barriers with few warps beside.  Odd rows, 8192 x 5121
// forward and backward: 752.  Backward past 5120 columns a block has 1024 threads of 64 registers, which the sums do not all fit (2048 x 16384
// forward and backward 308, 82 at the copy rate).
#include "gb_blocks.cuh"

#include <algorithm>
#include <atomic>

namespace {

using namespace gb_blocks;

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kMostStages = 8;
constexpr int kRingMax = 208 * 1024;

struct NormParams {
  int64_t T, H;
  const void *y, *r, *gate, *w, *pw;
  int64_t y_ld, r_ld, gate_ld, gate_rows;                // rows that share a row of the gate
  int w_type, pw_type;                                   // GB_DTYPE_*
  float a, b, eps, offset;
  float inv_h;
  void *h, *s;                                           // out; backward: s is in
  float *rstd, *post_rstd;                               // out or null; backward: in
  uint8_t* q;
  float* scale;
  int scale_rule;
  int stages;
  uint32_t stage_bytes;
  uint32_t in_at[5];                                     // where a stage holds the arrays of a row; ~0u: not read
  uint32_t w_at, pw_at, g_at;                            // behind the ring: the weights, and a gate that all rows of the block share
  int* status;
  // backward
  const void *dh, *ds;
  int64_t dh_ld, ds_ld;
  void *dy, *dr, *dg;                                    // dg: where every row has a gate of its own
  float *part_w, *part_pw, *part_g;                      // [blocks][H]
  int per_gate;                                          // blocks that work on the rows of one gate row; 0: no sums for a gate
  int gates;                                             // gate rows where there are more than blocks: a block takes every gridDim-th; else 0
  float* means;                                          // [T], value by value: mean(dh (o + w) x_hat)
};

GB_DEVINL float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
// Sum over the block's threads, in the same order each time.  `turn` changes the buffer from call to call: one barrier is enough.
GB_DEVINL float block_sum(float v, float (*red)[32], int& turn) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = warp_sum(v);
  float* to = red[turn & 1];
  ++turn;
  if (lane == 0) to[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? to[lane] : 0.0f);
}
GB_DEVINL float value_of(const void* p, int type, int64_t c) {
  if (type == GB_DTYPE_BF16) return to_f32<Bf16>(__ldg(static_cast<const uint16_t*>(p) + c));
  if (type == GB_DTYPE_FP16) return to_f32<Fp16>(__ldg(static_cast<const uint16_t*>(p) + c));
  return __ldg(static_cast<const float*>(p) + c);
}

// Eight columns of a row in fp32, as four pairs: products and sums go two at a time (a third fewer instructions, which the norms are
// bound by next to memory).
struct F8 { uint64_t v[4]; };
GB_DEVINL uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
GB_DEVINL uint64_t both(float v) { return pack_f32x2(v, v); }
GB_DEVINL F8 all8(float v) { const uint64_t b = both(v); return {{b, b, b, b}}; }
#define GB_EACH for (int i_ = 0; i_ < 4; ++i_)
GB_DEVINL F8 operator*(const F8& a, const F8& b) {
  F8 r;
#pragma unroll
  GB_EACH r.v[i_] = mul_f32x2(a.v[i_], b.v[i_]);
  return r;
}
GB_DEVINL F8 operator*(const F8& a, uint64_t b) { return a * F8{{b, b, b, b}}; }
GB_DEVINL F8 operator+(const F8& a, const F8& b) {
  F8 r;
#pragma unroll
  GB_EACH r.v[i_] = add_f32x2(a.v[i_], b.v[i_]);
  return r;
}
GB_DEVINL F8 fma8(const F8& a, const F8& b, const F8& c) {
  F8 r;
#pragma unroll
  GB_EACH r.v[i_] = fma_f32x2(a.v[i_], b.v[i_], c.v[i_]);
  return r;
}
GB_DEVINL F8 fma8(const F8& a, uint64_t b, const F8& c) { return fma8(a, F8{{b, b, b, b}}, c); }
GB_DEVINL void dot8(const F8& a, const F8& b, uint64_t& sum) {          // two sums: of the even columns and the odd ones
#pragma unroll
  GB_EACH sum = fma_f32x2(a.v[i_], b.v[i_], sum);
}
#undef GB_EACH
GB_DEVINL float halves(uint64_t v) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
  return lo + hi;
}
GB_DEVINL uint64_t words(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
// As they lie in memory.
template <typename T>
struct Raw8 { uint4 q[sizeof(typename T::word) / 2]; };
template <typename T>
GB_DEVINL Raw8<T> raw8(const typename T::word* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(typename T::word) / 2; ++i) r.q[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
GB_DEVINL F8 f8(const Raw8<T>& r) {
  if constexpr (sizeof(typename T::word) == 4) return {{words(r.q[0].x, r.q[0].y), words(r.q[0].z, r.q[0].w), words(r.q[1].x, r.q[1].y), words(r.q[1].z, r.q[1].w)}};
  else {
    F8 f;
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, Bf16>) f.v[i] = words(w[i] << 16, w[i] & 0xFFFF0000u);
      else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f.v[i] = pack_f32x2(h.x, h.y);
      }
    }
    return f;
  }
}
template <typename T>
GB_DEVINL F8 load8(const typename T::word* p) { return f8<T>(raw8<T>(p)); }
template <typename T>
GB_DEVINL Raw8<T> rounded(const F8& f) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("mov.b64 {%0, %1}, %2;" : "=r"(w[2 * i]), "=r"(w[2 * i + 1]) : "l"(f.v[i]));
  Raw8<T> r;
  if constexpr (sizeof(typename T::word) == 4) {
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r.q[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = __uint_as_float(w[2 * i]), hi = __uint_as_float(w[2 * i + 1]);
      if constexpr (std::is_same_v<T, Bf16>) h[i] = gb_pack_bf16x2(lo, hi);
      else { const __half2 v = __floats2half2_rn(lo, hi); h[i] = *reinterpret_cast<const uint32_t*>(&v); }
    }
    r.q[0] = make_uint4(h[0], h[1], h[2], h[3]);
  }
  return r;
}
template <typename T>
GB_DEVINL void store8(typename T::word* p, const Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(typename T::word) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.q[i];
}
template <typename T>
GB_DEVINL void store8(typename T::word* p, const F8& f) { store8<T>(p, rounded<T>(f)); }
// What a launch has is known to the compiler in the commonest forms: rows of exactly kV x 8 columns a thread, weights of the rows'
// own type with nothing added, all gradients there and asked for.  The others (other widths, weights around zero, fp32 weights, a gate for each
// sequence) look at bounds, types and absent inputs for every eight columns, a third of the instructions: 8192 x 5120 bf16
// forward 66 us, backward 116.
enum Form { kAny = 0, kPostGate = 1, kPost = 2, kPre = 3 };          // both norms with a gate that rows share, without a gate; the second norm alone

// Weights of eight columns in shared memory (of the longest rows, which fill it, where they lie), o + w; kRaw: of the rows' own type, o zero.
template <typename T, bool kRaw>
struct Weights {
  const uint8_t* p;
  int type;
  float offset;
  GB_DEVINL F8 get(int c) const {
    F8 v;
    if (kRaw) v = load8<T>(reinterpret_cast<const typename T::word*>(p) + c);
    else if (type == GB_DTYPE_BF16) v = load8<Bf16>(reinterpret_cast<const uint16_t*>(p) + c);
    else if (type == GB_DTYPE_FP16) v = load8<Fp16>(reinterpret_cast<const uint16_t*>(p) + c);
    else v = load8<Fp32>(reinterpret_cast<const uint32_t*>(p) + c);
    return kRaw || offset == 0.0f ? v : v + all8(offset);
  }
};
// The weights' way there, by one thread; they are waited for like a row.
GB_DEVINL void fetch_weights(const NormParams& p, uint8_t* smem, const void* gate, uint32_t gate_bytes, uint64_t* bar) {
  const auto bytes = [&](int type) { return (uint32_t)(p.H * (type == GB_DTYPE_FP32 ? 4 : 2)); };
  gb_mbar_expect_tx(bar, (p.w_at != ~0u ? bytes(p.w_type) : 0u) + (p.pw_at != ~0u ? bytes(p.pw_type) : 0u) + (p.g_at != ~0u ? gate_bytes : 0u));
  if (p.w_at != ~0u) gb_bulk_g2s(smem + p.w_at, p.w, bytes(p.w_type), bar);
  if (p.pw_at != ~0u) gb_bulk_g2s(smem + p.pw_at, p.pw, bytes(p.pw_type), bar);
  if (p.g_at != ~0u) gb_bulk_g2s(smem + p.g_at, gate, gate_bytes, bar);
}
template <typename R>
GB_DEVINL float as_stored(float v) { return to_f32<R>(from_f32<R>(v)); }

// The ring of rows.  A wait that runs out is remembered with the step it belongs to: the block leaves together behind that step's
// barrier, however far its fastest thread has come.
struct Ring {
  uint64_t* full;
  volatile int* gave_up;
  GB_DEVINL void wait(int i, int s, uint32_t phase, int* status, int code) const {     // step i, in stage s
    if (!gb_mbar_wait(&full[s], phase)) {
      atomicMin((int*)gave_up, i);
      atomicExch(status, code);
    }
  }
};

template <typename T, typename R, int kV, int kThreads, bool kFp8, Form kForm>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
norm_rows_kernel(const __grid_constant__ NormParams p) {
  using word = typename T::word;
  using rword = typename R::word;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kMostStages + 1];           // the last one: the weights
  __shared__ float red[2][32];
  __shared__ int gave_up;
  const int tid = threadIdx.x, H = (int)p.H, T_ = (int)p.T, step = (int)gridDim.x;
  gb_pdl_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) gb_mbar_init(&full[s], 1);
    gb_mbar_init(&full[kMostStages], 1);
    gave_up = 0x7FFFFFFF;
    gb_fence_barrier_init();
  }
  __syncthreads();
  gb_pdl_wait();
  const uint32_t y_bytes = (uint32_t)(H * (int)sizeof(word)), r_bytes = (uint32_t)(H * (int)sizeof(rword));
  constexpr bool kKnown = kForm != kAny;
  const bool has_w = kKnown || p.w, has_pw = kKnown ? kForm != kPre : p.pw != nullptr, has_gate = kKnown ? kForm == kPostGate : p.gate != nullptr;
  const bool own_gate = !kKnown && p.in_at[2] != ~0u;    // every row has a gate of its own
  auto fetch = [&](int64_t t, int s) {
    uint8_t* st = ring + (size_t)s * p.stage_bytes;
    gb_mbar_expect_tx(&full[s], p.stage_bytes);
    gb_bulk_g2s(st + p.in_at[0], static_cast<const word*>(p.y) + t * p.y_ld, y_bytes, &full[s]);
    gb_bulk_g2s(st + p.in_at[1], static_cast<const rword*>(p.r) + t * p.r_ld, r_bytes, &full[s]);
    if (own_gate) gb_bulk_g2s(st + p.in_at[2], static_cast<const word*>(p.gate) + t * p.gate_ld, y_bytes, &full[s]);
  };
  if (tid == 0) {
    fetch((int64_t)blockIdx.x, 0);                       // a block has a row at least
    fetch_weights(p, ring, p.gate, y_bytes, &full[kMostStages]);
    for (int s = 1; s < p.stages; ++s)
      if ((int64_t)blockIdx.x + (int64_t)s * step < T_) fetch((int64_t)blockIdx.x + (int64_t)s * step, s);
  }
  constexpr bool kLong = kThreads == 1024;
  const bool one_gate = kKnown ? has_gate : p.gate && (kLong ? p.gate_rows == p.T : p.g_at != ~0u);   // the same for all rows
  const Weights<T, kKnown> w{kLong ? static_cast<const uint8_t*>(p.w) : ring + p.w_at, p.w_type, p.offset},
      pw{kLong ? static_cast<const uint8_t*>(p.pw) : ring + p.pw_at, p.pw_type, p.offset};
  const Ring wheel{full, &gave_up};
  int turn = 0, i = 0, s = 0;
  uint32_t phase = 0;
  for (int64_t t = blockIdx.x; t < T_; t += step, ++i) {
    const uint8_t* st = ring + (size_t)s * p.stage_bytes;
    wheel.wait(i, s, phase, p.status, 91);
    F8 x[kV];
    float rp = 1.0f;
    uint64_t sum = 0;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const int c = (k * (int)blockDim.x + tid) * 8;
      x[k] = all8(0.0f);
      if (kKnown || c < H) {
        x[k] = load8<T>(reinterpret_cast<const word*>(st + p.in_at[0]) + c);
        dot8(x[k], x[k], sum);
      }
    }
    if (has_pw) rp = rsqrtf(fmaf(block_sum(halves(sum), red, turn), p.inv_h, p.eps));
    sum = 0;
    if (i == 0) wheel.wait(0, kMostStages, 0, p.status, 91);
    const word* gate_row = nullptr;
    if (own_gate) gate_row = reinterpret_cast<const word*>(st + p.in_at[2]);
    else if (one_gate) gate_row = kLong ? static_cast<const word*>(p.gate) : reinterpret_cast<const word*>(ring + p.g_at);
    else if (has_gate) gate_row = static_cast<const word*>(p.gate) + (int64_t)((uint32_t)t / (uint32_t)p.gate_rows) * p.gate_ld;
    rword* out = static_cast<rword*>(p.s) + t * H;
    const uint64_t scale_r = both(p.a), scale_u = both(p.b * rp);
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const int c = (k * (int)blockDim.x + tid) * 8;
      if (kKnown || c < H) {
        if (has_pw) x[k] = x[k] * pw.get(c);
        if (has_gate) x[k] = x[k] * load8<T>(gate_row + c);
        x[k] = fma8(x[k], scale_u, load8<R>(reinterpret_cast<const rword*>(st + p.in_at[1]) + c) * scale_r);
        const Raw8<R> kept = rounded<R>(x[k]);
        store8<R>(out + c, kept);
        if (!kFp8) x[k] = f8<R>(kept);
        dot8(x[k], x[k], sum);
      }
    }
    const float rs = rsqrtf(fmaf(block_sum(halves(sum), red, turn), p.inv_h, p.eps));
    if (gave_up <= i) break;
    if (tid == 0) {                                      // every thread has taken what it needs of the stage
      if (t + (int64_t)p.stages * step < T_) fetch(t + (int64_t)p.stages * step, s);
      if (p.rstd) p.rstd[t] = rs;
      if (p.post_rstd) p.post_rstd[t] = rp;
    }
    if (++s == p.stages) { s = 0; phase ^= 1; }
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const int c = (k * (int)blockDim.x + tid) * 8;
      x[k] = x[k] * both(rs);
      if (kKnown || c < H) {
        if (has_w) x[k] = x[k] * w.get(c);
        if (!kFp8) store8<T>(static_cast<word*>(p.h) + t * H + c, x[k]);
      }
      if constexpr (kFp8) {                              // sixteen neighbours have a block
        float scale, h[8];
        uint32_t q[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("mov.b64 {%0, %1}, %2;" : "=f"(h[2 * j]), "=f"(h[2 * j + 1]) : "l"(x[k].v[j]));
        quantize_block<8, 16>(h, p.scale_rule, scale, q);
        if (kKnown || c < H) {
          *reinterpret_cast<uint2*>(p.q + t * H + c) = make_uint2(q[0], q[1]);
          if ((tid & 15) == 0) p.scale[t * ((H + kBlock - 1) / kBlock) + c / kBlock] = scale;
        }
      }
    }
  }
  if (gave_up != 0x7FFFFFFF) __nanosleep(1000000);       // copies still in flight end before the memory goes
}

// kR rows at a time between the barriers: they share what is unpacked of the weights.
template <typename T, typename R, int kV, int kR, int kThreads, Form kForm>
__global__ void __launch_bounds__(kThreads, kThreads <= 256 ? 2 : 1)
norm_rows_grad_kernel(const __grid_constant__ NormParams p) {
  using word = typename T::word;
  using rword = typename R::word;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kMostStages + 1];           // the last one: the weights
  __shared__ float red[2][kR][32];
  __shared__ int gave_up;
  const int tid = threadIdx.x, H = (int)p.H;
  gb_pdl_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) gb_mbar_init(&full[s], 1);
    gb_mbar_init(&full[kMostStages], 1);
    gave_up = 0x7FFFFFFF;
    gb_fence_barrier_init();
  }
  __syncthreads();
  gb_pdl_wait();
  // the block's share of the rows, of all or of those of a gate row: first + begin, + step, ..; or all of those of some gate rows
  const int rows = p.per_gate == 0 ? (int)p.T : (int)p.gate_rows, first = p.per_gate == 0 ? 0 : (int)blockIdx.x / p.per_gate * rows;
  const int begin = p.per_gate == 0 ? (int)blockIdx.x : (int)blockIdx.x % p.per_gate, step = p.per_gate == 0 ? (int)gridDim.x : p.per_gate;
  const bool some_gates = kForm == kAny && p.gates != 0;
  const int mine = some_gates ? (p.gates - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * rows : (rows - begin + step - 1) / step;
  const auto row_at = [&](int n) -> int64_t {            // the n-th row of the share
    if (some_gates) return (int64_t)((int)blockIdx.x + n / rows * (int)gridDim.x) * rows + n % rows;
    return first + begin + (int64_t)n * step;
  };
  const uint32_t y_bytes = (uint32_t)(H * (int)sizeof(word)), r_bytes = (uint32_t)(H * (int)sizeof(rword));
  constexpr bool kKnown = kForm != kAny;
  const bool has_w = kKnown || p.w, has_pw = kKnown ? kForm != kPre : p.pw != nullptr, has_gate = kKnown ? kForm == kPostGate : p.gate != nullptr;
  const bool has_y = kKnown ? kForm != kPre : p.in_at[3] != ~0u, has_dh = kKnown || p.dh, has_ds = kKnown || p.ds;
  const bool own_gate = !kKnown && p.in_at[4] != ~0u;    // every row has a gate of its own
  auto fetch = [&](int n, int s) {
    const int64_t t = row_at(n);
    uint8_t* st = ring + (size_t)s * p.stage_bytes;
    gb_mbar_expect_tx(&full[s], p.stage_bytes);
    gb_bulk_g2s(st + p.in_at[0], static_cast<const rword*>(p.s) + t * H, r_bytes, &full[s]);
    if (p.in_at[1] != ~0u) gb_bulk_g2s(st + p.in_at[1], static_cast<const word*>(p.dh) + t * p.dh_ld, y_bytes, &full[s]);
    if (p.in_at[2] != ~0u) gb_bulk_g2s(st + p.in_at[2], static_cast<const rword*>(p.ds) + t * p.ds_ld, r_bytes, &full[s]);
    if (p.in_at[3] != ~0u) gb_bulk_g2s(st + p.in_at[3], static_cast<const word*>(p.y) + t * p.y_ld, y_bytes, &full[s]);
    if (own_gate) gb_bulk_g2s(st + p.in_at[4], static_cast<const word*>(p.gate) + t * p.gate_ld, y_bytes, &full[s]);
  };
  if (tid == 0) {
    if (mine > 0) fetch(0, 0);
    fetch_weights(p, ring, static_cast<const word*>(p.gate) + (p.per_gate != 0 ? (int64_t)(first / rows) * p.gate_ld : 0), y_bytes, &full[kMostStages]);
    for (int s = 1; s < p.stages; ++s)
      if (s < mine) fetch(s, s);
  }
  constexpr bool kLong = kV == 2;
  const Weights<T, kKnown> w_of{kLong ? static_cast<const uint8_t*>(p.w) : ring + p.w_at, p.w_type, p.offset},
      pw_of{kLong ? static_cast<const uint8_t*>(p.pw) : ring + p.pw_at, p.pw_type, p.offset};
  const word* gate_own = static_cast<const word*>(p.gate) + (p.per_gate != 0 ? (int64_t)(first / rows) * p.gate_ld : 0);
  const bool many_gates = !kKnown && p.gate && !own_gate && (kLong ? p.gates != 0 || (p.per_gate == 0 && p.gate_rows != p.T) : p.g_at == ~0u);   // not one for the block
  const Ring wheel{full, &gave_up};
  wheel.wait(0, kMostStages, 0, p.status, 92);
  F8 acc_w[kV], acc_pw[kV], acc_g[kV];
#pragma unroll
  for (int k = 0; k < kV; ++k) acc_w[k] = acc_pw[k] = acc_g[k] = all8(0.0f);
  // sums over the block of a value for each row, in the same order each time
  int turn = 0;
  const auto sums = [&](float (&m)[kR]) {
    const int warp = tid >> 5, lane = tid & 31, warps = (int)blockDim.x >> 5;
#pragma unroll
    for (int q = 0; q < kR; ++q) {
      m[q] = warp_sum(m[q]);
      if (lane == 0) red[turn][q][warp] = m[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kR; ++q) m[q] = warp_sum(lane < warps ? red[turn][q][lane] : 0.0f) * p.inv_h;
    turn ^= 1;
  };
  int s = 0;
  uint32_t phase = 0;
  float rs_next[kR], rp_next[kR];                        // of the rows to come
  const auto norms = [&](int n) {
#pragma unroll
    for (int q = 0; q < kR; ++q) {
      const int64_t t = row_at(n + q);
      rs_next[q] = n + q < mine ? __ldg(p.rstd + t) : 0.0f;
      rp_next[q] = n + q < mine && has_pw ? __ldg(p.post_rstd + t) : 1.0f;
    }
  };
  norms(0);
  for (int n = 0; n < mine; n += kR) {
    const uint8_t* st[kR];
    int64_t t[kR];
    bool on[kR];
    float rs[kR], rp[kR], m1[kR], m2[kR];
    F8 d[kR][kV];                                        // dh (o + w), dx, du (o + pw) in turn
#pragma unroll
    for (int q = 0; q < kR; ++q) {
      const int sq = s + q < p.stages ? s + q : s + q - p.stages;
      st[q] = ring + (size_t)sq * p.stage_bytes;
      on[q] = n + q < mine;
      t[q] = row_at(n + q);
      rs[q] = rs_next[q];
      rp[q] = rp_next[q];
      if (on[q]) wheel.wait(n + q, sq, phase ^ (s + q < p.stages ? 0u : 1u), p.status, 92);
    }
    norms(n + kR);
    uint64_t sum[kR];
#pragma unroll
    for (int q = 0; q < kR; ++q) sum[q] = 0;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const int c = (k * (int)blockDim.x + tid) * 8;
#pragma unroll
      for (int q = 0; q < kR; ++q) d[q][k] = all8(0.0f);
      if ((kKnown || c < H) && has_dh) {
        const F8 w = has_w ? w_of.get(c) : all8(1.0f);
#pragma unroll
        for (int q = 0; q < kR; ++q) {
          if (!on[q]) continue;
          const F8 xh = load8<R>(reinterpret_cast<const rword*>(st[q] + p.in_at[0]) + c) * both(rs[q]);
          d[q][k] = load8<T>(reinterpret_cast<const word*>(st[q] + p.in_at[1]) + c);
          acc_w[k] = fma8(d[q][k], xh, acc_w[k]);
          d[q][k] = d[q][k] * w;
          dot8(d[q][k], xh, sum[q]);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kR; ++q) { m1[q] = halves(sum[q]); sum[q] = 0; }
    sums(m1);
    Raw8<T> y_raw[kR][kV];
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const int c = (k * (int)blockDim.x + tid) * 8;
      if (kKnown || c < H) {
        const F8 w = has_pw ? pw_of.get(c) : all8(1.0f);
        F8 g = all8(1.0f);
#pragma unroll
        for (int q = 0; q < kR; ++q) {
          if (!on[q]) continue;
          F8& e = d[q][k];
          // dx; e is not scaled by 1 / rms yet
          e = fma8(load8<R>(reinterpret_cast<const rword*>(st[q] + p.in_at[0]) + c), both(-rs[q] * m1[q]), e);
          e = has_ds ? fma8(e, both(rs[q]), load8<R>(reinterpret_cast<const rword*>(st[q] + p.in_at[2]) + c)) : e * both(rs[q]);
          if (kKnown || p.dr) store8<R>(static_cast<rword*>(p.dr) + t[q] * H + c, e * both(p.a));
          F8 v = all8(0.0f);                             // y_hat, or y
          if (has_y) {
            y_raw[q][k] = raw8<T>(reinterpret_cast<const word*>(st[q] + p.in_at[3]) + c);
            v = f8<T>(y_raw[q][k]);
            if (has_pw) v = v * both(rp[q]);
          }
          e = e * both(p.b);
          if (has_gate) {
            if (q == 0 || own_gate || many_gates) {
              const word* from = reinterpret_cast<const word*>(own_gate ? st[q] + p.in_at[4] : kLong ? reinterpret_cast<const uint8_t*>(gate_own) : ring + p.g_at);
              if (many_gates) from = static_cast<const word*>(p.gate) + (int64_t)((uint32_t)t[q] / (uint32_t)p.gate_rows) * p.gate_ld;
              g = load8<T>(from + c);
            }
            const F8 u = v * w;
            if (!kKnown && p.dg) store8<T>(static_cast<word*>(p.dg) + t[q] * H + c, e * u);
            else if (kKnown || p.part_g) acc_g[k] = fma8(e, u, acc_g[k]);
            e = e * g;
          }
          if (has_pw) {
            acc_pw[k] = fma8(e, v, acc_pw[k]);
            e = e * w;
            dot8(e, v, sum[q]);
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kR; ++q) m2[q] = halves(sum[q]);
    sums(m2);
    if (gave_up <= n + kR - 1) break;
#pragma unroll
    for (int q = 0; q < kR; ++q) {
      if (tid == 0 && n + q + p.stages < mine) fetch(n + q + p.stages, s);
      if (++s == p.stages) { s = 0; phase ^= 1; }
    }
    if (kKnown || p.dy) {
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        const int c = (k * (int)blockDim.x + tid) * 8;
#pragma unroll
        for (int q = 0; q < kR; ++q) {
          if ((!kKnown && c >= H) || !on[q]) continue;
          if (has_pw) d[q][k] = fma8(f8<T>(y_raw[q][k]), both(-rp[q] * m2[q]), d[q][k]) * both(rp[q]);
          store8<T>(static_cast<word*>(p.dy) + t[q] * H + c, d[q][k]);
        }
      }
    }
    if (some_gates && p.part_g && (n + kR) % rows == 0) {  // the last row of a gate row's (two rows at a time: they are even in number)
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        const int c = (k * (int)blockDim.x + tid) * 8;
        if (c < H) store8<Fp32>(reinterpret_cast<uint32_t*>(p.part_g) + t[kR - 1] / rows * H + c, acc_g[k]);
        acc_g[k] = all8(0.0f);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kV; ++k) {
    const int c = (k * (int)blockDim.x + tid) * 8;
    const int64_t at = (int64_t)blockIdx.x * H + c;
    if (kKnown || c < H) {
      if (p.part_w) store8<Fp32>(reinterpret_cast<uint32_t*>(p.part_w) + at, acc_w[k]);
      if (p.part_pw) store8<Fp32>(reinterpret_cast<uint32_t*>(p.part_pw) + at, acc_pw[k]);
      if (p.part_g && !some_gates) store8<Fp32>(reinterpret_cast<uint32_t*>(p.part_g) + at, acc_g[k]);
    }
  }
  if (gave_up != 0x7FFFFFFF) __nanosleep(1000000);
}

// ------------------------------------------------------------------------------------------------ value by value
constexpr int kAnyThreads = 256;

// A row's inputs.  They are read by __ldg, so that several of a thread's columns are on their way past what it stores.
template <typename T, typename R>
struct Values {
  using word = typename T::word;
  using rword = typename R::word;
  const NormParams& p;
  int64_t t;
  const word *y_row, *gate_row, *dh_row;
  const rword *r_row, *ds_row, *s_row;
  GB_DEVINL Values(const NormParams& params, int64_t row) : p(params), t(row) {
    y_row = static_cast<const word*>(p.y) + t * p.y_ld;
    gate_row = p.gate ? static_cast<const word*>(p.gate) + (int64_t)((uint32_t)t / (uint32_t)p.gate_rows) * p.gate_ld : nullptr;
    dh_row = p.dh ? static_cast<const word*>(p.dh) + t * p.dh_ld : nullptr;
    r_row = static_cast<const rword*>(p.r) + t * p.r_ld;
    ds_row = p.ds ? static_cast<const rword*>(p.ds) + t * p.ds_ld : nullptr;
    s_row = static_cast<const rword*>(p.s) + t * p.H;
  }
  GB_DEVINL float y(int c) const { return to_f32<T>(__ldg(y_row + c)); }
  GB_DEVINL float gate(int c) const { return gate_row ? to_f32<T>(__ldg(gate_row + c)) : 1.0f; }
  GB_DEVINL float w(int c) const { return p.w ? value_of(p.w, p.w_type, c) + p.offset : 1.0f; }
  GB_DEVINL float pw(int c) const { return p.pw ? value_of(p.pw, p.pw_type, c) + p.offset : 1.0f; }
  GB_DEVINL float x_of(int c, float y, float rp) const {
    const float u = p.pw ? y * (rp * pw(c)) : y;
    return fmaf(p.b, u * gate(c), p.a * to_f32<R>(__ldg(r_row + c)));
  }
  // backward: p.s holds the stream
  GB_DEVINL float x_hat(int c, float rs) const { return to_f32<R>(__ldg(s_row + c)) * rs; }
  GB_DEVINL float dh(int c) const { return dh_row ? to_f32<T>(__ldg(dh_row + c)) : 0.0f; }
  GB_DEVINL float ds(int c) const { return to_f32<R>(__ldg(ds_row + c)); }
  GB_DEVINL float dx(int c, float rs, float m1) const {
    const float d = rs * fmaf(-x_hat(c, rs), m1, dh(c) * w(c));
    return p.ds ? d + ds(c) : d;
  }
};

// kCached: the row fits shared memory in fp32, where a thread keeps its columns from pass to pass; else every pass reads them again.
template <typename T, typename R, bool kFp8, bool kCached>
__global__ void __launch_bounds__(kAnyThreads)
norm_any_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ float row_s[];
  __shared__ float red[2][32];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  int turn = 0;
  const Values<T, R> v{p, (int64_t)blockIdx.x};
  const int H = (int)p.H;
  float rp = 1.0f, sum = 0.0f;
  if (p.pw) {
#pragma unroll 4
    for (int c = threadIdx.x; c < H; c += kAnyThreads) {
      const float y = v.y(c);
      if (kCached) row_s[c] = y;
      sum = fmaf(y, y, sum);
    }
    rp = rsqrtf(fmaf(block_sum(sum, red, turn), p.inv_h, p.eps));
  }
  sum = 0.0f;
  typename R::word* out = static_cast<typename R::word*>(p.s) + v.t * p.H;
#pragma unroll 4
  for (int c = threadIdx.x; c < H; c += kAnyThreads) {
    float x = v.x_of(c, kCached && p.pw ? row_s[c] : v.y(c), rp);
    const typename R::word kept = from_f32<R>(x);
    out[c] = kept;
    if (!kFp8) x = to_f32<R>(kept);
    if (kCached) row_s[c] = x;
    sum = fmaf(x, x, sum);
  }
  const float rs = rsqrtf(fmaf(block_sum(sum, red, turn), p.inv_h, p.eps));
  if (threadIdx.x == 0) {
    if (p.rstd) p.rstd[v.t] = rs;
    if (p.post_rstd) p.post_rstd[v.t] = rp;
  }
  const auto again = [&](int c) {                        // (block_sum's barrier lies in front of it: other threads' columns too)
    if (kCached) return row_s[c];
    const float x = v.x_of(c, v.y(c), rp);
    return kFp8 ? x : as_stored<R>(x);
  };
  if constexpr (!kFp8) {
    typename T::word* h = static_cast<typename T::word*>(p.h) + v.t * p.H;
#pragma unroll 4
    for (int c = threadIdx.x; c < H; c += kAnyThreads) h[c] = from_f32<T>(again(c) * rs * v.w(c));
  } else {
    const int blocks = (H + kBlock - 1) / kBlock;
    for (int b0 = 0; b0 < blocks; b0 += kAnyThreads / 16) {
      const int b = b0 + threadIdx.x / 16, c = b * kBlock + (threadIdx.x & 15) * 8;
      float h[8], scale;
      uint32_t q[2];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = c + j < H ? again(c + j) * rs * v.w(c + j) : 0.0f;
      quantize_block<8, 16>(h, p.scale_rule, scale, q);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < H) p.q[v.t * p.H + c + j] = (uint8_t)(q[j >> 2] >> (8 * (j & 3)));
      if (b < blocks && (threadIdx.x & 15) == 0) p.scale[v.t * blocks + b] = scale;
    }
  }
}

// The backward pass with the row and the columns' sums in shared memory: a block walks its share of the rows, a thread has every
// kAnyGradThreads-th column.
constexpr int kAnyGradThreads = 512;

template <typename T, typename R>
__global__ void __launch_bounds__(kAnyGradThreads)
norm_any_rows_grad_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ float row_s[];
  __shared__ float red[2][32];
  const int tid = threadIdx.x, H = (int)p.H;
  float *d_s = row_s, *x_s = d_s + H, *w_s = x_s + H, *pw_s = w_s + H, *g_s = pw_s + H;   // dh (o + w), dx, du (o + pw) in turn; x_hat, then y_hat; sums
  gb_pdl_launch_dependents();
  for (int c = tid; c < H; c += kAnyGradThreads) w_s[c] = pw_s[c] = g_s[c] = 0.0f;
  gb_pdl_wait();
  int turn = 0;
  const int rows = p.per_gate == 0 ? (int)p.T : (int)p.gate_rows, share = (int)blockIdx.x;
  const int begin = p.per_gate == 0 ? share : share % p.per_gate, step = p.per_gate == 0 ? (int)gridDim.x : p.per_gate;
  const int gates = p.gates != 0 ? p.gates : 1, first_gate = p.gates != 0 ? share : p.per_gate == 0 ? 0 : share / p.per_gate;
  for (int i = p.gates != 0 ? share : 0; i < gates; i += (int)gridDim.x) {
    const int gate = p.gates != 0 ? i : first_gate;
    for (int n = begin; n < rows; n += step) {
      const Values<T, R> v{p, (int64_t)gate * rows + n};
      const float rs = p.rstd[v.t], rp = p.pw ? p.post_rstd[v.t] : 1.0f;
      float m1 = 0.0f, m2 = 0.0f;
#pragma unroll 4
      for (int c = tid; c < H; c += kAnyGradThreads) {
        const float xh = v.x_hat(c, rs), dh = v.dh(c), k = dh * v.w(c);
        w_s[c] = fmaf(dh, xh, w_s[c]);
        d_s[c] = k;
        x_s[c] = xh;
        m1 = fmaf(k, xh, m1);
      }
      m1 = block_sum(m1, red, turn) * p.inv_h;
#pragma unroll 4
      for (int c = tid; c < H; c += kAnyGradThreads) {
        float dx = rs * fmaf(-x_s[c], m1, d_s[c]);
        if (p.ds) dx += v.ds(c);
        if (p.dr) static_cast<typename R::word*>(p.dr)[v.t * p.H + c] = from_f32<R>(p.a * dx);
        const float u = p.pw || p.dg || p.part_g ? v.y(c) * rp : 0.0f, pw = v.pw(c), e = p.b * dx, du = e * v.gate(c);
        if (p.dg) static_cast<typename T::word*>(p.dg)[v.t * p.H + c] = from_f32<T>(e * (u * pw));
        g_s[c] = fmaf(e, u * pw, g_s[c]);
        pw_s[c] = fmaf(du, u, pw_s[c]);
        d_s[c] = du * pw;
        x_s[c] = u;
        m2 = fmaf(du * pw, u, m2);
      }
      m2 = block_sum(m2, red, turn) * p.inv_h;
      if (p.dy)
#pragma unroll 4
        for (int c = tid; c < H; c += kAnyGradThreads)
          static_cast<typename T::word*>(p.dy)[v.t * p.H + c] = from_f32<T>(p.pw ? rp * fmaf(-x_s[c], m2, d_s[c]) : d_s[c]);
    }
    if (p.gates != 0 && p.part_g)
      for (int c = tid; c < H; c += kAnyGradThreads) {
        p.part_g[(int64_t)gate * p.H + c] = g_s[c];
        g_s[c] = 0.0f;
      }
  }
  for (int c = tid; c < H; c += kAnyGradThreads) {
    const int64_t at = (int64_t)share * p.H + c;
    if (p.part_w) p.part_w[at] = w_s[c];
    if (p.part_pw) p.part_pw[at] = pw_s[c];
    if (p.part_g && p.gates == 0) p.part_g[at] = g_s[c];
  }
}

// Rows that do not fit it.
template <typename T, typename R>
__global__ void __launch_bounds__(kAnyThreads)
norm_any_grad_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[2][32];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  int turn = 0;
  const Values<T, R> v{p, (int64_t)blockIdx.x};
  const float rs = p.rstd[v.t], rp = p.pw ? p.post_rstd[v.t] : 1.0f;
  float m1 = 0.0f, m2 = 0.0f;
  if (p.dh)
    for (int c = threadIdx.x; c < (int)p.H; c += kAnyThreads) m1 = fmaf(v.dh(c) * v.w(c), v.x_hat(c, rs), m1);
  m1 = block_sum(m1, red, turn) * p.inv_h;
  if (threadIdx.x == 0) p.means[v.t] = m1;
  for (int c = threadIdx.x; c < (int)p.H; c += kAnyThreads) {
    const float dx = v.dx(c, rs, m1);
    if (p.dr) static_cast<typename R::word*>(p.dr)[v.t * p.H + c] = from_f32<R>(p.a * dx);
    if (p.dg) static_cast<typename T::word*>(p.dg)[v.t * p.H + c] = from_f32<T>(p.b * dx * (v.y(c) * (rp * v.pw(c))));
    if (p.pw) m2 = fmaf(p.b * v.gate(c) * dx * v.pw(c), v.y(c) * rp, m2);
    else if (p.dy) static_cast<typename T::word*>(p.dy)[v.t * p.H + c] = from_f32<T>(p.b * v.gate(c) * dx);
  }
  if (!p.pw || !p.dy) return;
  m2 = block_sum(m2, red, turn) * p.inv_h;
  for (int c = threadIdx.x; c < (int)p.H; c += kAnyThreads) {
    const float du = p.b * v.gate(c) * v.dx(c, rs, m1);
    static_cast<typename T::word*>(p.dy)[v.t * p.H + c] = from_f32<T>(rp * fmaf(-v.y(c) * rp, m2, du * v.pw(c)));
  }
}

// The weights' gradients over a block's share of the rows; a thread has a column.
template <typename T, typename R>
__global__ void __launch_bounds__(kAnyThreads)
norm_any_columns_kernel(const __grid_constant__ NormParams p, int64_t column_blocks) {
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int64_t share = blockIdx.x / column_blocks, c = (blockIdx.x - share * column_blocks) * kAnyThreads + threadIdx.x;
  if (c >= p.H) return;
  const int64_t shares = gridDim.x / column_blocks;
  const int64_t rows = p.per_gate == 0 ? p.T : p.gate_rows;
  const int64_t begin = p.per_gate == 0 ? share : share % p.per_gate, step = p.per_gate == 0 ? shares : p.per_gate;
  float w = 0.0f, pw = 0.0f;
  for (int64_t gate = p.per_gate == 0 ? 0 : share / p.per_gate; gate < (p.gates != 0 ? p.gates : share + 1); gate += shares) {
    float g = 0.0f;
    for (int64_t n = begin; n < rows; n += step) {
      const Values<T, R> v{p, gate * rows + n};
      const float rs = p.rstd[v.t], rp = p.pw ? p.post_rstd[v.t] : 1.0f;
      w = fmaf(v.dh(c), v.x_hat(c, rs), w);
      if (p.part_pw || p.part_g) {
        const float dx = v.dx(c, rs, p.means[v.t]), y_hat = v.y(c) * rp;
        pw = fmaf(p.b * v.gate(c) * dx, y_hat, pw);
        g = fmaf(p.b * dx, y_hat * v.pw(c), g);
      }
    }
    if (p.part_g) p.part_g[(p.gates != 0 ? gate : share) * p.H + c] = g;
  }
  const int64_t at = share * p.H + c;
  if (p.part_w) p.part_w[at] = w;
  if (p.part_pw) p.part_pw[at] = pw;
}

// The shares' sums: a block adds up 32 columns of one result, warp w every 32nd share.
struct JoinParams {
  const float* part[3];       // w, pw, gate: shares of H sums each
  void* out[3];
  int type[3];
  int64_t H, shares, gate_shares;   // shares in all, of a gate row
  int64_t column_blocks;
};
constexpr int kJoinThreads = 1024;

__global__ void __launch_bounds__(kJoinThreads)
norm_join_kernel(const __grid_constant__ JoinParams p) {
  __shared__ float s[32][33];
  gb_pdl_launch_dependents();
  gb_pdl_wait();
  const int64_t job = blockIdx.x / p.column_blocks, col = (blockIdx.x - job * p.column_blocks) * 32 + (threadIdx.x & 31);
  int which = 2;
  int64_t gate = job;                                    // jobs: the weights that are asked for, then the gate's rows
  for (int k = 0; k < 2; ++k)
    if (p.part[k]) {
      if (gate == 0) { which = k; break; }
      --gate;
    }
  const int64_t n = which == 2 ? p.gate_shares : p.shares;
  const float* from = p.part[which] + (which == 2 ? gate * n * p.H : 0);
  float sum = 0.0f;
  if (col < p.H)
    for (int64_t i = threadIdx.x >> 5; i < n; i += 32) sum += from[i * p.H + col];
  s[threadIdx.x & 31][threadIdx.x >> 5] = sum;
  __syncthreads();
  const int c = threadIdx.x >> 5;
  sum = warp_sum(s[c][threadIdx.x & 31]);
  const int64_t at = (blockIdx.x - job * p.column_blocks) * 32 + c;
  if ((threadIdx.x & 31) != 0 || at >= p.H) return;
  const int64_t to = which == 2 ? gate * p.H + at : at;
  if (p.type[which] == GB_DTYPE_BF16) static_cast<uint16_t*>(p.out[which])[to] = from_f32<Bf16>(sum);
  else if (p.type[which] == GB_DTYPE_FP16) static_cast<uint16_t*>(p.out[which])[to] = from_f32<Fp16>(sum);
  else static_cast<float*>(p.out[which])[to] = sum;
}

// ------------------------------------------------------------------------------------------------ host
int size_of(int type) { return type == GB_DTYPE_FP32 ? 4 : 2; }

// Threads of a block, eight (kV = 1) or sixteen columns each; 0: rows too long.
struct Width { int v, threads, most; };
Width width_of(int64_t H) {
  if (H <= 2048) return {1, (int)((H + 255) / 256 * 32), 256};
  if (H <= 16384) return {2, (int)((H + 511) / 512 * 32), H <= 8192 ? 512 : 1024};
  return {0, 0, 0};
}

// For the backward pass: eight columns keep 24 sums in registers, and two rows at a time need 96 of them.
Width grad_width_of(int64_t H) {
  const int threads = (int)((H + 255) / 256 * 32);
  if (H <= 2048) return {1, threads, 256};
  if (H <= 5120) return {1, threads, 640};
  if (H <= 8192) return {1, threads, 1024};
  if (H <= 16384) return {2, (int)((H + 511) / 512 * 32), 1024};
  return {0, 0, 0};
}

bool whole(const void* p, int64_t ld, int size) { return !p || (((uintptr_t)p & 15u) == 0 && ld * size % 16 == 0); }

int check_args(const gb_residual_norm_args* a) {
  GB_REQUIRE(a != nullptr, "null arguments");
  GB_REQUIRE(a->dtype >= GB_DTYPE_BF16 && a->dtype <= GB_DTYPE_FP32, "unknown element type %d", a->dtype);
  GB_REQUIRE(a->stream_dtype == a->dtype || a->stream_dtype == GB_DTYPE_FP32, "the stream has the rows' type or fp32");
  GB_REQUIRE(a->T >= 0 && a->T < (1ll << 31) && a->H >= 1 && a->H < (1ll << 31), "bad shape T=%lld H=%lld", (long long)a->T, (long long)a->H);
  for (int t : {a->w ? a->w_dtype : 0, a->pw ? a->pw_dtype : 0}) GB_REQUIRE(t >= GB_DTYPE_BF16 && t <= GB_DTYPE_FP32, "unknown weight type %d", t);
  GB_REQUIRE(!a->gate || (a->gate_rows >= 1 && a->T % a->gate_rows == 0), "gate rows of %lld rows each do not make up %lld", (long long)a->gate_rows, (long long)a->T);
  GB_REQUIRE(a->y_ld >= a->H && a->r_ld >= a->H && (!a->gate || a->gate_ld >= a->H), "rows that do not overlap expected");
  return GB_OK;
}

NormParams params_of(const gb_residual_norm_args* a) {
  NormParams p = {};
  p.T = a->T; p.H = a->H;
  p.y = a->y; p.r = a->r; p.gate = a->gate; p.w = a->w; p.pw = a->pw;
  p.y_ld = a->y_ld; p.r_ld = a->r_ld; p.gate_ld = a->gate_ld; p.gate_rows = a->gate ? a->gate_rows : 1;
  p.w_type = a->w_dtype; p.pw_type = a->pw_dtype;
  p.a = a->residual_scale; p.b = a->branch_scale; p.eps = a->eps; p.offset = a->weight_offset;
  p.inv_h = (float)(1.0 / (double)a->H);
  p.status = gb_status_word();
  for (uint32_t& at : p.in_at) at = ~0u;
  p.w_at = p.pw_at = p.g_at = ~0u;
  return p;
}

// Blocks an SM, as many as the registers give, and stages of their rings: two at least where there is room, behind `fixed` bytes.
struct Plan { int per_sm, stages; };
Plan plan_of(int threads, int most_threads, int most_stages, uint32_t stage_bytes, uint32_t fixed) {
  int per_sm = most_threads / threads;
  if (per_sm < 1) per_sm = 1;
  if (per_sm > 16) per_sm = 16;
  while (per_sm > 1 && (uint32_t)kRingMax / per_sm < 2 * stage_bytes + fixed + 1024) --per_sm;
  const int stages = (int)(((uint32_t)kRingMax / per_sm - 1024 - fixed) / stage_bytes);
  return {per_sm, stages > most_stages ? most_stages : stages};
}
// Where the weights and a gate that a block's rows share lie behind the ring, from 0 on; their bytes.
uint32_t place_weights(const gb_residual_norm_args* a, bool in_shared, bool one_gate, uint32_t* w_at, uint32_t* pw_at, uint32_t* g_at) {
  uint32_t at = 0;
  const auto place = [&](bool there, int type, uint32_t* to) {
    *to = there ? at : ~0u;
    if (there) at += (uint32_t)(a->H * size_of(type));
  };
  place(in_shared && a->w != nullptr, a->w_dtype, w_at);
  place(in_shared && a->pw != nullptr, a->pw_dtype, pw_at);
  place(in_shared && one_gate, a->dtype, g_at);
  return at;
}
void behind_ring(NormParams& p, size_t ring) {
  for (uint32_t* at : {&p.w_at, &p.pw_at, &p.g_at})
    if (*at != ~0u) *at += (uint32_t)ring;
}

template <typename Go>
int with_types(int dtype, int stream_dtype, Go go) {
  if (dtype == GB_DTYPE_BF16) return stream_dtype == GB_DTYPE_FP32 ? go(Bf16(), Fp32()) : go(Bf16(), Bf16());
  if (dtype == GB_DTYPE_FP16) return stream_dtype == GB_DTYPE_FP32 ? go(Fp16(), Fp32()) : go(Fp16(), Fp16());
  return go(Fp32(), Fp32());
}
template <typename Go>
int with_width(const Width& w, Go go) {
  using std::integral_constant;
  if (w.v == 1) return go(integral_constant<int, 1>(), integral_constant<int, 256>());
  if (w.most == 512) return go(integral_constant<int, 2>(), integral_constant<int, 512>());
  return go(integral_constant<int, 2>(), integral_constant<int, 1024>());
}

// The kernel's shared memory is asked for once a device (half a microsecond a call).
template <auto kKernel>
int launch_ring(int blocks, int threads, size_t smem, cudaStream_t stream, const NormParams& p) {
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  GB_REQUIRE(dev >= 0 && dev < 64, "device %d out of range", dev);
  if (!(asked.load(std::memory_order_acquire) >> dev & 1u)) {
    GB_CUDA_OK(cudaFuncSetAttribute((const void*)kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingMax));
    asked.fetch_or(1ull << dev, std::memory_order_release);
  }
  GB_CUDA_OK(gb_launch(kKernel, dim3((unsigned)blocks), dim3((unsigned)threads), smem, stream, p));
  return GB_OK;
}

Form form_of(const gb_residual_norm_args* a, const Width& w) {
  if (a->H != (int64_t)w.v * w.threads * 8 || !a->w || a->w_dtype != a->dtype || (a->pw && a->pw_dtype != a->dtype) || a->weight_offset != 0.0f) return kAny;
  if (!a->gate) return a->pw ? kPost : kPre;
  return a->pw && a->gate_rows == a->T ? kPostGate : kAny;
}
// go(form) for one that is known at compile time.
template <typename Go>
int with_form(Form f, Go go) {
  using std::integral_constant;
  switch (f) {
    case kPostGate: return go(integral_constant<Form, kPostGate>());
    case kPost: return go(integral_constant<Form, kPost>());
    case kPre: return go(integral_constant<Form, kPre>());
    default: return go(integral_constant<Form, kAny>());
  }
}

template <bool kFp8>
int forward(const gb_residual_norm_args* a, NormParams p, cudaStream_t stream) {
  const int sms = gb_sm_count();
  if (sms <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  const int size = size_of(a->dtype), rsize = size_of(a->stream_dtype);
  const Width width = width_of(a->H);
  const bool full = a->gate && a->gate_rows == 1 && a->T > 1;
  p.in_at[0] = 0;
  p.in_at[1] = (uint32_t)(a->H * size);
  if (full) p.in_at[2] = (uint32_t)(a->H * (size + rsize));
  p.stage_bytes = (uint32_t)(a->H * (size * (full ? 2 : 1) + rsize));
  const uint32_t fixed = place_weights(a, width.most != 1024, a->gate && a->gate_rows == a->T && !full, &p.w_at, &p.pw_at, &p.g_at);
  const bool vec = width.v > 0 && a->H % 8 == 0 && whole(a->y, a->y_ld, size) && whole(a->r, a->r_ld, rsize) && whole(a->gate, a->gate_ld, size) &&
                   whole(a->w, 0, 1) && whole(a->pw, 0, 1) && whole(p.h, 0, 1) && whole(p.s, 0, 1) && whole(p.q, 0, 1) &&
                   p.stage_bytes + fixed <= (uint32_t)kRingMax - 1024;
  const Form form = form_of(a, width);
  return with_types(a->dtype, a->stream_dtype, [&](auto t, auto r) -> int {
    using T = decltype(t);
    using R = decltype(r);
    if (!vec) {
      if (a->H * 4 <= kRingMax) return launch_ring<norm_any_kernel<T, R, kFp8, true>>((int)a->T, kAnyThreads, (size_t)a->H * 4, stream, p);
      return launch_ring<norm_any_kernel<T, R, kFp8, false>>((int)a->T, kAnyThreads, 0, stream, p);
    }
    return with_width(width, [&](auto v, auto most) -> int {
      const Plan plan = plan_of(width.threads, 1024, 4, p.stage_bytes, fixed);
      p.stages = plan.stages;
      const int64_t blocks = a->T < (int64_t)sms * plan.per_sm ? a->T : (int64_t)sms * plan.per_sm;
      constexpr int kV = decltype(v)::value, kMost = decltype(most)::value;
      NormParams q = p;
      behind_ring(q, (size_t)p.stages * p.stage_bytes);
      const size_t smem = (size_t)p.stages * p.stage_bytes + fixed;
      return with_form(form, [&](auto f) -> int {
        return launch_ring<norm_rows_kernel<T, R, kV, kMost, kFp8, decltype(f)::value>>((int)blocks, width.threads, smem, stream, q);
      });
    });
  });
}

// How the rows are shared out for the backward pass: `blocks` shares, `per_gate` of them for the rows of a gate row (0: no sums of its gate).
// Gate rows that are more than the target are dealt out to that many blocks, one whole: sums of the weights' gradients are kept for a
// block, not for a gate row.
struct Shares { int64_t blocks; int per_gate; int64_t gates; };
Shares shares_of(const gb_residual_norm_args* a, bool gate_sums, int64_t target) {
  if (!gate_sums) return {a->T < target ? a->T : target, 0, 1};
  const int64_t gates = a->T / a->gate_rows;
  if (gates > target) return {target, 1, gates};
  int64_t per = target / gates;
  per = per > a->gate_rows ? a->gate_rows : per;
  return {gates * per, (int)per, gates};
}

struct GradPlan {
  bool vec, cached, gate_sums, gate_rows;                // cached: value by value, a row and the columns' sums in shared memory
  Width width;
  Plan plan;
  Shares shares;
  uint32_t at[5], stage_bytes, weight_at[3], fixed;
  int64_t w_at, pw_at, g_at, means_at, bytes;
};
GradPlan grad_plan(const gb_residual_norm_args* a, const gb_residual_norm_grads* g) {
  GradPlan r = {};
  const int size = size_of(a->dtype), rsize = size_of(a->stream_dtype);
  r.gate_rows = a->gate && a->gate_rows == 1 && a->T > 1;
  r.gate_sums = a->gate && g->d_gate && !r.gate_rows;
  r.width = grad_width_of(a->H);
  uint32_t at = 0;
  auto place = [&](bool read, int bytes) {
    const uint32_t here = read ? at : ~0u;
    if (read) at += (uint32_t)(a->H * bytes);
    return here;
  };
  const bool need_y = a->pw || (a->gate && g->d_gate);
  r.vec = r.width.v > 0 && a->H % 8 == 0;
  if (r.vec) {
    r.at[0] = place(true, rsize);
    r.at[1] = place(g->d_h != nullptr, size);
    r.at[2] = place(g->d_stream != nullptr, rsize);
    r.at[3] = place(need_y, size);
    r.at[4] = place(r.gate_rows, size);
    r.stage_bytes = at;
    // a gate row of the block's own; there are more than one for a block only where they are more than its SM takes blocks
    const bool one_gate = a->gate && !r.gate_rows && (a->gate_rows == a->T || (r.gate_sums && a->T / a->gate_rows <= gb_sm_count()));
    r.fixed = place_weights(a, r.width.v == 1, one_gate, &r.weight_at[0], &r.weight_at[1], &r.weight_at[2]);
    r.vec = at + r.fixed <= (uint32_t)kRingMax - 1024 && whole(a->y, a->y_ld, size) && whole(a->gate, a->gate_ld, size) && whole(a->w, 0, 1) && whole(a->pw, 0, 1) &&
            whole(g->stream, 0, 1) && whole(g->d_h, g->d_h_ld, size) && whole(g->d_stream, g->d_stream_ld, rsize) && whole(g->d_y, 0, 1) &&
            whole(g->d_r, 0, 1) && whole(g->d_gate, 0, 1);
  }
  if (r.vec) r.plan = plan_of(r.width.threads, r.width.most <= 256 ? 512 : 65536 / 96, kMostStages, r.stage_bytes, r.fixed);
  const int64_t sms = gb_sm_count();
  r.cached = !r.vec && a->H * 20 <= kRingMax;
  const int64_t any_per_sm = r.cached ? std::max<int64_t>(1, std::min<int64_t>(4, kRingMax / (a->H * 20 + 1024))) : 1;
  r.shares = shares_of(a, r.gate_sums, r.vec ? sms * r.plan.per_sm : r.cached ? sms * any_per_sm : 64);
  auto up = [](int64_t v) { return (v + 255) & ~(int64_t)255; };
  const int64_t sums = up(r.shares.blocks * a->H * 4);
  r.pw_at = g->d_w ? sums : 0;
  r.g_at = r.pw_at + (g->d_pw ? sums : 0);
  r.means_at = r.g_at + (r.gate_sums ? up(std::max(r.shares.blocks, r.shares.gates) * a->H * 4) : 0);
  r.bytes = r.means_at + (r.vec || r.cached ? 0 : up(a->T * 4));
  return r;
}

int launch_join(JoinParams j, int64_t jobs, cudaStream_t stream) {
  j.column_blocks = (j.H + 31) / 32;
  GB_REQUIRE(jobs * j.column_blocks < (1ll << 31), "too many gate rows");
  GB_CUDA_OK(gb_launch(norm_join_kernel, dim3((unsigned)(jobs * j.column_blocks)), dim3(kJoinThreads), 0, stream, j));
  return GB_OK;
}

}  // namespace

int gb_join_columns(const float* part, int64_t shares, int64_t columns, void* out, int dtype, cudaStream_t stream) {
  JoinParams j = {};
  j.part[0] = part; j.out[0] = out; j.type[0] = dtype;
  j.H = columns; j.shares = shares; j.gate_shares = shares;
  return launch_join(j, 1, stream);
}

extern "C" {

int gb_residual_norm(const gb_residual_norm_args* a, void* h, void* stream_out, float* rstd, float* post_rstd, void* stream) {
  const int rc = check_args(a);
  if (rc != GB_OK) return rc;
  if (a->T == 0) return GB_OK;
  GB_REQUIRE(a->y && a->r && h && stream_out, "null pointer argument");
  NormParams p = params_of(a);
  p.h = h; p.s = stream_out; p.rstd = rstd; p.post_rstd = a->pw ? post_rstd : nullptr;
  return forward<false>(a, p, (cudaStream_t)stream);
}

int gb_residual_norm_fp8(const gb_residual_norm_args* a, int scale_rule, void* q, float* scale, void* stream_out, void* stream) {
  const int rc = check_args(a);
  if (rc != GB_OK) return rc;
  if (a->T == 0) return GB_OK;
  GB_REQUIRE(a->y && a->r && q && scale && stream_out, "null pointer argument");
  GB_REQUIRE(scale_rule == GB_SCALE_RULE_RECIP || scale_rule == GB_SCALE_RULE_DIV, "unknown scale rule %d", scale_rule);
  NormParams p = params_of(a);
  p.q = static_cast<uint8_t*>(q); p.scale = scale; p.s = stream_out; p.scale_rule = scale_rule;
  return forward<true>(a, p, (cudaStream_t)stream);
}

int64_t gb_residual_norm_grad_workspace_bytes(const gb_residual_norm_args* a, const gb_residual_norm_grads* g) {
  return !a || !g || a->T < 1 || a->H < 1 ? 0 : grad_plan(a, g).bytes;
}

int gb_residual_norm_grad(const gb_residual_norm_args* a, const gb_residual_norm_grads* g, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_args(a);
  if (rc != GB_OK) return rc;
  GB_REQUIRE(g != nullptr, "null arguments");
  if (a->T == 0) return GB_OK;
  GB_REQUIRE(g->stream && g->rstd && (!a->pw || (g->post_rstd && a->y)) && (!g->d_gate || a->y), "null pointer argument");
  GB_REQUIRE((!g->d_h || g->d_h_ld >= a->H) && (!g->d_stream || g->d_stream_ld >= a->H), "rows that do not overlap expected");
  GB_REQUIRE((!g->d_w || a->w) && (!g->d_pw || a->pw) && (!g->d_gate || a->gate), "a gradient of what there is not");
  if (gb_sm_count() <= 0) return gb_fail(GB_ECUDA, "no usable CUDA device: %s", gb_last_error());
  const GradPlan plan = grad_plan(a, g);
  if (workspace_bytes < plan.bytes || (plan.bytes > 0 && !workspace))
    return gb_fail(GB_EWORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)plan.bytes);
  GB_REQUIRE(((uintptr_t)workspace & 15u) == 0, "the workspace must be 16-byte aligned");
  NormParams p = params_of(a);
  p.s = const_cast<void*>(g->stream);
  p.rstd = const_cast<float*>(g->rstd); p.post_rstd = const_cast<float*>(g->post_rstd);
  p.dh = g->d_h; p.ds = g->d_stream; p.dh_ld = g->d_h_ld; p.ds_ld = g->d_stream_ld;
  p.dy = g->d_y; p.dr = g->d_r; p.dg = plan.gate_rows ? g->d_gate : nullptr;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part_w = g->d_w ? reinterpret_cast<float*>(ws + plan.w_at) : nullptr;
  p.part_pw = g->d_pw ? reinterpret_cast<float*>(ws + plan.pw_at) : nullptr;
  p.part_g = plan.gate_sums ? reinterpret_cast<float*>(ws + plan.g_at) : nullptr;
  p.means = plan.vec || plan.cached ? nullptr : reinterpret_cast<float*>(ws + plan.means_at);
  p.per_gate = plan.shares.per_gate;
  p.gates = plan.shares.gates > plan.shares.blocks ? (int)plan.shares.gates : 0;
  const bool sums = p.part_w || p.part_pw || p.part_g;
  const cudaStream_t st = (cudaStream_t)stream;
  // all gradients there and asked for
  const bool all = g->d_h && g->d_stream && g->d_y && g->d_r && g->d_w && (!a->pw || g->d_pw) && (!a->gate || g->d_gate);
  const Form form = all && !p.gates ? form_of(a, plan.width) : kAny;
  const int rc2 = with_types(a->dtype, a->stream_dtype, [&](auto t, auto r) -> int {
    using T = decltype(t);
    using R = decltype(r);
    if (!plan.vec && plan.cached)
      return launch_ring<norm_any_rows_grad_kernel<T, R>>((int)plan.shares.blocks, kAnyGradThreads, (size_t)a->H * 20, st, p);
    if (!plan.vec) {
      GB_CUDA_OK(gb_launch(norm_any_grad_kernel<T, R>, dim3((unsigned)a->T), dim3(kAnyThreads), 0, st, p));
      if (!sums) return GB_OK;
      const int64_t column_blocks = (a->H + kAnyThreads - 1) / kAnyThreads, blocks = column_blocks * plan.shares.blocks;
      GB_REQUIRE(blocks < (1ll << 31), "too many gate rows");
      GB_CUDA_OK(gb_launch(norm_any_columns_kernel<T, R>, dim3((unsigned)blocks), dim3(kAnyThreads), 0, st, p, column_blocks));
      return GB_OK;
    }
    for (int k = 0; k < 5; ++k) p.in_at[k] = plan.at[k];
    p.stage_bytes = plan.stage_bytes;
    p.stages = plan.plan.stages;
    p.w_at = plan.weight_at[0]; p.pw_at = plan.weight_at[1]; p.g_at = plan.weight_at[2];
    behind_ring(p, (size_t)p.stages * p.stage_bytes);
    const auto go = [&](auto v, auto r_, auto most) -> int {
      constexpr int kV = decltype(v)::value, kR = decltype(r_)::value, kMost = decltype(most)::value;
      const size_t smem = (size_t)p.stages * p.stage_bytes + plan.fixed;
      return with_form(form, [&](auto f) -> int {
        return launch_ring<norm_rows_grad_kernel<T, R, kV, kR, kMost, decltype(f)::value>>((int)plan.shares.blocks, plan.width.threads, smem, st, p);
      });
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    if (plan.width.v == 2) return go(two, one, integral_constant<int, 1024>());
    if (plan.width.most == 1024) return go(one, one, integral_constant<int, 1024>());
    const bool pairs = p.stages >= 4 && !(p.gates && a->gate_rows % 2);   // two rows at hand, two on their way, both of one gate row
    if (plan.width.most == 640) return pairs ? go(one, two, integral_constant<int, 640>()) : go(one, one, integral_constant<int, 640>());
    return pairs ? go(one, two, integral_constant<int, 256>()) : go(one, one, integral_constant<int, 256>());
  });
  if (rc2 != GB_OK || !sums) return rc2;
  JoinParams j = {};
  j.part[0] = p.part_w; j.part[1] = p.part_pw; j.part[2] = p.part_g;
  j.out[0] = g->d_w; j.out[1] = g->d_pw; j.out[2] = g->d_gate;
  j.type[0] = a->w_dtype; j.type[1] = a->pw_dtype; j.type[2] = a->dtype;
  j.H = a->H; j.shares = plan.shares.blocks; j.gate_shares = plan.shares.per_gate;
  return launch_join(j, (p.part_w ? 1 : 0) + (p.part_pw ? 1 : 0) + (p.part_g ? plan.shares.gates : 0), st);
}

}  // extern "C"
