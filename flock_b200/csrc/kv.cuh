// A KV cache in memory the caller owns, and the kernels that fill and read it
// (flock_kv_* in include/flock_cuda.h).
//
// Cached element types.  f32, bf16 and e4m3 caches hold rows
// [key][kv head][128], the layers' own layout.  The 4-bit cache
// (FLOCK_KV_Q4) holds per head a plane of 64-byte rows [kv head][key][64] and
// a plane of f16 block scales [kv head][key][4]; a block is 32 values along
// the head in the Q4_0 rule (kernels/lib.ts:64 quantRowQ4): d = m / -8 with m
// the first value of largest magnitude, code = clamp(floor(x / d + 8.5), 0,
// 15), value (code - 8) * f16(d), byte i of the block = code i | code i+16
// << 4.  The head's four blocks are interleaved so that one attention lane's
// codes are one aligned load: byte i of block b of a key lies at
// 16 (i / 4) + 4 b + i % 4, of a value row at 8 (i / 2) + 2 b + i % 2.
// Head-major planes keep a head's keys contiguous: its scales (8 bytes a key)
// fill whole sectors, where [key][head] rows would use 8 bytes of each 32.
#pragma once
#include "../../include/flock_cuda.h"
#include "common.cuh"
#include "mbar.cuh"

namespace flock {

constexpr int KV_HD = 128;

// What every kernel here needs of a cache.
struct KvView {
  void* k;
  void* v;
  uint16_t* ks;   // FLOCK_KV_Q4: f16 scales [kv head][capacity][4]
  uint16_t* vs;
  int64_t capacity;
  int n_kv_heads;
};

// f16 magnitude a 4-bit block's scale saturates at: values past 8 * 65504 are
// clamped before the block is coded (as e4m3 saturates at 448).
constexpr float Q4_SCALE_MAX = 65504.0f;
constexpr float Q4_VALUE_MAX = 8.0f * Q4_SCALE_MAX;

// Index of (key, head) in rows of `row` elements: 64-bit, a long cache's
// element offsets pass 2^31.
FLOCK_DEV size_t kv_row(const KvView& c, int64_t key, int head) {
  return ((size_t)key * c.n_kv_heads + head) * KV_HD;
}
FLOCK_DEV size_t q4_row(const KvView& c, int64_t key, int head) {
  return ((size_t)head * c.capacity + key);
}

// Elements 4 lane .. 4 lane + 3 of a cached row, widened exactly.
template <int KV, bool IS_K>
FLOCK_DEV float4 kv_load4(const KvView& c, int64_t key, int head, int lane) {
  const void* base = IS_K ? c.k : c.v;
  if constexpr (KV == FLOCK_KV_Q4) {
    const size_t row = q4_row(c, key, head);
    const int b = lane >> 3, i0 = (4 * lane) & 31, byte0 = i0 & 15, sh = i0 & 16 ? 4 : 0;
    const uint8_t* r = static_cast<const uint8_t*>(base) + row * 64;
    uint32_t w;
    if (IS_K) {
      w = *reinterpret_cast<const uint32_t*>(r + 16 * (byte0 >> 2) + 4 * b);
    } else {
      const uint32_t lo = *reinterpret_cast<const uint16_t*>(r + 8 * (byte0 >> 1) + 2 * b);
      const uint32_t hi = *reinterpret_cast<const uint16_t*>(r + 8 * (byte0 >> 1) + 8 + 2 * b);
      w = lo | (hi << 16);
    }
    const float d = __half2float(__ushort_as_half((IS_K ? c.ks : c.vs)[row * 4 + b]));
    w = (w >> sh) & 0x0F0F0F0Fu;
    float x, y, z, t;
    dec_nib4(w, x, y, z, t);
    return make_float4(fmul(x, d), fmul(y, d), fmul(z, d), fmul(t, d));
  } else if constexpr (KV == FLOCK_KV_FP8) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) +
                                                          kv_row(c, key, head) + 4 * lane);
    const float2 a = fp8x2_widen(w), b = fp8x2_widen(w >> 16);
    return make_float4(a.x, a.y, b.x, b.y);
  } else if constexpr (KV == FLOCK_KV_BF16) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) +
                                                    kv_row(c, key, head) + 4 * lane);
    const float2 a = bf16x2_widen(w.x), b = bf16x2_widen(w.y);
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    return *reinterpret_cast<const float4*>(static_cast<const float*>(base) +
                                            kv_row(c, key, head) + 4 * lane);
  }
}

// One row (lane: elements 4 lane .. 4 lane + 3) into the 4-bit cache.
//
// The code of x is floor(x * (1 / d) + 8.5) in f64 with one rounding each, as
// flock_quant_q4 decides it: the codes of a row are the host's bytes.  f32
// gives the same wherever it lands further from an integer than its own error
// (2.5e-6: a reciprocal and a product of relative error 2^-22, the sum's 2^-20);
// a warp with a value within 1e-5 of one works its codes out in f64.  A block
// with a NaN gets a NaN scale (every value of it reads back NaN).
template <bool IS_K>
FLOCK_DEV void q4_store_row(const KvView& c, int64_t key, int head, float4 x4, int lane) {
  float x[4] = {x4.x, x4.y, x4.z, x4.w};
  auto mag = [](float v) { return __float_as_uint(v) & 0x7FFFFFFFu; };
  uint32_t top_bits = max(max(mag(x[0]), mag(x[1])), max(mag(x[2]), mag(x[3])));
  const bool nan = top_bits > 0x7F800000u;
  if (__any_sync(0xffffffffu, top_bits > __float_as_uint(Q4_VALUE_MAX))) {
    top_bits = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {  // a NaN becomes a bound, its block is marked below
      x[i] = fminf(fmaxf(x[i], -Q4_VALUE_MAX), Q4_VALUE_MAX);
      top_bits = max(top_bits, mag(x[i]));
    }
  }
  const uint32_t own = top_bits;
#pragma unroll
  for (int s = 1; s < 8; s <<= 1)  // over the block's 8 lanes
    top_bits = max(top_bits, __shfl_xor_sync(0xffffffffu, top_bits, s));
  // the first value of that magnitude: the first such lane's first
  const uint32_t octet = 0xFFu << (lane & 24);
  const int at = __ffs(__ballot_sync(0xffffffffu, own == top_bits) & octet) - 1;
  const float first = mag(x[0]) == own   ? x[0]
                      : mag(x[1]) == own ? x[1]
                      : mag(x[2]) == own ? x[2]
                                         : x[3];
  const float top = __shfl_sync(0xffffffffu, first, at);
  const bool nan_block = (__ballot_sync(0xffffffffu, nan) & octet) != 0;

  uint32_t code = 0;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(top));
  inv = top == 0.0f ? 0.0f : fmul(inv, -8.0f);
  // too small for f32's reciprocal: also f64
  bool close = top != 0.0f && fabsf(top) < 1e-30f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float t = ffma(x[i], inv, 8.5f);
    // 2^23 added rounding down leaves floor(t) in the low bits
    const float f = __fadd_rd(t, 8388608.0f);
    const float frac = fsub(t, fsub(f, 8388608.0f));
    close |= frac < 1e-5f || frac > 0.99999f;
    code |= min(__float_as_uint(f) & 31u, 15u) << (8 * i);
  }
  if (__any_sync(0xffffffffu, close)) {
    const double d = (double)top / -8.0;
    const double inv64 = d == 0.0 ? 0.0 : 1.0 / d;
    code = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const double t = __dadd_rn(__dmul_rn((double)x[i], inv64), 8.5);
      code |= (uint32_t)min(__double2loint(__dadd_rd(t, 4503599627370496.0)), 15) << (8 * i);
    }
  }
  // lanes 0-3 of a block hold values 0..15 (low nibbles), lanes 4-7 16..31
  const uint32_t high = __shfl_xor_sync(0xffffffffu, code, 4);
  const size_t row = q4_row(c, key, head);
  const int b = lane >> 3, p = lane & 7;
  if (p < 4) {
    const uint32_t w = code | (high << 4);  // bytes 4 p .. 4 p + 3 of block b
    uint8_t* r = static_cast<uint8_t*>(IS_K ? c.k : c.v) + row * 64;
    if (IS_K) {
      *reinterpret_cast<uint32_t*>(r + 16 * p + 4 * b) = w;
    } else {
      *reinterpret_cast<uint16_t*>(r + 16 * p + 2 * b) = (uint16_t)w;
      *reinterpret_cast<uint16_t*>(r + 16 * p + 8 + 2 * b) = (uint16_t)(w >> 16);
    }
  }
  if (p == 0)  // top / -8 is exact in f32 down to its subnormals, which round to a zero scale
    (IS_K ? c.ks : c.vs)[row * 4 + b] =
        nan_block ? (uint16_t)0x7E00u : __half_as_ushort(__float2half_rn(fmul(top, -0.125f)));
}

template <int KV, bool IS_K>
FLOCK_DEV void kv_store4(const KvView& c, int64_t key, int head, float4 x, int lane) {
  void* base = IS_K ? c.k : c.v;
  if constexpr (KV == FLOCK_KV_Q4) {
    q4_store_row<IS_K>(c, key, head, x, lane);
  } else if constexpr (KV == FLOCK_KV_FP8) {
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(base) + kv_row(c, key, head) + 4 * lane) =
        (uint32_t)fp8_bits(x.x) | (uint32_t)fp8_bits(x.y) << 8 | (uint32_t)fp8_bits(x.z) << 16 |
        (uint32_t)fp8_bits(x.w) << 24;
  } else if constexpr (KV == FLOCK_KV_BF16) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + kv_row(c, key, head) + 4 * lane) =
        make_uint2((uint32_t)bf16_bits(x.x) | (uint32_t)bf16_bits(x.y) << 16,
                   (uint32_t)bf16_bits(x.z) | (uint32_t)bf16_bits(x.w) << 16);
  } else {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + kv_row(c, key, head) + 4 * lane) = x;
  }
}

// One warp per (token, head), a row of k and one of v; grid (8 tokens, head), so
// no index is divided (64-bit divisions were half the instructions).  Bound: the
// f32 rows' bytes.  Two or four tokens a warp, to have more loads in flight,
// measured slower.
template <int KV>
static __global__ void __launch_bounds__(256) k_kv_append(KvView c, const float* k, const float* v,
                                                          int64_t row_stride, int64_t pos, int n) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int head = blockIdx.y;
  if (tok >= n) return;
  const int64_t src = tok * row_stride + (int64_t)head * KV_HD + 4 * lane;
  const float4 kx = __ldg(reinterpret_cast<const float4*>(k + src));
  const float4 vx = __ldg(reinterpret_cast<const float4*>(v + src));
  kv_store4<KV, true>(c, pos + tok, head, kx, lane);
  kv_store4<KV, false>(c, pos + tok, head, vx, lane);
}

// The cached rows [pos, pos + n) as f32 [n][kv heads][128].
template <int KV>
static __global__ void __launch_bounds__(256) k_kv_read(KvView c, int64_t pos, int n, float* k,
                                                        float* v) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t tok = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int head = blockIdx.y;
  if (tok >= n) return;
  const size_t dst = ((size_t)tok * c.n_kv_heads + head) * KV_HD + 4 * lane;
  const float4 kx = kv_load4<KV, true>(c, pos + tok, head, lane);
  const float4 vx = kv_load4<KV, false>(c, pos + tok, head, lane);
  *reinterpret_cast<float4*>(k + dst) = kx;
  *reinterpret_cast<float4*>(v + dst) = vx;
}

// Queries at positions pos .. pos + n_queries - 1, row i of q [n_heads][128]
// at q + i * q_stride.  Query position p sees key j iff j <= p and (window
// == 0 or j > p - window or j < sinks).
struct KvAttnArgs {
  KvView c;
  const float* q;
  float* out;
  int64_t q_stride, out_stride;
  int64_t pos;
  const int* ctl;  // a layer's step control: the position is ctl[0], pos its bound; or null
  int* err;        // a layer's error word: nonzero when a bounded wait ran out; or null
  int n_queries, n_heads, window, sinks;
};
// After griddepcontrol.wait: an earlier kernel of the step writes ctl.
FLOCK_DEV int kv_attn_pos(const KvAttnArgs& a) { return a.ctl ? a.ctl[0] : (int)a.pos; }

}  // namespace flock
