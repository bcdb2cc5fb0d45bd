// Attention of a few query rows (one decoded token's heads of a kv head, or a
// short draft) over a cache: k_kv_rows.
//
// Bound: the cache's bytes from HBM (a 4-bit key of one head is 72 + 72 bytes),
// and, near it, the instructions that widen the codes.  So every code is
// widened once, in registers, straight into the operand of a matrix
// instruction, for all query heads that share the kv head.
//
// mma.sync m16n8k16 (f32 accumulation) rather than tcgen05: with two to eight
// live rows there is nothing to amortise a pass of the operands through shared
// memory and tensor memory over; this path takes cached bytes from shared
// memory to the operand registers with no store in between.  Keys (then head
// dimensions) are the operand's 16 rows and query rows its 8 columns: the
// other way round 16 rows would be mostly empty and every step twice as long.
//
// f32 results from 16-bit operands.  Codes and e4m3 values are f16 values, so
// there queries and softmax weights are split as hi + lo, two f16 of 11 bits
// (22 bits; scaled by powers of two so that f16's range never cuts a part that
// matters).  bf16 and f32 elements need f32's range: hi + mid + lo, three bf16
// of 8 bits.  The parts sit in neighbouring COLUMNS, which a lane's accumulator
// holds side by side: one instruction multiplies both, an addition joins them.
//
// 4-bit blocks.  Codes minus 8 are the operands.  (A code left in an f16's low
// bits is the subnormal c 2^-24 and needs no more than an AND, but the tensor
// cores align a subnormal's product as if it were normal and drop the bits below:
// errors of 3e-6 instead of 3e-7.)  A block's products are multiplied by the
// key's scale in f32, one accumulator per block.  Values: the scale joins the
// weight, so the weight operand differs per block.  Scales further apart than
// 2^KR_SPREAD (a warp keeps watch) would leave the smaller ones' products too few
// bits in f16: the warp then begins again with the products as three bf16 parts.
//
// Work split: CTA (split z, row tile, kv head), its warps taking 16-key groups
// in turn, each with its own cp.async ring, running maximum, sum and output;
// warps join in shared memory, CTAs in the workspace, the last to arrive adding
// the splits in order (results do not depend on who is last).
#pragma once
#include <type_traits>

#include "kv.cuh"

namespace flock {

constexpr int KR_GROUP = 16;  // keys per warp step
constexpr int KR_SPREAD = 14;  // 4-bit value scales a warp takes in f16: 2^14 apart
constexpr int KR_MAX_ITEMS = 4096;  // (row tile, kv head) pairs that may be split: arrival counters
constexpr size_t KR_PART_OFFSET = KR_MAX_ITEMS * 4;

struct KvRowsArgs {
  KvAttnArgs a;
  int rows;         // n_queries * group: row r is query r / group, head r % group
  int group;        // query heads per kv head
  uint32_t* count;  // [items], zero between calls
  float* part;      // [item][gridDim.x][RT][128], then [item][gridDim.x][RT][2] (m, l)
};

// Shared-memory layout of one warp's 16-key stage, per cached type, for NT
// column tiles.  Key rows are read 16 bytes a lane, eight lanes covering 64
// bytes of two keys; value rows 8 or 16 bytes a lane, eight lanes covering
// pieces of four keys two apart.  Padding keeps both free of bank conflicts.
template <int KV, int NT>
struct KrTile;
template <int NT>
struct KrTile<FLOCK_KV_Q4, NT> {
  static constexpr int ROW = 64, K_STRIDE = 64, WARPS = NT == 1 ? 16 : 12, STAGES = 5;
  static constexpr int SCALES = 2 * KR_GROUP * 8;
};
template <int NT>
struct KrTile<FLOCK_KV_FP8, NT> {
  static constexpr int ROW = 128, K_STRIDE = 192, WARPS = 8, STAGES = 4, SCALES = 0;
};
template <int NT>
struct KrTile<FLOCK_KV_BF16, NT> {
  static constexpr int ROW = 256, K_STRIDE = 320, WARPS = 8, STAGES = 2, SCALES = 0;
};
template <int NT>
struct KrTile<FLOCK_KV_F32, NT> {
  static constexpr int ROW = 512, K_STRIDE = 576, WARPS = 6, STAGES = 2, SCALES = 0;
};
template <int KV, int NT>
struct KrLayout : KrTile<KV, NT> {
  using T = KrTile<KV, NT>;
  static constexpr bool F16 = KV == FLOCK_KV_Q4 || KV == FLOCK_KV_FP8;
  static constexpr int RT = F16 ? 4 * NT : 4;  // query rows per CTA
  static constexpr int V_PAIR = 2 * T::ROW + 32;  // two keys' value rows
  static constexpr int V_OFF = KR_GROUP * T::K_STRIDE;
  static constexpr int S_OFF = V_OFF + KR_GROUP / 2 * V_PAIR;
  static constexpr int STAGE = S_OFF + T::SCALES;
  static constexpr int THREADS = 32 * T::WARPS;
  static constexpr size_t SMEM = (size_t)T::WARPS * T::STAGES * STAGE;
};

FLOCK_DEV void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
FLOCK_DEV void cp_async8(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 8 : 0)
               : "memory");
}
FLOCK_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
FLOCK_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// d = a b + c; not volatile, so that the compiler may order it freely.
template <bool F16>
FLOCK_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                     float c1, float c2, float c3) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
          "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
          "f"(c3));
}
template <bool F16>
FLOCK_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma16<F16>(d, a, b0, b1, d[0], d[1], d[2], d[3]);
}
FLOCK_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 -> a pair of 16-bit values (nearest even), lo in the low half.
FLOCK_DEV uint32_t bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
FLOCK_DEV uint32_t hf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
FLOCK_DEV float2 h2f2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// x = hi + lo (f16), x = hi + mid + lo (bf16), for two values; every
// difference is exact.
FLOCK_DEV void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = hf2(x, y);
  const float2 f = h2f2(hi);
  lo = hf2(fsub(x, f.x), fsub(y, f.y));
}
FLOCK_DEV void split_bf16(float x, float y, uint32_t (&w)[3]) {
#pragma unroll
  for (int i = 0; i < 3; i++) {
    w[i] = bf2(x, y);
    x = fsub(x, __uint_as_float(w[i] << 16));
    y = fsub(y, __uint_as_float(w[i] & 0xffff0000u));
  }
}
// (a & b) | c in one instruction.
FLOCK_DEV uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
FLOCK_DEV uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
FLOCK_DEV uint32_t hmul2_u(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
FLOCK_DEV __half2 as_h2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
FLOCK_DEV uint32_t hadd2_u(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
FLOCK_DEV uint32_t hneg2_u(uint32_t a) {
  const __half2 r = __hneg2(*reinterpret_cast<const __half2*>(&a));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// An 8 x 8 matrix of 16-bit values, a row's eight over four lanes, transposed.
FLOCK_DEV uint32_t movm(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
// The eight codes of a word -> (code - 8) as four f16 pairs: 0x6400 | code is
// the f16 1024 + code, 0x6400 | 16 code is 1024 + 16 code, and the rest is
// taken off exactly.  v[e]: bits 4 e .. 4 e + 3 of both halfwords.
FLOCK_DEV void nib_f16(uint32_t w, uint32_t (&v)[4]) {
  const uint32_t hi = w >> 8;
  v[0] = hadd2_u(and_or(w, 0x000F000Fu, 0x64006400u), 0xE408E408u);                // - 1032
  v[1] = hfma2_u(and_or(w, 0x00F000F0u, 0x64006400u), 0x2C002C00u, 0xD480D480u);   // / 16 - 72
  v[2] = hadd2_u(and_or(hi, 0x000F000Fu, 0x64006400u), 0xE408E408u);
  v[3] = hfma2_u(and_or(hi, 0x00F000F0u, 0x64006400u), 0x2C002C00u, 0xD480D480u);
}
// Two e4m3 in the low half -> f16 pair, exactly.
FLOCK_DEV uint32_t fp8_f16(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The head dimension of row g (half 0) or g + 8 (half 1) of output tile u (0-7).
template <int KV>
FLOCK_DEV int kr_vdim(int u, int half, int g) {
  if (KV == FLOCK_KV_Q4) {  // nibble e of the lane's two bytes of block u / 2
    const int e = 2 * (u & 1) + half;
    return 32 * (u >> 1) + 16 * (e & 1) + 2 * g + (e >> 1);
  }
  if (KV == FLOCK_KV_FP8) return 16 * g + 2 * u + half;
  if (KV == FLOCK_KV_BF16) return 64 * (u >> 2) + 8 * g + 2 * (u & 3) + half;
  return 32 * (u >> 1) + 4 * g + 2 * (u & 1) + half;
}

// One stage of keys key0 .. key0 + 15 of a head into shared memory; keys
// outside [from, to) are zero-filled, so what lies there cannot reach a
// product.  kb, vb: the head's first rows; sb: this lane's scale plane at the
// head's first row.
template <int KV, int NT, bool WHOLE>
FLOCK_DEV void kr_load(uint32_t stage, const uint8_t* kb, const uint8_t* vb, const uint8_t* sb,
                       int64_t step, int key0, int from, int to, int lane) {
  using L = KrLayout<KV, NT>;
  constexpr int CHUNKS = L::ROW / 16;  // 16-byte chunks of a row
  constexpr int ROWS = 32 / CHUNKS;    // rows a warp's 32 chunks cover (f32: one)
  const int r0 = lane / CHUNKS, ch = lane % CHUNKS;
  // a 4-bit head's rows are contiguous, step = 64
  const uint8_t* ks = kb + (int64_t)(key0 + r0) * step + ch * 16;
  const uint8_t* vs = vb + (int64_t)(key0 + r0) * step + ch * 16;
  const uint32_t kd = stage + r0 * L::K_STRIDE + ch * 16;
  const uint32_t vd = stage + L::V_OFF + (r0 >> 1) * L::V_PAIR + (r0 & 1) * L::ROW + ch * 16;
#pragma unroll
  for (int i = 0; i < KR_GROUP / ROWS; i++) {
    const bool ok = WHOLE || (key0 + r0 + i * ROWS >= from && key0 + r0 + i * ROWS < to);
    const int64_t off = ok ? (int64_t)(i * ROWS) * step : (int64_t)(from - key0 - r0) * step;
    // value rows r0 + i ROWS: whole pairs apart, or the second of a pair
    const uint32_t vo = ROWS >= 2 ? i * (ROWS / 2) * L::V_PAIR : (i / 2) * L::V_PAIR + (i % 2) * L::ROW;
    cp_async16(kd + i * ROWS * L::K_STRIDE, ks + off, ok);
    cp_async16(vd + vo, vs + off, ok);
  }
  if (KV == FLOCK_KV_Q4) {
    const int r = lane & 15;
    const bool ok = WHOLE || (key0 + r >= from && key0 + r < to);
    cp_async8(stage + L::S_OFF + lane * 8, sb + (int64_t)(key0 + r) * 8, ok);
  }
}

// Key splits of a row tile: every warp at least a group of keys, as far as the
// grid allows.  Joining splits costs about 2.5 us, a group about 0.5: up to four
// groups a warp one CTA reads them all (320 keys: 4.9 us against 7 in two).
__host__ __device__ inline int kr_splits(int64_t groups, int warps, int64_t most) {
  const int64_t want = (groups + warps - 1) / warps;
  return want <= 4 || most < 2 ? 1 : (int)(want < most ? want : most);
}

FLOCK_DEV uint4 ld_u4(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
FLOCK_DEV uint2 ld_u2(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }
FLOCK_DEV uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Lane (g, c) = (lane / 4, lane % 4).  Scores: keys g and g + 8 of the stage,
// query row c of each column tile (f16: tile n holds rows 4 n .. 4 n + 3 as hi,
// lo columns; bf16: tile 0 hi, mid and tile 1 lo of rows 0-3).
template <int KV, int NT>
static __global__ void __launch_bounds__(KrLayout<KV, NT>::THREADS, 1)
    k_kv_rows(const KvRowsArgs p) {
  using L = KrLayout<KV, NT>;
  constexpr int RT = L::RT;
  constexpr bool Q4 = KV == FLOCK_KV_Q4;
  constexpr bool F16 = L::F16;
  constexpr int RL = F16 ? NT : 1;  // query rows of a lane
  extern __shared__ __align__(16) uint8_t kr_smem[];
  __shared__ float s_ml[L::WARPS][RT][2];
  __shared__ uint2 s_q[NT][8][32];    // the query operand: [tile][QK step][lane]
  __shared__ float s_unscale[RT];
  __shared__ int s_last;
  pdl_launch_dependents();
  pdl_wait();
  const KvAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int z = blockIdx.x, tile = blockIdx.y, head = blockIdx.z;
  const int first_q = tile * RT / p.group;
  const int last_q = (min(p.rows, (tile + 1) * RT) - 1) / p.group;
  // keys that some row of the tile sees: sinks [0, sk), then [lo, hi)
  const int pos = kv_attn_pos(a);
  const int hi = pos + last_q + 1;
  const int lo = a.window && pos + first_q + 1 > a.window ? pos + first_q + 1 - a.window : 0;
  const int sk = min(a.sinks, lo);
  const int sink_groups = (sk + KR_GROUP - 1) / KR_GROUP;
  const int lo16 = lo & ~(KR_GROUP - 1);
  const int groups = sink_groups + (hi - lo16 + KR_GROUP - 1) / KR_GROUP;
  // the splits these groups are worth, of those the grid has (see kr_splits)
  const int splits = kr_splits(groups, L::WARPS, gridDim.x);
  if (z >= splits) return;
  const int g0 = (int)((int64_t)z * groups / splits), g1 = (int)((int64_t)(z + 1) * groups / splits);
  // a row's own keys: sinks [0, row_sk), then [row_lo, row_hi)
  int row_lo[RL], row_hi[RL], row_sk[RL];
  int max_lo = 0, min_hi = hi;  // a group inside [max_lo, min_hi) is visible to every row
#pragma unroll
  for (int n = 0; n < RL; n++) {
    row_hi[n] = pos + min(tile * RT + 4 * n + c, p.rows - 1) / p.group + 1;
    row_lo[n] = a.window && row_hi[n] > a.window ? row_hi[n] - a.window : 0;
    row_sk[n] = min(a.sinks, row_lo[n]);
  }
  max_lo = a.window && pos + last_q + 1 > a.window ? pos + last_q + 1 - a.window : 0;
  min_hi = pos + first_q + 1;

  const uint32_t ring = smem_u32(kr_smem) + warp * L::STAGES * L::STAGE;
  const size_t hbase = Q4 ? q4_row(a.c, 0, head) * 64 : (size_t)head * L::ROW;
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + hbase;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + hbase;
  const uint8_t* sb = Q4 ? reinterpret_cast<const uint8_t*>((lane < 16 ? a.c.ks : a.c.vs) +
                                                            q4_row(a.c, 0, head) * 4)
                         : nullptr;
  const int64_t step = Q4 ? 64 : (int64_t)a.c.n_kv_heads * L::ROW;
  auto key_of = [&](int grp) {
    return grp < sink_groups ? grp * KR_GROUP : lo16 + (grp - sink_groups) * KR_GROUP;
  };
  auto fetch = [&](int grp, int st) {
    if (grp < g1) {
      const bool sink = grp < sink_groups;
      const int key0 = key_of(grp), from = sink ? 0 : lo, to = sink ? sk : hi;
      const uint32_t dst = ring + st * L::STAGE;
      if (key0 >= from && key0 + KR_GROUP <= to)
        kr_load<KV, NT, true>(dst, kb, vb, sb, step, key0, from, to, lane);
      else
        kr_load<KV, NT, false>(dst, kb, vb, sb, step, key0, from, to, lane);
    }
    cp_async_commit();
  };
  // The query rows' loads go out before the cached bytes': behind the rings'
  // prefetch (hundreds of KB an SM) they would wait for all of it.
  static_assert(RT <= L::WARPS, "a warp splits a query row");
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (warp < RT && tile * RT + warp < p.rows) {
    const int rr = tile * RT + warp;
    x = __ldg(reinterpret_cast<const float4*>(
        a.q + (rr / p.group) * a.q_stride + ((int64_t)head * p.group + rr % p.group) * KV_HD +
        4 * lane));
  }
#pragma unroll
  for (int s = 0; s < L::STAGES - 1; s++) fetch(g0 + warp + s * L::WARPS, s);

  // The query operand: the parts of q log2(e) / sqrt(128), for f16 scaled by
  // a power of two that brings the row's largest into [2^13, 2^14).  A warp
  // splits a row, four neighbouring dimensions a lane: one entry of each part.
  if (warp < RT) {
    const int r = warp;
    const float k = __double2float_rn(1.4426950408889634 / sqrt(128.0));
    x = make_float4(fmul(x.x, k), fmul(x.y, k), fmul(x.z, k), fmul(x.w, k));
    // where these four dimensions meet a lane's cached bytes: step ks, lane column qc
    const int qc = Q4 || KV == FLOCK_KV_F32 ? lane & 3 : KV == FLOCK_KV_FP8 ? (lane >> 2) & 3 : (lane >> 1) & 3;
    const int ks = Q4 || KV == FLOCK_KV_F32 ? lane >> 2
                   : KV == FLOCK_KV_FP8     ? (lane >> 4) * 4 + (lane & 3)
                                            : (lane >> 3) * 2 + (lane & 1);
    if (F16) {
      float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int biased = (int)(__float_as_uint(top) >> 23);
      // (up to f32's largest, whose exponent here is 114)
      const int e = biased == 0 ? 0 : max(-100, min(114, biased - 127 - 13));
      const float scale = __uint_as_float((uint32_t)(127 - e) << 23);
      if (Q4) {  // pairs two apart: bytes 0 and 2, 1 and 3 of a code word
        const float y = x.y;
        x.y = x.z;
        x.z = y;
      }
      uint2 h, l;
      split_f16(fmul(x.x, scale), fmul(x.y, scale), h.x, l.x);
      split_f16(fmul(x.z, scale), fmul(x.w, scale), h.y, l.y);
      s_q[r / 4][ks][4 * (2 * (r % 4)) + qc] = h;
      s_q[r / 4][ks][4 * (2 * (r % 4) + 1) + qc] = l;
      if (lane == 0) s_unscale[r] = __uint_as_float((uint32_t)(127 + e) << 23);
    } else {
      uint32_t w0[3], w1[3];
      split_bf16(x.x, x.y, w0);
      split_bf16(x.z, x.w, w1);
      s_q[0][ks][4 * (2 * r) + qc] = make_uint2(w0[0], w1[0]);
      s_q[0][ks][4 * (2 * r + 1) + qc] = make_uint2(w0[1], w1[1]);
      s_q[1][ks][4 * (2 * r) + qc] = make_uint2(w0[2], w1[2]);
      s_q[1][ks][4 * (2 * r + 1) + qc] = make_uint2(0, 0);
    }
  }
  __syncthreads();
  uint2 qb[NT][8];
  float unscale[RL];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int ks = 0; ks < 8; ks++) qb[n][ks] = s_q[n][ks][lane];
#pragma unroll
  for (int n = 0; n < RL; n++) unscale[n] = F16 ? s_unscale[4 * n + c] : 1.0f;
  float o[8][NT][4];
  // Weights are 2^(s - base), base = m - 10, m a running maximum that may lag by
  // 2^4: at most 2^14, inside f16, and a lo part loses nothing above 2^-35 of
  // the largest.  Value scales are divided by 2^dexp, a bound on those so far,
  // which the outputs get back at the end; those down to 2^-14 of it leave the
  // largest weight's products at 2^-4 and up, where a lo part's error is 2^-21.
  constexpr float HEADROOM = F16 ? 10.0f : 0.0f, LAG = F16 ? 4.0f : 8.0f;
  float m[RL], l[RL], base[RL];
  int dexp = -14;
  // The warp's groups; false: the value scales lie too far apart, and nothing of
  // this pass counts.  WIDE: whatever the scales.
  auto pass = [&](auto wide) -> bool {
    constexpr bool WIDE = decltype(wide)::value;
#pragma unroll
    for (int u = 0; u < 8; u++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[u][n][e] = 0.0f;
#pragma unroll
    for (int n = 0; n < RL; n++) {
      m[n] = -INFINITY;
      l[n] = base[n] = 0.0f;
    }
    dexp = WIDE ? 0 : -14;
    uint32_t dlim = 0x04000400u, dnorm = 0x74007400u;  // f16 pairs 2^dexp and 2^-dexp
    uint32_t dlow = 0, dmin = 0xFFFFFFFFu;  // u16 pairs: 2^(dexp - KR_SPREAD); smallest scale but 0, less 1

    int st = 0;
    for (int grp = g0 + warp; grp < g1; grp += L::WARPS) {
      cp_async_wait<L::STAGES - 2>();
      __syncwarp();  // the stage has landed for every lane, and every lane is done with the last one
      fetch(grp + (L::STAGES - 1) * L::WARPS, st == 0 ? L::STAGES - 1 : st - 1);
      const uint8_t* stage = kr_smem + (warp * L::STAGES + st) * L::STAGE;
      // ------------------------------------------------------------- scores
      float s[RL][2];  // keys g, g + 8
      const uint8_t* ka = stage + g * L::K_STRIDE + 16 * c;
      if constexpr (Q4) {
        const uint4 w0 = ld_u4(ka), w1 = ld_u4(ka + 8 * L::K_STRIDE);
        const uint2 e0 = ld_u2(stage + L::S_OFF + 8 * g), e1 = ld_u2(stage + L::S_OFF + 8 * g + 64);
#pragma unroll
        for (int n = 0; n < RL; n++) s[n][0] = s[n][1] = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; b++) {
          uint32_t x[4], y[4];
          nib_f16(word_of(w0, b), x);
          nib_f16(word_of(w1, b), y);
          const float2 d0 = h2f2(b < 2 ? e0.x : e0.y), d1 = h2f2(b < 2 ? e1.x : e1.y);
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float acc[4];
            const uint32_t a0[4] = {x[0], y[0], x[2], y[2]}, a1[4] = {x[1], y[1], x[3], y[3]};
            mma16<F16>(acc, a0, qb[n][2 * b].x, qb[n][2 * b].y, 0.f, 0.f, 0.f, 0.f);
            mma16<F16>(acc, a1, qb[n][2 * b + 1].x, qb[n][2 * b + 1].y);
            s[n][0] = ffma(b & 1 ? d0.y : d0.x, fadd(acc[0], acc[1]), s[n][0]);
            s[n][1] = ffma(b & 1 ? d1.y : d1.x, fadd(acc[2], acc[3]), s[n][1]);
          }
        }
      } else {
        float acc[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[n][h][e] = 0.0f;
        if constexpr (KV == FLOCK_KV_FP8) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint4 w0 = ld_u4(ka + 64 * h), w1 = ld_u4(ka + 64 * h + 8 * L::K_STRIDE);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t x = word_of(w0, i), y = word_of(w1, i);
              const uint32_t av[4] = {fp8_f16(x), fp8_f16(y), fp8_f16(x >> 16), fp8_f16(y >> 16)};
#pragma unroll
              for (int n = 0; n < NT; n++)
                mma16<F16>(acc[n][i & 1], av, qb[n][4 * h + i].x, qb[n][4 * h + i].y);
            }
          }
        } else if constexpr (KV == FLOCK_KV_BF16) {
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const uint4 w0 = ld_u4(ka + 64 * h), w1 = ld_u4(ka + 64 * h + 8 * L::K_STRIDE);
            const uint32_t a0[4] = {w0.x, w1.x, w0.y, w1.y}, a1[4] = {w0.z, w1.z, w0.w, w1.w};
#pragma unroll
            for (int n = 0; n < NT; n++) {
              mma16<F16>(acc[n][0], a0, qb[n][2 * h].x, qb[n][2 * h].y);
              mma16<F16>(acc[n][1], a1, qb[n][2 * h + 1].x, qb[n][2 * h + 1].y);
            }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 8; ks++) {
            const uint4 w0 = ld_u4(ka + 64 * ks), w1 = ld_u4(ka + 64 * ks + 8 * L::K_STRIDE);
            uint32_t x0[3], x1[3], y0[3], y1[3];
            split_bf16(__uint_as_float(w0.x), __uint_as_float(w0.y), x0);
            split_bf16(__uint_as_float(w0.z), __uint_as_float(w0.w), x1);
            split_bf16(__uint_as_float(w1.x), __uint_as_float(w1.y), y0);
            split_bf16(__uint_as_float(w1.z), __uint_as_float(w1.w), y1);
#pragma unroll
            for (int part = 0; part < 3; part++) {
              const uint32_t av[4] = {x0[part], y0[part], x1[part], y1[part]};
#pragma unroll
              for (int n = 0; n < (part == 2 ? 1 : NT); n++)  // lo lo is below f32's last bit
                mma16<F16>(acc[n][part & 1], av, qb[n][ks].x, qb[n][ks].y);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < RL; n++) {
          s[n][0] = fadd(fadd(acc[n][0][0], acc[n][1][0]), fadd(acc[n][0][1], acc[n][1][1]));
          s[n][1] = fadd(fadd(acc[n][0][2], acc[n][1][2]), fadd(acc[n][0][3], acc[n][1][3]));
          if (!F16) {
            s[n][0] = fadd(s[n][0], fadd(acc[1][0][0], acc[1][1][0]));
            s[n][1] = fadd(s[n][1], fadd(acc[1][0][2], acc[1][1][2]));
          }
        }
      }
      const int key0 = key_of(grp);
      {  // masks, only where the group is not wholly visible to every row
        const bool sink = grp < sink_groups;
        if (sink ? key0 + KR_GROUP > sk : key0 < max_lo || key0 + KR_GROUP > min_hi) {
#pragma unroll
          for (int n = 0; n < RL; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int key = key0 + g + 8 * i;
              // every row sees the tile's sinks; a row's own may reach into the main range
              const bool seen = sink ? key < sk
                                     : key >= lo && key < row_hi[n] && (key >= row_lo[n] || key < row_sk[n]);
              if (!seen) s[n][i] = -INFINITY;
            }
        }
      }
      // ------------------------------------------------------------ softmax
      // 4-bit: the value scales of the lane's two keys, a block's pair a word
      uint32_t vd[4];
      uint32_t dmax = 0;
      bool grow = false;
      if constexpr (Q4) {
        const uint2 e0 = ld_u2(stage + L::S_OFF + 128 + 8 * g), e1 = ld_u2(stage + L::S_OFF + 192 + 8 * g);
        vd[0] = __byte_perm(e0.x, e1.x, 0x5410);
        vd[1] = __byte_perm(e0.x, e1.x, 0x7632);
        vd[2] = __byte_perm(e0.y, e1.y, 0x5410);
        vd[3] = __byte_perm(e0.y, e1.y, 0x7632);
        if (!WIDE) {
          // magnitudes order as their bits do
          const uint32_t m0 = e0.x & 0x7FFF7FFFu, m1 = e0.y & 0x7FFF7FFFu, m2 = e1.x & 0x7FFF7FFFu,
                         m3 = e1.y & 0x7FFF7FFFu;
          const uint32_t h = __vimax3_u16x2(__vmaxu2(m0, m1), m2, m3);
          dmin = __viaddmin_u16x2(m3, 0xFFFFFFFFu,
                 __viaddmin_u16x2(m2, 0xFFFFFFFFu,
                 __viaddmin_u16x2(m1, 0xFFFFFFFFu, __viaddmin_u16x2(m0, 0xFFFFFFFFu, dmin))));
          grow = (__hgt2_mask(as_h2(h), as_h2(dlim)) | __hlt2_mask(as_h2(dmin), as_h2(dlow))) != 0;
          dmax = max(h & 0xFFFFu, h >> 16);
        }
      }
      float top[RL];
#pragma unroll
      for (int n = 0; n < RL; n++) {
        top[n] = fmaxf(s[n][0], s[n][1]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], d));
        top[n] = fmul(top[n], unscale[n]);
        grow = grow || top[n] > fadd(m[n], LAG);
      }
      if (__any_sync(0xffffffffu, grow)) {
        float fd = 1.0f;
        if (Q4 && !WIDE) {
          dmax = __reduce_max_sync(0xffffffffu, dmax);
          const int ne = max(dexp, min((int)(dmax >> 10) - 14, 16));  // below 2^(exponent - 14)
          fd = __uint_as_float((uint32_t)(127 + dexp - ne) << 23);
          dexp = ne;
          dlim = ne > 15 ? 0x7BFF7BFFu : (uint32_t)(ne + 15) * 0x04000400u;
          dnorm = ne < 15 ? (uint32_t)(15 - ne) * 0x04000400u : ne == 15 ? 0x02000200u : 0x01000100u;
          // 2^(ne - KR_SPREAD) as f16 bits, below 2^-14 a subnormal, below 2^-24 nothing
          const int le = ne - KR_SPREAD;
          const uint32_t low = le >= -14 ? (uint32_t)(le + 15) << 10 : le >= -24 ? 1u << (le + 24) : 0u;
          dlow = low * 0x00010001u;
          if (__reduce_min_sync(0xffffffffu, min(dmin & 0xFFFFu, dmin >> 16)) + 1 < low) return false;
        }
#pragma unroll
        for (int n = 0; n < RL; n++) {
          const float mn = fmaxf(m[n], top[n]);
          const float nb = mn == -INFINITY ? 0.0f : fsub(mn, HEADROOM);
          const float f = m[n] == -INFINITY ? 0.0f : exp2_approx(fsub(base[n], nb));
          l[n] = fmul(l[n], f);
#pragma unroll
          for (int u = 0; u < 8; u++)
#pragma unroll
            for (int k = F16 ? n : 0; k < (F16 ? n + 1 : NT); k++)
#pragma unroll
              for (int e = 0; e < 4; e++) o[u][k][e] = fmul(o[u][k][e], fmul(f, fd));
          m[n] = mn;
          base[n] = nb;
        }
      }
      float w[RL][2];
#pragma unroll
      for (int n = 0; n < RL; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          w[n][i] = exp2_approx(ffma(s[n][i], unscale[n], -base[n]));
          l[n] = fadd(l[n], w[n][i]);
        }
      // ------------------------------------------------------------- values
      // lane column c: keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
      const uint8_t* va = stage + L::V_OFF + c * L::V_PAIR;
      if constexpr (Q4) {
        uint32_t wh[NT], wl[NT];
#pragma unroll
        for (int n = 0; !WIDE && n < NT; n++) split_f16(w[n][0], w[n][1], wh[n], wl[n]);
        const uint2 v0 = ld_u2(va + 8 * g), v1 = ld_u2(va + L::ROW + 8 * g);
        const uint2 v2 = ld_u2(va + 4 * L::V_PAIR + 8 * g), v3 = ld_u2(va + 4 * L::V_PAIR + L::ROW + 8 * g);
#pragma unroll
        for (int b = 0; b < 4; b++) {
          // block b's two bytes of four keys, keys paired
          const uint32_t sel = b & 1 ? 0x7632u : 0x5410u;
          uint32_t x[4], y[4];
          nib_f16(__byte_perm(b < 2 ? v0.x : v0.y, b < 2 ? v1.x : v1.y, sel), x);
          nib_f16(__byte_perm(b < 2 ? v2.x : v2.y, b < 2 ? v3.x : v3.y, sel), y);
          if (WIDE) {  // codes in bf16, weight times scale in f32 and as three bf16 parts
            uint32_t av[2][4];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const float2 v = h2f2(i & 2 ? y[(i & 1) + 2 * (i >> 2)] : x[(i & 1) + 2 * (i >> 2)]);
              av[i >> 2][i & 3] = bf2(v.x, v.y);
            }
            const float2 d = h2f2(vd[b]);
#pragma unroll
            for (int n = 0; n < NT; n++) {
              uint32_t part[3];
              split_bf16(fmul(w[n][0], d.x), fmul(w[n][1], d.y), part);
              const uint32_t b0 = movm(__byte_perm(part[0], part[1], 0x5410)),
                             b1 = movm(__byte_perm(part[0], part[1], 0x7632)),
                             b2 = movm(part[2] & 0x0000FFFFu), b3 = movm(part[2] >> 16);
#pragma unroll
              for (int i = 0; i < 2; i++) {
                mma16<false>(o[2 * b + i][n], av[i], b2, b3);
                mma16<false>(o[2 * b + i][n], av[i], b0, b1);
              }
            }
            continue;
          }
          const uint32_t d = hmul2_u(vd[b], dnorm);
          const uint32_t a0[4] = {x[0], x[1], y[0], y[1]}, a1[4] = {x[2], x[3], y[2], y[3]};
#pragma unroll
          for (int n = 0; n < NT; n++) {
            // (hi + lo) d: the product's f16, then what its rounding left plus lo d
            const uint32_t ph = hmul2_u(wh[n], d);
            const uint32_t pl = hfma2_u(wl[n], d, hfma2_u(wh[n], d, hneg2_u(ph)));
            const uint32_t b0 = movm(__byte_perm(ph, pl, 0x5410)), b1 = movm(__byte_perm(ph, pl, 0x7632));
            mma16<F16>(o[2 * b][n], a0, b0, b1);
            mma16<F16>(o[2 * b + 1][n], a1, b0, b1);
          }
        }
      } else {
        uint32_t pb[NT][2];
        if constexpr (F16) {
#pragma unroll
          for (int n = 0; n < NT; n++) {
            uint32_t ph, pl;
            split_f16(w[n][0], w[n][1], ph, pl);
            pb[n][0] = movm(__byte_perm(ph, pl, 0x5410));
            pb[n][1] = movm(__byte_perm(ph, pl, 0x7632));
          }
        } else {
          uint32_t part[3];
          split_bf16(w[0][0], w[0][1], part);
          pb[0][0] = movm(__byte_perm(part[0], part[1], 0x5410));
          pb[0][1] = movm(__byte_perm(part[0], part[1], 0x7632));
          pb[1][0] = movm(part[2] & 0x0000FFFFu);
          pb[1][1] = movm(part[2] >> 16);
        }
        constexpr int K8 = 4 * L::V_PAIR;  // eight keys on
        if constexpr (KV == FLOCK_KV_FP8) {
          const uint4 v0 = ld_u4(va + 16 * g), v1 = ld_u4(va + L::ROW + 16 * g);
          const uint4 v2 = ld_u4(va + K8 + 16 * g), v3 = ld_u4(va + K8 + L::ROW + 16 * g);
#pragma unroll
          for (int u = 0; u < 8; u++) {
            const int sh = 16 * (u & 1);
            const uint32_t y0 = fp8_f16(word_of(v0, u >> 1) >> sh), y1 = fp8_f16(word_of(v1, u >> 1) >> sh),
                           y2 = fp8_f16(word_of(v2, u >> 1) >> sh), y3 = fp8_f16(word_of(v3, u >> 1) >> sh);
            const uint32_t av[4] = {__byte_perm(y0, y1, 0x5410), __byte_perm(y0, y1, 0x7632),
                                    __byte_perm(y2, y3, 0x5410), __byte_perm(y2, y3, 0x7632)};
#pragma unroll
            for (int n = 0; n < NT; n++) mma16<F16>(o[u][n], av, pb[n][0], pb[n][1]);
          }
        } else if constexpr (KV == FLOCK_KV_BF16) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint8_t* vh = va + 128 * h + 16 * g;
            const uint4 v0 = ld_u4(vh), v1 = ld_u4(vh + L::ROW), v2 = ld_u4(vh + K8),
                        v3 = ld_u4(vh + K8 + L::ROW);
#pragma unroll
            for (int q = 0; q < 4; q++) {
              const uint32_t y0 = word_of(v0, q), y1 = word_of(v1, q), y2 = word_of(v2, q), y3 = word_of(v3, q);
              const uint32_t av[4] = {__byte_perm(y0, y1, 0x5410), __byte_perm(y0, y1, 0x7632),
                                      __byte_perm(y2, y3, 0x5410), __byte_perm(y2, y3, 0x7632)};
#pragma unroll
              for (int n = 0; n < NT; n++) mma16<F16>(o[4 * h + q][n], av, pb[n][0], pb[n][1]);
            }
          }
        } else {
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const uint8_t* vh = va + 128 * h + 16 * g;
            const uint4 v0 = ld_u4(vh), v1 = ld_u4(vh + L::ROW), v2 = ld_u4(vh + K8),
                        v3 = ld_u4(vh + K8 + L::ROW);
#pragma unroll
            for (int q = 0; q < 2; q++) {
              auto f = [&](const uint4& v, int i) { return __uint_as_float(word_of(v, 2 * q + i)); };
              uint32_t x0[3], x1[3], y0[3], y1[3];
              split_bf16(f(v0, 0), f(v1, 0), x0);
              split_bf16(f(v0, 1), f(v1, 1), x1);
              split_bf16(f(v2, 0), f(v3, 0), y0);
              split_bf16(f(v2, 1), f(v3, 1), y1);
#pragma unroll
              for (int part = 0; part < 3; part++) {
                const uint32_t av[4] = {x0[part], x1[part], y0[part], y1[part]};
#pragma unroll
                for (int n = 0; n < (part == 2 ? 1 : NT); n++)
                  mma16<F16>(o[2 * h + q][n], av, pb[n][0], pb[n][1]);
              }
            }
          }
        }
      }
      st = st + 1 == L::STAGES ? 0 : st + 1;
    }
    return true;
  };
  if (!pass(std::false_type())) {
    if constexpr (Q4) {
      cp_async_wait<0>();
      __syncwarp();  // the ring is this warp's alone
#pragma unroll
      for (int s = 0; s < L::STAGES - 1; s++) fetch(g0 + warp + s * L::WARPS, s);
      pass(std::true_type());
    }
  }
  cp_async_wait<0>();

  // ---------------------------------------------------------- join the warps
  constexpr int OS = KV_HD + 4;  // row stride of the warps' outputs
  const int live = min(RT, p.rows - tile * RT);
  __syncthreads();  // the rings are done with: their memory holds the warps' outputs
  float* s_o = reinterpret_cast<float*>(kr_smem);  // [warp][RT][OS]
#pragma unroll
  for (int n = 0; n < RL; n++) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) l[n] = fadd(l[n], __shfl_xor_sync(0xffffffffu, l[n], d));
    if (4 * n + c < live) {
      const float back = Q4 ? __uint_as_float((uint32_t)(127 + dexp) << 23) : 1.0f;
      float* dst = s_o + (warp * RT + 4 * n + c) * OS;
#pragma unroll
      for (int u = 0; u < 8; u++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float x = fadd(o[u][n][2 * h], o[u][n][2 * h + 1]);
          if (!F16) x = fadd(x, o[u][NT - 1][2 * h]);
          dst[kr_vdim<KV>(u, h, g)] = fmul(x, back);
        }
      if (g == 0) {
        s_ml[warp][4 * n + c][0] = l[n] > 0.0f ? base[n] : -INFINITY;  // weights are relative to 2^base
        s_ml[warp][4 * n + c][1] = l[n];
      }
    }
  }
  __syncthreads();
  const int item = head * gridDim.y + tile;
  const int n_items = gridDim.y * gridDim.z;
  float* part_ml = p.part + (size_t)n_items * gridDim.x * RT * KV_HD;
  for (int i = threadIdx.x; i < live * KV_HD; i += L::THREADS) {
    const int r = i / KV_HD, d = i % KV_HD;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < L::WARPS; w++) mm = fmaxf(mm, s_ml[w][r][0]);
    const float b = mm == -INFINITY ? 0.0f : mm;
    float oo = 0.0f, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < L::WARPS; w++) {
      const float f = exp2_approx(fsub(s_ml[w][r][0], b));
      oo = ffma(f, s_o[(w * RT + r) * OS + d], oo);
      ll = ffma(f, s_ml[w][r][1], ll);
    }
    if (splits == 1) {
      const int rr = tile * RT + r;
      a.out[(rr / p.group) * a.out_stride + ((int64_t)head * p.group + rr % p.group) * KV_HD + d] =
          fdiv(oo, ll);
    } else {
      const size_t at = ((size_t)item * gridDim.x + z) * RT + r;
      p.part[at * KV_HD + d] = oo;
      if (d == 0) {
        part_ml[at * 2] = mm;
        part_ml[at * 2 + 1] = ll;
      }
    }
  }
  if (splits == 1) return;
  // --------------------------------------------------------- join the splits
  // one release-acquire arrival per CTA, behind the barrier that orders its
  // threads' stores before it
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                 : "=r"(before) : "l"(p.count + item) : "memory");
    s_last = before == (uint32_t)splits - 1;
    if (s_last) p.count[item] = 0;  // ready for the next call
  }
  __syncthreads();
  if (!s_last) return;
  // Thread (k, four outputs): the splits k, k + PAR, .. of them, all loads in
  // flight before the first use; the splits' factors 2^(m_s - m) meanwhile.
  const int quads = live * (KV_HD / 4);
  const int par = L::THREADS / quads;
  const int k = threadIdx.x / quads, r = (threadIdx.x % quads) / (KV_HD / 4),
            d = 4 * (threadIdx.x % (KV_HD / 4));
  const bool mine = threadIdx.x < par * quads;
  float* s_f = reinterpret_cast<float*>(kr_smem);  // [split][RT]
  float* s_l = s_f + splits * RT;
  float4* s_x = reinterpret_cast<float4*>(s_l + splits * RT);  // [k][quads]
  const size_t first = (size_t)item * gridDim.x * RT;
  constexpr int U = 4;  // loads in flight
  float4 x4[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; u++)
      if (mine && s0 + u * par < splits)
        x4[u] = __ldcg(reinterpret_cast<const float4*>(
            p.part + (first + (size_t)(s0 + u * par) * RT + r) * KV_HD + d));
  };
  load(k);
  for (int i = threadIdx.x; i < splits * RT; i += L::THREADS) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml) + first + i);
    s_f[i] = ml.x;
    s_l[i] = ml.y;
  }
  __syncthreads();
  if (warp < live) {
    float mm = -INFINITY;
    for (int s = lane; s < splits; s += 32) mm = fmaxf(mm, s_f[s * RT + warp]);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
    float ll = 0.0f;
    for (int s = lane; s < splits; s += 32) {
      const float f = exp2_approx(fsub(s_f[s * RT + warp], mm));
      s_f[s * RT + warp] = f;
      ll = ffma(f, s_l[s * RT + warp], ll);
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) ll = fadd(ll, __shfl_xor_sync(0xffffffffu, ll, x));
    if (lane == 0) s_ml[0][warp][1] = ll;
  }
  __syncthreads();
  float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = k; mine && s0 < splits; s0 += U * par) {
    if (s0 != k) load(s0);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (s0 + u * par < splits) {
        const float f = s_f[(s0 + u * par) * RT + r];
        oo = make_float4(ffma(f, x4[u].x, oo.x), ffma(f, x4[u].y, oo.y), ffma(f, x4[u].z, oo.z),
                         ffma(f, x4[u].w, oo.w));
      }
  }
  if (mine) s_x[threadIdx.x] = oo;
  __syncthreads();
  if (threadIdx.x < quads) {
    for (int i = 1; i < par; i++) {
      const float4 x = s_x[i * quads + threadIdx.x];
      oo = make_float4(fadd(oo.x, x.x), fadd(oo.y, x.y), fadd(oo.z, x.z), fadd(oo.w, x.w));
    }
    const float inv = fdiv(1.0f, s_ml[0][r][1]);
    const int rr = tile * RT + r;
    *reinterpret_cast<float4*>(a.out + (rr / p.group) * a.out_stride +
                               ((int64_t)head * p.group + rr % p.group) * KV_HD + d) =
        make_float4(fmul(oo.x, inv), fmul(oo.y, inv), fmul(oo.z, inv), fmul(oo.w, inv));
  }
}

}  // namespace flock
