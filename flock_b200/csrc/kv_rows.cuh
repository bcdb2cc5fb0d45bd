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
// memory to the operand registers with no store in between.
//
// f32 results from 16-bit operands.  Codes minus 8 and e4m3 values are f16
// values, so there queries and softmax weights are split as hi + lo, two f16
// of 11 bits (22 bits; scaled by powers of two so that f16's range never
// cuts a part that matters).  bf16 and f32 elements need f32's range: hi + mid
// + lo, three bf16 of 8 bits.  The parts sit in different ROWS of the 16-row
// operand, which a decode leaves empty anyway: one instruction multiplies all.
//
// 4-bit blocks.  Scores: a block's 32 products are summed as integers times
// query parts, then multiplied by the key's scale in f32 (one accumulator per
// block).  Values: the scale joins the weight before its split, so the weight
// operand differs per block.
//
// Work split: CTA (split z, row tile, kv head), its warps taking 16-key groups
// in turn, each with its own cp.async ring, running maximum, sum and output;
// warps join in shared memory, CTAs in the workspace, the last to arrive adding
// the splits in order (results do not depend on who is last).
#pragma once
#include "kv.cuh"

namespace flock {

constexpr int KR_GROUP = 16;  // keys per warp step
constexpr int KR_MAX_ITEMS = 4096;  // (row tile, kv head) pairs that may be split: arrival counters
constexpr size_t KR_PART_OFFSET = KR_MAX_ITEMS * 4;

struct KvRowsArgs {
  KvAttnArgs a;
  int rows;         // n_queries * group: row r is query r / group, head r % group
  int group;        // query heads per kv head
  int splits;
  uint32_t* count;  // [items], zero between calls
  float* part;      // [item][split][RT][128], then [item][split][RT][2] (m, l)
};

// Shared-memory layout of one warp's 16-key stage, per cached type.  Key rows
// are read 16 bytes a lane, eight lanes covering 64 bytes of two keys; value
// rows 8 or 16 bytes a lane, eight lanes covering pieces of four keys four
// apart.  Padding keeps both free of bank conflicts.
template <int KV>
struct KrTile;
template <>
struct KrTile<FLOCK_KV_Q4> {
  static constexpr int ROW = 64, K_STRIDE = 64, V_GROUP = 4 * 64 + 32, WARPS = 12, STAGES = 5;
  static constexpr int SCALES = 2 * KR_GROUP * 8;
};
template <>
struct KrTile<FLOCK_KV_FP8> {
  static constexpr int ROW = 128, K_STRIDE = 192, V_GROUP = 4 * 128 + 32, WARPS = 8, STAGES = 4;
  static constexpr int SCALES = 0;
};
template <>
struct KrTile<FLOCK_KV_BF16> {
  static constexpr int ROW = 256, K_STRIDE = 320, V_GROUP = 4 * 256 + 32, WARPS = 8, STAGES = 2;
  static constexpr int SCALES = 0;
};
template <>
struct KrTile<FLOCK_KV_F32> {
  static constexpr int ROW = 512, K_STRIDE = 576, V_GROUP = 4 * 512 + 32, WARPS = 6, STAGES = 2;
  static constexpr int SCALES = 0;
};
template <int KV>
struct KrLayout : KrTile<KV> {
  using T = KrTile<KV>;
  static constexpr int V_OFF = KR_GROUP * T::K_STRIDE;
  static constexpr int S_OFF = V_OFF + KR_GROUP / 4 * T::V_GROUP;
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

template <bool F16>
FLOCK_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
FLOCK_DEV uint32_t hadd2_u(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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

// The head dimension of column n of output tile t (0-15).
template <int KV>
FLOCK_DEV int kr_vdim(int t, int n) {
  if (KV == FLOCK_KV_Q4) return 32 * (t >> 2) + 16 * (t & 1) + 2 * n + ((t & 2) >> 1);
  if (KV == FLOCK_KV_FP8) return 16 * n + t;
  if (KV == FLOCK_KV_BF16) return 64 * (t >> 3) + 8 * n + (t & 7);
  return 32 * (t >> 2) + 4 * n + (t & 3);
}

// One stage of keys key0 .. key0 + 15 of a head into shared memory; keys
// outside [from, to) are zero-filled, so what lies there cannot reach a
// product.  kb, vb: the head's first rows; sb: this lane's scale plane at the
// head's first row.
template <int KV>
FLOCK_DEV void kr_load(uint32_t stage, const uint8_t* kb, const uint8_t* vb, const uint8_t* sb,
                       int64_t step, int key0, int from, int to, int lane) {
  using L = KrLayout<KV>;
  constexpr int CHUNKS = L::ROW / 16;  // 16-byte chunks of a row
  const bool whole = key0 >= from && key0 + KR_GROUP <= to;
#pragma unroll
  for (int i = 0; i < KR_GROUP * CHUNKS / 32; i++) {
    const int at = i * 32 + lane, r = at / CHUNKS, ch = at % CHUNKS;
    const bool ok = whole || (key0 + r >= from && key0 + r < to);
    // a 4-bit head's rows are contiguous: one offset for the whole group
    const int64_t off = KV == FLOCK_KV_Q4 ? (int64_t)key0 * 64 + at * 16
                                          : (int64_t)(ok ? key0 + r : from) * step + ch * 16;
    cp_async16(stage + r * L::K_STRIDE + ch * 16, kb + off, ok);
    cp_async16(stage + L::V_OFF + (r >> 2) * L::V_GROUP + (r & 3) * L::ROW + ch * 16, vb + off, ok);
  }
  if (KV == FLOCK_KV_Q4) {
    const int r = lane & 15;
    const bool ok = whole || (key0 + r >= from && key0 + r < to);
    cp_async8(stage + L::S_OFF + lane * 8, sb + (int64_t)(key0 + r) * 8, ok);
  }
}

FLOCK_DEV uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}
FLOCK_DEV uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}

// Query rows per CTA.  f16 parts: operand rows 0-7 hold the rows' hi parts,
// 8-15 their lo.  bf16 parts: 0-3 hi, 4-7 mid, 8-11 lo.
template <int KV>
constexpr int KR_ROWS = KV == FLOCK_KV_Q4 || KV == FLOCK_KV_FP8 ? 8 : 4;

// Keys of a stage are dealt to operand columns so that a lane's four score
// columns are four neighbouring keys: column n of score tile t is key
// 4 (n / 2) + 2 t + n % 2, and lane column c holds keys 4 c .. 4 c + 3.
template <int KV>
static __global__ void __launch_bounds__(KrLayout<KV>::THREADS, 1) k_kv_rows(const KvRowsArgs p) {
  using L = KrLayout<KV>;
  constexpr int RT = KR_ROWS<KV>;
  constexpr bool Q4 = KV == FLOCK_KV_Q4;
  constexpr bool F16 = Q4 || KV == FLOCK_KV_FP8;
  extern __shared__ __align__(16) uint8_t kr_smem[];
  __shared__ float s_ml[L::WARPS][RT][2];
  __shared__ uint4 s_q[8][32];  // the query operand: [QK step][lane]
  __shared__ float s_unscale[RT];
  __shared__ int s_last;
  pdl_launch_dependents();
  pdl_wait();
  const KvAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int z = blockIdx.x, tile = blockIdx.y, head = blockIdx.z;
  const int j = g % RT;  // this lane's query row
  const int row = tile * RT + j;
  const int first_q = tile * RT / p.group;
  const int last_q = (min(p.rows, (tile + 1) * RT) - 1) / p.group;
  // keys that some row of the tile sees: sinks [0, sk), then [lo, hi)
  const int pos = (int)a.pos;
  const int hi = pos + last_q + 1;
  const int lo = a.window && pos + first_q + 1 > a.window ? pos + first_q + 1 - a.window : 0;
  const int sk = min(a.sinks, lo);
  const int sink_groups = (sk + KR_GROUP - 1) / KR_GROUP;
  const int lo16 = lo & ~(KR_GROUP - 1);
  const int groups = sink_groups + (hi - lo16 + KR_GROUP - 1) / KR_GROUP;
  const int g0 = (int)((int64_t)z * groups / p.splits), g1 = (int)((int64_t)(z + 1) * groups / p.splits);
  // this row's own keys: sinks [0, row_sk), then [row_lo, row_hi)
  const int my_q = min(row, p.rows - 1) / p.group;
  const int row_hi = pos + my_q + 1;
  const int row_lo = a.window && row_hi > a.window ? row_hi - a.window : 0;
  const int row_sk = min(a.sinks, row_lo);

  const uint32_t ring = smem_u32(kr_smem) + warp * L::STAGES * L::STAGE;
  const size_t hbase = Q4 ? q4_row(a.c, 0, head) * 64 : (size_t)head * L::ROW;
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + hbase;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + hbase;
  const uint8_t* sb = Q4 ? reinterpret_cast<const uint8_t*>((lane < 16 ? a.c.ks : a.c.vs) +
                                                            q4_row(a.c, 0, head) * 4)
                         : nullptr;
  const int64_t step = (int64_t)a.c.n_kv_heads * L::ROW;
  auto key_of = [&](int grp) {
    return grp < sink_groups ? grp * KR_GROUP : lo16 + (grp - sink_groups) * KR_GROUP;
  };
  auto fetch = [&](int grp, int st) {
    if (grp < g1) {
      const bool sink = grp < sink_groups;
      kr_load<KV>(ring + st * L::STAGE, kb, vb, sb, step, key_of(grp), sink ? 0 : lo,
                  sink ? sk : hi, lane);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < L::STAGES - 1; s++) fetch(g0 + warp + s * L::WARPS, s);

  // The query operand: the parts of q log2(e) / sqrt(128), for f16 scaled by
  // a power of two that brings the row's largest into [2^13, 2^14).  A warp
  // splits a row, four neighbouring dimensions a lane: one operand entry.
  for (int r = warp; r < RT; r += L::WARPS) {
    const int rr = tile * RT + r;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (rr < p.rows)
      x = __ldg(reinterpret_cast<const float4*>(
          a.q + (rr / p.group) * a.q_stride + ((int64_t)head * p.group + rr % p.group) * KV_HD +
          4 * lane));
    const float k = __double2float_rn(1.4426950408889634 / sqrt(128.0));
    x = make_float4(fmul(x.x, k), fmul(x.y, k), fmul(x.z, k), fmul(x.w, k));
    const int qc = Q4 || KV == FLOCK_KV_F32 ? lane & 3 : KV == FLOCK_KV_FP8 ? (lane >> 2) & 3 : (lane >> 1) & 3;
    const int ks = Q4 || KV == FLOCK_KV_F32 ? lane >> 2
                   : KV == FLOCK_KV_FP8     ? (lane >> 4) * 4 + (lane & 3)
                                            : (lane >> 3) * 2 + (lane & 1);
    if (F16) {
      float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int biased = (int)(__float_as_uint(top) >> 23);
      const int e = biased == 0 ? 0 : max(-100, min(100, biased - 127 - 13));
      const float scale = __uint_as_float((uint32_t)(127 - e) << 23);
      if (lane == 0) s_unscale[r] = __uint_as_float((uint32_t)(127 + e) << 23);
      if (Q4) {  // pairs two apart: bytes 0 and 2, 1 and 3 of a code word
        const float y = x.y;
        x.y = x.z;
        x.z = y;
      }
      uint4 w;
      split_f16(fmul(x.x, scale), fmul(x.y, scale), w.x, w.y);
      split_f16(fmul(x.z, scale), fmul(x.w, scale), w.z, w.w);
      s_q[ks][4 * r + qc] = w;
    } else {
      uint32_t w0[3], w1[3];
      split_bf16(x.x, x.y, w0);
      split_bf16(x.z, x.w, w1);
      s_q[ks][4 * r + qc] = make_uint4(w0[0], w0[2], w1[0], w1[2]);
      s_q[ks][4 * (r + 4) + qc] = make_uint4(w0[1], 0, w1[1], 0);
    }
  }
  __syncthreads();
  uint32_t qa[8][4];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) {
    const uint4 w = s_q[ks][lane];
    qa[ks][0] = w.x;
    qa[ks][1] = w.y;
    qa[ks][2] = w.z;
    qa[ks][3] = w.w;
  }
  const float unscale = F16 ? s_unscale[j] : 1.0f;
  float o[16][4];
#pragma unroll
  for (int t = 0; t < 16; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) o[t][e] = 0.0f;
  // Weights are 2^(s - base), base = m + dexp - 6: m a running maximum that may
  // lag by 2^8, 2^dexp a bound on the value scales so far, so a weight times a
  // scale is at most 2^14, inside f16, and its lo part loses nothing above
  // 2^-31 of the largest.
  constexpr float HEADROOM = F16 ? 6.0f : 0.0f;
  float m = -INFINITY, l = 0.0f, base = 0.0f;
  int dexp = Q4 ? -24 : 0;
  float dlim = Q4 ? 5.9604645e-8f : 0.0f;  // 2^dexp

  int st = 0;
  for (int grp = g0 + warp; grp < g1; grp += L::WARPS) {
    cp_async_wait<L::STAGES - 2>();
    __syncwarp();  // the stage has landed for every lane, and every lane is done with the last one
    fetch(grp + (L::STAGES - 1) * L::WARPS, st == 0 ? L::STAGES - 1 : st - 1);
    const uint32_t stage = ring + st * L::STAGE;
    // ------------------------------------------------------------- scores
    float s[4];  // keys 4 c + i of this lane's row
    const uint32_t kaddr = stage + (4 * (g >> 1) + (g & 1)) * L::K_STRIDE + 16 * c;
    if constexpr (Q4) {
      const uint4 scales[2] = {lds128(stage + L::S_OFF + 32 * c),
                               lds128(stage + L::S_OFF + 32 * c + 16)};
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint4 w4 = lds128(kaddr + 2 * t * L::K_STRIDE);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        // keys 4 c + 2 t and the next, four blocks each
        const float2 k0[2] = {h2f2(scales[t].x), h2f2(scales[t].y)},
                     k1[2] = {h2f2(scales[t].z), h2f2(scales[t].w)};
        uint64_t sum = pack2(0.0f, 0.0f);
#pragma unroll
        for (int b = 0; b < 4; b++) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t v[4];
          nib_f16(w[b], v);
          mma16<F16>(acc, qa[2 * b], v[0], v[2]);
          mma16<F16>(acc, qa[2 * b + 1], v[1], v[3]);
          const uint64_t d = b & 1 ? pack2(k0[b >> 1].y, k1[b >> 1].y)
                                   : pack2(k0[b >> 1].x, k1[b >> 1].x);
          sum = ffma2(d, pack2(acc[0], acc[1]), sum);  // hi
          sum = ffma2(d, pack2(acc[2], acc[3]), sum);  // lo
        }
        const float2 r = unpack2(sum);
        s[2 * t] = r.x;
        s[2 * t + 1] = r.y;
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint32_t kt = kaddr + 2 * t * L::K_STRIDE;
        float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if constexpr (KV == FLOCK_KV_FP8) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint4 w4 = lds128(kt + 64 * h);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
              mma16<F16>(acc[i & 1], qa[4 * h + i], fp8_f16(w[i]), fp8_f16(w[i] >> 16));
          }
        } else if constexpr (KV == FLOCK_KV_BF16) {
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const uint4 w = lds128(kt + 64 * h);
            mma16<F16>(acc[0], qa[2 * h], w.x, w.y);
            mma16<F16>(acc[1], qa[2 * h + 1], w.z, w.w);
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 8; ks++) {
            const uint4 w = lds128(kt + 64 * ks);
            uint32_t b0[3], b1[3];
            split_bf16(__uint_as_float(w.x), __uint_as_float(w.y), b0);
            split_bf16(__uint_as_float(w.z), __uint_as_float(w.w), b1);
#pragma unroll
            for (int part = 0; part < 3; part++) mma16<F16>(acc[part & 1], qa[ks], b0[part], b1[part]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          s[2 * t + i] = fadd(fadd(acc[0][i], acc[1][i]), fadd(acc[0][2 + i], acc[1][2 + i]));
          if (!F16) s[2 * t + i] = fadd(s[2 * t + i], __shfl_xor_sync(0xffffffffu, s[2 * t + i], 16));
        }
      }
    }
    const int key0 = key_of(grp);
    {  // masks, only where the group is not wholly visible to every row
      const bool sink = grp < sink_groups;
      const int from = sink ? 0 : row_lo, to = sink ? sk : row_hi;
      if (__any_sync(0xffffffffu, key0 < from || key0 + KR_GROUP > to)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int key = key0 + 4 * c + i;
          // every row sees the tile's sinks; a row's own may reach into the main range
          const bool seen = sink ? key < sk
                                 : key >= lo && key < row_hi && (key >= row_lo || key < row_sk);
          if (!seen) s[i] = -INFINITY;
        }
      }
    }
    // ------------------------------------------------------------ softmax
    // the value scales of the lane's four keys, two blocks a word; the largest
    // magnitude of all sixteen as a bound for the f16 weights
    uint32_t vs[4][2];
    float dmax = 0.0f;
    if constexpr (Q4) {
      const uint4 e0 = lds128(stage + L::S_OFF + 128 + 32 * c);
      const uint4 e1 = lds128(stage + L::S_OFF + 128 + 32 * c + 16);
      vs[0][0] = e0.x, vs[0][1] = e0.y, vs[1][0] = e0.z, vs[1][1] = e0.w;
      vs[2][0] = e1.x, vs[2][1] = e1.y, vs[3][0] = e1.z, vs[3][1] = e1.w;
      auto habs = [](uint32_t x) {
        const uint32_t u = x & 0x7FFF7FFFu;
        return *reinterpret_cast<const __half2*>(&u);
      };
      __half2 h = habs(vs[0][0]);
#pragma unroll
      for (int i = 1; i < 8; i++) h = __hmax2(h, habs(vs[i >> 1][i & 1]));
      const float2 f = __half22float2(h);
      dmax = fmaxf(f.x, f.y);
    }
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmul(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)), unscale);
    if (__any_sync(0xffffffffu, top > fadd(m, 8.0f) || (Q4 && dmax > dlim))) {
      if (Q4) {
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) dmax = fmaxf(dmax, __shfl_xor_sync(0xffffffffu, dmax, x));
        dexp = max(dexp, min((int)(__float_as_uint(dmax) >> 23) - 126, 16));
        dlim = __uint_as_float((uint32_t)(127 + dexp) << 23);
      }
      const float mn = fmaxf(m, top);
      const float nb = mn == -INFINITY ? 0.0f : fadd(mn, (float)dexp - HEADROOM);
      const float f = m == -INFINITY ? 0.0f : exp2_approx(fsub(base, nb));
      l = fmul(l, f);
#pragma unroll
      for (int t = 0; t < 16; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[t][e] = fmul(o[t][e], f);  // rows g and g + 8: one query row
      m = mn;
      base = nb;
    }
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = exp2_approx(ffma(s[i], unscale, -base));
      l = fadd(l, w[i]);
    }
    // ------------------------------------------------------------- values
    const uint32_t vaddr = stage + L::V_OFF + c * L::V_GROUP;
    if constexpr (Q4) {
      uint2 v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = lds64(vaddr + i * 64 + 8 * g);
#pragma unroll
      for (int hb = 0; hb < 2; hb++) {
        float2 d[4];
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = h2f2(vs[i][hb]);
#pragma unroll
        for (int bb = 0; bb < 2; bb++) {
          const int b = 2 * hb + bb;
          uint32_t pa[4];
          split_f16(fmul(w[0], bb ? d[0].y : d[0].x), fmul(w[1], bb ? d[1].y : d[1].x), pa[0], pa[1]);
          split_f16(fmul(w[2], bb ? d[2].y : d[2].x), fmul(w[3], bb ? d[3].y : d[3].x), pa[2], pa[3]);
          // block b's two bytes of four keys, keys paired
          const uint32_t sel = bb ? 0x7632u : 0x5410u;
          const uint32_t k01 = __byte_perm(hb ? v[0].y : v[0].x, hb ? v[1].y : v[1].x, sel);
          const uint32_t k23 = __byte_perm(hb ? v[2].y : v[2].x, hb ? v[3].y : v[3].x, sel);
          uint32_t x[4], y[4];
          nib_f16(k01, x);
          nib_f16(k23, y);
#pragma unroll
          for (int e = 0; e < 4; e++)  // tile 4 b + e: nibble e of the halfword
            mma16<F16>(o[4 * b + e], pa, x[e], y[e]);
        }
      }
    } else {
      uint32_t pa[4];
      if constexpr (F16) {
        split_f16(w[0], w[1], pa[0], pa[1]);
        split_f16(w[2], w[3], pa[2], pa[3]);
      } else {
        uint32_t w0[3], w1[3];
        split_bf16(w[0], w[1], w0);
        split_bf16(w[2], w[3], w1);
        pa[0] = g < 4 ? w0[0] : w0[1];
        pa[2] = g < 4 ? w1[0] : w1[1];
        pa[1] = g < 4 ? w0[2] : 0;
        pa[3] = g < 4 ? w1[2] : 0;
      }
      auto word = [](const uint4& v, int q) { return q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w; };
      if constexpr (KV == FLOCK_KV_FP8) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = lds128(vaddr + i * 128 + 16 * g);
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = fp8_f16(word(v[i], q) >> (16 * h));
            mma16<F16>(o[4 * q + 2 * h], pa, __byte_perm(y[0], y[1], 0x5410),
                       __byte_perm(y[2], y[3], 0x5410));
            mma16<F16>(o[4 * q + 2 * h + 1], pa, __byte_perm(y[0], y[1], 0x7632),
                       __byte_perm(y[2], y[3], 0x7632));
          }
      } else if constexpr (KV == FLOCK_KV_BF16) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = lds128(vaddr + i * 256 + 128 * h + 16 * g);
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const uint32_t x0 = word(v[0], q), x1 = word(v[1], q), x2 = word(v[2], q),
                           x3 = word(v[3], q);
            mma16<F16>(o[8 * h + 2 * q], pa, __byte_perm(x0, x1, 0x5410), __byte_perm(x2, x3, 0x5410));
            mma16<F16>(o[8 * h + 2 * q + 1], pa, __byte_perm(x0, x1, 0x7632),
                       __byte_perm(x2, x3, 0x7632));
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 4; h++) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = lds128(vaddr + i * 512 + 128 * h + 16 * g);
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint32_t b0[3], b1[3];
            split_bf16(__uint_as_float(word(v[0], q)), __uint_as_float(word(v[1], q)), b0);
            split_bf16(__uint_as_float(word(v[2], q)), __uint_as_float(word(v[3], q)), b1);
#pragma unroll
            for (int part = 0; part < 3; part++) mma16<F16>(o[4 * h + q], pa, b0[part], b1[part]);
          }
        }
      }
    }
    st = st + 1 == L::STAGES ? 0 : st + 1;
  }
  cp_async_wait<0>();

  // ---------------------------------------------------------- join the warps
  l = fadd(l, __shfl_xor_sync(0xffffffffu, l, 1));
  l = fadd(l, __shfl_xor_sync(0xffffffffu, l, 2));
  __syncthreads();  // the rings are done with: their memory holds the warps' outputs
  float* s_o = reinterpret_cast<float*>(kr_smem);  // [warp][RT][128]
  const int live = min(RT, p.rows - tile * RT);
#pragma unroll
  for (int t = 0; t < 16; t++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int at = kr_vdim<KV>(t, 2 * c + e);
      float* dst = s_o + (warp * RT + j) * KV_HD + at;
      float x = fadd(o[t][e], o[t][2 + e]);
      if (!F16) x = fadd(x, __shfl_xor_sync(0xffffffffu, x, 16));
      if (g < live) *dst = x;
    }
  if (g < RT && c == 0) {
    s_ml[warp][j][0] = l > 0.0f ? base : -INFINITY;  // weights are relative to 2^base
    s_ml[warp][j][1] = l;
  }
  __syncthreads();
  const int item = head * gridDim.y + tile;
  const int n_items = gridDim.y * gridDim.z;
  float* part_ml = p.part + (size_t)n_items * p.splits * RT * KV_HD;
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
      oo = ffma(f, s_o[(w * RT + r) * KV_HD + d], oo);
      ll = ffma(f, s_ml[w][r][1], ll);
    }
    if (p.splits == 1) {
      const int rr = tile * RT + r;
      a.out[(rr / p.group) * a.out_stride + ((int64_t)head * p.group + rr % p.group) * KV_HD + d] =
          fdiv(oo, ll);
    } else {
      const size_t at = ((size_t)item * p.splits + z) * RT + r;
      p.part[at * KV_HD + d] = oo;
      if (d == 0) {
        part_ml[at * 2] = mm;
        part_ml[at * 2 + 1] = ll;
      }
    }
  }
  if (p.splits == 1) return;
  // --------------------------------------------------------- join the splits
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(p.count + item, 1u) == (uint32_t)p.splits - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (threadIdx.x == 0) p.count[item] = 0;  // ready for the next call
  // each split's factor 2^(m_s - m) and sum, [split][RT], then their weighted outputs
  float* s_f = reinterpret_cast<float*>(kr_smem);
  float* s_l = s_f + p.splits * RT;
  const size_t first = (size_t)item * p.splits * RT;
  for (int i = threadIdx.x; i < p.splits * RT; i += L::THREADS) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml) + first + i);
    s_f[i] = ml.x;
    s_l[i] = ml.y;
  }
  __syncthreads();
  for (int r = warp; r < live; r += L::WARPS) {
    float mm = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) mm = fmaxf(mm, s_f[s * RT + r]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    for (int s = lane; s < p.splits; s += 32)
      s_f[s * RT + r] = exp2_approx(fsub(s_f[s * RT + r], mm));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < live * (KV_HD / 4); i += L::THREADS) {
    const int r = i / (KV_HD / 4), d = 4 * (i % (KV_HD / 4)), rr = tile * RT + r;
    float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
    float ll = 0.0f;
    constexpr int U = 6;  // loads in flight
    for (int s0 = 0; s0 < p.splits; s0 += U) {
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (s0 + u < p.splits)
          x[u] = __ldcg(reinterpret_cast<const float4*>(
              p.part + (first + (size_t)(s0 + u) * RT + r) * KV_HD + d));
#pragma unroll
      for (int u = 0; u < U; u++)
        if (s0 + u < p.splits) {
          const float f = s_f[(s0 + u) * RT + r];
          oo = make_float4(ffma(f, x[u].x, oo.x), ffma(f, x[u].y, oo.y), ffma(f, x[u].z, oo.z),
                           ffma(f, x[u].w, oo.w));
          ll = ffma(f, s_l[(s0 + u) * RT + r], ll);
        }
    }
    const float inv = fdiv(1.0f, ll);
    *reinterpret_cast<float4*>(a.out + (rr / p.group) * a.out_stride +
                               ((int64_t)head * p.group + rr % p.group) * KV_HD + d) =
        make_float4(fmul(oo.x, inv), fmul(oo.y, inv), fmul(oo.z, inv), fmul(oo.w, inv));
  }
}

}  // namespace flock
