// Attention of a few query rows (one decoded token's heads of a kv head, or a
// short draft) over a cache: k_kv_rows.
//
// Bound: the cache's bytes from HBM (a 4-bit key of one head is 72 + 72 bytes),
// and, near it, the instructions that widen the codes.  So every code is
// widened once, in registers, straight into the operand of a matrix
// instruction, for all query heads that share the kv head.
//
// mma.sync m16n8k16 (bf16, f32 accumulation) rather than tcgen05: with two to
// four live rows there is nothing to amortise a pass of the operands through
// shared memory and tensor memory over; this path takes cached bytes from
// shared memory to the operand registers with no store in between.
//
// f32 results from bf16 operands.  A code minus 8, an e4m3 and a bf16 are bf16
// values; an f32 x is hi + mid + lo, three bf16 of 8 bits each (24 bits, f32's
// range).  Queries and softmax weights are split that way, and the three parts
// sit in different ROWS of the 16-row operand ("slots"), which a decode leaves
// empty anyway: one instruction multiplies all three.  f32 caches split their
// elements too, three instructions a step.
//
// 4-bit blocks.  Scores: a block's 32 products are summed exactly as integers
// times query parts, then multiplied by the key's scale in f32 (one
// accumulator per block).  Values: the scale joins the weight, p d_b, split
// after the product: one weight operand per block.
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

FLOCK_DEV void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
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
// Two f32 -> bf16 pair (nearest even), lo in the low half.
FLOCK_DEV uint32_t bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
FLOCK_DEV float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
FLOCK_DEV float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// x minus the bf16 parts a slot leaves to the ones before it (exact
// differences): part `slot` of hi + mid + lo for two values.
FLOCK_DEV uint32_t bf_part(float x, float y, int slot) {
  uint32_t w = bf2(x, y);
  if (slot >= 1) {
    x = fsub(x, bf_lo(w));
    y = fsub(y, bf_hi(w));
    w = bf2(x, y);
  }
  if (slot >= 2) {
    x = fsub(x, bf_lo(w));
    y = fsub(y, bf_hi(w));
    w = bf2(x, y);
  }
  return w;
}
// Codes at bits 0-3 and 16-19 -> (code - 8) as a bf16 pair: 0x4300 | code is
// the bf16 128 + code, and 136 is taken off exactly.
FLOCK_DEV uint32_t nib_bf2(uint32_t w) {
  const uint32_t u = (w & 0x000F000Fu) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u),
                                   __nv_bfloat162(__ushort_as_bfloat16(0x4308),
                                                  __ushort_as_bfloat16(0x4308)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Two e4m3 in the low half -> bf16 pair, exactly (e4m3 is a subset of both
// f16 and bf16).
FLOCK_DEV uint32_t fp8_bf2(uint32_t w) {
  const float2 f = fp8x2_widen(w);
  return bf2(f.x, f.y);
}

// The head dimension that element e (0-3) of lane column c meets in QK step ks
// (0-7): the order in which a lane's cached bytes unpack.  k_frag and the query
// operand agree on it, so any order is right.
template <int KV>
FLOCK_DEV int kr_kdim(int ks, int c, int e) {
  if (KV == FLOCK_KV_Q4)  // block ks / 2, low or high nibbles of bytes 4 c ..; pairs two apart
    return 32 * (ks >> 1) + 16 * (ks & 1) + 4 * c + ((e & 1) << 1 | e >> 1);
  if (KV == FLOCK_KV_FP8) return 64 * (ks >> 2) + 16 * c + 4 * (ks & 3) + e;
  if (KV == FLOCK_KV_BF16) return 32 * (ks >> 1) + 8 * c + 4 * (ks & 1) + e;
  return 16 * ks + 4 * c + e;
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
// product.
template <int KV>
FLOCK_DEV void kr_load(uint32_t stage, const KvView& c, int head, int64_t key0, int64_t from,
                       int64_t to, int lane) {
  using L = KrLayout<KV>;
  constexpr int CHUNKS = L::ROW / 16;  // 16-byte chunks of a row
  const uint8_t* kb = static_cast<const uint8_t*>(c.k);
  const uint8_t* vb = static_cast<const uint8_t*>(c.v);
  size_t base, step;
  if (KV == FLOCK_KV_Q4) {
    base = q4_row(c, 0, head) * 64;
    step = 64;
  } else {
    base = (size_t)head * L::ROW;
    step = (size_t)c.n_kv_heads * L::ROW;
  }
#pragma unroll
  for (int i = 0; i < KR_GROUP * CHUNKS / 32; i++) {
    const int at = i * 32 + lane, r = at / CHUNKS, ch = at % CHUNKS;
    const bool ok = key0 + r >= from && key0 + r < to;
    const size_t off = base + (size_t)(ok ? key0 + r : from) * step + ch * 16;
    cp_async16(stage + r * L::K_STRIDE + ch * 16, kb + off, ok);
    cp_async16(stage + L::V_OFF + (r >> 2) * L::V_GROUP + (r & 3) * L::ROW + ch * 16, vb + off, ok);
  }
  if (KV == FLOCK_KV_Q4) {
    const int r = lane & 15;
    const bool ok = key0 + r >= from && key0 + r < to;
    const uint16_t* s = (lane < 16 ? c.ks : c.vs) + q4_row(c, ok ? key0 + r : from, head) * 4;
    cp_async8(stage + L::S_OFF + lane * 8, s, ok);
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
FLOCK_DEV float2 h2f2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Keys of a stage are dealt to operand columns so that a lane's four score
// columns are four neighbouring keys: column n of score tile t is key
// 4 (n / 2) + 2 t + n % 2, and lane column c holds keys 4 c .. 4 c + 3.
template <int KV, int RT>
static __global__ void __launch_bounds__(KrLayout<KV>::THREADS, 1) k_kv_rows(const KvRowsArgs p) {
  using L = KrLayout<KV>;
  extern __shared__ __align__(16) uint8_t kr_smem[];
  __shared__ float s_ml[L::WARPS][RT][2];
  __shared__ int s_last;
  const KvAttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int z = blockIdx.x, tile = blockIdx.y, head = blockIdx.z;
  // slot and row of this lane's operand rows: row g is (slot, j), row g + 8
  // carries the last part of four rows and is empty for two
  const int j = g % RT, slot = g / RT;
  const int row = tile * RT + j;
  const int first_q = tile * RT / p.group;
  const int last_row = min(p.rows, (tile + 1) * RT) - 1;
  const int last_q = last_row / p.group;
  // keys that some row of the tile sees: sinks [0, sk), then [lo, hi)
  const int64_t hi = a.pos + last_q + 1;
  const int64_t lo = a.window && a.pos + first_q + 1 > a.window ? a.pos + first_q + 1 - a.window : 0;
  const int64_t sk = a.sinks < lo ? a.sinks : lo;
  const int sink_groups = (int)((sk + KR_GROUP - 1) / KR_GROUP);
  const int64_t lo16 = lo & ~(int64_t)(KR_GROUP - 1);
  const int groups = sink_groups + (int)((hi - lo16 + KR_GROUP - 1) / KR_GROUP);
  const int g0 = (int)((int64_t)z * groups / p.splits), g1 = (int)((int64_t)(z + 1) * groups / p.splits);
  // this row's own keys: sinks [0, row_sk), then [row_lo, row_hi)
  const int my_q = min(row, p.rows - 1) / p.group;
  const int64_t row_hi = a.pos + my_q + 1;
  const int64_t row_lo = a.window && row_hi > a.window ? row_hi - a.window : 0;
  const int64_t row_sk = a.sinks < row_lo ? a.sinks : row_lo;

  const uint32_t ring = smem_u32(kr_smem) + warp * L::STAGES * L::STAGE;
  auto key_of = [&](int grp) -> int64_t {
    return grp < sink_groups ? (int64_t)grp * KR_GROUP : lo16 + (int64_t)(grp - sink_groups) * KR_GROUP;
  };
  auto fetch = [&](int grp, int st) {
    if (grp < g1) {
      const bool sink = grp < sink_groups;
      kr_load<KV>(ring + st * L::STAGE, a.c, head, key_of(grp), sink ? 0 : lo, sink ? sk : hi, lane);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < L::STAGES - 1; s++) fetch(g0 + warp + s * L::WARPS, s);

  // the query operand: q * log2(e) / sqrt(128), its bf16 parts by slot
  uint32_t qa[8][4];
  {
    const float k = __double2float_rn(1.4426950408889634 / sqrt(128.0));
    const bool live = row < p.rows;
    const float* q = a.q + my_q * a.q_stride + ((int64_t)head * p.group + min(row, p.rows - 1) % p.group) * KV_HD;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = live ? fmul(__ldg(q + kr_kdim<KV>(ks, c, e)), k) : 0.0f;
      const bool used = slot < 3;
      qa[ks][0] = used ? bf_part(x[0], x[1], slot) : 0;
      qa[ks][2] = used ? bf_part(x[2], x[3], slot) : 0;
      const bool low = RT == 4 && g < 4;  // row g + 8: part 2 of row g
      qa[ks][1] = low ? bf_part(x[0], x[1], 2) : 0;
      qa[ks][3] = low ? bf_part(x[2], x[3], 2) : 0;
    }
  }
  float o[16][4];
#pragma unroll
  for (int t = 0; t < 16; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) o[t][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  int st = 0;
  for (int grp = g0 + warp; grp < g1; grp += L::WARPS) {
    cp_async_wait<L::STAGES - 2>();
    __syncwarp();  // the stage has landed for every lane, and every lane is done with the last one
    fetch(grp + (L::STAGES - 1) * L::WARPS, st == 0 ? L::STAGES - 1 : st - 1);
    const uint32_t stage = ring + st * L::STAGE;
    // ------------------------------------------------------------- scores
    float s[4];  // keys 4 c + i of this lane's row
    const uint32_t kaddr = stage + (4 * (g >> 1) + (g & 1)) * L::K_STRIDE + 16 * c;
    uint4 sc0, sc1;
    if (KV == FLOCK_KV_Q4) {
      sc0 = lds128(stage + L::S_OFF + 32 * c);
      sc1 = lds128(stage + L::S_OFF + 32 * c + 16);
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const uint32_t kt = kaddr + 2 * t * L::K_STRIDE;
      if constexpr (KV == FLOCK_KV_Q4) {
        const uint4 w4 = lds128(kt);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        const uint4 sc = t ? sc1 : sc0;  // keys 4 c + 2 t and the next, four blocks each
        const float2 d0[2] = {h2f2(sc.x), h2f2(sc.y)}, d1[2] = {h2f2(sc.z), h2f2(sc.w)};
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; b++) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          mma_bf16(acc, qa[2 * b], nib_bf2(w[b]), nib_bf2(w[b] >> 8));
          mma_bf16(acc, qa[2 * b + 1], nib_bf2(w[b] >> 4), nib_bf2(w[b] >> 12));
          if (RT == 4) {
            acc[0] = fadd(acc[0], acc[2]);
            acc[1] = fadd(acc[1], acc[3]);
          }
          s0 = ffma(b & 1 ? d0[b >> 1].y : d0[b >> 1].x, acc[0], s0);
          s1 = ffma(b & 1 ? d1[b >> 1].y : d1[b >> 1].x, acc[1], s1);
        }
        s[2 * t] = s0;
        s[2 * t + 1] = s1;
      } else {
        float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if constexpr (KV == FLOCK_KV_FP8) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint4 w4 = lds128(kt + 64 * h);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
              mma_bf16(acc[i & 1], qa[4 * h + i], fp8_bf2(w[i]), fp8_bf2(w[i] >> 16));
          }
        } else if constexpr (KV == FLOCK_KV_BF16) {
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const uint4 w = lds128(kt + 64 * h);
            mma_bf16(acc[0], qa[2 * h], w.x, w.y);
            mma_bf16(acc[1], qa[2 * h + 1], w.z, w.w);
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 8; ks++) {
            const uint4 w = lds128(kt + 64 * ks);
            const float x0 = __uint_as_float(w.x), x1 = __uint_as_float(w.y),
                        x2 = __uint_as_float(w.z), x3 = __uint_as_float(w.w);
#pragma unroll
            for (int part = 0; part < 3; part++)
              mma_bf16(acc[part & 1], qa[ks], bf_part(x0, x1, part), bf_part(x2, x3, part));
          }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          s[2 * t + i] = fadd(acc[0][i], acc[1][i]);
          if (RT == 4) s[2 * t + i] = fadd(s[2 * t + i], fadd(acc[0][2 + i], acc[1][2 + i]));
        }
      }
    }
    // a row's score is the sum over its slots
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (RT == 2) s[i] = fadd(s[i], __shfl_xor_sync(0xffffffffu, s[i], 8));
      s[i] = fadd(s[i], __shfl_xor_sync(0xffffffffu, s[i], 16));
    }
    const int64_t key0 = key_of(grp);
    {  // masks, only where the group is not wholly visible to every row
      const bool sink = grp < sink_groups;
      const int64_t from = sink ? 0 : row_lo, to = sink ? sk : row_hi;
      if (__any_sync(0xffffffffu, key0 < from || key0 + KR_GROUP > to)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int64_t key = key0 + 4 * c + i;
          // every row sees the tile's sinks; a row's own may reach into the main range
          const bool seen = sink ? key < sk
                                 : key >= lo && key < row_hi && (key >= row_lo || key < row_sk);
          if (!seen) s[i] = -INFINITY;
        }
      }
    }
    // ------------------------------------------------------------ softmax
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // The subtracted maximum may lag by up to 2^8: weights stay far inside
    // f32's range, and the outputs are rescaled in few groups only.
    if (__any_sync(0xffffffffu, top > fadd(m, 8.0f))) {
      const float mn = fmaxf(m, top);
      const float f = mn == -INFINITY ? 1.0f : exp2_approx(fsub(m, mn));
      l = fmul(l, f);
#pragma unroll
      for (int t = 0; t < 16; t++)
#pragma unroll
        for (int e = 0; e < (RT == 4 ? 4 : 2); e++)
          o[t][e] = fmul(o[t][e], f);  // rows g and g + 8 are slots of one row
      m = mn;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = exp2_approx(fsub(s[i], base));
      l = fadd(l, w[i]);
    }
    // ------------------------------------------------------------- values
    const uint32_t vaddr = stage + L::V_OFF + c * L::V_GROUP;
    auto weights = [&](uint32_t (&pa)[4], float x0, float x1, float x2, float x3) {
      pa[0] = slot < 3 ? bf_part(x0, x1, slot) : 0;
      pa[2] = slot < 3 ? bf_part(x2, x3, slot) : 0;
      pa[1] = RT == 4 && g < 4 ? bf_part(x0, x1, 2) : 0;
      pa[3] = RT == 4 && g < 4 ? bf_part(x2, x3, 2) : 0;
    };
    if constexpr (KV == FLOCK_KV_Q4) {
      uint2 v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = lds64(vaddr + i * 64 + 8 * g);
      const uint4 e0 = lds128(stage + L::S_OFF + 128 + 32 * c);
      const uint4 e1 = lds128(stage + L::S_OFF + 128 + 32 * c + 16);
      const uint32_t es[4][2] = {{e0.x, e0.y}, {e0.z, e0.w}, {e1.x, e1.y}, {e1.z, e1.w}};
#pragma unroll
      for (int hb = 0; hb < 2; hb++) {
        float2 d[4];
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = h2f2(es[i][hb]);
#pragma unroll
        for (int bb = 0; bb < 2; bb++) {
          const int b = 2 * hb + bb;
          // p d; a masked key's scale may be anything finite, its weight is 0
          uint32_t pa[4];
          weights(pa, fmul(w[0], bb ? d[0].y : d[0].x), fmul(w[1], bb ? d[1].y : d[1].x),
                  fmul(w[2], bb ? d[2].y : d[2].x), fmul(w[3], bb ? d[3].y : d[3].x));
          const uint32_t v0 = hb ? v[0].y : v[0].x, v1 = hb ? v[1].y : v[1].x,
                         v2 = hb ? v[2].y : v[2].x, v3 = hb ? v[3].y : v[3].x;
          const uint32_t k01 = __byte_perm(v0, v1, bb ? 0x7632 : 0x5410);
          const uint32_t k23 = __byte_perm(v2, v3, bb ? 0x7632 : 0x5410);
          // tile 4 b + e: nibble e of the halfword (low and high nibble of byte 0, then byte 1)
#pragma unroll
          for (int e = 0; e < 4; e++)
            mma_bf16(o[4 * b + e], pa, nib_bf2(k01 >> (4 * e)), nib_bf2(k23 >> (4 * e)));
        }
      }
    } else {
      uint32_t pa[4];
      weights(pa, w[0], w[1], w[2], w[3]);
      if constexpr (KV == FLOCK_KV_FP8) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = lds128(vaddr + i * 128 + 16 * g);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint32_t x[4] = {q == 0 ? v[0].x : q == 1 ? v[0].y : q == 2 ? v[0].z : v[0].w,
                                 q == 0 ? v[1].x : q == 1 ? v[1].y : q == 2 ? v[1].z : v[1].w,
                                 q == 0 ? v[2].x : q == 1 ? v[2].y : q == 2 ? v[2].z : v[2].w,
                                 q == 0 ? v[3].x : q == 1 ? v[3].y : q == 2 ? v[3].z : v[3].w};
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = fp8_bf2(x[i] >> (16 * h));
            mma_bf16(o[4 * q + 2 * h], pa, __byte_perm(y[0], y[1], 0x5410),
                     __byte_perm(y[2], y[3], 0x5410));
            mma_bf16(o[4 * q + 2 * h + 1], pa, __byte_perm(y[0], y[1], 0x7632),
                     __byte_perm(y[2], y[3], 0x7632));
          }
        }
      } else if constexpr (KV == FLOCK_KV_BF16) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = lds128(vaddr + i * 256 + 128 * h + 16 * g);
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = q == 0 ? v[i].x : q == 1 ? v[i].y : q == 2 ? v[i].z : v[i].w;
            mma_bf16(o[8 * h + 2 * q], pa, __byte_perm(x[0], x[1], 0x5410),
                     __byte_perm(x[2], x[3], 0x5410));
            mma_bf16(o[8 * h + 2 * q + 1], pa, __byte_perm(x[0], x[1], 0x7632),
                     __byte_perm(x[2], x[3], 0x7632));
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
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
              x[i] = __uint_as_float(q == 0 ? v[i].x : q == 1 ? v[i].y : q == 2 ? v[i].z : v[i].w);
#pragma unroll
            for (int part = 0; part < 3; part++)
              mma_bf16(o[4 * h + q], pa, bf_part(x[0], x[1], part), bf_part(x[2], x[3], part));
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
#pragma unroll
  for (int t = 0; t < 16; t++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float x = o[t][e];
      if (RT == 2) x = fadd(x, __shfl_xor_sync(0xffffffffu, x, 8));
      if (RT == 4) x = fadd(x, o[t][2 + e]);
      x = fadd(x, __shfl_xor_sync(0xffffffffu, x, 16));
      if (g < RT) s_o[(warp * RT + j) * KV_HD + kr_vdim<KV>(t, 2 * c + e)] = x;
    }
  if (g < RT && c == 0) {
    s_ml[warp][j][0] = m;
    s_ml[warp][j][1] = l;
  }
  __syncthreads();
  const int item = head * gridDim.y + tile;
  const int n_items = gridDim.y * gridDim.z;
  float* part_ml = p.part + (size_t)n_items * p.splits * RT * KV_HD;
  for (int i = threadIdx.x; i < RT * KV_HD; i += L::THREADS) {
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
      if (rr < p.rows)
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
  for (int i = threadIdx.x; i < RT * KV_HD; i += L::THREADS) {
    const int r = i / KV_HD, d = i % KV_HD, rr = tile * RT + r;
    if (rr >= p.rows) break;
    const size_t at = (size_t)item * p.splits * RT + r;
    float mm = -INFINITY;
    for (int s = 0; s < p.splits; s++) mm = fmaxf(mm, __ldcg(part_ml + (at + s * RT) * 2));
    float oo = 0.0f, ll = 0.0f;
    for (int s = 0; s < p.splits; s++) {
      const float f = exp2_approx(fsub(__ldcg(part_ml + (at + s * RT) * 2), mm));
      oo = ffma(f, __ldcg(p.part + (at + s * RT) * KV_HD + d), oo);
      ll = ffma(f, __ldcg(part_ml + (at + s * RT) * 2 + 1), ll);
    }
    a.out[(rr / p.group) * a.out_stride + ((int64_t)head * p.group + rr % p.group) * KV_HD + d] =
        fdiv(oo, ll);
  }
  if (threadIdx.x == 0) p.count[item] = 0;  // ready for the next call
}

}  // namespace flock
