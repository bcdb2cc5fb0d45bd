// Attention of many query rows (a prompt chunk, a long draft) over a cache on
// the tcgen05 tensor cores, to f32 accuracy: k_kv_prompt.
//
// CTA (row tile of 128 (query, head) rows of a kv head, key split), looping
// over 128-key tiles; per tile S = Q K^T and O += P V, f32 accumulators in
// tensor memory.  Bound: the tensor cores' f16 rate times the products below,
// with the softmax's instructions near it.
//
// f32 results from f16 operands.  q (scaled by a power of two per row) and the
// softmax weights are hi + lo, two f16.  An e4m3 value is an f16 value: two
// products (hi, lo times it), and so is a bf16 value once its tile is scaled by a
// power of two into f16's range.  A 4-bit value (code - 8) * scale has 15
// significant bits, an f32 24: hi + lo again, three products (lo lo is below
// 2^-22).
//
// Alone (PAIR false) a CTA widens every key for its 128 rows.  A pair, two CTAs
// of a cluster with neighbouring row tiles and the same keys, shares that work:
// the products are cta_group::2, 256 rows over both CTAs' tensor memory, and
// either CTA widens and keeps half of a B operand's rows (keys of K, output
// columns of V), in two stages.  1024 queries over 8192 4-bit keys, 16 / 8 heads:
// 187 us against 216; three products an operand pair at the sustained rate are
// 136, and the clock falls to 1.55 GHz under them.
//
// Roles, sixteen warps of 128 registers:
//   warps 0-7   softmax; thread = row = tensor-memory lane, warps 0-3 the
//               first 64 of its 128 scores, 4-7 the others (one thread a row
//               took 6500 cycles a tile, its 128 scores' chains alone on a
//               scheduler; so 3100).  They agree on the row's maximum in shared
//               memory, and write the weights' hi and lo parts over the scores in
//               tensor memory (the second product's A operand is read there).
//   warps 8-11  widen the next K and V tiles from global memory into the
//               128-byte-swizzled shared-memory operands (raw bytes are loaded
//               into registers a tile ahead).  The order of dimensions (K: those
//               q is given in; V: the output's columns) is whatever unpacks
//               without shuffling, and is undone at the ends.
//   warp 12     one thread (of the pair's first CTA) issues the products: O(t),
//               then S(t+2) over its weights, while the softmax of t+1 goes on.
//
// A barrier that a thread may find two phases on is two barriers, by the tile's
// parity: the weights' and the outputs'.
//
// The tensor cores' accumulators do not round to nearest: each step loses half a
// last bit on average, towards zero, so a sum of n steps shrinks by about n
// 2^-25 (1128 steps over 6000 keys: 2.3e-5).  The small products of a score go
// first, and the outputs move to an f32 sum in shared memory every KP_FLUSH
// tiles, added there in f32 (96 steps: 1e-6; 16 us of the 187).
//
// The running maximum may lag by 2^4 before the outputs are rescaled (as in
// k_kv_rows).
//
// f16 parts hold a number to 2^-22 of itself down to 2^-15 of its tile's largest,
// below that to 2^-38 of the largest.  That is enough while the largest is no
// outlier.  Where it is, a CTA's rows are worked out again in f32, a warp a row
// (kp_exact_rows), after a look at bounds that cost next to nothing:
//   scores  a row's largest |q| times a tile's largest |k| bounds what the lost
//           bits of q and k can move a score by;
//   values  the tiles' largest (4-bit: all scales) further apart than 2^KR_SPREAD,
//           or more than a few of a tile's elements below 2^-15 of its largest (a
//           key or a column of such is more; of 4096 normal ones about one).
// Large keys or values may belong to keys that a row does not see, to others'
// dimensions, or be infinite or NaN: the f32 rows are free of them.
//
// Every wait is bounded; a wait that runs out ends the CTA, which
// then writes NaN (and so does its partner) and sets a layer's error word.
#pragma once
#include "gemm_tc.cuh"
#include "kv_rows.cuh"

namespace flock {

constexpr int KP_ROWS = 128;     // query rows per CTA
constexpr int KP_KEYS = 128;     // keys per tile
constexpr int KP_THREADS = 512;
constexpr int KP_FLUSH = 4;      // key tiles an output accumulator takes
constexpr int KP_SUM_STRIDE = 132;  // floats of a row of the outputs' sum: rows 4 banks apart
constexpr int KP_OPND = 128 * 128 * 2;  // bytes of one 128 x 128 f16 operand

// Bounds of that look.  Scores: q's and k's f16 parts are off by 2^-25 each at
// most (q up to 2^14, k to 2^13), 128 terms by 2^-3.4, typically 2^-8, in units f: f up
// to 2^-12 moves a score by 2^-15.4, typically 2^-20.  e4m3 keys are exact, up to 448:
// 2^-9.2 of q's unit, typically 2^-13.
constexpr float KP_MAX_UNIT = 0x1p-12f, KP_MAX_UNIT_FP8 = 0x1p-6f;
// Values: elements of a warp's 32 keys below 2^-15 of the tile's largest (2^-2 as
// scaled), of which a column has 32 and a key 64 or 128.  Half of the elements are
// looked at, half of each key's and of each column's.
constexpr float KP_SMALL = 0.25f;
constexpr int KP_FEW = 24;

struct KvPromptArgs {
  KvAttnArgs a;
  int rows, group;  // row r is query r / group, head r % group
  int splits;
  float* part;      // [item][split][128 rows][128], then [..][128 rows][2] (base, l)
};

// 16-byte chunk c (8 columns) of row r of an operand of ROWS rows and 128
// columns: two 64-column halves of swizzled 128-byte rows.
template <int ROWS>
FLOCK_DEV uint32_t kp_off(int r, int c) {
  return (uint32_t)(c >> 3) * (ROWS * 128u) + sw128_off(r, c & 7);
}
// D (+)= A B^T over 128 K elements; A in tensor memory (a column holds two).
// PAIR: both CTAs' 128 rows of A and D, half of B's 128 rows in either.
template <bool PAIR>
FLOCK_DEV void kp_mma(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  const uint32_t idesc = umma_idesc_f16(PAIR ? 256 : 128, 128);
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const uint32_t off = (uint32_t)(k >> 2) * (PAIR ? 8192u : 16384u) + (uint32_t)(k & 3) * 32u;
    const uint64_t desc = umma_desc_sw128(b + off);
    const uint32_t acc = accumulate || k > 0 ? 1u : 0u;
    if constexpr (PAIR)
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
          " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
          "r"(a + 8u * k), "l"(desc), "r"(idesc), "r"(acc)
          : "memory");
    else
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
          " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
          "r"(a + 8u * k), "l"(desc), "r"(idesc), "r"(acc)
          : "memory");
  }
}
// The barrier (of both CTAs) arrives once the products issued so far are done.
template <bool PAIR>
FLOCK_DEV void kp_commit(uint64_t* b) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(b)), "h"((uint16_t)3)
        : "memory");
  else
    umma_commit(b);
}
template <bool PAIR>
FLOCK_DEV void kp_alloc(uint32_t* slot) {  // all 512 columns
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
}
template <bool PAIR>
FLOCK_DEV void kp_free(uint32_t t) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(t) : "memory");
  else
    tmem_dealloc(t, 512);
}
FLOCK_DEV void kp_cluster_sync() {  // every thread of both CTAs
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What a thread arrives for (PAIR: its warp, at the first CTA's barrier, whose
// thread issues the products of both).  What the barrier hands on, shared-memory
// operands and tensor memory, each thread has ordered itself before it arrives
// (proxy fence; store wait and tcgen05 fence), so the arrival need not be a
// release over the cluster, which waits 1000 cycles for every access of the warp.
template <bool PAIR>
FLOCK_DEV void kp_arrive(uint64_t* b) {
  if constexpr (PAIR) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
      asm volatile(
          "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n"
          " mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(smem_u32(b))
          : "memory");
  } else {
    mbar_arrive(b);
  }
}
// 32 columns of this thread's lane; waits for them, so that no use can come before.
FLOCK_DEV void kp_ld32(uint32_t t, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t)
      : "memory");
}
FLOCK_DEV void kp_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
FLOCK_DEV void kp_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
FLOCK_DEV void kp_bar(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The head dimension of q's column pair word w (0-63), half h, in the K
// operand's order; and of output column j (0-127), in V's.
template <int KV>
FLOCK_DEV constexpr int kp_kdim(int w, int h) {
  if (KV != FLOCK_KV_Q4) return 2 * w + h;
  // chunk w / 4 is word c of block b: nibbles at bits 0, 8, 4, 12 of both halfwords
  const int b = w >> 4, c = (w >> 2) & 3, i = w & 3;
  return 32 * b + 16 * (i >> 1) + 4 * c + (i & 1) + 2 * h;
}
template <int KV>
FLOCK_DEV constexpr int kp_vcol(int d) {
  if (KV != FLOCK_KV_Q4) return 8 * (d & 15) + (d >> 4);
  const int b = d >> 5, hi = (d >> 4) & 1, n = (d & 15) >> 1, byte = d & 1;
  return 32 * b + 8 * (2 * byte + hi) + n;
}

// Shared memory: the operands K hi, V hi, then K lo, V lo, and the outputs' sum.
template <int KV>
constexpr bool KP_LO = KV == FLOCK_KV_Q4 || KV == FLOCK_KV_F32;  // K and V in two parts
template <int KV>
constexpr size_t KP_SMEM =
    (KP_LO<KV> ? 4 : 2) * (size_t)KP_OPND + 128 * KP_SUM_STRIDE * 4 + 1024;

// Sixteen rows of a tile from the keys of tiles [t0, t1) in f32, by one warp, four
// rows and four keys at a time: outputs (normalised where nothing is joined later)
// into the rows' part of s_sum, (base, l) into part_ml.  A key that a row does not
// see is not part of its arithmetic, whatever it holds.  The sixteen scores are
// added up over the lanes together, each step halving the values a lane holds:
// lane 2 (4 i + j) has row i's with key j.  Rare, and slow: 1024 queries at 3000
// keys, 16 / 8 heads, 4 to 6 ms where the tensor cores take 0.1 to 0.25.
template <int KV>
FLOCK_DEV void kp_exact_rows(const KvPromptArgs& p, int tile, int head, int pos, int lo, int hi,
                             int sk, int t0, int t1, float* s_sum, float* part_ml) {
  const KvAttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sink_tiles = (sk + KP_KEYS - 1) / KP_KEYS, lo16 = lo & ~15;
  const float scale = __double2float_rn(1.4426950408889634 / sqrt(128.0));
#pragma unroll 1
  for (int i0 = 0; i0 < 16; i0 += 4) {
    const int row0 = tile * KP_ROWS + 16 * warp + i0;
    if (row0 >= p.rows) return;
    float4 q[4], o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = min(row0 + i, p.rows - 1);
      const float4 x = __ldg(reinterpret_cast<const float4*>(
                                 a.q + (r / p.group) * a.q_stride +
                                 ((int64_t)head * p.group + r % p.group) * KV_HD) + lane);
      q[i] = make_float4(fmul(x.x, scale), fmul(x.y, scale), fmul(x.z, scale), fmul(x.w, scale));
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // the lane's row (and its key of four): bounds, running maximum and sum
    const int row_hi = pos + min(row0 + (lane >> 3), p.rows - 1) / p.group + 1;
    const int row_lo = a.window && row_hi > a.window ? row_hi - a.window : 0;
    const int row_sk = min(a.sinks, row_lo);
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    for (int t = t0; t < t1; t++) {
      const bool sink = t < sink_tiles;
      const int key0 = sink ? t * KP_KEYS : lo16 + (t - sink_tiles) * KP_KEYS;
      const int from = max(key0, sink ? 0 : lo), to = min(key0 + KP_KEYS, sink ? sk : hi);
#pragma unroll 1
      for (int key = from; key < to; key += 4) {
        float4 k[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          k[j] = v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (key + j < to) {
            k[j] = kv_load4<KV, true>(a.c, key + j, head, lane);
            v[j] = kv_load4<KV, false>(a.c, key + j, head, lane);
          }
        }
        float s[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float4 x = q[i >> 2], y = k[i & 3];
          s[i] = ffma(x.x, y.x, ffma(x.y, y.y, ffma(x.z, y.z, fmul(x.w, y.w))));
        }
#pragma unroll
        for (int h = 8; h > 0; h >>= 1) {  // lanes 2 h apart trade halves
          const bool up = lane & (2 * h);
#pragma unroll
          for (int i = 0; i < h; i++) {
            const float give = up ? s[i] : s[i + h], own = up ? s[i + h] : s[i];
            s[i] = fadd(own, __shfl_xor_sync(0xffffffffu, give, 2 * h));
          }
        }
        float x = fadd(s[0], __shfl_xor_sync(0xffffffffu, s[0], 1));
        const int own = key + ((lane >> 1) & 3);
        if (own >= to || own >= row_hi || (own < row_lo && own >= row_sk)) x = -INFINITY;
        float top = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        top = fmaxf(m, fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4)));
        const float f = m == -INFINITY ? 0.0f : exp2_approx(fsub(m, top));
        const float w = x == -INFINITY ? 0.0f : exp2_approx(fsub(x, top));
        float sum = fadd(w, __shfl_xor_sync(0xffffffffu, w, 2));
        sum = fadd(sum, __shfl_xor_sync(0xffffffffu, sum, 4));
        l = ffma(l, f, sum);
        m = top;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float g = __shfl_sync(0xffffffffu, f, 8 * i);
          o[i] = make_float4(fmul(o[i].x, g), fmul(o[i].y, g), fmul(o[i].z, g), fmul(o[i].w, g));
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float e = __shfl_sync(0xffffffffu, w, 8 * i + 2 * j);
            if (e != 0.0f)
              o[i] = make_float4(ffma(e, v[j].x, o[i].x), ffma(e, v[j].y, o[i].y),
                                 ffma(e, v[j].z, o[i].z), ffma(e, v[j].w, o[i].w));
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float row_l = __shfl_sync(0xffffffffu, l, 8 * i);
      const float inv = p.splits == 1 ? fdiv(1.0f, row_l) : 1.0f;
      reinterpret_cast<float4*>(s_sum)[(16 * warp + i0 + i) * (KP_SUM_STRIDE / 4) + lane] =
          make_float4(fmul(o[i].x, inv), fmul(o[i].y, inv), fmul(o[i].z, inv), fmul(o[i].w, inv));
    }
    if (p.splits > 1 && (lane & 7) == 0 && row0 + (lane >> 3) < p.rows) {
      part_ml[(16 * warp + i0 + (lane >> 3)) * 2] = m;
      part_ml[(16 * warp + i0 + (lane >> 3)) * 2 + 1] = l;
    }
  }
}

template <int KV, bool PAIR>
static __global__ void __launch_bounds__(KP_THREADS, 1) k_kv_prompt(const KvPromptArgs p) {
  // operand rows here (keys of K, output columns of V), stages of them, their bytes
  constexpr int OR = PAIR ? 64 : 128, NB = PAIR ? 2 : 1, OP = KP_OPND / NB;
  constexpr bool Q4 = KV == FLOCK_KV_Q4, LO = KP_LO<KV>;
  constexpr bool WIDE = KV == FLOCK_KV_F32 || KV == FLOCK_KV_BF16;  // elements scaled by tile
  constexpr bool SCALED = KV != FLOCK_KV_FP8;
  extern __shared__ __align__(16) uint8_t kp_raw[];
  __shared__ uint64_t s_bar[14];
  __shared__ uint32_t s_tmem;
  __shared__ int s_err, s_ok[2];
  __shared__ int s_far[2];  // f16 parts do not do: found by the softmax warps, by the converters
  __shared__ float s_top[2][2][128];  // a row's maximum over either half, by tile parity
  __shared__ uint32_t s_dmax[2][4];   // converters: a warp's largest scale of K, V
  __shared__ uint32_t s_dmin[4];      // 4-bit: its smallest of V
  __shared__ float s_kscale[4];       // K tile's factor back, by tile % 4
  __shared__ int s_vexp[4];           // V tile's exponent
  uint8_t* base = kp_raw + ((1024u - (smem_u32(kp_raw) & 1023u)) & 1023u);
  uint8_t* sKh = base;
  uint8_t* sVh = base + KP_OPND;
  uint8_t* sKl = base + 2 * KP_OPND;
  uint8_t* sVl = base + 3 * KP_OPND;
  float* s_sum = reinterpret_cast<float*>(base + (LO ? 4 : 2) * KP_OPND);
  uint64_t *k_full = s_bar, *k_empty = s_bar + 2, *v_full = s_bar + 4, *v_empty = s_bar + 6,
           *s_full = s_bar + 8, *p_full = s_bar + 10, *q_full = s_bar + 12, *drained = s_bar + 13;
  auto stage = [](int t) { return NB == 2 ? t & 1 : 0; };
  auto phase = [](int t) { return (uint32_t)(NB == 2 ? t >> 1 : t) & 1; };
  const KvAttnArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x, z = blockIdx.y, head = blockIdx.z;
  const int rank = PAIR ? tile & 1 : 0;
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(k_full + i, PAIR ? 8 : 128);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, PAIR ? 8 : 128);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, PAIR ? 16 : 256);
    }
    mbar_init(q_full, PAIR ? 16 : 256);
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_err = s_far[0] = s_far[1] = 0;
  }
  if (warp == 12) kp_alloc<PAIR>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  if (PAIR) kp_cluster_sync();  // the other CTA's barriers are there to arrive at
  tc_fence_after();
  pdl_launch_dependents();  // after the allocation: a later grid's cannot hold what this one needs
  pdl_wait();
  const uint32_t tmem = s_tmem, tS = tmem, tO = tmem + 256, tQ = tmem + 384;

  // keys that some row of the tile (of both tiles of a pair) sees: sinks [0, sk),
  // then [lo, hi)
  const int pos = kv_attn_pos(a);
  const int first_q = (tile - rank) * KP_ROWS / p.group;
  const int last_q = (min(p.rows, (tile - rank + NB) * KP_ROWS) - 1) / p.group;
  const int hi = pos + last_q + 1;
  const int lo = a.window && pos + first_q + 1 > a.window ? pos + first_q + 1 - a.window : 0;
  const int sk = min(a.sinks, lo);
  const int sink_tiles = (sk + KP_KEYS - 1) / KP_KEYS;
  const int lo16 = lo & ~15;
  const int all = sink_tiles + (hi - lo16 + KP_KEYS - 1) / KP_KEYS;
  const int t0 = (int)((int64_t)z * all / p.splits), t1 = (int)((int64_t)(z + 1) * all / p.splits);
  const int n = t1 - t0;
  auto key_of = [&](int t) {
    return t0 + t < sink_tiles ? (t0 + t) * KP_KEYS : lo16 + (t0 + t - sink_tiles) * KP_KEYS;
  };
  auto fail = [&]() {
    *(volatile int*)&s_err = 1;
    if (a.err) atomicCAS(a.err, 0, 1);
  };

  if (warp < 8) {
    // ============================================================== softmax
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const int half = warp >> 2, r = tid & 127;  // scores (then output columns) 64 half ..
    const int row = tile * KP_ROWS + r;
    const bool live = row < p.rows;
    const int query = min(row, p.rows - 1) / p.group;
    const int row_hi = pos + query + 1;
    const int row_lo = a.window && row_hi > a.window ? row_hi - a.window : 0;
    const int row_sk = min(a.sinks, row_lo);
    // keys in [max_lo, min_hi) are seen by every row of this CTA
    const int own_last = (min(p.rows, (tile + 1) * KP_ROWS) - 1) / p.group;
    const int max_lo = a.window && pos + own_last + 1 > a.window ? pos + own_last + 1 - a.window : 0;
    const int min_hi = pos + min(tile * KP_ROWS, p.rows - 1) / p.group + 1;
    float unscale;
    {  // q log2(e) / sqrt(128), the row's largest in [2^13, 2^14), hi and lo parts
      // A warp reads whole rows (sixteen, 512 bytes each at once); a thread takes
      // its own from the outputs' sum, which is not in use yet.  (A thread's
      // own row straight from memory: 8 us.)
      const float k = __double2float_rn(1.4426950408889634 / sqrt(128.0));
      float4* sq = reinterpret_cast<float4*>(s_sum);
      float4 x16[16];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int rr = min(tile * KP_ROWS + 16 * warp + i, p.rows - 1);
        x16[i] = __ldg(reinterpret_cast<const float4*>(
                           a.q + (rr / p.group) * a.q_stride +
                           ((int64_t)head * p.group + rr % p.group) * KV_HD) + lane);
      }
#pragma unroll
      for (int i = 0; i < 16; i++) {
        auto mag = [](float y) { return __float_as_uint(y) & 0x7FFFFFFFu; };
        const uint32_t most = __reduce_max_sync(
            0xffffffffu, max(max(mag(x16[i].x), mag(x16[i].y)), max(mag(x16[i].z), mag(x16[i].w))));
        if (lane == 0) s_top[0][0][16 * warp + i] = __uint_as_float(most);
        sq[(16 * warp + i) * (KP_SUM_STRIDE / 4) + lane] = x16[i];
      }
      kp_bar(2, 256);
      const float top = fmul(s_top[0][0][r], k);
      const int biased = (int)(__float_as_uint(top) >> 23);
      const int e = max(-100, min(100, biased - 127 - 13));
      if (biased - 127 - 13 > 100) *(volatile int*)&s_far[0] = 1;
      const float scale = live ? __uint_as_float((uint32_t)(127 - e) << 23) : 0.0f;
      unscale = __uint_as_float((uint32_t)(127 + e) << 23);
      if (!SCALED && unscale > KP_MAX_UNIT_FP8) *(volatile int*)&s_far[0] = 1;
#pragma unroll
      for (int b = 0; b < 2; b++) {  // 32 dimensions: one block
        const int w0 = 32 * half + 16 * b;
        float x[32];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float4 v = sq[r * (KP_SUM_STRIDE / 4) + w0 / 2 + i];
          x[4 * i] = fmul(fmul(v.x, k), scale);
          x[4 * i + 1] = fmul(fmul(v.y, k), scale);
          x[4 * i + 2] = fmul(fmul(v.z, k), scale);
          x[4 * i + 3] = fmul(fmul(v.w, k), scale);
        }
        uint32_t h[16], l[16];
#pragma unroll
        for (int i = 0; i < 16; i++)  // every block's order is the first one's
          split_f16(x[kp_kdim<KV>(i, 0)], x[kp_kdim<KV>(i, 1)], h[i], l[i]);
        kp_st16(tQ + lanes + w0, h);
        kp_st16(tQ + lanes + 64 + w0, l);
      }
      kp_st_wait();
      tc_fence_before();
      kp_arrive<PAIR>(q_full);
    }
    float m = -INFINITY, base_ = 0.0f, l = 0.0f;
    int vexp = -1000;
    bool ok = true;
    for (int t = 0; t < n && ok; t++) {
      const uint32_t S = tS + 128u * (t & 1) + lanes;
      if (!mbar_wait(s_full + (t & 1), (t >> 1) & 1, &s_err)) fail();
      tc_fence_after();
      float s[64];
#pragma unroll
      for (int i = 0; i < 2; i++) kp_ld32(S + 64 * half + 32 * i, s + 32 * i);
      // not 0, which times a masked score is NaN; below 2^-126 a score is 0 anyway
      const float f = SCALED ? fmaxf(fmul(unscale, s_kscale[t & 3]), 0x1p-126f) : unscale;
      if (SCALED && f > KP_MAX_UNIT) *(volatile int*)&s_far[0] = 1;
      const int ve = SCALED ? s_vexp[t & 3] : 0;
      const int key0 = key_of(t);
      const bool sink = t0 + t < sink_tiles;
      if (sink ? key0 + KP_KEYS > sk : key0 < max_lo || key0 + KP_KEYS > min_hi) {
        // every row sees the tile's sinks; a row's own may reach into the main range
        const int from = sink ? 0 : max(lo, row_lo), to = sink ? sk : row_hi;
        const int also = sink ? 0 : row_sk;
#pragma unroll
        for (int i = 0; i < 64; i++) {
          const int key = key0 + 64 * half + i;
          if (!((key >= from && key < to) || (key >= lo && key < also))) s[i] = -INFINITY;
        }
      }
      float t4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < 64; i++) t4[i & 3] = fmaxf(t4[i & 3], s[i]);
      float top = fmul(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])), f);
      // the other half's; behind this barrier both halves have left the scores'
      // columns, which the weights overwrite
      s_top[t & 1][half][r] = top;
      if (tid == 0) s_ok[t & 1] = *(volatile int*)&s_err == 0;
      kp_bar(2, 256);
      ok = s_ok[t & 1];  // one thread's look, so that all leave the loop together
      top = fmaxf(top, s_top[t & 1][half ^ 1][r]);
      const bool grow = __any_sync(0xffffffffu, top > fadd(m, 4.0f) || ve > vexp);
      const bool flush = t > 0 && t % KP_FLUSH == 0;
      float go = 1.0f;  // the outputs so far, in the new units
      if (grow) {
        const float mn = fmaxf(m, top);
        const float nb = mn == -INFINITY ? 0.0f : fsub(mn, 10.0f);
        const float g = m == -INFINITY ? 0.0f : exp2_approx(fsub(base_, nb));
        const int ne = max(vexp, ve);
        l = fmul(l, g);
        go = fmul(g, pow2f(max(vexp - ne, -120)));
        m = mn;
        base_ = nb;
        vexp = ne;
      }
      if (t > 0 && (flush || __any_sync(0xffffffffu, go != 1.0f))) {
        // O(t-2) is complete with these scores, O(t-1) is waited for, and O(t)
        // waits for this thread
        if (ok && !mbar_wait(v_empty + ((t - 1) & 1), ((t - 1) >> 1) & 1, &s_err)) fail();
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const uint32_t at = tO + lanes + 64 * half + 32 * i;
          float4* sum = reinterpret_cast<float4*>(s_sum + r * KP_SUM_STRIDE + 64 * half + 32 * i);
          float o[32];
          kp_ld32(at, o);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            float4 x = t > KP_FLUSH ? sum[j] : make_float4(0.f, 0.f, 0.f, 0.f);
            if (flush)
              x = make_float4(fadd(x.x, o[4 * j]), fadd(x.y, o[4 * j + 1]), fadd(x.z, o[4 * j + 2]),
                              fadd(x.w, o[4 * j + 3]));
            if (flush || t > KP_FLUSH)
              sum[j] = make_float4(fmul(x.x, go), fmul(x.y, go), fmul(x.z, go), fmul(x.w, go));
          }
          if (!flush) {
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = fmul(o[j], go);
            kp_st16(at, reinterpret_cast<uint32_t*>(o));
            kp_st16(at + 16, reinterpret_cast<uint32_t*>(o) + 16);
          }
        }
      }
      // weights times the V tile's own power of two over the outputs'
      const float shift = fsub((float)(ve - vexp), base_);
      const uint64_t f2 = pack2(f, f), shift2 = pack2(shift, shift), one2 = pack2(1.0f, 1.0f);
      uint64_t sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 2; c++) {  // 32 keys
        uint32_t h[16], w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float2 x =
              unpack2(ffma2(pack2(s[32 * c + 2 * i], s[32 * c + 2 * i + 1]), f2, shift2));
          const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
          const uint64_t e2 = pack2(e.x, e.y);
          sum[i & 1] = ffma2(e2, one2, sum[i & 1]);
          h[i] = hf2(e.x, e.y);
          const float2 hi = h2f2(h[i]);
          const float2 rest = unpack2(fsub2(e2, pack2(hi.x, hi.y)));
          w[i] = hf2(rest.x, rest.y);
        }
        kp_st16(S + 32 * half + 16 * c, h);
        kp_st16(S + 64 + 32 * half + 16 * c, w);
      }
      const float2 sum0 = unpack2(sum[0]), sum1 = unpack2(sum[1]);
      l = ffma(fadd(fadd(sum0.x, sum0.y), fadd(sum1.x, sum1.y)), pow2f(min(vexp - ve, 120)), l);
      kp_st_wait();
      tc_fence_before();
      kp_arrive<PAIR>(p_full + (t & 1));
    }
    // ------------------------------------------------------------ epilogue
    // the last scores being there says that O(n-3) is complete: either of the two
    // after it has a barrier of its own, so that its parity says which
    for (int t = max(n - 2, 0); t < n; t++)
      if (ok && !mbar_wait(v_empty + (t & 1), (t >> 1) & 1, &s_err)) fail();
    kp_bar(3, 384);  // s_top is read, every wait decided, the converters are done
    s_top[0][half][r] = l;
    kp_bar(2, 256);
    ok = *(volatile int*)&s_err == 0;
    if (PAIR) {  // the other CTA's keys and columns are in these rows too
      int other;
      asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n"
                   " ld.volatile.shared::cluster.s32 %0, [a];\n}\n"
                   : "=r"(other) : "r"(smem_u32(&s_err)), "r"(rank ^ 1) : "memory");
      ok = ok && other == 0;
    }
    // behind the last outputs every converter of the pair has said what it found
    bool far = *(volatile int*)&s_far[0] || *(volatile int*)&s_far[1];
    if (PAIR && WIDE) {
      int other;
      asm volatile("{\n .reg .b32 a;\n fence.acq_rel.cluster;\n mapa.shared::cluster.u32 a, %1, %2;\n"
                   " ld.volatile.shared::cluster.s32 %0, [a];\n}\n"
                   : "=r"(other) : "r"(smem_u32(&s_far[1])), "r"(rank ^ 1) : "memory");
      far = far || other != 0;
    }
    l = fadd(s_top[0][0][r], s_top[0][1][r]);
    tc_fence_after();
    float o[64];
#pragma unroll
    for (int i = 0; i < 64; i++) o[i] = 0.0f;
    if (ok && n > 0) {
#pragma unroll
      for (int i = 0; i < 2; i++) kp_ld32(tO + lanes + 64 * half + 32 * i, o + 32 * i);
      if (n > KP_FLUSH) {
        const float4* sum = reinterpret_cast<const float4*>(s_sum + r * KP_SUM_STRIDE + 64 * half);
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const float4 x = sum[j];
          o[4 * j] = fadd(o[4 * j], x.x);
          o[4 * j + 1] = fadd(o[4 * j + 1], x.y);
          o[4 * j + 2] = fadd(o[4 * j + 2], x.z);
          o[4 * j + 3] = fadd(o[4 * j + 3], x.w);
        }
      }
    }
    // through shared memory, so that a warp writes whole rows (a thread its own
    // straight to memory: 4 us)
    const float mul = fmul(ok ? (n > 0 ? pow2f(max(vexp, -120)) : 0.0f) : NAN,
                           p.splits == 1 ? fdiv(1.0f, l) : 1.0f);
    const size_t part_row = (((size_t)head * gridDim.x + tile) * p.splits + z) * KP_ROWS;
    float* part_ml = p.part + (size_t)gridDim.z * gridDim.x * p.splits * KP_ROWS * KV_HD + part_row * 2;
    if (live && half == 0 && p.splits > 1) {
      part_ml[2 * r] = l > 0.0f ? base_ : -INFINITY;
      part_ml[2 * r + 1] = l;
    }
    kp_bar(2, 256);  // the sums are read
    // columns 64 half .. hold the dimensions 64 half .. (4-bit), 16 i + 8 half .. (e4m3)
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int d = Q4 ? 4 * i : 16 * (i >> 1) + 4 * (i & 1);
      *reinterpret_cast<float4*>(s_sum + r * KP_SUM_STRIDE + (Q4 ? 64 : 8) * half + d) =
          make_float4(fmul(o[kp_vcol<KV>(d)], mul), fmul(o[kp_vcol<KV>(d + 1)], mul),
                      fmul(o[kp_vcol<KV>(d + 2)], mul), fmul(o[kp_vcol<KV>(d + 3)], mul));
    }
    kp_bar(2, 256);
    if (__all_sync(0xffffffffu, far && ok)) {
      kp_exact_rows<KV>(p, tile, head, pos, lo, hi, sk, t0, t1, s_sum, part_ml);
      __syncwarp();
    }
#pragma unroll 4
    for (int i = 0; i < 16; i++) {
      const int rr = tile * KP_ROWS + 16 * warp + i;
      if (rr >= p.rows) break;
      float* dst = p.splits == 1 ? a.out + (rr / p.group) * a.out_stride +
                                       ((int64_t)head * p.group + rr % p.group) * KV_HD
                                 : p.part + (part_row + 16 * warp + i) * KV_HD;
      reinterpret_cast<float4*>(dst)[lane] =
          reinterpret_cast<const float4*>(s_sum)[(16 * warp + i) * (KP_SUM_STRIDE / 4) + lane];
    }
  } else if (warp < 12) {
    // =========================================================== converters
    const int w = tid - 256, cw = warp - 8;
    // K: the thread's key of the tile and which part of its row; of a pair either
    // CTA widens half of the keys
    const int kk = PAIR ? 64 * rank + (w & 63) : w, kr = PAIR ? w & 63 : w, kh = PAIR ? w >> 6 : 0;
    const int kg = w >> 3, vn = w & 7;   // V: keys 8 kg .. 8 kg + 7, byte column vn
    constexpr int KR = (Q4 ? 4 : WIDE ? 2 : 8) / NB;  // 16-byte loads of a K row held a tile ahead
    uint4 kraw[KR];
    constexpr int VW = (Q4 ? 2 : 4) / NB;  // words of a key held for V
    uint32_t vraw[8][VW];
    // 4-bit: the scales of the thread's K row and V rows, and, for the tile's
    // largest, those of key w
    uint2 kd = make_uint2(0, 0), k_any = make_uint2(0, 0), v_any = make_uint2(0, 0);
    constexpr int DW = 2 / NB;
    uint32_t vd[8][DW];
    constexpr int ROW = Q4 ? 64 : KV == FLOCK_KV_FP8 ? 128 : KV == FLOCK_KV_BF16 ? 256 : 512;
    const size_t hb = Q4 ? q4_row(a.c, 0, head) * 64 : (size_t)head * ROW;
    const int64_t step = Q4 ? 64 : (int64_t)a.c.n_kv_heads * ROW;
    const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + hb;
    const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + hb;
    const uint16_t* ks = Q4 ? a.c.ks + q4_row(a.c, 0, head) * 4 : nullptr;
    const uint16_t* vs = Q4 ? a.c.vs + q4_row(a.c, 0, head) * 4 : nullptr;
    // keys outside [from, to) are zeros: what lies there cannot reach a product
    auto range = [&](int t, int& from, int& to) {
      const bool sink = t0 + t < sink_tiles;
      from = sink ? 0 : lo;
      to = sink ? sk : hi;
    };
    auto load_words = [](const uint8_t* at, bool in, auto& out) {
      constexpr int N = sizeof(out) / 4;
      if constexpr (N == 1) {
        out[0] = in ? __ldg(reinterpret_cast<const uint32_t*>(at)) : 0;
      } else if constexpr (N == 2) {
        const uint2 x = in ? __ldg(reinterpret_cast<const uint2*>(at)) : make_uint2(0, 0);
        out[0] = x.x, out[1] = x.y;
      } else {
        const uint4 x = in ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
        out[0] = x.x, out[1] = x.y, out[2] = x.z, out[3] = x.w;
      }
    };
    auto load_k = [&](int t) {
      if (WIDE) return;
      int from, to;
      range(t, from, to);
      const int key = key_of(t) + kk;
      const bool in = key >= from && key < to;
#pragma unroll
      for (int i = 0; i < KR; i++)
        kraw[i] = in ? __ldg(reinterpret_cast<const uint4*>(kb + (int64_t)key * step) + KR * kh + i)
                     : make_uint4(0, 0, 0, 0);
      if (Q4) {
        const int any = key_of(t) + w;
        const bool has = any >= from && any < to;
        kd = in ? __ldg(reinterpret_cast<const uint2*>(ks) + key) : make_uint2(0, 0);
        k_any = has ? __ldg(reinterpret_cast<const uint2*>(ks) + any) : make_uint2(0, 0);
        v_any = has ? __ldg(reinterpret_cast<const uint2*>(vs) + any) : make_uint2(0, 0);
      }
    };
    auto load_v = [&](int t) {
      if (WIDE) return;
      int from, to;
      range(t, from, to);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int key = key_of(t) + 8 * kg + i;
        const bool in = key >= from && key < to;
        load_words(vb + (int64_t)key * step + 4 * VW * (NB * vn + rank), in, vraw[i]);
        if (Q4) load_words(reinterpret_cast<const uint8_t*>(vs) + (int64_t)key * 8 + 4 * rank, in, vd[i]);
      }
    };
    // f32 and bf16 rows are too long to hold: read for the tile's largest
    // magnitude, and again (from L2) when their buffer is free.
    auto wide4 = [&](const uint8_t* base, int key, int from, int to, int d) {
      if (key < from || key >= to) return make_float4(0.f, 0.f, 0.f, 0.f);
      const uint8_t* row = base + (int64_t)key * step;
      if constexpr (KV == FLOCK_KV_BF16) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(row + 2 * d));
        const float2 lo2 = bf16x2_widen(x.x), hi2 = bf16x2_widen(x.y);
        return make_float4(lo2.x, lo2.y, hi2.x, hi2.y);
      } else {
        return __ldg(reinterpret_cast<const float4*>(row + 4 * d));
      }
    };
    int vrun = -1000;  // the largest exponent of a V tile so far, and the smallest
    int vlow = 1000;
    auto found_far = [&]() {
      if (*(volatile int*)&s_far[1]) return;
      *(volatile int*)&s_far[1] = 1;
      if (PAIR) asm volatile("fence.acq_rel.cluster;" ::: "memory");  // ahead of the arrival
    };
    // A tile's scales times 2^e lie below 2^10, so a value (below 2^13) keeps
    // its lo part; e as far as f16 can hold 2^e.
    uint32_t knorm = 0, vnorm = 0;  // f16 pairs 2^e of the K and the V tile last looked at
    auto norms = [&](int t) {
      if (!SCALED) return;
      if (WIDE) {
        int from, to;
        range(t, from, to);
        auto mag = [](uint32_t m, float4 x) {
          const uint32_t y = 0x7FFFFFFFu;
          return max(max(m, max(__float_as_uint(x.x) & y, __float_as_uint(x.y) & y)),
                     max(__float_as_uint(x.z) & y, __float_as_uint(x.w) & y));
        };
        uint32_t bk = 0, bv = 0;
#pragma unroll 8
        for (int d = 0; d < 128; d += 4) bk = mag(bk, wide4(kb, key_of(t) + w, from, to, d));
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int d = 0; d < 16; d += 4)
            bv = mag(bv, wide4(vb, key_of(t) + 8 * kg + i, from, to, 16 * vn + d));
        bk = __reduce_max_sync(0xffffffffu, bk);
        bv = __reduce_max_sync(0xffffffffu, bv);
        if (lane == 0) {
          s_dmax[0][cw] = bk;
          s_dmax[1][cw] = bv;
        }
        kp_bar(1, 128);
        uint32_t mk = 0, mv = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          mk = max(mk, s_dmax[0][i]);
          mv = max(mv, s_dmax[1][i]);
        }
        kp_bar(1, 128);  // read before the next tile's are written
        // magnitudes lie below 2^(exponent field - 126): times 2^e below 2^13
        auto exponent = [](uint32_t m) { return max(-120, min(120, 139 - (int)(m >> 23))); };
        const int ek = exponent(mk);
        // a tile of far smaller values than an earlier one need not fill f16
        vrun = max(vrun, -exponent(mv));
        if (mv) vlow = min(vlow, -exponent(mv));
        if (vrun - vlow > KR_SPREAD || mv >= 0x7F800000u) found_far();
        const int ev = -max(-exponent(mv), vrun - 30);
        knorm = __float_as_uint(pow2f(ek));
        vnorm = __float_as_uint(pow2f(ev));
        if (w == 0) {
          s_kscale[t & 3] = pow2f(-ek);
          s_vexp[t & 3] = -ev;
        }
        return;
      }
      // magnitudes order as their bits do
      auto top = [](uint2 d) {
        const uint32_t h = __vmaxu2(d.x & 0x7FFF7FFFu, d.y & 0x7FFF7FFFu);
        return __reduce_max_sync(0xffffffffu, max(h & 0xFFFFu, h >> 16));
      };
      // the smallest of the values' scales but 0 (less 1, so that 0 is the largest)
      const uint32_t small2 = __viaddmin_u16x2(v_any.x & 0x7FFF7FFFu, 0xFFFFFFFFu,
                              __vadd2(v_any.y & 0x7FFF7FFFu, 0xFFFFFFFFu));
      const uint32_t small = __reduce_min_sync(0xffffffffu, min(small2 & 0xFFFFu, small2 >> 16));
      const uint32_t bk = top(k_any), bv = top(v_any);
      if (lane == 0) {
        s_dmax[0][cw] = bk;
        s_dmax[1][cw] = bv;
        s_dmin[cw] = small;
      }
      kp_bar(1, 128);
      uint32_t mk = 0, mv = 0, mn = 0xFFFFu;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        mk = max(mk, s_dmax[0][i]);
        mv = max(mv, s_dmax[1][i]);
        mn = min(mn, s_dmin[i]);
      }
      kp_bar(1, 128);  // read before the next tile's are written
      if (mn != 0xFFFFu) {  // exponents of the largest and of the smallest scale
        auto exponent = [](uint32_t b) { return b < 0x400u ? 22 - __clz((int)b) : (int)(b >> 10); };
        vrun = max(vrun, exponent(mv));
        vlow = min(vlow, exponent(mn + 1));
      }
      if (vrun - vlow > KR_SPREAD || max(mk, mv) >= 0x7C00u) found_far();
      // magnitude below 2^(exponent field - 14)
      const int ek = min(15, 10 - min((int)(mk >> 10) - 14, 16)), ev = min(15, 10 - min((int)(mv >> 10) - 14, 16));
      // f16 pair 2^e: e in -6 .. 15
      knorm = (uint32_t)(ek + 15) * 0x04000400u;
      vnorm = (uint32_t)(ev + 15) * 0x04000400u;
      if (w == 0) {
        s_kscale[t & 3] = pow2f(-ek);
        s_vexp[t & 3] = -ev;
      }
    };
    auto put_k = [&](int t) {
      uint8_t *oh = sKh + stage(t) * OP, *ol = sKl + stage(t) * OP;
      if constexpr (WIDE) {
        int from, to;
        range(t, from, to);
        const float f = __uint_as_float(knorm);
#pragma unroll 4
        for (int i = 0; i < 16 / NB; i++) {
          const int c = 8 * kh + i;
          const float4 x = wide4(kb, key_of(t) + kk, from, to, 8 * c);
          const float4 y = wide4(kb, key_of(t) + kk, from, to, 8 * c + 4);
          uint32_t h[4], l[4];
          split_f16(fmul(x.x, f), fmul(x.y, f), h[0], l[0]);
          split_f16(fmul(x.z, f), fmul(x.w, f), h[1], l[1]);
          split_f16(fmul(y.x, f), fmul(y.y, f), h[2], l[2]);
          split_f16(fmul(y.z, f), fmul(y.w, f), h[3], l[3]);
          *reinterpret_cast<uint4*>(oh + kp_off<OR>(kr, c)) = make_uint4(h[0], h[1], h[2], h[3]);
          if (LO) *reinterpret_cast<uint4*>(ol + kp_off<OR>(kr, c)) = make_uint4(l[0], l[1], l[2], l[3]);
        }
      } else if constexpr (Q4) {
        const uint32_t d01 = hmul2_u(kd.x, knorm), d23 = hmul2_u(kd.y, knorm);
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const uint32_t d = __byte_perm(b < 2 ? d01 : d23, 0, b & 1 ? 0x3232 : 0x1010);
#pragma unroll
          for (int c = 0; c < KR; c++) {
            uint32_t v[4], h[4], l[4];
            nib_f16(word_of(kraw[c], b), v);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              h[i] = hmul2_u(v[i], d);
              l[i] = hfma2_u(v[i], d, hneg2_u(h[i]));
            }
            const uint32_t off = kp_off<OR>(kr, 4 * b + KR * kh + c);
            *reinterpret_cast<uint4*>(oh + off) = make_uint4(h[0], h[2], h[1], h[3]);
            *reinterpret_cast<uint4*>(ol + off) = make_uint4(l[0], l[2], l[1], l[3]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < KR; i++) {
          uint32_t v[8];
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = fp8_f16(word_of(kraw[i], j >> 1) >> (16 * (j & 1)));
          const int c = 2 * (KR * kh + i);
          *reinterpret_cast<uint4*>(oh + kp_off<OR>(kr, c)) = make_uint4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<uint4*>(oh + kp_off<OR>(kr, c + 1)) = make_uint4(v[4], v[5], v[6], v[7]);
        }
      }
    };
    auto put_v = [&](int t, uint32_t norm) {
      uint8_t *oh = sVh + stage(t) * OP, *ol = sVl + stage(t) * OP;
      if constexpr (WIDE) {
        int from, to;
        range(t, from, to);
        const float f = __uint_as_float(norm);
        // a thread's elements below KP_SMALL, zeros among them
        __half2 small = __float2half2_rn(0.0f);
#pragma unroll
        for (int i = 0; i < 4 / NB; i++) {  // dimensions 16 vn + 8 rank + 4 i ..
          float4 x[8];
#pragma unroll
          for (int j = 0; j < 8; j++)
            x[j] = wide4(vb, key_of(t) + 8 * kg + j, from, to, 16 * vn + 8 * rank + 4 * i);
          auto at = [&](int j, int e) {
            return fmul(e == 0 ? x[j].x : e == 1 ? x[j].y : e == 2 ? x[j].z : x[j].w, f);
          };
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              split_f16(at(2 * j, e), at(2 * j + 1, e), h[j], l[j]);
              if ((e + j) % 2 == 0)
                small = __hadd2(small, __hlt2(__habs2(as_h2(h[j])), __float2half2_rn(KP_SMALL)));
            }
            const uint32_t off = kp_off<OR>(8 * (4 * i + e) + vn, kg);
            *reinterpret_cast<uint4*>(oh + off) = make_uint4(h[0], h[1], h[2], h[3]);
            if (LO) *reinterpret_cast<uint4*>(ol + off) = make_uint4(l[0], l[1], l[2], l[3]);
          }
        }
        const int first = key_of(t) + 8 * kg;
        const int in = min(8, max(0, to - first)) - min(8, max(0, from - first));  // keys of the range
        auto warp_sum = [](int n) { return (int)__reduce_add_sync(0xffffffffu, (uint32_t)n); };
        const int n2 = (int)__low2float(small) + (int)__high2float(small) - (8 - in) * (8 / NB);
        if (warp_sum(n2) > KP_FEW / 2) {  // again, all of them but the zeros
          int n = 0;
#pragma unroll 1
          for (int i = 0; i < 32 / NB; i++) {
            const float4 x = wide4(vb, first + (i & 7), from, to,
                                   16 * vn + 8 * rank + 4 * (i >> 3));
            auto is = [&](float y) { return y != 0.0f && fabsf(fmul(y, f)) < KP_SMALL; };
            n += is(x.x) + is(x.y) + is(x.z) + is(x.w);
          }
          if (warp_sum(n) > KP_FEW) found_far();
        }
      } else if constexpr (Q4) {
#pragma unroll
        for (int b = 0; b < 4 / NB; b++) {  // blocks (2 rank +) b
          const uint32_t sel = b & 1 ? 0x7632u : 0x5410u;
          uint32_t h[4][4], l[4][4];  // [nibble][key pair]
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t v[4];
            nib_f16(__byte_perm(vraw[2 * i][b >> 1], vraw[2 * i + 1][b >> 1], sel), v);
            const uint32_t d =
                hmul2_u(__byte_perm(vd[2 * i][b >> 1], vd[2 * i + 1][b >> 1], sel), norm);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              h[e][i] = hmul2_u(v[e], d);
              l[e][i] = hfma2_u(v[e], d, hneg2_u(h[e][i]));
            }
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const uint32_t off = kp_off<OR>(32 * b + 8 * e + vn, kg);
            *reinterpret_cast<uint4*>(oh + off) = make_uint4(h[e][0], h[e][1], h[e][2], h[e][3]);
            *reinterpret_cast<uint4*>(ol + off) = make_uint4(l[e][0], l[e][1], l[e][2], l[e][3]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2 * VW; j++) {  // dimensions 16 vn (+ 8 rank) + 2 j, + 1
          uint32_t x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) x[i] = fp8_f16(vraw[i][(j >> 1) & (VW - 1)] >> (16 * (j & 1)));
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t sel = h ? 0x7632u : 0x5410u;
            *reinterpret_cast<uint4*>(oh + kp_off<OR>(8 * (2 * j + h) + vn, kg)) =
                make_uint4(__byte_perm(x[0], x[1], sel), __byte_perm(x[2], x[3], sel),
                           __byte_perm(x[4], x[5], sel), __byte_perm(x[6], x[7], sel));
          }
        }
      }
    };
    bool ok = true;
    auto wait = [&](uint64_t* b, uint32_t parity) {
      if (ok && !mbar_wait(b, parity, &s_err)) {
        fail();
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);  // put_v adds up over the warp
    };
    // K(t + 1), then V(t); raw bytes are loaded as soon as the last tile's are
    // used up.  A failed wait skips the writes but keeps the barriers' counts.
    uint32_t vnorm_t = 0;  // of the V tile in hand
    auto k_tile = [&](int t) {
      norms(t);
      if (t >= NB) wait(k_empty + stage(t - NB), phase(t - NB));
      if (ok) put_k(t);
      fence_proxy_async_smem();
      kp_arrive<PAIR>(k_full + stage(t));
      if (t + 1 < n) load_k(t + 1);
    };
    if (n > 0) {
      load_k(0);
      load_v(0);
      k_tile(0);
      vnorm_t = vnorm;
    }
    for (int t = 0; t < n; t++) {
      if (t + 1 < n) k_tile(t + 1);
      if (t >= NB) wait(v_empty + ((t - NB) & 1), ((t - NB) >> 1) & 1);
      if (ok) put_v(t, vnorm_t);
      fence_proxy_async_smem();
      kp_arrive<PAIR>(v_full + stage(t));
      if (t + 1 < n) {
        vnorm_t = vnorm;
        load_v(t + 1);
      }
    }
    __syncwarp();
    asm volatile("bar.arrive 3, 384;" ::: "memory");
  } else {
    // ============================================================= products
    if (warp == 12 && lane == 0 && rank == 0) {
      bool ok = true;
      auto wait = [&](uint64_t* b, uint32_t parity) {
        if (ok && !mbar_wait(b, parity, &s_err)) {
          fail();
          ok = false;
        }
      };
      auto scores = [&](int t) {
        if (!ok) return;
        tc_fence_after();
        const uint32_t d = tS + 128u * (t & 1), kh = smem_u32(sKh) + stage(t) * OP;
        kp_mma<PAIR>(d, tQ + 64, kh, false);  // the small products first
        if (LO) kp_mma<PAIR>(d, tQ, smem_u32(sKl) + stage(t) * OP, true);
        kp_mma<PAIR>(d, tQ, kh, true);
        kp_commit<PAIR>(k_empty + stage(t));
        kp_commit<PAIR>(s_full + (t & 1));
      };
      wait(q_full, 0);
      for (int t = 0; t < min(n, 2); t++) {
        wait(k_full + stage(t), phase(t));
        scores(t);
      }
      // O(t), then S(t + 2) over O(t)'s weights: the softmax of two tiles is under
      // way.  The operands are there long before the weights.
      for (int t = 0; t < n && ok; t++) {
        wait(v_full + stage(t), phase(t));
        if (NB == 2 && t + 2 < n) wait(k_full + stage(t), phase(t + 2));
        wait(p_full + (t & 1), (t >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t P = tS + 128u * (t & 1), vh = smem_u32(sVh) + stage(t) * OP;
        kp_mma<PAIR>(tO, P + 64, vh, t % KP_FLUSH != 0);
        if (LO) kp_mma<PAIR>(tO, P, smem_u32(sVl) + stage(t) * OP, true);
        kp_mma<PAIR>(tO, P, vh, true);
        kp_commit<PAIR>(v_empty + (t & 1));
        if (t + 2 < n) {
          if (NB == 1) wait(k_full, phase(t + 2));
          scores(t + 2);
        }
      }
      if (!ok) {  // let what was issued finish before the memory is given back
        kp_commit<PAIR>(drained);
        mbar_wait(drained, 0, &s_err, false);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) kp_cluster_sync();  // nothing of the pair's is in flight, or will be read
  if (warp == 12) {
    tc_fence_after();
    kp_free<PAIR>(tmem);
  }
}

// The rows of one tile from its splits, in order: a warp per row, four
// outputs a lane.
static __global__ void __launch_bounds__(256) k_kv_prompt_join(const KvPromptArgs p, int tiles) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), head = blockIdx.y;
  if (row >= p.rows) return;
  const int tile = row / KP_ROWS, r = row % KP_ROWS;
  const size_t first = ((size_t)head * tiles + tile) * p.splits * KP_ROWS + r;
  const float* ml = p.part + (size_t)gridDim.y * tiles * p.splits * KP_ROWS * KV_HD;
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, __ldcg(ml + (first + (size_t)s * KP_ROWS) * 2));
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.0f;
#pragma unroll 4
  for (int s = 0; s < p.splits; s++) {
    const size_t at = first + (size_t)s * KP_ROWS;
    const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part + at * KV_HD) + lane);
    const float2 b = __ldcg(reinterpret_cast<const float2*>(ml) + at);
    const float f = exp2_approx(fsub(b.x, m));
    o = make_float4(ffma(f, x.x, o.x), ffma(f, x.y, o.y), ffma(f, x.z, o.z), ffma(f, x.w, o.w));
    l = ffma(f, b.y, l);
  }
  const float inv = fdiv(1.0f, l);
  const KvAttnArgs& a = p.a;
  *reinterpret_cast<float4*>(a.out + (row / p.group) * a.out_stride +
                             ((int64_t)head * p.group + row % p.group) * KV_HD + 4 * lane) =
      make_float4(fmul(o.x, inv), fmul(o.y, inv), fmul(o.z, inv), fmul(o.w, inv));
}

}  // namespace flock
