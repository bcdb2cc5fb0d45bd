// Verification of drafted tokens against the target's distribution with given
// uniform numbers (flock_verify_draft).
//
// For one sequence with drafts x_0 .. x_{n-1}, target logits t_0 .. t_n and
// draft logits s_0 .. s_{n-1}: p_i = softmax(t_i / T), q_i = softmax(s_i / T).
// Draft i is kept iff u_i q_i(x_i) < p_i(x_i) (no draft logits: q_i is 1 at
// x_i).  The token after the kept ones is drawn at u_n by inverse CDF from
// max(p_r - q_r, 0) at the first refused r, or from p_n when all were kept:
// that rule gives the target's own distribution whatever the draft's is.
//
// Two launches.  k_verify_stats reads every row once (the HBM bound: (2 n + 1)
// V floats a sequence) and leaves each chunk's maximum and sum of exponentials.
// k_verify_pick, one cluster per sequence, decides r from them and draws.
//
// Precision.  A keep decision compares two numbers known to ~1e-7 with a
// uniform number: f32 exponentials are enough.  The draw is another matter: it
// places u W among V borders, and a relative error e of the running sum moves
// about min(V, 1/e) borders past a given u with probability ~V e.  For the
// drawn row alone exponentials, their sums and the running sum are therefore
// f64 (V e ~ 1e-11), shared out over the cluster's CTAs (64 f64 lanes an SM).
#pragma once
#include <cooperative_groups.h>

#include "common.cuh"

namespace flock {

constexpr int VS_THREADS = 256;
constexpr int VP_THREADS = 512;
constexpr int VP_MAX_CLUSTER = 16;
constexpr int VERIFY_MAX_DRAFTS = 512;

struct VerifyArgs {
  const float* target;    // row (s, i) at (s (n + 1) + i) target_stride, i = 0 .. n
  const float* draft;     // row (s, i) at (s n + i) draft_stride, or null
  int64_t target_stride, draft_stride;
  const int32_t* ids;     // [n_seqs][n]
  const float* u;         // [n_seqs][n + 1]
  const int32_t* lens;    // [n_seqs] drafts of each sequence, or null: n
  int32_t* tokens;        // [n_seqs][n + 1]
  int32_t* accepted;      // [n_seqs]
  int n_seqs, n, vocab;
  double inv_t;           // 1 / T; 0 for greedy
  // partials of (row, chunk): rows are a sequence's n + 1 target rows, then
  // its n draft rows
  float* part_m;          // greedy: unused
  float* part_s;
  unsigned long long* part_key;  // greedy: ordered maximum and its index
  int chunks, chunk_len;  // chunk_len a multiple of 4
  int vec;                // rows are 16-byte aligned
};

FLOCK_DEV int verify_len(const VerifyArgs& a, int seq) {
  if (!a.lens) return a.n;
  const int l = a.lens[seq];
  return l < 0 ? 0 : l > a.n ? a.n : l;
}
FLOCK_DEV const float* verify_row(const VerifyArgs& a, int seq, int row) {
  return row <= a.n ? a.target + ((int64_t)seq * (a.n + 1) + row) * a.target_stride
                    : a.draft + ((int64_t)seq * a.n + (row - a.n - 1)) * a.draft_stride;
}

// Orders (value, lowest index first) by one unsigned comparison; 0 for a NaN,
// below every number.
FLOCK_DEV unsigned long long verify_key(float x, int index) {
  if (x != x) return 0;
  uint32_t b = __float_as_uint(fadd(x, 0.0f));  // -0 and 0 are one value
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)b << 32 | (uint32_t)~index;
}

FLOCK_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// CTA (chunk, row of a sequence): this chunk's maximum m and sum of
// e^((x - m) / T).  -inf logits are probability 0; a NaN or +inf makes the sum
// NaN, a row of -inf leaves it 0: a row without a distribution.
template <bool GREEDY>
static __global__ void __launch_bounds__(VS_THREADS) k_verify_stats(const VerifyArgs a) {
  pdl_launch_dependents();
  const int rows = GREEDY || !a.draft ? a.n + 1 : 2 * a.n + 1;
  const int seq = blockIdx.y / rows, row = blockIdx.y % rows;
  const int len = verify_len(a, seq);
  if (row <= a.n ? row > len : row - a.n - 1 >= len) return;
  const float* x = verify_row(a, seq, row);
  const int c0 = blockIdx.x * a.chunk_len, c1 = min(a.vocab, c0 + a.chunk_len);
  const float k = (float)(a.inv_t * 1.4426950408889634);
  float m = -INFINITY, s = 0.0f;
  unsigned long long key = 0;
  constexpr int B = 4;  // 16-byte loads of a pass; the next pass's are in flight meanwhile
  float v[4 * B], next[4 * B];
  auto load = [&](int i0) {
#pragma unroll
    for (int b = 0; b < B; b++) {
      const int i = i0 + 4 * b * VS_THREADS;
      if (a.vec && i + 4 <= c1) {
        const uint4 w = ldg_stream(x + i);
        next[4 * b] = __uint_as_float(w.x);
        next[4 * b + 1] = __uint_as_float(w.y);
        next[4 * b + 2] = __uint_as_float(w.z);
        next[4 * b + 3] = __uint_as_float(w.w);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) next[4 * b + j] = i + j < c1 ? __ldg(x + i + j) : -INFINITY;
      }
    }
  };
  load(c0 + 4 * threadIdx.x);
  for (int i0 = c0 + 4 * threadIdx.x; i0 < c1; i0 += 4 * B * VS_THREADS) {
#pragma unroll
    for (int j = 0; j < 4 * B; j++) v[j] = next[j];
    if (i0 + 4 * B * VS_THREADS < c1) load(i0 + 4 * B * VS_THREADS);
    if (GREEDY) {
#pragma unroll
      for (int j = 0; j < 4 * B; j++) {
        const int i = i0 + 4 * (j / 4) * VS_THREADS + j % 4;
        if (i < c1) {
          const unsigned long long t = verify_key(v[j], i);
          key = t > key ? t : key;
        }
      }
    } else {
      float mn = m;
#pragma unroll
      for (int j = 0; j < 4 * B; j++) mn = fmaxf(mn, v[j]);
      const float base = mn == -INFINITY ? 0.0f : mn;
      s = fmul(s, ex2(fmul(fsub(m, base), k)));
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4 * B; j++)
        part[j & 3] = fadd(part[j & 3], ex2(fmul(fsub(v[j], base), k)));
      s = fadd(s, fadd(fadd(part[0], part[1]), fadd(part[2], part[3])));
      m = mn;
    }
  }
  // join the threads: lanes, then warps
  __shared__ float sm[VS_THREADS / 32], ss[VS_THREADS / 32];
  __shared__ unsigned long long sk[VS_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t at = (size_t)blockIdx.y * a.chunks + blockIdx.x;
  if (GREEDY) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const unsigned long long t = __shfl_xor_sync(0xffffffffu, key, d);
      key = t > key ? t : key;
    }
    if (lane == 0) sk[warp] = key;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < VS_THREADS / 32; w++) key = sk[w] > key ? sk[w] : key;
      a.part_key[at] = key;
    }
    return;
  }
  auto join = [&](float om, float os) {
    const float mn = fmaxf(m, om), base = mn == -INFINITY ? 0.0f : mn;
    s = fadd(fmul(s, ex2(fmul(fsub(m, base), k))), fmul(os, ex2(fmul(fsub(om, base), k))));
    m = mn;
  };
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    join(__shfl_xor_sync(0xffffffffu, m, d), __shfl_xor_sync(0xffffffffu, s, d));
  if (lane == 0) {
    sm[warp] = m;
    ss[warp] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < VS_THREADS / 32; w++) join(sm[w], ss[w]);
    a.part_m[at] = m;
    a.part_s[at] = s;
  }
}

// The maximum and f64 sum of one row from its chunks' partials, by one warp.
FLOCK_DEV void verify_join(const VerifyArgs& a, size_t row, float& m, double& s) {
  const int lane = threadIdx.x & 31;
  const float* pm = a.part_m + row * a.chunks;
  const float* ps = a.part_s + row * a.chunks;
  // at most 64 chunks: two a lane, all loads in flight together
  float cm[2], cs[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int c = lane + 32 * h;
    cm[h] = c < a.chunks ? pm[c] : -INFINITY;
    cs[h] = c < a.chunks ? ps[c] : 0.0f;
  }
  m = fmaxf(cm[0], cm[1]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  s = 0.0;
#pragma unroll
  for (int h = 0; h < 2; h++)  // a chunk of -inf has the sum 0
    s += cm[h] == -INFINITY ? (double)cs[h]
                            : exp(((double)cm[h] - (double)m) * a.inv_t) * (double)cs[h];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
}

// e^((x - m) / T) for x <= m in f64, c = 16 / (T ln 2): e^z = 2^(n / 16) 2^(r /
// 16), n the integer nearest 16 z / ln 2 and |r| <= 1/2, 2^(r / 16) by the
// Taylor polynomial of e^(r ln 2 / 16) of degree 6 (remainder below 5e-16 of
// it), 2^(j / 16) from a table.  Relative error below 1e-15 for z > -40,
// growing as |z| 2e-17.  Logits below `lowest` (m - 700 T rounded up: at a small T
// it is m itself, which counts; above -inf at a large one) give 0.
__constant__ static const double k_pow16[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0};
struct VerifyRow {
  double m, c;
  float lowest;
};
FLOCK_DEV VerifyRow verify_row_of(float m, double inv_t) {
  return {(double)m, inv_t * 0x1.71547652b82fep+4, __double2float_ru((double)m - 700.0 / inv_t)};
}
FLOCK_DEV double verify_exp(float x, const VerifyRow& row, const double* pow16) {
  const double magic = 6755399441055744.0;  // 1.5 2^52: adding it rounds to an integer
  const double d = (double)x - row.m;
  const double t = fma(d, row.c, magic);
  const double r = fma(d, row.c, magic - t);
  double p = 0x1.430912f86c787p-37;  // (ln 2 / 16)^k / k!
  p = fma(p, r, 0x1.5d87fe78a6731p-30);
  p = fma(p, r, 0x1.3b2ab6fba4e77p-23);
  p = fma(p, r, 0x1.c6b08d704a0c0p-17);
  p = fma(p, r, 0x1.ebfbdff82c58fp-11);
  p = fma(p, r, 0x1.62e42fefa39efp-5);
  p = fma(p, r, 1.0);
  const int k = __double2loint(t);  // n, two's complement
  const double e = p * pow16[k & 15];
  return x >= row.lowest
             ? __hiloint2double(__double2hiint(e) + ((k >> 4) << 20), __double2loint(e)) : 0.0;
}

// The sum of one value per thread over the block, f64, the same in every
// thread; red: VP_THREADS / 32 values.
FLOCK_DEV double verify_sum(double v, double* red) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < VP_THREADS / 32; w++) v += red[w];
  return v;
}

// One cluster per sequence.  Every warp of it takes a contiguous `span` of the
// vocabulary, so that a sum per warp, added up in order, is the running sum at
// the warps' borders; the warp whose span holds u W then looks inside it.
// KEEP: a lane's exponentials of both rows stay in registers between the
// passes (spans up to 128 KEPT: V = 151936 in a cluster of 16); longer
// vocabularies compute them again.
constexpr int VP_KEPT = 5;
template <bool KEEP>
static __global__ void __launch_bounds__(VP_THREADS) k_verify_pick(const VerifyArgs a, int span) {
  namespace cg = cooperative_groups;
  constexpr int WARPS = VP_THREADS / 32;
  __shared__ int s_first;
  __shared__ float s_rm[2 * VERIFY_MAX_DRAFTS + 1];   // each row's maximum and sum
  __shared__ double s_rs[2 * VERIFY_MAX_DRAFTS + 1];
  __shared__ double s_red[WARPS], s_pow16[16];
  __shared__ double s_sum[2], s_total[2];  // read by the cluster's other CTAs
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), nr = (int)cluster.num_blocks();
  const int seq = blockIdx.x / nr, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  if (t < 16) s_pow16[t] = k_pow16[t];
  pdl_wait();  // the partials
  const int len = verify_len(a, seq);
  const bool sampled = a.draft != nullptr;
  const int rows = sampled ? 2 * a.n + 1 : a.n + 1;
  const size_t row0 = (size_t)seq * rows;
  const int32_t* ids = a.ids + (size_t)seq * a.n;
  const float* u = a.u + (size_t)seq * (a.n + 1);

  // every CTA decides the first refused draft for itself
  if (t == 0) s_first = len;
  for (int row = warp; row < rows; row += WARPS) {
    if (row <= a.n ? row > len : row - a.n - 1 >= len) continue;  // not read: no partials
    float m;
    double s;
    verify_join(a, row0 + row, m, s);
    if (lane == 0) {
      s_rm[row] = m;
      s_rs[row] = s;
    }
  }
  __syncthreads();
  for (int i = t; i < len; i += VP_THREADS) {
    const int x = ids[i];
    bool keep = false;
    if (x >= 0 && x < a.vocab) {
      auto prob = [&](int row) {
        return exp(((double)verify_row(a, seq, row)[x] - (double)s_rm[row]) * a.inv_t) / s_rs[row];
      };
      const double p = prob(i), q = sampled ? prob(a.n + 1 + i) : 1.0;
      keep = (double)u[i] * q < p;  // false for a row without a distribution
    }
    if (!keep) atomicMin(&s_first, i);
  }
  __syncthreads();
  const int r = s_first;
  const bool refused = r < len;
  const bool residual = refused && sampled;
  // one-hot draft: its token cannot be drawn again
  const int skip = refused && !sampled ? ids[r] : -1;
  const VerifyRow mp = verify_row_of(s_rm[r], a.inv_t);
  const VerifyRow mq = verify_row_of(residual ? s_rm[a.n + 1 + r] : 0.0f, a.inv_t);
  auto summable = [&](int row) { return s_rs[row] > 0.0 && s_rs[row] < (double)INFINITY; };
  const bool has = summable(r) && (!residual || summable(a.n + 1 + r));
  if (rank == 0) {
    int32_t* out = a.tokens + (size_t)seq * (a.n + 1);
    // token r too: the warp that draws it writes it behind the cluster's barriers
    for (int i = t; i <= a.n; i += VP_THREADS) out[i] = i < r ? ids[i] : -1;
    if (t == 0) a.accepted[seq] = r;
  }
  if (!has) return;  // the whole cluster agrees

  const float* xp = verify_row(a, seq, r);
  const float* xq = residual ? verify_row(a, seq, a.n + 1 + r) : nullptr;
  const int64_t from = ((int64_t)rank * WARPS + warp) * span;
  const int v0 = (int)(from < a.vocab ? from : a.vocab), v1 = (int)(from + span < a.vocab ? from + span : a.vocab);
  // four neighbouring logits from i on, -inf past the span
  auto four = [&](const float* x, int i, float (&v)[4]) {
    if (a.vec && i + 4 <= v1) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(x + i));
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = i + j < v1 ? __ldg(x + i + j) : -INFINITY;
    }
  };
  // f(index, exponential, draft's exponential) over the span, a lane four at a
  // time; the first of two passes computes them (KEEP) or both do
  double ke[KEEP ? VP_KEPT : 1][4], kf[KEEP ? VP_KEPT : 1][4];
  auto compute = [&](const float (&x)[4], const float (&y)[4], double (&e)[4], double (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      e[j] = verify_exp(x[j], mp, s_pow16);
      f[j] = residual ? verify_exp(y[j], mq, s_pow16) : 0.0;
    }
  };
  auto each = [&](bool first, auto f) {
    if constexpr (KEEP) {
      if (first) {
        float x[VP_KEPT][4], y[VP_KEPT][4];
#pragma unroll
        for (int b = 0; b < VP_KEPT; b++) {
          four(xp, v0 + 4 * lane + 128 * b, x[b]);
          if (residual) four(xq, v0 + 4 * lane + 128 * b, y[b]);
        }
#pragma unroll
        for (int b = 0; b < VP_KEPT; b++) compute(x[b], y[b], ke[b], kf[b]);
      }
#pragma unroll
      for (int b = 0; b < VP_KEPT; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) f(v0 + 4 * lane + 128 * b + j, ke[b][j], kf[b][j]);
    } else {
      for (int i = v0 + 4 * lane; i < v1; i += 128) {
        float x[4], y[4];
        four(xp, i, x);
        if (residual) four(xq, i, y);
        compute(x, y, ke[0], kf[0]);
#pragma unroll
        for (int j = 0; j < 4; j++) f(i + j, ke[0][j], kf[0][j]);
      }
    }
  };
  double ip = 1.0, iq = 1.0;
  if (residual) {  // the rows' f64 sums
    double a0 = 0.0, a1 = 0.0;
    each(true, [&](int, double e, double f) {
      a0 += e;
      a1 += f;
    });
    a0 = verify_sum(a0, s_red);
    a1 = verify_sum(a1, s_red);
    if (t == 0) {
      s_sum[0] = a0;
      s_sum[1] = a1;
    }
    cluster.sync();
    // a lane per CTA: the remote loads (0.2 us each) in flight together
    double sp = 0.0, sq = 0.0;
    if (lane < nr) {
      const double* o = cluster.map_shared_rank(s_sum, lane);
      sp = o[0];
      sq = o[1];
    }
#pragma unroll
    for (int d = VP_MAX_CLUSTER / 2; d > 0; d >>= 1) {
      sp += __shfl_xor_sync(0xffffffffu, sp, d);
      sq += __shfl_xor_sync(0xffffffffu, sq, d);
    }
    sp = __shfl_sync(0xffffffffu, sp, 0);
    sq = __shfl_sync(0xffffffffu, sq, 0);
    ip = 1.0 / sp;
    iq = 1.0 / sq;
  }
  // all: the weights are the target's own (nothing was left of the residual)
  auto weight = [&](int i, double e, double f, bool all) {
    return all ? e : residual ? fmax(e * ip - f * iq, 0.0) : i == skip ? 0.0 : e;
  };
  double before = 0.0, end = 0.0, w = 0.0;
  bool all = !refused;
  for (int turn = 0; turn < 2; turn++) {
    double mine = 0.0;
    each(turn == 0 && !residual, [&](int i, double e, double f) { mine += weight(i, e, f, all); });
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    __syncthreads();
    if (lane == 0) s_red[warp] = mine;
    __syncthreads();
    if (t == 0) {
      double sum = 0.0;
      for (int i = 0; i < WARPS; i++) sum += s_red[i];
      s_total[turn] = sum;
    }
    cluster.sync();
    // running sums over the CTAs, a lane each, the same in every CTA: one after the
    // other in fours, and so the fours, which never fall and stay as they are over a
    // CTA without weight (a scan by doubling adds neighbours in different orders)
    const double total = lane < nr ? *cluster.map_shared_rank(s_total + turn, lane) : 0.0;
    double run = 0.0, fours = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const double o = __shfl_sync(0xffffffffu, total, (lane & ~3) + i);
      run += i <= (lane & 3) ? o : 0.0;
    }
#pragma unroll
    for (int i = 0; i + 1 < VP_MAX_CLUSTER / 4; i++) {
      const double o = __shfl_sync(0xffffffffu, run, 4 * i + 3);
      fours += i < lane >> 2 ? o : 0.0;
    }
    run += fours;
    before = rank == 0 ? 0.0 : __shfl_sync(0xffffffffu, run, rank - 1);
    end = __shfl_sync(0xffffffffu, run, rank);
    w = __shfl_sync(0xffffffffu, run, nr - 1);
    if (w > 0.0 || all) break;  // the whole cluster agrees
    all = true;
  }
  // no CTA leaves while another may read its shared memory
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  // This warp's [before, end) of the running sum: its CTA's, cut at the warps
  // before it, and none without weight.  The CTA's end and the warps' sums round
  // apart: cut at that end, and the last warp of weight reaches it, the parts cover
  // [0, w) once, so one warp draws, and it has a token to draw.
  const double cta_end = end;
  const uint32_t weighted = __ballot_sync(0xffffffffu, lane < WARPS && s_red[lane % WARPS] > 0.0);
  for (int i = 0; i < warp; i++) before += s_red[i];
  end = weighted >> warp > 1 ? fmin(before + s_red[warp], cta_end) : cta_end;
  const bool some = weighted >> warp & 1;
  double goal = fmax((double)u[a.n], 0.0) * w;  // fmax: 0 for a NaN
  if (!(goal < w)) goal = w * 0.9999999999999999;
  if (some && before <= goal && goal < end) {
    int pick = -1, last = v0;
    double c = before;
    auto look = [&](int i, const double (&e)[4], const double (&f)[4]) {
      double v[4], sum = 0.0;
      int top = -1;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        v[j] = weight(i + j, e[j], f[j], all);
        sum += v[j];
        if (v[j] > 0.0) top = i + j;
      }
      double run = sum;  // inclusive over the lanes
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += o;
      }
      // of the lanes with weight: the others' sums may pass it by their rounding
      const uint32_t over = __ballot_sync(0xffffffffu, top >= 0 && c + run > goal);
      if (over && pick < 0) {
        int found = top;  // rounding may leave it to the lane's last weight
        double upto = c + (run - sum) + sum;
#pragma unroll
        for (int j = 3; j >= 0; j--) {
          if (v[j] > 0.0 && upto > goal) found = i + j;
          upto -= v[j];
        }
        pick = __shfl_sync(0xffffffffu, found, __ffs(over) - 1);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      last = top >= 0 ? top : last;
      c += __shfl_sync(0xffffffffu, run, 31);
    };
    if constexpr (KEEP) {
#pragma unroll
      for (int b = 0; b < VP_KEPT; b++)
        if (pick < 0) look(v0 + 4 * lane + 128 * b, ke[b], kf[b]);
    } else {
      for (int i0 = v0; i0 < v1 && pick < 0; i0 += 128) {
        float x[4], y[4];
        four(xp, i0 + 4 * lane, x);
        if (residual) four(xq, i0 + 4 * lane, y);
        compute(x, y, ke[0], kf[0]);
        look(i0 + 4 * lane, ke[0], kf[0]);
      }
    }
    if (lane == 0) a.tokens[(size_t)seq * (a.n + 1) + r] = pick >= 0 ? pick : last;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Greedy: drafts are kept while they equal the target's argmax (the lowest
// index among the maxima), and the argmax at the first difference follows.
static __global__ void __launch_bounds__(128) k_verify_greedy(const VerifyArgs a) {
  __shared__ int s_first;
  pdl_wait();
  const int seq = blockIdx.x, t = threadIdx.x, len = verify_len(a, seq);
  const int32_t* ids = a.ids + (size_t)seq * a.n;
  auto top = [&](int row) {
    const unsigned long long* p = a.part_key + ((size_t)seq * (a.n + 1) + row) * a.chunks;
    unsigned long long key = 0;
    for (int c = 0; c < a.chunks; c++) key = p[c] > key ? p[c] : key;
    return key ? (int)~(uint32_t)key : -1;
  };
  if (t == 0) s_first = len;
  __syncthreads();
  for (int i = t; i < len; i += 128)
    if (top(i) != ids[i] || ids[i] < 0) atomicMin(&s_first, i);
  __syncthreads();
  const int r = s_first;
  int32_t* out = a.tokens + (size_t)seq * (a.n + 1);
  for (int i = t; i <= a.n; i += 128) out[i] = i < r ? ids[i] : i == r ? top(r) : -1;
  if (t == 0) a.accepted[seq] = r;
}

}  // namespace flock
