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
  constexpr int B = 4;  // 16-byte loads in flight per thread
  for (int i0 = c0 + 4 * threadIdx.x; i0 < c1; i0 += 4 * B * VS_THREADS) {
    float v[4 * B];
#pragma unroll
    for (int b = 0; b < B; b++) {
      const int i = i0 + 4 * b * VS_THREADS;
      if (a.vec && i + 4 <= c1) {
        const uint4 w = ldg_stream(x + i);
        v[4 * b] = __uint_as_float(w.x);
        v[4 * b + 1] = __uint_as_float(w.y);
        v[4 * b + 2] = __uint_as_float(w.z);
        v[4 * b + 3] = __uint_as_float(w.w);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[4 * b + j] = i + j < c1 ? __ldg(x + i + j) : -INFINITY;
      }
    }
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
#pragma unroll
      for (int j = 0; j < 4 * B; j++) s = fadd(s, ex2(fmul(fsub(v[j], base), k)));
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
  m = -INFINITY;
  for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, pm[c]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  s = 0.0;
  for (int c = lane; c < a.chunks; c += 32)  // a chunk of -inf has the sum 0
    s += pm[c] == -INFINITY ? (double)ps[c]
                            : exp(((double)pm[c] - (double)m) * a.inv_t) * (double)ps[c];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
}

// Inclusive sums of one value per thread over the block (VP_THREADS), f64;
// returns the thread's exclusive sum and the block's total.
FLOCK_DEV double verify_scan(double v, double* red, double& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double s = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
  for (int w = 0; w < VP_THREADS / 32; w++) {
    if (w == warp) before = total;
    total += red[w];
  }
  // the exclusive sum of a thread is the inclusive sum of the one before it
  const double prev = __shfl_up_sync(0xffffffffu, s, 1);
  return lane == 0 ? before : before + prev;
}

// One cluster per sequence; CTA `rank` holds vocabulary [rank L, (rank + 1) L),
// thread t of it the contiguous elements [t E, (t + 1) E) of that.  CACHED: the
// f64 exponentials of both rows stay in shared memory between the passes (V /
// cluster * 16 bytes); a vocabulary too long for that computes them again.
template <bool CACHED>
static __global__ void __launch_bounds__(VP_THREADS) k_verify_pick(const VerifyArgs a, int L) {
  namespace cg = cooperative_groups;
  extern __shared__ double vp_smem[];
  __shared__ int s_first;
  __shared__ float s_rm[2 * VERIFY_MAX_DRAFTS + 1];   // each row's maximum and sum
  __shared__ double s_rs[2 * VERIFY_MAX_DRAFTS + 1];
  __shared__ double s_red[VP_THREADS / 32];
  __shared__ double s_sum[2], s_total;  // read by the cluster's other CTAs
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), nr = (int)cluster.num_blocks();
  const int seq = blockIdx.x / nr, t = threadIdx.x;
  pdl_wait();  // the partials
  const int len = verify_len(a, seq);
  const bool sampled = a.draft != nullptr;
  const int rows = sampled ? 2 * a.n + 1 : a.n + 1;
  const size_t row0 = (size_t)seq * rows;
  const int32_t* ids = a.ids + (size_t)seq * a.n;
  const float* u = a.u + (size_t)seq * (a.n + 1);

  // every CTA decides the first refused draft for itself
  if (t == 0) s_first = len;
  for (int row = t >> 5; row < rows; row += VP_THREADS / 32) {
    if (row <= a.n ? row > len : row - a.n - 1 >= len) continue;  // not read: no partials
    float m;
    double s;
    verify_join(a, row0 + row, m, s);
    if ((t & 31) == 0) {
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
  const double mp = s_rm[r], mq = residual ? s_rm[a.n + 1 + r] : 0.0f;
  auto summable = [&](int row) { return s_rs[row] > 0.0 && s_rs[row] < (double)INFINITY; };
  const bool has = summable(r) && (!residual || summable(a.n + 1 + r));
  if (rank == 0) {
    int32_t* out = a.tokens + (size_t)seq * (a.n + 1);
    for (int i = t; i <= a.n; i += VP_THREADS)
      if (i != r || !has) out[i] = i < r ? ids[i] : -1;
    if (t == 0) a.accepted[seq] = r;
  }
  if (!has) return;  // the whole cluster agrees

  const float* xp = verify_row(a, seq, r);
  const float* xq = residual ? verify_row(a, seq, a.n + 1 + r) : nullptr;
  const int v0 = rank * L, v1 = min(a.vocab, v0 + L);
  double* ep = vp_smem;
  double* eq = vp_smem + L;
  auto expo = [&](const float* x, int i, double m) {
    return exp(((double)__ldg(x + i) - m) * a.inv_t);
  };
  // the rows' f64 sums over the cluster (only a residual needs them)
  double sp = 1.0, sq = 1.0;
  if (CACHED || residual) {
    double a0 = 0.0, a1 = 0.0;
    for (int i = v0 + t; i < v1; i += VP_THREADS) {
      const double e = expo(xp, i, mp);
      a0 += e;
      if (CACHED) ep[i - v0] = e;
      if (residual) {
        const double f = expo(xq, i, mq);
        a1 += f;
        if (CACHED) eq[i - v0] = f;
      }
    }
    if (residual) {
      double t0, t1;
      verify_scan(a0, s_red, t0);
      verify_scan(a1, s_red, t1);
      if (t == 0) {
        s_sum[0] = t0;
        s_sum[1] = t1;
      }
      cluster.sync();
      sp = sq = 0.0;
      for (int c = 0; c < nr; c++) {
        const double* o = cluster.map_shared_rank(s_sum, c);
        sp += o[0];
        sq += o[1];
      }
    } else {
      __syncthreads();
    }
  }
  const double ip = 1.0 / sp, iq = 1.0 / sq;
  const int E = (L + VP_THREADS - 1) / VP_THREADS;
  const int j0 = min(v1, v0 + t * E), j1 = min(v1, j0 + E);
  // all: the weights are the target's own (nothing was left of the residual)
  auto weight = [&](int i, bool all) {
    const double e = CACHED ? ep[i - v0] : expo(xp, i, mp);
    if (all) return e;
    if (residual) return fmax(e * ip - (CACHED ? eq[i - v0] : expo(xq, i, mq)) * iq, 0.0);
    return i == skip ? 0.0 : e;
  };
  bool all = !refused;
  double mine, before, total, w = 0.0;
  while (true) {
    mine = 0.0;
    for (int i = j0; i < j1; i++) mine += weight(i, all);
    before = verify_scan(mine, s_red, total);
    if (t == 0) s_total = total;
    cluster.sync();
    double base = 0.0;
    w = 0.0;
    for (int c = 0; c < nr; c++) {
      if (c == rank) base = w;
      w += *cluster.map_shared_rank(&s_total, c);
    }
    before += base;
    cluster.sync();  // s_total is read before it is written again, and before any CTA leaves
    if (w > 0.0 || all) break;
    all = true;
  }
  // The first index whose running sum passes u W.  The threads' half-open
  // ranges [before, end) cut [0, W) without gaps, `end` being the next
  // thread's `before`, so one thread draws.
  double goal = (double)u[a.n] * w;
  if (!(goal < w)) goal = w * 0.9999999999999999;
  double end = __shfl_down_sync(0xffffffffu, before, 1);
  const int lane = t & 31, warp = t >> 5;
  __syncthreads();
  if (lane == 0) s_red[warp] = before;
  if (t == 0) s_sum[0] = before;  // this CTA's first running sum
  cluster.sync();
  if (lane == 31)
    end = warp + 1 < VP_THREADS / 32 ? s_red[warp + 1]
          : rank + 1 < nr            ? cluster.map_shared_rank(s_sum, rank + 1)[0]
                                     : w;
  if (before <= goal && goal < end) {
    double c = before;
    int pick = min(j0, a.vocab - 1);
    for (int i = j0; i < j1; i++) {
      const double x = weight(i, all);
      c += x;
      if (x > 0.0) pick = i;
      if (c > goal) break;
    }
    a.tokens[(size_t)seq * (a.n + 1) + r] = pick;
  }
  cluster.sync();  // s_sum is read before its CTA leaves
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
