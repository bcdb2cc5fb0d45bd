// Draft verification (include/flock_cuda.h flock_verify_draft).
#include <cuda_runtime.h>

#include "flock_internal.h"
#include "verify.cuh"

using namespace flock;

namespace {

constexpr int64_t VERIFY_MAX_VOCAB = 4194304;
constexpr int64_t VERIFY_MAX_PARTIALS = FLOCK_WORKSPACE_BYTES / 8;

struct OnDevice {
  int before = -1, want;
  explicit OnDevice(int ordinal) : want(ordinal) {}
  int enter() {
    FLOCK_CK(cudaGetDevice(&before));
    if (before != want) FLOCK_CK(cudaSetDevice(want));
    return FLOCK_OK;
  }
  ~OnDevice() {
    if (before >= 0 && before != want) cudaSetDevice(before);
  }
};

template <bool KEEP>
int launch_pick(cudaStream_t st, const VerifyArgs& a, int cluster, int span) {
  auto k = k_verify_pick<KEEP>;
  if (cluster > 8) {  // past the portable size: asked for once per device
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    FLOCK_CK(cudaGetDevice(&dev));
    if (!(allowed.load() >> (dev & 63) & 1)) {
      FLOCK_CK(cudaFuncSetAttribute((const void*)k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      allowed.fetch_or((uint64_t)1 << (dev & 63));
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n_seqs * cluster);
  cfg.blockDim = dim3(VP_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FLOCK_CK(cudaLaunchKernelEx(&cfg, k, a, span));
  return FLOCK_OK;
}

}  // namespace

extern "C" {

int flock_verify_draft(flock_dev* dev, const float* target, int64_t target_stride,
                       const float* draft, int64_t draft_stride, const int32_t* ids,
                       const float* u, const int32_t* lens, int n_seqs, int n_drafts,
                       int64_t vocab, double temperature, int32_t* tokens, int32_t* accepted,
                       void* workspace, void* stream) {
  if (!dev || n_seqs < 0 || n_drafts < 0 || vocab < 1) {
    set_error("verify_draft: dev must not be NULL, n_seqs and n_drafts not negative, vocab >= 1");
    return FLOCK_E_ARG;
  }
  if (n_drafts > VERIFY_MAX_DRAFTS || vocab > VERIFY_MAX_VOCAB) {
    set_error("verify_draft: n_drafts %d must be at most %d and vocab %lld at most %lld", n_drafts,
              VERIFY_MAX_DRAFTS, (long long)vocab, (long long)VERIFY_MAX_VOCAB);
    return FLOCK_E_LIMIT;
  }
  // log2(e) / temperature has to be a normal f32 (k_verify_stats)
  if (temperature != 0.0 && !(temperature >= 1e-38 && temperature <= 1e38)) {
    set_error("verify_draft: temperature %g must be 0 (greedy) or in 1e-38 .. 1e38", temperature);
    return FLOCK_E_ARG;
  }
  if (n_seqs == 0) return FLOCK_OK;
  const bool greedy = temperature == 0.0;
  if (!target || (n_drafts && !ids) || (!greedy && !u) || !tokens || !accepted || !workspace) {
    set_error("verify_draft: target, ids, u, tokens, accepted and workspace must not be NULL");
    return FLOCK_E_ARG;
  }
  // floats and ints at 4 bytes, the workspace's 8-byte keys and more at 16: a
  // misaligned address would fault the GPU
  auto off = [](const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0; };
  if (off(workspace, 16) || off(target, 4) || off(draft, 4) || off(ids, 4) || off(u, 4) ||
      off(lens, 4) || off(tokens, 4) || off(accepted, 4)) {
    set_error("verify_draft: the workspace must be 16-byte aligned, every other address 4-byte "
              "aligned");
    return FLOCK_E_ARG;
  }
  if (target_stride == 0) target_stride = vocab;
  if (draft_stride == 0) draft_stride = vocab;
  if (target_stride < vocab || draft_stride < vocab) {
    set_error("verify_draft: row strides %lld and %lld must be at least vocab %lld",
              (long long)target_stride, (long long)draft_stride, (long long)vocab);
    return FLOCK_E_ARG;
  }
  if (greedy || n_drafts == 0) draft = nullptr;
  const int64_t rows = (int64_t)n_seqs * (draft ? 2 * n_drafts + 1 : n_drafts + 1);
  if (rows > 65535) {
    set_error("verify_draft: %lld rows of logits in one call, at most 65535", (long long)rows);
    return FLOCK_E_LIMIT;
  }
  OnDevice on(dev->ordinal);
  FLOCK_TRY(on.enter());
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  VerifyArgs a = {};
  a.target = target;
  a.draft = draft;
  a.target_stride = target_stride;
  a.draft_stride = draft_stride;
  a.ids = ids;
  a.u = u;
  a.lens = lens;
  a.tokens = tokens;
  a.accepted = accepted;
  a.n_seqs = n_seqs;
  a.n = n_drafts;
  a.vocab = (int)vocab;
  a.inv_t = greedy ? 0.0 : 1.0 / temperature;
  // chunks of a row: enough CTAs to fill the GPU's SMs about four times over,
  // none under one pass of a CTA's loads
  const int64_t pass = 16 * VS_THREADS;
  int64_t chunks = (4 * (int64_t)dev->sm_count + rows - 1) / rows;
  const int64_t passes = (vocab + pass - 1) / pass;
  chunks = chunks < 1 ? 1 : chunks > passes ? passes : chunks;
  if (chunks > 64) chunks = 64;
  if (chunks * rows > VERIFY_MAX_PARTIALS) chunks = VERIFY_MAX_PARTIALS / rows;
  a.chunk_len = (int)(((vocab + chunks - 1) / chunks + 3) / 4 * 4);
  a.chunks = (int)((vocab + a.chunk_len - 1) / a.chunk_len);
  a.part_m = static_cast<float*>(workspace);
  a.part_s = a.part_m + (size_t)rows * a.chunks;
  a.part_key = static_cast<unsigned long long*>(workspace);
  a.vec = ((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) & 15) == 0 &&
          target_stride % 4 == 0 && (!draft || draft_stride % 4 == 0);
  const dim3 grid((unsigned)a.chunks, (unsigned)rows);
  if (greedy) {
    k_verify_stats<true><<<grid, VS_THREADS, 0, st>>>(a);
    FLOCK_CK(cudaGetLastError());
    FLOCK_CK(launch_ex(st, k_verify_greedy, dim3((unsigned)n_seqs), dim3(128), 0, true, a));
    return FLOCK_OK;
  }
  k_verify_stats<false><<<grid, VS_THREADS, 0, st>>>(a);
  FLOCK_CK(cudaGetLastError());
  // CTAs per sequence: about a thousand tokens each, as many as a cluster may
  // have.  More sequences than such clusters find room (seven of 16 CTAs that
  // fill an SM each) do better in clusters of eight whose CTAs share SMs and
  // compute the exponentials twice (32 sequences: 90 us against 101).
  const bool many = (int64_t)n_seqs * VP_MAX_CLUSTER > dev->sm_count;
  const int most = many ? VP_MAX_CLUSTER / 2 : VP_MAX_CLUSTER;
  int cluster = 1;
  while (cluster < most && (int64_t)cluster * 1024 < vocab) cluster *= 2;
  // each warp's span of the vocabulary, in whole groups of four
  const int64_t warps = (int64_t)cluster * (VP_THREADS / 32);
  const int span = (int)(((vocab + warps - 1) / warps + 3) / 4 * 4);
  return span <= 128 * VP_KEPT && !many ? launch_pick<true>(st, a, cluster, span)
                               : launch_pick<false>(st, a, cluster, span);
}

}  // extern "C"
