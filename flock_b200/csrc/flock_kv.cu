// Caches in caller-owned memory: append, read back and attention with a
// sliding window and sinks (include/flock_cuda.h flock_kv_*).
#include <cuda_runtime.h>

#include <new>

#include "arg_checks.h"
#include "flock_internal.h"
#include "kv.cuh"
#include "kv_layer.h"
#include "kv_prompt.cuh"
#include "kv_rows.cuh"

using namespace flock;

struct flock_kv {
  flock_dev* dev = nullptr;
  int kv_dtype = 0;
  KvView view{};
  uint8_t* workspace = nullptr;
  DBuf own_k, own_v, own_ks, own_vs, own_ws;  // allocated here when the caller gave none
};

namespace {

constexpr int64_t KV_MAX_CAPACITY = (int64_t)1 << 30;

// The handle's device made current for the call, the caller's restored after.
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A pointer the caller says is device memory of `dev`: asked of the runtime
// once, when a handle is made.
int check_device_pointer(const flock_dev* dev, const void* p, const char* what) {
  cudaPointerAttributes at = {};
  const cudaError_t e = cudaPointerGetAttributes(&at, p);
  if (e != cudaSuccess || at.type == cudaMemoryTypeUnregistered || at.type == cudaMemoryTypeHost) {
    cudaGetLastError();
    set_error("%s is not device memory", what);
    return FLOCK_E_ARG;
  }
  if (at.device != dev->ordinal) {
    set_error("%s is on device %d, the handle on device %d", what, at.device, dev->ordinal);
    return FLOCK_E_ARG;
  }
  if (!aligned16(p)) {
    set_error("%s is not 16-byte aligned", what);
    return FLOCK_E_ARG;
  }
  return FLOCK_OK;
}

int check_range(const flock_kv* c, const char* who, int64_t pos, int n) {
  if (!range_inside(pos, n, c->view.capacity)) {
    set_error("%s: %d positions from %lld on are not inside a cache of %lld keys", who, n,
              (long long)pos, (long long)c->view.capacity);
    return FLOCK_E_STATE;
  }
  return FLOCK_OK;
}

dim3 row_grid(const flock_kv* c, int n) {  // 8 tokens a CTA, a warp each
  return dim3((unsigned)((n + 7) / 8), (unsigned)c->view.n_kv_heads);
}

size_t plane_bytes(int kv_dtype, int n_kv_heads, int64_t capacity) {
  const size_t values = (size_t)capacity * n_kv_heads * KV_HD;
  return kv_dtype == FLOCK_KV_Q4     ? values / 2
         : kv_dtype == FLOCK_KV_FP8  ? values
         : kv_dtype == FLOCK_KV_BF16 ? values * 2
                                     : values * 4;
}

template <typename F>
int by_dtype(int kv_dtype, F f) {
  switch (kv_dtype) {
    case FLOCK_KV_Q4: return f(std::integral_constant<int, FLOCK_KV_Q4>());
    case FLOCK_KV_FP8: return f(std::integral_constant<int, FLOCK_KV_FP8>());
    case FLOCK_KV_BF16: return f(std::integral_constant<int, FLOCK_KV_BF16>());
    default: return f(std::integral_constant<int, FLOCK_KV_F32>());
  }
}

// Keys that some query of the call sees, sinks included (with the position on
// the device and a window: of the bound).
int64_t visible_keys(const KvAttnArgs& a) {
  const int64_t lo = a.window && a.pos + 1 > a.window ? a.pos + 1 - a.window : 0;
  return a.pos + a.n_queries - lo + (a.sinks < lo ? a.sinks : lo);
}

// k_kv_rows or k_kv_prompt.  The first's time grows with rows times keys, the
// second's starts at 12 to 25 us and grows with the keys of 128 rows.  us, first
// against second, 8 kv heads, rows @ keys:
//   4-bit  32 @ 32000 60 / 69   48 @ 32000 76 / 69    48 @ 8169 28 / 33    64 @ 8169 36 / 33
//   e4m3   24 @ 32000 43 / 51   32 @ 32000 59 / 51    48 @ 8169 26 / 27    64 @ 8169 35 / 27
//   bf16   32 @ 32000 139 / 204 48 @ 32000 265 / 205  128 @ 1000 25 / 30   48 @ 8169 74 / 59
//   f32    16 @ 32000 211 / 243 24 @ 32000 275 / 244  32 @ 1000 22 / 33    48 @ 1000 33 / 33
template <int KV>
bool few_rows(int64_t rows, int64_t keys, int64_t n_kv_heads) {
  constexpr int always = KV == FLOCK_KV_F32 ? 16 : KV == FLOCK_KV_FP8 ? 24 : 32;
  constexpr int64_t work = KV == FLOCK_KV_F32 ? 300000 : KV == FLOCK_KV_BF16 ? 1024000 : 3200000;
  return rows <= always || (rows <= 128 && rows * keys * n_kv_heads <= work);
}

// A few query rows per kv head: k_kv_rows.
template <int KV, int NT>
int launch_rows(int sm_count, uint8_t* workspace, const KvAttnArgs& a, cudaStream_t st) {
  using L = KrLayout<KV, NT>;
  constexpr int RT = L::RT;
  KvRowsArgs p = {};
  p.a = a;
  p.group = a.n_heads / a.c.n_kv_heads;
  p.rows = a.n_queries * p.group;
  const int tiles = (p.rows + RT - 1) / RT;
  const int64_t items = (int64_t)tiles * a.c.n_kv_heads;
  // one CTA per SM; with the position on the device the kernel decides, at most
  // the splits of the bound (sink and window groups, two of them cut)
  const int64_t lo = a.window && !a.ctl && a.pos + 1 > a.window ? a.pos + 1 - a.window : 0;
  int64_t keys = a.pos + a.n_queries - lo + (a.sinks < lo ? a.sinks : lo);
  if (a.ctl && a.window && keys > (int64_t)a.window + a.n_queries + a.sinks)
    keys = (int64_t)a.window + a.n_queries + a.sinks;
  const int64_t room = items < KR_MAX_ITEMS ? sm_count / items : 1;
  const int splits = kr_splits(keys / KR_GROUP + 3, L::WARPS, room);
  p.count = reinterpret_cast<uint32_t*>(workspace);
  p.part = reinterpret_cast<float*>(workspace + KR_PART_OFFSET);
  FLOCK_TRY(kernel_setup((const void*)k_kv_rows<KV, NT>, (int)L::SMEM));
  FLOCK_CK(launch_ex(st, k_kv_rows<KV, NT>,
                     dim3((unsigned)splits, (unsigned)tiles, (unsigned)a.c.n_kv_heads),
                     dim3(L::THREADS), L::SMEM, true, p));
  return FLOCK_OK;
}

// Many query rows: k_kv_prompt on the tensor cores, 128 rows a CTA, alone or in pairs.
template <int KV, bool PAIR>
int launch_prompt(uint8_t* workspace, const KvAttnArgs& a, cudaStream_t st) {
  KvPromptArgs p = {};
  p.a = a;
  p.group = a.n_heads / a.c.n_kv_heads;
  p.rows = a.n_queries * p.group;
  int tiles = (p.rows + KP_ROWS - 1) / KP_ROWS;
  if (PAIR) tiles = (tiles + 1) & ~1;
  const int64_t items = (int64_t)tiles * a.c.n_kv_heads;
  // key splits of a tile, at least two key tiles each, as many for every tile as the
  // workspace's 125 partial outputs allow: none from 63 (tile, kv head) items on
  const int64_t want = (visible_keys(a) + 2 * KP_KEYS - 1) / (2 * KP_KEYS);
  constexpr int64_t most = (FLOCK_WORKSPACE_BYTES - KR_PART_OFFSET) / (KP_ROWS * (KV_HD + 2) * 4);
  const int64_t room = most / items;
  p.splits = (int)(want < room ? want : room);
  if (p.splits < 1) p.splits = 1;
  p.part = reinterpret_cast<float*>(workspace + KR_PART_OFFSET);
  FLOCK_TRY(kernel_setup((const void*)k_kv_prompt<KV, PAIR>, (int)KP_SMEM<KV>));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)tiles, (unsigned)p.splits, (unsigned)a.c.n_kv_heads);
  cfg.blockDim = dim3(KP_THREADS);
  cfg.dynamicSmemBytes = KP_SMEM<KV>;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {PAIR ? 2u : 1u, 1u, 1u};
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  FLOCK_CK(cudaLaunchKernelEx(&cfg, k_kv_prompt<KV, PAIR>, p));
  if (p.splits > 1)
    FLOCK_CK(launch_ex(st, k_kv_prompt_join,
                       dim3((unsigned)((p.rows + 7) / 8), (unsigned)a.c.n_kv_heads), dim3(256), 0,
                       true, p, tiles));
  return FLOCK_OK;
}

}  // namespace

int flock::kv_attention_enqueue(int sm_count, int kv_dtype, const KvAttnArgs& a,
                                uint8_t* workspace, cudaStream_t st) {
  const int64_t rows = (int64_t)a.n_queries * (a.n_heads / a.c.n_kv_heads);
  return by_dtype(kv_dtype, [&](auto kv) -> int {
    constexpr int KV = decltype(kv)::value;
    if (!few_rows<KV>(rows, visible_keys(a), a.c.n_kv_heads)) {
      // Two tiles as a pair of CTAs where the operands are widened at a cost: 1024
      // queries at 3000 keys of 16 / 8 heads 100 us against 120 (4-bit), 228
      // against 292 (bf16); e4m3 gains 1 to 3% and loses 15% in a window.  A tile
      // without a partner costs one: three tiles at 4000 keys 46 us against 38,
      // thirteen in a window of 1500 keys 54 against 59.
      const int64_t tiles = (rows + KP_ROWS - 1) / KP_ROWS;
      if constexpr (KV != FLOCK_KV_FP8)
        if (tiles % 2 == 0 || tiles > 8) return launch_prompt<KV, true>(workspace, a, st);
      return launch_prompt<KV, false>(workspace, a, st);
    }
    if constexpr (KV == FLOCK_KV_Q4 || KV == FLOCK_KV_FP8)
      if (rows <= 4) return launch_rows<KV, 1>(sm_count, workspace, a, st);  // one column tile
    return launch_rows<KV, 2>(sm_count, workspace, a, st);
  });
}

extern "C" {

int flock_pointer_device(const void* p) {
  cudaPointerAttributes at = {};
  if (!p || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return at.type == cudaMemoryTypeDevice ? at.device : -1;
}

int flock_kv_create(flock_dev* dev, int kv_dtype, int n_kv_heads, int head_dim, int64_t capacity,
                    void* k, void* v, void* k_scales, void* v_scales, void* workspace,
                    flock_kv** out) {
  if (!dev || !out) {
    set_error("kv_create: dev and out must not be NULL");
    return FLOCK_E_ARG;
  }
  if (kv_dtype != FLOCK_KV_F32 && kv_dtype != FLOCK_KV_BF16 && kv_dtype != FLOCK_KV_FP8 &&
      kv_dtype != FLOCK_KV_Q4) {
    set_error("kv_create: kv_dtype %d is not FLOCK_KV_F32, _BF16, _FP8 or _Q4", kv_dtype);
    return FLOCK_E_ARG;
  }
  if (head_dim != KV_HD) {
    set_error("kv_create: head_dim %d: the kernels are built for head_dim 128", head_dim);
    return FLOCK_E_UNSUPPORTED;
  }
  if (n_kv_heads < 1 || n_kv_heads > 65535 || capacity < 1 || capacity > KV_MAX_CAPACITY) {
    set_error("kv_create: n_kv_heads %d must be in 1..65535 and capacity %lld in 1..%lld",
              n_kv_heads, (long long)capacity, (long long)KV_MAX_CAPACITY);
    return FLOCK_E_ARG;
  }
  const bool q4 = kv_dtype == FLOCK_KV_Q4;
  if (q4 && capacity % 16) {
    set_error("kv_create: a 4-bit cache's capacity %lld must be a multiple of 16",
              (long long)capacity);
    return FLOCK_E_ARG;
  }
  if ((!k) != (!v) || (k && q4 && (!k_scales || !v_scales)) ||
      ((k_scales || v_scales) && (!q4 || !k))) {
    set_error("kv_create: give both planes or none, and both scale planes with a 4-bit cache's "
              "planes only");
    return FLOCK_E_ARG;
  }
  OnDevice on(dev->ordinal);
  FLOCK_TRY(on.enter());
  flock_kv* c = new (std::nothrow) flock_kv();
  if (!c) {
    set_error("kv_create: out of host memory");
    return FLOCK_E_NOMEM;
  }
  auto fill = [&]() -> int {
    const size_t bytes = plane_bytes(kv_dtype, n_kv_heads, capacity);
    const size_t sbytes = (size_t)capacity * n_kv_heads * 4 * sizeof(uint16_t);
    if (k) {
      FLOCK_TRY(check_device_pointer(dev, k, "kv_create: k"));
      FLOCK_TRY(check_device_pointer(dev, v, "kv_create: v"));
      if (q4) {
        FLOCK_TRY(check_device_pointer(dev, k_scales, "kv_create: k_scales"));
        FLOCK_TRY(check_device_pointer(dev, v_scales, "kv_create: v_scales"));
      }
    } else {
      FLOCK_TRY(c->own_k.alloc(bytes));
      FLOCK_TRY(c->own_v.alloc(bytes));
      FLOCK_CK(cudaMemset(c->own_k.p, 0, bytes));
      FLOCK_CK(cudaMemset(c->own_v.p, 0, bytes));
      k = c->own_k.p;
      v = c->own_v.p;
      if (q4) {
        FLOCK_TRY(c->own_ks.alloc(sbytes));
        FLOCK_TRY(c->own_vs.alloc(sbytes));
        FLOCK_CK(cudaMemset(c->own_ks.p, 0, sbytes));
        FLOCK_CK(cudaMemset(c->own_vs.p, 0, sbytes));
        k_scales = c->own_ks.p;
        v_scales = c->own_vs.p;
      }
    }
    if (workspace) {
      FLOCK_TRY(check_device_pointer(dev, workspace, "kv_create: workspace"));
    } else {
      FLOCK_TRY(c->own_ws.alloc(FLOCK_WORKSPACE_BYTES));
      FLOCK_CK(cudaMemset(c->own_ws.p, 0, FLOCK_WORKSPACE_BYTES));
      workspace = c->own_ws.p;
    }
    if (c->own_k.p || c->own_ws.p) FLOCK_CK(cudaStreamSynchronize(nullptr));
    return FLOCK_OK;
  };
  const int rc = fill();
  if (rc != FLOCK_OK) {
    delete c;
    return rc;
  }
  c->dev = dev_retain(dev);
  c->kv_dtype = kv_dtype;
  c->view.k = k;
  c->view.v = v;
  c->view.ks = static_cast<uint16_t*>(k_scales);
  c->view.vs = static_cast<uint16_t*>(v_scales);
  c->view.capacity = capacity;
  c->view.n_kv_heads = n_kv_heads;
  c->workspace = static_cast<uint8_t*>(workspace);
  *out = c;
  return FLOCK_OK;
}

int flock_kv_free(flock_kv* c) {
  if (!c) return FLOCK_OK;
  flock_dev* dev = c->dev;
  {
    OnDevice on(dev->ordinal);
    FLOCK_TRY(on.enter());
    delete c;
  }
  dev_release(dev);
  return FLOCK_OK;
}

int flock_kv_append(flock_kv* c, const float* k, const float* v, int64_t row_stride, int64_t pos,
                    int n, void* stream) {
  if (!c || (n > 0 && (!k || !v))) {
    set_error("kv_append: the cache, k and v must not be NULL");
    return FLOCK_E_ARG;
  }
  FLOCK_TRY(check_range(c, "kv_append", pos, n));
  const int64_t row = (int64_t)c->view.n_kv_heads * KV_HD;
  if (row_stride == 0) row_stride = row;
  if (row_stride < row || row_stride % 4 || !aligned16(k) || !aligned16(v)) {
    set_error("kv_append: row_stride %lld must be a multiple of 4, at least %lld, and k and v "
              "16-byte aligned", (long long)row_stride, (long long)row);
    return FLOCK_E_ARG;
  }
  if (n == 0) return FLOCK_OK;
  OnDevice on(c->dev->ordinal);
  FLOCK_TRY(on.enter());
  const dim3 grid = row_grid(c, n);
  return by_dtype(c->kv_dtype, [&](auto kv) -> int {
    FLOCK_CK(launch_ex(static_cast<cudaStream_t>(stream), k_kv_append<decltype(kv)::value>,
                       grid, dim3(256), 0, true, c->view, k, v, row_stride, pos, n));
    return FLOCK_OK;
  });
}

int flock_kv_read(flock_kv* c, int64_t pos, int n, float* k, float* v, void* stream) {
  if (!c || (n > 0 && (!k || !v)) || !aligned16(k) || !aligned16(v)) {
    set_error("kv_read: the cache, k and v must not be NULL, k and v 16-byte aligned");
    return FLOCK_E_ARG;
  }
  FLOCK_TRY(check_range(c, "kv_read", pos, n));
  if (n == 0) return FLOCK_OK;
  OnDevice on(c->dev->ordinal);
  FLOCK_TRY(on.enter());
  const dim3 grid = row_grid(c, n);
  return by_dtype(c->kv_dtype, [&](auto kv) -> int {
    FLOCK_CK(launch_ex(static_cast<cudaStream_t>(stream), k_kv_read<decltype(kv)::value>,
                       grid, dim3(256), 0, true, c->view, pos, n, k, v));
    return FLOCK_OK;
  });
}

int flock_kv_attention(flock_kv* c, const float* q, int64_t q_stride, int n_heads, int n_queries,
                       int64_t pos, int window, int sinks, float* out, int64_t out_stride,
                       void* stream) {
  if (!c || (n_queries > 0 && (!q || !out))) {
    set_error("kv_attention: the cache, q and out must not be NULL");
    return FLOCK_E_ARG;
  }
  if (n_heads < 1 || n_heads % c->view.n_kv_heads) {
    set_error("kv_attention: n_heads %d must be a multiple of n_kv_heads %d", n_heads,
              c->view.n_kv_heads);
    return FLOCK_E_ARG;
  }
  if (window < 0 || sinks < 0) {
    set_error("kv_attention: window %d and sinks %d must not be negative (window 0: no window)",
              window, sinks);
    return FLOCK_E_ARG;
  }
  FLOCK_TRY(check_range(c, "kv_attention", pos, n_queries));
  const int64_t row = (int64_t)n_heads * KV_HD;
  if (q_stride == 0) q_stride = row;
  if (out_stride == 0) out_stride = row;
  if (q_stride < row || q_stride % 4 || out_stride < row || out_stride % 4 || !aligned16(q) ||
      !aligned16(out)) {
    set_error("kv_attention: q_stride %lld and out_stride %lld must be multiples of 4, at least "
              "%lld, and q and out 16-byte aligned", (long long)q_stride, (long long)out_stride,
              (long long)row);
    return FLOCK_E_ARG;
  }
  if ((int64_t)n_queries * (n_heads / c->view.n_kv_heads) > (int64_t)1 << 30) {
    set_error("kv_attention: %d queries of %d heads over %d kv heads are more than 2^30 rows",
              n_queries, n_heads, c->view.n_kv_heads);
    return FLOCK_E_LIMIT;
  }
  if (n_queries == 0) return FLOCK_OK;
  OnDevice on(c->dev->ordinal);
  FLOCK_TRY(on.enter());
  KvAttnArgs a = {};
  a.c = c->view;
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.pos = pos;
  a.n_queries = n_queries;
  a.n_heads = n_heads;
  a.window = window;
  a.sinks = sinks;
  return kv_attention_enqueue(c->dev->sm_count, c->kv_dtype, a, c->workspace,
                              static_cast<cudaStream_t>(stream));
}

}  // extern "C"
