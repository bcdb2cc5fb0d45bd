// What the layers need of flock_kv.cu: attention over a cache view on a stream.
#pragma once
#include <cuda_runtime.h>

#include "kv.cuh"

namespace flock {
// Causal attention of a.n_queries queries (KvAttnArgs), the kernel chosen by the
// rows per kv head; workspace: FLOCK_WORKSPACE_BYTES, zero-filled once.
int kv_attention_enqueue(int sm_count, int kv_dtype, const KvAttnArgs& a, uint8_t* workspace,
                         cudaStream_t st);
}  // namespace flock
