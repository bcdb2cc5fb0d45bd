// GENERATED by kernels/gen_ffi.py from include/flock_cuda.h -- do not edit.
// The Deno.dlopen symbol table of libflock_cuda.so, the status and enum
// constants, and the byte layout of flock_layer_config.  The TypeScript
// modules beside it (lib.ts, layer.ts, model.ts, shard.ts) keep the
// reference kernels/ module surface on top of these symbols.

export const FLOCK_OK = 0;
export const FLOCK_E_ARG = -1;
export const FLOCK_E_CUDA = -2;
export const FLOCK_E_STATE = -3;
export const FLOCK_E_MISSING = -4;
export const FLOCK_E_LIMIT = -5;
export const FLOCK_E_NCCL = -6;
export const FLOCK_E_NOMEM = -7;
export const FLOCK_E_UNSUPPORTED = -8;
export const FLOCK_Q8_0 = 8;
export const FLOCK_Q4_0 = 4;
export const FLOCK_F32 = 32;
export const FLOCK_ROPE_NEOX = 0;
export const FLOCK_ROPE_NORM = 1;
export const FLOCK_ATTN_EXACT = 0;
export const FLOCK_ATTN_FAST = 1;
export const FLOCK_PREFILL_EXACT = 0;
export const FLOCK_PREFILL_TENSOR = 1;
export const FLOCK_KV_F32 = 0;
export const FLOCK_KV_BF16 = 1;
export const FLOCK_KV_FP8 = 2;
export const FLOCK_KV_Q4 = 3;
export const FLOCK_MATVEC_EXACT = 0;
export const FLOCK_MATVEC_FAST = 1;
export const FLOCK_WORKSPACE_BYTES = 8388608;
export const FLOCK_TP_NCCL = 0;
export const FLOCK_TP_PEER = 1;
export const FLOCK_DECODE_KERNELS = 0;
export const FLOCK_DECODE_PERSISTENT = 1;
export const FLOCK_DECODE_EAGER = 2;
export const FLOCK_DECODE_STREAM = 3;

export const symbols = {
  // ()
  flock_last_error: { parameters: [], result: "pointer" },
  // ()
  flock_version: { parameters: [], result: "pointer" },
  // (ordinal, out)
  flock_dev_open: { parameters: ["i32", "buffer"], result: "i32" },
  // (dev)
  flock_dev_close: { parameters: ["pointer"], result: "i32" },
  // (dev)
  flock_dev_sync: { parameters: ["pointer"], result: "i32" },
  // (dev, out)
  flock_dev_sm_count: { parameters: ["pointer", "buffer"], result: "i32" },
  // (dev)
  flock_dev_timer_start: { parameters: ["pointer"], result: "i32" },
  // (dev, ms)
  flock_dev_timer_stop: { parameters: ["pointer", "buffer"], result: "i32" },
  // (packed, rows, cols, qs_out, scales_out)
  flock_repack_q8: { parameters: ["buffer", "i64", "i64", "buffer", "buffer"], result: "i32" },
  // (packed, rows, cols, qs_out, scales_out)
  flock_repack_q4: { parameters: ["buffer", "i64", "i64", "buffer", "buffer"], result: "i32" },
  // (w, rows, cols, out)
  flock_quant_q8: { parameters: ["buffer", "i64", "i64", "buffer"], result: "i32" },
  // (w, rows, cols, out)
  flock_quant_q4: { parameters: ["buffer", "i64", "i64", "buffer"], result: "i32" },
  // (dev, dtype, packed, rows, cols, out)
  flock_tensor_from_packed: { parameters: ["pointer", "i32", "buffer", "i64", "i64", "buffer"], result: "i32" },
  // (dev, dtype, qs, scales, rows, cols, out)
  flock_tensor_from_split: { parameters: ["pointer", "i32", "buffer", "buffer", "i64", "i64", "buffer"], result: "i32" },
  // (dev, data, n, out)
  flock_tensor_from_f32: { parameters: ["pointer", "buffer", "i64", "buffer"], result: "i32" },
  // (t)
  flock_tensor_free: { parameters: ["pointer"], result: "i32" },
  // (t, out)
  flock_tensor_bytes: { parameters: ["pointer", "buffer"], result: "i32" },
  // (dev, data, bytes, out)
  flock_tensor_from_bytes: { parameters: ["pointer", "buffer", "i64", "buffer"], result: "i32" },
  // (t, offset, bytes, out)
  flock_tensor_read: { parameters: ["pointer", "i64", "i64", "buffer"], result: "i32" },
  // (dev, w, x, n_tokens, out)
  flock_op_matvec: { parameters: ["pointer", "pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (dev, w, n_tokens, iters, ms_per_call)
  flock_op_matvec_timed: { parameters: ["pointer", "pointer", "i32", "i32", "buffer"], result: "i32" },
  // (dev, w, n_tokens, iters, ms_per_call)
  flock_op_matvec_timed_cold: { parameters: ["pointer", "pointer", "i32", "i32", "buffer"], result: "i32" },
  // (dev, w, x, out)
  flock_op_matvec_fast: { parameters: ["pointer", "pointer", "buffer", "buffer"], result: "i32" },
  // (dev, w, iters, cold, ms_per_call)
  flock_op_matvec_fast_timed: { parameters: ["pointer", "pointer", "i32", "i32", "buffer"], result: "i32" },
  // (dev, w, x, M, y)
  flock_op_gemm: { parameters: ["pointer", "pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (dev, w, M, iters, ms_per_call, ms_image)
  flock_op_gemm_timed: { parameters: ["pointer", "pointer", "i32", "i32", "buffer", "buffer"], result: "i32" },
  // (dev, w, M, iters, ms_per_call, ms_image)
  flock_op_gemm_timed_cold: { parameters: ["pointer", "pointer", "i32", "i32", "buffer", "buffer"], result: "i32" },
  // (dev, n_ranks, n, wait_ms, calls, first_status)
  flock_op_peer_exchange_lone: { parameters: ["pointer", "i32", "i64", "i32", "i32", "buffer"], result: "i32" },
  // (dev, x, g, n, n_vecs, eps, out)
  flock_op_rmsnorm: { parameters: ["pointer", "buffer", "buffer", "i32", "i32", "f32", "buffer"], result: "i32" },
  // (dev, x, n_tokens, n_heads, head_dim, pos0, inv_freq, pairing, out)
  flock_op_rope: { parameters: ["pointer", "buffer", "i32", "i32", "i32", "i32", "buffer", "i32", "buffer"], result: "i32" },
  // (dev, gate, up, n, out)
  flock_op_swiglu: { parameters: ["pointer", "buffer", "buffer", "i64", "buffer"], result: "i32" },
  // (dev, a, b, n, out)
  flock_op_add: { parameters: ["pointer", "buffer", "buffer", "i64", "buffer"], result: "i32" },
  // (dev, q, k, v, n_heads, n_kv_heads, head_dim, n_keys, mode, out)
  flock_op_attention: { parameters: ["pointer", "buffer", "buffer", "buffer", "i32", "i32", "i32", "i32", "i32", "buffer"], result: "i32" },
  // (dev, q, k, v, n_heads, n_kv_heads, head_dim, n_queries, pos0, out)
  flock_op_attention_prefill: { parameters: ["pointer", "buffer", "buffer", "buffer", "i32", "i32", "i32", "i32", "i32", "buffer"], result: "i32" },
  // (dev, table, ids, n, out)
  flock_op_embed: { parameters: ["pointer", "pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (dev, x, n, index, value)
  flock_op_argmax: { parameters: ["pointer", "buffer", "i64", "buffer", "buffer"], result: "i32" },
  // (x, n, index_out, value_out, stream)
  flock_argmax_noalloc: { parameters: ["buffer", "i64", "buffer", "buffer", "buffer"], result: "i32" },
  // (p)
  flock_pointer_device: { parameters: ["buffer"], result: "i32" },
  // (dev, kv_dtype, n_kv_heads, head_dim, capacity, k, v, k_scales, v_scales, workspace, out)
  flock_kv_create: { parameters: ["pointer", "i32", "i32", "i32", "i64", "buffer", "buffer", "buffer", "buffer", "buffer", "buffer"], result: "i32" },
  // (c)
  flock_kv_free: { parameters: ["pointer"], result: "i32" },
  // (c, k, v, row_stride, pos, n, stream)
  flock_kv_append: { parameters: ["pointer", "buffer", "buffer", "i64", "i64", "i32", "buffer"], result: "i32" },
  // (c, pos, n, k, v, stream)
  flock_kv_read: { parameters: ["pointer", "i64", "i32", "buffer", "buffer", "buffer"], result: "i32" },
  // (c, q, q_stride, n_heads, n_queries, pos, window, sinks, out, out_stride, stream)
  flock_kv_attention: { parameters: ["pointer", "buffer", "i64", "i32", "i32", "i64", "i32", "i32", "buffer", "i64", "buffer"], result: "i32" },
  // (dev, target, target_stride, draft, draft_stride, ids, u, lens, n_seqs, n_drafts, vocab, temperature, tokens, accepted, workspace, stream)
  flock_verify_draft: { parameters: ["pointer", "buffer", "i64", "buffer", "i64", "buffer", "buffer", "buffer", "i32", "i32", "i64", "f64", "buffer", "buffer", "buffer", "buffer"], result: "i32" },
  // (dev, cfg, n_tensors, names, tensors, out)
  flock_layer_create: { parameters: ["pointer", "buffer", "i32", "buffer", "buffer", "buffer"], result: "i32" },
  // (layer)
  flock_layer_free: { parameters: ["pointer"], result: "i32" },
  // (layer, hidden, n_tokens)
  flock_layer_encode: { parameters: ["pointer", "buffer", "i32"], result: "i32" },
  // (layer, n_tokens, out)
  flock_layer_read_output: { parameters: ["pointer", "i32", "buffer"], result: "i32" },
  // (layer)
  flock_layer_reset: { parameters: ["pointer"], result: "i32" },
  // (layer, out)
  flock_layer_n_keys: { parameters: ["pointer", "buffer"], result: "i32" },
  // (layer, n_keys)
  flock_layer_rewind: { parameters: ["pointer", "i32"], result: "i32" },
  // (layer, window, sinks)
  flock_layer_set_window: { parameters: ["pointer", "i32", "i32"], result: "i32" },
  // (layer, k_out, v_out)
  flock_layer_read_cache: { parameters: ["pointer", "buffer", "buffer"], result: "i32" },
  // (layer, k, v, n_keys)
  flock_layer_write_cache: { parameters: ["pointer", "buffer", "buffer", "i32"], result: "i32" },
  // (layers, n_layers, x, seq, offset, reset, out)
  flock_range_forward: { parameters: ["buffer", "i32", "buffer", "i32", "i32", "i32", "buffer"], result: "i32" },
  // (dev, cfg, vocab, n_layers, layer_tensors, embd, output_norm, output, cut, out)
  flock_model_create: { parameters: ["pointer", "buffer", "i32", "i32", "buffer", "pointer", "pointer", "pointer", "i32", "buffer"], result: "i32" },
  // (dev, cfg, vocab, n_layers, layer_tensors, embd, output_norm, output_slice, comm, out)
  flock_model_create_tp: { parameters: ["pointer", "buffer", "i32", "i32", "buffer", "pointer", "pointer", "pointer", "pointer", "buffer"], result: "i32" },
  // (m, mode)
  flock_model_set_tp_exchange: { parameters: ["pointer", "i32"], result: "i32" },
  // (m, mode)
  flock_model_get_tp_exchange: { parameters: ["pointer", "buffer"], result: "i32" },
  // (m)
  flock_model_free: { parameters: ["pointer"], result: "i32" },
  // (m, ids, n, next_id)
  flock_model_step: { parameters: ["pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (m, ids, n, logits)
  flock_model_logits: { parameters: ["pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (m, ids, n, out)
  flock_model_hidden_state: { parameters: ["pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (m, ids, n, out)
  flock_model_normed_state: { parameters: ["pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (m, ids, n, out)
  flock_model_embed: { parameters: ["pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (m, ids, n, offset, out)
  flock_model_encode_partial: { parameters: ["pointer", "buffer", "i32", "i32", "buffer"], result: "i32" },
  // (m, flat, seq, next_id)
  flock_model_project_hidden: { parameters: ["pointer", "buffer", "i32", "buffer"], result: "i32" },
  // (m, prompt, n_prompt, max_tokens, eos, n_eos, out_ids, n_out)
  flock_model_generate: { parameters: ["pointer", "buffer", "i32", "i32", "buffer", "i32", "buffer", "buffer"], result: "i32" },
  // (m, n_steps, out_ids)
  flock_model_decode_device: { parameters: ["pointer", "i32", "buffer"], result: "i32" },
  // (m)
  flock_model_reset: { parameters: ["pointer"], result: "i32" },
  // (m, n_keys)
  flock_model_rewind: { parameters: ["pointer", "i32"], result: "i32" },
  // (m, out)
  flock_model_pos: { parameters: ["pointer", "buffer"], result: "i32" },
  // (m, out)
  flock_model_held: { parameters: ["pointer", "buffer"], result: "i32" },
  // (m, mode)
  flock_model_set_decode_mode: { parameters: ["pointer", "i32"], result: "i32" },
  // (m, mode)
  flock_model_get_decode_mode: { parameters: ["pointer", "buffer"], result: "i32" },
  // (m, enable)
  flock_model_trace: { parameters: ["pointer", "i32"], result: "i32" },
  // (m, out, cap, n_ctas, stride)
  flock_model_trace_read: { parameters: ["pointer", "buffer", "i64", "buffer", "buffer"], result: "i32" },
  // (m, window, sinks)
  flock_model_set_window: { parameters: ["pointer", "i32", "i32"], result: "i32" },
  // (m, ids, n, draft, u, temperature, tokens, n_tokens)
  flock_model_step_draft: { parameters: ["pointer", "buffer", "i32", "buffer", "buffer", "f64", "buffer", "buffer"], result: "i32" },
  // (m, stream)
  flock_model_wait_stream: { parameters: ["pointer", "buffer"], result: "i32" },
  // (m, id)
  flock_model_set_token: { parameters: ["pointer", "i32"], result: "i32" },
  // (m, out)
  flock_model_current_token: { parameters: ["pointer", "buffer"], result: "i32" },
  // (x, n, seq, hidden, offset, flags, out, cap, out_len)
  flock_wire_pack: { parameters: ["buffer", "i64", "u32", "u32", "u32", "u32", "buffer", "i64", "buffer"], result: "i32" },
  // (frame, len, out, cap, meta)
  flock_wire_unpack: { parameters: ["buffer", "i64", "buffer", "i64", "buffer"], result: "i32" },
  // (layers, n_layers, frame, frame_len, out, out_cap, out_len)
  flock_range_forward_wire: { parameters: ["buffer", "i32", "buffer", "i64", "buffer", "i64", "buffer"], result: "i32" },
  // (path, out)
  flock_gguf_open: { parameters: ["buffer", "buffer"], result: "i32" },
  // (g)
  flock_gguf_free: { parameters: ["pointer"], result: "i32" },
  // (g, n_tensors, data_start, version, n_layers)
  flock_gguf_info: { parameters: ["pointer", "buffer", "buffer", "buffer", "buffer"], result: "i32" },
  // (g, i, name, name_cap, dtype, rows, cols, offset, bytes)
  flock_gguf_tensor_info: { parameters: ["pointer", "i64", "buffer", "i32", "buffer", "buffer", "buffer", "buffer", "buffer"], result: "i32" },
  // (g, name, index)
  flock_gguf_find: { parameters: ["pointer", "buffer", "buffer"], result: "i32" },
  // (g, key, out)
  flock_gguf_meta_int: { parameters: ["pointer", "buffer", "buffer"], result: "i32" },
  // (g, key, out)
  flock_gguf_meta_f64: { parameters: ["pointer", "buffer", "buffer"], result: "i32" },
  // (g, key, out, cap)
  flock_gguf_meta_str: { parameters: ["pointer", "buffer", "buffer", "i32"], result: "i32" },
  // (g, first, last, gap, starts, ends, cap, n)
  flock_gguf_layer_ranges: { parameters: ["pointer", "i32", "i32", "i64", "buffer", "buffer", "i32", "buffer"], result: "i32" },
  // (dev, g, name, staging, out)
  flock_gguf_load_tensor: { parameters: ["pointer", "pointer", "buffer", "i64", "buffer"], result: "i32" },
  // (g, name, chunk, qs, scales)
  flock_gguf_split_host: { parameters: ["pointer", "buffer", "i64", "buffer", "buffer"], result: "i32" },
  // (dev, qs, scales, rows, cols, n_shards, direction, binding_limit, out)
  flock_shard_matvec_create: { parameters: ["pointer", "buffer", "buffer", "i64", "i64", "i32", "i32", "i64", "buffer"], result: "i32" },
  // (s)
  flock_shard_matvec_free: { parameters: ["pointer"], result: "i32" },
  // (s, x, y)
  flock_shard_matvec_run: { parameters: ["pointer", "buffer", "buffer"], result: "i32" },
  // (s, parts)
  flock_shard_matvec_partials: { parameters: ["pointer", "buffer"], result: "i32" },
  // (s, out)
  flock_shard_matvec_wire_bytes: { parameters: ["pointer", "buffer"], result: "i32" },
  // (dev, qs, scales, vocab, hidden, n_shards, out)
  flock_sharded_head_create: { parameters: ["pointer", "buffer", "buffer", "i64", "i64", "i32", "buffer"], result: "i32" },
  // (h)
  flock_sharded_head_free: { parameters: ["pointer"], result: "i32" },
  // (h, x, logits, token)
  flock_sharded_head_run: { parameters: ["pointer", "buffer", "buffer", "buffer"], result: "i32" },
  // (h, values, index, row_offset)
  flock_sharded_head_shard_argmax: { parameters: ["pointer", "buffer", "buffer", "buffer"], result: "i32" },
  // (id_out)
  flock_comm_unique_id: { parameters: ["buffer"], result: "i32" },
  // (dev, n_ranks, rank, id, timeout_ms, out)
  flock_comm_init: { parameters: ["pointer", "i32", "i32", "buffer", "i32", "buffer"], result: "i32" },
  // (c)
  flock_comm_free: { parameters: ["pointer"], result: "i32" },
  // (c, m, n_tokens, peer)
  flock_comm_send_hidden: { parameters: ["pointer", "pointer", "i32", "i32"], result: "i32" },
  // (c, m, n_tokens, peer)
  flock_comm_recv_hidden: { parameters: ["pointer", "pointer", "i32", "i32"], result: "i32" },
  // (m, c, ids, n, sync, next_id)
  flock_pipeline_step: { parameters: ["pointer", "pointer", "buffer", "i32", "i32", "buffer"], result: "i32" },
  // (m, start, n, out)
  flock_model_history: { parameters: ["pointer", "i32", "i32", "buffer"], result: "i32" },
  // (c, in, out, n)
  flock_comm_allreduce_f32: { parameters: ["pointer", "buffer", "buffer", "i64"], result: "i32" },
  // (c, in, out, bytes_per_rank)
  flock_comm_allgather_bytes: { parameters: ["pointer", "buffer", "buffer", "i64"], result: "i32" },
} as const;

export type FlockSymbols = typeof symbols;
export type FlockLib = Deno.DynamicLibrary<FlockSymbols>["symbols"];

/** sizeof(flock_layer_config) and each field's byte offset (C layout). */
export const LAYER_CONFIG_BYTES = 64;
export const LAYER_CONFIG_FIELDS = {
  hidden: { offset: 0, type: "int32_t" },
  n_heads: { offset: 4, type: "int32_t" },
  n_kv_heads: { offset: 8, type: "int32_t" },
  head_dim: { offset: 12, type: "int32_t" },
  ffn: { offset: 16, type: "int32_t" },
  eps: { offset: 20, type: "float" },
  rope_base: { offset: 24, type: "double" },
  max_keys: { offset: 32, type: "int32_t" },
  max_prefill: { offset: 36, type: "int32_t" },
  rope_pairing: { offset: 40, type: "int32_t" },
  attention: { offset: 44, type: "int32_t" },
  prefill: { offset: 48, type: "int32_t" },
  kv_dtype: { offset: 52, type: "int32_t" },
  matvec: { offset: 56, type: "int32_t" },
} as const;

export type LayerConfigC = { [K in keyof typeof LAYER_CONFIG_FIELDS]: number };

/** Pack a flock_layer_config into the bytes the C ABI reads. */
export function packLayerConfig(c: LayerConfigC): Uint8Array {
  const buf = new Uint8Array(LAYER_CONFIG_BYTES);
  const dv = new DataView(buf.buffer);
  dv.setInt32(0, c.hidden, true);
  dv.setInt32(4, c.n_heads, true);
  dv.setInt32(8, c.n_kv_heads, true);
  dv.setInt32(12, c.head_dim, true);
  dv.setInt32(16, c.ffn, true);
  dv.setFloat32(20, c.eps, true);
  dv.setFloat64(24, c.rope_base, true);
  dv.setInt32(32, c.max_keys, true);
  dv.setInt32(36, c.max_prefill, true);
  dv.setInt32(40, c.rope_pairing, true);
  dv.setInt32(44, c.attention, true);
  dv.setInt32(48, c.prefill, true);
  dv.setInt32(52, c.kv_dtype, true);
  dv.setInt32(56, c.matvec, true);
  return buf;
}

let opened: Deno.DynamicLibrary<FlockSymbols> | null = null;

/** dlopen libflock_cuda.so once (FLOCK_LIB overrides the path).  There is
 *  no fallback: a missing library is an error, not a CPU path. */
export function flock(path?: string): FlockLib {
  if (!opened) {
    const p = path ?? Deno.env.get("FLOCK_LIB") ??
      new URL("../flock_b200/libflock_cuda.so", import.meta.url).pathname;
    opened = Deno.dlopen(p, symbols);
  }
  return opened.symbols;
}

/** flock_last_error() as a string. */
export function lastError(): string {
  const p = flock().flock_last_error();
  return p ? new Deno.UnsafePointerView(p).getCString() : "";
}

/** The reference throws `Error`s with named messages; a non-zero status
 *  becomes the same kind of throw, carrying flock_last_error() and the code. */
export class FlockError extends Error {
  constructor(readonly code: number, message: string) {
    super(message || `flock error ${code}`);
  }
}

export function check(rc: number): void {
  if (rc !== FLOCK_OK) throw new FlockError(rc, lastError());
}

/** One out-slot for a handle (flock_X** parameters). */
export function handleSlot(): BigUint64Array {
  return new BigUint64Array(1);
}

export function slotPointer(slot: BigUint64Array): Deno.PointerValue {
  return Deno.UnsafePointer.create(slot[0]);
}

/** A NUL-terminated UTF-8 string for a `const char*` parameter. */
export function cstr(s: string): Uint8Array {
  return new TextEncoder().encode(s + "\0");
}

/** An array of handles for a `T* const*` parameter. */
export function pointerArray(ps: Deno.PointerValue[]): BigUint64Array {
  return BigUint64Array.from(ps.map((p) => BigInt(Deno.UnsafePointer.value(p))));
}
