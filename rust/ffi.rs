// ffi.rs: the raw binding of libsgk.so (include/sgk.h), generated by rust/gen_ffi.py.
// Do not edit by hand: change the header and run the generator.
//
// Every prototype of the header is declared here, in the header's order. The safe layer
// of the crate (FullAttentionMetalState, BlockAwarePrefixCache, ...) keeps its signatures
// and calls these through `check`, which turns a status code into the crate's InferError.
#![allow(non_camel_case_types, dead_code, clippy::too_many_arguments)]

use crate::error::InferError;

// ---- status codes and constants ----
pub const SGK_OK: i32 = 0;
pub const SGK_ERR_DIMENSION: i32 = 1;
pub const SGK_ERR_CONFIG: i32 = 2;
pub const SGK_ERR_BACKEND: i32 = 3;
pub const SGK_ERR_MEMORY_GUARD: i32 = 4;
pub const SGK_ERR_SHAPE: i32 = 5;
pub const SGK_ERR_TIMEOUT: i32 = 6;
pub const SGK_KV_F32: i32 = 0;
pub const SGK_KV_BF16: i32 = 1;
pub const SGK_KV_U8G32: i32 = 2;
pub const SGK_KV_U4G32: i32 = 3;
pub const SGK_PAGE_TOKENS: usize = 16;
pub const SGK_NOALLOC_SCRATCH_BYTES: usize = 4 << 20;
pub const SGK_NOALLOC_MAX_Q_DIM: usize = 16384;

// ---- opaque handles (only ever used behind a pointer) ----
#[repr(C)]
pub struct SgkState {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkPool {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkSeq {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkKv {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkBatch {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkStep {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkLinstate {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkPrefix {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkBudget {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkExchange {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkTokenWindow {
    _private: [u8; 0],
}
#[repr(C)]
pub struct SgkDprefix {
    _private: [u8; 0],
}

// ---- plain structs passed by pointer ----
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct SgkRope {
    pub rope_dims: i32,
    pub frequency_dim: i32,
    pub theta: f32,
    pub position_scale: f32,
    pub eps: f32,
    pub interleaved: i32,
}
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct SgkAffineWeight {
    pub d_packed: *const u32,
    pub d_scales: *const u16,
    pub d_biases: *const u16,
    pub bits: i32,
    pub group_size: i32,
}
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct SgkTokenIo {
    pub d_table: *const std::ffi::c_void,
    pub table_dtype: i32,
    pub vocab: i64,
    pub hidden: i32,
    pub embedding_scale: f32,
    pub recast_bf16: i32,
    pub d_x: *mut f32,
    pub d_lm_weight: *const std::ffi::c_void,
    pub lm_weight_dtype: i32,
    pub d_final: *const f32,
    pub table_affine: *const SgkAffineWeight,
    pub lm_affine: *const SgkAffineWeight,
}
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct SgkLinearShape {
    pub num_key_heads: i32,
    pub num_value_heads: i32,
    pub key_head_dim: i32,
    pub value_head_dim: i32,
}

#[link(name = "sgk")]
extern "C" {
    pub fn sgk_last_error() -> *const std::os::raw::c_char;
    pub fn sgk_version() -> *const std::os::raw::c_char;
    pub fn sgk_state_create(device: i32, out: *mut *mut SgkState) -> i32;
    pub fn sgk_state_destroy(state: *mut SgkState);
    pub fn sgk_state_stream(state: *mut SgkState) -> *mut std::ffi::c_void;
    pub fn sgk_state_sync(state: *mut SgkState) -> i32;
    pub fn sgk_state_device_status(state: *mut SgkState, status_out: *mut i32) -> i32;
    pub fn sgk_state_set_concurrent_streams(state: *mut SgkState, enabled: i32) -> i32;
    pub fn sgk_state_launches(state: *const SgkState) -> i64;
    pub fn sgk_state_chain_begin(state: *mut SgkState, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_state_chain_end(state: *mut SgkState) -> i32;
    pub fn sgk_state_selftest_wait_timeout(state: *mut SgkState) -> i32;
    pub fn sgk_pool_create(state: *mut SgkState, layers: i32, kv_heads: i32, head_dim: i32, dtype: i32, page_tokens: i32, num_pages: i64, max_seqs: i32, max_seq_tokens: i64, out: *mut *mut SgkPool) -> i32;
    pub fn sgk_pool_destroy(pool: *mut SgkPool);
    pub fn sgk_pool_num_pages(pool: *const SgkPool) -> i64;
    pub fn sgk_pool_free_pages(pool: *const SgkPool) -> i64;
    pub fn sgk_pool_page_bytes(pool: *const SgkPool) -> i64;
    pub fn sgk_pool_used_bytes(pool: *const SgkPool) -> i64;
    pub fn sgk_pool_shuffle_free_list(pool: *mut SgkPool, seed: u64) -> i32;
    pub fn sgk_pool_page_refcount(pool: *const SgkPool, page: i64, out: *mut i32) -> i32;
    pub fn sgk_pool_set_scrub_on_free(pool: *mut SgkPool, enabled: i32) -> i32;
    pub fn sgk_seq_create(pool: *mut SgkPool, capacity_tokens: i64, out: *mut *mut SgkSeq) -> i32;
    pub fn sgk_seq_destroy(seq: *mut SgkSeq);
    pub fn sgk_seq_reserve(seq: *mut SgkSeq, tokens: i64) -> i32;
    pub fn sgk_seq_block_table(seq: *const SgkSeq, pages_out: *mut i32, cap: i64, n_out: *mut i64) -> i32;
    pub fn sgk_seq_reset(seq: *mut SgkSeq, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_seq_release_before(seq: *mut SgkSeq, row: i64) -> i32;
    pub fn sgk_seq_release_between(seq: *mut SgkSeq, first_row: i64, row: i64) -> i32;
    pub fn sgk_seq_layer(seq: *mut SgkSeq, layer: i32, q_heads: i32, out: *mut *mut SgkKv) -> i32;
    pub fn sgk_kv_create(state: *mut SgkState, capacity: i64, q_heads: i32, kv_heads: i32, head_dim: i32, dtype: i32, page_tokens: i32, out: *mut *mut SgkKv) -> i32;
    pub fn sgk_kv_create_shuffled(state: *mut SgkState, capacity: i64, q_heads: i32, kv_heads: i32, head_dim: i32, dtype: i32, seed: u64, out: *mut *mut SgkKv) -> i32;
    pub fn sgk_kv_destroy(kv: *mut SgkKv);
    pub fn sgk_kv_len(kv: *const SgkKv) -> i64;
    pub fn sgk_kv_capacity(kv: *const SgkKv) -> i64;
    pub fn sgk_kv_kv_dim(kv: *const SgkKv) -> i32;
    pub fn sgk_kv_q_heads(kv: *const SgkKv) -> i32;
    pub fn sgk_kv_kv_heads(kv: *const SgkKv) -> i32;
    pub fn sgk_kv_head_dim(kv: *const SgkKv) -> i32;
    pub fn sgk_kv_dtype(kv: *const SgkKv) -> i32;
    pub fn sgk_kv_byte_len(kv: *const SgkKv) -> i64;
    pub fn sgk_kv_truncate(kv: *mut SgkKv, len: i64) -> i32;
    pub fn sgk_kv_enqueue_truncate(kv: *mut SgkKv, stream: *mut std::ffi::c_void, len: i64) -> i32;
    pub fn sgk_kv_set_attention_sinks(kv: *mut SgkKv, rows: i64) -> i32;
    pub fn sgk_kv_attention_sinks(kv: *const SgkKv) -> i64;
    pub fn sgk_kv_seed_f32(kv: *mut SgkKv, k: *const f32, k_len: usize, v: *const f32, v_len: usize, n_rows: i64) -> i32;
    pub fn sgk_kv_append_row_f32(kv: *mut SgkKv, k: *const f32, k_len: usize, v: *const f32, v_len: usize) -> i32;
    pub fn sgk_kv_append_rows_f32(kv: *mut SgkKv, k: *const f32, k_len: usize, v: *const f32, v_len: usize, n_rows: i64) -> i32;
    pub fn sgk_kv_enqueue_append(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32) -> i32;
    pub fn sgk_kv_enqueue_append_rows(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, n_rows: i64) -> i32;
    pub fn sgk_kv_enqueue_rope_append(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_k_raw: *const f32, d_v: *const f32, d_knorm_weight: *const f32, rope: *const SgkRope) -> i32;
    pub fn sgk_kv_enqueue_rope_append_rows(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_k_raw: *const f32, d_v: *const f32, n_rows: i64, d_knorm_weight: *const f32, rope: *const SgkRope) -> i32;
    pub fn sgk_kv_enqueue_verify_rows(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, n_rows: i32, sliding_window: i64, attn_scalar: f32) -> i32;
    pub fn sgk_rms_norm_rope_decode(state: *mut SgkState, x: *const f32, weight: *const f32, heads: i32, head_dim: i32, rope: *const SgkRope, position: i64, out: *mut f32) -> i32;
    pub fn sgk_kv_attention_decode(kv: *mut SgkKv, q: *const f32, q_len: usize, window_start: i64, attn_scalar: f32, out: *mut f32) -> i32;
    pub fn sgk_kv_enqueue_attention(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_q: *const f32, d_out: *mut f32, window_start: i64, attn_scalar: f32) -> i32;
    pub fn sgk_kv_enqueue_attention_noalloc(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_q: *const f32, d_out: *mut f32, window_start: i64, attn_scalar: f32) -> i32;
    pub fn sgk_kv_enqueue_append_attention(kv: *mut SgkKv, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, sliding_window: i64, attn_scalar: f32) -> i32;
    pub fn sgk_kv_gather_rows(kv: *mut SgkKv, row0: i64, n: i64, k_out: *mut std::ffi::c_void, v_out: *mut std::ffi::c_void) -> i32;
    pub fn sgk_kv_gather_rows_u8(kv: *mut SgkKv, row0: i64, n: i64, k_codes: *mut u8, k_scale: *mut u16, k_bias: *mut u16, v_codes: *mut u8, v_scale: *mut u16, v_bias: *mut u16) -> i32;
    pub fn sgk_kv_gather_rows_u4(kv: *mut SgkKv, row0: i64, n: i64, k_codes: *mut u8, k_scale: *mut u16, k_bias: *mut u16, v_codes: *mut u8, v_scale: *mut u16, v_bias: *mut u16) -> i32;
    pub fn sgk_kv_gather_rows_f32(kv: *mut SgkKv, row0: i64, n: i64, k_out: *mut f32, v_out: *mut f32) -> i32;
    pub fn sgk_kv_enqueue_gather_rows_f32(kv: *mut SgkKv, stream: *mut std::ffi::c_void, row0: i64, n: i64, d_k: *mut f32, d_v: *mut f32) -> i32;
    pub fn sgk_kv_block_table(kv: *const SgkKv, pages_out: *mut i32, cap: i64, n_out: *mut i64) -> i32;
    pub fn sgk_kv_set_attention_kernel(kv: *mut SgkKv, which: i32) -> i32;
    pub fn sgk_batch_create(state: *mut SgkState, kvs: *mut *mut SgkKv, n: i32, out: *mut *mut SgkBatch) -> i32;
    pub fn sgk_batch_destroy(batch: *mut SgkBatch);
    pub fn sgk_batch_enqueue_append(batch: *mut SgkBatch, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32) -> i32;
    pub fn sgk_batch_enqueue_attention(batch: *mut SgkBatch, stream: *mut std::ffi::c_void, d_q: *const f32, d_out: *mut f32, sliding_window: i64, attn_scalar: f32) -> i32;
    pub fn sgk_batch_enqueue_step(batch: *mut SgkBatch, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, sliding_window: i64, attn_scalar: f32) -> i32;
    pub fn sgk_batch_enqueue_truncate(batch: *mut SgkBatch, stream: *mut std::ffi::c_void, lens: *const i64) -> i32;
    pub fn sgk_batch_enqueue_verify_rows(batch: *mut SgkBatch, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, n_rows: i32, sliding_window: i64, attn_scalar: f32) -> i32;
    pub fn sgk_batch_set_splits(batch: *mut SgkBatch, splits: i32) -> i32;
    pub fn sgk_batch_get_splits(batch: *const SgkBatch, splits_out: *mut i32) -> i32;
    pub fn sgk_batch_set_kernel(batch: *mut SgkBatch, which: i32) -> i32;
    pub fn sgk_batch_last_kernel(batch: *const SgkBatch, which_out: *mut i32) -> i32;
    pub fn sgk_step_create(state: *mut SgkState, layers: *mut *mut SgkBatch, n_layers: i32, out: *mut *mut SgkStep) -> i32;
    pub fn sgk_step_destroy(step: *mut SgkStep);
    pub fn sgk_step_enqueue(step: *mut SgkStep, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, sliding_windows: *const i64, attn_scalar: f32) -> i32;
    pub fn sgk_step_capture(step: *mut SgkStep, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, sliding_windows: *const i64, attn_scalar: f32) -> i32;
    pub fn sgk_step_replay(step: *mut SgkStep, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_step_run_host(step: *mut SgkStep, k: *const f32, v: *const f32, q: *const f32, out: *mut f32, sliding_windows: *const i64, attn_scalar: f32) -> i32;
    pub fn sgk_step_launches(step: *const SgkStep) -> i64;
    pub fn sgk_linstate_create(state: *mut SgkState, layers: i32, conv_len: i64, ssm_len: i64, ssm_bf16: i32, out: *mut *mut SgkLinstate) -> i32;
    pub fn sgk_linstate_destroy(ls: *mut SgkLinstate);
    pub fn sgk_linstate_bytes(ls: *const SgkLinstate) -> i64;
    pub fn sgk_linstate_write(ls: *mut SgkLinstate, layer: i32, conv: *const f32, ssm: *const f32) -> i32;
    pub fn sgk_linstate_read(ls: *mut SgkLinstate, layer: i32, conv: *mut f32, ssm: *mut f32) -> i32;
    pub fn sgk_linstate_snapshot(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, snapshot_out: *mut *mut SgkLinstate) -> i32;
    pub fn sgk_linstate_restore(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, snapshot: *const SgkLinstate) -> i32;
    pub fn sgk_lm_head_enqueue_argmax(state: *mut SgkState, stream: *mut std::ffi::c_void, d_weight: *const std::ffi::c_void, weight_dtype: i32, vocab: i64, hidden: i32, d_x: *const f32, n_rows: i32, index_offset: i32, d_index_out: *mut i32, d_value_out: *mut f32) -> i32;
    pub fn sgk_lm_head_enqueue_argmax_affine(state: *mut SgkState, stream: *mut std::ffi::c_void, weight: *const SgkAffineWeight, vocab: i64, hidden: i32, d_x: *const f32, n_rows: i32, index_offset: i32, d_index_out: *mut i32, d_value_out: *mut f32) -> i32;
    pub fn sgk_embed_enqueue_from_index_affine(state: *mut SgkState, stream: *mut std::ffi::c_void, table: *const SgkAffineWeight, vocab: i64, hidden: i32, d_index: *const i32, embedding_scale: f32, recast_bf16: i32, d_out: *mut f32) -> i32;
    pub fn sgk_embed_enqueue_from_index(state: *mut SgkState, stream: *mut std::ffi::c_void, d_table: *const std::ffi::c_void, table_dtype: i32, vocab: i64, hidden: i32, d_index: *const i32, embedding_scale: f32, recast_bf16: i32, d_out: *mut f32) -> i32;
    pub fn sgk_batch_enqueue_step_exchange(batch: *mut SgkBatch, stream: *mut std::ffi::c_void, d_k: *const f32, d_v: *const f32, d_q: *const f32, ex: *mut SgkExchange, d_local_row: *mut f32, d_peer_rows: *const *mut f32, slice_offset: i64, sliding_window: i64, attn_scalar: f32) -> i32;
    pub fn sgk_peer_export(state: *mut SgkState, d_ptr: *mut std::ffi::c_void, handle_out: *mut u8) -> i32;
    pub fn sgk_peer_open(state: *mut SgkState, handle: *const u8, d_ptr_out: *mut *mut std::ffi::c_void) -> i32;
    pub fn sgk_peer_close(state: *mut SgkState, d_ptr: *mut std::ffi::c_void) -> i32;
    pub fn sgk_exchange_create(state: *mut SgkState, rank: i32, n_ranks: i32, out: *mut *mut SgkExchange, flags_handle_out: *mut u8) -> i32;
    pub fn sgk_exchange_destroy(ex: *mut SgkExchange);
    pub fn sgk_exchange_connect(ex: *mut SgkExchange, peer_rank: i32, peer_flags_handle: *const u8) -> i32;
    pub fn sgk_exchange_enqueue(ex: *mut SgkExchange, stream: *mut std::ffi::c_void, d_local_row: *mut f32, d_peer_rows: *const *mut f32, slice_offset: i64, slice_floats: i32) -> i32;
    pub fn sgk_token_window_create(state: *mut SgkState, depth: i32, out: *mut *mut SgkTokenWindow) -> i32;
    pub fn sgk_token_window_destroy(w: *mut SgkTokenWindow);
    pub fn sgk_token_window_output_slot(w: *mut SgkTokenWindow) -> *mut i32;
    pub fn sgk_token_window_previous_slot(w: *mut SgkTokenWindow) -> *const i32;
    pub fn sgk_token_window_submit(w: *mut SgkTokenWindow, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_token_window_pop(w: *mut SgkTokenWindow, token_out: *mut i32) -> i32;
    pub fn sgk_token_window_inflight(w: *const SgkTokenWindow) -> i32;
    pub fn sgk_token_window_enqueued(w: *const SgkTokenWindow) -> i64;
    pub fn sgk_token_window_depth(w: *const SgkTokenWindow) -> i32;
    pub fn sgk_token_window_drain(w: *mut SgkTokenWindow) -> i32;
    pub fn sgk_token_capture(step: *mut SgkStep, window: *mut SgkTokenWindow, io: *const SgkTokenIo, d_k: *const f32, d_v: *const f32, d_q: *const f32, d_out: *mut f32, sliding_windows: *const i64, attn_scalar: f32) -> i32;
    pub fn sgk_token_seed(step: *mut SgkStep, first_token: i32, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_token_submit(step: *mut SgkStep, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_linstate_enqueue_capture(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, capture: *mut SgkLinstate) -> i32;
    pub fn sgk_linstate_conv_ptr(ls: *mut SgkLinstate, layer: i32) -> *mut std::ffi::c_void;
    pub fn sgk_linstate_enqueue_conv_step(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, layer: i32, d_qkv: *const f32, d_weight: *const f32, conv_dim: i32, conv_kernel_dim: i32, d_out: *mut f32) -> i32;
    pub fn sgk_linstate_enqueue_gated_delta_step(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, layer: i32, shape: *const SgkLinearShape, d_q: *const f32, d_k: *const f32, d_v: *const f32, d_g: *const f32, d_beta: *const f32, d_out: *mut f32) -> i32;
    pub fn sgk_linstate_enqueue_conv_seq(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, layer: i32, d_qkv: *const f32, d_weight: *const f32, conv_dim: i32, conv_kernel_dim: i32, n_tokens: i32, d_out: *mut f32) -> i32;
    pub fn sgk_linstate_enqueue_gated_delta_seq(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, layer: i32, shape: *const SgkLinearShape, d_q: *const f32, d_k: *const f32, d_v: *const f32, d_g: *const f32, d_beta: *const f32, n_tokens: i32, d_out: *mut f32) -> i32;
    pub fn sgk_linstate_enqueue_gated_delta_step_batch(states: *const *mut SgkLinstate, n_states: i32, stream: *mut std::ffi::c_void, layer: i32, shape: *const SgkLinearShape, d_q: *const f32, d_k: *const f32, d_v: *const f32, d_g: *const f32, d_beta: *const f32, d_out: *mut f32) -> i32;
    pub fn sgk_linstate_enqueue_decode_step(ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, layer: i32, shape: *const SgkLinearShape, d_qkv: *const f32, d_conv_weight: *const f32, conv_kernel_dim: i32, d_beta_input: *const f32, d_gate_input: *const f32, d_a_log: *const f32, d_dt_bias: *const f32, d_out: *mut f32) -> i32;
    pub fn sgk_linstate_ssm_ptr(ls: *mut SgkLinstate, layer: i32) -> *mut std::ffi::c_void;
    pub fn sgk_hash_root(out: *mut u8);
    pub fn sgk_hash_for_session(key: *const std::os::raw::c_char, key_len: usize, present: i32, out: *mut u8);
    pub fn sgk_hash_chain(prev: *const u8, tokens: *const u64, n: usize, out: *mut u8);
    pub fn sgk_prefix_create(pool: *mut SgkPool, block_tokens: i64, capacity_blocks: i64, blocks_per_session: i64, budget_bytes: i64, out: *mut *mut SgkPrefix) -> i32;
    pub fn sgk_prefix_destroy(pc: *mut SgkPrefix);
    pub fn sgk_prefix_block_tokens(pc: *const SgkPrefix) -> i64;
    pub fn sgk_prefix_match(pc: *mut SgkPrefix, root: *const u8, tokens: *const u64, n: usize, tokens_out: *mut i64, hash_out: *mut u8, entry_out: *mut u64) -> i32;
    pub fn sgk_prefix_insert(pc: *mut SgkPrefix, session: *const u8, hash: *const u8, tokens: i64, seq: *mut SgkSeq, ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, inserted_out: *mut i32) -> i32;
    pub fn sgk_prefix_insert_chain(pc: *mut SgkPrefix, root: *const u8, tokens: *const u64, n: usize, from_tokens: i64, seq: *mut SgkSeq, stream: *mut std::ffi::c_void, inserted_out: *mut i32, last_hash_out: *mut u8) -> i32;
    pub fn sgk_prefix_restore(pc: *mut SgkPrefix, entry: u64, seq: *mut SgkSeq, ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, mode: i32, bytes_copied_out: *mut i64) -> i32;
    pub fn sgk_prefix_evict_lru(pc: *mut SgkPrefix, evicted_out: *mut i32, bytes_out: *mut i64) -> i32;
    pub fn sgk_prefix_bytes(pc: *const SgkPrefix) -> i64;
    pub fn sgk_prefix_pinned_bytes(pc: *const SgkPrefix) -> i64;
    pub fn sgk_prefix_len(pc: *const SgkPrefix) -> i64;
    pub fn sgk_prefix_evicted_count(pc: *const SgkPrefix) -> i64;
    pub fn sgk_prefix_session_count(pc: *const SgkPrefix, session: *const u8) -> i64;
    pub fn sgk_prefix_dump(pc: *const SgkPrefix, which: i32, cap: i64, sessions: *mut u8, hashes: *mut u8, tokens: *mut i64) -> i64;
    pub fn sgk_dprefix_create(pool: *mut SgkPool, capacity: i64, out: *mut *mut SgkDprefix) -> i32;
    pub fn sgk_dprefix_destroy(dp: *mut SgkDprefix);
    pub fn sgk_dprefix_get(dp: *mut SgkDprefix, prompt: *const u64, n: usize, seq: *mut SgkSeq, ls: *mut SgkLinstate, stream: *mut std::ffi::c_void, cached_len_out: *mut i64) -> i32;
    pub fn sgk_dprefix_put(dp: *mut SgkDprefix, tokens: *const u64, n: usize, seq: *mut SgkSeq, ls: *mut SgkLinstate, stream: *mut std::ffi::c_void) -> i32;
    pub fn sgk_dprefix_len(dp: *const SgkDprefix) -> i64;
    pub fn sgk_dprefix_entry_tokens(dp: *const SgkDprefix, index: i64, tokens_out: *mut u64, cap: i64) -> i64;
    pub fn sgk_longest_prefix_entry_index(flat_tokens: *const u64, lens: *const usize, n_entries: usize, prompt: *const u64, n: usize) -> i64;
    pub fn sgk_budget_create(static_cap: u64, total_memory: u64, headroom_bytes: u64, device_cap: u64, out: *mut *mut SgkBudget) -> i32;
    pub fn sgk_budget_destroy(b: *mut SgkBudget);
    pub fn sgk_budget_set_usage(b: *mut SgkBudget, current: u64, reserved: u64);
    pub fn sgk_budget_limit(b: *const SgkBudget, limit_out: *mut u64) -> i32;
    pub fn sgk_budget_check_allocation(b: *const SgkBudget, requested: u64, projected_out: *mut u64, available_out: *mut u64) -> i32;
    pub fn sgk_util_fill_normal(state: *mut SgkState, stream: *mut std::ffi::c_void, d_out: *mut f32, n: i64, seed: u64, stream_id: u64, index0: u64) -> i32;
    pub fn sgk_util_malloc(state: *mut SgkState, bytes: usize, d_out: *mut *mut std::ffi::c_void) -> i32;
    pub fn sgk_util_free(state: *mut SgkState, d_ptr: *mut std::ffi::c_void) -> i32;
    pub fn sgk_util_h2d(state: *mut SgkState, d_dst: *mut std::ffi::c_void, src: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn sgk_util_d2h(state: *mut SgkState, dst: *mut std::ffi::c_void, d_src: *const std::ffi::c_void, bytes: usize) -> i32;
    pub fn sgk_util_copy_blocks(state: *mut SgkState, stream: *mut std::ffi::c_void, d_dst: *mut std::ffi::c_void, d_src: *const std::ffi::c_void, dst_pages: *const i32, src_pages: *const i32, n_pages: i32, page_bytes: i64) -> i32;
}

/// Status of a libsgk call as the crate's error type (src/error.rs:12-75 of the reference).
pub fn check(rc: i32) -> Result<(), InferError> {
    if rc == SGK_OK {
        return Ok(());
    }
    // SAFETY: sgk_last_error returns a NUL-terminated thread-local string owned by the library.
    let msg = unsafe { std::ffi::CStr::from_ptr(sgk_last_error()) }.to_string_lossy().into_owned();
    Err(match rc {
        SGK_ERR_DIMENSION => InferError::Dimension(msg),
        SGK_ERR_CONFIG => InferError::Config(msg),
        SGK_ERR_MEMORY_GUARD => InferError::MemoryGuard(msg),
        SGK_ERR_SHAPE => InferError::Shape(msg),
        // SGK_ERR_BACKEND and SGK_ERR_TIMEOUT: the variant the Metal backend's failures use
        _ => InferError::Metal(msg),
    })
}
