// GENERATED by rust/gen_ffi.py from include/lumen_b200.h - do not edit by hand.
// Raw bindings of liblumen_b200.so.  Not compiled or tested where this was written (no rustc).
#![allow(non_camel_case_types)]

use std::os::raw::{c_char, c_int, c_void};

pub const LUMEN_OK: c_int = 0;
pub const LUMEN_ERR_INVALID: c_int = 1;
pub const LUMEN_ERR_SHAPE: c_int = 2;
pub const LUMEN_ERR_KV_OVERFLOW: c_int = 3;
pub const LUMEN_ERR_ROPE_RANGE: c_int = 4;
pub const LUMEN_ERR_EMBED_RANGE: c_int = 5;
pub const LUMEN_ERR_CACHE_COUNT: c_int = 6;
pub const LUMEN_ERR_CUDA: c_int = 7;
pub const LUMEN_ERR_NCCL: c_int = 8;
pub const LUMEN_ERR_TIMEOUT: c_int = 9;
pub const LUMEN_ERR_DTYPE: c_int = 10;
pub const LUMEN_ERR_PARAM_NAME: c_int = 11;
pub const LUMEN_ERR_UNSUPPORTED: c_int = 12;
pub const LUMEN_ERR_MISSING_PARAM: c_int = 13;
pub const LUMEN_NCCL_ID_BYTES: c_int = 128;
pub const LUMEN_W_Q: c_int = 0;
pub const LUMEN_W_K: c_int = 1;
pub const LUMEN_W_V: c_int = 2;
pub const LUMEN_W_O: c_int = 3;
pub const LUMEN_MLP_NONE: c_int = 0;
pub const LUMEN_MLP_DENSE: c_int = 1;
pub const LUMEN_MLP_MOE: c_int = 2;
pub const LUMEN_F32: c_int = 0;
pub const LUMEN_BF16: c_int = 1;

#[repr(C)]
pub struct lumen_ctx {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_tensor {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_rope {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_kv_cache {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_llama_kv_cache {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_self_attention {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_llama {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_model {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_page_pool {
    _private: [u8; 0],
}
#[repr(C)]
pub struct lumen_page_batch {
    _private: [u8; 0],
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct lumen_llama_config {
    pub vocab_size: usize,
    pub hidden_size: usize,
    pub intermediate_size: usize,
    pub num_hidden_layers: usize,
    pub num_attention_heads: usize,
    pub num_key_value_heads: usize,
    pub rms_norm_eps: f32,
    pub max_seq_len: usize,
    pub rope_theta: f32,
    pub head_dim: usize,
    pub qk_norm: c_int,
    pub weight_dtype: c_int,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct lumen_decoder_layer {
    pub heads: usize,
    pub dim: usize,
    pub rot_dim: usize,
    pub vdim: usize,
    pub kv_rank: usize,
    pub rot_dims: usize,
    pub rot_base: f64,
    pub scale: f32,
    pub mlp_kind: c_int,
    pub ff: usize,
    pub experts: usize,
    pub top: usize,
    pub expert_ff: usize,
    pub expert_limit: f32,
    pub shared_ff: usize,
    pub shared_limit: f32,
    pub mixer: c_int,
    pub kv_heads: usize,
    pub kv_from: c_int,
    pub chunk: usize,
    pub rot_factor: f64,
    pub rot_low: f64,
    pub rot_high: f64,
    pub rot_original: f64,
    pub gate_cap: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct lumen_decoder_config {
    pub vocab_size: usize,
    pub width: usize,
    pub num_layers: usize,
    pub layers: *const lumen_decoder_layer,
    pub norm_eps: f32,
    pub max_seq_len: usize,
    pub bigram_buckets: usize,
    pub bigram_mul_prev: usize,
    pub bigram_mul_cur: usize,
    pub side_dim: usize,
    pub weight_dtype: c_int,
    pub embed_scale: f32,
    pub tied_head: c_int,
    pub norms: c_int,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct lumen_sample_params {
    pub temperature: f32,
    pub top_p: f32,
    pub repetition_penalty: f32,
    pub recent_tokens: *const i32,
    pub n_recent: usize,
    pub uniform: f32,
}

#[link(name = "lumen_b200")]
extern "C" {
    pub fn lumen_nccl_unique_id(id_out_128_bytes: *mut c_void) -> c_int;
    pub fn lumen_ctx_create(device: c_int, tp_rank: c_int, tp_size: c_int, nccl_unique_id: *const c_void, out: *mut *mut lumen_ctx) -> c_int;
    pub fn lumen_ctx_destroy(ctx: *mut lumen_ctx) -> c_int;
    pub fn lumen_ctx_synchronize(ctx: *mut lumen_ctx) -> c_int;
    pub fn lumen_ctx_stream(ctx: *mut lumen_ctx) -> *mut c_void;
    pub fn lumen_ctx_launch_count(ctx: *const lumen_ctx) -> u64;
    pub fn lumen_last_error(ctx: *const lumen_ctx) -> *const c_char;
    pub fn lumen_status_string(status: c_int) -> *const c_char;
    pub fn lumen_version() -> c_int;
    pub fn lumen_tensor_from_host(ctx: *mut lumen_ctx, data: *const f32, shape: *const usize, ndim: c_int, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_tensor_from_host_bf16(ctx: *mut lumen_ctx, data: *const u16, shape: *const usize, ndim: c_int, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_tensor_empty(ctx: *mut lumen_ctx, shape: *const usize, ndim: c_int, dtype: c_int, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_tensor_ndim(t: *const lumen_tensor) -> c_int;
    pub fn lumen_tensor_shape(t: *const lumen_tensor, shape_out: *mut usize) -> c_int;
    pub fn lumen_tensor_numel(t: *const lumen_tensor) -> usize;
    pub fn lumen_tensor_dtype(t: *const lumen_tensor) -> c_int;
    pub fn lumen_tensor_data(t: *const lumen_tensor) -> *mut c_void;
    pub fn lumen_tensor_to_host(t: *const lumen_tensor, out: *mut f32) -> c_int;
    pub fn lumen_tensor_set(t: *mut lumen_tensor, data: *const f32) -> c_int;
    pub fn lumen_tensor_reshape(t: *const lumen_tensor, shape: *const i64, ndim: c_int, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_tensor_free(t: *mut lumen_tensor) -> c_int;
    pub fn lumen_matmul(ctx: *mut lumen_ctx, a: *const lumen_tensor, w: *const lumen_tensor, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_linear_forward(ctx: *mut lumen_ctx, x: *const lumen_tensor, w: *const lumen_tensor, bias: *const lumen_tensor, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_rmsnorm(ctx: *mut lumen_ctx, x: *const lumen_tensor, weight: *const lumen_tensor, eps: f32, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_silu(ctx: *mut lumen_ctx, x: *const lumen_tensor, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_mul(ctx: *mut lumen_ctx, a: *const lumen_tensor, b: *const lumen_tensor, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_add(ctx: *mut lumen_ctx, a: *const lumen_tensor, b: *const lumen_tensor, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_embedding(ctx: *mut lumen_ctx, ids: *const lumen_tensor, table: *const lumen_tensor, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_fused_softmax(ctx: *mut lumen_ctx, x: *const lumen_tensor, scale: f32, causal: c_int, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_gemv(ctx: *mut lumen_ctx, x_dev: *const f32, w_dev: *const c_void, w_dtype: c_int, layout_kn: c_int, k: usize, n: usize, y_dev: *mut f32) -> c_int;
    pub fn lumen_gemv_kn_static(ctx: *mut lumen_ctx, x_dev: *const f32, w_dev: *const c_void, w_dtype: c_int, k: usize, n: usize, y_dev: *mut f32) -> c_int;
    pub fn lumen_rope_new(ctx: *mut lumen_ctx, dim: usize, max_seq_len: usize, theta: f32, out: *mut *mut lumen_rope) -> c_int;
    pub fn lumen_rope_from_tables(ctx: *mut lumen_ctx, dim: usize, max_seq_len: usize, cos_host: *const f32, sin_host: *const f32, out: *mut *mut lumen_rope) -> c_int;
    pub fn lumen_rope_forward(rope: *mut lumen_rope, x_bhsd: *const lumen_tensor, offset: usize, out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_rope_free(rope: *mut lumen_rope) -> c_int;
    pub fn lumen_kv_new(ctx: *mut lumen_ctx, b: usize, h_kv: usize, max_seq: usize, d: usize, out: *mut *mut lumen_kv_cache) -> c_int;
    pub fn lumen_kv_reset(c: *mut lumen_kv_cache) -> c_int;
    pub fn lumen_kv_len(c: *const lumen_kv_cache) -> usize;
    pub fn lumen_kv_free(c: *mut lumen_kv_cache) -> c_int;
    pub fn lumen_kv_read(c: *const lumen_kv_cache, k_out: *mut f32, v_out: *mut f32) -> c_int;
    pub fn lumen_kv_write(c: *mut lumen_kv_cache, k_in: *const f32, v_in: *const f32, len: usize) -> c_int;
    pub fn lumen_llama_kv_new(ctx: *mut lumen_ctx, kv_heads: usize, max_seq_len: usize, head_dim: usize, out: *mut *mut lumen_llama_kv_cache) -> c_int;
    pub fn lumen_llama_kv_update(c: *mut lumen_llama_kv_cache, k: *const lumen_tensor, v: *const lumen_tensor, start_pos: usize) -> c_int;
    pub fn lumen_llama_kv_get_view(c: *const lumen_llama_kv_cache, current_len: usize, k_out: *mut *mut lumen_tensor, v_out: *mut *mut lumen_tensor) -> c_int;
    pub fn lumen_llama_kv_free(c: *mut lumen_llama_kv_cache) -> c_int;
    pub fn lumen_self_attention_new(ctx: *mut lumen_ctx, embed_dim: usize, n_head: usize, n_kv_head: usize, max_seq_len: usize, rope_theta: f32, causal: c_int, out: *mut *mut lumen_self_attention) -> c_int;
    pub fn lumen_self_attention_set_weight(attn: *mut lumen_self_attention, which: c_int, w: *const lumen_tensor) -> c_int;
    pub fn lumen_self_attention_forward(attn: *mut lumen_self_attention, x: *const lumen_tensor, cache: *mut lumen_kv_cache, out: *mut *mut lumen_tensor, cache_out: *mut *mut lumen_kv_cache) -> c_int;
    pub fn lumen_self_attention_free(attn: *mut lumen_self_attention) -> c_int;
    pub fn lumen_attention_decode(ctx: *mut lumen_ctx, q_dev: *const f32, k_new_dev: *const f32, v_new_dev: *const f32, n_head: usize, cache: *mut lumen_kv_cache, rope: *mut lumen_rope, causal: c_int, out_dev: *mut f32) -> c_int;
    pub fn lumen_llama_new(ctx: *mut lumen_ctx, cfg: *const lumen_llama_config, out: *mut *mut lumen_llama) -> c_int;
    pub fn lumen_tp_param_slice(cfg: *const lumen_llama_config, tp_rank: c_int, tp_size: c_int, name: *const c_char, out: *mut usize) -> c_int;
    pub fn lumen_llama_set_param(m: *mut lumen_llama, name: *const c_char, host_data: *const c_void, shape: *const usize, ndim: c_int, dtype: c_int) -> c_int;
    pub fn lumen_llama_init_kv_caches(m: *mut lumen_llama, batch: usize, caches_out: *mut *mut lumen_kv_cache) -> c_int;
    pub fn lumen_llama_reset_kv_caches(m: *mut lumen_llama, caches: *mut *mut lumen_kv_cache, n_caches: usize) -> c_int;
    pub fn lumen_llama_forward(m: *mut lumen_llama, ids_host: *const f32, b: usize, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, pos: usize, logits_host: *mut f32) -> c_int;
    pub fn lumen_llama_forward_last(m: *mut lumen_llama, ids_host: *const f32, b: usize, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, pos: usize, logits_host: *mut f32) -> c_int;
    pub fn lumen_llama_forward_device(m: *mut lumen_llama, ids_dev: *const f32, b: usize, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, logits_dev: *mut f32) -> c_int;
    pub fn lumen_sample_top_p(ctx: *mut lumen_ctx, logits_dev: *const f32, vocab: usize, params: *const lumen_sample_params, token_out: *mut i32) -> c_int;
    pub fn lumen_llama_forward_sample(m: *mut lumen_llama, ids_host: *const f32, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, params: *const lumen_sample_params, token_out: *mut i32) -> c_int;
    pub fn lumen_llama_free(m: *mut lumen_llama) -> c_int;
    pub fn lumen_llama_weight_bytes(m: *const lumen_llama) -> usize;
    pub fn lumen_llama_decode_trace(m: *mut lumen_llama, out: *mut u64, capacity: usize, n_out: *mut usize) -> c_int;
    pub fn lumen_decoder_new(ctx: *mut lumen_ctx, cfg: *const lumen_decoder_config, out: *mut *mut lumen_model) -> c_int;
    pub fn lumen_model_set_param(m: *mut lumen_model, name: *const c_char, host_data: *const c_void, shape: *const usize, ndim: c_int, dtype: c_int) -> c_int;
    pub fn lumen_model_init_kv_caches(m: *mut lumen_model, batch: usize, caches_out: *mut *mut lumen_kv_cache) -> c_int;
    pub fn lumen_model_reset_kv_caches(m: *mut lumen_model, caches: *mut *mut lumen_kv_cache, n_caches: usize) -> c_int;
    pub fn lumen_model_forward(m: *mut lumen_model, ids_host: *const f32, b: usize, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, logits_host: *mut f32) -> c_int;
    pub fn lumen_model_forward_last(m: *mut lumen_model, ids_host: *const f32, b: usize, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, logits_host: *mut f32) -> c_int;
    pub fn lumen_model_forward_device(m: *mut lumen_model, ids_dev: *const f32, b: usize, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, logits_dev: *mut f32) -> c_int;
    pub fn lumen_model_forward_sample(m: *mut lumen_model, ids_host: *const f32, s: usize, caches: *mut *mut lumen_kv_cache, n_caches: usize, params: *const lumen_sample_params, token_out: *mut i32) -> c_int;
    pub fn lumen_model_weight_bytes(m: *const lumen_model) -> usize;
    pub fn lumen_model_free(m: *mut lumen_model) -> c_int;
    pub fn lumen_page_pool_new(ctx: *mut lumen_ctx, pages: usize, page_size: usize, h_kv: usize, d: usize, dtype: c_int, out: *mut *mut lumen_page_pool) -> c_int;
    pub fn lumen_page_pool_k(pool: *const lumen_page_pool) -> *mut c_void;
    pub fn lumen_page_pool_v(pool: *const lumen_page_pool) -> *mut c_void;
    pub fn lumen_page_pool_mass(pool: *const lumen_page_pool) -> *mut f32;
    pub fn lumen_page_pool_free(pool: *mut lumen_page_pool) -> c_int;
    pub fn lumen_page_batch_new(pool: *const lumen_page_pool, n_head: usize, n_seq: usize, q_lens: *const i32, kv_lens: *const i32, first_pos: *const i32, tables: *const i32, table_stride: usize, causal: c_int, out: *mut *mut lumen_page_batch) -> c_int;
    pub fn lumen_page_batch_free(batch: *mut lumen_page_batch) -> c_int;
    pub fn lumen_paged_append(pool: *mut lumen_page_pool, batch: *const lumen_page_batch, rope: *const lumen_rope, q_dev: *const f32, k_dev: *const f32, v_dev: *const f32, q_stride: usize, kv_stride: usize, q_norm_dev: *const f32, k_norm_dev: *const f32, eps: f32, q_out_dev: *mut c_void) -> c_int;
    pub fn lumen_paged_attention(pool: *const lumen_page_pool, batch: *const lumen_page_batch, q_dev: *const c_void, scale: f32, out_dev: *mut c_void, out_dtype: c_int, lse_dev: *mut f32) -> c_int;
    pub fn lumen_paged_attention_mass(pool: *mut lumen_page_pool, batch: *const lumen_page_batch, q_dev: *const c_void, scale: f32, lse_dev: *const f32) -> c_int;
    pub fn lumen_paged_evict(pool: *mut lumen_page_pool, from: *const lumen_page_batch, to: *const lumen_page_batch, recent: usize, kept_dev: *mut i32, kept_stride: usize) -> c_int;
    pub fn lumen_gemv_repeat(ctx: *mut lumen_ctx, x_dev: *const f32, w_devs: *const *const c_void, n_w: usize, w_dtype: c_int, layout_kn: c_int, k: usize, n: usize, y_dev: *mut f32, iters: usize, us_per_call_out: *mut f32) -> c_int;
    pub fn lumen_attention_decode_repeat(ctx: *mut lumen_ctx, q_dev: *const f32, k_new_dev: *const f32, v_new_dev: *const f32, n_head: usize, caches: *const *mut lumen_kv_cache, n_caches: usize, rope: *mut lumen_rope, out_dev: *mut f32, iters: usize, us_per_call_out: *mut f32) -> c_int;
}
