//! Raw bindings to libtangq (generated by gen_bindings.py from include/tangq.h; do not edit).
#![allow(non_camel_case_types)]

use std::os::raw::{c_char, c_int, c_uint, c_void};

#[repr(C)]
pub struct tq_ctx {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_qweight {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_pages {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_comm {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_llama {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_moe {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_mla {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_dweight {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_tofazen {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_numuzen {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_dotanex {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_sakinex {
    _private: [u8; 0],
}

#[repr(C)]
pub struct tq_graph {
    _private: [u8; 0],
}

pub const TQ_OK: c_int = 0;
pub const TQ_EINVAL: c_int = 1;
pub const TQ_ECUDA: c_int = 2;
pub const TQ_ENCCL: c_int = 3;
pub const TQ_ETIMEOUT: c_int = 4;
pub const TQ_ENOMEM: c_int = 5;
pub const TQ_EUNSUPPORTED: c_int = 6;

pub const TQ_F32: c_int = 0;
pub const TQ_BF16: c_int = 1;
pub const TQ_F16: c_int = 2;
pub const TQ_I8: c_int = 3;
pub const TQ_U8: c_int = 4;
pub const TQ_I32: c_int = 5;
pub const TQ_F64: c_int = 6;

pub const TQ_Q4_F32: c_int = 0;
pub const TQ_Q4_F16: c_int = 1;
pub const TQ_Q8_F32: c_int = 2;
pub const TQ_I8_ROW: c_int = 3;

pub const TQ_TZ_EMBED: c_int = 0;
pub const TQ_TZ_POS: c_int = 1;
pub const TQ_TZ_FINAL_NORM: c_int = 2;
pub const TQ_TZ_HEAD: c_int = 3;
pub const TQ_TZ_NORM: c_int = 4;
pub const TQ_TZ_Q: c_int = 5;
pub const TQ_TZ_K: c_int = 6;
pub const TQ_TZ_V: c_int = 7;
pub const TQ_TZ_O: c_int = 8;
pub const TQ_TZ_GATE: c_int = 9;
pub const TQ_TZ_UP: c_int = 10;
pub const TQ_TZ_DOWN: c_int = 11;

pub const TQ_NZ_ATTENTION: c_int = 0;
pub const TQ_NZ_GLA: c_int = 1;

pub const TQ_NZ_EMBED: c_int = 0;
pub const TQ_NZ_FINAL_NORM: c_int = 1;
pub const TQ_NZ_NORM1: c_int = 2;
pub const TQ_NZ_NORM1B: c_int = 3;
pub const TQ_NZ_NORM2: c_int = 4;
pub const TQ_NZ_NORM2B: c_int = 5;
pub const TQ_NZ_Q: c_int = 6;
pub const TQ_NZ_K: c_int = 7;
pub const TQ_NZ_V: c_int = 8;
pub const TQ_NZ_G: c_int = 9;
pub const TQ_NZ_O: c_int = 10;
pub const TQ_NZ_Q_NORM: c_int = 11;
pub const TQ_NZ_K_NORM: c_int = 12;
pub const TQ_NZ_O_NORM: c_int = 13;
pub const TQ_NZ_A1: c_int = 14;
pub const TQ_NZ_A2: c_int = 15;
pub const TQ_NZ_A2_BIAS: c_int = 16;
pub const TQ_NZ_ROUTER: c_int = 17;
pub const TQ_NZ_GATE: c_int = 18;
pub const TQ_NZ_UP: c_int = 19;
pub const TQ_NZ_DOWN: c_int = 20;

pub const TQ_DX_ATTENTION: c_int = 0;
pub const TQ_DX_LATENT: c_int = 1;
pub const TQ_DX_LIGHTNING: c_int = 2;

pub const TQ_DX_NONE: c_int = 0;
pub const TQ_DX_DENSE: c_int = 1;
pub const TQ_DX_MOE: c_int = 2;

pub const TQ_DX_EMBED: c_int = 0;
pub const TQ_DX_FINAL_NORM: c_int = 1;
pub const TQ_DX_HEAD: c_int = 2;
pub const TQ_DX_NORM1: c_int = 3;
pub const TQ_DX_NORM2: c_int = 4;
pub const TQ_DX_HC1_IN: c_int = 5;
pub const TQ_DX_HC1_OUT: c_int = 6;
pub const TQ_DX_HC1_MIX: c_int = 7;
pub const TQ_DX_HC2_IN: c_int = 8;
pub const TQ_DX_HC2_OUT: c_int = 9;
pub const TQ_DX_HC2_MIX: c_int = 10;
pub const TQ_DX_Q: c_int = 11;
pub const TQ_DX_K: c_int = 12;
pub const TQ_DX_V: c_int = 13;
pub const TQ_DX_G: c_int = 14;
pub const TQ_DX_O: c_int = 15;
pub const TQ_DX_Q_NORM: c_int = 16;
pub const TQ_DX_K_NORM: c_int = 17;
pub const TQ_DX_SINK: c_int = 18;
pub const TQ_DX_O_NORM: c_int = 19;
pub const TQ_DX_DQ: c_int = 20;
pub const TQ_DX_DQ_NORM: c_int = 21;
pub const TQ_DX_UQ: c_int = 22;
pub const TQ_DX_DKV: c_int = 23;
pub const TQ_DX_DKV_NORM: c_int = 24;
pub const TQ_DX_UK: c_int = 25;
pub const TQ_DX_UV: c_int = 26;
pub const TQ_DX_ROUTER: c_int = 27;
pub const TQ_DX_CORRECTION: c_int = 28;
pub const TQ_DX_GATE: c_int = 29;
pub const TQ_DX_UP: c_int = 30;
pub const TQ_DX_DOWN: c_int = 31;
pub const TQ_DX_SHARED_GATE: c_int = 32;
pub const TQ_DX_SHARED_UP: c_int = 33;
pub const TQ_DX_SHARED_DOWN: c_int = 34;

pub const TQ_SX_EMBED: c_int = 0;
pub const TQ_SX_FINAL_NORM: c_int = 1;
pub const TQ_SX_HEAD: c_int = 2;
pub const TQ_SX_NORM1: c_int = 3;
pub const TQ_SX_NORM2: c_int = 4;
pub const TQ_SX_CANON1: c_int = 5;
pub const TQ_SX_CANON2: c_int = 6;
pub const TQ_SX_Q: c_int = 7;
pub const TQ_SX_K: c_int = 8;
pub const TQ_SX_V: c_int = 9;
pub const TQ_SX_Q_CONV: c_int = 10;
pub const TQ_SX_K_CONV: c_int = 11;
pub const TQ_SX_V_CONV: c_int = 12;
pub const TQ_SX_LEFT_O: c_int = 13;
pub const TQ_SX_Z: c_int = 14;
pub const TQ_SX_Z_BIAS: c_int = 15;
pub const TQ_SX_X: c_int = 16;
pub const TQ_SX_X_BIAS: c_int = 17;
pub const TQ_SX_G: c_int = 18;
pub const TQ_SX_RIGHT_O: c_int = 19;
pub const TQ_SX_ROUTER: c_int = 20;
pub const TQ_SX_ROUTER_BIAS: c_int = 21;
pub const TQ_SX_GATE: c_int = 22;
pub const TQ_SX_UP: c_int = 23;
pub const TQ_SX_DOWN: c_int = 24;
pub const TQ_SX_SHARED_GATE: c_int = 25;
pub const TQ_SX_SHARED_UP: c_int = 26;
pub const TQ_SX_SHARED_DOWN: c_int = 27;
pub const TQ_SX_SHARED_SWITCH: c_int = 28;

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_sampler_config {
    pub temperature: f64,
    pub top_k: u64,
    pub top_p: f64,
    pub repetition_penalty: f64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_llama_config {
    pub n_layers: u32,
    pub d_model: u32,
    pub n_heads: u32,
    pub n_kv_heads: u32,
    pub head_dim: u32,
    pub ffn: u32,
    pub vocab: u32,
    pub max_seq: u32,
    pub max_batch: u32,
    pub eps: f32,
    pub rope_base: f64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_moe_config {
    pub d_model: u32,
    pub ffn: u32,
    pub n_experts: u32,
    pub top_k: u32,
    pub n_shared: u32,
    pub renormalize: u32,
    pub ep_rank: u32,
    pub ep_size: u32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_mla_config {
    pub d_model: u32,
    pub n_heads: u32,
    pub q_lora: u32,
    pub kv_lora: u32,
    pub nope_dim: u32,
    pub rope_dim: u32,
    pub v_dim: u32,
    pub max_batch: u32,
    pub max_pos: u32,
    pub norm_eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_diff_attn_config {
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub window: u32,
    pub keep_first: u32,
    pub scale: f32,
    pub lambda: f32,
    pub out_scale: f32,
    pub eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_tofazen_config {
    pub n_layers: u32,
    pub width: u32,
    pub vocab: u32,
    pub max_positions: u32,
    pub max_seq: u32,
    pub max_slots: u32,
    pub dtype: c_int,
    pub eps: f32,
    pub residual_mult: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_tofazen_layer {
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub ff: u32,
    pub kv_from: c_int,
    pub window: u32,
    pub keep_first: u32,
    pub scale: f32,
    pub lambda: f32,
    pub out_scale: f32,
    pub limit: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_window_attn_config {
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub window: u32,
    pub scale: f32,
    pub softcap: f32,
    pub sink: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_conv_heads_config {
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub k0: u32,
    pub v0: u32,
    pub channels: u32,
    pub taps: u32,
    pub rot_dims: u32,
    pub norm: c_int,
    pub pool: u32,
    pub pool_rows: u32,
    pub rot_mult: f32,
    pub eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_gla_config {
    pub heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub rank: u32,
    pub tau: f32,
    pub q_scale: f32,
    pub eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_numuzen_config {
    pub n_layers: u32,
    pub width: u32,
    pub vocab: u32,
    pub max_seq: u32,
    pub max_slots: u32,
    pub dtype: c_int,
    pub eps: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_numuzen_layer {
    pub kind: u32,
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub window: u32,
    pub rot_dims: u32,
    pub rank: u32,
    pub experts: u32,
    pub top: u32,
    pub ff: u32,
    pub scale: f32,
    pub softcap: f32,
    pub tau: f32,
    pub limit: f32,
    pub rot_base: f64,
    pub rot_factor: f64,
    pub rot_original: f64,
    pub rot_fast: f64,
    pub rot_slow: f64,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_dotanex_config {
    pub n_layers: u32,
    pub width: u32,
    pub vocab: u32,
    pub streams: u32,
    pub max_seq: u32,
    pub max_slots: u32,
    pub dtype: c_int,
    pub eps: f32,
    pub expand_bytes: usize,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_dotanex_layer {
    pub kind: u32,
    pub weights_of: c_int,
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub window: u32,
    pub rot_dims: u32,
    pub q_rank: u32,
    pub kv_rank: u32,
    pub rot_dim: u32,
    pub ff_kind: u32,
    pub ff: u32,
    pub experts: u32,
    pub identity: u32,
    pub top: u32,
    pub shared_ff: u32,
    pub scale: f32,
    pub limit: f32,
    pub shared_limit: f32,
    pub rot_base: f64,
    pub rot_factor: f64,
    pub rot_original: f64,
    pub rot_low: f64,
    pub rot_high: f64,
    pub rot_fast: f64,
    pub rot_slow: f64,
    pub decay: *const f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_sakinex_config {
    pub n_layers: u32,
    pub width: u32,
    pub vocab: u32,
    pub taps: u32,
    pub max_seq: u32,
    pub max_slots: u32,
    pub dtype: c_int,
    pub eps: f32,
    pub residual_mult: f32,
}

#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct tq_sakinex_layer {
    pub weights_of: c_int,
    pub add_embedding: c_int,
    pub heads: u32,
    pub kv_heads: u32,
    pub dim: u32,
    pub vdim: u32,
    pub window: u32,
    pub pool: u32,
    pub taps: u32,
    pub rot_dims: u32,
    pub state_width: u32,
    pub experts: u32,
    pub top: u32,
    pub ff: u32,
    pub shared_ff: u32,
    pub scale: f32,
    pub left_scale: f32,
    pub right_scale: f32,
    pub rot_base: f64,
    pub rot_factor: f64,
    pub rot_original: f64,
    pub rot_fast: f64,
    pub rot_slow: f64,
}

#[link(name = "tangq")]
extern "C" {
    pub fn tq_ctx_create(device: c_int, stream: *mut c_void, out: *mut *mut tq_ctx) -> c_int;
    pub fn tq_ctx_destroy(ctx: *mut tq_ctx) -> c_int;
    pub fn tq_last_error(ctx: *const tq_ctx) -> *const c_char;
    pub fn tq_sync(ctx: *mut tq_ctx) -> c_int;
    pub fn tq_ctx_stream(ctx: *mut tq_ctx) -> *mut c_void;
    pub fn tq_version() -> c_int;
    pub fn tq_buf_alloc(ctx: *mut tq_ctx, bytes: usize, dev_out: *mut *mut c_void) -> c_int;
    pub fn tq_buf_free(ctx: *mut tq_ctx, dev: *mut c_void) -> c_int;
    pub fn tq_upload(ctx: *mut tq_ctx, dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> c_int;
    pub fn tq_download(ctx: *mut tq_ctx, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> c_int;
    pub fn tq_memset(ctx: *mut tq_ctx, dst_dev: *mut c_void, byte: c_int, bytes: usize) -> c_int;
    pub fn tq_convert(ctx: *mut tq_ctx, src_dev: *const c_void, src_dtype: c_int, dst_dev: *mut c_void, dst_dtype: c_int, n: usize) -> c_int;
    pub fn tq_qweight_from_blocks(ctx: *mut tq_ctx, kind: c_int, blocks_host: *const c_void, rows: usize, cols: usize, out: *mut *mut tq_qweight) -> c_int;
    pub fn tq_qweight_from_arrays(ctx: *mut tq_ctx, kind: c_int, payload_host: *const c_void, scales_host: *const c_void, rows: usize, cols: usize, out: *mut *mut tq_qweight) -> c_int;
    pub fn tq_qweight_from_device_arrays(ctx: *mut tq_ctx, kind: c_int, payload_dev: *const c_void, scales_dev: *const c_void, rows: usize, cols: usize, out: *mut *mut tq_qweight) -> c_int;
    pub fn tq_quantize_matrix(ctx: *mut tq_ctx, src_dev: *const c_void, src_dtype: c_int, ld: usize, rows: usize, cols: usize, kind: c_int, out: *mut *mut tq_qweight) -> c_int;
    pub fn tq_qweight_free(ctx: *mut tq_ctx, w: *mut tq_qweight) -> c_int;
    pub fn tq_qweight_shape(w: *const tq_qweight, rows: *mut usize, cols: *mut usize, kind: *mut c_int) -> c_int;
    pub fn tq_qweight_bytes(w: *const tq_qweight) -> usize;
    pub fn tq_dequantize(ctx: *mut tq_ctx, w: *const tq_qweight, out_dev: *mut f32, ints_dev: *mut i8) -> c_int;
    pub fn tq_qlinear(ctx: *mut tq_ctx, w: *const tq_qweight, x_dev: *const c_void, x_dtype: c_int, ldx: usize, m: usize, y_dev: *mut c_void, y_dtype: c_int, ldy: usize, residual_dev: *const f32) -> c_int;
    pub fn tq_q_matvec_host(ctx: *mut tq_ctx, w: *const tq_qweight, x_host: *const c_void, y_host: *mut c_void, dtype: c_int, m: usize) -> c_int;
    pub fn tq_q_matvec_host_async(ctx: *mut tq_ctx, w: *const tq_qweight, x_host: *const c_void, y_host: *mut c_void, dtype: c_int, m: usize) -> c_int;
    pub fn tq_qweight_concat_rows(ctx: *mut tq_ctx, parts: *const *const tq_qweight, n_parts: usize, out: *mut *mut tq_qweight) -> c_int;
    pub fn tq_qweight_interleave_gate_up(ctx: *mut tq_ctx, w_gate_up: *const tq_qweight, out: *mut *mut tq_qweight) -> c_int;
    pub fn tq_rms_norm(ctx: *mut tq_ctx, x_dev: *const c_void, x_dtype: c_int, residual_dev: *const f32, weight_dev: *const c_void, w_dtype: c_int, n_groups: usize, dim: usize, eps: f32, out_dev: *mut c_void, out_dtype: c_int, sum_out_dev: *mut f32) -> c_int;
    pub fn tq_rope_tables(ctx: *mut tq_ctx, head_dim: usize, max_seq_len: usize, base: f64, cos_dev: *mut f32, sin_dev: *mut f32) -> c_int;
    pub fn tq_rope_forward(ctx: *mut tq_ctx, x_dev: *const c_void, x_dtype: c_int, cos_dev: *const f32, sin_dev: *const f32, positions_dev: *const c_int, seq_len: usize, n_heads: usize, head_dim: usize, start_pos: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_swiglu(ctx: *mut tq_ctx, gate_dev: *const c_void, up_dev: *const c_void, in_dtype: c_int, ld: usize, rows: usize, n: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_embedding(ctx: *mut tq_ctx, weight_dev: *const c_void, w_dtype: c_int, ids_dev: *const c_int, seq_len: usize, dim: usize, vocab: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_argmax_rows(ctx: *mut tq_ctx, x_dev: *const f32, slices: usize, rows: usize, cols: usize, idx_out_dev: *mut c_int) -> c_int;
    pub fn tq_sample(ctx: *mut tq_ctx, logits_dev: *const f32, slices: usize, rows: usize, cols: usize, cfg: *const tq_sampler_config, rng_states_dev: *mut u64, past_tokens_dev_or_null: *const c_int, past_lens_dev_or_null: *const c_int, past_ld: usize, tokens_out_dev: *mut c_int) -> c_int;
    pub fn tq_generate_advance(ctx: *mut tq_ctx, chosen_dev: *const c_int, rows: usize, tokens_io_dev: *mut c_int, positions_io_dev: *mut c_int, out_tokens_dev: *mut c_int, out_ld: usize, step_io_dev_or_null: *mut c_int, lens_io_dev_or_null: *mut c_int) -> c_int;
    pub fn tq_kv_attention(ctx: *mut tq_ctx, q_dev: *const f32, k_cache_dev: *const f32, v_cache_dev: *const f32, cache_start: usize, q_len: usize, n_heads: usize, n_kv_heads: usize, head_dim: usize, out_dev: *mut f32) -> c_int;
    pub fn tq_gqa_decode(ctx: *mut tq_ctx, q_dev: *const c_void, k_cache_dev: *const c_void, v_cache_dev: *const c_void, lens_dev: *const c_int, batch: usize, n_heads: usize, n_kv_heads: usize, head_dim: usize, seq_stride: usize, max_len: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_gqa_decode_noalloc(ctx: *mut tq_ctx, q_dev: *const c_void, k_cache_dev: *const c_void, v_cache_dev: *const c_void, lens_dev: *const c_int, batch: usize, n_heads: usize, n_kv_heads: usize, head_dim: usize, seq_stride: usize, max_len: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_gqa_prefill(ctx: *mut tq_ctx, q_dev: *const c_void, k_cache_dev: *const c_void, v_cache_dev: *const c_void, cache_start_dev: *const c_int, batch: usize, q_len: usize, n_heads: usize, n_kv_heads: usize, head_dim: usize, seq_stride: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_token_logprobs(ctx: *mut tq_ctx, logits_dev: *const c_void, dtype: c_int, ld: usize, slices: usize, rows: usize, cols: usize, tokens_dev_or_null: *const c_int, n_tokens: usize, top: usize, logprob_out_dev: *mut f32, entropy_out_dev_or_null: *mut f32, top_ids_out_dev: *mut c_int, top_logprob_out_dev: *mut f32) -> c_int;
    pub fn tq_pages_create(ctx: *mut tq_ctx, n_pages: usize, page_rows: usize, n_seqs: usize, table_ld: usize, refs_dev_or_null: *mut c_int, tables_dev_or_null: *mut c_int, lens_dev_or_null: *mut c_int, out: *mut *mut tq_pages) -> c_int;
    pub fn tq_pages_destroy(pages: *mut tq_pages) -> c_int;
    pub fn tq_pages_arrays(pages: *mut tq_pages, bases_host: *const *mut c_void, n_arrays: usize, row_bytes: usize) -> c_int;
    pub fn tq_pages_data(pages: *const tq_pages, refs_dev: *mut *mut c_int, tables_dev: *mut *mut c_int, lens_dev: *mut *mut c_int) -> c_int;
    pub fn tq_pages_extend(pages: *mut tq_pages, seqs_dev: *const c_int, counts_dev_or_null: *const c_int, n: usize) -> c_int;
    pub fn tq_pages_fork(pages: *mut tq_pages, src_dev: *const c_int, dst_dev: *const c_int, keep_dev_or_null: *const c_int, n: usize) -> c_int;
    pub fn tq_pages_free(pages: *mut tq_pages, seqs_dev: *const c_int, n: usize) -> c_int;
    pub fn tq_pages_compact(pages: *mut tq_pages, used_out_dev_or_null: *mut c_int) -> c_int;
    pub fn tq_gqa_decode_paged(ctx: *mut tq_ctx, q_dev: *const c_void, k_pages_dev: *const c_void, v_pages_dev: *const c_void, pages: *const tq_pages, seqs_dev_or_null: *const c_int, batch: usize, group_starts_dev_or_null: *const c_int, shared_dev_or_null: *const c_int, n_groups: usize, max_shared: usize, n_heads: usize, n_kv_heads: usize, head_dim: usize, max_len: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_comm_unique_id(id_out128: *mut c_void) -> c_int;
    pub fn tq_comm_create(ctx: *mut tq_ctx, id128: *const c_void, rank: c_int, world: c_int, out: *mut *mut tq_comm) -> c_int;
    pub fn tq_comm_destroy(ctx: *mut tq_ctx, comm: *mut tq_comm) -> c_int;
    pub fn tq_comm_abort(comm: *mut tq_comm) -> c_int;
    pub fn tq_comm_rank(comm: *const tq_comm) -> c_int;
    pub fn tq_comm_world(comm: *const tq_comm) -> c_int;
    pub fn tq_all_reduce_f32(ctx: *mut tq_ctx, comm: *mut tq_comm, buf_dev: *mut f32, n: usize) -> c_int;
    pub fn tq_comm_enable_peer(ctx: *mut tq_ctx, comm: *mut tq_comm, max_elems: usize) -> c_int;
    pub fn tq_comm_peer_local(ctx: *mut tq_ctx, rank: c_int, world: c_int, peer_bufs_dev: *const *mut c_void, max_elems: usize, out: *mut *mut tq_comm) -> c_int;
    pub fn tq_comm_peer_bytes(world: c_int, max_elems: usize) -> usize;
    pub fn tq_comm_set_wait_limit(comm: *mut tq_comm, polls: c_uint) -> c_int;
    pub fn tq_all_gather(ctx: *mut tq_ctx, comm: *mut tq_comm, send_dev: *const c_void, recv_dev: *mut c_void, bytes_per_rank: usize) -> c_int;
    pub fn tq_all_to_all(ctx: *mut tq_ctx, comm: *mut tq_comm, send_dev: *const c_void, recv_dev: *mut c_void, bytes_per_peer: usize) -> c_int;
    pub fn tq_llama_create(ctx: *mut tq_ctx, cfg: *const tq_llama_config, comm_or_null: *mut tq_comm, out: *mut *mut tq_llama) -> c_int;
    pub fn tq_llama_destroy(model: *mut tq_llama) -> c_int;
    pub fn tq_llama_set_layer(model: *mut tq_llama, layer: usize, wqkv: *const tq_qweight, wo: *const tq_qweight, wgate_up: *const tq_qweight, wdown: *const tq_qweight, attn_norm_bf16_dev: *const c_void, ffn_norm_bf16_dev: *const c_void) -> c_int;
    pub fn tq_llama_set_head(model: *mut tq_llama, embed_bf16_dev: *const c_void, final_norm_bf16_dev: *const c_void, lm_head: *const tq_qweight) -> c_int;
    pub fn tq_llama_kv_cache(model: *mut tq_llama, layer: usize, k_cache_dev: *mut *mut c_void, v_cache_dev: *mut *mut c_void, seq_stride_elems: *mut usize) -> c_int;
    pub fn tq_llama_kv_trim(model: *mut tq_llama, seq_lens_io_dev: *mut c_int, batch: usize, keep: usize) -> c_int;
    pub fn tq_llama_hidden(model: *mut tq_llama, hidden_dev: *mut *mut f32) -> c_int;
    pub fn tq_llama_decode(model: *mut tq_llama, token_ids_dev: *const c_int, positions_dev: *const c_int, batch: usize, max_len: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_llama_decode_at(model: *mut tq_llama, token_ids_dev: *const c_int, positions_dev: *const c_int, rope_positions_dev: *const c_int, batch: usize, max_len: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_llama_decode_paged(model: *mut tq_llama, token_ids_dev: *const c_int, pages: *const tq_pages, seqs_dev_or_null: *const c_int, batch: usize, group_starts_dev_or_null: *const c_int, shared_dev_or_null: *const c_int, n_groups: usize, max_shared: usize, max_len: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_llama_prefill(model: *mut tq_llama, token_ids_dev: *const c_int, cache_start_dev: *const c_int, batch: usize, q_len: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_moe_router(ctx: *mut tq_ctx, h_bf16_dev: *const c_void, wg_bf16_dev: *const c_void, n_tokens: usize, d_model: usize, n_experts: usize, top_k: usize, renormalize: c_int, idx_out_dev: *mut c_int, weight_out_dev: *mut f32, logits_out_dev: *mut f64) -> c_int;
    pub fn tq_moe_create(ctx: *mut tq_ctx, cfg: *const tq_moe_config, wg_bf16_dev: *const c_void, w_gate_up_stacked: *const tq_qweight, w_down_stacked: *const tq_qweight, shared_gate_up: *const *const tq_qweight, shared_down: *const *const tq_qweight, out: *mut *mut tq_moe) -> c_int;
    pub fn tq_moe_destroy(moe: *mut tq_moe) -> c_int;
    pub fn tq_moe_ffn(moe: *mut tq_moe, h_bf16_dev: *const c_void, n_tokens: usize, out_dev: *mut f32, comm_or_null: *mut tq_comm, idx_out_dev: *mut c_int, weight_out_dev: *mut f32) -> c_int;
    pub fn tq_moe_ffn_dispatch(moe: *mut tq_moe, h_bf16_dev: *const c_void, n_tokens: usize, out_dev: *mut f32, comm_or_null: *mut tq_comm, idx_out_dev_or_null: *mut c_int, weight_out_dev_or_null: *mut f32) -> c_int;
    pub fn tq_mla_decode(ctx: *mut tq_ctx, q_full_bf16_dev: *const c_void, cache_bf16_dev: *const c_void, lens_dev: *const c_int, batch: usize, n_heads: usize, kv_lora: usize, rope_dim: usize, seq_stride: usize, max_len: usize, softmax_scale: f32, o_lat_bf16_dev: *mut c_void) -> c_int;
    pub fn tq_mla_absorb_q(ctx: *mut tq_ctx, w_qk_stacked: *const tq_qweight, q_nope_bf16_dev: *const c_void, q_rope_bf16_dev: *const c_void, batch: usize, n_heads: usize, nope_dim: usize, q_full_bf16_dev: *mut c_void) -> c_int;
    pub fn tq_mla_unabsorb(ctx: *mut tq_ctx, w_uv_stacked: *const tq_qweight, o_lat_bf16_dev: *const c_void, batch: usize, n_heads: usize, v_dim: usize, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_mla_create(ctx: *mut tq_ctx, cfg: *const tq_mla_config, q_a: *const tq_qweight, q_a_norm_gain_bf16_dev_or_null: *const c_void, q_b: *const tq_qweight, w_qk_stacked: *const tq_qweight, w_uv_stacked: *const tq_qweight, w_o: *const tq_qweight, rope_cos_dev: *const f32, rope_sin_dev: *const f32, out: *mut *mut tq_mla) -> c_int;
    pub fn tq_mla_destroy(layer: *mut tq_mla) -> c_int;
    pub fn tq_mla_layer_decode(layer: *mut tq_mla, h_bf16_dev: *const c_void, cache_bf16_dev: *const c_void, lens_dev: *const c_int, batch: usize, seq_stride: usize, max_len: usize, comm_or_null: *mut tq_comm, out_dev: *mut f32) -> c_int;
    pub fn tq_dweight_create(ctx: *mut tq_ctx, rows: usize, cols: usize, dtype: c_int, out: *mut *mut tq_dweight) -> c_int;
    pub fn tq_dweight_put(ctx: *mut tq_ctx, w: *mut tq_dweight, src: *const c_void, src_dtype: c_int, rows: usize, cols: usize, row0: usize, col0: usize, interleave: c_int) -> c_int;
    pub fn tq_dweight_free(ctx: *mut tq_ctx, w: *mut tq_dweight) -> c_int;
    pub fn tq_dweight_data(w: *const tq_dweight, dev: *mut *mut c_void, rows_padded: *mut usize, cols_padded: *mut usize) -> c_int;
    pub fn tq_dlinear(ctx: *mut tq_ctx, w: *const tq_dweight, x_dev: *const c_void, ldx: usize, m: usize, y_dev: *mut c_void, y_dtype: c_int, ldy: usize) -> c_int;
    pub fn tq_clamped_glu(ctx: *mut tq_ctx, gate_dev: *const c_void, up_dev: *const c_void, in_dtype: c_int, n: usize, limit: f32, alpha: f32, out_dev: *mut c_void, out_dtype: c_int) -> c_int;
    pub fn tq_dense_group_chunk(dtype: c_int, cols: usize, rows: usize, n_groups: usize) -> usize;
    pub fn tq_dlinear_grouped(ctx: *mut tq_ctx, w: *const tq_dweight, x_dev: *const c_void, ldx: usize, rows: usize, jobs_dev: *const c_int, n_jobs_dev: *const c_int, max_jobs: usize, chunk: usize, group_rows: usize, x_rows_dev_or_null: *const c_int, row_scale_dev_or_null: *const f32, glu_limit: f32, glu_alpha: f32, y_dev: *mut c_void, y_dtype: c_int, ldy: usize) -> c_int;
    pub fn tq_embedding_pos(ctx: *mut tq_ctx, table_dev: *const c_void, pos_table_dev: *const c_void, dtype: c_int, ids_dev: *const c_int, seq_rows_dev_or_null: *const c_int, starts_dev: *const c_int, slots_dev_or_null: *const c_int, n_seqs: usize, rows: usize, dim: usize, vocab: usize, n_pos: usize, max_seq: usize, n_slots: usize, out_dev: *mut f32, row_pos_dev: *mut c_int, cache_row_dev: *mut c_int) -> c_int;
    pub fn tq_diff_attention(ctx: *mut tq_ctx, cfg: *const tq_diff_attn_config, dtype: c_int, q_dev: *const c_void, ldq: usize, k_cache_dev: *const c_void, v_cache_dev: *const c_void, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, max_len: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_tofazen_create(ctx: *mut tq_ctx, cfg: *const tq_tofazen_config, layers: *const tq_tofazen_layer, out: *mut *mut tq_tofazen) -> c_int;
    pub fn tq_tofazen_destroy(model: *mut tq_tofazen) -> c_int;
    pub fn tq_tofazen_put(model: *mut tq_tofazen, tensor: c_int, layer: usize, src: *const c_void, src_dtype: c_int, rows: usize, cols: usize) -> c_int;
    pub fn tq_tofazen_step(model: *mut tq_tofazen, token_ids_dev: *const c_int, rows: usize, seq_rows_dev_or_null: *const c_int, starts_dev: *const c_int, slots_dev_or_null: *const c_int, n_seqs: usize, max_q: usize, max_len: usize, logit_rows_dev_or_null: *const c_int, n_logits: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_tofazen_hidden(model: *mut tq_tofazen, hidden_dev: *mut *mut f32) -> c_int;
    pub fn tq_tofazen_trace(model: *mut tq_tofazen, streams_dev_or_null: *mut f32) -> c_int;
    pub fn tq_yarn_frequencies(dims: usize, base: f64, factor: f64, original: f64, fast: f64, slow: f64, freq_host: *mut f32, mult_host: *mut f32) -> c_int;
    pub fn tq_add_norm(ctx: *mut tq_ctx, x_dev: *mut f32, y_dev_or_null: *const f32, y_rows_dev_or_null: *const c_int, n_y: usize, gain_post_dev_or_null: *const f32, gain_next_dev_or_null: *const f32, rows: usize, width: usize, eps: f32, out_dev_or_null: *mut c_void, out_dtype: c_int, ld_out: usize) -> c_int;
    pub fn tq_qk_norm_rope(ctx: *mut tq_ctx, dtype: c_int, heads: usize, kv_heads: usize, dim: usize, q_dev: *mut c_void, ldq: usize, raw_dev: *const c_void, keys_dev: *mut c_void, cache_rows: usize, q_gain_dev: *const c_void, k_gain_dev: *const c_void, rot_dims: usize, freq_dev: *const f32, rot_mult: f32, eps: f32, row_pos_dev: *const c_int, cache_row_dev: *const c_int, rows: usize) -> c_int;
    pub fn tq_head_norm_rope(ctx: *mut tq_ctx, dtype: c_int, heads: usize, kv_heads: usize, dim: usize, q_dev: *mut c_void, ldq: usize, q_head: usize, raw_dev_or_null: *const c_void, keys_dev_or_null: *mut c_void, cache_rows: usize, q_gain_dev_or_null: *const c_void, k_gain_dev_or_null: *const c_void, rot_first: usize, rot_dims: usize, interleaved: c_int, freq_dev: *const f32, rot_mult: f32, eps: f32, row_pos_dev: *const c_int, cache_row_dev: *const c_int, rows: usize) -> c_int;
    pub fn tq_banded_frequencies(dims: usize, base: f64, factor: f64, low: f64, high: f64, original: f64, freq_host: *mut f32) -> c_int;
    pub fn tq_stream_mix(ctx: *mut tq_ctx, streams: usize, src_streams: usize, src_dev: *const f32, dst_dev_or_null: *mut f32, y_dev_or_null: *const f32, y_rows_dev_or_null: *const c_int, y_weight_dev_or_null: *const f32, n_y: usize, self_dev_or_null: *const c_void, y_more_dev_or_null: *const f32, mix_dev_or_null: *const f32, w_out_dev_or_null: *const f32, w_in_dev_or_null: *const f32, gain_dev_or_null: *const f32, rows: usize, width: usize, eps: f32, out_dev_or_null: *mut c_void, out_dtype: c_int, ld_out: usize, sum_dev_or_null: *mut f32) -> c_int;
    pub fn tq_stream_step(ctx: *mut tq_ctx, src_dev: *const f32, dst_dev: *mut f32, y_dev: *const f32, y_rows_dev_or_null: *const c_int, y_weight_dev_or_null: *const f32, n_y: usize, y_more_dev_or_null: *const f32, y_more_gate_dev_or_null: *const f32, ld_gate: usize, inject_dev_or_null: *const f32, mix_one_dev: *const f32, w_out_dev: *const f32, gain_dev: *const f32, rows: usize, width: usize, eps: f32, conv_w_dev_or_null: *const f32, conv_state_dev_or_null: *mut c_void, taps: usize, max_seq: usize, row_pos_dev: *const c_int, cache_row_dev: *const c_int, out_dev: *mut c_void, out_dtype: c_int, ld_out: usize, sum_dev_or_null: *mut f32) -> c_int;
    pub fn tq_window_attention(ctx: *mut tq_ctx, cfg: *const tq_window_attn_config, dtype: c_int, q_dev: *const c_void, ldq: usize, gate_dev_or_null: *const c_void, ldg: usize, k_cache_dev: *const c_void, v_cache_dev: *const c_void, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, max_len: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_window_attention_sinks(ctx: *mut tq_ctx, cfg: *const tq_window_attn_config, sinks_dev_or_null: *const f32, dtype: c_int, q_dev: *const c_void, ldq: usize, gate_dev_or_null: *const c_void, ldg: usize, k_cache_dev: *const c_void, v_cache_dev: *const c_void, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, max_len: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_window_attention_pooled(ctx: *mut tq_ctx, cfg: *const tq_window_attn_config, sinks_dev_or_null: *const f32, dtype: c_int, q_dev: *const c_void, ldq: usize, gate_dev_or_null: *const c_void, ldg: usize, k_cache_dev: *const c_void, v_cache_dev: *const c_void, cache_rows: usize, pool: usize, pooled_keys_dev_or_null: *const c_void, pooled_values_dev_or_null: *const c_void, pool_rows: usize, max_seq: usize, out_scale: f32, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, max_len: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_conv_residual(ctx: *mut tq_ctx, dtype: c_int, channels: usize, taps: usize, w_dev: *const f32, state_dev: *mut c_void, max_seq: usize, cache_rows: usize, x_dev: *const c_void, ldx: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, max_len: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_conv_heads(ctx: *mut tq_ctx, cfg: *const tq_conv_heads_config, dtype: c_int, raw_dev: *const c_void, ld: usize, w_dev_or_null: *const f32, state_dev_or_null: *mut c_void, freq_dev_or_null: *const f32, max_seq: usize, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, max_len: usize, q_dev: *mut c_void, ldq: usize, keys_dev: *mut c_void, values_dev: *mut c_void, pooled_keys_dev_or_null: *mut c_void, pooled_values_dev_or_null: *mut c_void) -> c_int;
    pub fn tq_min_gru(ctx: *mut tq_ctx, dtype: c_int, width: usize, z_dev: *const c_void, u_dev: *const c_void, gate_dev: *const c_void, ld: usize, z_bias_dev: *const f32, u_bias_dev: *const f32, out_scale: f32, state_dev: *mut f32, max_seq: usize, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_gla(ctx: *mut tq_ctx, cfg: *const tq_gla_config, dtype: c_int, q_dev: *const c_void, k_dev: *const c_void, v_dev: *const c_void, gate_dev: *const c_void, ld: usize, a1_dev: *const f32, ld_a1: usize, a2_dev: *const f32, a2_bias_dev: *const f32, norm_dev: *const f32, state_dev: *mut f32, max_seq: usize, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_lightning(ctx: *mut tq_ctx, dtype: c_int, heads: usize, dim: usize, vdim: usize, eps: f32, decay_dev: *const f32, q_dev: *const c_void, k_dev: *const c_void, v_dev: *const c_void, gate_dev: *const c_void, ld: usize, norm_dev: *const f32, state_dev: *mut f32, max_seq: usize, cache_rows: usize, seq_rows_dev_or_null: *const c_int, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, rows: usize, max_q: usize, out_dev: *mut c_void, ldo: usize) -> c_int;
    pub fn tq_latent_decode(ctx: *mut tq_ctx, heads: usize, dim: usize, rot: usize, rank: usize, scale: f32, rot_dims: usize, freq_dev: *const f32, rot_mult: f32, rotate: c_int, q_lat_dev: *const c_void, q_dev: *const c_void, ldq: usize, cache_dev: *const c_void, cache_rows: usize, row_pos_dev: *const c_int, cache_row_dev: *const c_int, n_seqs: usize, max_len: usize, out_dev: *mut c_void) -> c_int;
    pub fn tq_route(ctx: *mut tq_ctx, logits_dev: *const f32, rows: usize, experts: usize, top: usize, score: c_int, renorm: c_int, chunk: usize, expert_dev: *mut c_int, weight_dev: *mut f32, slot_dev: *mut c_int, slot_row_dev: *mut c_int, jobs_dev: *mut c_int, n_jobs_dev: *mut c_int) -> c_int;
    pub fn tq_route_rule(ctx: *mut tq_ctx, logits_dev: *const f32, rows: usize, experts: usize, top: usize, score: c_int, renorm: c_int, correction_dev_or_null: *const f32, identity: usize, chunk: usize, expert_dev: *mut c_int, weight_dev: *mut f32, slot_dev: *mut c_int, slot_row_dev: *mut c_int, jobs_dev: *mut c_int, n_jobs_dev: *mut c_int) -> c_int;
    pub fn tq_route_biased(ctx: *mut tq_ctx, logits_dev: *const f32, ld: usize, rows: usize, experts: usize, top: usize, score: c_int, renorm: c_int, bias_dev_or_null: *const f32, correction_dev_or_null: *const f32, identity: usize, chunk: usize, expert_dev: *mut c_int, weight_dev: *mut f32, slot_dev: *mut c_int, slot_row_dev: *mut c_int, jobs_dev: *mut c_int, n_jobs_dev: *mut c_int) -> c_int;
    pub fn tq_numuzen_create(ctx: *mut tq_ctx, cfg: *const tq_numuzen_config, layers: *const tq_numuzen_layer, out: *mut *mut tq_numuzen) -> c_int;
    pub fn tq_numuzen_destroy(model: *mut tq_numuzen) -> c_int;
    pub fn tq_numuzen_put(model: *mut tq_numuzen, tensor: c_int, layer: usize, expert: usize, src: *const c_void, src_dtype: c_int, rows: usize, cols: usize) -> c_int;
    pub fn tq_numuzen_step(model: *mut tq_numuzen, token_ids_dev: *const c_int, rows: usize, seq_rows_dev_or_null: *const c_int, starts_dev: *const c_int, slots_dev_or_null: *const c_int, n_seqs: usize, max_q: usize, max_len: usize, logit_rows_dev_or_null: *const c_int, n_logits: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_numuzen_hidden(model: *mut tq_numuzen, hidden_dev: *mut *mut f32) -> c_int;
    pub fn tq_numuzen_trace(model: *mut tq_numuzen, streams_dev_or_null: *mut f32) -> c_int;
    pub fn tq_dotanex_create(ctx: *mut tq_ctx, cfg: *const tq_dotanex_config, layers: *const tq_dotanex_layer, out: *mut *mut tq_dotanex) -> c_int;
    pub fn tq_dotanex_destroy(model: *mut tq_dotanex) -> c_int;
    pub fn tq_dotanex_put(model: *mut tq_dotanex, tensor: c_int, layer: usize, expert: usize, src: *const c_void, src_dtype: c_int, rows: usize, cols: usize) -> c_int;
    pub fn tq_dotanex_step(model: *mut tq_dotanex, token_ids_dev: *const c_int, rows: usize, seq_rows_dev_or_null: *const c_int, starts_dev: *const c_int, slots_dev_or_null: *const c_int, n_seqs: usize, max_q: usize, max_len: usize, logit_rows_dev_or_null: *const c_int, n_logits: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_dotanex_trace(model: *mut tq_dotanex, sums_dev_or_null: *mut f32) -> c_int;
    pub fn tq_sakinex_create(ctx: *mut tq_ctx, cfg: *const tq_sakinex_config, layers: *const tq_sakinex_layer, out: *mut *mut tq_sakinex) -> c_int;
    pub fn tq_sakinex_destroy(model: *mut tq_sakinex) -> c_int;
    pub fn tq_sakinex_put(model: *mut tq_sakinex, tensor: c_int, layer: usize, expert: usize, src: *const c_void, src_dtype: c_int, rows: usize, cols: usize) -> c_int;
    pub fn tq_sakinex_step(model: *mut tq_sakinex, token_ids_dev: *const c_int, rows: usize, seq_rows_dev_or_null: *const c_int, starts_dev: *const c_int, slots_dev_or_null: *const c_int, n_seqs: usize, max_q: usize, max_len: usize, logit_rows_dev_or_null: *const c_int, n_logits: usize, logits_dev: *mut f32) -> c_int;
    pub fn tq_sakinex_trace(model: *mut tq_sakinex, streams_dev_or_null: *mut f32) -> c_int;
    pub fn tq_graph_begin(ctx: *mut tq_ctx) -> c_int;
    pub fn tq_graph_end(ctx: *mut tq_ctx, out: *mut *mut tq_graph) -> c_int;
    pub fn tq_graph_launch(ctx: *mut tq_ctx, graph: *mut tq_graph) -> c_int;
    pub fn tq_graph_free(ctx: *mut tq_ctx, graph: *mut tq_graph) -> c_int;
    pub fn tq_launch_count(ctx: *const tq_ctx) -> u64;
}
