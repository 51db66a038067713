// Generated by gen_bindings.py from include/runit_hip.h; do not edit.
#![allow(non_camel_case_types, clippy::too_many_arguments)]
use std::os::raw::{c_char, c_int, c_void};

#[repr(C)] pub struct RtCtx { _p: [u8; 0] }
#[repr(C)] pub struct RtEvent { _p: [u8; 0] }
#[repr(C)] pub struct RtGraph { _p: [u8; 0] }
#[repr(C)] pub struct RtGguf { _p: [u8; 0] }
#[repr(C)] pub struct RtStep { _p: [u8; 0] }

/// rt_step_layer (include/runit_hip.h)
#[repr(C)] #[derive(Clone, Copy)]
pub struct RtStepLayer {
    pub wq: *const c_void, pub wk: *const c_void, pub wv: *const c_void,
    pub wo: *const c_void, pub wg: *const c_void, pub wu: *const c_void,
    pub wd: *const c_void,
    pub bq: *const u16, pub bk: *const u16, pub bv: *const u16,
    pub attn_norm: *const f32, pub ffn_norm: *const f32,
    pub k_cache: *mut f32, pub v_cache: *mut f32,
}
/// rt_step_model (include/runit_hip.h)
#[repr(C)]
pub struct RtStepModel {
    pub layers: u32, pub hidden: u32, pub heads: u32, pub kv_heads: u32,
    pub head_dim: u32, pub ff: u32, pub vocab: u32, pub max_seq: u32,
    pub eps: f32, pub theta: f32,
    pub layer: *const RtStepLayer,
    pub token_embd: *const c_void, pub lm_head: *const c_void,
    pub output_norm: *const f32, pub token: *mut u32, pub logits: *mut f32,
}
/// rt_paged_batch (include/runit_hip.h)
#[repr(C)] #[derive(Clone, Copy)]
pub struct RtPagedBatch {
    pub k_pages: *mut c_void, pub v_pages: *mut c_void,
    pub f16: u32, pub num_pages: u32, pub page_size: u32, pub num_kv_heads: u32,
    pub head_dim: u32, pub table_stride: u32, pub n_seqs: u32, pub rows: u32,
    pub page_stride: u64,
    pub table: *const u32, pub row_start: *const u32, pub kv_len: *const u32,
}

extern "C" {
    pub fn rt_ctx_create(out: *mut *mut RtCtx, code_object_path: *const c_char) -> c_int;
    pub fn rt_ctx_destroy(ctx: *mut RtCtx);
    pub fn rt_flush(ctx: *mut RtCtx) -> c_int;
    pub fn rt_last_error(ctx: *const RtCtx) -> *const c_char;
    pub fn rt_global_last_error() -> *const c_char;
    pub fn rt_device_cu_count(ctx: *const RtCtx) -> c_int;
    pub fn rt_has_kernel(ctx: *mut RtCtx, name: *const c_char) -> c_int;
    pub fn rt_malloc(ctx: *mut RtCtx, bytes: usize, out: *mut *mut c_void) -> c_int;
    pub fn rt_free(ctx: *mut RtCtx, ptr: *mut c_void) -> c_int;
    pub fn rt_upload(ctx: *mut RtCtx, dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> c_int;
    pub fn rt_download(ctx: *mut RtCtx, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> c_int;
    pub fn rt_memset(ctx: *mut RtCtx, dst_dev: *mut c_void, value: c_int, bytes: usize) -> c_int;
    pub fn rt_copy_d2d(ctx: *mut RtCtx, dst_dev: *mut c_void, src_dev: *const c_void, bytes: usize) -> c_int;
    pub fn rt_event_create(ctx: *mut RtCtx, out: *mut *mut RtEvent) -> c_int;
    pub fn rt_event_record(ctx: *mut RtCtx, ev: *mut RtEvent) -> c_int;
    pub fn rt_event_elapsed_ms(ctx: *mut RtCtx, start: *mut RtEvent, stop: *mut RtEvent, ms: *mut f32) -> c_int;
    pub fn rt_event_destroy(ev: *mut RtEvent);
    pub fn rt_capture_begin(ctx: *mut RtCtx) -> c_int;
    pub fn rt_capture_end(ctx: *mut RtCtx, out: *mut *mut RtGraph) -> c_int;
    pub fn rt_graph_launch(ctx: *mut RtCtx, g: *mut RtGraph) -> c_int;
    pub fn rt_graph_destroy(g: *mut RtGraph);
    pub fn rt_gemv_q8_0_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_add_f32_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_f16(ctx: *mut RtCtx, weight: *const c_void, input: *const u16, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_add_f16(ctx: *mut RtCtx, weight: *const c_void, input: *const u16, output: *mut u16, residual: *const u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_add_f32res_f16(ctx: *mut RtCtx, weight: *const c_void, input: *const u16, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_f32in_f32out_mr(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_add_f32_f32in_mr(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0_add_f32_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0_f16(ctx: *mut RtCtx, weight: *const c_void, input: *const u16, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0_add_f16(ctx: *mut RtCtx, weight: *const c_void, input: *const u16, output: *mut u16, residual: *const u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4k_f32in_f32out(ctx: *mut RtCtx, weight_q4k: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4k_add_f32_f32in(ctx: *mut RtCtx, weight_q4k: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4k_f16(ctx: *mut RtCtx, weight_q4k: *const c_void, input: *const u16, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4k_add_f16(ctx: *mut RtCtx, weight_q4k: *const c_void, input: *const u16, output: *mut u16, residual: *const u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4k_add_f32res_f16(ctx: *mut RtCtx, weight_q4k: *const c_void, input: *const u16, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6k_f32in_f32out(ctx: *mut RtCtx, weight_q6k: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6k_add_f32_f32in(ctx: *mut RtCtx, weight_q6k: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6k_f32in(ctx: *mut RtCtx, weight_q6k: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6k_add_f32_f32in_noalloc(ctx: *mut RtCtx, weight_q6k: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5_0_f32in_f32out(ctx: *mut RtCtx, weight_q5_0: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5_0_add_f32_f32in(ctx: *mut RtCtx, weight_q5_0: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5_0_f32in(ctx: *mut RtCtx, weight_q5_0: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5k_f32in_f32out(ctx: *mut RtCtx, weight_q5k: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5k_add_f32_f32in(ctx: *mut RtCtx, weight_q5k: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5k_f32in(ctx: *mut RtCtx, weight_q5k: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0g_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0g_add_f32_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4_0g_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4kg_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4kg_add_f32_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q4kg_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5kg_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5kg_add_f32_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q5kg_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6kg_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6kg_add_f32_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q6kg_f32in(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut u16, m: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q4_0g_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q4kg_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q5kg_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_dequant_q4_0g_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q4kg_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q5kg_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q6kg_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_fused_qkv_q8_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q8_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q4_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q4k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q4k_q6k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q4kg_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q4kg_q6kg_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q8_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q4_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q4k_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q5_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_qkv_bias_q5k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x_vec: *const f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q5_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_q5k_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x_vec: *const f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_dequant_q8_0_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q4_0_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q4k_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q6k_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q5_0_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q5k_f32(ctx: *mut RtCtx, input: *const c_void, output: *mut f32, n_blocks: u32) -> c_int;
    pub fn rt_dequant_q4k_f16(ctx: *mut RtCtx, input: *const c_void, output: *mut u16, n_blocks: u32) -> c_int;
    pub fn rt_gemm_q8_0_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q4_0_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q4k_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q5_0_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q5k_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q6k_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q4_0g_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q4kg_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q5kg_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_q6kg_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, y: *mut f32, m_rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemm_set_f32(ctx: *mut RtCtx, count: u32, fmts: *const *const c_char, weight: *const *const c_void, y: *const *mut f32, n: *const u32, bias: *const *const u16, res: *const f32, x: *const f32, m_rows: u32, k: u32, gamma: *const f32, eps: f32, xn: *mut f32, silu_pair: u32) -> c_int;
    pub fn rt_gemm_qkv_rope_f32(ctx: *mut RtCtx, fmt_q: *const c_char, w_q: *const c_void, fmt_k: *const c_char, w_k: *const c_void, fmt_v: *const c_char, w_v: *const c_void, b_q: *const u16, b_k: *const u16, b_v: *const u16, x: *const f32, gamma: *const f32, eps: f32, xn: *mut f32, q: *mut f32, k: *mut f32, v: *mut f32, k_cache: *mut f32, v_cache: *mut f32, m_rows: u32, hidden: u32, q_dim: u32, kv_dim: u32, head_dim: u32, start_pos: u32, theta: f32, max_seq: u32) -> c_int;
    pub fn rt_gemm_ffn_block_f32(ctx: *mut RtCtx, fmt_o: *const c_char, w_o: *const c_void, fmt_gate: *const c_char, w_gate: *const c_void, fmt_up: *const c_char, w_up: *const c_void, fmt_down: *const c_char, w_down: *const c_void, att: *const f32, x: *mut f32, x_mid: *mut f32, gamma: *const f32, eps: f32, g: *mut f32, u: *mut f32, xn: *mut f32, m_rows: u32, h: u32, qd: u32, ff: u32) -> c_int;
    pub fn rt_gemm_attn_ffn_block_f32(ctx: *mut RtCtx, q: *const f32, k_cache: *const f32, v_cache: *const f32, kv_len: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, kv_head_stride: u32, q_start: u32, att: *mut f32, fmt_o: *const c_char, w_o: *const c_void, fmt_gate: *const c_char, w_gate: *const c_void, fmt_up: *const c_char, w_up: *const c_void, fmt_down: *const c_char, w_down: *const c_void, x: *mut f32, x_mid: *mut f32, gamma: *const f32, eps: f32, g: *mut f32, u: *mut f32, xn: *mut f32, m_rows: u32, h: u32, ff: u32) -> c_int;
    pub fn rt_gemv_rows_q8_0_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q8_0_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q8_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q8_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4_0_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4_0_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q4_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q4_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4k_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4k_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q4k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q4k_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q6k_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q6k_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q6k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q6k_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q5_0_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q5_0_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q5_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q5_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q5k_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q5k_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q5k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q5k_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4_0g_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4_0g_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q4_0g_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q4_0g_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4kg_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q4kg_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q4kg_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q4kg_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q5kg_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q5kg_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q5kg_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q5kg_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q6kg_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_gemv_rows_q6kg_add_f32(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, res: *const f32, y: *mut f32, rows: u32, n: u32, k: u32) -> c_int;
    pub fn rt_qkv_bias_rows_q6kg_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, q: *mut f32, k_out: *mut f32, v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_fused_ffn_rows_q6kg_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act: *mut f32, rows: u32, ff: u32, k: u32) -> c_int;
    pub fn rt_argmax_f32(ctx: *mut RtCtx, input: *const f32, result: *mut u32, n: u32) -> c_int;
    pub fn rt_argmax_f16(ctx: *mut RtCtx, input: *const u16, result: *mut u32, n: u32) -> c_int;
    pub fn rt_synth_normal_f32(ctx: *mut RtCtx, out: *mut f32, n: u64, seed: u64, mean: f32, std: f32) -> c_int;
    pub fn rt_synth_normal_f16(ctx: *mut RtCtx, out: *mut u16, n: u64, seed: u64, mean: f32, std: f32) -> c_int;
    pub fn rt_synth_q8_0(ctx: *mut RtCtx, out: *mut c_void, n_blocks: u64, seed: u64, std: f32) -> c_int;
    pub fn rt_synth_q4_0(ctx: *mut RtCtx, out: *mut c_void, n_blocks: u64, seed: u64, std: f32) -> c_int;
    pub fn rt_synth_q4k(ctx: *mut RtCtx, out: *mut c_void, n_blocks: u64, seed: u64, std: f32) -> c_int;
    pub fn rt_synth_q6k(ctx: *mut RtCtx, out: *mut c_void, n_blocks: u64, seed: u64, std: f32) -> c_int;
    pub fn rt_synth_q5_0(ctx: *mut RtCtx, out: *mut c_void, n_blocks: u64, seed: u64, std: f32) -> c_int;
    pub fn rt_synth_q5k(ctx: *mut RtCtx, out: *mut c_void, n_blocks: u64, seed: u64, std: f32) -> c_int;
    pub fn rt_rms_norm_f32_f32_f32g(ctx: *mut RtCtx, x: *const f32, y: *mut f32, gamma: *const f32, eps: f32, hidden: u32, num_rows: u32) -> c_int;
    pub fn rt_fused_rope_qk_f32(ctx: *mut RtCtx, q: *mut f32, k: *mut f32, head_dim: u32, q_heads: u32, kv_heads: u32, pos: u32, theta: f32) -> c_int;
    pub fn rt_kv_copy_to_cache_f32(ctx: *mut RtCtx, src: *const f32, dst: *mut f32, pos: u32, max_seq: u32, head_dim: u32, num_kv_heads: u32) -> c_int;
    pub fn rt_decode_attention_f32(ctx: *mut RtCtx, q: *const f32, k: *const f32, v: *const f32, out: *mut f32, batch: u32, kv_len: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, kv_head_stride: u32) -> c_int;
    pub fn rt_decode_attention_rope_f32(ctx: *mut RtCtx, q_raw: *const f32, k_raw: *const f32, v_raw: *const f32, k_cache: *mut f32, v_cache: *mut f32, out: *mut f32, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32) -> c_int;
    pub fn rt_decode_attention_rope_oproj_q8_0_f32(ctx: *mut RtCtx, q_raw: *const f32, k_raw: *const f32, v_raw: *const f32, k_cache: *mut f32, v_cache: *mut f32, w_o: *const c_void, x_io: *mut f32, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32) -> c_int;
    pub fn rt_decode_attention_rope_oproj_q4k_f32(ctx: *mut RtCtx, q_raw: *const f32, k_raw: *const f32, v_raw: *const f32, k_cache: *mut f32, v_cache: *mut f32, w_o: *const c_void, x_io: *mut f32, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32) -> c_int;
    pub fn rt_decode_attention_rope_oproj_q4kg_f32(ctx: *mut RtCtx, q_raw: *const f32, k_raw: *const f32, v_raw: *const f32, k_cache: *mut f32, v_cache: *mut f32, w_o: *const c_void, x_io: *mut f32, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32) -> c_int;
    pub fn rt_launch_count(ctx: *const RtCtx) -> u64;
    pub fn rt_last_launch_name(ctx: *const RtCtx) -> *const c_char;
    pub fn rt_add_f16_into_f32(ctx: *mut RtCtx, src: *const u16, acc: *mut f32, n: u32) -> c_int;
    pub fn rt_add_bias_broadcast_f32(ctx: *mut RtCtx, x: *mut f32, bias: *const u16, seq: u32, dim: u32) -> c_int;
    pub fn rt_rope_batch_inplace_f32(ctx: *mut RtCtx, x: *mut f32, head_dim: u32, num_heads: u32, start_pos: u32, theta: f32, seq: u32) -> c_int;
    pub fn rt_rope_kv_write_batch_f32(ctx: *mut RtCtx, q: *mut f32, k: *const f32, v: *const f32, k_cache: *mut f32, v_cache: *mut f32, head_dim: u32, num_heads: u32, num_kv_heads: u32, start_pos: u32, theta: f32, seq: u32, max_seq: u32) -> c_int;
    pub fn rt_kv_write_batch_f32(ctx: *mut RtCtx, k: *const f32, v: *const f32, k_cache: *mut f32, v_cache: *mut f32, start_pos: u32, seq: u32, max_seq: u32, head_dim: u32, num_kv_heads: u32) -> c_int;
    pub fn rt_flash_attention_f32(ctx: *mut RtCtx, q: *const f32, k: *const f32, v: *const f32, out: *mut f32, batch: u32, q_len: u32, kv_len: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, kv_head_stride: u32, q_start: u32) -> c_int;
    pub fn rt_add_f32(ctx: *mut RtCtx, a: *const f32, b: *const f32, out: *mut f32, n: u32) -> c_int;
    pub fn rt_silu_mul_f32(ctx: *mut RtCtx, gate: *const f32, up: *const f32, out: *mut f32, n: u32) -> c_int;
    pub fn rt_argmax_rows_first_f32(ctx: *mut RtCtx, in_: *const f32, result: *mut u32, rows: u32, n: u32) -> c_int;
    pub fn rt_rope_kv_append_paged_f32(ctx: *mut RtCtx, batch: *const RtPagedBatch, q: *const f32, k: *const f32, v: *const f32, q_out: *mut f32, num_heads: u32, theta: f32) -> c_int;
    pub fn rt_paged_attention_f32(ctx: *mut RtCtx, batch: *const RtPagedBatch, q: *const f32, out: *mut f32, num_heads: u32) -> c_int;
    pub fn rt_shared_prefix_attention_f32(ctx: *mut RtCtx, batch: *const RtPagedBatch, q: *const f32, out: *mut f32, num_heads: u32, shared_table: *const u32, shared_len: u32) -> c_int;
    pub fn rt_token_logprobs_f32(ctx: *mut RtCtx, logits: *const f32, tokens: *const u32, rows: u32, n: u32, row_stride: u64, logprob: *mut f32, entropy: *mut f32, rank: *mut u32, top: u32, top_ids: *mut u32, top_logprobs: *mut f32) -> c_int;
    pub fn rt_token_logprobs_f16(ctx: *mut RtCtx, logits: *const u16, tokens: *const u32, rows: u32, n: u32, row_stride: u64, logprob: *mut f32, entropy: *mut f32, rank: *mut u32, top: u32, top_ids: *mut u32, top_logprobs: *mut f32) -> c_int;
    pub fn rt_embed_q8_0_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q4_0_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q4k_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q6k_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q5_0_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q5k_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q4_0g_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q4kg_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q5kg_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_q6kg_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_f16_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_f32_f32(ctx: *mut RtCtx, table: *const c_void, token: *const u32, out: *mut f32, k: u32) -> c_int;
    pub fn rt_embed_rows_q8_0_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q4_0_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q4k_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q6k_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q5_0_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q5k_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q4_0g_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q4kg_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q5kg_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_q6kg_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_f16_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_embed_rows_f32_f32(ctx: *mut RtCtx, table: *const c_void, tokens: *const u32, out: *mut f32, k: u32, rows: u32) -> c_int;
    pub fn rt_rms_norm_fused_qkv_bias_q8_0_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_rms_norm_fused_ffn_q8_0_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_rms_norm_gemv_q8_0_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_gemv_q8_0_add_f32_f32in_ssq(ctx: *mut RtCtx, weight: *const c_void, input: *const f32, output: *mut f32, residual: *const f32, m: u32, k: u32, ssq: *mut f32) -> c_int;
    pub fn rt_decode_attention_rope_oproj_q8_0_f32_ssq(ctx: *mut RtCtx, q_raw: *const f32, k_raw: *const f32, v_raw: *const f32, k_cache: *mut f32, v_cache: *mut f32, w_o: *const c_void, x_io: *mut f32, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32, ssq: *mut f32) -> c_int;
    pub fn rt_rms_norm_fused_qkv_bias_q8_0_f32_ssq(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32, ssq: *const f32, nparts: u32) -> c_int;
    pub fn rt_rms_norm_fused_ffn_q8_0_f32_ssq(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act_out: *mut f32, ff_dim: u32, k: u32, ssq: *const f32, nparts: u32) -> c_int;
    pub fn rt_rms_norm_fused_qkv_bias_q4k_q6k_f32(ctx: *mut RtCtx, w_q: *const c_void, w_k: *const c_void, w_v: *const c_void, x: *const f32, gamma: *const f32, eps: f32, out_q: *mut f32, out_k: *mut f32, out_v: *mut f32, bias_q: *const u16, bias_k: *const u16, bias_v: *const u16, q_dim: u32, kv_dim: u32, k: u32) -> c_int;
    pub fn rt_rms_norm_fused_ffn_q4k_f32(ctx: *mut RtCtx, w_gate: *const c_void, w_up: *const c_void, x: *const f32, gamma: *const f32, eps: f32, act_out: *mut f32, ff_dim: u32, k: u32) -> c_int;
    pub fn rt_rms_norm_gemv_q6k_f32in_f32out(ctx: *mut RtCtx, weight: *const c_void, x: *const f32, gamma: *const f32, eps: f32, output: *mut f32, m: u32, k: u32) -> c_int;
    pub fn rt_stream_read(ctx: *mut RtCtx, src: *const c_void, bytes: usize, sink: *mut u32, sink_dwords: usize) -> c_int;
    pub fn rt_stream_copy(ctx: *mut RtCtx, dst: *mut c_void, src: *const c_void, bytes: usize) -> c_int;
    pub fn rt_gguf_open(path: *const c_char, out: *mut *mut RtGguf) -> c_int;
    pub fn rt_gguf_close(g: *mut RtGguf);
    pub fn rt_gguf_last_error() -> *const c_char;
    pub fn rt_gguf_version(g: *const RtGguf) -> u32;
    pub fn rt_gguf_alignment(g: *const RtGguf) -> u64;
    pub fn rt_gguf_data_offset(g: *const RtGguf) -> u64;
    pub fn rt_gguf_tensor_count(g: *const RtGguf) -> u64;
    pub fn rt_gguf_find_tensor(g: *const RtGguf, name: *const c_char) -> i64;
    pub fn rt_gguf_tensor_info(g: *const RtGguf, i: u64, name: *mut *const c_char, n_dims: *mut u32, dims: *mut u64, dtype: *mut u32, offset: *mut u64, bytes: *mut u64) -> c_int;
    pub fn rt_gguf_tensor_data(g: *const RtGguf, i: u64) -> *const c_void;
    pub fn rt_gguf_upload(ctx: *mut RtCtx, g: *const RtGguf, i: u64, dst_dev: *mut c_void) -> c_int;
    pub fn rt_gguf_meta_count(g: *const RtGguf) -> u64;
    pub fn rt_gguf_find_meta(g: *const RtGguf, key: *const c_char) -> i64;
    pub fn rt_gguf_meta_info(g: *const RtGguf, i: u64, key: *mut *const c_char, type_: *mut u32, elem_type: *mut u32, count: *mut u64) -> c_int;
    pub fn rt_gguf_meta_int(g: *const RtGguf, i: u64, out: *mut i64) -> c_int;
    pub fn rt_gguf_meta_float(g: *const RtGguf, i: u64, out: *mut f64) -> c_int;
    pub fn rt_gguf_meta_string(g: *const RtGguf, i: u64) -> *const c_char;
    pub fn rt_gguf_meta_array_numbers(g: *const RtGguf, i: u64, out: *mut f64, max: u64) -> c_int;
    pub fn rt_gguf_meta_array_string(g: *const RtGguf, i: u64, k: u64, s: *mut *const c_char, len: *mut u64) -> c_int;
    pub fn rt_decode_step_q8_0_create(ctx: *mut RtCtx, model: *const RtStepModel, pos: u32, out: *mut *mut RtStep) -> c_int;
    pub fn rt_decode_step_run(ctx: *mut RtCtx, step: *mut RtStep) -> c_int;
    pub fn rt_decode_step_status(ctx: *mut RtCtx, step: *mut RtStep) -> c_int;
    pub fn rt_decode_step_destroy(step: *mut RtStep);
}
