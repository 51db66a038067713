// Generated by gen_bindings.py from include/runit_hip.h; do not edit.
//! The reference's `dispatch::*` surface (crates/kernels/src/dispatch.rs) over the
//! C ABI: one wrapper per kernel entry point, same names and argument order.
#![allow(clippy::too_many_arguments)]
use crate::{ffi, status, Buffer, HipContext, Result};
use std::os::raw::c_void;

pub fn gemv_q8_0_f32in_f32out(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q8_0_add_f32_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_add_f32_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q8_0_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q8_0_f16(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_f16(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q8_0_add_f16(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_add_f16(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut u16, residual.as_ptr() as *const u16, m, k) })
}
pub fn gemv_q8_0_add_f32res_f16(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_add_f32res_f16(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q8_0_f32in_f32out_mr(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_f32in_f32out_mr(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q8_0_add_f32_f32in_mr(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_add_f32_f32in_mr(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q4_0_f32in_f32out(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q4_0_add_f32_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0_add_f32_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q4_0_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q4_0_f16(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0_f16(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q4_0_add_f16(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0_add_f16(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut u16, residual.as_ptr() as *const u16, m, k) })
}
pub fn gemv_q4k_f32in_f32out(ctx: &HipContext, weight_q4k: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4k_f32in_f32out(ctx.raw(), weight_q4k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q4k_add_f32_f32in(ctx: &HipContext, weight_q4k: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4k_add_f32_f32in(ctx.raw(), weight_q4k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q4k_f16(ctx: &HipContext, weight_q4k: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4k_f16(ctx.raw(), weight_q4k.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q4k_add_f16(ctx: &HipContext, weight_q4k: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4k_add_f16(ctx.raw(), weight_q4k.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut u16, residual.as_ptr() as *const u16, m, k) })
}
pub fn gemv_q4k_add_f32res_f16(ctx: &HipContext, weight_q4k: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4k_add_f32res_f16(ctx.raw(), weight_q4k.as_ptr() as *const c_void, input.as_ptr() as *const u16, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q6k_f32in_f32out(ctx: &HipContext, weight_q6k: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6k_f32in_f32out(ctx.raw(), weight_q6k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q6k_add_f32_f32in(ctx: &HipContext, weight_q6k: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6k_add_f32_f32in(ctx.raw(), weight_q6k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q6k_f32in(ctx: &HipContext, weight_q6k: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6k_f32in(ctx.raw(), weight_q6k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q6k_add_f32_f32in_noalloc(ctx: &HipContext, weight_q6k: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6k_add_f32_f32in_noalloc(ctx.raw(), weight_q6k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q5_0_f32in_f32out(ctx: &HipContext, weight_q5_0: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5_0_f32in_f32out(ctx.raw(), weight_q5_0.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q5_0_add_f32_f32in(ctx: &HipContext, weight_q5_0: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5_0_add_f32_f32in(ctx.raw(), weight_q5_0.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q5_0_f32in(ctx: &HipContext, weight_q5_0: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5_0_f32in(ctx.raw(), weight_q5_0.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q5k_f32in_f32out(ctx: &HipContext, weight_q5k: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5k_f32in_f32out(ctx.raw(), weight_q5k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q5k_add_f32_f32in(ctx: &HipContext, weight_q5k: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5k_add_f32_f32in(ctx.raw(), weight_q5k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q5k_f32in(ctx: &HipContext, weight_q5k: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5k_f32in(ctx.raw(), weight_q5k.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q4_0g_f32in_f32out(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0g_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q4_0g_add_f32_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0g_add_f32_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q4_0g_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4_0g_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q4kg_f32in_f32out(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4kg_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q4kg_add_f32_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4kg_add_f32_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q4kg_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q4kg_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q5kg_f32in_f32out(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5kg_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q5kg_add_f32_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5kg_add_f32_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q5kg_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q5kg_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn gemv_q6kg_f32in_f32out(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6kg_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q6kg_add_f32_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6kg_add_f32_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k) })
}
pub fn gemv_q6kg_f32in(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q6kg_f32in(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut u16, m, k) })
}
pub fn fused_ffn_q4_0g_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q4_0g_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn fused_ffn_q4kg_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q4kg_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn fused_ffn_q5kg_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q5kg_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn dequant_q4_0g_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q4_0g_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q4kg_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q4kg_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q5kg_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q5kg_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q6kg_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q6kg_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn fused_qkv_q8_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_q8_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q8_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q8_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q4_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q4_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q4k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q4k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q4k_q6k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q4k_q6k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q4kg_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q4kg_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q4kg_q6kg_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q4kg_q6kg_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_ffn_q8_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q8_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn fused_ffn_q4_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q4_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn fused_ffn_q4k_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q4k_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn fused_qkv_bias_q5_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q5_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_qkv_bias_q5k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x_vec: &Buffer, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_qkv_bias_q5k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn fused_ffn_q5_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q5_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn fused_ffn_q5k_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x_vec: &Buffer, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_q5k_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x_vec.as_ptr() as *const f32, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn dequant_q8_0_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q8_0_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q4_0_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q4_0_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q4k_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q4k_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q6k_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q6k_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q5_0_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q5_0_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q5k_f32(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q5k_f32(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut f32, n_blocks) })
}
pub fn dequant_q4k_f16(ctx: &HipContext, input: &Buffer, output: &Buffer, n_blocks: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_dequant_q4k_f16(ctx.raw(), input.as_ptr() as *const c_void, output.as_ptr() as *mut u16, n_blocks) })
}
pub fn gemm_q8_0_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q8_0_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q4_0_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q4_0_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q4k_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q4k_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q5_0_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q5_0_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q5k_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q5k_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q6k_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q6k_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q4_0g_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q4_0g_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q4kg_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q4kg_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q5kg_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q5kg_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_q6kg_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, y: &Buffer, m_rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_q6kg_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, y.as_ptr() as *mut f32, m_rows, n, k) })
}
pub fn gemm_qkv_rope_f32(ctx: &HipContext, fmt_q: &Buffer, w_q: &Buffer, fmt_k: &Buffer, w_k: &Buffer, fmt_v: &Buffer, w_v: &Buffer, b_q: &Buffer, b_k: &Buffer, b_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, xn: &Buffer, q: &Buffer, k: &Buffer, v: &Buffer, k_cache: &Buffer, v_cache: &Buffer, m_rows: u32, hidden: u32, q_dim: u32, kv_dim: u32, head_dim: u32, start_pos: u32, theta: f32, max_seq: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_qkv_rope_f32(ctx.raw(), fmt_q.as_ptr() as *const c_char, w_q.as_ptr() as *const c_void, fmt_k.as_ptr() as *const c_char, w_k.as_ptr() as *const c_void, fmt_v.as_ptr() as *const c_char, w_v.as_ptr() as *const c_void, b_q.as_ptr() as *const u16, b_k.as_ptr() as *const u16, b_v.as_ptr() as *const u16, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, xn.as_ptr() as *mut f32, q.as_ptr() as *mut f32, k.as_ptr() as *mut f32, v.as_ptr() as *mut f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, m_rows, hidden, q_dim, kv_dim, head_dim, start_pos, theta, max_seq) })
}
pub fn gemm_ffn_block_f32(ctx: &HipContext, fmt_o: &Buffer, w_o: &Buffer, fmt_gate: &Buffer, w_gate: &Buffer, fmt_up: &Buffer, w_up: &Buffer, fmt_down: &Buffer, w_down: &Buffer, att: &Buffer, x: &Buffer, x_mid: &Buffer, gamma: &Buffer, eps: f32, g: &Buffer, u: &Buffer, xn: &Buffer, m_rows: u32, h: u32, qd: u32, ff: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_ffn_block_f32(ctx.raw(), fmt_o.as_ptr() as *const c_char, w_o.as_ptr() as *const c_void, fmt_gate.as_ptr() as *const c_char, w_gate.as_ptr() as *const c_void, fmt_up.as_ptr() as *const c_char, w_up.as_ptr() as *const c_void, fmt_down.as_ptr() as *const c_char, w_down.as_ptr() as *const c_void, att.as_ptr() as *const f32, x.as_ptr() as *mut f32, x_mid.as_ptr() as *mut f32, gamma.as_ptr() as *const f32, eps, g.as_ptr() as *mut f32, u.as_ptr() as *mut f32, xn.as_ptr() as *mut f32, m_rows, h, qd, ff) })
}
pub fn gemm_attn_ffn_block_f32(ctx: &HipContext, q: &Buffer, k_cache: &Buffer, v_cache: &Buffer, kv_len: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, kv_head_stride: u32, q_start: u32, att: &Buffer, fmt_o: &Buffer, w_o: &Buffer, fmt_gate: &Buffer, w_gate: &Buffer, fmt_up: &Buffer, w_up: &Buffer, fmt_down: &Buffer, w_down: &Buffer, x: &Buffer, x_mid: &Buffer, gamma: &Buffer, eps: f32, g: &Buffer, u: &Buffer, xn: &Buffer, m_rows: u32, h: u32, ff: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemm_attn_ffn_block_f32(ctx.raw(), q.as_ptr() as *const f32, k_cache.as_ptr() as *const f32, v_cache.as_ptr() as *const f32, kv_len, num_heads, num_kv_heads, head_dim, kv_head_stride, q_start, att.as_ptr() as *mut f32, fmt_o.as_ptr() as *const c_char, w_o.as_ptr() as *const c_void, fmt_gate.as_ptr() as *const c_char, w_gate.as_ptr() as *const c_void, fmt_up.as_ptr() as *const c_char, w_up.as_ptr() as *const c_void, fmt_down.as_ptr() as *const c_char, w_down.as_ptr() as *const c_void, x.as_ptr() as *mut f32, x_mid.as_ptr() as *mut f32, gamma.as_ptr() as *const f32, eps, g.as_ptr() as *mut f32, u.as_ptr() as *mut f32, xn.as_ptr() as *mut f32, m_rows, h, ff) })
}
pub fn gemv_rows_q8_0_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q8_0_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q8_0_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q8_0_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q8_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q8_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q8_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q8_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q4_0_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4_0_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q4_0_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4_0_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q4_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q4_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q4_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q4_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q4k_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4k_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q4k_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4k_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q4k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q4k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q4k_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q4k_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q6k_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q6k_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q6k_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q6k_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q6k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q6k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q6k_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q6k_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q5_0_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q5_0_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q5_0_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q5_0_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q5_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q5_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q5_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q5_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q5k_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q5k_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q5k_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q5k_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q5k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q5k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q5k_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q5k_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q4_0g_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4_0g_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q4_0g_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4_0g_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q4_0g_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q4_0g_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q4_0g_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q4_0g_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q4kg_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4kg_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q4kg_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q4kg_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q4kg_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q4kg_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q4kg_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q4kg_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q5kg_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q5kg_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q5kg_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q5kg_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q5kg_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q5kg_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q5kg_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q5kg_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn gemv_rows_q6kg_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q6kg_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn gemv_rows_q6kg_add_f32(ctx: &HipContext, weight: &Buffer, x: &Buffer, res: &Buffer, y: &Buffer, rows: u32, n: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_rows_q6kg_add_f32(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, res.as_ptr() as *const f32, y.as_ptr() as *mut f32, rows, n, k) })
}
pub fn qkv_bias_rows_q6kg_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, q: &Buffer, k_out: &Buffer, v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, rows: u32, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_qkv_bias_rows_q6kg_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, q.as_ptr() as *mut f32, k_out.as_ptr() as *mut f32, v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, rows, q_dim, kv_dim, k) })
}
pub fn fused_ffn_rows_q6kg_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act: &Buffer, rows: u32, ff: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_ffn_rows_q6kg_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act.as_ptr() as *mut f32, rows, ff, k) })
}
pub fn argmax_f32(ctx: &HipContext, input: &Buffer, result: &Buffer, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_argmax_f32(ctx.raw(), input.as_ptr() as *const f32, result.as_ptr() as *mut u32, n) })
}
pub fn argmax_f16(ctx: &HipContext, input: &Buffer, result: &Buffer, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_argmax_f16(ctx.raw(), input.as_ptr() as *const u16, result.as_ptr() as *mut u32, n) })
}
pub fn synth_normal_f32(ctx: &HipContext, out: &Buffer, n: u64, seed: u64, mean: f32, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_normal_f32(ctx.raw(), out.as_ptr() as *mut f32, n, seed, mean, std) })
}
pub fn synth_normal_f16(ctx: &HipContext, out: &Buffer, n: u64, seed: u64, mean: f32, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_normal_f16(ctx.raw(), out.as_ptr() as *mut u16, n, seed, mean, std) })
}
pub fn synth_q8_0(ctx: &HipContext, out: &Buffer, n_blocks: u64, seed: u64, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_q8_0(ctx.raw(), out.as_ptr() as *mut c_void, n_blocks, seed, std) })
}
pub fn synth_q4_0(ctx: &HipContext, out: &Buffer, n_blocks: u64, seed: u64, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_q4_0(ctx.raw(), out.as_ptr() as *mut c_void, n_blocks, seed, std) })
}
pub fn synth_q4k(ctx: &HipContext, out: &Buffer, n_blocks: u64, seed: u64, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_q4k(ctx.raw(), out.as_ptr() as *mut c_void, n_blocks, seed, std) })
}
pub fn synth_q6k(ctx: &HipContext, out: &Buffer, n_blocks: u64, seed: u64, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_q6k(ctx.raw(), out.as_ptr() as *mut c_void, n_blocks, seed, std) })
}
pub fn synth_q5_0(ctx: &HipContext, out: &Buffer, n_blocks: u64, seed: u64, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_q5_0(ctx.raw(), out.as_ptr() as *mut c_void, n_blocks, seed, std) })
}
pub fn synth_q5k(ctx: &HipContext, out: &Buffer, n_blocks: u64, seed: u64, std: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_synth_q5k(ctx.raw(), out.as_ptr() as *mut c_void, n_blocks, seed, std) })
}
pub fn rms_norm_f32_f32_f32g(ctx: &HipContext, x: &Buffer, y: &Buffer, gamma: &Buffer, eps: f32, hidden: u32, num_rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_f32_f32_f32g(ctx.raw(), x.as_ptr() as *const f32, y.as_ptr() as *mut f32, gamma.as_ptr() as *const f32, eps, hidden, num_rows) })
}
pub fn fused_rope_qk_f32(ctx: &HipContext, q: &Buffer, k: &Buffer, head_dim: u32, q_heads: u32, kv_heads: u32, pos: u32, theta: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_fused_rope_qk_f32(ctx.raw(), q.as_ptr() as *mut f32, k.as_ptr() as *mut f32, head_dim, q_heads, kv_heads, pos, theta) })
}
pub fn kv_copy_to_cache_f32(ctx: &HipContext, src: &Buffer, dst: &Buffer, pos: u32, max_seq: u32, head_dim: u32, num_kv_heads: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_kv_copy_to_cache_f32(ctx.raw(), src.as_ptr() as *const f32, dst.as_ptr() as *mut f32, pos, max_seq, head_dim, num_kv_heads) })
}
pub fn decode_attention_f32(ctx: &HipContext, q: &Buffer, k: &Buffer, v: &Buffer, out: &Buffer, batch: u32, kv_len: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, kv_head_stride: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_decode_attention_f32(ctx.raw(), q.as_ptr() as *const f32, k.as_ptr() as *const f32, v.as_ptr() as *const f32, out.as_ptr() as *mut f32, batch, kv_len, num_heads, num_kv_heads, head_dim, kv_head_stride) })
}
pub fn decode_attention_rope_f32(ctx: &HipContext, q_raw: &Buffer, k_raw: &Buffer, v_raw: &Buffer, k_cache: &Buffer, v_cache: &Buffer, out: &Buffer, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_decode_attention_rope_f32(ctx.raw(), q_raw.as_ptr() as *const f32, k_raw.as_ptr() as *const f32, v_raw.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, out.as_ptr() as *mut f32, pos, max_seq, num_heads, num_kv_heads, head_dim, theta) })
}
pub fn decode_attention_rope_oproj_q8_0_f32(ctx: &HipContext, q_raw: &Buffer, k_raw: &Buffer, v_raw: &Buffer, k_cache: &Buffer, v_cache: &Buffer, w_o: &Buffer, x_io: &Buffer, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_decode_attention_rope_oproj_q8_0_f32(ctx.raw(), q_raw.as_ptr() as *const f32, k_raw.as_ptr() as *const f32, v_raw.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, w_o.as_ptr() as *const c_void, x_io.as_ptr() as *mut f32, pos, max_seq, num_heads, num_kv_heads, head_dim, theta, hidden) })
}
pub fn decode_attention_rope_oproj_q4k_f32(ctx: &HipContext, q_raw: &Buffer, k_raw: &Buffer, v_raw: &Buffer, k_cache: &Buffer, v_cache: &Buffer, w_o: &Buffer, x_io: &Buffer, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_decode_attention_rope_oproj_q4k_f32(ctx.raw(), q_raw.as_ptr() as *const f32, k_raw.as_ptr() as *const f32, v_raw.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, w_o.as_ptr() as *const c_void, x_io.as_ptr() as *mut f32, pos, max_seq, num_heads, num_kv_heads, head_dim, theta, hidden) })
}
pub fn decode_attention_rope_oproj_q4kg_f32(ctx: &HipContext, q_raw: &Buffer, k_raw: &Buffer, v_raw: &Buffer, k_cache: &Buffer, v_cache: &Buffer, w_o: &Buffer, x_io: &Buffer, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_decode_attention_rope_oproj_q4kg_f32(ctx.raw(), q_raw.as_ptr() as *const f32, k_raw.as_ptr() as *const f32, v_raw.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, w_o.as_ptr() as *const c_void, x_io.as_ptr() as *mut f32, pos, max_seq, num_heads, num_kv_heads, head_dim, theta, hidden) })
}
pub fn add_f16_into_f32(ctx: &HipContext, src: &Buffer, acc: &Buffer, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_add_f16_into_f32(ctx.raw(), src.as_ptr() as *const u16, acc.as_ptr() as *mut f32, n) })
}
pub fn add_bias_broadcast_f32(ctx: &HipContext, x: &Buffer, bias: &Buffer, seq: u32, dim: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_add_bias_broadcast_f32(ctx.raw(), x.as_ptr() as *mut f32, bias.as_ptr() as *const u16, seq, dim) })
}
pub fn rope_batch_inplace_f32(ctx: &HipContext, x: &Buffer, head_dim: u32, num_heads: u32, start_pos: u32, theta: f32, seq: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rope_batch_inplace_f32(ctx.raw(), x.as_ptr() as *mut f32, head_dim, num_heads, start_pos, theta, seq) })
}
pub fn rope_kv_write_batch_f32(ctx: &HipContext, q: &Buffer, k: &Buffer, v: &Buffer, k_cache: &Buffer, v_cache: &Buffer, head_dim: u32, num_heads: u32, num_kv_heads: u32, start_pos: u32, theta: f32, seq: u32, max_seq: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rope_kv_write_batch_f32(ctx.raw(), q.as_ptr() as *mut f32, k.as_ptr() as *const f32, v.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, head_dim, num_heads, num_kv_heads, start_pos, theta, seq, max_seq) })
}
pub fn kv_write_batch_f32(ctx: &HipContext, k: &Buffer, v: &Buffer, k_cache: &Buffer, v_cache: &Buffer, start_pos: u32, seq: u32, max_seq: u32, head_dim: u32, num_kv_heads: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_kv_write_batch_f32(ctx.raw(), k.as_ptr() as *const f32, v.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, start_pos, seq, max_seq, head_dim, num_kv_heads) })
}
pub fn flash_attention_f32(ctx: &HipContext, q: &Buffer, k: &Buffer, v: &Buffer, out: &Buffer, batch: u32, q_len: u32, kv_len: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, kv_head_stride: u32, q_start: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_flash_attention_f32(ctx.raw(), q.as_ptr() as *const f32, k.as_ptr() as *const f32, v.as_ptr() as *const f32, out.as_ptr() as *mut f32, batch, q_len, kv_len, num_heads, num_kv_heads, head_dim, kv_head_stride, q_start) })
}
pub fn add_f32(ctx: &HipContext, a: &Buffer, b: &Buffer, out: &Buffer, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_add_f32(ctx.raw(), a.as_ptr() as *const f32, b.as_ptr() as *const f32, out.as_ptr() as *mut f32, n) })
}
pub fn silu_mul_f32(ctx: &HipContext, gate: &Buffer, up: &Buffer, out: &Buffer, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_silu_mul_f32(ctx.raw(), gate.as_ptr() as *const f32, up.as_ptr() as *const f32, out.as_ptr() as *mut f32, n) })
}
pub fn argmax_rows_first_f32(ctx: &HipContext, in_: &Buffer, result: &Buffer, rows: u32, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_argmax_rows_first_f32(ctx.raw(), in_.as_ptr() as *const f32, result.as_ptr() as *mut u32, rows, n) })
}
pub fn rope_kv_append_paged_f32(ctx: &HipContext, batch: &ffi::RtPagedBatch, q: &Buffer, k: &Buffer, v: &Buffer, q_out: &Buffer, num_heads: u32, theta: f32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rope_kv_append_paged_f32(ctx.raw(), batch, q.as_ptr() as *const f32, k.as_ptr() as *const f32, v.as_ptr() as *const f32, q_out.as_ptr() as *mut f32, num_heads, theta) })
}
pub fn paged_attention_f32(ctx: &HipContext, batch: &ffi::RtPagedBatch, q: &Buffer, out: &Buffer, num_heads: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_paged_attention_f32(ctx.raw(), batch, q.as_ptr() as *const f32, out.as_ptr() as *mut f32, num_heads) })
}
pub fn shared_prefix_attention_f32(ctx: &HipContext, batch: &ffi::RtPagedBatch, q: &Buffer, out: &Buffer, num_heads: u32, shared_table: &Buffer, shared_len: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_shared_prefix_attention_f32(ctx.raw(), batch, q.as_ptr() as *const f32, out.as_ptr() as *mut f32, num_heads, shared_table.as_ptr() as *const u32, shared_len) })
}
pub fn paged_gather_f32(ctx: &HipContext, batch: &ffi::RtPagedBatch, k: &Buffer, v: &Buffer) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_paged_gather_f32(ctx.raw(), batch, k.as_ptr() as *mut f32, v.as_ptr() as *mut f32) })
}
pub fn paged_gather_f16(ctx: &HipContext, batch: &ffi::RtPagedBatch, k: &Buffer, v: &Buffer) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_paged_gather_f16(ctx.raw(), batch, k.as_ptr() as *mut u16, v.as_ptr() as *mut u16) })
}
pub fn paged_copy(ctx: &HipContext, batches: &[ffi::RtPagedBatch], src: &Buffer, dst: &Buffer, n: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_paged_copy(ctx.raw(), batches.as_ptr(), batches.len() as u32, src.as_ptr() as *const u32, dst.as_ptr() as *const u32, n) })
}
pub fn adjust_logits_f32(ctx: &HipContext, logits: &Buffer, out: &Buffer, rows: u32, n: u32, row_stride: u64, rules: &ffi::RtLogitRules) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_adjust_logits_f32(ctx.raw(), logits.as_ptr() as *const f32, out.as_ptr() as *mut f32, rows, n, row_stride, rules) })
}
pub fn adjust_logits_f16(ctx: &HipContext, logits: &Buffer, out: &Buffer, rows: u32, n: u32, row_stride: u64, rules: &ffi::RtLogitRules) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_adjust_logits_f16(ctx.raw(), logits.as_ptr() as *const u16, out.as_ptr() as *mut u16, rows, n, row_stride, rules) })
}
pub fn token_logprobs_f32(ctx: &HipContext, logits: &Buffer, tokens: &Buffer, rows: u32, n: u32, row_stride: u64, logprob: &Buffer, entropy: &Buffer, rank: &Buffer, top: u32, top_ids: &Buffer, top_logprobs: &Buffer) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_token_logprobs_f32(ctx.raw(), logits.as_ptr() as *const f32, tokens.as_ptr() as *const u32, rows, n, row_stride, logprob.as_ptr() as *mut f32, entropy.as_ptr() as *mut f32, rank.as_ptr() as *mut u32, top, top_ids.as_ptr() as *mut u32, top_logprobs.as_ptr() as *mut f32) })
}
pub fn token_logprobs_f16(ctx: &HipContext, logits: &Buffer, tokens: &Buffer, rows: u32, n: u32, row_stride: u64, logprob: &Buffer, entropy: &Buffer, rank: &Buffer, top: u32, top_ids: &Buffer, top_logprobs: &Buffer) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_token_logprobs_f16(ctx.raw(), logits.as_ptr() as *const u16, tokens.as_ptr() as *const u32, rows, n, row_stride, logprob.as_ptr() as *mut f32, entropy.as_ptr() as *mut f32, rank.as_ptr() as *mut u32, top, top_ids.as_ptr() as *mut u32, top_logprobs.as_ptr() as *mut f32) })
}
pub fn embed_q8_0_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q8_0_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q4_0_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q4_0_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q4k_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q4k_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q6k_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q6k_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q5_0_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q5_0_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q5k_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q5k_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q4_0g_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q4_0g_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q4kg_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q4kg_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q5kg_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q5kg_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_q6kg_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_q6kg_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_f16_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_f16_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_f32_f32(ctx: &HipContext, table: &Buffer, token: &Buffer, out: &Buffer, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_f32_f32(ctx.raw(), table.as_ptr() as *const c_void, token.as_ptr() as *const u32, out.as_ptr() as *mut f32, k) })
}
pub fn embed_rows_q8_0_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q8_0_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q4_0_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q4_0_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q4k_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q4k_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q6k_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q6k_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q5_0_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q5_0_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q5k_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q5k_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q4_0g_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q4_0g_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q4kg_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q4kg_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q5kg_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q5kg_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_q6kg_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_q6kg_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_f16_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_f16_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn embed_rows_f32_f32(ctx: &HipContext, table: &Buffer, tokens: &Buffer, out: &Buffer, k: u32, rows: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_embed_rows_f32_f32(ctx.raw(), table.as_ptr() as *const c_void, tokens.as_ptr() as *const u32, out.as_ptr() as *mut f32, k, rows) })
}
pub fn rms_norm_fused_qkv_bias_q8_0_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_fused_qkv_bias_q8_0_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn rms_norm_fused_ffn_q8_0_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_fused_ffn_q8_0_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn rms_norm_gemv_q8_0_f32in_f32out(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_gemv_q8_0_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, output.as_ptr() as *mut f32, m, k) })
}
pub fn gemv_q8_0_add_f32_f32in_ssq(ctx: &HipContext, weight: &Buffer, input: &Buffer, output: &Buffer, residual: &Buffer, m: u32, k: u32, ssq: &Buffer) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_gemv_q8_0_add_f32_f32in_ssq(ctx.raw(), weight.as_ptr() as *const c_void, input.as_ptr() as *const f32, output.as_ptr() as *mut f32, residual.as_ptr() as *const f32, m, k, ssq.as_ptr() as *mut f32) })
}
pub fn decode_attention_rope_oproj_q8_0_f32_ssq(ctx: &HipContext, q_raw: &Buffer, k_raw: &Buffer, v_raw: &Buffer, k_cache: &Buffer, v_cache: &Buffer, w_o: &Buffer, x_io: &Buffer, pos: u32, max_seq: u32, num_heads: u32, num_kv_heads: u32, head_dim: u32, theta: f32, hidden: u32, ssq: &Buffer) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_decode_attention_rope_oproj_q8_0_f32_ssq(ctx.raw(), q_raw.as_ptr() as *const f32, k_raw.as_ptr() as *const f32, v_raw.as_ptr() as *const f32, k_cache.as_ptr() as *mut f32, v_cache.as_ptr() as *mut f32, w_o.as_ptr() as *const c_void, x_io.as_ptr() as *mut f32, pos, max_seq, num_heads, num_kv_heads, head_dim, theta, hidden, ssq.as_ptr() as *mut f32) })
}
pub fn rms_norm_fused_qkv_bias_q8_0_f32_ssq(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32, ssq: &Buffer, nparts: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_fused_qkv_bias_q8_0_f32_ssq(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k, ssq.as_ptr() as *const f32, nparts) })
}
pub fn rms_norm_fused_ffn_q8_0_f32_ssq(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act_out: &Buffer, ff_dim: u32, k: u32, ssq: &Buffer, nparts: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_fused_ffn_q8_0_f32_ssq(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act_out.as_ptr() as *mut f32, ff_dim, k, ssq.as_ptr() as *const f32, nparts) })
}
pub fn rms_norm_fused_qkv_bias_q4k_q6k_f32(ctx: &HipContext, w_q: &Buffer, w_k: &Buffer, w_v: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, out_q: &Buffer, out_k: &Buffer, out_v: &Buffer, bias_q: &Buffer, bias_k: &Buffer, bias_v: &Buffer, q_dim: u32, kv_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_fused_qkv_bias_q4k_q6k_f32(ctx.raw(), w_q.as_ptr() as *const c_void, w_k.as_ptr() as *const c_void, w_v.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, out_q.as_ptr() as *mut f32, out_k.as_ptr() as *mut f32, out_v.as_ptr() as *mut f32, bias_q.as_ptr() as *const u16, bias_k.as_ptr() as *const u16, bias_v.as_ptr() as *const u16, q_dim, kv_dim, k) })
}
pub fn rms_norm_fused_ffn_q4k_f32(ctx: &HipContext, w_gate: &Buffer, w_up: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, act_out: &Buffer, ff_dim: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_fused_ffn_q4k_f32(ctx.raw(), w_gate.as_ptr() as *const c_void, w_up.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, act_out.as_ptr() as *mut f32, ff_dim, k) })
}
pub fn rms_norm_gemv_q6k_f32in_f32out(ctx: &HipContext, weight: &Buffer, x: &Buffer, gamma: &Buffer, eps: f32, output: &Buffer, m: u32, k: u32) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_rms_norm_gemv_q6k_f32in_f32out(ctx.raw(), weight.as_ptr() as *const c_void, x.as_ptr() as *const f32, gamma.as_ptr() as *const f32, eps, output.as_ptr() as *mut f32, m, k) })
}
pub fn stream_read(ctx: &HipContext, src: &Buffer, bytes: usize, sink: &Buffer, sink_dwords: usize) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_stream_read(ctx.raw(), src.as_ptr() as *const c_void, bytes, sink.as_ptr() as *mut u32, sink_dwords) })
}
pub fn stream_copy(ctx: &HipContext, dst: &Buffer, src: &Buffer, bytes: usize) -> Result<()> {
    status(ctx.raw(), unsafe { ffi::rt_stream_copy(ctx.raw(), dst.as_ptr() as *mut c_void, src.as_ptr() as *const c_void, bytes) })
}
