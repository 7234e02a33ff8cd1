//! Raw declarations of `include/mi_moe_f8.h`, one to one: experts and linear layers on e4m3 weights, tokens sorted by expert.
#![allow(non_camel_case_types, non_snake_case)]

use std::os::raw::{c_int, c_void};

#[repr(C)]
#[derive(Clone, Copy)]
pub struct mi_moe_f8_experts {
    pub gate: *const c_void,
    pub up: *const c_void,
    pub down: *const c_void,
    pub gate_scales: *const f32,
    pub up_scales: *const f32,
    pub down_scales: *const f32,
}

extern "C" {
    pub fn mi_moe_sort_tokens_workspace_size(T: i64, top_k: i32, n_experts: i32, bytes: *mut usize) -> c_int;
    pub fn mi_moe_sort_tokens(x: *const c_void, topk_idx: *const u32, T: i64, top_k: i32, n_experts: i32, hidden: i32, dtype: i32, rows: *mut c_void, order: *mut u32, inverse: *mut i32, offsets: *mut u32, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn mi_moe_sort_tokens_grad(drows: *const c_void, inverse: *const i32, T: i64, top_k: i32, hidden: i32, dtype: i32, dx: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn mi_moe_unsort_tokens(rows: *const c_void, topk_w: *const c_void, w_dtype: i32, inverse: *const i32, T: i64, top_k: i32, hidden: i32, dtype: i32, out: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn mi_moe_unsort_tokens_grad(dout: *const c_void, rows: *const c_void, topk_w: *const c_void, w_dtype: i32, inverse: *const i32, T: i64, top_k: i32, hidden: i32, dtype: i32, drows: *mut c_void, dweights: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn mi_moe_quantize_f8(x: *const c_void, dtype: i32, rows: i64, cols: i64, block_rows: i32, codes: *mut c_void, scales: *mut f32, stream: *mut c_void) -> c_int;
    pub fn mi_moe_dequantize_f8(codes: *const c_void, scales: *const f32, rows: i64, cols: i64, block_rows: i32, dtype: i32, out: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn mi_moe_linear_f8_workspace_size(M: i64, N: i32, K: i32, bytes: *mut usize) -> c_int;
    pub fn mi_moe_linear_f8(x: *const c_void, w: *const c_void, scales: *const f32, linear_bias: *const c_void, M: i64, N: i32, K: i32, transpose: i32, dtype: i32, y: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn mi_moe_grouped_linear_f8(x: *const c_void, w: *const c_void, scales: *const f32, offsets: *const u32, rows: i64, n_experts: i32, N: i32, K: i32, transpose: i32, dtype: i32, y: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn mi_moe_switch_glu_f8_workspace_size(T: i64, hidden: i32, intermediate: i32, n_experts: i32, top_k: i32, grad: i32, bytes: *mut usize) -> c_int;
    pub fn mi_moe_switch_glu_f8(x: *const c_void, topk_idx: *const u32, topk_w: *const c_void, w_dtype: i32, experts: *const mi_moe_f8_experts, T: i64, hidden: i32, intermediate: i32, n_experts: i32, top_k: i32, dtype: i32, out: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn mi_moe_switch_glu_f8_grad(dout: *const c_void, x: *const c_void, topk_idx: *const u32, topk_w: *const c_void, w_dtype: i32, experts: *const mi_moe_f8_experts, T: i64, hidden: i32, intermediate: i32, n_experts: i32, top_k: i32, dtype: i32, dx: *mut c_void, dweights: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
}
