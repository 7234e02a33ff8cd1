//! Raw declarations of `include/mi_moe_layer.h`, one to one: what a decoder layer runs around the expert block.
#![allow(non_snake_case)]

use std::os::raw::{c_int, c_void};

use crate::{mi_moe_debug_out, mi_moe_handle};

pub const MI_MOE_SCORING_SOFTMAX: i32 = 0;
pub const MI_MOE_SCORING_SIGMOID: i32 = 1;
pub const MI_MOE_GROUP_SCORE_MAX: i32 = 0;
pub const MI_MOE_GROUP_SCORE_TOP2: i32 = 1;

extern "C" {
    pub fn mi_moe_add_rms_norm(x: *const c_void, residual: *const c_void, weight: *const c_void, eps: f32, T: i64, hidden: i32, dtype: i32, sum: *mut c_void, y: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn mi_moe_add_rms_norm_rows8(x: *const c_void, residual: *const c_void, weight: *const c_void, eps: f32, T: i64, hidden: i32, dtype: i32, sum: *mut c_void, rows8: *mut c_void, row_scales: *mut f32, stream: *mut c_void) -> c_int;
    pub fn mi_moe_add_rms_norm_grad_workspace_size(T: i64, hidden: i32, bytes: *mut usize) -> c_int;
    pub fn mi_moe_add_rms_norm_grad(dy: *const c_void, sum: *const c_void, dsum: *const c_void, weight: *const c_void, eps: f32, T: i64, hidden: i32, dtype: i32, dx: *mut c_void, dweight: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn mi_moe_forward_routed(h: mi_moe_handle, x: *const u16, topk_idx: *const u32, topk_w: *const u16, T: i64, out: *mut u16, workspace: *mut c_void, workspace_bytes: usize, dbg: *const mi_moe_debug_out, stream: *mut c_void) -> c_int;
    pub fn mi_moe_select_experts(logits: *const c_void, dtype: i32, bias: *const f32, T: i64, n_experts: i32, top_k: i32, scoring: i32, n_groups: i32, top_groups: i32, group_score: i32, renormalize: i32, scale: f32, topk_idx: *mut u32, topk_w: *mut c_void, w_dtype: i32, stream: *mut c_void) -> c_int;
    pub fn mi_moe_select_experts_grad(dw: *const c_void, w_dtype: i32, logits: *const c_void, dtype: i32, topk_idx: *const u32, T: i64, n_experts: i32, top_k: i32, scoring: i32, renormalize: i32, scale: f32, dlogits: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn mi_moe_quantized_linear_rows8_workspace_size(M: i64, K: i32, bytes: *mut usize) -> c_int;
    pub fn mi_moe_quantized_linear_rows8(x: *const c_void, row_scales: *const f32, w: *const u32, scales: *const c_void, biases: *const c_void, linear_bias: *const c_void, M: i64, N: i32, K: i32, group_size: i32, bits: i32, dtype: i32, y: *mut c_void, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
}
