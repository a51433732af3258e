// GENERATED by rust/ferrox-hip-sys/generate.py from include/ferrox_hip.h -- do not edit.
//! Raw FFI bindings of `libferrox_hip.so`, the MI355X (gfx950) backend of Ferrox's training hot path.
//! Every entry point returns an `int` status (`FX_OK` = 0); `fx_last_error()` holds the message of the last failure
//! on the calling thread.  Tensor pointers are device pointers unless the parameter is named `host_*`.
#![allow(non_camel_case_types, non_upper_case_globals, non_snake_case, clippy::too_many_arguments)]
use std::os::raw::{c_char, c_int, c_void};

/// Opaque context (one device, one compute stream, one pool per dtype).
#[repr(C)]
pub struct fx_ctx {
    _private: [u8; 0],
}

/// Opaque recorded step (fx_graph_begin .. fx_graph_end).
#[repr(C)]
pub struct fx_graph {
    _private: [u8; 0],
}

pub const FX_OK: c_int = 0;
pub const FX_ERR_INVALID: c_int = 1;
pub const FX_ERR_HIP: c_int = 2;
pub const FX_ERR_OOM: c_int = 3;
pub const FX_ERR_UNSUPPORTED: c_int = 4;
pub const FX_F32: c_int = 0;
pub const FX_F64: c_int = 1;
pub const FX_MAX_BUCKETS: usize = 8;
pub const FX_CONV_FWD: c_int = 0;
pub const FX_CONV_DGRAD: c_int = 1;
pub const FX_CONV_WGRAD: c_int = 2;
pub const FX_NOALLOC_SCRATCH_BYTES: usize = 4 << 20;

pub const FX_ADD: c_int = 0;
pub const FX_SUB: c_int = 1;
pub const FX_MUL: c_int = 2;
pub const FX_DIV: c_int = 3;
pub const FX_EQUAL: c_int = 4;
pub const FX_GREATER: c_int = 5;
pub const FX_GREATER_EQUAL: c_int = 6;
pub const FX_LESS: c_int = 7;
pub const FX_LESS_EQUAL: c_int = 8;
pub const FX_MIN: c_int = 9;
pub const FX_MAX: c_int = 10;
pub const FX_POW: c_int = 11;
pub const FX_NEG: c_int = 0;
pub const FX_SQRT: c_int = 1;
pub const FX_EXP: c_int = 2;
pub const FX_LOG: c_int = 3;
pub const FX_RELU: c_int = 4;
pub const FX_SIGMOID: c_int = 5;
pub const FX_TANH: c_int = 6;
pub const FX_ABS: c_int = 7;
pub const FX_RECIPROCAL: c_int = 8;
pub const FX_SIGN: c_int = 9;
pub const FX_LOGICAL_NOT: c_int = 10;
pub const FX_ADD_SCALAR: c_int = 0;
pub const FX_SUB_SCALAR: c_int = 1;
pub const FX_MUL_SCALAR: c_int = 2;
pub const FX_DIV_SCALAR: c_int = 3;
pub const FX_GREATER_SCALAR: c_int = 4;
pub const FX_GREATER_EQUAL_SCALAR: c_int = 5;
pub const FX_LESS_EQUAL_SCALAR: c_int = 6;
pub const FX_LESS_SCALAR: c_int = 7;
pub const FX_POW_SCALAR: c_int = 8;

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fx_bucket_config {
    pub min_elems: i64,
    pub max_elems: i64,
    pub max_blocks: i64,
    pub to_evict: i64,
    pub eviction_threshold_ms: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fx_pool_config {
    pub n_buckets: i32,
    pub literal_ids: i32,
    pub best_fit: i32,
    pub reserved: i32,
    pub buckets: [fx_bucket_config; FX_MAX_BUCKETS as usize],
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fx_pool_stats {
    pub total_allocations: i64,
    pub active_allocations: i64,
    pub pool_hits: i64,
    pub pool_misses: i64,
    pub underflow_misses: i64,
    pub allocation_counter: i64,
    pub active_table_len: i64,
    pub device_allocs: i64,
    pub device_frees: i64,
    pub bytes_in_use: i64,
    pub bytes_pooled: i64,
    pub peak_bytes: i64,
}

#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct fx_bucket_stats {
    pub pooled_blocks: i64,
    pub total_allocations: i64,
    pub total_evictions: i64,
    pub av_allocations: i64,
    pub max_allocations: i64,
}

#[link(name = "ferrox_hip")]
extern "C" {
    pub fn fx_init(device: c_int, cfg_or_null: *const fx_pool_config, out: *mut *mut fx_ctx) -> c_int;
    pub fn fx_destroy(ctx: *mut fx_ctx) -> c_int;
    pub fn fx_sync(ctx: *mut fx_ctx) -> c_int;
    pub fn fx_device_name(ctx: *mut fx_ctx, buf: *mut c_char, buf_len: i64) -> c_int;
    pub fn fx_last_error() -> *const c_char;
    pub fn fx_stream(ctx: *mut fx_ctx) -> *mut c_void;
    pub fn fx_timer_start(ctx: *mut fx_ctx) -> c_int;
    pub fn fx_timer_stop(ctx: *mut fx_ctx, elapsed_ms: *mut f32) -> c_int;
    pub fn fx_alloc(ctx: *mut fx_ctx, dtype: c_int, n_elems: i64, ptr: *mut *mut c_void, granted_elems: *mut i64, alloc_id: *mut u64) -> c_int;
    pub fn fx_free(ctx: *mut fx_ctx, dtype: c_int, ptr: *mut c_void, alloc_id: u64) -> c_int;
    pub fn fx_pool_cleanup(ctx: *mut fx_ctx, dtype: c_int) -> c_int;
    pub fn fx_pool_reset(ctx: *mut fx_ctx, dtype: c_int) -> c_int;
    pub fn fx_pool_stats_get(ctx: *mut fx_ctx, dtype: c_int, out: *mut fx_pool_stats) -> c_int;
    pub fn fx_pool_bucket_stats_get(ctx: *mut fx_ctx, dtype: c_int, bucket: c_int, out: *mut fx_bucket_stats) -> c_int;
    pub fn fx_h2d(ctx: *mut fx_ctx, dst_dev: *mut c_void, host_src: *const c_void, bytes: i64) -> c_int;
    pub fn fx_d2h(ctx: *mut fx_ctx, host_dst: *mut c_void, src_dev: *const c_void, bytes: i64) -> c_int;
    pub fn fx_d2d(ctx: *mut fx_ctx, dst_dev: *mut c_void, src_dev: *const c_void, bytes: i64) -> c_int;
    pub fn fx_conv2d_workspace_bytes(kind: c_int, dtype: c_int, mode: c_int, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> i64;
    pub fn fx_conv2d_tune_f32(ctx: *mut fx_ctx, kind: c_int, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, with_bias: c_int, act: c_int) -> c_int;
    pub fn fx_fill_f32(ctx: *mut fx_ctx, out: *mut f32, value: f32, n: i64) -> c_int;
    pub fn fx_fill_uniform_f32(ctx: *mut fx_ctx, out: *mut f32, n: i64, seed: u64, lo: f32, hi: f32) -> c_int;
    pub fn fx_fill_normal_f32(ctx: *mut fx_ctx, out: *mut f32, n: i64, seed: u64, mean: f32, std: f32) -> c_int;
    pub fn fx_materialize_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, host_shape: *const i64, host_strides: *const i64, ndim: c_int, n: i64) -> c_int;
    pub fn fx_binary_f32(ctx: *mut fx_ctx, op: c_int, a: *const f32, b: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_add_f32(ctx: *mut fx_ctx, a: *const f32, b: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_sub_f32(ctx: *mut fx_ctx, a: *const f32, b: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_mul_f32(ctx: *mut fx_ctx, a: *const f32, b: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_div_f32(ctx: *mut fx_ctx, a: *const f32, b: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_equal_f32(ctx: *mut fx_ctx, a: *const f32, b: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_scalar_f32(ctx: *mut fx_ctx, op: c_int, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_add_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_sub_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_mul_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_div_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_greater_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_greater_equal_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_less_equal_scalar_f32(ctx: *mut fx_ctx, a: *const f32, s: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_unary_f32(ctx: *mut fx_ctx, op: c_int, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_neg_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_sqrt_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_exp_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_log_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_relu_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_sigmoid_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_tanh_f32(ctx: *mut fx_ctx, a: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_clamp_f32(ctx: *mut fx_ctx, a: *const f32, lo: f32, hi: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_in_range_f32(ctx: *mut fx_ctx, a: *const f32, lo: f32, hi: f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_relu_bwd_f32(ctx: *mut fx_ctx, g: *const f32, x: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_sigmoid_bwd_f32(ctx: *mut fx_ctx, g: *const f32, s: *const f32, out: *mut f32, n: i64, literal: c_int) -> c_int;
    pub fn fx_tanh_bwd_f32(ctx: *mut fx_ctx, g: *const f32, t: *const f32, out: *mut f32, n: i64) -> c_int;
    pub fn fx_softmax_axis_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_sum_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_mean_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_max_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, idx_out: *mut i64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_min_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, idx_out: *mut i64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_prod_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_gemm_f32(ctx: *mut fx_ctx, trans_a: c_int, trans_b: c_int, M: i64, N: i64, K: i64, A: *const f32, B: *const f32, C: *mut f32) -> c_int;
    pub fn fx_im2col_f32(ctx: *mut fx_ctx, x: *const f32, col: *mut f32, B: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_col2im_f32(ctx: *mut fx_ctx, col: *const f32, out: *mut f32, B: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, layout: c_int) -> c_int;
    pub fn fx_conv2d_fwd_f32(ctx: *mut fx_ctx, x: *const f32, w: *const f32, y: *mut f32, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_conv2d_dgrad_f32(ctx: *mut fx_ctx, g: *const f32, w: *const f32, dx: *mut f32, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, mode: c_int, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_conv2d_wgrad_f32(ctx: *mut fx_ctx, x: *const f32, g: *const f32, dw: *mut f32, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, mode: c_int, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_maxpool2d_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_avgpool2d_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_max_unpool2d_f32(ctx: *mut fx_ctx, grad_out: *const f32, input: *const f32, pooled: *const f32, grad_in: *mut f32, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_avg_unpool2d_f32(ctx: *mut fx_ctx, grad_out: *const f32, grad_in: *mut f32, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_bias_act_f32(ctx: *mut fx_ctx, y: *mut f32, bias: *const f32, outer: i64, C: i64, inner: i64, act: c_int) -> c_int;
    pub fn fx_conv2d_fwd_bias_act_f32(ctx: *mut fx_ctx, x: *const f32, w: *const f32, bias: *const f32, y: *mut f32, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, act: c_int, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_gemm_bias_act_f32(ctx: *mut fx_ctx, trans_a: c_int, trans_b: c_int, M: i64, N: i64, K: i64, A: *const f32, B: *const f32, bias: *const f32, C: *mut f32, act: c_int) -> c_int;
    pub fn fx_conv2d_wgrad_relu_bias_f32(ctx: *mut fx_ctx, x: *const f32, g: *const f32, act: *const f32, dw: *mut f32, db: *mut f32, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_conv2d_dgrad_relu_f32(ctx: *mut fx_ctx, g: *const f32, act: *const f32, w: *const f32, dx: *mut f32, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_gemm_tn_colsum_f32(ctx: *mut fx_ctx, M: i64, N: i64, K: i64, A: *const f32, B: *const f32, C: *mut f32, colsum: *mut f32) -> c_int;
    pub fn fx_linear_bwd_f32(ctx: *mut fx_ctx, B: i64, input: i64, out: i64, dY: *const f32, W: *const f32, X: *const f32, dX: *mut f32, dW: *mut f32, db: *mut f32, relu_below: c_int) -> c_int;
    pub fn fx_batchnorm_stats_f32(ctx: *mut fx_ctx, x: *const f32, mean: *mut f32, var: *mut f32, running_mean: *mut f32, running_var: *mut f32, momentum: f64, outer: i64, C: i64, inner: i64) -> c_int;
    pub fn fx_batchnorm_fwd_f32(ctx: *mut fx_ctx, x: *const f32, mean: *const f32, var: *const f32, gamma: *const f32, beta: *const f32, eps: f64, y: *mut f32, outer: i64, C: i64, inner: i64, act: c_int) -> c_int;
    pub fn fx_batchnorm_bwd_f32(ctx: *mut fx_ctx, dy: *const f32, x: *const f32, y_act: *const f32, mean: *const f32, var: *const f32, gamma: *const f32, eps: f64, dx: *mut f32, dgamma: *mut f32, dbeta: *mut f32, outer: i64, C: i64, inner: i64, batch_stats: c_int) -> c_int;
    pub fn fx_dropout_f32(ctx: *mut fx_ctx, x: *const f32, mask: *mut f32, y: *mut f32, n: i64, p: f64, seed: u64) -> c_int;
    pub fn fx_bias_grad_f32(ctx: *mut fx_ctx, g: *const f32, out: *mut f32, outer: i64, C: i64, inner: i64) -> c_int;
    pub fn fx_relu_bwd_bias_grad_f32(ctx: *mut fx_ctx, g: *const f32, y: *const f32, gm: *mut f32, dbias: *mut f32, outer: i64, C: i64, inner: i64) -> c_int;
    pub fn fx_softmax_ce_fwd_f32(ctx: *mut fx_ctx, logits: *const f32, targets: *const f32, probs: *mut f32, loss: *mut f32, B: i64, C: i64) -> c_int;
    pub fn fx_softmax_ce_bwd_f32(ctx: *mut fx_ctx, probs: *const f32, targets: *const f32, grad_loss: *const f32, dlogits: *mut f32, B: i64, C: i64) -> c_int;
    pub fn fx_softmax_ce_fwd_unit_grad_f32(ctx: *mut fx_ctx, logits: *const f32, targets: *const f32, probs: *mut f32, loss: *mut f32, dlogits: *mut f32, B: i64, C: i64) -> c_int;
    pub fn fx_adam_step_f32(ctx: *mut fx_ctx, p: *mut f32, g: *const f32, m: *mut f32, v: *mut f32, n: i64, lr: f32, beta1: f32, beta2: f32, eps: f32, weight_decay: f32, bc1: f32, bc2: f32) -> c_int;
    pub fn fx_adam_amsgrad_step_f32(ctx: *mut fx_ctx, p: *mut f32, g: *const f32, m: *mut f32, v: *mut f32, vmax: *mut f32, n: i64, lr: f32, beta1: f32, beta2: f32, eps: f32, weight_decay: f32, bc1: f32, bc2: f32) -> c_int;
    pub fn fx_sgd_step_f32(ctx: *mut fx_ctx, p: *mut f32, g: *const f32, n: i64, lr: f32) -> c_int;
    pub fn fx_sgd_momentum_step_f32(ctx: *mut fx_ctx, p: *mut f32, g: *const f32, buf: *mut f32, n: i64, lr: f32, momentum: f32, weight_decay: f32, nesterov: c_int) -> c_int;
    pub fn fx_adam_step_multi_f32(ctx: *mut fx_ctx, count: c_int, p: *const *mut f32, g: *const *const f32, m: *const *mut f32, v: *const *mut f32, n: *const i64, lr: f32, beta1: f32, beta2: f32, eps: f32, weight_decay: f32, bc1: f32, bc2: f32) -> c_int;
    pub fn fx_adam_amsgrad_step_multi_f32(ctx: *mut fx_ctx, count: c_int, p: *const *mut f32, g: *const *const f32, m: *const *mut f32, v: *const *mut f32, vmax: *const *mut f32, n: *const i64, lr: f32, beta1: f32, beta2: f32, eps: f32, weight_decay: f32, bc1: f32, bc2: f32) -> c_int;
    pub fn fx_adam_step_multi_bc_f32(ctx: *mut fx_ctx, count: c_int, p: *const *mut f32, g: *const *const f32, m: *const *mut f32, v: *const *mut f32, vmax: *const *mut f32, n: *const i64, lr: f32, beta1: f32, beta2: f32, eps: f32, weight_decay: f32, bc: *const f32) -> c_int;
    pub fn fx_sgd_step_multi_f32(ctx: *mut fx_ctx, count: c_int, p: *const *mut f32, g: *const *const f32, n: *const i64, lr: f32) -> c_int;
    pub fn fx_sgd_momentum_step_multi_f32(ctx: *mut fx_ctx, count: c_int, p: *const *mut f32, g: *const *const f32, buf: *const *mut f32, n: *const i64, lr: f32, momentum: f32, weight_decay: f32, nesterov: c_int) -> c_int;
    pub fn fx_embedding_fwd_f32(ctx: *mut fx_ctx, W: *const f32, ids: *const i64, out: *mut f32, n: i64, vocab: i64, dim: i64, scale: f32) -> c_int;
    pub fn fx_embedding_bwd_f32(ctx: *mut fx_ctx, g: *const f32, ids: *const i64, dW: *mut f32, n: i64, vocab: i64, dim: i64, scale: f32) -> c_int;
    pub fn fx_rmsnorm_fwd_f32(ctx: *mut fx_ctx, x: *const f32, res: *const f32, w: *const f32, eps: f64, h: *mut f32, y: *mut f32, rstd: *mut f32, rows: i64, dim: i64) -> c_int;
    pub fn fx_rmsnorm_bwd_f32(ctx: *mut fx_ctx, dy: *const f32, dh: *const f32, h: *const f32, w: *const f32, rstd: *const f32, dx: *mut f32, dw: *mut f32, rows: i64, dim: i64) -> c_int;
    pub fn fx_gemm_bias_act_residual_f32(ctx: *mut fx_ctx, trans_a: c_int, trans_b: c_int, M: i64, N: i64, K: i64, A: *const f32, B: *const f32, bias: *const f32, residual: *const f32, pre: *mut f32, C: *mut f32, act: c_int) -> c_int;
    pub fn fx_linear_act_bwd_f32(ctx: *mut fx_ctx, B: i64, input: i64, out: i64, dY: *const f32, W: *const f32, X: *const f32, pre: *const f32, act: c_int, dpre: *mut f32, dX: *mut f32, dW: *mut f32, db: *mut f32) -> c_int;
    pub fn fx_gated_recurrence_fwd_f32(ctx: *mut fx_ctx, z: *const f32, x: *const f32, h0: *const f32, h: *mut f32, B: i64, steps: i64, dim: i64) -> c_int;
    pub fn fx_gated_recurrence_bwd_f32(ctx: *mut fx_ctx, dh: *const f32, z: *const f32, x: *const f32, h: *const f32, h0: *const f32, dh_next: *const f32, dz: *mut f32, dx: *mut f32, dh0: *mut f32, B: i64, steps: i64, dim: i64) -> c_int;
    pub fn fx_grad_norm_multi_f32(ctx: *mut fx_ctx, count: c_int, g: *const *const f32, n: *const i64, norm: *mut f32) -> c_int;
    pub fn fx_clip_grad_norm_multi_f32(ctx: *mut fx_ctx, count: c_int, g: *const *const f32, out: *const *mut f32, n: *const i64, max_norm: f64, norm: *mut f32) -> c_int;
    pub fn fx_fill_f64(ctx: *mut fx_ctx, out: *mut f64, value: f64, n: i64) -> c_int;
    pub fn fx_fill_uniform_f64(ctx: *mut fx_ctx, out: *mut f64, n: i64, seed: u64, lo: f64, hi: f64) -> c_int;
    pub fn fx_fill_normal_f64(ctx: *mut fx_ctx, out: *mut f64, n: i64, seed: u64, mean: f64, std: f64) -> c_int;
    pub fn fx_materialize_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, host_shape: *const i64, host_strides: *const i64, ndim: c_int, n: i64) -> c_int;
    pub fn fx_binary_f64(ctx: *mut fx_ctx, op: c_int, a: *const f64, b: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_add_f64(ctx: *mut fx_ctx, a: *const f64, b: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_sub_f64(ctx: *mut fx_ctx, a: *const f64, b: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_mul_f64(ctx: *mut fx_ctx, a: *const f64, b: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_div_f64(ctx: *mut fx_ctx, a: *const f64, b: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_equal_f64(ctx: *mut fx_ctx, a: *const f64, b: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_scalar_f64(ctx: *mut fx_ctx, op: c_int, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_add_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_sub_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_mul_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_div_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_greater_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_greater_equal_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_less_equal_scalar_f64(ctx: *mut fx_ctx, a: *const f64, s: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_unary_f64(ctx: *mut fx_ctx, op: c_int, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_neg_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_sqrt_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_exp_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_log_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_relu_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_sigmoid_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_tanh_f64(ctx: *mut fx_ctx, a: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_clamp_f64(ctx: *mut fx_ctx, a: *const f64, lo: f64, hi: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_in_range_f64(ctx: *mut fx_ctx, a: *const f64, lo: f64, hi: f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_relu_bwd_f64(ctx: *mut fx_ctx, g: *const f64, x: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_sigmoid_bwd_f64(ctx: *mut fx_ctx, g: *const f64, s: *const f64, out: *mut f64, n: i64, literal: c_int) -> c_int;
    pub fn fx_tanh_bwd_f64(ctx: *mut fx_ctx, g: *const f64, t: *const f64, out: *mut f64, n: i64) -> c_int;
    pub fn fx_softmax_axis_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_sum_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_mean_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_max_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, idx_out: *mut i64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_min_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, idx_out: *mut i64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_reduce_prod_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, outer: i64, axis: i64, inner: i64) -> c_int;
    pub fn fx_gemm_f64(ctx: *mut fx_ctx, trans_a: c_int, trans_b: c_int, M: i64, N: i64, K: i64, A: *const f64, B: *const f64, C: *mut f64) -> c_int;
    pub fn fx_im2col_f64(ctx: *mut fx_ctx, x: *const f64, col: *mut f64, B: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_col2im_f64(ctx: *mut fx_ctx, col: *const f64, out: *mut f64, B: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, layout: c_int) -> c_int;
    pub fn fx_conv2d_fwd_f64(ctx: *mut fx_ctx, x: *const f64, w: *const f64, y: *mut f64, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_conv2d_dgrad_f64(ctx: *mut fx_ctx, g: *const f64, w: *const f64, dx: *mut f64, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, mode: c_int, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_conv2d_wgrad_f64(ctx: *mut fx_ctx, x: *const f64, g: *const f64, dw: *mut f64, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, mode: c_int, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_maxpool2d_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_avgpool2d_f64(ctx: *mut fx_ctx, input: *const f64, out: *mut f64, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_max_unpool2d_f64(ctx: *mut fx_ctx, grad_out: *const f64, input: *const f64, pooled: *const f64, grad_in: *mut f64, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_avg_unpool2d_f64(ctx: *mut fx_ctx, grad_out: *const f64, grad_in: *mut f64, N: i64, C: i64, H: i64, W: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_bias_act_f64(ctx: *mut fx_ctx, y: *mut f64, bias: *const f64, outer: i64, C: i64, inner: i64, act: c_int) -> c_int;
    pub fn fx_conv2d_fwd_bias_act_f64(ctx: *mut fx_ctx, x: *const f64, w: *const f64, bias: *const f64, y: *mut f64, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, act: c_int, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_gemm_bias_act_f64(ctx: *mut fx_ctx, trans_a: c_int, trans_b: c_int, M: i64, N: i64, K: i64, A: *const f64, B: *const f64, bias: *const f64, C: *mut f64, act: c_int) -> c_int;
    pub fn fx_conv2d_wgrad_relu_bias_f64(ctx: *mut fx_ctx, x: *const f64, g: *const f64, act: *const f64, dw: *mut f64, db: *mut f64, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64, workspace: *mut c_void, ws_bytes: i64) -> c_int;
    pub fn fx_conv2d_dgrad_relu_f64(ctx: *mut fx_ctx, g: *const f64, act: *const f64, w: *const f64, dx: *mut f64, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_gemm_tn_colsum_f64(ctx: *mut fx_ctx, M: i64, N: i64, K: i64, A: *const f64, B: *const f64, C: *mut f64, colsum: *mut f64) -> c_int;
    pub fn fx_linear_bwd_f64(ctx: *mut fx_ctx, B: i64, input: i64, out: i64, dY: *const f64, W: *const f64, X: *const f64, dX: *mut f64, dW: *mut f64, db: *mut f64, relu_below: c_int) -> c_int;
    pub fn fx_batchnorm_stats_f64(ctx: *mut fx_ctx, x: *const f64, mean: *mut f64, var: *mut f64, running_mean: *mut f64, running_var: *mut f64, momentum: f64, outer: i64, C: i64, inner: i64) -> c_int;
    pub fn fx_batchnorm_fwd_f64(ctx: *mut fx_ctx, x: *const f64, mean: *const f64, var: *const f64, gamma: *const f64, beta: *const f64, eps: f64, y: *mut f64, outer: i64, C: i64, inner: i64, act: c_int) -> c_int;
    pub fn fx_batchnorm_bwd_f64(ctx: *mut fx_ctx, dy: *const f64, x: *const f64, y_act: *const f64, mean: *const f64, var: *const f64, gamma: *const f64, eps: f64, dx: *mut f64, dgamma: *mut f64, dbeta: *mut f64, outer: i64, C: i64, inner: i64, batch_stats: c_int) -> c_int;
    pub fn fx_dropout_f64(ctx: *mut fx_ctx, x: *const f64, mask: *mut f64, y: *mut f64, n: i64, p: f64, seed: u64) -> c_int;
    pub fn fx_bias_grad_f64(ctx: *mut fx_ctx, g: *const f64, out: *mut f64, outer: i64, C: i64, inner: i64) -> c_int;
    pub fn fx_relu_bwd_bias_grad_f64(ctx: *mut fx_ctx, g: *const f64, y: *const f64, gm: *mut f64, dbias: *mut f64, outer: i64, C: i64, inner: i64) -> c_int;
    pub fn fx_softmax_ce_fwd_f64(ctx: *mut fx_ctx, logits: *const f64, targets: *const f64, probs: *mut f64, loss: *mut f64, B: i64, C: i64) -> c_int;
    pub fn fx_softmax_ce_bwd_f64(ctx: *mut fx_ctx, probs: *const f64, targets: *const f64, grad_loss: *const f64, dlogits: *mut f64, B: i64, C: i64) -> c_int;
    pub fn fx_softmax_ce_fwd_unit_grad_f64(ctx: *mut fx_ctx, logits: *const f64, targets: *const f64, probs: *mut f64, loss: *mut f64, dlogits: *mut f64, B: i64, C: i64) -> c_int;
    pub fn fx_adam_step_f64(ctx: *mut fx_ctx, p: *mut f64, g: *const f64, m: *mut f64, v: *mut f64, n: i64, lr: f64, beta1: f64, beta2: f64, eps: f64, weight_decay: f64, bc1: f64, bc2: f64) -> c_int;
    pub fn fx_adam_amsgrad_step_f64(ctx: *mut fx_ctx, p: *mut f64, g: *const f64, m: *mut f64, v: *mut f64, vmax: *mut f64, n: i64, lr: f64, beta1: f64, beta2: f64, eps: f64, weight_decay: f64, bc1: f64, bc2: f64) -> c_int;
    pub fn fx_sgd_step_f64(ctx: *mut fx_ctx, p: *mut f64, g: *const f64, n: i64, lr: f64) -> c_int;
    pub fn fx_sgd_momentum_step_f64(ctx: *mut fx_ctx, p: *mut f64, g: *const f64, buf: *mut f64, n: i64, lr: f64, momentum: f64, weight_decay: f64, nesterov: c_int) -> c_int;
    pub fn fx_adam_step_multi_f64(ctx: *mut fx_ctx, count: c_int, p: *const *mut f64, g: *const *const f64, m: *const *mut f64, v: *const *mut f64, n: *const i64, lr: f64, beta1: f64, beta2: f64, eps: f64, weight_decay: f64, bc1: f64, bc2: f64) -> c_int;
    pub fn fx_adam_amsgrad_step_multi_f64(ctx: *mut fx_ctx, count: c_int, p: *const *mut f64, g: *const *const f64, m: *const *mut f64, v: *const *mut f64, vmax: *const *mut f64, n: *const i64, lr: f64, beta1: f64, beta2: f64, eps: f64, weight_decay: f64, bc1: f64, bc2: f64) -> c_int;
    pub fn fx_adam_step_multi_bc_f64(ctx: *mut fx_ctx, count: c_int, p: *const *mut f64, g: *const *const f64, m: *const *mut f64, v: *const *mut f64, vmax: *const *mut f64, n: *const i64, lr: f64, beta1: f64, beta2: f64, eps: f64, weight_decay: f64, bc: *const f64) -> c_int;
    pub fn fx_sgd_step_multi_f64(ctx: *mut fx_ctx, count: c_int, p: *const *mut f64, g: *const *const f64, n: *const i64, lr: f64) -> c_int;
    pub fn fx_sgd_momentum_step_multi_f64(ctx: *mut fx_ctx, count: c_int, p: *const *mut f64, g: *const *const f64, buf: *const *mut f64, n: *const i64, lr: f64, momentum: f64, weight_decay: f64, nesterov: c_int) -> c_int;
    pub fn fx_embedding_fwd_f64(ctx: *mut fx_ctx, W: *const f64, ids: *const i64, out: *mut f64, n: i64, vocab: i64, dim: i64, scale: f64) -> c_int;
    pub fn fx_embedding_bwd_f64(ctx: *mut fx_ctx, g: *const f64, ids: *const i64, dW: *mut f64, n: i64, vocab: i64, dim: i64, scale: f64) -> c_int;
    pub fn fx_rmsnorm_fwd_f64(ctx: *mut fx_ctx, x: *const f64, res: *const f64, w: *const f64, eps: f64, h: *mut f64, y: *mut f64, rstd: *mut f64, rows: i64, dim: i64) -> c_int;
    pub fn fx_rmsnorm_bwd_f64(ctx: *mut fx_ctx, dy: *const f64, dh: *const f64, h: *const f64, w: *const f64, rstd: *const f64, dx: *mut f64, dw: *mut f64, rows: i64, dim: i64) -> c_int;
    pub fn fx_gemm_bias_act_residual_f64(ctx: *mut fx_ctx, trans_a: c_int, trans_b: c_int, M: i64, N: i64, K: i64, A: *const f64, B: *const f64, bias: *const f64, residual: *const f64, pre: *mut f64, C: *mut f64, act: c_int) -> c_int;
    pub fn fx_linear_act_bwd_f64(ctx: *mut fx_ctx, B: i64, input: i64, out: i64, dY: *const f64, W: *const f64, X: *const f64, pre: *const f64, act: c_int, dpre: *mut f64, dX: *mut f64, dW: *mut f64, db: *mut f64) -> c_int;
    pub fn fx_gated_recurrence_fwd_f64(ctx: *mut fx_ctx, z: *const f64, x: *const f64, h0: *const f64, h: *mut f64, B: i64, steps: i64, dim: i64) -> c_int;
    pub fn fx_gated_recurrence_bwd_f64(ctx: *mut fx_ctx, dh: *const f64, z: *const f64, x: *const f64, h: *const f64, h0: *const f64, dh_next: *const f64, dz: *mut f64, dx: *mut f64, dh0: *mut f64, B: i64, steps: i64, dim: i64) -> c_int;
    pub fn fx_grad_norm_multi_f64(ctx: *mut fx_ctx, count: c_int, g: *const *const f64, n: *const i64, norm: *mut f64) -> c_int;
    pub fn fx_clip_grad_norm_multi_f64(ctx: *mut fx_ctx, count: c_int, g: *const *const f64, out: *const *mut f64, n: *const i64, max_norm: f64, norm: *mut f64) -> c_int;
    pub fn fx_conv2d_last_path(ctx: *mut fx_ctx) -> *const c_char;
    pub fn fx_conv2d_bwd_relu_supported(ctx: *mut fx_ctx, kind: c_int, dtype: c_int, B: i64, Cin: i64, H: i64, W: i64, Cout: i64, kh: i64, kw: i64, sh: i64, sw: i64, ph: i64, pw: i64) -> c_int;
    pub fn fx_graph_begin(ctx: *mut fx_ctx) -> c_int;
    pub fn fx_graph_end(ctx: *mut fx_ctx, out: *mut *mut fx_graph) -> c_int;
    pub fn fx_graph_launch(ctx: *mut fx_ctx, graph: *mut fx_graph) -> c_int;
    pub fn fx_graph_info(graph: *mut fx_graph, nodes: *mut i64, kernel_nodes: *mut i64, held_blocks: *mut i64) -> c_int;
    pub fn fx_graph_destroy(ctx: *mut fx_ctx, graph: *mut fx_graph) -> c_int;
    pub fn fx_scratch_info(ctx: *mut fx_ctx, current: *mut *mut c_void, bytes: *mut i64, parked_regions: *mut i64, live_graphs: *mut i64) -> c_int;
    pub fn fx_device_mem_info(ctx: *mut fx_ctx, free_bytes: *mut i64, total_bytes: *mut i64) -> c_int;
    pub fn fx_host_alloc(ctx: *mut fx_ctx, bytes: i64, out: *mut *mut c_void) -> c_int;
    pub fn fx_host_free(ctx: *mut fx_ctx, ptr: *mut c_void) -> c_int;
    pub fn fx_h2d_async(ctx: *mut fx_ctx, dst: *mut c_void, src_pinned: *const c_void, bytes: i64) -> c_int;
    pub fn fx_reduce_max_noalloc_f32(ctx: *mut fx_ctx, input: *const f32, out: *mut f32, idx_out: *mut i64, outer: i64, axis: i64, inner: i64) -> c_int;
}

/// `Ok(())` for `FX_OK`, otherwise the library's message for the calling thread.
pub fn check(rc: c_int) -> Result<(), String> {
    if rc == FX_OK {
        return Ok(());
    }
    let msg = unsafe { std::ffi::CStr::from_ptr(fx_last_error()) };
    Err(msg.to_string_lossy().into_owned())
}
