// Raw bindings to libferro_b200.so: one declaration per entry of include/ferro_b200.h.
// Generated by `python -m ferro_b200.rust_bindings`; do not edit by hand.
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_int, c_void};

/// cudaStream_t (cudarc: `stream.cu_stream()` cast to this).
pub type Stream = *mut c_void;

pub const FB_UN_NEG: c_int = 0;
pub const FB_UN_RELU: c_int = 1;
pub const FB_UN_EXP: c_int = 2;
pub const FB_UN_SIGMOID: c_int = 3;
pub const FB_UN_TANH: c_int = 4;
pub const FB_UN_SQRT: c_int = 5;
pub const FB_UN_ABS: c_int = 6;
pub const FB_UN_SIGN: c_int = 7;
pub const FB_UN_LOG: c_int = 8;
pub const FB_UN_POWF: c_int = 9;
pub const FB_UN_CLAMP: c_int = 10;
pub const FB_UN_GTZ: c_int = 11;
pub const FB_UN_GELU: c_int = 12;
pub const FB_UN_GELU_ERF: c_int = 13;
pub const FB_UN_GELU_ERF_GRAD: c_int = 14;
pub const FB_UN_SILU: c_int = 15;
pub const FB_UN_KIND_COUNT: c_int = 16;
pub const FB_BIN_ADD: c_int = 0;
pub const FB_BIN_SUB: c_int = 1;
pub const FB_BIN_MUL: c_int = 2;
pub const FB_BIN_DIV: c_int = 3;
pub const FB_BIN_RELU_BACKWARD: c_int = 4;
pub const FB_BIN_TANH_BWD: c_int = 5;
pub const FB_BIN_SIGMOID_BWD: c_int = 6;
pub const FB_BIN_SQRT_BWD: c_int = 7;
pub const FB_BIN_ABS_BWD: c_int = 8;
pub const FB_BIN_LOG_BWD: c_int = 9;
pub const FB_BIN_POWF_BWD: c_int = 10;
pub const FB_BIN_CLAMP_BWD: c_int = 11;
pub const FB_BIN_KIND_COUNT: c_int = 12;
pub const FB_RED_SUM: c_int = 0;
pub const FB_RED_MEAN: c_int = 1;
pub const FB_ROPE_INTERLEAVED: c_int = 0;
pub const FB_ROPE_HALF: c_int = 1;
pub const FB_ROPE_PLAIN: c_int = 0;
pub const FB_ROPE_LINEAR: c_int = 1;
pub const FB_ROPE_BASE: c_int = 2;
pub const FB_ROPE_BY_PARTS: c_int = 3;
pub const FB_OK: c_int = 0;
pub const FB_ERR_INVALID_SHAPE: c_int = 1;
pub const FB_ERR_INVALID_ARG: c_int = 2;
pub const FB_ERR_CUDA: c_int = 3;
pub const FB_ERR_UNSUPPORTED: c_int = 4;
pub const FB_ERR_WORKSPACE: c_int = 5;
pub const FB_ERR_COMM: c_int = 6;
pub const FB_ERR_FORMAT: c_int = 7;
pub const FB_MAX_RANK: c_int = 16;
pub const FB_VERSION: c_int = 1;
pub const FB_CHAIN_MAX_STEPS: c_int = 32;
pub const FB_CHAIN_MAX_OPERANDS: c_int = 6;
pub const FB_LN_STATIC_SCRATCH_BYTES: c_int = 16777216;
pub const FB_MOE_MAX_EXPERTS: c_int = 1024;
pub const FB_MOE_MAX_K: c_int = 32;
pub const FB_DDP_UNIQUE_ID_BYTES: c_int = 128;
pub const FB_CH_LOAD: c_int = 0;
pub const FB_CH_UNARY: c_int = 1;
pub const FB_CH_BINARY: c_int = 2;
pub const FB_CH_IMM: c_int = 3;
pub const FB_CH_V: c_int = 0;
pub const FB_CH_T: c_int = 1;
pub const FB_CH_SRC_OTHER_REG: c_int = 0;
pub const FB_CH_SRC_IMM: c_int = 1;
pub const FB_CH_SRC_OPERAND0: c_int = 8;
pub const FB_CH_SWAP: c_int = 64;
pub const FB_ST_F32: c_int = 0;
pub const FB_ST_I64: c_int = 1;

/// Opaque handle (`fb_host_ln`).
#[repr(C)] pub struct HostLn { _private: [u8; 0] }
/// Opaque handle (`fb_ddp_comm`).
#[repr(C)] pub struct DdpComm { _private: [u8; 0] }

pub type DlpackReleaseFn = Option<unsafe extern "C" fn(owner: *mut c_void)>;

#[repr(C)] #[derive(Clone, Copy)]
pub struct ChainStep {
    pub opcode: i32,
    pub dst: i32,
    pub kind: i32,
    pub src: i32,
    pub p0: f32,
    pub p1: f32,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct ChainOperand {
    pub ptr: *const f32,
    pub len: u64,
    pub offset: i64,
    pub strides: [i64; 16],
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct View {
    pub ptr: *const f32,
    pub len: u64,
    pub offset: i64,
    pub rank: i32,
    pub shape: [u64; 16],
    pub strides: [i64; 16],
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct AdamwHparams {
    pub lr: f32,
    pub beta1: f32,
    pub beta2: f32,
    pub bc1: f32,
    pub bc2: f32,
    pub eps: f32,
    pub weight_decay: f32,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct TensorQuad {
    pub p: *mut f32,
    pub m: *mut f32,
    pub v: *mut f32,
    pub g: *const f32,
    pub n: u64,
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct StEntry {
    pub name: *const c_char,
    pub dtype: i32,
    pub rank: i32,
    pub shape: [u64; 16],
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct DlpackDesc {
    pub data: *mut c_void,
    pub on_device: i32,
    pub device_id: i32,
    pub dtype: i32,
    pub rank: i32,
    pub contiguous: i32,
    pub reserved: i32,
    pub numel: u64,
    pub shape: [u64; 16],
    pub strides: [i64; 16],
}
#[repr(C)] #[derive(Clone, Copy)]
pub struct Rng {
    pub s0: u64,
    pub s1: u64,
}

#[link(name = "ferro_b200")]
extern "C" {
    pub fn fb_version() -> c_int;
    pub fn fb_last_error() -> *const c_char;
    pub fn fb_launch_count() -> u64;
    pub fn fb_device_faults(reset: c_int) -> c_int;
    pub fn fb_selftest_bounded_wait(stream: Stream, limit_ms: u32) -> c_int;
    pub fn fb_unary(stream: Stream, kind: c_int, p0: f32, p1: f32, x: *const f32, out: *mut f32, n: u64) -> c_int;
    pub fn fb_binary(stream: Stream, kind: c_int, p0: f32, p1: f32, a: *const f32, b: *const f32, out: *mut f32, n: u64) -> c_int;
    pub fn fb_binary_bc(stream: Stream, kind: c_int, p0: f32, p1: f32, a: *const f32, sa: *const u64, rank_a: c_int, b: *const f32, sb: *const u64, rank_b: c_int, out: *mut f32, out_shape: *const u64, rank_out: c_int) -> c_int;
    pub fn fb_unary_strided(stream: Stream, kind: c_int, p0: f32, p1: f32, x: *const f32, x_len: u64, x_strides: *const i64, x_offset: i64, shape: *const u64, rank: c_int, out: *mut f32) -> c_int;
    pub fn fb_binary_strided(stream: Stream, kind: c_int, p0: f32, p1: f32, a: *const f32, a_len: u64, a_strides: *const i64, a_offset: i64, b: *const f32, b_len: u64, b_strides: *const i64, b_offset: i64, shape: *const u64, rank: c_int, out: *mut f32) -> c_int;
    pub fn fb_materialize(stream: Stream, x: *const f32, x_len: u64, strides: *const i64, offset: i64, shape: *const u64, rank: c_int, out: *mut f32) -> c_int;
    pub fn fb_chain(stream: Stream, steps: *const ChainStep, n_steps: c_int, operands: *const ChainOperand, n_operands: c_int, shape: *const u64, rank: c_int, out: *mut f32) -> c_int;
    pub fn fb_chain_catalogue(enable: c_int) -> c_int;
    pub fn fb_fill(stream: Stream, dst: *mut f32, value: f32, n: u64) -> c_int;
    pub fn fb_affine_inplace(stream: Stream, dst: *mut f32, mul: f32, add: f32, n: u64) -> c_int;
    pub fn fb_binary_inplace(stream: Stream, kind: c_int, dst: *mut f32, src: *const f32, n: u64) -> c_int;
    pub fn fb_axpy_inplace(stream: Stream, alpha: f32, dst: *mut f32, src: *const f32, n: u64) -> c_int;
    pub fn fb_copy(stream: Stream, dst: *mut f32, src: *const f32, n: u64) -> c_int;
    pub fn fb_gather_rows(stream: Stream, w: *const f32, idx: *const i64, n: u64, dim_size: u64, inner: u64, out: *mut f32, bad_index: *mut i64) -> c_int;
    pub fn fb_reduce_workspace_bytes(n: u64) -> u64;
    pub fn fb_reduce(stream: Stream, kind: c_int, x: *const f32, n: u64, out: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_reduce_dim_workspace_bytes(outer: u64, red: u64, inner: u64) -> u64;
    pub fn fb_sum_dim(stream: Stream, x: *const f32, outer: u64, red: u64, inner: u64, out: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_mean_dim(stream: Stream, x: *const f32, outer: u64, red: u64, inner: u64, out: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_max_dim(stream: Stream, x: *const f32, outer: u64, red: u64, inner: u64, values: *mut f32, indices: *mut i64, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_softmax_fwd(stream: Stream, x: *const f32, rows: u64, cols: u64, y: *mut f32) -> c_int;
    pub fn fb_log_softmax_fwd(stream: Stream, x: *const f32, rows: u64, cols: u64, y: *mut f32) -> c_int;
    pub fn fb_softmax_bwd(stream: Stream, g: *const f32, y: *const f32, rows: u64, cols: u64, dx: *mut f32) -> c_int;
    pub fn fb_log_softmax_bwd(stream: Stream, g: *const f32, y: *const f32, rows: u64, cols: u64, dx: *mut f32) -> c_int;
    pub fn fb_bias_act_scale_softmax_fwd(stream: Stream, x: *const f32, bias: *const f32, relu: c_int, scale: f32, rows: u64, cols: u64, y: *mut f32) -> c_int;
    pub fn fb_softmax_fused_bwd_workspace_bytes(rows: u64, cols: u64) -> u64;
    pub fn fb_bias_act_scale_softmax_bwd(stream: Stream, g: *const f32, y: *const f32, x: *const f32, bias: *const f32, relu: c_int, scale: f32, rows: u64, cols: u64, dx: *mut f32, dbias: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_nll_workspace_bytes(rows: u64) -> u64;
    pub fn fb_log_softmax_nll_fwd(stream: Stream, logits: *const f32, targets: *const i64, rows: u64, cols: u64, loss: *mut f32, row_max: *mut f32, row_lse: *mut f32, argmax: *mut i64, bad_target: *mut i64, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_log_softmax_nll_bwd(stream: Stream, logits: *const f32, targets: *const i64, row_max: *const f32, row_lse: *const f32, grad_scale: f32, rows: u64, cols: u64, dlogits: *mut f32) -> c_int;
    pub fn fb_gather_dim(stream: Stream, x: *const f32, in_shape: *const u64, index: *const i64, out_shape: *const u64, rank: c_int, dim: c_int, out: *mut f32, bad_index: *mut i64) -> c_int;
    pub fn fb_scatter_add_dim(stream: Stream, g: *const f32, index: *const i64, in_shape: *const u64, out_shape: *const u64, rank: c_int, dim: c_int, gx: *mut f32, bad_index: *mut i64) -> c_int;
    pub fn fb_segment_csr_build(ids: *const u64, edges: u64, groups: u64, csr_host: *mut i64) -> c_int;
    pub fn fb_segment_sum(stream: Stream, x: *const f32, csr: *const i64, groups: u64, edges: u64, width: u64, out: *mut f32) -> c_int;
    pub fn fb_segment_sum_bwd(stream: Stream, g: *const f32, csr: *const i64, groups: u64, edges: u64, width: u64, dx: *mut f32) -> c_int;
    pub fn fb_segment_softmax_fwd(stream: Stream, x: *const f32, csr: *const i64, groups: u64, edges: u64, width: u64, y: *mut f32, not_finite: *mut c_int) -> c_int;
    pub fn fb_segment_softmax_bwd(stream: Stream, g: *const f32, y: *const f32, csr: *const i64, groups: u64, edges: u64, width: u64, dx: *mut f32) -> c_int;
    pub fn fb_reduce_view_workspace_bytes(x: *const View, dim: c_int) -> u64;
    pub fn fb_sum_dim_view(stream: Stream, x: *const View, dim: c_int, out: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_mean_dim_view(stream: Stream, x: *const View, dim: c_int, out: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_max_dim_view(stream: Stream, x: *const View, dim: c_int, values: *mut f32, indices: *mut i64, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_softmax_view_fwd(stream: Stream, x: *const View, dim: c_int, y: *mut f32) -> c_int;
    pub fn fb_log_softmax_view_fwd(stream: Stream, x: *const View, dim: c_int, y: *mut f32) -> c_int;
    pub fn fb_softmax_view_bwd(stream: Stream, g: *const View, y: *const View, dim: c_int, dx: *mut f32) -> c_int;
    pub fn fb_log_softmax_view_bwd(stream: Stream, g: *const View, y: *const View, dim: c_int, dx: *mut f32) -> c_int;
    pub fn fb_layer_norm_fwd(stream: Stream, x: *const f32, weight: *const f32, bias: *const f32, rows: u64, cols: u64, eps: f32, y: *mut f32, h: *mut f32, stds: *mut f32, mean: *mut f32, rstd: *mut f32) -> c_int;
    pub fn fb_layer_norm_bwd_workspace_bytes(rows: u64, cols: u64) -> u64;
    pub fn fb_layer_norm_bwd(stream: Stream, g: *const f32, h: *const f32, stds: *const f32, x: *const f32, mean: *const f32, rstd: *const f32, weight: *const f32, rows: u64, cols: u64, dx: *mut f32, dweight: *mut f32, dbias: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_residual_layer_norm_fwd(stream: Stream, x: *const f32, residual: *const f32, weight: *const f32, bias: *const f32, rows: u64, cols: u64, eps: f32, y: *mut f32, h: *mut f32, stds: *mut f32, mean: *mut f32, rstd: *mut f32, sum_out: *mut f32) -> c_int;
    pub fn fb_rms_norm_fwd(stream: Stream, x: *const f32, weight: *const f32, rows: u64, cols: u64, eps: f32, y: *mut f32, rstd: *mut f32) -> c_int;
    pub fn fb_rms_norm_bwd(stream: Stream, g: *const f32, x: *const f32, rstd: *const f32, weight: *const f32, rows: u64, cols: u64, dx: *mut f32, dweight: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_layer_norm_bwd_static(stream: Stream, g: *const f32, h: *const f32, stds: *const f32, x: *const f32, mean: *const f32, rstd: *const f32, weight: *const f32, rows: u64, cols: u64, dx: *mut f32, dweight: *mut f32, dbias: *mut f32) -> c_int;
    pub fn fb_sgd_step(stream: Stream, p: *mut f32, v: *mut f32, g: *const f32, n: u64, lr: f32, momentum: f32, nesterov: c_int) -> c_int;
    pub fn fb_adamw_step(stream: Stream, p: *mut f32, m: *mut f32, v: *mut f32, g: *const f32, n: u64, hp: AdamwHparams) -> c_int;
    pub fn fb_adamw_step_capturable(stream: Stream, p: *mut f32, m: *mut f32, v: *mut f32, g: *const f32, t: *const f32, n: u64, lr: f32, beta1: f32, beta2: f32, eps: f32, weight_decay: f32) -> c_int;
    pub fn fb_scalar_increment(stream: Stream, t: *mut f32, beta1: f32, beta2: f32) -> c_int;
    pub fn fb_adamw_multi(stream: Stream, table: *const TensorQuad, n_tensors: c_int, total_elems: u64, hp: AdamwHparams, g_scale: f32) -> c_int;
    pub fn fb_sgd_multi(stream: Stream, table: *const TensorQuad, n_tensors: c_int, total_elems: u64, lr: f32, momentum: f32, nesterov: c_int, g_scale: f32) -> c_int;
    pub fn fb_grad_norm_workspace_bytes() -> u64;
    pub fn fb_grad_sumsq_multi(stream: Stream, table: *const TensorQuad, n_tensors: c_int, total_elems: u64, g_scale: f32, sumsq: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_clip_scale(stream: Stream, sumsq: *const f32, max_norm: f32, norm_out: *mut f32, scale_out: *mut f32) -> c_int;
    pub fn fb_adamw_multi_clipped(stream: Stream, table: *const TensorQuad, n_tensors: c_int, total_elems: u64, hp: AdamwHparams, g_scale: f32, clip_scale: *const f32) -> c_int;
    pub fn fb_sgd_multi_clipped(stream: Stream, table: *const TensorQuad, n_tensors: c_int, total_elems: u64, lr: f32, momentum: f32, nesterov: c_int, g_scale: f32, clip_scale: *const f32) -> c_int;
    pub fn fb_bias_act_fwd(stream: Stream, x: *const f32, bias: *const f32, act: c_int, rows: u64, cols: u64, out: *mut f32) -> c_int;
    pub fn fb_bias_act_bwd(stream: Stream, g: *const f32, x: *const f32, bias: *const f32, act: c_int, rows: u64, cols: u64, dx: *mut f32, dbias: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_mse_fwd_bwd(stream: Stream, pred: *const f32, target: *const f32, n: u64, grad_scale: f32, loss: *mut f32, dpred: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_rope_turns(rot_dim: u64, base: f64, scaling: c_int, factor: f64, original_len: f64, low: f64, high: f64, turns_host: *mut i64) -> c_int;
    pub fn fb_rope(stream: Stream, x: *const View, positions: *const i64, position_rows: u64, start: i64, turns: *const i64, rot_dim: u64, layout: c_int, scale: f32, inverse: c_int, out: *mut f32, out_len: u64, out_strides: *const i64, out_offset: i64) -> c_int;
    pub fn fb_dropout_fwd(stream: Stream, x: *const f32, bias: *const f32, residual: *const f32, rows: u64, cols: u64, p: f32, seed: u64, offset: u64, counter: *const i64, out: *mut f32) -> c_int;
    pub fn fb_dropout_bwd_workspace_bytes(rows: u64, cols: u64) -> u64;
    pub fn fb_dropout_bwd(stream: Stream, g: *const f32, rows: u64, cols: u64, p: f32, seed: u64, offset: u64, counter: *const i64, dx: *mut f32, dbias: *mut f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_dropout_advance(stream: Stream, counter: *mut i64, n: u64) -> c_int;
    pub fn fb_moe_gate_fwd(stream: Stream, logits: *const f32, tokens: u64, experts: u64, k: u64, renorm: c_int, weights: *mut f32, ids: *mut i64) -> c_int;
    pub fn fb_moe_gate_bwd(stream: Stream, dweights: *const f32, logits: *const f32, weights: *const f32, ids: *const i64, tokens: u64, experts: u64, k: u64, renorm: c_int, dlogits: *mut f32) -> c_int;
    pub fn fb_moe_sort_workspace_bytes(n: u64, experts: u64) -> u64;
    pub fn fb_moe_sort(stream: Stream, ids: *const i64, n: u64, experts: u64, place: *mut i64, order: *mut i64, offsets: *mut i64, bad_index: *mut i64, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn fb_moe_dispatch_fwd(stream: Stream, x: *const f32, place: *const i64, tokens: u64, k: u64, cols: u64, xs: *mut f32, slots: u64) -> c_int;
    pub fn fb_moe_dispatch_bwd(stream: Stream, dxs: *const f32, place: *const i64, tokens: u64, k: u64, cols: u64, slots: u64, dx: *mut f32) -> c_int;
    pub fn fb_moe_combine_fwd(stream: Stream, ys: *const f32, weights: *const f32, place: *const i64, tokens: u64, k: u64, cols: u64, slots: u64, y: *mut f32) -> c_int;
    pub fn fb_moe_combine_bwd(stream: Stream, dy: *const f32, ys: *const f32, weights: *const f32, place: *const i64, tokens: u64, k: u64, cols: u64, slots: u64, dys: *mut f32, dweights: *mut f32) -> c_int;
    pub fn fb_host_ln_create(chunks: c_int, out: *mut *mut HostLn) -> c_int;
    pub fn fb_host_ln_device_bytes(rows: u64, cols: u64, chunks: c_int) -> u64;
    pub fn fb_host_ln_run(h: *mut HostLn, rows: u64, cols: u64, eps: f32, x: *const f32, g: *const f32, weight: *const f32, bias: *const f32, y: *mut f32, dx: *mut f32, mean: *mut f32, rstd: *mut f32, dweight_dbias: *mut f32, device_staging: *mut c_void, staging_bytes: u64) -> c_int;
    pub fn fb_host_ln_synchronize(h: *mut HostLn) -> c_int;
    pub fn fb_host_ln_destroy(h: *mut HostLn) -> c_int;
    pub fn fb_safetensors_image_bytes(entries: *const StEntry, n: c_int, data_offsets: *mut u64) -> u64;
    pub fn fb_safetensors_write(stream: Stream, entries: *const StEntry, n: c_int, sources: *const *const c_void, sources_on_device: c_int, image: *mut c_void, image_bytes: u64) -> c_int;
    pub fn fb_safetensors_count(image: *const c_void, image_bytes: u64) -> c_int;
    pub fn fb_safetensors_entry(image: *const c_void, image_bytes: u64, index: c_int, name_out: *mut c_char, name_cap: u64, entry_out: *mut StEntry, data_begin: *mut u64, data_end: *mut u64) -> c_int;
    pub fn fb_safetensors_read(stream: Stream, image: *const c_void, image_bytes: u64, tensor_name: *const c_char, dtype: c_int, numel: u64, dst: *mut c_void, dst_on_device: c_int) -> c_int;
    pub fn fb_dlpack_export(data: *const c_void, byte_offset: u64, dtype: c_int, ndim: c_int, shape: *const i64, strides: *const i64, device_ordinal: c_int, owner: *mut c_void, release: DlpackReleaseFn, managed_out: *mut *mut c_void) -> c_int;
    pub fn fb_dlpack_handoff(producer: Stream, has_consumer: c_int, consumer: i64) -> c_int;
    pub fn fb_dlpack_describe(managed: *const c_void, out: *mut DlpackDesc) -> c_int;
    pub fn fb_dlpack_import_into(stream: Stream, managed: *const c_void, dst: *mut c_void, dst_bytes: u64) -> c_int;
    pub fn fb_dlpack_delete(managed: *mut c_void);
    pub fn fb_rng_seed(rng: *mut Rng, seed: u64);
    pub fn fb_rng_skip(rng: *mut Rng, draws: u64);
    pub fn fb_rng_uniform(rng: *mut Rng) -> f32;
    pub fn fb_rng_normal(rng: *mut Rng) -> f32;
    pub fn fb_rng_fill_uniform(rng: *mut Rng, out: *mut f32, n: u64, scale: f32, shift: f32) -> c_int;
    pub fn fb_rng_fill_normal(rng: *mut Rng, out: *mut f32, n: u64, scale: f32, shift: f32) -> c_int;
    pub fn fb_rng_fill_rowscaled_normal(rng: *mut Rng, out: *mut f32, rows: u64, cols: u64, lo: f32, span: f32) -> c_int;
    pub fn fb_rng_fill_index(rng: *mut Rng, out: *mut i64, n: u64, classes: u64) -> c_int;
    pub fn fb_ddp_unique_id(id: *mut c_void) -> c_int;
    pub fn fb_ddp_comm_init(id: *const c_void, rank: c_int, world: c_int, out: *mut *mut DdpComm) -> c_int;
    pub fn fb_ddp_rank(comm: *const DdpComm) -> c_int;
    pub fn fb_ddp_world(comm: *const DdpComm) -> c_int;
    pub fn fb_ddp_nccl_version() -> c_int;
    pub fn fb_ddp_allreduce_bucket(comm: *mut DdpComm, stream: Stream, bucket: *mut f32, n: u64) -> c_int;
    pub fn fb_ddp_allreduce_buckets(comm: *mut DdpComm, stream: Stream, buckets: *const *mut f32, lens: *const u64, n_buckets: c_int) -> c_int;
    pub fn fb_ddp_average_bucket(comm: *mut DdpComm, stream: Stream, bucket: *mut f32, n: u64) -> c_int;
    pub fn fb_ddp_poll(comm: *mut DdpComm) -> c_int;
    pub fn fb_ddp_comm_abort(comm: *mut DdpComm) -> c_int;
    pub fn fb_ddp_comm_destroy(comm: *mut DdpComm) -> c_int;
}
