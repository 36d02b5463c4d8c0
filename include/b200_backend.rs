// b200_backend.rs -- `impl Backend for B200Backend` over the C ABI of rt_b200.h.
//
// GENERATED by include/gen_rust_shim.py from include/rt_b200.h; do not edit by hand.
// UNVERIFIED SOURCE: no Rust toolchain exists where librt_b200.so is built.  It is what a maintainer of the reference would
// add as src/backend/b200/mod.rs (feature "b200"); the compiled and tested twin with the same method list and the same
// calls is rusttensor_b200/csrc/host/b200_backend.hpp.  Citations are lines of the reference's src/backend/mod.rs.
#![allow(clippy::too_many_arguments)]
use crate::backend::Backend;
use crate::error::Error;
use crate::graph::{Op, OpType};
use std::ffi::CStr;
use std::os::raw::{c_char, c_int, c_void};
use std::sync::{Arc, Mutex, OnceLock};

pub mod ffi {
    use super::*;
    #[repr(C)] pub struct RtCtx { _p: [u8; 0] }
    #[repr(C)] pub struct RtGraph { _p: [u8; 0] }
    #[repr(C)] pub struct RtUpload { _p: [u8; 0] }
    #[repr(C)] pub struct RtFusedProgram { _p: [u8; 0] }
    #[repr(C)] pub struct RtEvent { _p: [u8; 0] }
    pub type RtStatus = i32;
    pub const RT_OK: c_int = 0;
    pub const RT_ERR_SHAPE_MISMATCH: c_int = 1;
    pub const RT_ERR_INCOMPATIBLE_SHAPES: c_int = 2;
    pub const RT_ERR_INVALID_INDEX: c_int = 3;
    pub const RT_ERR_INVALID_OPERATION: c_int = 4;
    pub const RT_ERR_INTERNAL: c_int = 5;
    pub const RT_ERR_DIMENSION_MISMATCH: c_int = 6;
    pub const RT_ERR_CUDA: c_int = 7;
    pub const RT_ERR_OOM: c_int = 8;
    pub const RT_ERR_UNIMPLEMENTED: c_int = 9;
    pub const RT_ERR_EMPTY_TENSOR: c_int = 10;
    pub const RT_ERR_TIMEOUT: c_int = 14;
    pub const RT_ERR_NCCL: c_int = 15;
    pub const RT_ERR_INITIALIZATION: c_int = 16;
    pub const RT_RELU: c_int = 0;
    pub const RT_ELU: c_int = 1;
    pub const RT_EXP: c_int = 2;
    pub const RT_LN: c_int = 3;
    pub const RT_SIN: c_int = 4;
    pub const RT_TANH: c_int = 5;
    pub const RT_SIGMOID: c_int = 6;
    pub const RT_SOFTPLUS: c_int = 7;
    pub const RT_SQUARE: c_int = 8;
    pub const RT_SQRT: c_int = 9;
    pub const RT_ABS: c_int = 10;
    pub const RT_CLIP: c_int = 11;
    pub const RT_MUL_SCALAR: c_int = 12;
    pub const RT_DIV_SCALAR: c_int = 13;
    pub const RT_COS: c_int = 14;
    pub const RT_TAN: c_int = 15;
    pub const RT_UNARY_COUNT: c_int = 16;
    pub const RT_ADD: c_int = 0;
    pub const RT_SUB: c_int = 1;
    pub const RT_MUL: c_int = 2;
    pub const RT_DIV: c_int = 3;
    pub const RT_POWF: c_int = 4;
    pub const RT_MAXIMUM: c_int = 5;
    pub const RT_MINIMUM: c_int = 6;
    pub const RT_EQUAL: c_int = 7;
    pub const RT_NOT_EQUAL: c_int = 8;
    pub const RT_GREATER: c_int = 9;
    pub const RT_GREATER_EQUAL: c_int = 10;
    pub const RT_LESS: c_int = 11;
    pub const RT_LESS_EQUAL: c_int = 12;
    pub const RT_BINARY_COUNT: c_int = 13;
    pub const RT_F_LOAD: c_int = 0;
    pub const RT_RED_SUM: c_int = 0;
    pub const RT_RED_MEAN: c_int = 1;
    pub const RT_RED_MAX: c_int = 2;
    pub const RT_RED_MIN: c_int = 3;
    pub const RT_RED_PROD: c_int = 4;
    pub const RT_RED_LOGSUMEXP: c_int = 5;
    pub const RT_RED_ARGMAX: c_int = 6;
    pub const RT_RED_ARGMIN: c_int = 7;
    pub const RT_RED_COUNT: c_int = 8;
    pub const RT_ACT_NONE: c_int = 0;
    pub const RT_ACT_RELU: c_int = 1;
    pub const RT_ACT_TANH: c_int = 2;
    pub const RT_ACT_SIGMOID: c_int = 3;
    #[link(name = "rt_b200")]
    extern "C" {
        pub fn rt_ctx_create(device: c_int, out: *mut *mut RtCtx) -> RtStatus;
        pub fn rt_ctx_destroy(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_last_error(ctx: *mut RtCtx) -> *const c_char;
        pub fn rt_device_count() -> c_int;
        pub fn rt_malloc(ctx: *mut RtCtx, bytes: usize, out: *mut *mut c_void) -> RtStatus;
        pub fn rt_free(ctx: *mut RtCtx, ptr: *mut c_void) -> RtStatus;
        pub fn rt_memcpy_h2d(ctx: *mut RtCtx, dst: *mut c_void, host_src: *const c_void, bytes: usize) -> RtStatus;
        pub fn rt_memcpy_d2h(ctx: *mut RtCtx, host_dst: *mut c_void, src: *const c_void, bytes: usize) -> RtStatus;
        pub fn rt_memcpy_h2d_async(ctx: *mut RtCtx, dst: *mut c_void, pinned_src: *const c_void, bytes: usize) -> RtStatus;
        pub fn rt_memcpy_d2h_async(ctx: *mut RtCtx, pinned_dst: *mut c_void, src: *const c_void, bytes: usize) -> RtStatus;
        pub fn rt_memcpy_d2d(ctx: *mut RtCtx, dst: *mut c_void, src: *const c_void, bytes: usize) -> RtStatus;
        pub fn rt_fill(ctx: *mut RtCtx, dst: *mut f32, value: f32, n: i64) -> RtStatus;
        pub fn rt_random_uniform(ctx: *mut RtCtx, out: *mut f32, n: i64, low: f32, high: f32, seed: u64, offset: u64) -> RtStatus;
        pub fn rt_random_normal(ctx: *mut RtCtx, out: *mut f32, n: i64, mean: f32, std_dev: f32, seed: u64, offset: u64) -> RtStatus;
        pub fn rt_bernoulli(ctx: *mut RtCtx, out: *mut f32, n: i64, p: f32, seed: u64, offset: u64) -> RtStatus;
        pub fn rt_host_alloc(ctx: *mut RtCtx, bytes: usize, out: *mut *mut c_void) -> RtStatus;
        pub fn rt_host_free(ctx: *mut RtCtx, ptr: *mut c_void) -> RtStatus;
        pub fn rt_sync(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_upload_create(ctx: *mut RtCtx, bytes: usize, out: *mut *mut RtUpload) -> RtStatus;
        pub fn rt_upload_destroy(ctx: *mut RtCtx, up: *mut RtUpload) -> RtStatus;
        pub fn rt_upload_host_buffer(ctx: *mut RtCtx, up: *mut RtUpload, pinned: *mut *mut c_void) -> RtStatus;
        pub fn rt_upload_submit(ctx: *mut RtCtx, up: *mut RtUpload, dst: *mut c_void) -> RtStatus;
        pub fn rt_upload_submit_all(ctx: *mut RtCtx, ups: *const *mut RtUpload, dsts: *const *mut c_void, n: c_int) -> RtStatus;
        pub fn rt_upload_submit_parts(ctx: *mut RtCtx, up: *mut RtUpload, n: c_int, offsets: *const i64, bytes: *const i64, dsts: *const *mut c_void) -> RtStatus;
        pub fn rt_publish_to_host(ctx: *mut RtCtx, pinned_dst: *mut f32, src: *const f32, n: i64) -> RtStatus;
        pub fn rt_side_stream_begin(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_side_stream_end(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_side_stream_join(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_event_create(ctx: *mut RtCtx, out: *mut *mut RtEvent) -> RtStatus;
        pub fn rt_event_destroy(ctx: *mut RtCtx, ev: *mut RtEvent) -> RtStatus;
        pub fn rt_event_record(ctx: *mut RtCtx, ev: *mut RtEvent) -> RtStatus;
        pub fn rt_event_synchronize(ctx: *mut RtCtx, ev: *mut RtEvent) -> RtStatus;
        pub fn rt_stream(ctx: *mut RtCtx) -> *mut c_void;
        pub fn rt_mem_stats(ctx: *mut RtCtx, bytes_reserved: *mut i64, bytes_in_use: *mut i64, n_device_allocs: *mut i64) -> RtStatus;
        pub fn rt_kernel_launch_count(ctx: *mut RtCtx, launches: *mut i64) -> RtStatus;
        pub fn rt_fused_launch_counts(ctx: *mut RtCtx, compiled: *mut i64, interpreted: *mut i64) -> RtStatus;
        pub fn rt_device_status(ctx: *mut RtCtx, code: *mut c_int) -> RtStatus;
        pub fn rt_set_tensor_cores(ctx: *mut RtCtx, enable: c_int) -> RtStatus;
        pub fn rt_set_concurrent_backward(ctx: *mut RtCtx, enable: c_int) -> RtStatus;
        pub fn rt_tc_issue_rate(ctx: *mut RtCtx, m: c_int, n: c_int, a_in_tmem: c_int, iters: c_int, issue_cycles: *mut f64, complete_cycles: *mut f64) -> RtStatus;
        pub fn rt_graph_begin(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_graph_end(ctx: *mut RtCtx, out: *mut *mut RtGraph) -> RtStatus;
        pub fn rt_graph_launch(ctx: *mut RtCtx, g: *mut RtGraph) -> RtStatus;
        pub fn rt_graph_destroy(ctx: *mut RtCtx, g: *mut RtGraph) -> RtStatus;
        pub fn rt_graph_num_nodes(ctx: *mut RtCtx, g: *mut RtGraph, n: *mut i64) -> RtStatus;
        pub fn rt_timer_start(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_timer_stop(ctx: *mut RtCtx, elapsed_ms: *mut f32) -> RtStatus;
        pub fn rt_stamp(ctx: *mut RtCtx, dst: *mut u64) -> RtStatus;
        pub fn rt_unary(ctx: *mut RtCtx, op: c_int, x: *const f32, y: *mut f32, n: i64, p0: f32, p1: f32) -> RtStatus;
        pub fn rt_unary_backward(ctx: *mut RtCtx, op: c_int, x: *const f32, g: *const f32, dx: *mut f32, n: i64, p0: f32, p1: f32) -> RtStatus;
        pub fn rt_binary(ctx: *mut RtCtx, op: c_int, a: *const f32, a_shape: *const i64, a_ndim: c_int, b: *const f32, b_shape: *const i64, b_ndim: c_int, out: *mut f32) -> RtStatus;
        pub fn rt_binary_backward(ctx: *mut RtCtx, op: c_int, a: *const f32, a_shape: *const i64, a_ndim: c_int, b: *const f32, b_shape: *const i64, b_ndim: c_int, g: *const f32, da: *mut f32, db: *mut f32) -> RtStatus;
        pub fn rt_unbroadcast(ctx: *mut RtCtx, g: *const f32, g_shape: *const i64, g_ndim: c_int, target_shape: *const i64, t_ndim: c_int, out: *mut f32) -> RtStatus;
        pub fn rt_broadcast_to(ctx: *mut RtCtx, x: *const f32, x_shape: *const i64, x_ndim: c_int, out_shape: *const i64, out_ndim: c_int, out: *mut f32) -> RtStatus;
        pub fn rt_transpose2d(ctx: *mut RtCtx, x: *const f32, rows: i64, cols: i64, out: *mut f32) -> RtStatus;
        pub fn rt_slice_assign(ctx: *mut RtCtx, dst: *mut f32, dst_shape: *const i64, ndim: c_int, starts: *const i64, src: *const f32, src_shape: *const i64) -> RtStatus;
        pub fn rt_slice(ctx: *mut RtCtx, x: *const f32, x_shape: *const i64, ndim: c_int, starts: *const i64, out_shape: *const i64, out: *mut f32) -> RtStatus;
        pub fn rt_concat_list(ctx: *mut RtCtx, count: c_int, srcs: *const *const f32, lens: *const i64, outer: i64, out: *mut f32) -> RtStatus;
        pub fn rt_fused_elementwise(ctx: *mut RtCtx, program: *const RtFusedProgram) -> RtStatus;
        pub fn rt_fused_reduction_possible(ctx: *mut RtCtx, which: c_int, ops: u64) -> RtStatus;
        pub fn rt_fused_reduction_known(ctx: *mut RtCtx, program: *const RtFusedProgram, which: c_int) -> RtStatus;
        pub fn rt_fused_column_sums(ctx: *mut RtCtx, program: *const RtFusedProgram, which: c_int, sums: *mut f32) -> RtStatus;
        pub fn rt_fused_logsumexp(ctx: *mut RtCtx, program: *const RtFusedProgram, out: *mut f32) -> RtStatus;
        pub fn rt_gather_rows(ctx: *mut RtCtx, src: *const f32, rows: i64, row_len: i64, idx: *const i32, n_idx: i64, out: *mut f32) -> RtStatus;
        pub fn rt_gather_rows_list(ctx: *mut RtCtx, n_src: c_int, srcs: *const *const f32, row_lens: *const i64, rows: i64, idx: *const i32, n_idx: i64, outs: *const *mut f32) -> RtStatus;
        pub fn rt_upload_gather_rows(ctx: *mut RtCtx, up: *mut RtUpload, n_src: c_int, srcs: *const *const f32, row_lens: *const i64, rows: i64, n_idx: i64, outs: *const *mut f32) -> RtStatus;
        pub fn rt_embedding(ctx: *mut RtCtx, table: *const f32, rows: i64, cols: i64, ids: *const i32, n: i64, scale: f32, out: *mut f32) -> RtStatus;
        pub fn rt_embedding_backward(ctx: *mut RtCtx, g: *const f32, ids: *const i32, n: i64, rows: i64, cols: i64, scale: f32, dtable: *mut f32, accumulate: c_int) -> RtStatus;
        pub fn rt_token_ids(ctx: *mut RtCtx, x: *const f32, n: i64, ids: *mut i32) -> RtStatus;
        pub fn rt_sum_rows_accumulate(ctx: *mut RtCtx, x: *const f32, rows: i64, cols: i64, out: *mut f32) -> RtStatus;
        pub fn rt_reduce(ctx: *mut RtCtx, kind: c_int, x: *const f32, outer: i64, len: i64, inner: i64, out: *mut f32) -> RtStatus;
        pub fn rt_reduce_backward(ctx: *mut RtCtx, kind: c_int, x: *const f32, g: *const f32, outer: i64, len: i64, inner: i64, dx: *mut f32) -> RtStatus;
        pub fn rt_sum_all_host(ctx: *mut RtCtx, x: *const f32, n: i64, host_out: *mut f32) -> RtStatus;
        pub fn rt_log_softmax(ctx: *mut RtCtx, x: *const f32, outer: i64, len: i64, inner: i64, y: *mut f32) -> RtStatus;
        pub fn rt_log_softmax_backward(ctx: *mut RtCtx, x: *const f32, g: *const f32, outer: i64, len: i64, inner: i64, dx: *mut f32) -> RtStatus;
        pub fn rt_lstm_cell_c(ctx: *mut RtCtx, gates: *const f32, c_prev: *const f32, batch: i64, hidden: i64, c: *mut f32) -> RtStatus;
        pub fn rt_lstm_cell_c_backward(ctx: *mut RtCtx, gates: *const f32, c_prev: *const f32, dc: *const f32, batch: i64, hidden: i64, dgates: *mut f32, dc_prev: *mut f32) -> RtStatus;
        pub fn rt_lstm_cell_h(ctx: *mut RtCtx, gates: *const f32, c: *const f32, batch: i64, hidden: i64, h: *mut f32) -> RtStatus;
        pub fn rt_lstm_cell_h_backward(ctx: *mut RtCtx, gates: *const f32, c: *const f32, dh: *const f32, batch: i64, hidden: i64, dgates: *mut f32, dc: *mut f32) -> RtStatus;
        pub fn rt_lstm_sequence_polls(ctx: *mut RtCtx, polls: i64) -> RtStatus;
        pub fn rt_lstm_sequence(ctx: *mut RtCtx, pre: *const f32, w: *const f32, ldw: i64, h0: *const f32, c0: *const f32, steps: i64, batch: i64, hidden: i64, saved: *mut f32, h: *mut f32) -> RtStatus;
        pub fn rt_lstm_sequence_backward(ctx: *mut RtCtx, saved: *const f32, w: *const f32, ldw: i64, c0: *const f32, dh: *const f32, steps: i64, batch: i64, hidden: i64, dgates: *mut f32, dh0: *mut f32, dc0: *mut f32) -> RtStatus;
        pub fn rt_gated_scan(ctx: *mut RtCtx, f: *const f32, v: *const f32, ld: i64, h0: *const f32, steps: i64, batch: i64, hidden: i64, h: *mut f32) -> RtStatus;
        pub fn rt_gated_scan_backward(ctx: *mut RtCtx, f: *const f32, v: *const f32, ld: i64, h0: *const f32, h: *const f32, dh: *const f32, steps: i64, batch: i64, hidden: i64, df: *mut f32, dv: *mut f32, ldd: i64, dh0: *mut f32) -> RtStatus;
        pub fn rt_softmax_cross_entropy(ctx: *mut RtCtx, logits: *const f32, targets: *const f32, rows: i64, classes: i64, loss: *mut f32) -> RtStatus;
        pub fn rt_softmax_cross_entropy_backward(ctx: *mut RtCtx, logits: *const f32, targets: *const f32, g: *const f32, rows: i64, classes: i64, dlogits: *mut f32, dtargets: *mut f32) -> RtStatus;
        pub fn rt_softmax_nll_scaled(ctx: *mut RtCtx, logits: *const f32, targets: *const f32, rows: i64, classes: i64, scale: f32, divisor: f32, loss: *mut f32) -> RtStatus;
        pub fn rt_softmax_nll_scaled_backward(ctx: *mut RtCtx, logits: *const f32, targets: *const f32, rows: i64, classes: i64, c: f32, dlogits: *mut f32) -> RtStatus;
        pub fn rt_softmax_nll_with_grad(ctx: *mut RtCtx, logits: *const f32, targets: *const f32, rows: i64, classes: i64, scale: f32, divisor: f32, g: *const f32, c: f32, loss: *mut f32, dlogits: *mut f32) -> RtStatus;
        pub fn rt_softmax_nll_list(ctx: *mut RtCtx, count: c_int, logits: *const *const f32, targets: *const *const f32, rows: i64, classes: i64, scale: f32, divisor: f32, n_more: c_int, more: *const *const f32, loss: *mut f32) -> RtStatus;
        pub fn rt_reduce_sum_static_scratch(ctx: *mut RtCtx, x: *const f32, outer: i64, len: i64, inner: i64, out: *mut f32) -> RtStatus;
        pub fn rt_max_pool2d(ctx: *mut RtCtx, x: *const f32, n: i64, c: i64, h: i64, w: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, y: *mut f32, idx: *mut f32) -> RtStatus;
        pub fn rt_max_pool2d_backward(ctx: *mut RtCtx, g: *const f32, idx: *const f32, n: i64, c: i64, h: i64, w: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, dx: *mut f32) -> RtStatus;
        pub fn rt_relu_max_pool2d(ctx: *mut RtCtx, x: *const f32, n: i64, c: i64, h: i64, w: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, y: *mut f32, idx: *mut f32) -> RtStatus;
        pub fn rt_relu_max_pool2d_backward(ctx: *mut RtCtx, x: *const f32, g: *const f32, idx: *const f32, n: i64, c: i64, h: i64, w: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, dx: *mut f32) -> RtStatus;
        pub fn rt_relu_max_pool2x2_backward_from_output(ctx: *mut RtCtx, y: *const f32, g: *const f32, idx: *const f32, n: i64, c: i64, h: i64, w: i64, dx: *mut f32) -> RtStatus;
        pub fn rt_gemm(ctx: *mut RtCtx, trans_a: c_int, trans_b: c_int, m: i64, n: i64, k: i64, a: *const f32, lda: i64, b: *const f32, ldb: i64, c: *mut f32, ldc: i64, accumulate: c_int) -> RtStatus;
        pub fn rt_gemm_bias_act(ctx: *mut RtCtx, m: i64, n: i64, k: i64, a: *const f32, lda: i64, b: *const f32, ldb: i64, bias: *const f32, act: c_int, c: *mut f32, ldc: i64) -> RtStatus;
        pub fn rt_gemm_bias_act_list(ctx: *mut RtCtx, count: c_int, a: *const *const f32, c: *const *mut f32, m: i64, n: i64, k: i64, b: *const f32, bias: *const f32, act: c_int) -> RtStatus;
        pub fn rt_gemm_sum_products(ctx: *mut RtCtx, count: c_int, a: *const *const f32, g: *const *const f32, m: i64, k: i64, n: i64, c: *mut f32) -> RtStatus;
        pub fn rt_sum_rows_accumulate_list(ctx: *mut RtCtx, count: c_int, x: *const *const f32, rows: i64, cols: i64, out: *mut f32) -> RtStatus;
        pub fn rt_column_sums_list(ctx: *mut RtCtx, count: c_int, xs: *const *const f32, rows: *const i64, cols: *const i64, outs: *const *mut f32) -> RtStatus;
        pub fn rt_matmul_backward(ctx: *mut RtCtx, a: *const f32, b: *const f32, g: *const f32, m: i64, k: i64, n: i64, da: *mut f32, db: *mut f32) -> RtStatus;
        pub fn rt_matmul_backward_accumulate(ctx: *mut RtCtx, a: *const f32, b: *const f32, g: *const f32, m: i64, k: i64, n: i64, da: *mut f32, db_sum: *mut f32) -> RtStatus;
        pub fn rt_conv2d(ctx: *mut RtCtx, x: *const f32, w: *const f32, bias: *const f32, n: i64, cin: i64, h: i64, wd: i64, cout: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, y: *mut f32) -> RtStatus;
        pub fn rt_conv2d_relu_max_pool2x2(ctx: *mut RtCtx, x: *const f32, w: *const f32, bias: *const f32, n: i64, cin: i64, h: i64, wd: i64, cout: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, y: *mut f32, idx: *mut f32) -> RtStatus;
        pub fn rt_conv2d_backward(ctx: *mut RtCtx, x: *const f32, w: *const f32, g: *const f32, n: i64, cin: i64, h: i64, wd: i64, cout: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, dx: *mut f32, dw: *mut f32, db: *mut f32) -> RtStatus;
        pub fn rt_conv2d_transpose(ctx: *mut RtCtx, x: *const f32, w: *const f32, bias: *const f32, n: i64, cin: i64, h: i64, wd: i64, cout: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, y: *mut f32) -> RtStatus;
        pub fn rt_conv2d_transpose_backward(ctx: *mut RtCtx, x: *const f32, w: *const f32, g: *const f32, n: i64, cin: i64, h: i64, wd: i64, cout: i64, kh: c_int, kw: c_int, sh: c_int, sw: c_int, ph: c_int, pw: c_int, dx: *mut f32, dw: *mut f32, db: *mut f32) -> RtStatus;
        pub fn rt_sgd_step(ctx: *mut RtCtx, param: *mut f32, grad: *const f32, n: i64, lr: f32) -> RtStatus;
        pub fn rt_momentum_sgd_step(ctx: *mut RtCtx, param: *mut f32, grad: *const f32, velocity: *mut f32, n: i64, lr: f32, momentum: f32) -> RtStatus;
        pub fn rt_adagrad_step(ctx: *mut RtCtx, param: *mut f32, grad: *const f32, accum: *mut f32, n: i64, lr: f32, epsilon: f32) -> RtStatus;
        pub fn rt_adam_step(ctx: *mut RtCtx, param: *mut f32, grad: *const f32, m: *mut f32, v: *mut f32, n: i64, lr: f32, beta1: f32, beta2: f32, epsilon: f32, t: i64) -> RtStatus;
        pub fn rt_optimizer_step_multi(ctx: *mut RtCtx, kind: c_int, n_tensors: c_int, params: *const *mut f32, grads: *const *const f32, state1: *const *mut f32, state2: *const *mut f32, sizes: *const i64, lr: f32, beta1: f32, beta2: f32, epsilon: f32, momentum: f32, t: i64, grad_scale: f32, clip: c_int, clip_lo: f32, clip_hi: f32) -> RtStatus;
        pub fn rt_muon_step_multi(ctx: *mut RtCtx, n_tensors: c_int, params: *const *mut f32, grads: *const *const f32, momenta: *const *mut f32, rows: *const i64, cols: *const i64, lr: f32, momentum: f32, nesterov: c_int, weight_decay: f32, steps: c_int, grad_scale: f32) -> RtStatus;
        pub fn rt_orthogonalize_list(ctx: *mut RtCtx, count: c_int, xs: *const *const f32, rows: *const i64, cols: *const i64, steps: c_int, outs: *const *mut f32) -> RtStatus;
        pub fn rt_pack_flat(ctx: *mut RtCtx, n_tensors: c_int, srcs: *const *const f32, sizes: *const i64, flat: *mut f32, clip: c_int, clip_lo: f32, clip_hi: f32) -> RtStatus;
        pub fn rt_dp_unique_id(id: *mut u8) -> RtStatus;
        pub fn rt_dp_init(ctx: *mut RtCtx, rank: c_int, world: c_int, id: *const u8) -> RtStatus;
        pub fn rt_dp_init_deadline(ctx: *mut RtCtx, rank: c_int, world: c_int, id: *const u8, timeout_ms: i64) -> RtStatus;
        pub fn rt_dp_allreduce_sum(ctx: *mut RtCtx, buf: *mut f32, n: i64) -> RtStatus;
        pub fn rt_dp_async_error(ctx: *mut RtCtx, nccl_code: *mut c_int) -> RtStatus;
        pub fn rt_dp_wait_event(ctx: *mut RtCtx, ev: *mut RtEvent) -> RtStatus;
        pub fn rt_dp_finalize(ctx: *mut RtCtx) -> RtStatus;
        pub fn rt_ipc_export(ctx: *mut RtCtx, device_ptr: *mut c_void, handle: *mut u8) -> RtStatus;
        pub fn rt_ipc_open(ctx: *mut RtCtx, handle: *const u8, peer_ptr: *mut *mut c_void) -> RtStatus;
        pub fn rt_ipc_close(ctx: *mut RtCtx, peer_ptr: *mut c_void) -> RtStatus;
        pub fn rt_dp_step_begin(ctx: *mut RtCtx, step_state: *mut c_int) -> RtStatus;
        pub fn rt_optimizer_step_multi_device_t(ctx: *mut RtCtx, kind: c_int, n_tensors: c_int, params: *const *mut f32, grads: *const *const f32, state1: *const *mut f32, state2: *const *mut f32, sizes: *const i64, lr: f32, beta1: f32, beta2: f32, epsilon: f32, momentum: f32, step_state: *const c_int, grad_scale: f32, clip: c_int, clip_lo: f32, clip_hi: f32) -> RtStatus;
        pub fn rt_optimizer_step_multi_next(ctx: *mut RtCtx, kind: c_int, n_tensors: c_int, params: *const *mut f32, grads: *const *const f32, state1: *const *mut f32, state2: *const *mut f32, sizes: *const i64, lr: f32, beta1: f32, beta2: f32, epsilon: f32, momentum: f32, step_state: *mut c_int, grad_scale: f32, clip: c_int, clip_lo: f32, clip_hi: f32) -> RtStatus;
        pub fn rt_pack_flat_alternating(ctx: *mut RtCtx, n_tensors: c_int, srcs: *const *const f32, sizes: *const i64, flat0: *mut f32, flat1: *mut f32, step_state: *const c_int, clip: c_int, clip_lo: f32, clip_hi: f32) -> RtStatus;
        pub fn rt_pack_flat_signal(ctx: *mut RtCtx, n_tensors: c_int, srcs: *const *const f32, sizes: *const i64, flat0: *mut f32, flat1: *mut f32, step_state: *const c_int, clip: c_int, clip_lo: f32, clip_hi: f32, peer_flags: *const *mut c_int, rank: c_int, world: c_int) -> RtStatus;
        pub fn rt_dp_signal_peers(ctx: *mut RtCtx, peer_flags: *const *mut c_int, rank: c_int, world: c_int, step_state: *const c_int) -> RtStatus;
        pub fn rt_dp_wait_peers(ctx: *mut RtCtx, local_flags: *const c_int, rank: c_int, world: c_int, step_state: *mut c_int, spin_limit: u32) -> RtStatus;
        pub fn rt_optimizer_step_multi_peers(ctx: *mut RtCtx, kind: c_int, n_tensors: c_int, params: *const *mut f32, grads: *const *const f32, state1: *const *mut f32, state2: *const *mut f32, sizes: *const i64, lr: f32, beta1: f32, beta2: f32, epsilon: f32, momentum: f32, grad_scale: f32, flats0: *const *const f32, flats1: *const *const f32, rank: c_int, world: c_int, step_state: *const c_int) -> RtStatus;
    }
}
use ffi::*;

// ---- context: one per process and device, like the reference's global CUDA context (src/backend/cuda/context.rs) ----
struct CtxPtr(*mut RtCtx);
unsafe impl Send for CtxPtr {}
unsafe impl Sync for CtxPtr {}
static CTX: OnceLock<CtxPtr> = OnceLock::new();
static RNG: Mutex<(u64, u64)> = Mutex::new((0x5eed, 0)); // (seed, counter offset) of the random factories
fn ctx() -> *mut RtCtx {
    CTX.get_or_init(|| {
        let mut c: *mut RtCtx = std::ptr::null_mut();
        let dev = std::env::var("LOCAL_RANK").ok().and_then(|s| s.parse().ok()).unwrap_or(0);
        let st = unsafe { rt_ctx_create(dev, &mut c) };
        assert_eq!(st, RT_OK, "rt_ctx_create failed: this backend needs a CUDA device (sm_100a)");
        CtxPtr(c)
    }).0
}

fn check(st: RtStatus) -> Result<(), Error> {
    if st == RT_OK { return Ok(()); }
    let msg = unsafe { CStr::from_ptr(rt_last_error(ctx())) }.to_string_lossy().into_owned();
    Err(match st {
        RT_ERR_SHAPE_MISMATCH => Error::ShapeMismatch { expected: vec![], actual: vec![] }, // shapes are checked host side first, with details
        RT_ERR_INCOMPATIBLE_SHAPES => Error::IncompatibleShapes { op: msg, shape_a: vec![], shape_b: vec![] },
        RT_ERR_INVALID_INDEX => Error::InvalidIndex(vec![]),
        RT_ERR_INVALID_OPERATION => Error::InvalidOperation(msg),
        RT_ERR_INTERNAL => Error::InternalLogicError(msg),
        RT_ERR_DIMENSION_MISMATCH => Error::DimensionMismatch(0, 0),
        RT_ERR_OOM => Error::OutOfMemory,
        RT_ERR_UNIMPLEMENTED => Error::Unimplemented(msg),
        RT_ERR_EMPTY_TENSOR => Error::EmptyTensor,
        RT_ERR_INITIALIZATION => Error::InitializationError,
        _ => Error::CudaError(msg), // RT_ERR_CUDA, RT_ERR_TIMEOUT, RT_ERR_NCCL
    })
}

// ---- storage: a reference-counted device buffer + shape.  Buffers are immutable once produced, so `Clone` (an Arc
// clone) is observably the deep copy the trait asks for (mod.rs:39); the in-place methods copy on write. ----
#[derive(Debug)]
struct DeviceBuf { ptr: *mut f32, bytes: usize }
unsafe impl Send for DeviceBuf {}
unsafe impl Sync for DeviceBuf {}
impl Drop for DeviceBuf { fn drop(&mut self) { if !self.ptr.is_null() { unsafe { rt_free(ctx(), self.ptr as *mut c_void) }; } } }

#[derive(Debug, Clone)]
pub struct B200Storage { buf: Arc<DeviceBuf>, shape: Vec<usize> }
impl std::fmt::Display for B200Storage {
    fn fmt(&self, f: &mut std::fmt::Formatter) -> std::fmt::Result { write!(f, "B200Storage{:?}", self.shape) }
}
impl B200Storage {
    fn alloc(shape: &[usize]) -> Result<Self, Error> {
        let n: usize = shape.iter().product();
        let mut p: *mut c_void = std::ptr::null_mut();
        check(unsafe { rt_malloc(ctx(), 4 * n.max(1), &mut p) })?;
        Ok(Self { buf: Arc::new(DeviceBuf { ptr: p as *mut f32, bytes: 4 * n.max(1) }), shape: shape.to_vec() })
    }
    fn ptr(&self) -> *const f32 { self.buf.ptr }
    fn ptr_mut(&self) -> *mut f32 { self.buf.ptr } // fresh outputs only
    fn numel(&self) -> usize { self.shape.iter().product() }
    fn dims(&self) -> Vec<i64> { self.shape.iter().map(|&d| d as i64).collect() }
    fn unique_ptr_mut(&mut self) -> Result<*mut f32, Error> { // copy on write before an in-place update
        if Arc::strong_count(&self.buf) > 1 {
            let c = Self::alloc(&self.shape)?;
            check(unsafe { rt_memcpy_d2d(ctx(), c.buf.ptr as *mut c_void, self.buf.ptr as *const c_void, 4 * self.numel()) })?;
            self.buf = c.buf;
        }
        Ok(self.buf.ptr)
    }
}

// [outer, len, inner] view of `shape` around `axis`
fn split(shape: &[usize], axis: usize) -> (i64, i64, i64) {
    (shape[..axis].iter().product::<usize>() as i64, shape[axis] as i64, shape[axis + 1..].iter().product::<usize>() as i64)
}
fn broadcast_shape(op: &str, a: &[usize], b: &[usize]) -> Result<Vec<usize>, Error> {
    crate::util::broadcast_shapes(a, b).map_err(|_| Error::IncompatibleShapes { op: op.into(), shape_a: a.to_vec(), shape_b: b.to_vec() })
}
fn unary(code: c_int, x: &B200Storage, p0: f32, p1: f32) -> Result<B200Storage, Error> {
    let out = B200Storage::alloc(&x.shape)?;
    check(unsafe { rt_unary(ctx(), code, x.ptr(), out.ptr_mut(), x.numel() as i64, p0, p1) })?;
    Ok(out)
}
fn unary_bwd(code: c_int, op: &Op<B200Backend>, g: &B200Storage, p0: f32, p1: f32) -> Result<B200Storage, Error> {
    let x = &*op.inputs[0].data(); // f' is recomputed from the INPUT, as in the reference's CPU backend
    if x.shape != g.shape { return Err(Error::ShapeMismatch { expected: x.shape.clone(), actual: g.shape.clone() }); }
    let out = B200Storage::alloc(&x.shape)?;
    check(unsafe { rt_unary_backward(ctx(), code, x.ptr(), g.ptr(), out.ptr_mut(), x.numel() as i64, p0, p1) })?;
    Ok(out)
}
fn binary(code: c_int, name: &str, a: &B200Storage, b: &B200Storage) -> Result<B200Storage, Error> {
    let out = B200Storage::alloc(&broadcast_shape(name, &a.shape, &b.shape)?)?;
    let (da, db) = (a.dims(), b.dims());
    check(unsafe { rt_binary(ctx(), code, a.ptr(), da.as_ptr(), da.len() as c_int, b.ptr(), db.as_ptr(), db.len() as c_int, out.ptr_mut()) })?;
    Ok(out)
}
fn binary_bwd(code: c_int, op: &Op<B200Backend>, g: &B200Storage) -> Result<(B200Storage, B200Storage), Error> {
    let (a, b) = (&*op.inputs[0].data(), &*op.inputs[1].data());
    let (ga, gb) = (B200Storage::alloc(&a.shape)?, B200Storage::alloc(&b.shape)?); // un-broadcast inside the kernels
    let (da, db) = (a.dims(), b.dims());
    check(unsafe { rt_binary_backward(ctx(), code, a.ptr(), da.as_ptr(), da.len() as c_int, b.ptr(), db.as_ptr(), db.len() as c_int,
                                      g.ptr(), ga.ptr_mut(), gb.ptr_mut()) })?;
    Ok((ga, gb))
}
fn reduce(kind: c_int, x: &B200Storage, axis: Option<usize>) -> Result<B200Storage, Error> {
    let (shape, (o, l, i)) = match axis {
        None => (vec![], (1, x.numel() as i64, 1)),           // global reductions have shape [] (mod.rs:293)
        Some(a) if a < x.shape.len() => { let mut s = x.shape.clone(); s.remove(a); (s, split(&x.shape, a)) }
        Some(a) => return Err(Error::InvalidIndex(vec![a])),
    };
    let out = B200Storage::alloc(&shape)?;
    check(unsafe { rt_reduce(ctx(), kind, x.ptr(), o, l, i, out.ptr_mut()) })?;
    Ok(out)
}
fn reduce_bwd(kind: c_int, x: &B200Storage, g: &B200Storage, axis: Option<usize>) -> Result<B200Storage, Error> {
    let (o, l, i) = match axis { None => (1, x.numel() as i64, 1), Some(a) => split(&x.shape, a) };
    let out = B200Storage::alloc(&x.shape)?;
    check(unsafe { rt_reduce_backward(ctx(), kind, x.ptr(), g.ptr(), o, l, i, out.ptr_mut()) })?;
    Ok(out)
}
fn random(shape: &[usize], f: impl Fn(*mut f32, i64, u64, u64) -> RtStatus) -> Result<B200Storage, Error> {
    let out = B200Storage::alloc(shape)?;
    let n = out.numel();
    if n == 0 { return B200Backend::zeros(shape); }
    let mut st = RNG.lock().unwrap();
    check(f(out.ptr_mut(), n as i64, st.0, st.1))?;
    st.1 += ((n + 3) / 4) as u64; // a call consumes (n + 3) / 4 counter values
    Ok(out)
}

#[derive(Debug, Clone, Copy)]
pub struct B200Backend;

impl Backend for B200Backend {
    type Storage = B200Storage;

    // ---- factories and access (mod.rs:44-88, 248-252) ----
    fn zeros(shape: &[usize]) -> Result<Self::Storage, Error> {
        let s = B200Storage::alloc(shape)?;
        check(unsafe { rt_fill(ctx(), s.ptr_mut(), 0.0, s.numel() as i64) })?;
        Ok(s)
    }
    fn ones(shape: &[usize]) -> Result<Self::Storage, Error> {
        let s = B200Storage::alloc(shape)?;
        check(unsafe { rt_fill(ctx(), s.ptr_mut(), 1.0, s.numel() as i64) })?;
        Ok(s)
    }
    fn from_vec(data: Vec<f32>, shape: &[usize]) -> Result<Self::Storage, Error> {
        let n: usize = shape.iter().product();
        if data.len() != n { return Err(Error::ShapeMismatch { expected: shape.to_vec(), actual: vec![data.len()] }); }
        let s = B200Storage::alloc(shape)?;
        check(unsafe { rt_memcpy_h2d(ctx(), s.ptr_mut() as *mut c_void, data.as_ptr() as *const c_void, 4 * n) })?;
        Ok(s)
    }
    fn kaiming_uniform(fan_in: usize, shape: &[usize]) -> Result<Self::Storage, Error> {            // mod.rs:57, src/init.rs:7-52
        if shape.is_empty() { return Err(Error::InvalidOperation("Cannot initialize tensor with empty shape".into())); }
        if shape.iter().any(|&d| d == 0) { return Self::zeros(shape); }
        if fan_in == 0 { return Err(Error::InvalidOperation("Fan-in cannot be zero for Kaiming initialization".into())); }
        let bound = (6.0 / fan_in as f32).sqrt();
        Self::random_uniform(shape, -bound, bound)
    }
    fn random_uniform(shape: &[usize], low: f32, high: f32) -> Result<Self::Storage, Error> {        // mod.rs:63
        random(shape, |p, n, seed, off| unsafe { rt_random_uniform(ctx(), p, n, low, high, seed, off) })
    }
    fn random_normal(shape: &[usize], mean: f32, std_dev: f32) -> Result<Self::Storage, Error> {     // mod.rs:66
        random(shape, |p, n, seed, off| unsafe { rt_random_normal(ctx(), p, n, mean, std_dev, seed, off) })
    }
    fn bernoulli(shape: &[usize], p: f32) -> Result<Self::Storage, Error> {                          // mod.rs:69
        random(shape, |q, n, seed, off| unsafe { rt_bernoulli(ctx(), q, n, p, seed, off) })
    }
    fn device(_s: &Self::Storage) -> crate::Device { crate::Device::Cuda(0) }
    fn shape(s: &Self::Storage) -> &[usize] { &s.shape }
    fn size(s: &Self::Storage) -> usize { s.numel() }
    fn into_raw_vec(s: Self::Storage) -> Result<Vec<f32>, Error> { Self::copy_to_host(&s) }
    fn set_data(s: &mut Self::Storage, data: Self::Storage) -> Result<(), Error> { *s = data; Ok(()) }
    fn set_shape(s: &mut Self::Storage, shape: &[usize]) -> Result<(), Error> {
        if shape.iter().product::<usize>() != s.numel() { return Err(Error::ShapeMismatch { expected: shape.to_vec(), actual: s.shape.clone() }); }
        s.shape = shape.to_vec();
        Ok(())
    }
    fn copy_to_host(s: &Self::Storage) -> Result<Vec<f32>, Error> {                                  // mod.rs:248 (synchronises)
        let mut v = vec![0f32; s.numel()];
        check(unsafe { rt_memcpy_d2h(ctx(), v.as_mut_ptr() as *mut c_void, s.ptr() as *const c_void, 4 * v.len()) })?;
        Ok(v)
    }
    fn update_from_host(s: &mut Self::Storage, data: &[f32]) -> Result<(), Error> {                  // mod.rs:252
        if data.len() != s.numel() { return Err(Error::ShapeMismatch { expected: s.shape.clone(), actual: vec![data.len()] }); }
        let p = s.unique_ptr_mut()?;
        check(unsafe { rt_memcpy_h2d(ctx(), p as *mut c_void, data.as_ptr() as *const c_void, 4 * data.len()) })
    }
    fn map<F>(x: &Self::Storage, f: F) -> Result<Self::Storage, Error> where F: Fn(f32) -> f32 + Send + Sync + 'static {
        let v: Vec<f32> = Self::copy_to_host(x)?.into_iter().map(f).collect(); // an arbitrary host closure: host round trip, as in the reference's CUDA backend
        Self::from_vec(v, &x.shape)
    }

    // ---- element-wise, comparisons, reductions and their gradients (one forwarding call each) ----
    fn exp(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_EXP, x, 0.0, 0.0) }
    fn exp_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_EXP, op, g, 0.0, 0.0) }
    fn ln(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_LN, x, 0.0, 0.0) }
    fn ln_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_LN, op, g, 0.0, 0.0) }
    fn relu(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_RELU, x, 0.0, 0.0) }
    fn relu_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_RELU, op, g, 0.0, 0.0) }
    fn sigmoid(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_SIGMOID, x, 0.0, 0.0) }
    fn sigmoid_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_SIGMOID, op, g, 0.0, 0.0) }
    fn abs(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_ABS, x, 0.0, 0.0) }
    fn abs_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_ABS, op, g, 0.0, 0.0) }
    fn sqrt(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_SQRT, x, 0.0, 0.0) }
    fn sqrt_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_SQRT, op, g, 0.0, 0.0) }
    fn tanh(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_TANH, x, 0.0, 0.0) }
    fn tanh_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_TANH, op, g, 0.0, 0.0) }
    fn softplus(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_SOFTPLUS, x, 0.0, 0.0) }
    fn softplus_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_SOFTPLUS, op, g, 0.0, 0.0) }
    fn square(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_SQUARE, x, 0.0, 0.0) }
    fn square_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_SQUARE, op, g, 0.0, 0.0) }
    fn sin(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_SIN, x, 0.0, 0.0) }
    fn sin_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_SIN, op, g, 0.0, 0.0) }
    fn cos(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_COS, x, 0.0, 0.0) }
    fn cos_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_COS, op, g, 0.0, 0.0) }
    fn tan(x: &Self::Storage) -> Result<Self::Storage, Error> { unary(RT_TAN, x, 0.0, 0.0) }
    fn tan_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> { unary_bwd(RT_TAN, op, g, 0.0, 0.0) }
    fn mul(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_MUL, "mul", a, b) }
    fn add(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_ADD, "add", a, b) }
    fn sub(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_SUB, "sub", a, b) }
    fn div(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_DIV, "div", a, b) }
    fn powf(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_POWF, "powf", a, b) }
    fn maximum(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_MAXIMUM, "maximum", a, b) }
    fn minimum(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_MINIMUM, "minimum", a, b) }
    fn equal(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_EQUAL, "equal", a, b) }
    fn not_equal(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_NOT_EQUAL, "not_equal", a, b) }
    fn greater(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_GREATER, "greater", a, b) }
    fn greater_equal(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_GREATER_EQUAL, "greater_equal", a, b) }
    fn less(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_LESS, "less", a, b) }
    fn less_equal(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> { binary(RT_LESS_EQUAL, "less_equal", a, b) }
    fn mul_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_MUL, op, g) }
    fn add_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_ADD, op, g) }
    fn sub_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_SUB, op, g) }
    fn div_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_DIV, op, g) }
    fn powf_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_POWF, op, g) }
    fn maximum_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_MAXIMUM, op, g) }
    fn minimum_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { binary_bwd(RT_MINIMUM, op, g) }
    fn max(x: &Self::Storage, axis: Option<usize>) -> Result<Self::Storage, Error> { reduce(RT_RED_MAX, x, axis) }
    fn min(x: &Self::Storage, axis: Option<usize>) -> Result<Self::Storage, Error> { reduce(RT_RED_MIN, x, axis) }
    fn prod(x: &Self::Storage, axis: Option<usize>) -> Result<Self::Storage, Error> { reduce(RT_RED_PROD, x, axis) }
    fn logsumexp(x: &Self::Storage, axis: Option<usize>) -> Result<Self::Storage, Error> { reduce(RT_RED_LOGSUMEXP, x, axis) }
    fn mean(x: &Self::Storage, axis: Option<usize>) -> Result<Self::Storage, Error> { reduce(RT_RED_MEAN, x, axis) }
    fn max_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let axis = match op.op_type { OpType::Max(a) => a, _ => return Err(Error::InternalLogicError("max_backward: wrong op type".into())) };
        reduce_bwd(RT_RED_MAX, &*op.inputs[0].data(), g, axis)
    }
    fn min_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let axis = match op.op_type { OpType::Min(a) => a, _ => return Err(Error::InternalLogicError("min_backward: wrong op type".into())) };
        reduce_bwd(RT_RED_MIN, &*op.inputs[0].data(), g, axis)
    }
    fn prod_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let axis = match op.op_type { OpType::Prod(a) => a, _ => return Err(Error::InternalLogicError("prod_backward: wrong op type".into())) };
        reduce_bwd(RT_RED_PROD, &*op.inputs[0].data(), g, axis)
    }
    fn logsumexp_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let axis = match op.op_type { OpType::LogSumExp(a) => a, _ => return Err(Error::InternalLogicError("logsumexp_backward: wrong op type".into())) };
        reduce_bwd(RT_RED_LOGSUMEXP, &*op.inputs[0].data(), g, axis)
    }
    fn mean_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let axis = match op.op_type { OpType::Mean(a) => a, _ => return Err(Error::InternalLogicError("mean_backward: wrong op type".into())) };
        reduce_bwd(RT_RED_MEAN, &*op.inputs[0].data(), g, axis)
    }
    fn sum_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let axis = match op.op_type { OpType::Sum(a) => a, _ => return Err(Error::InternalLogicError("sum_backward: wrong op type".into())) };
        reduce_bwd(RT_RED_SUM, &*op.inputs[0].data(), g, axis)
    }
    fn elu(x: &Self::Storage, alpha: f32) -> Result<Self::Storage, Error> { unary(RT_ELU, x, alpha, 0.0) }
    fn elu_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let alpha = match op.op_type { OpType::Elu(a) => a, _ => return Err(Error::InternalLogicError("elu_backward: wrong op type".into())) };
        unary_bwd(RT_ELU, op, g, alpha, 0.0)
    }
    fn clip(x: &Self::Storage, min_val: f32, max_val: f32) -> Result<Self::Storage, Error> { unary(RT_CLIP, x, min_val, max_val) }
    fn clip_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let (lo, hi) = match op.op_type { OpType::Clip { min_val, max_val } => (min_val, max_val), _ => return Err(Error::InternalLogicError("clip_backward: wrong op type".into())) };
        unary_bwd(RT_CLIP, op, g, lo, hi)
    }
    fn mul_scalar(x: &Self::Storage, scalar: f32) -> Result<Self::Storage, Error> { unary(RT_MUL_SCALAR, x, scalar, 0.0) }
    fn div_scalar(x: &Self::Storage, scalar: f32) -> Result<Self::Storage, Error> {
        if scalar == 0.0 { return Err(Error::InvalidOperation("Division by zero scalar".into())); }
        unary(RT_DIV_SCALAR, x, scalar, 0.0)
    }
    fn sum_along_axis(x: &Self::Storage, axis: usize) -> Result<Self::Storage, Error> { reduce(RT_RED_SUM, x, Some(axis)) }
    fn max_along_axis(x: &Self::Storage, axis: usize) -> Result<Self::Storage, Error> { reduce(RT_RED_MAX, x, Some(axis)) }
    fn argmax(x: &Self::Storage, axis: usize) -> Result<Self::Storage, Error> { reduce(RT_RED_ARGMAX, x, Some(axis)) }
    fn argmin(x: &Self::Storage, axis: usize) -> Result<Self::Storage, Error> { reduce(RT_RED_ARGMIN, x, Some(axis)) }
    fn sum_all(x: &Self::Storage) -> Result<f32, Error> {                                            // mod.rs:293 (synchronises)
        let mut v = 0f32;
        check(unsafe { rt_sum_all_host(ctx(), x.ptr(), x.numel() as i64, &mut v) })?;
        Ok(v)
    }
    fn log_softmax(x: &Self::Storage, axis: usize) -> Result<Self::Storage, Error> {                 // mod.rs:307
        let (o, l, i) = split(&x.shape, axis);
        let out = B200Storage::alloc(&x.shape)?;
        check(unsafe { rt_log_softmax(ctx(), x.ptr(), o, l, i, out.ptr_mut()) })?;
        Ok(out)
    }
    fn log_softmax_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {      // mod.rs:349
        let axis = match op.op_type { OpType::LogSoftmax(a) => a, _ => return Err(Error::InternalLogicError("log_softmax_backward: wrong op type".into())) };
        let x = &*op.inputs[0].data();
        let (o, l, i) = split(&x.shape, axis);
        let out = B200Storage::alloc(&x.shape)?;
        check(unsafe { rt_log_softmax_backward(ctx(), x.ptr(), g.ptr(), o, l, i, out.ptr_mut()) })?;
        Ok(out)
    }

    // ---- layout ----
    fn transpose(x: &Self::Storage) -> Result<Self::Storage, Error> {                                // mod.rs:275 (matrices)
        if x.shape.len() != 2 { return Err(Error::Unimplemented("transpose of tensors with more than two axes".into())); }
        let out = B200Storage::alloc(&[x.shape[1], x.shape[0]])?;
        check(unsafe { rt_transpose2d(ctx(), x.ptr(), x.shape[0] as i64, x.shape[1] as i64, out.ptr_mut()) })?;
        Ok(out)
    }
    fn broadcast_to(x: &Self::Storage, shape: &[usize]) -> Result<Self::Storage, Error> {            // mod.rs:277
        let out = B200Storage::alloc(shape)?;
        let (dx, ds): (Vec<i64>, Vec<i64>) = (x.dims(), shape.iter().map(|&d| d as i64).collect());
        check(unsafe { rt_broadcast_to(ctx(), x.ptr(), dx.as_ptr(), dx.len() as c_int, ds.as_ptr(), ds.len() as c_int, out.ptr_mut()) })?;
        Ok(out)
    }
    fn slice(x: &Self::Storage, ranges: &[std::ops::Range<usize>]) -> Result<Self::Storage, Error> { // mod.rs:522
        let shape: Vec<usize> = ranges.iter().map(|r| r.end - r.start).collect();
        let out = B200Storage::alloc(&shape)?;
        let (dx, st, os): (Vec<i64>, Vec<i64>, Vec<i64>) = (x.dims(), ranges.iter().map(|r| r.start as i64).collect(), shape.iter().map(|&d| d as i64).collect());
        check(unsafe { rt_slice(ctx(), x.ptr(), dx.as_ptr(), dx.len() as c_int, st.as_ptr(), os.as_ptr(), out.ptr_mut()) })?;
        Ok(out)
    }
    fn slice_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {            // mod.rs:535: zero fill + write the block
        let (input_shape, ranges) = match &op.op_type { OpType::Slice { input_shape, ranges } => (input_shape, ranges), _ => return Err(Error::InternalLogicError("slice_backward: wrong op type".into())) };
        let out = Self::zeros(input_shape)?;
        let (ds, st, gs): (Vec<i64>, Vec<i64>, Vec<i64>) = (out.dims(), ranges.iter().map(|r| r.start as i64).collect(), g.dims());
        check(unsafe { rt_slice_assign(ctx(), out.ptr_mut(), ds.as_ptr(), ds.len() as c_int, st.as_ptr(), g.ptr(), gs.as_ptr()) })?;
        Ok(out)
    }
    fn concat(tensors: &[&Self::Storage], axis: usize) -> Result<Self::Storage, Error> {            // mod.rs:550: one block write per input
        let mut shape = tensors[0].shape.clone();
        shape[axis] = tensors.iter().map(|t| t.shape[axis]).sum();
        let out = B200Storage::alloc(&shape)?;
        let ds = out.dims();
        let mut start = vec![0i64; shape.len()];
        for t in tensors {
            let ts = t.dims();
            check(unsafe { rt_slice_assign(ctx(), out.ptr_mut(), ds.as_ptr(), ds.len() as c_int, start.as_ptr(), t.ptr(), ts.as_ptr()) })?;
            start[axis] += t.shape[axis] as i64;
        }
        Ok(out)
    }
    fn concat_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Vec<Self::Storage>, Error> {      // mod.rs:563: one slice per input
        let (axis, shapes) = match &op.op_type { OpType::Concat { axis, input_shapes } => (*axis, input_shapes), _ => return Err(Error::InternalLogicError("concat_backward: wrong op type".into())) };
        let mut start = 0usize;
        let mut outs = Vec::with_capacity(shapes.len());
        for s in shapes {
            let ranges: Vec<std::ops::Range<usize>> = s.iter().enumerate().map(|(d, &n)| if d == axis { start..start + n } else { 0..n }).collect();
            outs.push(Self::slice(g, &ranges)?);
            start += s[axis];
        }
        Ok(outs)
    }
    fn expand_dims(x: &Self::Storage, axis: usize) -> Result<Self::Storage, Error> {                 // metadata only: the buffer is shared
        let mut s = x.clone();
        s.shape.insert(axis, 1);
        Ok(s)
    }
    fn expand_dims_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let mut s = g.clone();
        s.shape = op.inputs[0].data().shape.clone();
        Ok(s)
    }
    fn squeeze(x: &Self::Storage, axis: Option<usize>) -> Result<Self::Storage, Error> {
        let mut s = x.clone();
        match axis {
            Some(a) => { if s.shape.get(a) != Some(&1) { return Err(Error::InvalidOperation("squeeze: axis extent is not 1".into())); } s.shape.remove(a); }
            None => s.shape.retain(|&d| d != 1),
        }
        Ok(s)
    }
    fn squeeze_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {
        let shape = match &op.op_type { OpType::Squeeze { original_input_shape, .. } => original_input_shape.clone(), _ => return Err(Error::InternalLogicError("squeeze_backward: wrong op type".into())) };
        let mut s = g.clone();
        s.shape = shape;
        Ok(s)
    }

    // ---- contractions ----
    fn matmul(a: &Self::Storage, b: &Self::Storage) -> Result<Self::Storage, Error> {                // mod.rs:93
        if a.shape.len() != 2 || b.shape.len() != 2 || a.shape[1] != b.shape[0] {
            return Err(Error::IncompatibleShapes { op: "matmul".into(), shape_a: a.shape.clone(), shape_b: b.shape.clone() });
        }
        let (m, k, n) = (a.shape[0] as i64, a.shape[1] as i64, b.shape[1] as i64);
        let out = B200Storage::alloc(&[m as usize, n as usize])?;
        check(unsafe { rt_gemm(ctx(), 0, 0, m, n, k, a.ptr(), k, b.ptr(), n, out.ptr_mut(), n, 0) })?;
        Ok(out)
    }
    fn matmul_backward(op: &Op<Self>, g: &Self::Storage) -> Result<(Self::Storage, Self::Storage), Error> { // mod.rs:324: g*B^T, A^T*g, no transposes materialised
        let (a, b) = (&*op.inputs[0].data(), &*op.inputs[1].data());
        let (da, db) = (B200Storage::alloc(&a.shape)?, B200Storage::alloc(&b.shape)?);
        check(unsafe { rt_matmul_backward(ctx(), a.ptr(), b.ptr(), g.ptr(), a.shape[0] as i64, a.shape[1] as i64, b.shape[1] as i64, da.ptr_mut(), db.ptr_mut()) })?;
        Ok((da, db))
    }
    fn conv2d(x: &Self::Storage, w: &Self::Storage, bias: Option<&Self::Storage>, stride: (usize, usize), padding: (usize, usize)) -> Result<Self::Storage, Error> { // mod.rs:101
        let (n, cin, h, wd, cout, kh, kw) = (x.shape[0], x.shape[1], x.shape[2], x.shape[3], w.shape[0], w.shape[2], w.shape[3]);
        let (ho, wo) = ((h + 2 * padding.0 - kh) / stride.0 + 1, (wd + 2 * padding.1 - kw) / stride.1 + 1);
        let out = B200Storage::alloc(&[n, cout, ho, wo])?;
        check(unsafe { rt_conv2d(ctx(), x.ptr(), w.ptr(), bias.map_or(std::ptr::null(), |b| b.ptr()), n as i64, cin as i64, h as i64, wd as i64, cout as i64,
                                 kh as c_int, kw as c_int, stride.0 as c_int, stride.1 as c_int, padding.0 as c_int, padding.1 as c_int, out.ptr_mut()) })?;
        Ok(out)
    }
    fn conv2d_backward(x: &Self::Storage, w: &Self::Storage, g: &Self::Storage, stride: (usize, usize), padding: (usize, usize))
        -> Result<(Self::Storage, Self::Storage, Option<Self::Storage>), Error> {                      // mod.rs:111
        let (dx, dw, db) = (B200Storage::alloc(&x.shape)?, B200Storage::alloc(&w.shape)?, B200Storage::alloc(&[w.shape[0]])?);
        check(unsafe { rt_conv2d_backward(ctx(), x.ptr(), w.ptr(), g.ptr(), x.shape[0] as i64, x.shape[1] as i64, x.shape[2] as i64, x.shape[3] as i64,
                                          w.shape[0] as i64, w.shape[2] as c_int, w.shape[3] as c_int, stride.0 as c_int, stride.1 as c_int,
                                          padding.0 as c_int, padding.1 as c_int, dx.ptr_mut(), dw.ptr_mut(), db.ptr_mut()) })?;
        Ok((dx, dw, Some(db)))
    }
    fn conv2d_transpose(x: &Self::Storage, w: &Self::Storage, bias: Option<&Self::Storage>, stride: (usize, usize), padding: (usize, usize)) -> Result<Self::Storage, Error> { // mod.rs:125
        let (n, cin, h, wd, cout, kh, kw) = (x.shape[0], x.shape[1], x.shape[2], x.shape[3], w.shape[1], w.shape[2], w.shape[3]);
        let (oh, ow) = ((h - 1) * stride.0 + kh - 2 * padding.0, (wd - 1) * stride.1 + kw - 2 * padding.1);
        let out = B200Storage::alloc(&[n, cout, oh, ow])?;
        check(unsafe { rt_conv2d_transpose(ctx(), x.ptr(), w.ptr(), bias.map_or(std::ptr::null(), |b| b.ptr()), n as i64, cin as i64, h as i64, wd as i64, cout as i64,
                                           kh as c_int, kw as c_int, stride.0 as c_int, stride.1 as c_int, padding.0 as c_int, padding.1 as c_int, out.ptr_mut()) })?;
        Ok(out)
    }
    fn conv2d_transpose_backward(x: &Self::Storage, w: &Self::Storage, g: &Self::Storage, stride: (usize, usize), padding: (usize, usize))
        -> Result<(Self::Storage, Self::Storage, Option<Self::Storage>), Error> {                      // mod.rs:135
        let (dx, dw, db) = (B200Storage::alloc(&x.shape)?, B200Storage::alloc(&w.shape)?, B200Storage::alloc(&[w.shape[1]])?);
        check(unsafe { rt_conv2d_transpose_backward(ctx(), x.ptr(), w.ptr(), g.ptr(), x.shape[0] as i64, x.shape[1] as i64, x.shape[2] as i64, x.shape[3] as i64,
                                                    w.shape[1] as i64, w.shape[2] as c_int, w.shape[3] as c_int, stride.0 as c_int, stride.1 as c_int,
                                                    padding.0 as c_int, padding.1 as c_int, dx.ptr_mut(), dw.ptr_mut(), db.ptr_mut()) })?;
        Ok((dx, dw, Some(db)))
    }
    fn max_pool2d(x: &Self::Storage, kernel_size: (usize, usize), stride: (usize, usize), padding: (usize, usize)) -> Result<(Self::Storage, Self::Storage), Error> { // mod.rs:144
        let (n, c, h, w) = (x.shape[0], x.shape[1], x.shape[2], x.shape[3]);
        let (ho, wo) = ((h + 2 * padding.0 - kernel_size.0) / stride.0 + 1, (w + 2 * padding.1 - kernel_size.1) / stride.1 + 1);
        let (y, idx) = (B200Storage::alloc(&[n, c, ho, wo])?, B200Storage::alloc(&[n, c, ho, wo])?);
        check(unsafe { rt_max_pool2d(ctx(), x.ptr(), n as i64, c as i64, h as i64, w as i64, kernel_size.0 as c_int, kernel_size.1 as c_int,
                                     stride.0 as c_int, stride.1 as c_int, padding.0 as c_int, padding.1 as c_int, y.ptr_mut(), idx.ptr_mut()) })?;
        Ok((y, idx))
    }
    fn max_pool2d_backward(op: &Op<Self>, g: &Self::Storage) -> Result<Self::Storage, Error> {       // mod.rs:151: inputs = [x, indices]
        let (k, s, p) = match op.op_type { OpType::MaxPool2D { kernel_size, stride, padding } => (kernel_size, stride, padding), _ => return Err(Error::InternalLogicError("max_pool2d_backward: wrong op type".into())) };
        let (x, idx) = (&*op.inputs[0].data(), &*op.inputs[1].data());
        let dx = B200Storage::alloc(&x.shape)?;
        check(unsafe { rt_max_pool2d_backward(ctx(), g.ptr(), idx.ptr(), x.shape[0] as i64, x.shape[1] as i64, x.shape[2] as i64, x.shape[3] as i64,
                                              k.0 as c_int, k.1 as c_int, s.0 as c_int, s.1 as c_int, p.0 as c_int, p.1 as c_int, dx.ptr_mut()) })?;
        Ok(dx)
    }

    // ---- optimizer steps, in place (mod.rs:18-36, 256-272) ----
    fn sgd_step(w: &mut Self::Storage, dw: &Self::Storage, lr: f32) -> Result<(), Error> {
        let n = w.numel() as i64;
        check(unsafe { rt_sgd_step(ctx(), w.unique_ptr_mut()?, dw.ptr(), n, lr) })
    }
    fn momentum_sgd_step(p: &mut Self::Storage, g: &Self::Storage, v: &mut Self::Storage, lr: f32, momentum: f32) -> Result<(), Error> {
        let n = p.numel() as i64;
        check(unsafe { rt_momentum_sgd_step(ctx(), p.unique_ptr_mut()?, g.ptr(), v.unique_ptr_mut()?, n, lr, momentum) })
    }
    fn adagrad_step(p: &mut Self::Storage, g: &Self::Storage, acc: &mut Self::Storage, lr: f32, epsilon: f32) -> Result<(), Error> {
        let n = p.numel() as i64;
        check(unsafe { rt_adagrad_step(ctx(), p.unique_ptr_mut()?, g.ptr(), acc.unique_ptr_mut()?, n, lr, epsilon) })
    }
    fn adam_step(p: &mut Self::Storage, g: &Self::Storage, m: &mut Self::Storage, v: &mut Self::Storage, lr: f32, beta1: f32, beta2: f32,
                 epsilon: f32, t: usize) -> Result<(), Error> {
        let n = p.numel() as i64;
        check(unsafe { rt_adam_step(ctx(), p.unique_ptr_mut()?, g.ptr(), m.unique_ptr_mut()?, v.unique_ptr_mut()?, n, lr, beta1, beta2, epsilon, t as i64) })
    }
}
