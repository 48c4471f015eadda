//! Raw bindings to `libturq.so` (include/turq.h). Generated by gen_bindings.py; do not edit.
//!
//! Every entry returns a `turq_status` as `i32` (0 = OK) and never unwinds across the boundary.
#![allow(non_camel_case_types)]
#![no_std]

use core::ffi::{c_char, c_void};

/// Opaque handle owned by the library.
#[repr(C)]
pub struct turq_ctx {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct turq_qtensor {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct turq_tp {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct turq_host_call {
    _private: [u8; 0],
}

/// Opaque handle owned by the library.
#[repr(C)]
pub struct turq_kv_cache {
    _private: [u8; 0],
}

pub const TURQ_VERSION: i32 = 100;
pub const TURQ_STATIC_SCRATCH_BYTES: usize = 4 << 20;
pub const TURQ_TP_HANDLE_BYTES: usize = 64;

// enum turq_status
pub const TURQ_OK: i32 = 0;
pub const TURQ_E_INVALID_ARG: i32 = 1;
pub const TURQ_E_SHAPE: i32 = 2;
pub const TURQ_E_DTYPE: i32 = 3;
pub const TURQ_E_ALIGN: i32 = 4;
pub const TURQ_E_CUDA: i32 = 5;
pub const TURQ_E_NCCL: i32 = 6;
pub const TURQ_E_TIMEOUT: i32 = 7;
pub const TURQ_E_NO_DEVICE: i32 = 8;
pub const TURQ_E_LIMIT: i32 = 9;

// enum turq_dtype
pub const TURQ_F32: i32 = 0;
pub const TURQ_F16: i32 = 1;
pub const TURQ_Q8_0: i32 = 8;
pub const TURQ_Q4_K: i32 = 12;
pub const TURQ_Q5_K: i32 = 13;
pub const TURQ_Q6_K: i32 = 14;
pub const TURQ_Q8_K: i32 = 15;
pub const TURQ_BF16: i32 = 30;

// enum turq_mode
pub const TURQ_MODE_AUTO: i32 = 0;
pub const TURQ_MODE_INT8_ACT: i32 = 1;
pub const TURQ_MODE_EXACT_F32: i32 = 2;
pub const TURQ_MODE_TENSOR_CORE: i32 = 3;

extern "C" {
    pub fn turq_version() -> i32;
    pub fn turq_q8k_variant() -> i32;
    pub fn turq_status_string(status: i32) -> *const c_char;
    pub fn turq_block_elems(dtype: i32) -> i32;
    pub fn turq_block_bytes(dtype: i32) -> i32;
    pub fn turq_row_bytes(dtype: i32, k: i64) -> usize;
    pub fn turq_ctx_create(device: i32, out: *mut *mut turq_ctx) -> i32;
    pub fn turq_ctx_destroy(ctx: *mut turq_ctx) -> i32;
    pub fn turq_last_error(ctx: *const turq_ctx) -> *const c_char;
    pub fn turq_ctx_reserve(ctx: *mut turq_ctx, max_m: i64, max_k: i64, max_n: i64) -> i32;
    pub fn turq_ctx_set_auto_policy(ctx: *mut turq_ctx, mode: i32) -> i32;
    pub fn turq_ctx_poll_status(ctx: *mut turq_ctx, stream: *mut c_void) -> i32;
    pub fn turq_ctx_launch_count(ctx: *const turq_ctx) -> i64;
    pub fn turq_qtensor_from_host(
        ctx: *mut turq_ctx,
        dtype: i32,
        n_rows: i64,
        n_cols: i64,
        host_blocks: *const c_void,
        nbytes: usize,
        out: *mut *mut turq_qtensor,
    ) -> i32;
    pub fn turq_qtensor_from_device(
        ctx: *mut turq_ctx,
        dtype: i32,
        n_rows: i64,
        n_cols: i64,
        dev_blocks: *const c_void,
        nbytes: usize,
        stream: *mut c_void,
        out: *mut *mut turq_qtensor,
    ) -> i32;
    pub fn turq_qtensor_slice_rows(
        ctx: *mut turq_ctx,
        src: *const turq_qtensor,
        row0: i64,
        n: i64,
        out: *mut *mut turq_qtensor,
    ) -> i32;
    pub fn turq_qtensor_slice_cols(
        ctx: *mut turq_ctx,
        src: *const turq_qtensor,
        col0: i64,
        n: i64,
        out: *mut *mut turq_qtensor,
    ) -> i32;
    pub fn turq_qtensor_free(qt: *mut turq_qtensor) -> i32;
    pub fn turq_qtensor_info(
        qt: *const turq_qtensor,
        dtype: *mut i32,
        n_rows: *mut i64,
        n_cols: *mut i64,
        wire_bytes: *mut usize,
    ) -> i32;
    pub fn turq_dequantize(
        ctx: *mut turq_ctx,
        qt: *const turq_qtensor,
        out_dtype: i32,
        dev_out: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_embedding(
        ctx: *mut turq_ctx,
        qt: *const turq_qtensor,
        dev_ids: *const i32,
        n_ids: i64,
        out_dtype: i32,
        dev_out: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_quantize_weights(
        ctx: *mut turq_ctx,
        dtype: i32,
        dev_x: *const f32,
        n_rows: i64,
        n_cols: i64,
        dev_blocks: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_quantize_act(
        ctx: *mut turq_ctx,
        fmt: i32,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        k: i64,
        dev_blocks: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qmatmul(
        ctx: *mut turq_ctx,
        qt: *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        dev_y: *mut f32,
        mode: i32,
        dev_bias: *const f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qmatmul_multi(
        ctx: *mut turq_ctx,
        count: i32,
        qts: *const *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        dev_ys: *const *mut f32,
        mode: i32,
        dev_biases: *const *const f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qmatmul_host(
        ctx: *mut turq_ctx,
        qt: *const turq_qtensor,
        host_x: *const f32,
        m: i64,
        host_y: *mut f32,
        mode: i32,
        host_bias: *const f32,
    ) -> i32;
    pub fn turq_qmatmul_multi_host(
        ctx: *mut turq_ctx,
        count: i32,
        qts: *const *const turq_qtensor,
        host_x: *const f32,
        m: i64,
        host_ys: *const *mut f32,
        mode: i32,
        host_biases: *const *const f32,
    ) -> i32;
    pub fn turq_host_call_create(
        ctx: *mut turq_ctx,
        count: i32,
        qts: *const *const turq_qtensor,
        host_x: *const f32,
        m: i64,
        host_ys: *const *mut f32,
        out: *mut *mut turq_host_call,
    ) -> i32;
    pub fn turq_host_call_run(call: *mut turq_host_call) -> i32;
    pub fn turq_host_call_destroy(call: *mut turq_host_call) -> i32;
    pub fn turq_qmatmul_static(
        ctx: *mut turq_ctx,
        qt: *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        dev_y: *mut f32,
        dev_bias: *const f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qmatmul_swiglu(
        ctx: *mut turq_ctx,
        gate: *const turq_qtensor,
        up: *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        dev_out: *mut f32,
        mode: i32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_rmsnorm_qmatmul_multi(
        ctx: *mut turq_ctx,
        count: i32,
        qts: *const *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        dev_norm_weight: *const f32,
        eps: f32,
        dev_h_out: *mut f32,
        dev_ys: *const *mut f32,
        mode: i32,
        dev_biases: *const *const f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_topk(
        ctx: *mut turq_ctx,
        dev_vals: *const f32,
        dev_ids: *const i32,
        m: i64,
        n: i64,
        k: i32,
        id_offset: i32,
        dev_out_vals: *mut f32,
        dev_out_ids: *mut i32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_lm_head_topk(
        ctx: *mut turq_ctx,
        qt: *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        k: i32,
        id_offset: i32,
        dev_out_vals: *mut f32,
        dev_out_ids: *mut i32,
        dev_logits: *mut f32,
        mode: i32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_rope_table(
        ctx: *mut turq_ctx,
        host_freqs: *const f64,
        n_freqs: i32,
        n_positions: i64,
        scale: f64,
        dev_table: *mut f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qk_norm_rope(
        ctx: *mut turq_ctx,
        dev_q: *const c_void,
        q_stride: i64,
        dev_k: *const c_void,
        k_stride: i64,
        x_dtype: i32,
        n_tokens: i64,
        n_q_heads: i32,
        n_kv_heads: i32,
        head_dim: i32,
        dev_q_weight: *const f32,
        dev_k_weight: *const f32,
        eps: f32,
        dev_table: *const f32,
        n_positions: i64,
        rotary_dim: i32,
        interleaved: i32,
        dev_positions: *const i32,
        out_dtype: i32,
        dev_q_out: *mut c_void,
        dev_k_out: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_kv_cache_bytes(
        dtype: i32,
        n_pages: i64,
        page_size: i32,
        n_kv_heads: i32,
        head_dim: i32,
    ) -> usize;
    pub fn turq_kv_cache_create(
        ctx: *mut turq_ctx,
        dtype: i32,
        n_pages: i64,
        page_size: i32,
        n_kv_heads: i32,
        head_dim: i32,
        dev_memory: *mut c_void,
        nbytes: usize,
        out: *mut *mut turq_kv_cache,
    ) -> i32;
    pub fn turq_kv_cache_free(cache: *mut turq_kv_cache) -> i32;
    pub fn turq_kv_cache_layout(
        cache: *const turq_kv_cache,
        dev_memory: *mut *mut c_void,
        offsets: *mut i64,
    ) -> i32;
    pub fn turq_kv_append(
        ctx: *mut turq_ctx,
        cache: *mut turq_kv_cache,
        dev_q: *const c_void,
        q_stride: i64,
        dev_k: *const c_void,
        k_stride: i64,
        dev_v: *const c_void,
        v_stride: i64,
        x_dtype: i32,
        n_tokens: i64,
        n_q_heads: i32,
        dev_q_weight: *const f32,
        dev_k_weight: *const f32,
        eps: f32,
        dev_table: *const f32,
        n_positions: i64,
        rotary_dim: i32,
        interleaved: i32,
        dev_positions: *const i32,
        dev_slots: *const i64,
        out_dtype: i32,
        dev_q_out: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_kv_write(
        ctx: *mut turq_ctx,
        cache: *mut turq_kv_cache,
        dev_k: *const c_void,
        k_stride: i64,
        dev_v: *const c_void,
        v_stride: i64,
        x_dtype: i32,
        n_tokens: i64,
        dev_slots: *const i64,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_kv_read(
        ctx: *mut turq_ctx,
        cache: *const turq_kv_cache,
        dev_slots: *const i64,
        n_tokens: i64,
        out_dtype: i32,
        dev_k_out: *mut c_void,
        dev_v_out: *mut c_void,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_kv_attention_workspace(
        cache: *const turq_kv_cache,
        n_tokens: i64,
        n_seqs: i32,
        n_q_heads: i32,
        max_new: i64,
        max_context: i64,
    ) -> usize;
    pub fn turq_kv_attention(
        ctx: *mut turq_ctx,
        cache: *const turq_kv_cache,
        dev_q: *const c_void,
        q_stride: i64,
        q_dtype: i32,
        n_tokens: i64,
        n_q_heads: i32,
        dev_starts: *const i32,
        dev_contexts: *const i32,
        dev_page_table: *const i32,
        table_stride: i64,
        n_seqs: i32,
        max_new: i64,
        max_context: i64,
        scale: f32,
        causal: i32,
        out_dtype: i32,
        dev_out: *mut c_void,
        dev_workspace: *mut c_void,
        workspace_bytes: usize,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_tp_create(
        ctx: *mut turq_ctx,
        rank: i32,
        world: i32,
        max_bytes: usize,
        out: *mut *mut turq_tp,
    ) -> i32;
    pub fn turq_tp_export(tp: *const turq_tp, handle_out: *mut c_void) -> i32;
    pub fn turq_tp_connect(tp: *mut turq_tp, handles: *const c_void) -> i32;
    pub fn turq_tp_destroy(tp: *mut turq_tp) -> i32;
    pub fn turq_tp_set_wait_limit(tp: *mut turq_tp, cycles: i64) -> i32;
    pub fn turq_tp_set_fuse_limit(tp: *mut turq_tp, bytes: i64) -> i32;
    pub fn turq_tp_set_twoshot_limit(tp: *mut turq_tp, bytes: i64) -> i32;
    pub fn turq_tp_set_chunk_rows(tp: *mut turq_tp, rows: i64) -> i32;
    pub fn turq_tp_reset(tp: *mut turq_tp) -> i32;
    pub fn turq_tp_allreduce(
        tp: *mut turq_tp,
        dev_in: *const f32,
        dev_out: *mut f32,
        count: i64,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_tp_allgather(
        tp: *mut turq_tp,
        dev_in: *const f32,
        m: i64,
        widths: *const i64,
        dev_out: *mut f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qmatmul_rowparallel(
        tp: *mut turq_tp,
        qt: *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        dev_y: *mut f32,
        mode: i32,
        dev_bias: *const f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_qmatmul_gather(
        tp: *mut turq_tp,
        qt: *const turq_qtensor,
        dev_x: *const c_void,
        x_dtype: i32,
        m: i64,
        widths: *const i64,
        dev_out: *mut f32,
        mode: i32,
        dev_bias: *const f32,
        stream: *mut c_void,
    ) -> i32;
    pub fn turq_tp_connect_loopback(tp: *mut turq_tp) -> i32;
    pub fn turq_tp_loopback_fill(
        tp: *mut turq_tp,
        peer: i32,
        dev_src: *const f32,
        count: i64,
        signal: i32,
        stream: *mut c_void,
    ) -> i32;
}
