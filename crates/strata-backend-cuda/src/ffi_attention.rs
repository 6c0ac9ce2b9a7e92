//! `extern "C"` declarations of `include/strata_attention.h`: attention over a
//! paged cache and the scoring of tokens, on device buffers. Contexts and status
//! codes are [`crate::ffi`]'s; [`crate::attention`] calls them.

#![allow(non_camel_case_types)]

use std::os::raw::{c_int, c_void};

use crate::ffi::StrataCtx;

/// `strata_kv_cache`: one layer's pages, tables and lengths.
#[repr(C)]
pub(crate) struct strata_kv_cache {
    pub(crate) k_dev: *mut c_void,
    pub(crate) v_dev: *mut c_void,
    pub(crate) table_dev: *const i32,
    pub(crate) len_dev: *const i32,
    pub(crate) n_pages: i64,
    pub(crate) page_size: i64,
    pub(crate) n_kv_head: i64,
    pub(crate) head_dim: i64,
    pub(crate) page_stride: i64,
    pub(crate) token_stride: i64,
    pub(crate) head_stride: i64,
    pub(crate) max_pages: i64,
    pub(crate) table_stride: i64,
}

/// `strata_kv_append`: the shape of one append.
#[repr(C)]
pub(crate) struct strata_kv_append {
    pub(crate) n_seq: i64,
    pub(crate) seq_len: i64,
    pub(crate) seq_offsets: *const i64,
    pub(crate) n_head: i64,
    pub(crate) n_rot: i64,
    pub(crate) q_stride: i64,
    pub(crate) k_stride: i64,
    pub(crate) v_stride: i64,
    pub(crate) q_out_stride: i64,
    pub(crate) freq_base: f64,
    pub(crate) dtype: u32,
    pub(crate) q_dtype: u32,
    pub(crate) neighbours: c_int,
}

/// `strata_attention`: the shape of one attention call.
#[repr(C)]
pub(crate) struct strata_attention {
    pub(crate) n_seq: i64,
    pub(crate) seq_len: i64,
    pub(crate) seq_offsets: *const i64,
    pub(crate) n_head: i64,
    pub(crate) q_stride: i64,
    pub(crate) o_stride: i64,
    pub(crate) window: i64,
    pub(crate) sinks: i64,
    pub(crate) scale: f64,
    pub(crate) dtype: u32,
}

extern "C" {
    pub(crate) fn strata_cuda_kv_append_dev(
        ctx: *mut StrataCtx,
        desc: *const strata_kv_append,
        cache: *const strata_kv_cache,
        q_dev: *const c_void,
        k_dev: *const c_void,
        v_dev: *const c_void,
        q_out_dev: *mut c_void,
        stream: *mut c_void,
    ) -> c_int;
    pub(crate) fn strata_cuda_attention_work_bytes(
        desc: *const strata_attention,
        cache: *const strata_kv_cache,
        bytes: *mut u64,
    ) -> c_int;
    pub(crate) fn strata_cuda_attention_dev(
        ctx: *mut StrataCtx,
        desc: *const strata_attention,
        cache: *const strata_kv_cache,
        q_dev: *const c_void,
        o_dev: *mut c_void,
        work_dev: *mut c_void,
        work_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub(crate) fn strata_cuda_logprobs_dev(
        ctx: *mut StrataCtx,
        logits_dev: *const f32,
        rows: i64,
        vocab: i64,
        stride: i64,
        targets_dev: *const i32,
        logprobs_dev: *mut f32,
        entropy_dev: *mut f32,
        top: i64,
        top_ids_dev: *mut i32,
        top_logprobs_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
}
