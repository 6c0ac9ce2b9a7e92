//! `extern "C"` declarations of `include/strata_sequence.h`: the sequence
//! operators (short convolution, gated delta rule, sampling) on device buffers.
//! Contexts and status codes are [`crate::ffi`]'s; [`crate::sequence`] calls them.

#![allow(non_camel_case_types)]

use std::os::raw::{c_int, c_void};

use crate::ffi::StrataCtx;

/// `strata_short_conv`: the shape of one convolution call.
#[repr(C)]
pub(crate) struct strata_short_conv {
    pub(crate) n_seq: i64,
    pub(crate) seq_len: i64,
    pub(crate) seq_offsets: *const i64,
    pub(crate) channels: i64,
    pub(crate) taps: i64,
    pub(crate) x_stride: i64,
    pub(crate) y_stride: i64,
    pub(crate) dtype: u32,
    pub(crate) silu: c_int,
}

/// `strata_gated_delta`: the shape of one gated delta rule call.
#[repr(C)]
pub(crate) struct strata_gated_delta {
    pub(crate) n_seq: i64,
    pub(crate) seq_len: i64,
    pub(crate) seq_offsets: *const i64,
    pub(crate) n_k_head: i64,
    pub(crate) n_v_head: i64,
    pub(crate) k_dim: i64,
    pub(crate) v_dim: i64,
    pub(crate) q_stride: i64,
    pub(crate) k_stride: i64,
    pub(crate) v_stride: i64,
    pub(crate) o_stride: i64,
    pub(crate) gate_stride: i64,
    pub(crate) beta_stride: i64,
    pub(crate) scale: f64,
    pub(crate) l2_eps: f64,
    pub(crate) dtype: u32,
    pub(crate) tiled: c_int,
    pub(crate) raw_gates: c_int,
}

extern "C" {
    pub(crate) fn strata_cuda_short_conv_dev(
        ctx: *mut StrataCtx,
        desc: *const strata_short_conv,
        x_dev: *const c_void,
        w_dev: *const f32,
        bias_dev: *const f32,
        state_dev: *mut f32,
        y_dev: *mut c_void,
        stream: *mut c_void,
    ) -> c_int;
    pub(crate) fn strata_cuda_gated_delta_work_bytes(desc: *const strata_gated_delta, bytes: *mut u64) -> c_int;
    pub(crate) fn strata_cuda_gated_delta_dev(
        ctx: *mut StrataCtx,
        desc: *const strata_gated_delta,
        q_dev: *const c_void,
        k_dev: *const c_void,
        v_dev: *const c_void,
        gate_dev: *const f32,
        beta_dev: *const f32,
        coef_dev: *const f32,
        shift_dev: *const f32,
        state_dev: *mut f32,
        o_dev: *mut c_void,
        work_dev: *mut c_void,
        work_bytes: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub(crate) fn strata_cuda_sample_dev(
        ctx: *mut StrataCtx,
        logits_dev: *const f32,
        rows: i64,
        vocab: i64,
        stride: i64,
        temperature_dev: *const f32,
        top_k_dev: *const i32,
        top_p_dev: *const f32,
        min_p_dev: *const f32,
        uniform_dev: *const f64,
        ids_dev: *mut i32,
        logprobs_dev: *mut f32,
        stream: *mut c_void,
    ) -> c_int;
}
