//! The sequence operators (`include/strata_sequence.h`) for an engine that
//! keeps a token's activations on the device: what the reference runs on the
//! host in `crates/strata-core/src/gdn.rs` and, behind the penalties, in
//! `crates/strata-core/src/sampler.rs`.
//!
//! Buffers are device memory of the backend's device (from any allocator of
//! the CUDA runtime or driver); a call only enqueues work on `stream` (null:
//! the backend's own). What each buffer holds, and which ones may be null, is
//! in the header.

use std::os::raw::c_void;

use strata_core::error::{Error, Result};
use strata_gguf::quant::QuantType;

use crate::ffi;
use crate::ffi_sequence::{
    strata_cuda_gated_delta_dev, strata_cuda_gated_delta_work_bytes, strata_cuda_sample_dev,
    strata_cuda_short_conv_dev, strata_gated_delta, strata_short_conv,
};
use crate::CudaBackend;

/// The type of the activations; states, weights and gates are f32.
#[derive(Debug, Clone, Copy, PartialEq, Eq)]
pub enum Activations {
    /// 32-bit floats.
    F32,
    /// bfloat16.
    Bf16,
}

impl Activations {
    fn id(self) -> u32 {
        match self {
            Self::F32 => 0,   // STRATA_QUANT_F32
            Self::Bf16 => 30, // STRATA_QUANT_BF16
        }
    }
}

/// Which rows of a call's buffers are whose tokens.
#[derive(Debug, Clone, Copy)]
pub enum Sequences<'a> {
    /// `count` sequences of `len` tokens each, one after another.
    Uniform {
        /// Number of sequences.
        count: i64,
        /// Tokens of each.
        len: i64,
    },
    /// Sequence `i` has the rows from `offsets[i]` up to `offsets[i + 1]`.
    Offsets(&'a [i64]),
}

impl Sequences<'_> {
    /// `n_seq`, `seq_len` and `seq_offsets` of a call.
    fn parts(&self) -> (i64, i64, *const i64) {
        match *self {
            Self::Uniform { count, len } => (count, len, std::ptr::null()),
            // no offsets at all are no sequences, which the library refuses
            Self::Offsets(rows) => (rows.len() as i64 - 1, 0, rows.as_ptr()),
        }
    }
}

/// The shape of a short convolution (`strata_short_conv`); strides of 0 are packed.
#[derive(Debug, Clone, Copy)]
pub struct ShortConv<'a> {
    /// The call's tokens.
    pub sequences: Sequences<'a>,
    /// Channels of a token.
    pub channels: i64,
    /// Taps of a channel, 1 to 8.
    pub taps: i64,
    /// Elements from one token to the next in `x`.
    pub x_stride: i64,
    /// Elements from one token to the next in `y`.
    pub y_stride: i64,
    /// The type of `x` and `y`.
    pub activations: Activations,
    /// Whether the sums go through SiLU.
    pub silu: bool,
}

/// The shape of a gated delta rule call (`strata_gated_delta`); strides of 0 are packed.
#[derive(Debug, Clone, Copy)]
pub struct GatedDelta<'a> {
    /// The call's tokens.
    pub sequences: Sequences<'a>,
    /// Heads of q and k.
    pub n_k_head: i64,
    /// Heads of v and o, a multiple of `n_k_head`.
    pub n_v_head: i64,
    /// Elements of a head of q and k.
    pub k_dim: i64,
    /// Elements of a head of v and o.
    pub v_dim: i64,
    /// Elements from one token to the next in `q`, `k`, `v` and `o`.
    pub strides: [i64; 4],
    /// Floats from one token to the next in `gate` and `beta`.
    pub gate_strides: [i64; 2],
    /// What the outputs are multiplied with.
    pub scale: f64,
    /// Added to the sum of squares that q and k are normalised by; negative: they are taken as they are.
    pub l2_eps: f64,
    /// The type of `q`, `k`, `v` and `o`.
    pub activations: Activations,
    /// Whether value head `h` reads key head `h mod n_k_head` (else `h / (n_v_head / n_k_head)`).
    pub tiled: bool,
    /// Whether `gate` and `beta` are as the projections give them.
    pub raw_gates: bool,
}

impl GatedDelta<'_> {
    fn desc(&self) -> strata_gated_delta {
        let (n_seq, seq_len, seq_offsets) = self.sequences.parts();
        strata_gated_delta {
            n_seq,
            seq_len,
            seq_offsets,
            n_k_head: self.n_k_head,
            n_v_head: self.n_v_head,
            k_dim: self.k_dim,
            v_dim: self.v_dim,
            q_stride: self.strides[0],
            k_stride: self.strides[1],
            v_stride: self.strides[2],
            o_stride: self.strides[3],
            gate_stride: self.gate_strides[0],
            beta_stride: self.gate_strides[1],
            scale: self.scale,
            l2_eps: self.l2_eps,
            dtype: self.activations.id(),
            tiled: i32::from(self.tiled),
            raw_gates: i32::from(self.raw_gates),
        }
    }

    /// Bytes of device workspace that [`CudaBackend::gated_delta`] needs (0: none).
    pub fn work_bytes(&self) -> Result<u64> {
        let desc = self.desc();
        let mut bytes = 0;
        let rc = unsafe { strata_cuda_gated_delta_work_bytes(&desc, &mut bytes) };
        if rc == ffi::STRATA_OK {
            Ok(bytes)
        } else {
            Err(Error::Backend {
                message: format!("gated_delta: bad shape (status {rc})"),
            })
        }
    }
}

/// The device buffers of a gated delta rule call.
#[derive(Debug, Clone, Copy)]
pub struct GatedDeltaBuffers {
    /// Queries.
    pub q: *const c_void,
    /// Keys.
    pub k: *const c_void,
    /// Values.
    pub v: *const c_void,
    /// Log decays, or what they are made of.
    pub gate: *const f32,
    /// Steps, or what they are made of.
    pub beta: *const f32,
    /// Decay rates of raw gates (null without).
    pub coef: *const f32,
    /// Shifts of raw gates, or null.
    pub shift: *const f32,
    /// The states, updated in place.
    pub state: *mut f32,
    /// Outputs.
    pub o: *mut c_void,
    /// Workspace of `work_bytes` bytes, or null where none is needed.
    pub work: *mut c_void,
    /// Its size.
    pub work_bytes: u64,
}

/// The device buffers of a sampling call: one setting a row, null where it is off.
#[derive(Debug, Clone, Copy)]
pub struct SampleBuffers {
    /// Rows of logits.
    pub logits: *const f32,
    /// Temperatures.
    pub temperature: *const f32,
    /// Numbers of tokens that top-k keeps.
    pub top_k: *const i32,
    /// Masses that top-p keeps.
    pub top_p: *const f32,
    /// Least probabilities, relative to the largest.
    pub min_p: *const f32,
    /// Random numbers in [0, 1).
    pub uniform: *const f64,
    /// The tokens taken (-1: none is left).
    pub ids: *mut i32,
    /// Their log-probabilities, or null.
    pub logprobs: *mut f32,
}

impl CudaBackend {
    /// The short causal convolution over `shape`'s tokens, its states updated in place.
    ///
    /// # Safety
    /// The pointers are device memory of the sizes that the header gives for
    /// `shape`, and stay so until the work on `stream` is done.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn short_conv(
        &self,
        shape: &ShortConv<'_>,
        x: *const c_void,
        w: *const f32,
        bias: *const f32,
        state: *mut f32,
        y: *mut c_void,
        stream: *mut c_void,
    ) -> Result<()> {
        let (n_seq, seq_len, seq_offsets) = shape.sequences.parts();
        let desc = strata_short_conv {
            n_seq,
            seq_len,
            seq_offsets,
            channels: shape.channels,
            taps: shape.taps,
            x_stride: shape.x_stride,
            y_stride: shape.y_stride,
            dtype: shape.activations.id(),
            silu: i32::from(shape.silu),
        };
        let rc = unsafe { strata_cuda_short_conv_dev(self.ctx, &desc, x, w, bias, state, y, stream) };
        self.check(rc, QuantType::F32)
    }

    /// The gated delta rule over `shape`'s tokens, its states updated in place.
    /// A device wait that expires is reported by [`CudaBackend::synchronize`].
    ///
    /// # Safety
    /// As for [`CudaBackend::short_conv`]; calls that may overlap need a workspace each.
    pub unsafe fn gated_delta(&self, shape: &GatedDelta<'_>, b: &GatedDeltaBuffers, stream: *mut c_void) -> Result<()> {
        let desc = shape.desc();
        let rc = unsafe {
            strata_cuda_gated_delta_dev(
                self.ctx,
                &desc,
                b.q,
                b.k,
                b.v,
                b.gate,
                b.beta,
                b.coef,
                b.shift,
                b.state,
                b.o,
                b.work,
                b.work_bytes,
                stream,
            )
        };
        self.check(rc, QuantType::F32)
    }

    /// One token for each of `rows` rows of `vocab` logits, `stride` floats
    /// apart (0: packed). Penalties are the caller's to apply before.
    ///
    /// # Safety
    /// As for [`CudaBackend::short_conv`].
    pub unsafe fn sample(&self, rows: i64, vocab: i64, stride: i64, b: &SampleBuffers, stream: *mut c_void)
        -> Result<()> {
        let rc = unsafe {
            strata_cuda_sample_dev(
                self.ctx,
                b.logits,
                rows,
                vocab,
                stride,
                b.temperature,
                b.top_k,
                b.top_p,
                b.min_p,
                b.uniform,
                b.ids,
                b.logprobs,
                stream,
            )
        };
        self.check(rc, QuantType::F32)
    }

    /// Waits for the work on the backend's own stream, and reports a device
    /// wait that has expired on any.
    pub fn synchronize(&self) -> Result<()> {
        let rc = unsafe { ffi::strata_cuda_synchronize(self.ctx) };
        self.check(rc, QuantType::F32)
    }
}
