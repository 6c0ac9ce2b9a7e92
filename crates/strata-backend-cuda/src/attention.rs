//! Attention over a paged cache and the scoring of tokens
//! (`include/strata_attention.h`) for an engine that keeps a token's activations
//! on the device: what the reference runs on the host in
//! `crates/strata-core/src/qsa.rs`.
//!
//! Buffers are device memory of the backend's device; a call only enqueues work
//! on `stream` (null: the backend's own). What each buffer holds, and which ones
//! may be null, is in the header. [`crate::CudaBackend::synchronize`] reports a
//! device wait that has expired.

use std::os::raw::c_void;

use strata_core::error::{Error, Result};
use strata_gguf::quant::QuantType;

use crate::ffi;
use crate::ffi_attention::{
    strata_attention, strata_cuda_attention_dev, strata_cuda_attention_work_bytes, strata_cuda_kv_append_dev,
    strata_cuda_logprobs_dev, strata_kv_append, strata_kv_cache,
};
use crate::sequence::{Activations, Sequences};
use crate::CudaBackend;

/// A paged cache of one layer's keys and values, bf16 (`strata_kv_cache`);
/// strides of 0 are packed.
#[derive(Debug, Clone, Copy)]
pub struct KvCache {
    /// The keys' pages.
    pub k: *mut c_void,
    /// The values' pages.
    pub v: *mut c_void,
    /// A row of page numbers a sequence.
    pub table: *const i32,
    /// Tokens of each sequence, those of the call included.
    pub len: *const i32,
    /// Pages of a pool.
    pub n_pages: i64,
    /// Tokens of a page, a multiple of 16.
    pub page_size: i64,
    /// Heads of keys and values.
    pub n_kv_head: i64,
    /// Elements of a head, a multiple of 8 up to 256.
    pub head_dim: i64,
    /// Elements from one page, token and head to the next.
    pub strides: [i64; 3],
    /// Entries of a row of the table.
    pub max_pages: i64,
    /// Entries from one row of the table to the next.
    pub table_stride: i64,
}

impl KvCache {
    fn desc(&self) -> strata_kv_cache {
        strata_kv_cache {
            k_dev: self.k,
            v_dev: self.v,
            table_dev: self.table,
            len_dev: self.len,
            n_pages: self.n_pages,
            page_size: self.page_size,
            n_kv_head: self.n_kv_head,
            head_dim: self.head_dim,
            page_stride: self.strides[0],
            token_stride: self.strides[1],
            head_stride: self.strides[2],
            max_pages: self.max_pages,
            table_stride: self.table_stride,
        }
    }
}

/// The shape of an append (`strata_kv_append`); strides of 0 are packed.
#[derive(Debug, Clone, Copy)]
pub struct KvAppend<'a> {
    /// The call's tokens.
    pub sequences: Sequences<'a>,
    /// Heads of the queries (0: none).
    pub n_head: i64,
    /// Elements of a head that are turned.
    pub n_rot: i64,
    /// Elements from one token to the next in `q`, `k`, `v` and `q_out`.
    pub strides: [i64; 4],
    /// The base of the angles' frequencies.
    pub freq_base: f64,
    /// The type of `q`, `k` and `v`.
    pub activations: Activations,
    /// The type of `q_out`.
    pub queries: Activations,
    /// Whether pairs are neighbours (else halves apart).
    pub neighbours: bool,
}

/// The shape of an attention call (`strata_attention`); strides of 0 are packed.
#[derive(Debug, Clone, Copy)]
pub struct Attention<'a> {
    /// The call's tokens.
    pub sequences: Sequences<'a>,
    /// Heads of the queries, a multiple of the cache's.
    pub n_head: i64,
    /// Elements from one token to the next in `q` and `o`.
    pub strides: [i64; 2],
    /// Tokens that a token sees back from itself; 0: all.
    pub window: i64,
    /// First tokens that stay visible outside the window.
    pub sinks: i64,
    /// What scores are multiplied with.
    pub scale: f64,
    /// The type of `q` and `o`.
    pub activations: Activations,
}

impl Attention<'_> {
    fn desc(&self) -> strata_attention {
        let (n_seq, seq_len, seq_offsets) = self.sequences.parts();
        strata_attention {
            n_seq,
            seq_len,
            seq_offsets,
            n_head: self.n_head,
            q_stride: self.strides[0],
            o_stride: self.strides[1],
            window: self.window,
            sinks: self.sinks,
            scale: self.scale,
            dtype: self.activations.id(),
        }
    }

    /// Bytes of device workspace that [`CudaBackend::attention`] needs (0: none).
    pub fn work_bytes(&self, cache: &KvCache) -> Result<u64> {
        let (desc, cache) = (self.desc(), cache.desc());
        let mut bytes = 0;
        let rc = unsafe { strata_cuda_attention_work_bytes(&desc, &cache, &mut bytes) };
        if rc == ffi::STRATA_OK {
            Ok(bytes)
        } else {
            Err(Error::Backend {
                message: format!("attention: bad shape (status {rc})"),
            })
        }
    }
}

/// The device buffers of a scoring call.
#[derive(Debug, Clone, Copy)]
pub struct LogprobBuffers {
    /// Rows of logits.
    pub logits: *const f32,
    /// The token of each row that is scored, or null.
    pub targets: *const i32,
    /// Their log-probabilities, or null.
    pub logprobs: *mut f32,
    /// The rows' entropies, or null.
    pub entropy: *mut f32,
    /// The likeliest tokens, null where there are none to give.
    pub top_ids: *mut i32,
    /// Their log-probabilities, null where there are none to give.
    pub top_logprobs: *mut f32,
}

impl CudaBackend {
    /// Appends the call's keys and values to `cache`, turned by their positions, and turns its queries.
    ///
    /// # Safety
    /// The pointers are device memory of the sizes that the header gives for
    /// `shape` and `cache`, and stay so until the work on `stream` is done.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn kv_append(
        &self,
        shape: &KvAppend<'_>,
        cache: &KvCache,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        q_out: *mut c_void,
        stream: *mut c_void,
    ) -> Result<()> {
        let (n_seq, seq_len, seq_offsets) = shape.sequences.parts();
        let desc = strata_kv_append {
            n_seq,
            seq_len,
            seq_offsets,
            n_head: shape.n_head,
            n_rot: shape.n_rot,
            q_stride: shape.strides[0],
            k_stride: shape.strides[1],
            v_stride: shape.strides[2],
            q_out_stride: shape.strides[3],
            freq_base: shape.freq_base,
            dtype: shape.activations.id(),
            q_dtype: shape.queries.id(),
            neighbours: i32::from(shape.neighbours),
        };
        let cache = cache.desc();
        let rc = unsafe { strata_cuda_kv_append_dev(self.ctx, &desc, &cache, q, k, v, q_out, stream) };
        self.check(rc, QuantType::F32)
    }

    /// Attention of the call's queries over `cache`.
    ///
    /// # Safety
    /// As for [`CudaBackend::kv_append`]; calls that may overlap need a workspace each.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn attention(
        &self,
        shape: &Attention<'_>,
        cache: &KvCache,
        q: *const c_void,
        o: *mut c_void,
        work: *mut c_void,
        work_bytes: u64,
        stream: *mut c_void,
    ) -> Result<()> {
        let (desc, cache) = (shape.desc(), cache.desc());
        let rc = unsafe { strata_cuda_attention_dev(self.ctx, &desc, &cache, q, o, work, work_bytes, stream) };
        self.check(rc, QuantType::F32)
    }

    /// Log-probabilities of given tokens, entropies and the `top` likeliest tokens of
    /// `rows` rows of `vocab` logits, `stride` floats apart (0: packed).
    ///
    /// # Safety
    /// As for [`CudaBackend::kv_append`].
    pub unsafe fn logprobs(
        &self,
        rows: i64,
        vocab: i64,
        stride: i64,
        top: i64,
        b: &LogprobBuffers,
        stream: *mut c_void,
    ) -> Result<()> {
        let rc = unsafe {
            strata_cuda_logprobs_dev(
                self.ctx,
                b.logits,
                rows,
                vocab,
                stride,
                b.targets,
                b.logprobs,
                b.entropy,
                top,
                b.top_ids,
                b.top_logprobs,
                stream,
            )
        };
        self.check(rc, QuantType::F32)
    }
}
