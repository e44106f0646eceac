//! The batched GPU sampler for C and Python callers that embed llm-rs
//! without its scheduler, in llm-ffi's style (lib.rs: opaque handles,
//! `#[no_mangle] extern "C"`, null / 0 sentinels for failure).  Built with
//! the `hip-sampler` feature.

use std::ffi::c_void;
use llm_kernel::hip_sampler::{pages_work_words, HipSampler, LlmkLogprobsArgs, LlmkPageCache,
                               LlmkProcessLogitsArgs, LlmkSampleBatchArgs,
                               LLMK_ERR_INVALID_ARGUMENT};

/// A sampler on `device` for batches up to `max_batch` rows of up to
/// `max_vocab` logits; null on failure.
#[no_mangle]
pub extern "C" fn llm_sampler_create(device: i32, max_batch: u32, max_vocab: u32) -> *mut c_void {
    match HipSampler::new(device, max_batch, max_vocab) {
        Ok(s) => Box::into_raw(Box::new(s)) as *mut c_void,
        Err(_) => std::ptr::null_mut(),
    }
}

/// One batched sampling step on `stream`: 0 on success, else the library's
/// error code.
/// # SAFETY: `sampler` from llm_sampler_create; `args` valid, its device
/// pointers alive until the stream reaches the call.
#[no_mangle]
pub unsafe extern "C" fn llm_sample_batch(sampler: *mut c_void, args: *const LlmkSampleBatchArgs,
                                          stream: *mut c_void) -> i32 {
    if sampler.is_null() || args.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    let s = &*(sampler as *const HipSampler);
    match s.sample_batch(&*args, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// Speculative-decoding verification of one draft token per row (see
/// `HipSampler::verify_batch`): 0 on success, else the error code.
/// # SAFETY: as llm_sample_batch; every array is device memory.
#[no_mangle]
pub unsafe extern "C" fn llm_verify_batch(sampler: *mut c_void, batch: u32, vocab: u32,
                                          ids: *const u32, probs: *const f32, list_cap: u32,
                                          counts: *const u32, draft_tokens: *const u32,
                                          draft_probs: *const f32, draft_stride: u64,
                                          u_accept: *const f32, u_resample: *const f32,
                                          out_tokens: *mut u32, out_accepted: *mut u32,
                                          stream: *mut c_void) -> i32 {
    if sampler.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    let s = &*(sampler as *const HipSampler);
    match s.verify_batch(batch, vocab, ids, probs, list_cap, counts, draft_tokens, draft_probs,
                         draft_stride, u_accept, u_resample, out_tokens, out_accepted, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// Processed logits (see `HipSampler::process_logits`): 0 on success, else the
/// error code.
/// # SAFETY: as llm_sample_batch.
#[no_mangle]
pub unsafe extern "C" fn llm_process_logits(sampler: *mut c_void, args: *const LlmkProcessLogitsArgs,
                                            stream: *mut c_void) -> i32 {
    if sampler.is_null() || args.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    match (*(sampler as *const HipSampler)).process_logits(&*args, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// Log-probabilities (see `HipSampler::logprobs`): 0 on success, else the
/// error code.
/// # SAFETY: as llm_sample_batch.
#[no_mangle]
pub unsafe extern "C" fn llm_logprobs(sampler: *mut c_void, args: *const LlmkLogprobsArgs,
                                      stream: *mut c_void) -> i32 {
    if sampler.is_null() || args.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    match (*(sampler as *const HipSampler)).logprobs(&*args, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// The words of a page cache's work array; 0 where the sizes are refused.
#[no_mangle]
pub extern "C" fn llm_pages_work_words(rows: u32, num_pages: u32) -> u64 {
    pages_work_words(rows, num_pages).unwrap_or(0)
}

/// One step of a paged cache's rows (see `HipSampler::pages_update`): 0 on
/// success, else the error code.
/// # SAFETY: as llm_sample_batch; the cache's arrays are device memory.
#[no_mangle]
pub unsafe extern "C" fn llm_pages_update(sampler: *mut c_void, cache: *const LlmkPageCache,
                                          parents: *const i32, new_lengths: *const i32,
                                          out_granted: *mut u32, stream: *mut c_void) -> i32 {
    if sampler.is_null() || cache.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    let s = &*(sampler as *const HipSampler);
    match s.pages_update(&*cache, parents, new_lengths, out_granted, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// Moves a cache's pages in use to the front (see `HipSampler::pages_compact`):
/// 0 on success, else the error code.
/// # SAFETY: as llm_pages_update; `out_map` has `num_pages` entries.
#[no_mangle]
pub unsafe extern "C" fn llm_pages_compact(sampler: *mut c_void, cache: *const LlmkPageCache,
                                           out_map: *mut u32, stream: *mut c_void) -> i32 {
    if sampler.is_null() || cache.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    match (*(sampler as *const HipSampler)).pages_compact(&*cache, out_map, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// Copies page `src[i]` to page `dst[i]` in every pool (see
/// `HipSampler::pages_copy`): 0 on success, else the error code.
/// # SAFETY: as llm_sample_batch; every array is device memory.
#[no_mangle]
pub unsafe extern "C" fn llm_pages_copy(sampler: *mut c_void, n_pools: u32, pools: *const u64,
                                        page_bytes: u64, num_pages: u32, n: u32, src: *const u32,
                                        dst: *const u32, stream: *mut c_void) -> i32 {
    if sampler.is_null() {
        return LLMK_ERR_INVALID_ARGUMENT;
    }
    let s = &*(sampler as *const HipSampler);
    match s.pages_copy(n_pools, pools, page_bytes, num_pages, n, src, dst, stream) {
        Ok(()) => 0,
        Err(e) => e.code,
    }
}

/// Reads and clears the status bits raised since the last read; 0 also
/// when the handle is null or the read fails.
/// # SAFETY: `sampler` from llm_sampler_create or null.
#[no_mangle]
pub unsafe extern "C" fn llm_sampler_status(sampler: *mut c_void, stream: *mut c_void) -> u32 {
    if sampler.is_null() {
        return 0;
    }
    let s = &*(sampler as *const HipSampler);
    s.status(stream).unwrap_or(0)
}

/// Frees a sampler from llm_sampler_create (null: nothing).
/// # SAFETY: `sampler` from llm_sampler_create, not used afterwards.
#[no_mangle]
pub unsafe extern "C" fn llm_sampler_destroy(sampler: *mut c_void) {
    if !sampler.is_null() {
        drop(Box::from_raw(sampler as *mut HipSampler));
    }
}
