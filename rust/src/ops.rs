//! The decode step's operators: draws from given uniforms and the 8-bit language-model head, over
//! the C ABI of include/llamars_sampler.h (every pointer a device pointer, every call enqueued on
//! `stream`, a cudaStream_t of the current device, without host synchronisation).
//!
//! Not compiled in this repository's build image (it has no Rust toolchain); the ABI declared
//! here is checked by tests/csrc/rust_ops_abi.c in the CPU test suite.
use std::os::raw::{c_int, c_void};

use crate::ffi;
use crate::sampler::{check, SamplerError};

/// Element types of logits, activations and weights.
#[repr(i32)]
#[derive(Clone, Copy, Debug, PartialEq, Eq)]
pub enum Dtype {
    F32 = 0,
    Bf16 = 1,
    F16 = 2,
}

/// One row's filters: top_k 0, top_p 1 and min_p 0 are off, temperature <= 0 is greedy.
#[repr(C)]
#[derive(Clone, Copy, Debug, PartialEq)]
#[allow(non_camel_case_types)]
pub struct lrs_draw_params {
    pub temperature: f32,
    pub top_k: u32,
    pub top_p: f32,
    pub min_p: f32,
}

extern "C" {
    pub fn lrs_draw_device(
        d_logits: *const c_void,
        dtype: c_int,
        rows: u32,
        n: u32,
        ld: u64,
        d_params: *const lrs_draw_params,
        d_uniform: *const f32,
        d_tokens: *mut u32,
        d_probs: *mut f32,
        d_kept: *mut u32,
        d_status: *mut i32,
        stream: *mut c_void,
    ) -> c_int;
    pub fn lrs_quantize_rows(
        d_x: *const c_void,
        dtype: c_int,
        rows: u32,
        k: u32,
        ld_x: u64,
        d_q: *mut u8,
        ld_q: u64,
        d_scale: *mut f32,
        ld_scale: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn lrs_quantize_blocks(
        d_x: *const c_void,
        dtype: c_int,
        rows: u32,
        k: u32,
        ld_x: u64,
        d_q: *mut u8,
        ld_q: u64,
        d_scale: *mut f32,
        ld_scale: u64,
        stream: *mut c_void,
    ) -> c_int;
    pub fn lrs_fp8_logits(
        d_a: *const u8,
        ld_a: u64,
        d_a_scale: *const f32,
        ld_as: u64,
        d_w: *const u8,
        ld_w: u64,
        d_w_scale: *const f32,
        ld_ws: u64,
        rows: u32,
        n: u32,
        k: u32,
        d_out: *mut c_void,
        out_dtype: c_int,
        ld_out: u64,
        stream: *mut c_void,
    ) -> c_int;
}

/// A token a row from given uniforms (lrs_draw_device).
///
/// # Safety
/// Device pointers valid for `rows` rows on the current device; `d_probs`, `d_kept` and
/// `d_status` may be null.
#[allow(clippy::too_many_arguments)]
pub unsafe fn draw_device(
    d_logits: *const c_void,
    dtype: Dtype,
    rows: u32,
    n: u32,
    ld: u64,
    d_params: *const lrs_draw_params,
    d_uniform: *const f32,
    d_tokens: *mut u32,
    d_probs: *mut f32,
    d_kept: *mut u32,
    d_status: *mut i32,
    stream: *mut c_void,
) -> Result<(), SamplerError> {
    check(
        lrs_draw_device(d_logits, dtype as c_int, rows, n, ld, d_params, d_uniform, d_tokens, d_probs, d_kept, d_status,
                        stream),
        std::ptr::null::<ffi::lrs_ctx>(),
    )
}

/// A matrix in device memory: row r starts at `data + r * ld` elements.
#[derive(Clone, Copy, Debug)]
pub struct Matrix {
    pub data: *mut c_void,
    pub rows: u32,
    pub cols: u32,
    pub ld: u64,
}

/// e4m3 codes of `x`'s rows in blocks of 128 columns, or (`tall`) of 128 x 128 blocks, with their
/// scales (lrs_quantize_rows, lrs_quantize_blocks).
///
/// # Safety
/// Device pointers of the sizes the C header gives, on the current device.
pub unsafe fn quantize(x: Matrix, dtype: Dtype, tall: bool, d_q: *mut u8, ld_q: u64, d_scale: *mut f32, ld_scale: u64,
                       stream: *mut c_void) -> Result<(), SamplerError> {
    let f = if tall { lrs_quantize_blocks } else { lrs_quantize_rows };
    check(
        f(x.data, dtype as c_int, x.rows, x.cols, x.ld, d_q, ld_q, d_scale, ld_scale, stream),
        std::ptr::null::<ffi::lrs_ctx>(),
    )
}

/// The head's product of codes, out.rows x out.cols (lrs_fp8_logits); matrices whose sizes do not agree are
/// refused (LRS_E_INVALID).
///
/// # Safety
/// Device pointers of the sizes the C header gives, on the current device.
pub unsafe fn fp8_logits(a: Matrix, d_a_scale: *const f32, ld_as: u64, w: Matrix, d_w_scale: *const f32, ld_ws: u64,
                         out: Matrix, out_dtype: Dtype, stream: *mut c_void) -> Result<(), SamplerError> {
    if w.cols != a.cols || out.rows != a.rows || out.cols != w.rows {
        return Err(SamplerError {
            code: ffi::LRS_E_INVALID,
            message: format!("fp8_logits: {} x {} times {} x {} into {} x {}", a.rows, a.cols, w.rows, w.cols, out.rows, out.cols),
        });
    }
    check(
        lrs_fp8_logits(a.data as *const u8, a.ld, d_a_scale, ld_as, w.data as *const u8, w.ld, d_w_scale, ld_ws, a.rows,
                       w.rows, a.cols, out.data, out_dtype as c_int, out.ld, stream),
        std::ptr::null::<ffi::lrs_ctx>(),
    )
}
