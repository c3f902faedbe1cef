//! `#[repr(C)]` mirrors of `include/deltacore_layers.h`: the operators around the token mixers of a block stack.
//!
//! Not compiled here, as the crate's root; `tests/test_layers_abi.py` checks the structs, constants and functions against the
//! header and the library.
use super::dc_stream_t;
use std::ffi::{c_int, c_void};

pub const DC_E4M3: i32 = 2;
pub const DC_RMS_MAX_WIDTH: i64 = 16384;
pub const DC_CONV_MAX_TAPS: i64 = 8;
pub const DC_SCAN_MAX_STATE: i64 = 64;
pub const DC_CONV_SILU: u32 = 0x1;
pub const DC_SCAN_SOFTPLUS: u32 = 0x1;

/// The residual stream's addition and the RMS norm of the sum.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct dc_rms_norm_args {
    pub rows: i64,
    pub width: i64,
    pub x_stride: i64,
    pub residual_in_stride: i64,
    pub residual_out_stride: i64,
    pub y_stride: i64,
    pub x_dtype: i32,
    pub residual_dtype: i32,
    pub out_dtype: i32,
    pub group: i32,
    pub eps: f32,
    pub x: *const c_void,
    pub residual_in: *const c_void,
    pub weight: *const f32,
    pub residual_out: *mut c_void,
    pub y: *mut c_void,
    pub scale: *mut f32,
}

/// Its backward.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct dc_rms_norm_bwd_args {
    pub rows: i64,
    pub width: i64,
    pub d_y_stride: i64,
    pub d_r_stride: i64,
    pub r_stride: i64,
    pub d_x_stride: i64,
    pub d_residual_stride: i64,
    pub y_dtype: i32,
    pub r_dtype: i32,
    pub x_dtype: i32,
    pub eps: f32,
    pub d_y: *const c_void,
    pub d_r: *const c_void,
    pub r: *const c_void,
    pub weight: *const f32,
    pub d_x: *mut c_void,
    pub d_residual: *mut c_void,
    pub d_weight: *mut f32,
    pub workspace: *mut c_void,
    pub workspace_bytes: u64,
}

/// The causal depthwise convolution, over a prompt or (`seq = 1`) one token.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct dc_causal_conv_args {
    pub batch: i64,
    pub seq: i64,
    pub channels: i64,
    pub x_batch_stride: i64,
    pub x_token_stride: i64,
    pub y_batch_stride: i64,
    pub y_token_stride: i64,
    pub taps: i32,
    pub in_dtype: i32,
    pub out_dtype: i32,
    pub flags: u32,
    pub x: *const c_void,
    pub weight: *const f32,
    pub bias: *const f32,
    pub window_in: *const f32,
    pub lengths: *const i32,
    pub y: *mut c_void,
    pub window_out: *mut f32,
}

/// Its backward.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct dc_causal_conv_bwd_args {
    pub batch: i64,
    pub seq: i64,
    pub channels: i64,
    pub x_batch_stride: i64,
    pub x_token_stride: i64,
    pub d_y_batch_stride: i64,
    pub d_y_token_stride: i64,
    pub d_x_batch_stride: i64,
    pub d_x_token_stride: i64,
    pub taps: i32,
    pub in_dtype: i32,
    pub out_dtype: i32,
    pub flags: u32,
    pub d_y: *const c_void,
    pub d_window_out: *const f32,
    pub x: *const c_void,
    pub weight: *const f32,
    pub bias: *const f32,
    pub window_in: *const f32,
    pub lengths: *const i32,
    pub d_x: *mut c_void,
    pub d_weight: *mut f32,
    pub d_bias: *mut f32,
    pub d_window_in: *mut f32,
    pub workspace: *mut c_void,
    pub workspace_bytes: u64,
}

/// The selective state space scan, over a prompt or one token.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct dc_selective_scan_args {
    pub batch: i64,
    pub seq: i64,
    pub channels: i64,
    pub state: i64,
    pub groups: i64,
    pub u_batch_stride: i64,
    pub u_token_stride: i64,
    pub dt_batch_stride: i64,
    pub dt_token_stride: i64,
    pub z_batch_stride: i64,
    pub z_token_stride: i64,
    pub b_batch_stride: i64,
    pub b_token_stride: i64,
    pub c_batch_stride: i64,
    pub c_token_stride: i64,
    pub y_batch_stride: i64,
    pub y_token_stride: i64,
    pub in_dtype: i32,
    pub out_dtype: i32,
    pub flags: u32,
    pub u: *const c_void,
    pub dt: *const c_void,
    pub a: *const f32,
    pub b: *const c_void,
    pub c: *const c_void,
    pub d: *const f32,
    pub z: *const c_void,
    pub dt_bias: *const f32,
    pub state_in: *const f32,
    pub lengths: *const i32,
    pub y: *mut c_void,
    pub state_out: *mut f32,
    pub checkpoints: *mut f32,
    pub workspace: *mut c_void,
    pub workspace_bytes: u64,
}

/// Its backward.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct dc_selective_scan_bwd_args {
    pub fwd: dc_selective_scan_args,
    pub d_y_batch_stride: i64,
    pub d_y_token_stride: i64,
    pub d_y: *const c_void,
    pub d_state_out: *const f32,
    pub d_u: *mut c_void,
    pub d_dt: *mut c_void,
    pub d_a: *mut f32,
    pub d_b: *mut c_void,
    pub d_c: *mut c_void,
    pub d_d: *mut f32,
    pub d_z: *mut c_void,
    pub d_dt_bias: *mut f32,
    pub d_state_in: *mut f32,
    pub workspace: *mut c_void,
    pub workspace_bytes: u64,
}

#[link(name = "deltacore")]
extern "C" {
    pub fn dc_rms_norm(args: *const dc_rms_norm_args, stream: dc_stream_t) -> c_int;
    pub fn dc_rms_norm_bwd_workspace_size(args: *const dc_rms_norm_bwd_args) -> u64;
    pub fn dc_rms_norm_bwd(args: *const dc_rms_norm_bwd_args, stream: dc_stream_t) -> c_int;
    pub fn dc_causal_conv(args: *const dc_causal_conv_args, stream: dc_stream_t) -> c_int;
    pub fn dc_causal_conv_bwd_workspace_size(args: *const dc_causal_conv_bwd_args) -> u64;
    pub fn dc_causal_conv_bwd(args: *const dc_causal_conv_bwd_args, stream: dc_stream_t) -> c_int;
    pub fn dc_selective_scan_checkpoint_size(args: *const dc_selective_scan_args) -> u64;
    pub fn dc_selective_scan_workspace_size(args: *const dc_selective_scan_args) -> u64;
    pub fn dc_selective_scan(args: *const dc_selective_scan_args, stream: dc_stream_t) -> c_int;
    pub fn dc_selective_scan_step(args: *const dc_selective_scan_args, stream: dc_stream_t) -> c_int;
    pub fn dc_selective_scan_bwd_workspace_size(args: *const dc_selective_scan_bwd_args) -> u64;
    pub fn dc_selective_scan_bwd(args: *const dc_selective_scan_bwd_args, stream: dc_stream_t) -> c_int;
}
