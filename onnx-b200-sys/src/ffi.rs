// Generated by gen_ffi.py from include/onnxb200.h -- do not edit by hand.
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_int, c_void};

pub const ONNXB200_OK: c_int = 0;
pub const ONNXB200_ERR_VALIDATION: c_int = 1;
pub const ONNXB200_ERR_EXECUTION: c_int = 2;
pub const ONNXB200_ERR_UNSUPPORTED: c_int = 3;
pub const ONNXB200_ERR_TIMEOUT: c_int = 4;
pub const ONNXB200_ERR_RESOURCE_EXHAUSTED: c_int = 5;
pub const ONNXB200_ERR_INVALID_GRAPH: c_int = 6;
pub const ONNXB200_ERR_INVALID_OPERATOR: c_int = 7;
pub const ONNXB200_ERR_CANCELLED: c_int = 8;
pub const ONNXB200_ERR_INVALID_ARGUMENT: c_int = 9;
pub const ONNXB200_ERR_IO: c_int = 10;
pub const ONNXB200_ERR_PROTOBUF: c_int = 11;
pub const ONNXB200_ERR_INVALID_MODEL: c_int = 12;
pub const ONNXB200_PREC_DEFAULT: c_int = -1;
pub const ONNXB200_PREC_3XTF32: c_int = 0;
pub const ONNXB200_PREC_TF32: c_int = 1;
pub const ONNXB200_PREC_BF16: c_int = 2;
pub const ONNXB200_PREC_FP32: c_int = 3;
pub const ONNXB200_LAYOUT_NCHW: c_int = 0;
pub const ONNXB200_LAYOUT_NHWC: c_int = 1;
pub const ONNXB200_AUTOPAD_NOTSET: c_int = 0;
pub const ONNXB200_AUTOPAD_SAME_UPPER: c_int = 1;
pub const ONNXB200_AUTOPAD_SAME_LOWER: c_int = 2;
pub const ONNXB200_AUTOPAD_VALID: c_int = 3;
pub const ONNXB200_EPI_BIAS: c_int = 1;
pub const ONNXB200_EPI_BN: c_int = 2;
pub const ONNXB200_EPI_RESIDUAL: c_int = 4;
pub const ONNXB200_EPI_RELU: c_int = 8;
pub const ONNXB200_COPY_H2D: c_int = 0;
pub const ONNXB200_COPY_D2H: c_int = 1;
pub const ONNXB200_COPY_D2D: c_int = 2;
pub const ONNXB200_NOALLOC_SCRATCH_BYTES: usize = 25165824;
pub const ONNXB200_TYPE_F32: c_int = 0;
pub const ONNXB200_TYPE_F16: c_int = 1;
pub const ONNXB200_TYPE_BF16: c_int = 2;
pub const ONNXB200_TYPE_E4M3: c_int = 3;
pub const ONNXB200_RMSNORM_MAX_COLS: c_int = 49152;
pub const ONNXB200_ATTR_INT: c_int = 0;
pub const ONNXB200_ATTR_FLOAT: c_int = 1;
pub const ONNXB200_ATTR_INTS: c_int = 2;
pub const ONNXB200_ATTR_STRING: c_int = 3;
pub const ONNXB200_STEP_CONV_TC: c_int = 1;
pub const ONNXB200_STEP_CONV_DIRECT: c_int = 2;
pub const ONNXB200_STEP_GEMM: c_int = 3;
pub const ONNXB200_STEP_MAXPOOL: c_int = 4;
pub const ONNXB200_STEP_GAP: c_int = 5;
pub const ONNXB200_STEP_ADD: c_int = 6;
pub const ONNXB200_STEP_RELU: c_int = 7;
pub const ONNXB200_STEP_AFFINE: c_int = 8;
pub const ONNXB200_STEP_CONVERT: c_int = 9;

#[repr(C)]
pub struct Handle {
    _private: [u8; 0],
}

#[repr(C)]
pub struct ConvPlan {
    _private: [u8; 0],
}

#[repr(C)]
pub struct Graph {
    _private: [u8; 0],
}

#[repr(C)]
pub struct Multi {
    _private: [u8; 0],
}

#[repr(C)]
pub struct Model {
    _private: [u8; 0],
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct Options {
    pub precision: c_int,
    pub workspace_bytes: usize,
    pub use_cuda_graph: c_int,
    pub wait_timeout_ms: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ConvDesc {
    pub n: i64,
    pub c: i64,
    pub h: i64,
    pub w: i64,
    pub c_out: i64,
    pub kh: i64,
    pub kw: i64,
    pub stride_h: i64,
    pub stride_w: i64,
    pub pad_top: i64,
    pub pad_left: i64,
    pub pad_bottom: i64,
    pub pad_right: i64,
    pub dil_h: i64,
    pub dil_w: i64,
    pub group: i64,
    pub auto_pad: c_int,
    pub layout: c_int,
    pub epilogue: c_int,
    pub precision: c_int,
    pub bn_epsilon: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ConvNdDesc {
    pub spatial: c_int,
    pub n: i64,
    pub c: i64,
    pub c_out: i64,
    pub group: i64,
    pub in_: [i64; 3],
    pub kernel: [i64; 3],
    pub stride: [i64; 3],
    pub pad_begin: [i64; 3],
    pub pad_end: [i64; 3],
    pub dilation: [i64; 3],
    pub auto_pad: c_int,
    pub relu: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct RmsnormDesc {
    pub rows: i64,
    pub cols: i64,
    pub ldx: i64,
    pub ldr: i64,
    pub lds: i64,
    pub ldy: i64,
    pub y_scale_row: i64,
    pub y_scale_block: i64,
    pub type_: c_int,
    pub weight_type: c_int,
    pub out_type: c_int,
    pub epsilon: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct QuantizeDesc {
    pub rows: i64,
    pub cols: i64,
    pub ldx: i64,
    pub ldq: i64,
    pub scale_row: i64,
    pub scale_block: i64,
    pub type_: c_int,
    pub block_rows: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct MatmulBlocksDesc {
    pub m: i64,
    pub n: i64,
    pub k: i64,
    pub lda: i64,
    pub ldb: i64,
    pub ldy: i64,
    pub a_scale_row: i64,
    pub a_scale_block: i64,
    pub b_scale_row: i64,
    pub b_scale_block: i64,
    pub out_type: c_int,
    pub flags: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct Attr {
    pub name: *const c_char,
    pub type_: c_int,
    pub i: i64,
    pub f: f32,
    pub ints: *const i64,
    pub n_ints: c_int,
    pub s: *const c_char,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct Node {
    pub op_type: *const c_char,
    pub inputs: *const *const c_char,
    pub n_inputs: c_int,
    pub outputs: *const *const c_char,
    pub n_outputs: c_int,
    pub attrs: *const Attr,
    pub n_attrs: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct TensorInfo {
    pub name: *const c_char,
    pub data: *const f32,
    pub shape: *const i64,
    pub rank: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct GraphStats {
    pub n_nodes_in: c_int,
    pub n_steps: c_int,
    pub n_fused: c_int,
    pub kernels_per_run: i64,
    pub arena_bytes: i64,
    pub weight_bytes: i64,
    pub captured: c_int,
    pub bf16_tensors: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShapeInfo {
    pub name: *const c_char,
    pub dims: [i64; 8],
    pub rank: c_int,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct StepProfile {
    pub kind: c_int,
    pub ms: f32,
    pub flops: f64,
    pub bytes: f64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct ModelInfo {
    pub ir_version: i64,
    pub opset: i64,
    pub n_nodes: c_int,
    pub n_initializers: c_int,
    pub n_skipped_initializers: c_int,
    pub n_skipped_attributes: c_int,
    pub n_inputs: c_int,
    pub n_outputs: c_int,
    pub producer_name: *const c_char,
    pub graph_name: *const c_char,
}

#[link(name = "onnxb200")]
extern "C" {
    pub fn onnxb200_version() -> c_int;
    pub fn onnxb200_default_options(opts: *mut Options);
    pub fn onnxb200_create(device: c_int, opts: *const Options, out: *mut *mut Handle) -> c_int;
    pub fn onnxb200_destroy(h: *mut Handle) -> c_int;
    pub fn onnxb200_last_error(h: *const Handle) -> *const c_char;
    pub fn onnxb200_status_string(status: c_int) -> *const c_char;
    pub fn onnxb200_set_stream(h: *mut Handle, cuda_stream: *mut c_void) -> c_int;
    pub fn onnxb200_get_stream(h: *mut Handle) -> *mut c_void;
    pub fn onnxb200_synchronize(h: *mut Handle) -> c_int;
    pub fn onnxb200_kernel_launches(h: *const Handle) -> i64;
    pub fn onnxb200_num_sms(h: *const Handle) -> c_int;
    pub fn onnxb200_malloc(h: *mut Handle, bytes: usize, ptr: *mut *mut c_void) -> c_int;
    pub fn onnxb200_free(h: *mut Handle, ptr: *mut c_void) -> c_int;
    pub fn onnxb200_memcpy(h: *mut Handle, dst: *mut c_void, src: *const c_void, bytes: usize, kind: c_int) -> c_int;
    pub fn onnxb200_conv2d_output_shape(d: *const ConvDesc, out: *mut i64) -> c_int;
    pub fn onnxb200_conv_nd_output_shape(d: *const ConvNdDesc, out: *mut i64, rank: *mut c_int) -> c_int;
    pub fn onnxb200_conv_nd(h: *mut Handle, d: *const ConvNdDesc, x: *const f32, w: *const f32, bias: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_conv2d(h: *mut Handle, d: *const ConvDesc, x: *const f32, w: *const f32, bias: *const f32, bn_scale: *const f32, bn_bias: *const f32, bn_mean: *const f32, bn_var: *const f32, residual: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_conv_plan_create(h: *mut Handle, d: *const ConvDesc, w: *const f32, bias: *const f32, bn_scale: *const f32, bn_bias: *const f32, bn_mean: *const f32, bn_var: *const f32, out: *mut *mut ConvPlan) -> c_int;
    pub fn onnxb200_conv_plan_run(h: *mut Handle, p: *const ConvPlan, x: *const f32, residual: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_conv_plan_destroy(p: *mut ConvPlan) -> c_int;
    pub fn onnxb200_conv2d_nhwc_noalloc(cuda_stream: *mut c_void, d: *const ConvDesc, x: *const f32, w: *const f32, bias: *const f32, bn_scale: *const f32, bn_bias: *const f32, bn_mean: *const f32, bn_var: *const f32, residual: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_matmul_output_shape(a_shape: *const i64, a_rank: c_int, b_shape: *const i64, b_rank: c_int, out_shape: *mut i64, out_rank: *mut c_int) -> c_int;
    pub fn onnxb200_matmul(h: *mut Handle, a: *const f32, a_shape: *const i64, a_rank: c_int, b: *const f32, b_shape: *const i64, b_rank: c_int, bias: *const f32, flags: c_int, precision: c_int, y: *mut f32) -> c_int;
    pub fn onnxb200_gemm(h: *mut Handle, a: *const f32, b: *const f32, c: *const f32, c_shape: *const i64, c_rank: c_int, m: i64, n: i64, k: i64, trans_a: c_int, trans_b: c_int, alpha: f32, beta: f32, flags: c_int, precision: c_int, y: *mut f32) -> c_int;
    pub fn onnxb200_maxpool2d(h: *mut Handle, layout: c_int, n: i64, c: i64, hh: i64, ww: i64, kh: i64, kw: i64, stride_h: i64, stride_w: i64, pad_top: i64, pad_left: i64, pad_bottom: i64, pad_right: i64, ceil_mode: c_int, x: *const f32, y: *mut f32, indices: *mut i64, out: *mut i64) -> c_int;
    pub fn onnxb200_global_avgpool(h: *mut Handle, layout: c_int, n: i64, c: i64, hh: i64, ww: i64, x: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_add(h: *mut Handle, a: *const f32, a_shape: *const i64, a_rank: c_int, b: *const f32, b_shape: *const i64, b_rank: c_int, relu: c_int, y: *mut f32) -> c_int;
    pub fn onnxb200_relu(h: *mut Handle, x: *const f32, count: i64, y: *mut f32) -> c_int;
    pub fn onnxb200_batchnorm(h: *mut Handle, layout: c_int, n: i64, c: i64, hh: i64, ww: i64, x: *const f32, scale: *const f32, bias: *const f32, mean: *const f32, var: *const f32, epsilon: f32, y: *mut f32) -> c_int;
    pub fn onnxb200_nchw_to_nhwc(h: *mut Handle, n: i64, c: i64, hh: i64, ww: i64, c_pad: i64, x: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_nhwc_to_nchw(h: *mut Handle, n: i64, c: i64, hh: i64, ww: i64, x: *const f32, y: *mut f32) -> c_int;
    pub fn onnxb200_rmsnorm(h: *mut Handle, d: *const RmsnormDesc, x: *const c_void, residual: *const c_void, weight: *const c_void, sum: *mut c_void, y: *mut c_void, y_scale: *mut f32) -> c_int;
    pub fn onnxb200_quantize_blocks(h: *mut Handle, d: *const QuantizeDesc, x: *const c_void, q: *mut c_void, scale: *mut f32) -> c_int;
    pub fn onnxb200_matmul_blocks(h: *mut Handle, d: *const MatmulBlocksDesc, a: *const c_void, a_scale: *const f32, b: *const c_void, b_scale: *const f32, bias: *const f32, y: *mut c_void) -> c_int;
    pub fn onnxb200_graph_build(h: *mut Handle, nodes: *const Node, n_nodes: c_int, initializers: *const TensorInfo, n_init: c_int, inputs: *const TensorInfo, n_inputs: c_int, outputs: *const *const c_char, n_outputs: c_int, out: *mut *mut Graph) -> c_int;
    pub fn onnxb200_graph_run(h: *mut Handle, g: *mut Graph, inputs: *const *const f32, outputs: *const *mut f32) -> c_int;
    pub fn onnxb200_graph_run_host(h: *mut Handle, g: *mut Graph, inputs: *const *const f32, outputs: *const *mut f32) -> c_int;
    pub fn onnxb200_graph_run_host_pipelined(h: *mut Handle, g: *mut Graph, n_batches: c_int, inputs: *const *const f32, outputs: *const *mut f32) -> c_int;
    pub fn onnxb200_graph_output_shape(g: *const Graph, index: c_int, shape: *mut i64, rank: *mut c_int) -> c_int;
    pub fn onnxb200_infer_shapes(nodes: *const Node, n_nodes: c_int, known: *const TensorInfo, n_known: c_int, shapes: *mut ShapeInfo, max_shapes: c_int, n_shapes: *mut c_int, err: *mut c_char, err_len: usize) -> c_int;
    pub fn onnxb200_graph_profile(h: *mut Handle, g: *mut Graph, inputs: *const *const f32, outputs: *const *mut f32, steps: *mut StepProfile, max_steps: c_int, n_steps: *mut c_int) -> c_int;
    pub fn onnxb200_graph_get_stats(g: *const Graph, st: *mut GraphStats) -> c_int;
    pub fn onnxb200_graph_destroy(g: *mut Graph) -> c_int;
    pub fn onnxb200_multi_build(devices: *const c_int, n_devices: c_int, opts: *const Options, nodes: *const Node, n_nodes: c_int, initializers: *const TensorInfo, n_init: c_int, inputs: *const TensorInfo, n_inputs: c_int, outputs: *const *const c_char, n_outputs: c_int, out: *mut *mut Multi, err: *mut c_char, err_len: usize) -> c_int;
    pub fn onnxb200_multi_run_host(m: *mut Multi, n_batches: c_int, inputs: *const *const f32, outputs: *const *mut f32) -> c_int;
    pub fn onnxb200_multi_get_info(m: *const Multi, n_devices: *mut c_int, batch: *mut i64, slice_begin: *mut i64, last_run_ms: *mut f32) -> c_int;
    pub fn onnxb200_multi_output_shape(m: *const Multi, index: c_int, shape: *mut i64, rank: *mut c_int) -> c_int;
    pub fn onnxb200_multi_last_error(m: *const Multi) -> *const c_char;
    pub fn onnxb200_multi_destroy(m: *mut Multi) -> c_int;
    pub fn onnxb200_model_parse(data: *const c_void, len: usize, base_dir: *const c_char, out: *mut *mut Model, err: *mut c_char, err_len: usize) -> c_int;
    pub fn onnxb200_model_load(path: *const c_char, out: *mut *mut Model, err: *mut c_char, err_len: usize) -> c_int;
    pub fn onnxb200_model_get_info(m: *const Model, info: *mut ModelInfo) -> c_int;
    pub fn onnxb200_model_get_nodes(m: *const Model, nodes: *mut *const Node, n: *mut c_int) -> c_int;
    pub fn onnxb200_model_get_initializers(m: *const Model, t: *mut *const TensorInfo, n: *mut c_int) -> c_int;
    pub fn onnxb200_model_get_inputs(m: *const Model, t: *mut *const TensorInfo, n: *mut c_int) -> c_int;
    pub fn onnxb200_model_get_outputs(m: *const Model, names: *mut *const *const c_char, n: *mut c_int) -> c_int;
    pub fn onnxb200_model_destroy(m: *mut Model) -> c_int;
    pub fn onnxb200_graph_build_from_model(h: *mut Handle, m: *const Model, input_shapes: *const TensorInfo, n_input_shapes: c_int, out: *mut *mut Graph) -> c_int;
}
