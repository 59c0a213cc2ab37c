"""Host-side mirror of the reference's operator interface on top of the C ABI.

``Operator`` follows ``trait Operator`` (src/ops/registry.rs:14-27): ``compute``
takes input tensors and returns freshly allocated outputs (the reference replaces
``outputs[i]`` wholesale, src/ops/nn/conv.rs:199-200), ``output_shapes`` infers
shapes from a node, ``validate`` checks a node.  Tensors are NCHW fp32 torch CUDA
tensors.  Unlike the reference's ``compute`` (which ignores node attributes,
src/ops/nn/conv.rs:180-199, src/ops/math/gemm.rs:35-38), operators built with
``from_node`` carry the node's attributes.

``OperatorRegistry`` keeps the reference's (name, domain, version) keys
(src/ops/registry.rs:30-98); ``create_operator_for_node`` resolves the newest
registered version not above the requested opset (the reference compares
character codes instead, src/ops/registry.rs:105-106, and never matches).
"""
from __future__ import annotations

import ctypes
import importlib
import math
import os
import threading
import warnings
from typing import Dict, List, NamedTuple, Optional, Sequence

import torch

from . import _capi as C
from .runtime import (Handle, InvalidOperator, UnsupportedFeature, ValidationError, dptr)


def _load_calls():
    """The native module for repeated calls (make -C csrc calls), or None: ctypes does without it."""
    if not os.path.exists(os.path.join(os.path.dirname(os.path.abspath(__file__)), "_calls.so")):
        return None
    try:
        module = importlib.import_module("._calls", __package__)
        built_for = getattr(module, "torch_version", "of an unknown version")
        if built_for != torch.__version__:
            raise ImportError(f"built for torch {built_for}, not {torch.__version__}")
        return module
    except ImportError as e:
        warnings.warn(f"onnx-rs_b200/_calls.so is not used ({e}); calls go through ctypes", RuntimeWarning, stacklevel=2)
        return None


def _native():
    """ops._calls, loaded where it is asked for first: importing the package does not need it."""
    if "_calls" not in globals():
        globals()["_calls"] = _load_calls()
    return _calls


def __getattr__(name):
    if name == "_calls":
        return _native()
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


class ExecutionContext:
    """Operator-level context (src/ops/registry.rs:8-11) plus the device handle."""

    def __init__(self, handle: Handle, options: Optional[Dict[str, str]] = None):
        self.handle = handle
        self.options = dict(options or {})


def _attrs(node) -> dict:
    return dict(node.get("attrs", {})) if isinstance(node, dict) else dict(getattr(node, "attrs", {}))


def _prec(ctx: ExecutionContext, prec) -> int:
    if prec is None:
        p = ctx.options.get("precision")
        return C.PRECISIONS[p] if p else C.PREC_DEFAULT
    return C.PRECISIONS[prec] if isinstance(prec, str) else int(prec)


class Operator:
    op_type = ""

    def compute(self, inputs: Sequence[Optional[torch.Tensor]], ctx: ExecutionContext) -> List[torch.Tensor]:
        raise NotImplementedError

    def input_shapes(self, node, input_shapes):
        return list(input_shapes)

    def output_shapes(self, node, input_shapes) -> List[Optional[List[int]]]:
        raise NotImplementedError

    def validate(self, node) -> None:
        n_in = len(node["inputs"]) if isinstance(node, dict) else len(node.inputs)
        if n_in < self.min_inputs:
            raise ValidationError(C.ERR_VALIDATION,
                                  f"{self.op_type} operator requires at least {self.min_inputs} inputs, got {n_in}")

    min_inputs = 1


# --------------------------------------------------------------------------- Conv
class Conv(Operator):
    """Conv (src/ops/nn/conv.rs:115-323): 2-D with an optional fused epilogue
    (BatchNormalization, residual Add, Relu) on the tensor-core path; 1-D (NCL,
    run as 2-D of height 1) and 3-D (NCDHW, CUDA cores) with bias and Relu.
    strides / pads / dilations default per rank (ONNX: ones, zeros, ones)."""
    op_type = "Conv"
    min_inputs = 2

    def __init__(self, strides=None, pads=None, dilations=None, group=1, auto_pad="NOTSET",
                 precision=None, relu=False):
        self.strides = None if strides is None else list(strides)
        self.pads = None if pads is None else list(pads)
        self.dilations = None if dilations is None else list(dilations)
        self.group = int(group)
        self.auto_pad = auto_pad
        self.precision = precision
        self.relu = relu

    @classmethod
    def from_node(cls, node, **kw):
        a = _attrs(node)
        return cls(a.get("strides"), a.get("pads"), a.get("dilations"), a.get("group", 1),
                   a.get("auto_pad", "NOTSET"), **kw)

    def _attr(self, sp):
        """strides, pads (begin..., end...), dilations for `sp` spatial dims."""
        st = self.strides if self.strides is not None else [1] * sp
        pd = self.pads if self.pads is not None else [0] * (2 * sp)
        dl = self.dilations if self.dilations is not None else [1] * sp
        if len(st) != sp or len(pd) != 2 * sp or len(dl) != sp:
            raise ValidationError(C.ERR_VALIDATION, f"Conv: attributes do not match {sp} spatial dims")
        return st, pd, dl

    def nd_desc(self, x_shape, w_shape):
        """onnxb200_conv_nd_desc for a 1-D, 2-D or 3-D input."""
        sp = len(x_shape) - 2
        if sp < 1 or sp > 3 or len(w_shape) != len(x_shape):
            raise ValidationError(C.ERR_VALIDATION, "Conv supports only 1D, 2D, and 3D convolutions")
        st, pd, dl = self._attr(sp)
        d = C.ConvNdDesc()
        d.spatial = sp
        d.n, d.c = x_shape[0], x_shape[1]
        d.c_out = w_shape[0]
        d.group = self.group
        for i in range(sp):
            d.in_[i] = x_shape[2 + i]
            d.kernel[i] = w_shape[2 + i]
            d.stride[i] = st[i]
            d.pad_begin[i] = pd[i]
            d.pad_end[i] = pd[sp + i]
            d.dilation[i] = dl[i]
        d.auto_pad = C.AUTOPAD[self.auto_pad]
        d.relu = 1 if self.relu else 0
        return d

    def desc(self, x_shape, w_shape, layout=C.LAYOUT_NCHW, epilogue=0, prec=C.PREC_DEFAULT, eps=1e-5):
        d = C.ConvDesc()
        if layout == C.LAYOUT_NHWC:
            d.n, d.h, d.w, d.c = x_shape
        else:
            d.n, d.c, d.h, d.w = x_shape
        d.c_out, _, d.kh, d.kw = w_shape
        st, pd, dl = self._attr(2)
        d.stride_h, d.stride_w = st
        d.pad_top, d.pad_left, d.pad_bottom, d.pad_right = pd
        d.dil_h, d.dil_w = dl
        d.group = self.group
        d.auto_pad = C.AUTOPAD[self.auto_pad]
        d.layout = layout
        d.epilogue = epilogue
        d.precision = prec
        d.bn_epsilon = eps
        return d

    def output_shape(self, x_shape, w_shape) -> List[int]:
        if len(x_shape) != 4:
            d = self.nd_desc(x_shape, w_shape)
            out = C.i64_array([0] * 5)
            rank = ctypes.c_int()
            rc = C.lib().onnxb200_conv_nd_output_shape(ctypes.byref(d), out, ctypes.byref(rank))
            if rc != 0:
                raise ValidationError(rc, "Conv: invalid shapes or attributes")
            return [int(v) for v in out[:rank.value]]
        d = self.desc(x_shape, w_shape)
        out = C.i64_array([0] * 4)
        rc = C.lib().onnxb200_conv2d_output_shape(ctypes.byref(d), out)
        if rc != 0:
            raise ValidationError(rc, "Conv: invalid shapes or attributes")
        return [int(v) for v in out[:4]]

    def output_shapes(self, node, input_shapes):
        if len(input_shapes) < 2:
            raise ValidationError(C.ERR_VALIDATION, f"Conv requires at least 2 inputs, got {len(input_shapes)}")
        x, w = input_shapes[0], input_shapes[1]
        if x is None or w is None:
            return [None]
        return [type(self).from_node(node).output_shape(x, w)]

    def compute(self, inputs, ctx, bn=None, residual=None, layout=C.LAYOUT_NCHW):
        """inputs = [X, W, B?]; bn = (scale, B, mean, var, eps) fuses BatchNormalization."""
        x, w = inputs[0], inputs[1]
        b = inputs[2] if len(inputs) > 2 else None
        h = ctx.handle
        if x.dim() != 4:  # 1-D / 3-D: bias and Relu only
            if bn is not None or residual is not None or layout != C.LAYOUT_NCHW:
                raise UnsupportedFeature(C.ERR_UNSUPPORTED, "Conv: fused BN / residual / NHWC are 2-D only")
            y = torch.empty(self.output_shape(tuple(x.shape), tuple(w.shape)), dtype=torch.float32,
                            device=x.device)
            d = self.nd_desc(tuple(x.shape), tuple(w.shape))
            h.check(C.lib().onnxb200_conv_nd(h.ptr, ctypes.byref(d), dptr(x), dptr(w), dptr(b), dptr(y)), "Conv")
            return [y]
        epi = (C.EPI_BIAS if b is not None else 0) | (C.EPI_BN if bn is not None else 0) | \
              (C.EPI_RESIDUAL if residual is not None else 0) | (C.EPI_RELU if self.relu else 0)
        eps = bn[4] if bn is not None else 1e-5
        d = self.desc(tuple(x.shape), tuple(w.shape), layout, epi, _prec(ctx, self.precision), eps)
        out = C.i64_array([0] * 4)
        h.check(C.lib().onnxb200_conv2d_output_shape(ctypes.byref(d), out), "Conv")
        n, co, oh, ow = [int(v) for v in out[:4]]
        shape = (n, co, oh, ow) if layout == C.LAYOUT_NCHW else (n, oh, ow, co)
        y = torch.empty(shape, dtype=torch.float32, device=x.device)
        bnp = list(bn[:4]) if bn is not None else [None] * 4
        h.check(C.lib().onnxb200_conv2d(h.ptr, ctypes.byref(d), dptr(x), dptr(w), dptr(b), dptr(bnp[0]),
                                        dptr(bnp[1]), dptr(bnp[2]), dptr(bnp[3]), dptr(residual), dptr(y)), "Conv")
        return [y]


class ConvPlan:
    """Prepared convolution (onnxb200_conv_plan_*): weights packed and BN folded once.

    ``layout`` is the layout of x / residual / y at run time (NHWC runs the
    kernel directly on the caller's buffers)."""

    def __init__(self, ctx: ExecutionContext, conv: Conv, x_shape, w, bias=None, bn=None,
                 layout=C.LAYOUT_NHWC, residual=False):
        self.ctx = ctx
        h = ctx.handle
        epi = (C.EPI_BIAS if bias is not None else 0) | (C.EPI_BN if bn is not None else 0) | \
              (C.EPI_RESIDUAL if residual else 0) | (C.EPI_RELU if conv.relu else 0)
        self.desc = conv.desc(tuple(x_shape), tuple(w.shape), layout, epi, _prec(ctx, conv.precision),
                              bn[4] if bn is not None else 1e-5)
        out = C.i64_array([0] * 4)
        h.check(C.lib().onnxb200_conv2d_output_shape(ctypes.byref(self.desc), out), "Conv")
        n, co, oh, ow = [int(v) for v in out[:4]]
        self.out_shape = (n, co, oh, ow) if layout == C.LAYOUT_NCHW else (n, oh, ow, co)
        bnp = list(bn[:4]) if bn is not None else [None] * 4
        ptr = ctypes.c_void_p()
        h.check(C.lib().onnxb200_conv_plan_create(h.ptr, ctypes.byref(self.desc), dptr(w), dptr(bias),
                                                  dptr(bnp[0]), dptr(bnp[1]), dptr(bnp[2]), dptr(bnp[3]),
                                                  ctypes.byref(ptr)), "conv plan")
        self.ptr = ptr

    def run(self, x: torch.Tensor, y: torch.Tensor, residual: Optional[torch.Tensor] = None):
        h = self.ctx.handle
        h.check(C.lib().onnxb200_conv_plan_run(h.ptr, self.ptr, dptr(x), dptr(residual), dptr(y)), "conv plan run")
        return y

    def close(self):
        if getattr(self, "ptr", None):
            C.lib().onnxb200_conv_plan_destroy(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# --------------------------------------------------------------------------- MatMul / Gemm
class MatMul(Operator):
    """MatMul (src/ops/math/matmul.rs:60-124): numpy-broadcast batched matmul."""
    op_type = "MatMul"
    min_inputs = 2

    def __init__(self, precision=None):
        self.precision = precision

    @classmethod
    def from_node(cls, node, **kw):
        return cls(**kw)

    @staticmethod
    def output_shape(a_shape, b_shape) -> List[int]:
        out = C.i64_array([0] * 10)
        r = ctypes.c_int()
        rc = C.lib().onnxb200_matmul_output_shape(C.i64_array(a_shape), len(a_shape), C.i64_array(b_shape),
                                                  len(b_shape), out, ctypes.byref(r))
        if rc != 0:
            raise ValidationError(rc, f"Incompatible shapes for MatMul: {list(a_shape)} and {list(b_shape)}")
        return [int(v) for v in out[:r.value]]

    def output_shapes(self, node, input_shapes):
        a, b = input_shapes[0], input_shapes[1]
        return [None if a is None or b is None else self.output_shape(a, b)]

    def compute(self, inputs, ctx, bias=None, relu=False):
        a, b = inputs[0], inputs[1]
        shape = self.output_shape(tuple(a.shape), tuple(b.shape))
        y = torch.empty(shape, dtype=torch.float32, device=a.device)
        h = ctx.handle
        h.check(C.lib().onnxb200_matmul(h.ptr, dptr(a), C.i64_array(a.shape), a.dim(), dptr(b),
                                        C.i64_array(b.shape), b.dim(), dptr(bias), C.EPI_RELU if relu else 0,
                                        _prec(ctx, self.precision), dptr(y)), "MatMul")
        return [y]


class Gemm(Operator):
    """Gemm (src/ops/math/gemm.rs:17-44) with alpha, beta, transA, transB honoured."""
    op_type = "Gemm"
    min_inputs = 2

    def __init__(self, alpha=1.0, beta=1.0, trans_a=0, trans_b=0, precision=None, relu=False):
        self.alpha, self.beta = float(alpha), float(beta)
        self.trans_a, self.trans_b = int(trans_a), int(trans_b)
        self.precision = precision
        self.relu = relu

    @classmethod
    def from_node(cls, node, **kw):
        a = _attrs(node)
        return cls(a.get("alpha", 1.0), a.get("beta", 1.0), a.get("transA", 0), a.get("transB", 0), **kw)

    def output_shapes(self, node, input_shapes):
        a, b = input_shapes[0], input_shapes[1]
        if a is None or b is None:
            return [None]
        g = type(self).from_node(node)
        m = a[1] if g.trans_a else a[0]
        n = b[0] if g.trans_b else b[1]
        return [[m, n]]

    def compute(self, inputs, ctx):
        a, b = inputs[0], inputs[1]
        c = inputs[2] if len(inputs) > 2 else None
        if a.dim() != 2 or b.dim() != 2:
            raise ValidationError(C.ERR_VALIDATION, "Gemm inputs must be 2D matrices")
        m, k = (a.shape[1], a.shape[0]) if self.trans_a else (a.shape[0], a.shape[1])
        k2, n = (b.shape[1], b.shape[0]) if self.trans_b else (b.shape[0], b.shape[1])
        if k != k2:
            raise ValidationError(C.ERR_VALIDATION, f"Incompatible dimensions for Gemm: {k} and {k2}")
        y = torch.empty((m, n), dtype=torch.float32, device=a.device)
        h = ctx.handle
        cs = C.i64_array(c.shape if c is not None else [1])
        h.check(C.lib().onnxb200_gemm(h.ptr, dptr(a), dptr(b), dptr(c), cs, 0 if c is None else c.dim(), m, n, k,
                                      self.trans_a, self.trans_b, self.alpha, self.beta,
                                      C.EPI_RELU if self.relu else 0, _prec(ctx, self.precision), dptr(y)), "Gemm")
        return [y]


# --------------------------------------------------------------------------- pooling
class MaxPool(Operator):
    """MaxPool (src/ops/nn/pool.rs:168-193) with the node's attributes (the
    reference hard-codes 2x2/2, pool.rs:185-187)."""
    op_type = "MaxPool"

    def __init__(self, kernel_shape=(2, 2), strides=(2, 2), pads=(0, 0, 0, 0), ceil_mode=0):
        self.kernel_shape, self.strides, self.pads = list(kernel_shape), list(strides), list(pads)
        self.ceil_mode = int(ceil_mode)

    @classmethod
    def from_node(cls, node, **kw):
        a = _attrs(node)
        return cls(a.get("kernel_shape", (2, 2)), a.get("strides", (1, 1)), a.get("pads", (0, 0, 0, 0)),
                   a.get("ceil_mode", 0))

    def out_hw(self, h, w):
        kh, kw = self.kernel_shape
        sh, sw = self.strides
        pt, pl, pb, pr = self.pads
        if self.ceil_mode:
            return (h + pt + pb - kh + sh - 1) // sh + 1, (w + pl + pr - kw + sw - 1) // sw + 1
        return (h + pt + pb - kh) // sh + 1, (w + pl + pr - kw) // sw + 1

    def output_shapes(self, node, input_shapes):
        x = input_shapes[0]
        if x is None:
            return [None]
        oh, ow = type(self).from_node(node).out_hw(x[2], x[3])
        return [[x[0], x[1], oh, ow]]

    def compute(self, inputs, ctx, with_indices=False, layout=C.LAYOUT_NCHW):
        x = inputs[0]
        if layout == C.LAYOUT_NHWC:
            n, hh, ww, c = x.shape
        else:
            n, c, hh, ww = x.shape
        oh, ow = self.out_hw(hh, ww)
        shape = (n, c, oh, ow) if layout == C.LAYOUT_NCHW else (n, oh, ow, c)
        y = torch.empty(shape, dtype=torch.float32, device=x.device)
        ind = torch.empty((n, c, oh, ow), dtype=torch.int64, device=x.device) if with_indices else None
        h = ctx.handle
        out = C.i64_array([0] * 4)
        h.check(C.lib().onnxb200_maxpool2d(h.ptr, layout, n, c, hh, ww, *self.kernel_shape, *self.strides,
                                           *self.pads, self.ceil_mode, dptr(x), dptr(y),
                                           None if ind is None else ctypes.c_void_p(ind.data_ptr()), out),
                "MaxPool")
        return [y, ind] if with_indices else [y]


class GlobalAveragePool(Operator):
    """GlobalAveragePool (src/ops/nn/pool.rs:275-295 -> global_pool :493-557)."""
    op_type = "GlobalAveragePool"

    @classmethod
    def from_node(cls, node, **kw):
        return cls()

    def output_shapes(self, node, input_shapes):
        x = input_shapes[0]
        return [None if x is None else [x[0], x[1]] + [1] * (len(x) - 2)]

    def compute(self, inputs, ctx, layout=C.LAYOUT_NCHW):
        x = inputs[0]
        if layout == C.LAYOUT_NHWC:
            n, hh, ww, c = x.shape
        else:
            n, c, hh, ww = x.shape
        y = torch.empty((n, c, 1, 1), dtype=torch.float32, device=x.device)
        h = ctx.handle
        h.check(C.lib().onnxb200_global_avgpool(h.ptr, layout, n, c, hh, ww, dptr(x), dptr(y)), "GlobalAveragePool")
        return [y]


# --------------------------------------------------------------------------- elementwise
class Relu(Operator):
    """Relu (src/ops/activations.rs:92-96, relu :244-246)."""
    op_type = "Relu"

    @classmethod
    def from_node(cls, node, **kw):
        return cls()

    def output_shapes(self, node, input_shapes):
        return [input_shapes[0]]

    def compute(self, inputs, ctx):
        x = inputs[0]
        y = torch.empty_like(x)
        ctx.handle.check(C.lib().onnxb200_relu(ctx.handle.ptr, dptr(x), x.numel(), dptr(y)), "Relu")
        return [y]


class Add(Operator):
    """Add = element_wise_binary_op(+) with broadcasting (src/ops/tensor.rs:1124-1218)."""
    op_type = "Add"
    min_inputs = 2

    def __init__(self, relu=False):
        self.relu = relu

    @classmethod
    def from_node(cls, node, **kw):
        return cls(**kw)

    @staticmethod
    def broadcast(a, b):
        r = max(len(a), len(b))
        a = [1] * (r - len(a)) + list(a)
        b = [1] * (r - len(b)) + list(b)
        out = []
        for i, (x, y) in enumerate(zip(a, b)):
            if x != y and x != 1 and y != 1:
                raise ValidationError(C.ERR_VALIDATION,
                                      f"Cannot broadcast shapes {a} and {b}: incompatible dimensions at index {i}")
            out.append(y if x == 1 else x)
        return out

    def output_shapes(self, node, input_shapes):
        a, b = input_shapes[0], input_shapes[1]
        return [None if a is None or b is None else self.broadcast(a, b)]

    def compute(self, inputs, ctx):
        a, b = inputs[0], inputs[1]
        y = torch.empty(self.broadcast(a.shape, b.shape), dtype=torch.float32, device=a.device)
        h = ctx.handle
        h.check(C.lib().onnxb200_add(h.ptr, dptr(a), C.i64_array(a.shape), a.dim(), dptr(b), C.i64_array(b.shape),
                                     b.dim(), 1 if self.relu else 0, dptr(y)), "Add")
        return [y]


class BatchNormalization(Operator):
    """ONNX BatchNormalization (inference).  Not in the reference registry."""
    op_type = "BatchNormalization"
    min_inputs = 5

    def __init__(self, epsilon=1e-5):
        self.epsilon = float(epsilon)

    @classmethod
    def from_node(cls, node, **kw):
        return cls(_attrs(node).get("epsilon", 1e-5))

    def output_shapes(self, node, input_shapes):
        return [input_shapes[0]]

    def compute(self, inputs, ctx, layout=C.LAYOUT_NCHW):
        x, scale, bias, mean, var = inputs[:5]
        if layout == C.LAYOUT_NHWC:
            n, hh, ww, c = x.shape
        else:
            n, c, hh, ww = x.shape
        y = torch.empty_like(x)
        h = ctx.handle
        h.check(C.lib().onnxb200_batchnorm(h.ptr, layout, n, c, hh, ww, dptr(x), dptr(scale), dptr(bias),
                                           dptr(mean), dptr(var), self.epsilon, dptr(y)), "BatchNormalization")
        return [y]


class Flatten(Operator):
    """ONNX Flatten (a view; the reference only infers its shape, src/memory/planner.rs:1735)."""
    op_type = "Flatten"

    def __init__(self, axis=1):
        self.axis = int(axis)

    @classmethod
    def from_node(cls, node, **kw):
        return cls(_attrs(node).get("axis", 1))

    def output_shapes(self, node, input_shapes):
        x = input_shapes[0]
        if x is None:
            return [None]
        ax = type(self).from_node(node).axis
        ax = ax + len(x) if ax < 0 else ax
        a = 1
        for v in x[:ax]:
            a *= v
        b = 1
        for v in x[ax:]:
            b *= v
        return [[a, b]]

    def compute(self, inputs, ctx):
        x = inputs[0]
        return [x.reshape(self.output_shapes({"attrs": {"axis": self.axis}}, [list(x.shape)])[0])]


# --------------------------------------------------------------------------- 8-bit linear path
_TYPE = {torch.float32: C.TYPE_F32, torch.float16: C.TYPE_F16, torch.bfloat16: C.TYPE_BF16}
_E4M3 = torch.float8_e4m3fn
_ONNX_TYPE = {1: torch.float32, 10: torch.float16, 16: torch.bfloat16}  # TensorProto.DataType
_QBLOCK = 128


def _type(t, what):
    code = _TYPE.get(t.dtype)
    if code is None:
        raise ValidationError(C.ERR_VALIDATION, f"{what}: expected float32, float16 or bfloat16, got {t.dtype}")
    return code


def _check_device(h, what, *tensors):
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device.index != h.device):
            raise ValidationError(C.ERR_VALIDATION, f"{what}: expected tensors on cuda:{h.device}, got {t.device}")


def _row_stride(t, what):
    """Row stride of a tensor read as the matrix [product of leading dims, last dim]."""
    if t.dim() == 0:
        raise ValidationError(C.ERR_VALIDATION, f"{what}: expected at least one dimension")
    cols = t.shape[-1]
    if t.numel() == 0 or t.is_contiguous():
        return cols
    stride = t.stride()
    if cols > 1 and stride[-1] != 1:
        raise ValidationError(C.ERR_VALIDATION, f"{what}: expected rows of consecutive elements")
    ld = step = None
    for size, st in zip(reversed(t.shape[:-1]), reversed(stride[:-1])):
        if size == 1:
            continue
        if ld is None:
            ld, step = st, st * size
        elif st != step:
            raise ValidationError(C.ERR_VALIDATION, f"{what}: the leading dimensions do not have one stride")
        else:
            step = st * size
    if ld is None:
        return cols
    if ld < cols:
        raise ValidationError(C.ERR_VALIDATION, f"{what}: the rows overlap")
    return ld


def _stored_stride(cols):
    """Row stride of e4m3 rows that start on 16-byte boundaries (what the tensor-core product reads)."""
    return (cols + 15) // 16 * 16


def _dense(shape, dtype):
    """(shape, strides, dtype) of a new contiguous tensor."""
    strides, step = [], 1
    for n in reversed(shape):
        strides.append(step)
        step *= max(1, n)
    return tuple(shape), tuple(reversed(strides)), dtype


def _stored_rows(lead, cols):
    """(shape, strides, dtype) of new e4m3 rows [*lead, cols], _stored_stride(cols) apart."""
    _, strides, _ = _dense((*lead, _stored_stride(cols)), _E4M3)
    return (*lead, cols), strides, _E4M3


def _stored_scales(lead, rows, blocks):
    """(shape, strides, dtype) of new scales [*lead, blocks]; those of one block of columns lie side by
    side, as the product reads them."""
    _, strides, _ = _dense(lead, torch.float32)
    return (*lead, blocks), (*strides, max(1, rows)), torch.float32


def _new_on(dev):
    """f(shape, strides, dtype): a new uninitialised tensor on a device."""
    return lambda shape, strides, dtype: torch.empty_strided(shape, strides, dtype=dtype, device=dev)


def _scale_strides(s, rows, blocks, what):
    """(tensor, row stride, block stride) of scales read as the matrix [rows, blocks]."""
    if s.dtype != torch.float32:
        raise ValidationError(C.ERR_VALIDATION, f"{what}: expected float32 scales, got {s.dtype}")
    if s.dim() == 0 or s.shape[-1] != blocks or s.numel() != rows * blocks:
        raise ValidationError(C.ERR_VALIDATION, f"{what}: expected {rows} x {blocks} scales, got {tuple(s.shape)}")
    if s.dim() != 2:
        s = s.reshape(rows, blocks)
    sr, sb = s.stride()
    if sr == 0 and sb == 0:  # one value for all: two zeros stand for dense rows at the C entry
        s = s.contiguous()
        sr, sb = s.stride()
    return s, sr, sb


def _launch(h, what, entry, desc, *args):
    """Calls a C entry in order with torch's current stream, whatever stream the handle runs on."""
    cur = torch._C._cuda_getCurrentRawStream(h.device)
    run = h.stream_ptr
    # the handle's own stream is a blocking one: ordered with the legacy default stream by itself
    if cur == run or (cur == 0 and run == h.own_stream_ptr):
        rc = entry(h.ptr, desc, *args)
    else:
        cur = torch.cuda.current_stream(h.device)
        side = torch.cuda.ExternalStream(run, device=h.device)
        side.wait_stream(cur)
        rc = entry(h.ptr, desc, *args)
        cur.wait_stream(side)
    if rc != 0:
        h.check(rc, what)


def _address(fn):
    return ctypes.cast(fn, ctypes.c_void_p).value


def _ptr(t):
    return None if t is None else t.data_ptr()


def _layout(t):
    """What a call's checks and descriptor depend on: never where the elements are."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


class _Kept(NamedTuple):
    """What an operator keeps of a call: nothing of it depends on where the elements are."""
    desc: ctypes.Structure
    specs: tuple     # (shape, strides, dtype) of each output, None where there is none
    relaid: Sequence  # (input, function that lays it out anew) on every call
    plan: object     # of the native module, or None


# Held to publish what operators keep, never during a call's own work; a finaliser that the collector
# runs meanwhile may change an operator's settings.
_keeping = threading.RLock()


class _Described:
    """Operators whose checks, descriptors and output layouts are kept from call to call, by the
    operator's settings and the layout of the inputs.  Where the native module _calls is built, a call
    whose layouts were seen before is made there (csrc/torch_calls.cpp).  Threads may share an operator:
    _plans is replaced as a whole, together with what _kept holds, and what a call made under settings
    that have changed since is not kept."""
    entry = None   # name of the C entry
    slots = ()     # its pointers behind the descriptor: an input, or -1 - an output
    _plans = None

    def __setattr__(self, name, value):
        """A changed setting: what was kept does not hold any more."""
        with _keeping:
            object.__setattr__(self, name, value)
            self.__dict__.pop("_kept", None)
            self.__dict__.pop("_plans", None)

    def __getstate__(self):
        # pointers are neither copied nor pickled
        return {k: v for k, v in self.__dict__.items() if k not in ("_kept", "_plans")}

    def _call(self, h, *tensors):
        plans = self._plans
        if plans:
            out = _native().run(plans, h.address, h.device, h.own_stream_ptr, *tensors)
            if type(out) is list:
                return out
            if out is not None:
                h.check(out, self.op_type)
        desc, specs, relaid, _ = self._described(h, self._prepare, *tensors)
        for i, lay in relaid:
            tensors = (*tensors[:i], lay(tensors[i]), *tensors[i + 1:])
        new = _new_on(tensors[0].device)
        outs = [None if spec is None else new(*spec) for spec in specs]
        _launch(h, self.op_type, getattr(C.lib(), self.entry), ctypes.byref(desc),
                *(_ptr(tensors[s] if s >= 0 else outs[-1 - s]) for s in self.slots))
        return [t for t in outs if t is not None]

    def _described(self, handle, make, *tensors):
        kept = self.__dict__.setdefault("_kept", {})  # before the settings are read: a change takes it away
        key = (handle.device, self._settings(), *map(_layout, tensors))
        got = kept.get(key)
        if got is None:
            got = make(handle, *tensors)
            with _keeping:
                if self.__dict__.get("_kept") is kept:
                    if len(kept) >= 64:
                        del kept[next(iter(kept))]  # the oldest
                    kept[key] = got
                    plans = [p for p in (getattr(g, "plan", None) for g in kept.values()) if p is not None]
                    self.__dict__["_plans"] = plans[::-1]  # the newest comes first
        return got

    def _prepare(self, h, *tensors):
        """Checks a call and makes its plan for _calls.run."""
        desc, specs, relaid = self._describe(h, *tensors)
        if relaid or _native() is None:
            return _Kept(desc, specs, relaid, None)
        present = [i for i, spec in enumerate(specs) if spec is not None]
        slots = tuple((s if tensors[s] is not None else None) if s >= 0 else
                      (-1 - present.index(-1 - s) if specs[-1 - s] is not None else None) for s in self.slots)
        return _Kept(desc, specs, relaid, _native().Plan(
            _address(getattr(C.lib(), self.entry)), _address(C.lib().onnxb200_get_stream), ctypes.addressof(desc), desc,
            h.device, tensors, tuple(specs[i] for i in present), slots))


class RMSNormalization(_Described, Operator):
    """ONNX RMSNormalization (opset 23) over the last axis.  Not in the reference registry.

    compute([x, scale], ctx, residual=None) returns [y], or with ``quantize`` [q, q_scale]: e4m3
    values and one fp32 scale for every 128 columns of a row, the operand form of
    MatMulBlockScaled.  With a residual, h = x + residual is normalised and h (rounded to x's
    type) is returned as the last output.  Where x and scale differ in type, y has x's, or with
    ``y_like="scale"`` the scale's: so ONNX defines it, and so operators made from nodes do."""
    op_type = "RMSNormalization"
    min_inputs = 2
    entry = "onnxb200_rmsnorm"
    slots = (0, 2, 1, -3, -1, -2)  # x, residual, scale; h, y, y_scale

    def __init__(self, epsilon=1e-5, axis=-1, quantize=False, y_like="x"):
        self._check_y_like(y_like)
        self.epsilon = float(epsilon)
        self.axis = int(axis)
        self.quantize = bool(quantize)
        self.y_like = y_like

    @classmethod
    def from_node(cls, node, **kw):
        a = _attrs(node)
        if a.get("stash_type", 1) != 1:
            raise UnsupportedFeature(C.ERR_UNSUPPORTED,
                                     f"RMSNormalization: computes in float32 (stash_type 1), got stash_type {a['stash_type']}")
        kw.setdefault("y_like", "scale")
        return cls(a.get("epsilon", 1e-5), a.get("axis", -1), **kw)

    def _settings(self):
        return self.epsilon, self.axis, self.quantize, self.y_like

    @staticmethod
    def _check_y_like(y_like):
        if y_like not in ("x", "scale"):
            raise ValidationError(C.ERR_VALIDATION, f"RMSNormalization: y_like must be 'x' or 'scale', got {y_like!r}")

    def _check_axis(self, rank):
        if self.axis not in (-1, rank - 1):
            raise UnsupportedFeature(C.ERR_UNSUPPORTED, f"RMSNormalization: only the last axis, got {self.axis}")

    def output_shapes(self, node, input_shapes):
        x = input_shapes[0]
        if x is not None:
            type(self).from_node(node)._check_axis(len(x))
        return [x]

    def _describe(self, h, x, w, residual):
        what = "RMSNormalization"
        _check_device(h, what, x, w, residual)
        d = C.RmsNormDesc()
        d.type = _type(x, what)
        d.weight_type = _type(w, what)
        d.ldx = _row_stride(x, what)
        self._check_axis(x.dim())
        lead, cols = tuple(x.shape[:-1]), x.shape[-1]
        if w.dim() != 1 or w.shape[0] != cols or not w.is_contiguous():
            raise ValidationError(C.ERR_VALIDATION, f"{what}: expected a contiguous scale of {cols} elements")
        if residual is not None:
            if residual.shape != x.shape or residual.dtype != x.dtype:
                raise ValidationError(C.ERR_VALIDATION, f"{what}: the residual must have x's shape and type")
            d.ldr = _row_stride(residual, what)
        rows = math.prod(lead)
        d.rows, d.cols = rows, cols
        d.epsilon = self.epsilon
        self._check_y_like(self.y_like)
        y = x if self.y_like == "x" else w
        d.out_type = d.type if y is x else d.weight_type
        if self.quantize:
            d.out_type = C.TYPE_E4M3
            d.ldy = _stored_stride(cols)
            d.y_scale_row, d.y_scale_block = 1, max(1, rows)
        blocks = (cols + _QBLOCK - 1) // _QBLOCK
        return d, (_stored_rows(lead, cols) if self.quantize else _dense(x.shape, y.dtype),
                   _stored_scales(lead, rows, blocks) if self.quantize else None,
                   _dense(x.shape, x.dtype) if residual is not None else None), ()

    def compute(self, inputs, ctx, residual=None):
        return self._call(ctx.handle, inputs[0], inputs[1], residual)


class QuantizeBlocks(_Described, Operator):
    """e4m3 values and fp32 scales of a matrix: compute([x], ctx) returns [q, scale].  block_rows = 1
    gives one scale for every 128 columns of a row (activations, any leading dims), block_rows = 128
    one for 128 rows by 128 columns (weights, 2-D).  Not in the reference registry."""
    op_type = "QuantizeBlocks"
    entry = "onnxb200_quantize_blocks"
    slots = (0, -1, -2)

    def __init__(self, block_rows=1):
        if block_rows not in (1, _QBLOCK):
            raise ValidationError(C.ERR_VALIDATION, f"QuantizeBlocks: block_rows must be 1 or {_QBLOCK}, got {block_rows}")
        self.block_rows = int(block_rows)

    def _settings(self):
        return self.block_rows

    @classmethod
    def from_node(cls, node, **kw):
        return cls(_attrs(node).get("block_rows", 1), **kw)

    @staticmethod
    def _check_rank(block_rows, rank):
        if rank == 0 or (block_rows != 1 and rank != 2):
            raise ValidationError(C.ERR_VALIDATION, "QuantizeBlocks: " + ("weights must be 2-D" if rank else "expected at least one dimension"))

    def output_shapes(self, node, input_shapes):
        x = input_shapes[0]
        if x is None:
            return [None, None]
        br = type(self).from_node(node).block_rows
        self._check_rank(br, len(x))
        blocks = (x[-1] + _QBLOCK - 1) // _QBLOCK
        return [list(x), list(x[:-1]) + [blocks] if br == 1 else [(x[0] + _QBLOCK - 1) // _QBLOCK, blocks]]

    def _describe(self, h, x):
        what = "QuantizeBlocks"
        _check_device(h, what, x)
        d = C.QuantizeDesc()
        d.type = _type(x, what)
        d.ldx = _row_stride(x, what)
        self._check_rank(self.block_rows, x.dim())
        lead, cols = tuple(x.shape[:-1]), x.shape[-1]
        rows, blocks = math.prod(lead), (cols + _QBLOCK - 1) // _QBLOCK
        d.rows, d.cols, d.ldq = rows, cols, _stored_stride(cols)
        d.block_rows = self.block_rows
        if self.block_rows == 1:
            d.scale_row, d.scale_block = 1, max(1, rows)
        else:
            d.scale_row, d.scale_block = max(1, blocks), 1
        return d, (_stored_rows(lead, cols), _stored_scales(lead, rows, blocks) if self.block_rows == 1 else
                   _dense(((rows + _QBLOCK - 1) // _QBLOCK, blocks), torch.float32)), ()

    def compute(self, inputs, ctx):
        return self._call(ctx.handle, inputs[0])


class MatMulBlockScaled(_Described, Operator):
    """y = A . B^T of e4m3 operands with a scale for every block of 128: compute([a, a_scale, b,
    b_scale, bias?], ctx) returns [y].  a is [..., k] with a_scale [..., ceil(k / 128)], b is
    [n, k] with b_scale [ceil(n / 128), ceil(k / 128)] (QuantizeBlocks(128)), bias fp32 [n]; y is
    [..., n] in ``dtype``, after Relu if asked.  Not in the reference registry."""
    op_type = "MatMulBlockScaled"
    min_inputs = 4
    entry = "onnxb200_matmul_blocks"
    slots = (0, 1, 2, 3, 4, -1)

    def __init__(self, dtype=torch.float32, relu=False):
        self._check_dtype(dtype)
        self.dtype = dtype
        self.relu = bool(relu)

    @staticmethod
    def _check_dtype(dtype):
        if dtype not in _TYPE:
            raise ValidationError(C.ERR_VALIDATION,
                                  f"MatMulBlockScaled: expected float32, float16 or bfloat16, got {dtype}")

    def _settings(self):
        return self.dtype, self.relu

    @classmethod
    def from_node(cls, node, **kw):
        a = _attrs(node)
        kw.setdefault("dtype", _ONNX_TYPE.get(a.get("dtype", 1)))
        kw.setdefault("relu", a.get("relu", 0))
        return cls(**kw)

    def output_shapes(self, node, input_shapes):
        a, b = input_shapes[0], input_shapes[2]
        return [None if a is None or b is None else list(a[:-1]) + [b[0]]]

    def _describe(self, h, a, a_scale, b, b_scale, bias):
        what = "MatMulBlockScaled"
        _check_device(h, what, a, a_scale, b, b_scale, bias)
        if a.dtype != _E4M3 or b.dtype != _E4M3:
            raise ValidationError(C.ERR_VALIDATION, f"{what}: expected float8_e4m3fn operands, got {a.dtype} and {b.dtype}")
        d = C.MatmulBlocksDesc()
        d.lda = _row_stride(a, what)
        d.ldb = _row_stride(b, what)
        if b.dim() != 2 or a.shape[-1] != b.shape[1]:
            raise ValidationError(C.ERR_VALIDATION, f"Incompatible shapes for {what}: {list(a.shape)} and {list(b.shape)}")
        n, k = b.shape
        m = math.prod(a.shape[:-1])
        blocks, rows_b = (k + _QBLOCK - 1) // _QBLOCK, (n + _QBLOCK - 1) // _QBLOCK
        if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()):
            raise ValidationError(C.ERR_VALIDATION, f"{what}: expected a contiguous float32 bias of {n} elements")
        d.m, d.n, d.k = m, n, k
        # scales that are not addressable by two strides are laid out anew on every call
        strides, relaid = [], []
        for i, s, rows in ((1, a_scale, m), (3, b_scale, rows_b)):
            t, sr, sb = _scale_strides(s, rows, blocks, what)
            strides += [sr, sb]
            if t.data_ptr() != s.data_ptr():
                relaid.append((i, lambda s, rows=rows: _scale_strides(s, rows, blocks, what)[0]))
        d.a_scale_row, d.a_scale_block, d.b_scale_row, d.b_scale_block = strides
        self._check_dtype(self.dtype)
        d.out_type = _TYPE[self.dtype]
        d.flags = C.EPI_RELU if self.relu else 0
        return d, (_dense((*a.shape[:-1], n), self.dtype),), relaid

    def compute(self, inputs, ctx):
        a, a_scale, b, b_scale = inputs[:4]
        bias = inputs[4] if len(inputs) > 4 else None
        return self._call(ctx.handle, a, a_scale, b, b_scale, bias)


# --------------------------------------------------------------------------- registry
class OperatorRegistry:
    """(name, domain, version)-keyed registry (src/ops/registry.rs:30-128)."""

    def __init__(self):
        self.operators: Dict[tuple, type] = {}

    def register_operator(self, name: str, domain: str, version: int, op_cls) -> None:
        key = (name, domain, int(version))
        if key in self.operators:
            raise InvalidOperator(C.ERR_INVALID_OPERATOR,
                                  f"Operator {domain}.{name} (version {version}) is already registered")
        self.operators[key] = op_cls

    def get_operator(self, name: str, domain: str, version: int):
        return self.operators.get((name, domain, int(version)))

    @classmethod
    def initialize_standard_operators(cls) -> "OperatorRegistry":
        r = cls()
        # versions as registered by the reference (src/ops/registry.rs:74-95); BN, Add
        # and Flatten are additions for this path.
        for name, ver, op in (("MatMul", 9, MatMul), ("Gemm", 9, Gemm), ("Conv", 11, Conv),
                              ("MaxPool", 11, MaxPool), ("GlobalAveragePool", 1, GlobalAveragePool),
                              ("Relu", 6, Relu), ("Add", 7, Add), ("BatchNormalization", 9, BatchNormalization),
                              ("Flatten", 9, Flatten)):
            r.register_operator(name, "", ver, op)
        # the 8-bit linear path: RMSNormalization is ONNX's (opset 23), the others have no ONNX form
        r.register_operator("RMSNormalization", "", 23, RMSNormalization)
        r.register_operator("QuantizeBlocks", "b200", 1, QuantizeBlocks)
        r.register_operator("MatMulBlockScaled", "b200", 1, MatMulBlockScaled)
        return r

    def create_operator_for_node(self, node, opset: int = 17, **kw) -> Operator:
        name = node["op"] if isinstance(node, dict) else node.op_type
        domain = (node.get("domain", "") if isinstance(node, dict) else getattr(node, "domain", "")) or ""
        best = None
        for (n, d, v), op in self.operators.items():
            if n == name and d == domain and v <= opset and (best is None or v > best[0]):
                best = (v, op)
        if best is None:
            raise InvalidOperator(C.ERR_INVALID_OPERATOR,
                                  f"Operator {domain}.{name} (opset {opset}) not found in registry")
        return best[1].from_node(node, **kw)
