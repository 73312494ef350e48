"""euler-b200: B200 (sm_100a) convolution kernels behind the Euler API.

This package is the Python door to the C-ABI library ``lib/libeuler_b200.so`` (sources in
``csrc/``, interface in ``include/euler_b200.h``).  It mirrors the reference's public surface
(``include/euler.hpp``): an ``eld_conv_t`` descriptor with the same field names, ``setup()`` and
``elx_conv(desc, output, input, weights, bias)``.  ``Linear``, ``BlockNorm``, ``Route``, ``Experts``, ``Rotary``,
``CacheAppend`` and ``Attention`` are the operators of transformer blocks, with the same describe / prepare / enqueue protocol.

There is no CPU implementation here.  Importing works without a GPU (the library loads and its
symbols can be inspected), but every compute call needs an sm_100 device and fails loudly
otherwise; a missing or stale shared library raises at import time.
"""
from __future__ import annotations

import ctypes as C
import os
import subprocess
from pathlib import Path
from types import SimpleNamespace

PKG_DIR = Path(__file__).resolve().parent
ROOT = PKG_DIR.parent
LIB_PATH = PKG_DIR / "lib" / "libeuler_b200.so"
HOST_LIB_PATH = PKG_DIR / "lib" / "libel.so"

# ----------------------------------------------------------------------------- constants
ELB_OK, ELB_UNIMPLEMENTED, ELB_GENERAL_ERROR = 0, 1, 2
ELD_OK, ELD_UNIMPLEMENTED, ELD_GENERAL_ERROR = 0, 1, 2
ELX_OK, ELX_UNIMPLEMENTED, ELX_GENERAL_ERROR = 0, 1, 2
CONV_AUTO, CONV_DIRECT_1X1, CONV_DIRECT, CONV_DIRECT_VMG, CONV_WINOGRAD, DECONV_DIRECT = range(6)
data_type_undef, f32, f16, u8, s8, s32, bf16 = range(7)
(format_undef, nchw, nhwc, nChw16c, nChw8c, oihw, hwio, OIhw16i16o, OIhw8i8o, goihw, ghwio, gOIhw16i16o,
 gOIhw8i8o) = range(13)
forward_training, forward_inference, backward_data, backward_weights = range(4)
FINE, COARSE, CALIBRATED = range(3)
ACT_NONE, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU = range(5)
NORM_NONE, NORM_RMS, NORM_LAYER = range(3)
SCORE_SOFTMAX, SCORE_SIGMOID = range(2)
ROTARY_HALVES, ROTARY_NEIGHBOURS = range(2)
SCALE_NONE, SCALE_LINEAR, SCALE_BY_PARTS = range(3)
EL_NO_CALI = 3.4028234663852886e38
KERNEL_NAMES = {0: "none", 1: "i8_gemm_umma", 2: "i8_conv_umma", 3: "i8_simt", 4: "wino_f32_umma",
                5: "wino_i8_umma", 6: "i8_depthwise", 7: "f32_direct_umma", 8: "f32_small_ic", 9: "conv_halo"}


def build(verbose: bool = False) -> Path:
    """Compile the CUDA library and the C++ host library (see _build.py)."""
    from . import _build
    return _build.build(verbose)


# ----------------------------------------------------------------------------- C structs
class ElbConvDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in
                ("n", "g", "ic", "oc", "ih", "iw", "oh", "ow", "kh", "kw", "pad_l", "pad_r", "pad_t", "pad_b",
                 "stride_h", "stride_w", "dilation_h", "dilation_w", "dt_input", "dt_weights", "dt_output",
                 "dt_bias", "fmt_input", "fmt_weights", "fmt_output", "prop_kind", "algorithm", "tile_size",
                 "with_relu", "with_bias", "with_ip_sum", "with_op_sum", "with_argmax", "f16c_opt",
                 "disable_autoparam")] + \
               [("relu_lower", C.c_float), ("relu_upper", C.c_float), ("execution_mode", C.c_int32)] + \
               [(k, C.c_float) for k in ("input_scale", "input_z", "tinput_scale", "tinput_z", "output_scale",
                                         "output_z", "sum_scale", "sum_z")] + \
               [("sampling_kind", C.c_int32), ("flatting_t", C.c_int32), ("device", C.c_int32)]


class ElbConvInfo(C.Structure):
    _fields_ = [("algorithm", C.c_int32), ("tile_size", C.c_int32), ("kernel", C.c_int32), ("device", C.c_int32)] + \
               [(k, C.c_uint64) for k in ("size_input", "size_weights", "size_output", "size_bias", "bytes_input",
                                          "bytes_weights", "bytes_output", "bytes_bias", "workspace_bytes")] + \
               [("launches_per_call", C.c_int32), ("launched_kernel", C.c_int32)]


class ElbLinearDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("ic", "oc", "dt_input", "dt_output", "dt_bias", "fmt_weights", "activation", "gated",
                                         "with_bias", "with_residual")] + \
               [("scale", C.c_float), ("device", C.c_int32)] + \
               [(k, C.c_int64) for k in ("ld_input", "ld_output", "ld_residual")]


class ElbNormDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("channels", "dt", "dt_residual", "dt_weights", "post", "pre")] + \
               [(k, C.c_float) for k in ("post_eps", "pre_eps", "weight_offset", "scale")] + \
               [(k, C.c_int32) for k in ("with_residual", "gate_rows", "device")] + \
               [(k, C.c_int64) for k in ("ld_input", "ld_residual", "ld_gate", "ld_sum", "ld_output")]


class ElbRouteDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("experts", "top_k", "dt_logits", "score", "with_bias", "groups", "top_groups",
                                         "group_best", "renormalise")] + \
               [("scale", C.c_float), ("device", C.c_int32), ("ld_logits", C.c_int64)]


class ElbExpertsDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("experts", "top_k", "ic", "mid", "dt", "activation", "gated", "device")] + \
               [(k, C.c_int64) for k in ("max_rows", "ld_input", "ld_output")]


class ElbRotaryDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("heads", "kv_heads", "head_dim", "rotary_dim", "dt", "layout", "scaling", "inverse")] + \
               [(k, C.c_float) for k in ("base", "factor", "slow", "fast", "magnitude")] + [("original", C.c_int32), ("device", C.c_int32)] + \
               [(k, C.c_int64) for k in ("ld_q", "ld_k", "ld_q_out", "ld_k_out")]


class ElbAppendDesc(C.Structure):
    _fields_ = [("rotary", ElbRotaryDesc), ("page_size", C.c_int32), ("reserved", C.c_int32)] + \
               [(k, C.c_int64) for k in ("ld_v", "ld_page", "ld_head", "ld_token")]


class ElbAttentionDesc(C.Structure):
    _fields_ = [(k, C.c_int32) for k in ("heads", "kv_heads", "head_dim", "dt", "page_size", "causal")] + \
               [("scale", C.c_float), ("device", C.c_int32)] + \
               [(k, C.c_int64) for k in ("ld_input", "ld_output", "ld_page", "ld_head", "ld_token")]


def _load():
    if not LIB_PATH.exists():
        raise ImportError(f"{LIB_PATH} is missing: run `python -c 'import __graft_entry__ as g; g.build()'` "
                          "(there is no CPU fallback)")
    lib = C.CDLL(str(LIB_PATH))
    vp, i32, u64 = C.c_void_p, C.c_int32, C.c_uint64
    sig = {
        "elb_conv_sizes": (i32, [C.POINTER(ElbConvDesc), C.POINTER(ElbConvInfo)]),
        "elb_conv_create": (i32, [C.POINTER(ElbConvDesc), C.POINTER(vp)]),
        "elb_conv_info": (i32, [vp, C.POINTER(ElbConvInfo)]),
        "elb_conv_execute": (i32, [vp, vp, vp, vp, vp]),
        "elb_conv_enqueue": (i32, [vp, vp, vp, vp, vp, vp]),
        "elb_conv_input_step_supported": (i32, [vp]),
        "elb_conv_enqueue_strided": (i32, [vp, vp, vp, i32, i32, i32, vp]),
        "elb_conv_prepare": (i32, [vp, vp, vp]),
        "elb_conv_set_accumulator_dump": (i32, [vp, vp]),
        "elb_conv_device_status": (i32, [vp]),
        "elb_conv_launch_count": (u64, [vp]),
        "elb_conv_set_stage_events": (i32, [vp, C.POINTER(vp)]),
        "elb_conv_destroy": (None, [vp]),
        "elb_last_error": (C.c_char_p, []),
        "elb_device_supported": (i32, [i32]),
        "elb_reorder_nchw_to_nChw16c": (i32, [vp, vp, i32, i32, i32, i32, i32, vp]),
        "elb_reorder_nChw16c_to_nchw": (i32, [vp, vp, i32, i32, i32, i32, i32, vp]),
        "elb_reorder": (i32, [vp, i32, vp, i32, i32, i32, i32, i32, i32, i32, vp]),
        "elb_subsample_nChw16c": (i32, [vp, vp, i32, i32, i32, i32, i32, i32, i32, vp]),
        "elb_selftest_bounded_wait": (i32, [i32, C.c_ulonglong]),
        "elb_conv_set_trace": (i32, [vp, vp]),
        "elb_conv_execute_async": (i32, [vp, vp, vp, vp, vp]),
        "elb_conv_wait": (i32, [vp]),
        "elb_conv_set_name": (i32, [vp, C.c_char_p]),
        "elb_stack_create": (i32, [C.POINTER(ElbConvDesc), C.POINTER(i32), i32, C.POINTER(vp)]),
        "elb_stack_prepare": (i32, [vp, i32, vp, vp]),
        "elb_stack_enqueue": (i32, [vp, vp, vp, vp]),
        "elb_stack_execute": (i32, [vp, vp, vp, C.c_int64]),
        "elb_stack_layer": (i32, [vp, i32, C.POINTER(vp)]),
        "elb_stack_sizes": (i32, [vp, C.POINTER(i32), C.POINTER(u64), C.POINTER(u64)]),
        "elb_stack_launch_count": (u64, [vp]),
        "elb_stack_layer_output": (i32, [vp, i32, C.POINTER(vp), C.POINTER(u64)]),
        "elb_stack_set_layer_events": (i32, [vp, C.POINTER(vp), i32]),
        "elb_stack_destroy": (None, [vp]),
        "elb_conv_multi_create": (i32, [C.POINTER(ElbConvDesc), C.POINTER(i32), i32, C.POINTER(vp)]),
        "elb_conv_multi_execute": (i32, [vp, vp, vp, vp, vp]),
        "elb_conv_multi_parts": (i32, [vp, C.POINTER(i32), C.POINTER(i32), C.POINTER(i32), C.POINTER(i32)]),
        "elb_conv_multi_destroy": (None, [vp]),
        "elb_wino_f32_conv_noalloc": (i32, [C.POINTER(ElbConvDesc), vp, vp, vp, vp, vp]),
        "elb_wino_f32_noalloc_status": (i32, []),
        "elb_linear_create": (i32, [C.POINTER(ElbLinearDesc), C.POINTER(vp)]),
        "elb_linear_prepare": (i32, [vp, vp, vp]),
        "elb_linear_enqueue": (i32, [vp, vp, vp, vp, C.c_int64, vp]),
        "elb_norm_create": (i32, [C.POINTER(ElbNormDesc), C.POINTER(vp)]),
        "elb_norm_prepare": (i32, [vp, vp, vp, vp, vp]),
        "elb_norm_enqueue": (i32, [vp, vp, vp, vp, vp, vp, C.c_int64, vp]),
        "elb_route_create": (i32, [C.POINTER(ElbRouteDesc), C.POINTER(vp)]),
        "elb_route_prepare": (i32, [vp, vp]),
        "elb_route_enqueue": (i32, [vp, vp, vp, vp, C.c_int64, vp]),
        "elb_experts_create": (i32, [C.POINTER(ElbExpertsDesc), C.POINTER(vp)]),
        "elb_experts_prepare": (i32, [vp, vp, vp]),
        "elb_experts_enqueue": (i32, [vp, vp, vp, vp, vp, C.c_int64, vp]),
        "elb_rotary_create": (i32, [C.POINTER(ElbRotaryDesc), C.POINTER(vp)]),
        "elb_rotary_prepare": (i32, [vp, vp]),
        "elb_rotary_enqueue": (i32, [vp, vp, vp, vp, vp, vp, C.c_int64, vp]),
        "elb_append_create": (i32, [C.POINTER(ElbAppendDesc), C.POINTER(vp)]),
        "elb_append_prepare": (i32, [vp, vp]),
        "elb_append_enqueue": (i32, [vp] * 10 + [C.c_int64] * 4 + [vp]),
        "elb_attention_create": (i32, [C.POINTER(ElbAttentionDesc), C.POINTER(vp)]),
        "elb_attention_enqueue": (i32, [vp] * 8 + [C.c_int64] * 4 + [vp]),
        "elb_op_device_status": (i32, [vp]),
        "elb_op_device": (i32, [vp]),
        "elb_op_launch_count": (u64, [vp]),
        "elb_op_workspace_bytes": (u64, [vp]),
        "elb_op_destroy": (None, [vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)          # AttributeError here = stale library
        fn.restype, fn.argtypes = res, args
    return lib


lib = _load()
EXPORTED_SYMBOLS = ["elb_conv_sizes", "elb_conv_create", "elb_conv_info", "elb_conv_execute", "elb_conv_enqueue",
                    "elb_conv_prepare", "elb_conv_set_accumulator_dump", "elb_conv_device_status",
                    "elb_conv_launch_count", "elb_conv_set_stage_events", "elb_conv_destroy", "elb_last_error", "elb_device_supported",
                    "elb_reorder_nchw_to_nChw16c", "elb_reorder_nChw16c_to_nchw", "elb_reorder", "elb_subsample_nChw16c",
                    "elb_conv_execute_async", "elb_conv_wait", "elb_conv_set_name", "elb_conv_set_trace",
                    "elb_selftest_bounded_wait", "elb_stack_create", "elb_stack_prepare", "elb_stack_enqueue",
                    "elb_stack_execute", "elb_stack_layer", "elb_stack_sizes", "elb_stack_launch_count",
                    "elb_stack_layer_output", "elb_stack_set_layer_events", "elb_stack_destroy", "elb_conv_multi_create", "elb_conv_multi_execute", "elb_conv_multi_parts",
                    "elb_conv_multi_destroy", "elb_wino_f32_conv_noalloc", "elb_wino_f32_noalloc_status",
                    "elb_conv_input_step_supported", "elb_conv_enqueue_strided",
                    "elb_linear_create", "elb_linear_prepare", "elb_linear_enqueue", "elb_norm_create", "elb_norm_prepare",
                    "elb_norm_enqueue", "elb_route_create", "elb_route_prepare", "elb_route_enqueue", "elb_experts_create",
                    "elb_experts_prepare", "elb_experts_enqueue", "elb_rotary_create", "elb_rotary_prepare", "elb_rotary_enqueue",
                    "elb_append_create", "elb_append_prepare", "elb_append_enqueue", "elb_attention_create", "elb_attention_enqueue", "elb_op_device_status", "elb_op_device", "elb_op_launch_count",
                    "elb_op_workspace_bytes", "elb_op_destroy"]


def last_error() -> str:
    return lib.elb_last_error().decode()


def _ptr(x):
    """Address of a torch tensor / numpy array / int / None."""
    if x is None:
        return None
    try:
        return x.data_ptr()                 # (first: what the calls of a running program pass)
    except AttributeError:
        pass
    if isinstance(x, int):
        return x
    if hasattr(x, "ctypes"):
        return x.ctypes.data
    raise TypeError(f"cannot take the address of {type(x)}")


class eld_conv_t:
    """Python mirror of ``euler::eld_conv_t`` (include/euler.hpp:110-187): same field names, same
    defaults (src/eld_conv.cpp:21-50), ``setup()`` returns ELD_* codes and fills ``sizes`` /
    ``byte_sizes``; the plan (``xc``) is released by ``close()`` or garbage collection."""

    def __init__(self):
        self.dims = SimpleNamespace(n=0, g=1, ic=0, oc=0, ih=0, iw=0, oh=0, ow=0, kh=0, kw=0)
        self.pads = SimpleNamespace(l=1, r=1, t=1, b=1)
        self.strides = SimpleNamespace(h=1, w=1)
        self.dilations = SimpleNamespace(h=1, w=1)
        self.data_type = SimpleNamespace(input=f32, weights=f32, output=f32, bias=f32)
        self.formats = SimpleNamespace(input=nChw16c, weights=OIhw16i16o, output=nChw16c)
        self.prop_kind = forward_inference
        self.algorithm = CONV_DIRECT
        self.tile_size = 0
        self.with_relu = self.with_bias = self.with_ip_sum = self.with_op_sum = self.with_argmax = False
        self.f16c_opt = False
        self.is_inference = True
        self.use_scratch_pad = False
        self.disable_autoparam = True
        self.eager_mode = True
        self.stream_sync = False
        self.relu_bound = SimpleNamespace(lower=0.0, upper=EL_NO_CALI)
        self.nthreads = 0
        self.execution_mode = 0
        self.flatting = SimpleNamespace(o=0, t=0)
        self.blocking = SimpleNamespace(i=0, o=0)
        self.partition = SimpleNamespace(i=1, o=1, g=1)
        self.streaming_hint = SimpleNamespace(input=0, output=0)
        self.input_quant = SimpleNamespace(scale=EL_NO_CALI, z=EL_NO_CALI)
        self.wino_tinput_quant = SimpleNamespace(scale=EL_NO_CALI, z=EL_NO_CALI)
        self.output_quant = SimpleNamespace(scale=EL_NO_CALI, z=EL_NO_CALI)
        self.sum_quant = SimpleNamespace(scale=1.0, z=0.0)
        self.sampling_kind = FINE
        self.name = "ioi"
        self.device = -1
        self.sizes = SimpleNamespace(input=0, weights=0, output=0, bias=0)
        self.byte_sizes = SimpleNamespace(input=0, weights=0, output=0, bias=0)
        self.xc = None
        self.info = None

    def _c_desc(self) -> ElbConvDesc:
        d, p = self.dims, self.pads
        return ElbConvDesc(
            d.n, d.g, d.ic, d.oc, d.ih, d.iw, d.oh, d.ow, d.kh, d.kw, p.l, p.r, p.t, p.b, self.strides.h,
            self.strides.w, self.dilations.h, self.dilations.w, self.data_type.input, self.data_type.weights,
            self.data_type.output, self.data_type.bias, self.formats.input, self.formats.weights,
            self.formats.output, self.prop_kind, self.algorithm, self.tile_size, int(self.with_relu),
            int(self.with_bias), int(self.with_ip_sum), int(self.with_op_sum), int(self.with_argmax),
            int(self.f16c_opt), int(self.disable_autoparam), self.relu_bound.lower, self.relu_bound.upper,
            self.execution_mode, self.input_quant.scale, self.input_quant.z, self.wino_tinput_quant.scale,
            self.wino_tinput_quant.z, self.output_quant.scale, self.output_quant.z, self.sum_quant.scale,
            self.sum_quant.z, int(self.sampling_kind), int(self.flatting.t), self.device)

    def setup(self, fully_setup: bool = True) -> int:
        desc = self._c_desc()
        info = ElbConvInfo()
        self.close()
        if fully_setup:
            plan = C.c_void_p()
            rc = lib.elb_conv_create(C.byref(desc), C.byref(plan))
            if rc != ELB_OK:
                return rc
            self.xc = plan
            lib.elb_conv_info(self.xc, C.byref(info))
            lib.elb_conv_set_name(self.xc, str(self.name).encode())
        else:
            rc = lib.elb_conv_sizes(C.byref(desc), C.byref(info))
            if rc != ELB_OK:
                return rc
        self.info = info
        self.algorithm, self.tile_size = info.algorithm, info.tile_size
        self.sizes = SimpleNamespace(input=info.size_input, weights=info.size_weights, output=info.size_output,
                                     bias=info.size_bias)
        self.byte_sizes = SimpleNamespace(input=info.bytes_input, weights=info.bytes_weights,
                                          output=info.bytes_output, bias=info.bytes_bias)
        return ELD_OK

    @property
    def kernel(self) -> str:
        return KERNEL_NAMES.get(self.info.kernel if self.info else 0, "?")

    @property
    def launched_kernel(self) -> str:
        """The kernel that a call launches: ``kernel``, or "conv_halo" where the plan serves the request with it."""
        return KERNEL_NAMES.get(self.info.launched_kernel if self.info else 0, "?")

    def prepare(self, weights, bias) -> int:
        return lib.elb_conv_prepare(self.xc, _ptr(weights), _ptr(bias))

    def enqueue(self, output, input, weights=None, bias=None, stream=None) -> int:
        """Device pointers only; returns after the kernels are enqueued on ``stream``."""
        return lib.elb_conv_enqueue(self.xc, _ptr(output), _ptr(input), _ptr(weights), _ptr(bias), stream)

    def input_step_supported(self) -> bool:
        return bool(lib.elb_conv_input_step_supported(self.xc))

    def enqueue_strided(self, output, input, src_h: int, src_w: int, step: int, stream=None) -> int:
        """As enqueue on a prepared plan, but ``input`` holds src_h x src_w pixels per plane of which every
        ``step``-th row and column is read (a subsample folded into the kernel's loads)."""
        return lib.elb_conv_enqueue_strided(self.xc, _ptr(output), _ptr(input), src_h, src_w, step, stream)

    def set_accumulator_dump(self, dev_int32) -> int:
        return lib.elb_conv_set_accumulator_dump(self.xc, _ptr(dev_int32))

    def device_status(self) -> int:
        return lib.elb_conv_device_status(self.xc)

    def launch_count(self) -> int:
        return int(lib.elb_conv_launch_count(self.xc))

    def set_stage_events(self, handles) -> int:
        """Four cudaEvent_t handles (ints) recorded around the three Winograd kernels; None = off."""
        if handles is None:
            return lib.elb_conv_set_stage_events(self.xc, None)
        arr = (C.c_void_p * 4)(*[int(h) for h in handles])
        return lib.elb_conv_set_stage_events(self.xc, arr)

    def wait(self) -> int:
        """Complete the asynchronous calls made with ``eager_mode = False`` (what a later call with
        ``stream_sync = True`` does in the reference, src/elx_conv.cpp:234-235)."""
        return lib.elb_conv_wait(self.xc)

    def close(self):
        if self.xc is not None:
            lib.elb_conv_destroy(self.xc)
            self.xc = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def elx_conv(desc: eld_conv_t, output, input, weights, bias) -> int:
    """``euler::elx_conv`` (include/euler.hpp:190): run the convolution and wait.  Arguments may be
    torch tensors (CUDA or CPU), numpy arrays or raw addresses; output comes first."""
    if desc.xc is None:
        raise RuntimeError("elx_conv: descriptor is not set up")
    if desc.eager_mode:
        return lib.elb_conv_execute(desc.xc, _ptr(output), _ptr(input), _ptr(weights), _ptr(bias))
    # eager_mode = False: enqueue and return; stream_sync = True waits (src/elx_conv.cpp:228-236)
    rc = lib.elb_conv_execute_async(desc.xc, _ptr(output), _ptr(input), _ptr(weights), _ptr(bias))
    if rc == ELB_OK and desc.stream_sync:
        rc = lib.elb_conv_wait(desc.xc)
    return rc


def _elem_bytes(x) -> int:
    if hasattr(x, "element_size"):
        return x.element_size()
    return x.dtype.itemsize


def reorder(dst, dst_format: int, src, src_format: int, *dims, stream=None) -> int:
    """``euler::reorder<T, dst_format, src_format>(dst, src, dims...)`` (include/euler_reorder.hpp:9-64)
    for DEVICE tensors: dims are (n, c, h, w), (o, i, h, w) or (g, o, i, h, w) as in the reference.
    The call is asynchronous on ``stream`` (default stream when None)."""
    if len(dims) == 4:
        g, (a, b, h, w) = 1, dims
    elif len(dims) == 5:
        g, a, b, h, w = dims
    else:
        raise ValueError("reorder takes 4 or 5 extents")
    return lib.elb_reorder(_ptr(dst), dst_format, _ptr(src), src_format, g, a, b, h, w, _elem_bytes(src), _ptr(stream))


def subsample(dst, src, n: int, c: int, h: int, w: int, step_h: int = 2, step_w: int = 2, stream=None) -> int:
    """Keep every step_h-th row and step_w-th column of a device nChw16c tensor (the glue between two
    layers of a stack; the reference's harness chains layers on the host, tests/elt_conv.cpp:399-410)."""
    return lib.elb_subsample_nChw16c(_ptr(dst), _ptr(src), n, c, h, w, step_h, step_w, _elem_bytes(src), _ptr(stream))


class ConvStack:
    """A chain of convolutions that stays on the device (``elb_stack_*``): ``descs`` are set-up-able
    ``eld_conv_t`` descriptors, ``subsample_after[k]`` = 2 keeps every second row and column of layer
    k's output.  The reference's harness chains layers on the host (tests/elt_conv.cpp:399-410)."""

    def __init__(self, descs, subsample_after=None):
        n = len(descs)
        arr = (ElbConvDesc * n)(*[d._c_desc() for d in descs])
        steps = (C.c_int32 * n)(*[int(v) for v in (subsample_after or [1] * n)])
        h = C.c_void_p()
        rc = lib.elb_stack_create(arr, steps, n, C.byref(h))
        if rc != ELB_OK:
            raise RuntimeError(f"elb_stack_create rc={rc}: {last_error()}")
        self.h, self.n_layers = h, n
        nl, bi, bo = C.c_int32(), C.c_uint64(), C.c_uint64()
        lib.elb_stack_sizes(self.h, C.byref(nl), C.byref(bi), C.byref(bo))
        self.bytes_input, self.bytes_output = bi.value, bo.value

    def prepare(self, layer: int, weights, bias) -> int:
        return lib.elb_stack_prepare(self.h, layer, _ptr(weights), _ptr(bias))

    def enqueue(self, output, input, stream=None) -> int:
        return lib.elb_stack_enqueue(self.h, _ptr(output), _ptr(input), stream)

    def execute(self, output, input, images: int) -> int:
        return lib.elb_stack_execute(self.h, _ptr(output), _ptr(input), images)

    def layer_plan(self, layer: int):
        p = C.c_void_p()
        lib.elb_stack_layer(self.h, layer, C.byref(p))
        return p

    def layer_kernel(self, layer: int) -> str:
        info = ElbConvInfo()
        lib.elb_conv_info(self.layer_plan(layer), C.byref(info))
        return KERNEL_NAMES.get(info.kernel, "?")

    def launch_count(self) -> int:
        return int(lib.elb_stack_launch_count(self.h))

    def layer_output(self, layer: int):
        """(device address, bytes) of layer k's output tensor inside the stack; address None for the last layer."""
        p, b = C.c_void_p(), C.c_uint64()
        lib.elb_stack_layer_output(self.h, layer, C.byref(p), C.byref(b))
        return p.value, b.value

    def set_layer_events(self, handles) -> int:
        if handles is None:
            return lib.elb_stack_set_layer_events(self.h, None, 0)
        arr = (C.c_void_p * len(handles))(*[int(h) for h in handles])
        return lib.elb_stack_set_layer_events(self.h, arr, len(handles))

    def close(self):
        if self.h is not None:
            lib.elb_stack_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class MultiConv:
    """One convolution whose minibatch is split over the GPUs of this box (``elb_conv_multi_*``):
    GPU r runs images [r*N/G, (r+1)*N/G) of the host tensors; weights are replicated."""

    def __init__(self, desc: eld_conv_t, devices=None, n_devices: int = 0):
        cd = desc._c_desc()
        h = C.c_void_p()
        arr = (C.c_int32 * len(devices))(*devices) if devices else None
        rc = lib.elb_conv_multi_create(C.byref(cd), arr, len(devices) if devices else n_devices, C.byref(h))
        if rc != ELB_OK:
            raise RuntimeError(f"elb_conv_multi_create rc={rc}: {last_error()}")
        self.h = h

    def parts(self):
        n = C.c_int32(64)
        dev, first, cnt = (C.c_int32 * 64)(), (C.c_int32 * 64)(), (C.c_int32 * 64)()
        lib.elb_conv_multi_parts(self.h, C.byref(n), dev, first, cnt)
        return [(dev[i], first[i], cnt[i]) for i in range(n.value)]

    def execute(self, output, input, weights, bias) -> int:
        return lib.elb_conv_multi_execute(self.h, _ptr(output), _ptr(input), _ptr(weights), _ptr(bias))

    def close(self):
        if self.h is not None:
            lib.elb_conv_multi_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_DTYPE_NAMES = {f32: "float32", f16: "float16", bf16: "bfloat16", s32: "int32"}


def _dev(x, device):
    """Address of a tensor of ``device`` (torch tensor, raw address or None) that a call does not use."""
    if x is None or type(x) is int:
        return x
    if x.get_device() != device:
        raise ValueError(f"the plan's enqueue calls take tensors of device {device}")
    return x.data_ptr()


class _Spec:
    """What a plan wants of a tensor: rows of ``n`` elements of an ELB type, ``ld`` apart, on the plan's device."""
    __slots__ = ("type", "n", "ld", "what", "device", "dtype", "row_bytes")

    def __init__(self, type, n, ld, what, device):
        self.type, self.n, self.ld, self.what, self.device = type, n, ld or n, what, device
        self.dtype = None                                                # the tensors' own name for the type, once one has been met
        self.row_bytes = n * (2 if type in (f16, bf16) else 4) if self.ld == n else float("inf")


def _rows(x, spec, rows):
    """Address of a device tensor of which a call reads or writes ``rows`` rows: a torch tensor that holds them, a raw address, which is taken as it
    is, or None.  (A property of a tensor costs 30 to 70 ns here, beside a call's 4 us: dense tensors are looked at three times.)"""
    if x is None or type(x) is int:
        return x
    if not (x.dtype is spec.dtype and x.is_contiguous() and x.nbytes >= rows * spec.row_bytes) and rows > 0:
        _check_rows(x, spec, rows)
    if x.get_device() != spec.device:
        raise ValueError(f"{spec.what}: the plan's enqueue calls take tensors of device {spec.device}")
    return x.data_ptr()


def _check_rows(x, spec, rows):
    """As ``_rows``, for any tensor: a dense one of enough elements where rows are dense or it has one dimension; otherwise the last dimension holds
    a row, and the others, taken together, ``rows`` of them, ``ld`` elements apart."""
    n, ld = spec.n, spec.ld
    name, shape, stride = str(x.dtype).replace("torch.", ""), tuple(x.shape), tuple(x.stride())
    if x.is_contiguous() and (ld == n or len(shape) == 1):
        fits = x.numel() >= (rows - 1) * ld + n
    else:
        fits = bool(shape) and shape[-1] >= n and (n == 1 or stride[-1] == 1)
        held = 1
        for size, step in zip(reversed(shape[:-1]), reversed(stride[:-1])):
            fits = fits and (size == 1 or step == held * ld)
            held *= size
        fits = fits and held >= rows
    if not fits or name != _DTYPE_NAMES[spec.type]:
        raise ValueError(f"{spec.what}: {rows} rows of {n} elements in {_DTYPE_NAMES[spec.type]}, {ld} apart, are wanted, got {shape} with strides {stride} in {name}")
    spec.dtype = x.dtype


def _dense(x, shape, dtypes, what):
    """Address of a weight tensor for an operator's prepare, which reads all of ``shape``: a dense torch tensor or numpy array of that many
    elements of one of ``dtypes`` (ELB types), a raw address, or None."""
    if x is None or isinstance(x, int):
        return x
    n = 1
    for d in shape:
        n *= d
    contiguous = x.is_contiguous() if hasattr(x, "is_contiguous") else x.flags["C_CONTIGUOUS"]
    count = x.numel() if hasattr(x, "numel") else x.size
    name = str(x.dtype).replace("torch.", "")
    if not contiguous or count != n or name not in [_DTYPE_NAMES[t] for t in dtypes]:
        raise ValueError(f"{what}: a dense tensor of {n} elements {shape} in {[_DTYPE_NAMES[t] for t in dtypes]} is wanted, got {tuple(x.shape)} "
                         f"in {name}{'' if contiguous else ', not dense'}")
    return _ptr(x)


class _Op:
    """A plan of one of the operators of transformer blocks (``elb_op_t``).  ``prepare`` copies the weights (host or
    device tensors, read once; later calls do nothing), ``enqueue`` runs on ``stream`` (a cudaStream_t; None: the legacy default stream, not
    torch's current one) and returns an ELB_* code; rows of tensors are ``ld_*`` elements apart (0: dense).  Torch tensors must hold the call's
    rows in the plan's types, on its device, or ``enqueue`` raises ValueError; raw addresses are taken as they are."""
    h = None

    def _create(self, create, desc):
        h = C.c_void_p()
        rc = create(C.byref(desc), C.byref(h))
        if rc != ELB_OK:
            raise RuntimeError(f"rc={rc}: {last_error()}")
        self.h = h
        self.device = lib.elb_op_device(h)

    def _spec(self, type, n, ld, what):
        return _Spec(type, n, ld, what, self.device)

    def device_status(self) -> int:
        return lib.elb_op_device_status(self.h)

    def launch_count(self) -> int:
        return int(lib.elb_op_launch_count(self.h))

    def workspace_bytes(self) -> int:
        return int(lib.elb_op_workspace_bytes(self.h))

    def close(self):
        if self.h is not None:
            lib.elb_op_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Linear(_Op):
    """output = residual + scale * act(input weights^T + bias), or scale * act(gate) * up where ``gated`` (weights and bias
    then hold the oc gate rows, then the oc up rows).  ``dtype``: bf16 or f16 operands; ``out_dtype``: the same or f32."""

    def __init__(self, ic: int, oc: int, dtype: int = bf16, out_dtype: int | None = None, activation: int = ACT_NONE, gated: bool = False,
                 with_bias: bool = False, bias_dtype: int = f32, with_residual: bool = False, scale: float = 1.0, weights_format: int = oihw,
                 ld_input: int = 0, ld_output: int = 0, ld_residual: int = 0, device: int = -1):
        self._create(lib.elb_linear_create, ElbLinearDesc(ic, oc, dtype, dtype if out_dtype is None else out_dtype, bias_dtype, weights_format,
                                                          activation, int(gated), int(with_bias), int(with_residual), scale, device,
                                                          ld_input, ld_output, ld_residual))
        wide = 2 * oc if gated else oc
        self._weights = ((wide, ic) if weights_format == oihw else (ic, wide), (dtype,))
        self._bias = ((wide,), (bias_dtype,))
        out = dtype if out_dtype is None else out_dtype
        self._output, self._input = self._spec(out, oc, ld_output, "output"), self._spec(dtype, ic, ld_input, "input")
        self._residual = self._spec(out, oc, ld_residual, "residual") if with_residual else None

    def prepare(self, weights, bias=None) -> int:
        return lib.elb_linear_prepare(self.h, _dense(weights, *self._weights, "weights"), _dense(bias, *self._bias, "bias"))

    def enqueue(self, output, input, residual=None, *, rows: int, stream=None) -> int:
        return lib.elb_linear_enqueue(self.h, _rows(output, self._output, rows), _rows(input, self._input, rows),
                                      _rows(residual, self._residual, rows) if self._residual else _dev(residual, self.device), rows, stream)


class BlockNorm(_Op):
    """sum = residual + scale * gate * post(input); output = pre(sum): what lies between two blocks.  ``post`` / ``pre``:
    NORM_*; ``gate_rows``: consecutive rows that share a row of the gate (0: no gate)."""

    def __init__(self, channels: int, dtype: int = bf16, residual_dtype: int | None = None, weights_dtype: int = f32, post: int = NORM_NONE,
                 pre: int = NORM_RMS, post_eps: float = 1e-6, pre_eps: float = 1e-6, weight_offset: float = 0.0, scale: float = 1.0,
                 with_residual: bool = True, gate_rows: int = 0, ld_input: int = 0, ld_residual: int = 0, ld_gate: int = 0, ld_sum: int = 0,
                 ld_output: int = 0, device: int = -1):
        self._create(lib.elb_norm_create, ElbNormDesc(channels, dtype, dtype if residual_dtype is None else residual_dtype, weights_dtype, post, pre,
                                                      post_eps, pre_eps, weight_offset, scale, int(with_residual), gate_rows, device,
                                                      ld_input, ld_residual, ld_gate, ld_sum, ld_output))
        self._vector = ((channels,), (weights_dtype,), "weights")
        stream = dtype if residual_dtype is None else residual_dtype
        self._output = self._spec(dtype, channels, ld_output, "output") if pre != NORM_NONE else None
        self._sum, self._input = self._spec(stream, channels, ld_sum, "sum"), self._spec(dtype, channels, ld_input, "input")
        self._residual = self._spec(stream, channels, ld_residual, "residual") if with_residual else None
        self._gate = self._spec(dtype, channels, ld_gate, "gate") if gate_rows else None
        self._gate_rows = gate_rows

    def prepare(self, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None) -> int:
        return lib.elb_norm_prepare(self.h, *(_dense(v, *self._vector) for v in (post_weight, post_bias, pre_weight, pre_bias)))

    def enqueue(self, output, sum, input, residual=None, gate=None, *, rows: int, stream=None) -> int:
        return lib.elb_norm_enqueue(self.h, _rows(output, self._output, rows) if self._output else _dev(output, self.device), _rows(sum, self._sum, rows),
                                    _rows(input, self._input, rows), _rows(residual, self._residual, rows) if self._residual else _dev(residual, self.device),
                                    _rows(gate, self._gate, -(-rows // self._gate_rows)) if self._gate else _dev(gate, self.device), rows, stream)


class Route(_Op):
    """The top_k experts of each row of logits, best first, and their weights.  ``with_bias``: a bias for balance counts for
    the choice alone; ``groups`` / ``top_groups`` / ``group_best``: only experts of the groups with the best choices."""

    def __init__(self, experts: int, top_k: int, dtype: int = f32, score: int = SCORE_SOFTMAX, with_bias: bool = False, groups: int = 1,
                 top_groups: int = 1, group_best: int = 1, renormalise: bool = True, scale: float = 1.0, ld_logits: int = 0, device: int = -1):
        self._create(lib.elb_route_create, ElbRouteDesc(experts, top_k, dtype, score, int(with_bias), groups, top_groups, group_best,
                                                        int(renormalise), scale, device, ld_logits))
        self._bias = ((experts,), (f32,), "bias")
        self._ids, self._weights, self._logits = self._spec(s32, top_k, 0, "ids"), self._spec(f32, top_k, 0, "weights"), self._spec(dtype, experts, ld_logits, "logits")

    def prepare(self, bias=None) -> int:
        return lib.elb_route_prepare(self.h, _dense(bias, *self._bias))

    def enqueue(self, ids, weights, logits, *, rows: int, stream=None) -> int:
        """ids: int32 [rows, top_k], weights: float32 [rows, top_k] or None, both dense."""
        return lib.elb_route_enqueue(self.h, _rows(ids, self._ids, rows), _rows(weights, self._weights, rows), _rows(logits, self._logits, rows), rows, stream)


class Experts(_Op):
    """output[t] = sum_j weights[t][j] * w_out[e] f(w_in[e] input[t]), e = ids[t][j]; an id outside 0 .. experts - 1 adds
    nothing.  w_in: [experts, mid (gated: 2 * mid, gate rows first), ic], w_out: [experts, ic, mid]."""

    def __init__(self, experts: int, top_k: int, ic: int, mid: int, max_rows: int, dtype: int = bf16, activation: int = ACT_SILU,
                 gated: bool = True, ld_input: int = 0, ld_output: int = 0, device: int = -1):
        self._create(lib.elb_experts_create, ElbExpertsDesc(experts, top_k, ic, mid, dtype, activation, int(gated), device, max_rows,
                                                            ld_input, ld_output))
        self._in = ((experts, 2 * mid if gated else mid, ic), (dtype,), "w_in")
        self._out = ((experts, ic, mid), (dtype,), "w_out")
        self._output, self._input = self._spec(dtype, ic, ld_output, "output"), self._spec(dtype, ic, ld_input, "input")
        self._ids, self._weights = self._spec(s32, top_k, 0, "ids"), self._spec(f32, top_k, 0, "weights")

    def prepare(self, w_in, w_out) -> int:
        return lib.elb_experts_prepare(self.h, _dense(w_in, *self._in), _dense(w_out, *self._out))

    def enqueue(self, output, input, ids, weights, *, rows: int, stream=None) -> int:
        return lib.elb_experts_enqueue(self.h, _rows(output, self._output, rows), _rows(input, self._input, rows), _rows(ids, self._ids, rows),
                                       _rows(weights, self._weights, rows), rows, stream)


class Rotary(_Op):
    """Queries and keys turned by their positions: pairs (i, i + r/2) or (2i, 2i + 1) of the first r = ``rotary_dim`` channels (None: all) of each
    head.  Either may have no heads; outputs may be their inputs' tensors.  ``prepare`` takes frequencies of its own, float32 [r / 2]."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, rotary_dim: int | None = None, dtype: int = bf16, layout: int = ROTARY_HALVES,
                 scaling: int = SCALE_NONE, inverse: bool = False, base: float = 10000.0, factor: float = 1.0, slow: float = 1.0, fast: float = 4.0,
                 magnitude: float = 1.0, original: int = 8192, ld_q: int = 0, ld_k: int = 0, ld_q_out: int = 0, ld_k_out: int = 0, device: int = -1):
        turn = head_dim if rotary_dim is None else rotary_dim
        self._create(lib.elb_rotary_create, ElbRotaryDesc(heads, kv_heads, head_dim, turn, dtype, layout, scaling, int(inverse), base, factor, slow,
                                                          fast, magnitude, original, device, ld_q, ld_k, ld_q_out, ld_k_out))
        self._frequencies = ((turn // 2,), (f32,), "frequencies")
        wide = ((heads, ld_q, "q"), (kv_heads, ld_k, "k"), (heads, ld_q_out, "q_out"), (kv_heads, ld_k_out, "k_out"))
        self._q, self._k, self._q_out, self._k_out = (self._spec(dtype, h * head_dim, ld, what) if h else None for h, ld, what in wide)
        self._positions = self._spec(s32, 1, 0, "positions")

    def prepare(self, frequencies=None) -> int:
        return lib.elb_rotary_prepare(self.h, _dense(frequencies, *self._frequencies))

    def enqueue(self, q_out, k_out, q, k, positions, *, rows: int, stream=None) -> int:
        return lib.elb_rotary_enqueue(self.h, _heads(q_out, self._q_out, rows, self.device), _heads(k_out, self._k_out, rows, self.device),
                                      _heads(q, self._q, rows, self.device), _heads(k, self._k, rows, self.device), _flat(positions, rows, self._positions),
                                      rows, stream)


class _Cache:
    """What a plan wants of a cache's tensor: [pages, kv_heads, page_size, head_dim], the middle two in either order, as its strides say."""
    __slots__ = ("type", "shape", "strides", "device", "dtype", "dense", "seen")

    def __init__(self, type, kv_heads, page_size, head_dim, ld_page, ld_head, ld_token, device):
        token = ld_token or head_dim
        head = ld_head or page_size * token
        page = ld_page or (kv_heads * head if head > token else page_size * token)
        self.type, self.device, self.dtype, self.seen = type, device, None, None         # seen: the last whole shape that has been found right
        self.shape, self.strides = (kv_heads, page_size, head_dim), (page, head, token, 1)
        self.dense = self.strides == (kv_heads * page_size * head_dim, page_size * head_dim, head_dim, 1)

    def take(self, x, what, pages):
        """(address, pages) of a cache"""
        if x is None or type(x) is int:
            if pages is None:
                raise ValueError(f"{what}: pages are wanted beside an address")
            return x, pages
        shape = x.shape
        if not (shape == self.seen and x.dtype is self.dtype and x.is_contiguous()):
            self.check(x, what, tuple(shape))
            self.seen = shape if self.dense and x.is_contiguous() and tuple(shape[1:]) == self.shape else None
        if x.get_device() != self.device:
            raise ValueError(f"{what}: the plan's enqueue calls take tensors of device {self.device}")
        if pages is None:
            pages = shape[0]
        elif pages > shape[0]:
            raise ValueError(f"{what}: {pages} pages are wanted, got {shape[0]}")
        return x.data_ptr(), pages

    def check(self, x, what, shape):
        name, stride, (heads, tokens, dim) = str(x.dtype).replace("torch.", ""), tuple(x.stride()), self.shape
        page, head, token, _ = self.strides

        def lies(a, b, sa, sb):
            return len(shape) == 4 and shape[1:] == (a, b, dim) and all(n == 1 or s == w for n, s, w in zip(shape, stride, (page, sa, sb, 1)))
        if name != _DTYPE_NAMES[self.type] or not (lies(heads, tokens, head, token) or lies(tokens, heads, token, head)):
            raise ValueError(f"{what}: pages of {heads} heads and {tokens} tokens of {dim} channels in {_DTYPE_NAMES[self.type]}, strides {self.strides} of page, "
                             f"head and token, are wanted, got {shape} with strides {stride} in {name}")
        self.dtype = x.dtype


def _heads(x, spec, rows, device):
    """Address of a tensor of which a call uses ``rows`` rows of heads: [rows, heads, channels] or [rows, heads * channels]; without heads, none."""
    if spec is None:
        return _dev(x, device)
    if x is None or type(x) is int:
        return x
    if x.dtype is spec.dtype and x.is_contiguous() and x.nbytes >= rows * spec.row_bytes and x.get_device() == spec.device:
        return x.data_ptr()
    if len(x.shape) == 3 and x.shape[2] != spec.n and (spec.ld != spec.n or not x.is_contiguous()):        # (one row is contiguous wherever the next would lie)
        (held, heads, dim), (row, head, one) = x.shape, x.stride()
        if not (heads * dim == spec.n and held >= rows and (held == 1 or row == spec.ld) and (heads == 1 or head == dim) and (dim == 1 or one == 1)) or \
                str(x.dtype).replace("torch.", "") != _DTYPE_NAMES[spec.type]:
            raise ValueError(f"{spec.what}: {rows} rows of {spec.n} elements in {_DTYPE_NAMES[spec.type]}, {spec.ld} apart, are wanted, got {tuple(x.shape)} with "
                             f"strides {tuple(x.stride())} in {x.dtype}")
        if x.get_device() != device:
            raise ValueError(f"{spec.what}: the plan's enqueue calls take tensors of device {device}")
        return x.data_ptr()
    return _rows(x, spec, rows)


def _flat(x, n, spec):
    """Address of a dense vector of at least n elements."""
    if x is None or type(x) is int:
        return x
    if x.dtype is not spec.dtype or not x.is_contiguous() or x.numel() < n:
        if str(x.dtype).replace("torch.", "") != _DTYPE_NAMES[spec.type] or not x.is_contiguous() or x.numel() < n:
            raise ValueError(f"{spec.what}: a dense tensor of {n} elements in {_DTYPE_NAMES[spec.type]} is wanted, got {tuple(x.shape)} in {x.dtype}")
        spec.dtype = x.dtype
    if x.get_device() != spec.device:
        raise ValueError(f"{spec.what}: the plan's enqueue calls take tensors of device {spec.device}")
    return x.data_ptr()


class _OverSequences(_Op):
    """A plan whose calls go over a batch of sequences: ``table`` [seqs, width], ``lengths`` [seqs] and ``starts`` [seqs + 1], all int32."""

    def _sequences(self):
        self._table, self._lengths, self._starts = (self._spec(s32, 1, 0, what) for what in ("table", "lengths", "starts"))

    def _batch(self, table, lengths, starts, seqs, width):
        """(table, lengths, starts, width)"""
        if table is not None and type(table) is not int:
            shape = table.shape
            if len(shape) != 2 or shape[0] < seqs:
                raise ValueError(f"table: {seqs} rows of pages are wanted, got {tuple(shape)}")
            if width is None:
                width = shape[1]
            elif width != shape[1]:
                raise ValueError(f"table: rows of {width} pages are wanted, got {tuple(shape)}")
        if width is None:
            raise ValueError("table: width is wanted beside an address")
        return _flat(table, seqs * width, self._table), _flat(lengths, seqs, self._lengths), _flat(starts, seqs + 1, self._starts), width


class CacheAppend(_OverSequences):
    """New tokens come into a cache of pages: q turned into ``q_out``, k turned into its place in ``k_cache``, v copied to its place in ``v_cache``.
    Caches are [pages, kv_heads, page_size, head_dim], or as ``ld_*`` say; ``rotary_dim`` 0: nothing turns."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, page_size: int, rotary_dim: int | None = None, dtype: int = bf16, layout: int = ROTARY_HALVES,
                 scaling: int = SCALE_NONE, base: float = 10000.0, factor: float = 1.0, slow: float = 1.0, fast: float = 4.0, magnitude: float = 1.0,
                 original: int = 8192, ld_q: int = 0, ld_k: int = 0, ld_v: int = 0, ld_q_out: int = 0, ld_page: int = 0, ld_head: int = 0, ld_token: int = 0,
                 device: int = -1):
        turn = head_dim if rotary_dim is None else rotary_dim
        self._create(lib.elb_append_create, ElbAppendDesc(ElbRotaryDesc(heads, kv_heads, head_dim, turn, dtype, layout, scaling, 0, base, factor, slow, fast,
                                                                        magnitude, original, device, ld_q, ld_k, ld_q_out, 0),
                                                          page_size, 0, ld_v, ld_page, ld_head, ld_token))
        self._frequencies = ((turn // 2,), (f32,), "frequencies")
        wide = ((heads, ld_q, "q"), (kv_heads, ld_k, "k"), (kv_heads, ld_v, "v"), (heads, ld_q_out, "q_out"))
        self._q, self._k, self._v, self._q_out = (self._spec(dtype, h * head_dim, ld, what) if h else None for h, ld, what in wide)
        self._cache = _Cache(dtype, kv_heads, page_size, head_dim, ld_page, ld_head, ld_token, self.device)
        self._sequences()

    def prepare(self, frequencies=None) -> int:
        return lib.elb_append_prepare(self.h, _dense(frequencies, *self._frequencies))

    def enqueue(self, q_out, k_cache, v_cache, q, k, v, table, lengths, starts=None, *, rows: int, seqs: int, pages: int | None = None, width: int | None = None,
                stream=None) -> int:
        dev, cache = self.device, self._cache
        kc, pages = cache.take(k_cache, "k_cache", pages)
        vc, pages = cache.take(v_cache, "v_cache", pages)
        table, lengths, starts, width = self._batch(table, lengths, starts, seqs, width)
        return lib.elb_append_enqueue(self.h, _heads(q_out, self._q_out, rows, dev), kc, vc, _heads(q, self._q, rows, dev), _heads(k, self._k, rows, dev),
                                      _heads(v, self._v, rows, dev), table, lengths, starts, rows, seqs, pages, width, stream)


class Attention(_OverSequences):
    """output[t] = sum_j softmax_j(scale * q[t] k[j]) v[j] over the keys that token t sees.  k and v: a cache of pages of ``page_size`` tokens, as
    CacheAppend writes it, with ``table`` and ``lengths``; or, ``page_size`` 0, tensors [seqs, keys, kv_heads, head_dim] (strides as ``ld_*`` say), of which
    ``lengths`` may leave the last keys out.  ``causal``: a sequence's new tokens are its last ones.  Nothing to prepare."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, dtype: int = bf16, page_size: int = 0, causal: bool = True, scale: float = 0.0, ld_input: int = 0,
                 ld_output: int = 0, ld_page: int = 0, ld_head: int = 0, ld_token: int = 0, device: int = -1):
        self._create(lib.elb_attention_create, ElbAttentionDesc(heads, kv_heads, head_dim, dtype, page_size, int(causal), scale, device, ld_input, ld_output,
                                                                ld_page, ld_head, ld_token))
        self._input, self._output = self._spec(dtype, heads * head_dim, ld_input, "input"), self._spec(dtype, heads * head_dim, ld_output, "output")
        self._cache = _Cache(dtype, kv_heads, page_size, head_dim, ld_page, ld_head, ld_token, self.device) if page_size else None
        head = ld_head or head_dim
        self._dense, self._dtype = (kv_heads, head_dim, ld_page, head, ld_token or kv_heads * head, dtype), None
        self._sequences()

    def _keys(self, x, what, seqs, width):
        """(address, keys of a sequence) of dense keys or values"""
        if x is None or type(x) is int:
            if width is None:
                raise ValueError(f"{what}: width is wanted beside an address")
            return x, width
        kv_heads, dim, ld_page, head, token, kind = self._dense
        shape, stride, name = tuple(x.shape), tuple(x.stride()), str(x.dtype).replace("torch.", "")

        def lies(keys, heads, sk, sh, rest):
            return heads == kv_heads and rest == dim and (keys <= 1 or sk == token) and (heads == 1 or sh == head) and (dim == 1 or stride[3] == 1) and \
                (shape[0] <= 1 or keys == 0 or stride[0] == (ld_page or keys * token)) and (width is None or keys == width)
        keys = None
        if len(shape) == 4 and name == _DTYPE_NAMES[kind] and shape[0] >= seqs:
            if lies(shape[1], shape[2], stride[1], stride[2], shape[3]):
                keys = shape[1]
            elif lies(shape[2], shape[1], stride[2], stride[1], shape[3]):
                keys = shape[2]
        if keys is None:
            raise ValueError(f"{what}: {seqs} sequences of {'keys' if width is None else width}, {kv_heads} heads of {dim} channels in {_DTYPE_NAMES[kind]}, strides "
                             f"{(ld_page or 'dense', token, head)} of sequence, key and head, are wanted, got {shape} with strides {stride} in {name}")
        if x.get_device() != self.device:
            raise ValueError(f"{what}: the plan's enqueue calls take tensors of device {self.device}")
        return x.data_ptr(), keys

    def enqueue(self, output, input, k, v, table=None, lengths=None, starts=None, *, rows: int, seqs: int, pages: int | None = None, width: int | None = None,
                stream=None) -> int:
        if self._cache:
            k, pages = self._cache.take(k, "k", pages)
            v, pages = self._cache.take(v, "v", pages)
            table, lengths, starts, width = self._batch(table, lengths, starts, seqs, width)
        else:
            k, width = self._keys(k, "k", seqs, width)
            v, width = self._keys(v, "v", seqs, width)
            if table is not None:
                raise ValueError("table: the plan's keys and values are dense")
            lengths, starts, pages = _flat(lengths, seqs, self._lengths), _flat(starts, seqs + 1, self._starts), 0
        return lib.elb_attention_enqueue(self.h, _heads(output, self._output, rows, self.device), _heads(input, self._input, rows, self.device), k, v, table, lengths,
                                         starts, rows, seqs, pages, width, stream)
