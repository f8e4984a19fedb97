"""ctypes mirror of the blocks and functions of include/cc1d_mixer.h that linear attention and the layer norm add."""
import ctypes as C

import cabi_mixer as mixer
from cabi import i32, i64, vp

f32 = C.c_float


class LayerNormParams(C.Structure):
    _fields_ = [("rows", i64), ("dim", i32), ("x_dtype", i32), ("r_dtype", i32), ("w_dtype", i32), ("eps", f32), ("reserved0", i32),
                ("x", vp), ("x_stride", i64), ("residual", vp), ("residual_stride", i64), ("weight", vp), ("bias", vp), ("h", vp), ("h_stride", i64),
                ("y", vp), ("y_stride", i64), ("stats", vp)]


class LayerNormBwdParams(C.Structure):
    _fields_ = [("rows", i64), ("dim", i32), ("x_dtype", i32), ("r_dtype", i32), ("w_dtype", i32), ("reserved0", i32), ("reserved1", i32), ("h", vp), ("h_stride", i64), ("stats", vp),
                ("weight", vp), ("dy", vp), ("dy_stride", i64), ("dh", vp), ("dh_stride", i64), ("dx", vp), ("dx_stride", i64),
                ("dresidual", vp), ("dresidual_stride", i64), ("dweight", vp), ("dbias", vp)]


STRUCTS = {"cc1d_layer_norm_params": LayerNormParams, "cc1d_layer_norm_bwd_params": LayerNormBwdParams}


def declare_linear(lib):
    size = C.POINTER(C.c_size_t)
    for name, st in (("linear", mixer.DeltaParams), ("linear_bwd", mixer.DeltaBwdParams), ("linear_step", mixer.DeltaStepParams),
                     ("layer_norm", LayerNormParams), ("layer_norm_bwd", LayerNormBwdParams)):
        getattr(lib, "cc1d_validate_" + name).argtypes = [C.POINTER(st)]
    for name, st in (("linear_workspace", mixer.DeltaParams), ("linear_saved", mixer.DeltaParams), ("linear_bwd_workspace", mixer.DeltaBwdParams),
                     ("layer_norm_bwd_workspace", LayerNormBwdParams)):
        getattr(lib, "cc1d_%s_bytes" % name).argtypes = [C.POINTER(st), size]
    for name, st in (("linear_fwd", mixer.DeltaParams), ("linear_bwd", mixer.DeltaBwdParams), ("layer_norm_bwd", LayerNormBwdParams)):
        getattr(lib, "cc1d_" + name).argtypes = [C.POINTER(st), vp, C.c_size_t, vp]
    for name, st in (("linear_step", mixer.DeltaStepParams), ("layer_norm_fwd", LayerNormParams)):
        getattr(lib, "cc1d_" + name).argtypes = [C.POINTER(st), vp]
    return lib
