"""ctypes mirror of include/cc1d_mixer.h.  Field order and types must match the header exactly."""
import ctypes as C

from cabi import DTYPES, _ptr, i32, i64, vp

f32 = C.c_float


def _tensor(name, *axes):
    return [(name, vp)] + [("%s_stride_%s" % (name, a), i64) for a in axes]


class DeltaParams(C.Structure):
    _fields_ = ([(n, i32) for n in ("batch", "seqlen", "heads", "v_heads", "dim_k", "dim_v", "sequences", "x_dtype", "g_dtype", "beta_dtype",
                                    "qk_l2norm", "cu_seqlens_is_int64")] + [("scale", f32), ("reserved0", i32)] +
                sum((_tensor(n, "b", "l", "h") for n in ("q", "k", "v", "g", "beta")), []) + [("cu_seqlens", vp)] +
                _tensor("initial_states", "n", "h", "k") + _tensor("out", "b", "l", "h") + _tensor("final_states", "n", "h", "k") + [("saved", vp)])


class DeltaBwdParams(C.Structure):
    _fields_ = ([("fwd", DeltaParams)] + _tensor("dout", "b", "l", "h") + _tensor("dfinal_states", "n", "h", "k") +
                sum((_tensor(n, "b", "l", "h") for n in ("dq", "dk", "dv")), []) + [("dg", vp), ("dbeta", vp)] +
                _tensor("dinitial_states", "n", "h", "k"))


class DeltaStepParams(C.Structure):
    _fields_ = ([(n, i32) for n in ("batch", "seqlen", "heads", "v_heads", "dim_k", "dim_v", "state_slots", "x_dtype", "g_dtype", "beta_dtype",
                                    "qk_l2norm")] + [("scale", f32)] + sum((_tensor(n, "b", "l", "h") for n in ("q", "k", "v", "g", "beta")), []) +
                _tensor("state", "n", "h", "k") + _tensor("out", "b", "l", "h") + [("state_indices", vp)])


class NormParams(C.Structure):
    _fields_ = [("rows", i64), ("dim", i32), ("x_dtype", i32), ("r_dtype", i32), ("w_dtype", i32), ("eps", f32), ("reserved0", i32),
                ("x", vp), ("x_stride", i64), ("residual", vp), ("residual_stride", i64), ("weight", vp), ("h", vp), ("h_stride", i64),
                ("y", vp), ("y_stride", i64), ("y8", vp), ("y8_stride", i64), ("scales", vp)]


class NormBwdParams(C.Structure):
    _fields_ = [("rows", i64), ("dim", i32), ("x_dtype", i32), ("r_dtype", i32), ("w_dtype", i32), ("eps", f32), ("reserved0", i32),
                ("h", vp), ("h_stride", i64), ("weight", vp), ("dy", vp), ("dy_stride", i64), ("dh", vp), ("dh_stride", i64),
                ("dx", vp), ("dx_stride", i64), ("dresidual", vp), ("dresidual_stride", i64), ("dweight", vp)]


class DequantizeParams(C.Structure):
    _fields_ = [("rows", i64), ("dim", i32), ("y_dtype", i32), ("y8", vp), ("y8_stride", i64), ("scales", vp), ("y", vp), ("y_stride", i64)]


STRUCTS = {"cc1d_delta_params": DeltaParams, "cc1d_delta_bwd_params": DeltaBwdParams, "cc1d_delta_step_params": DeltaStepParams,
           "cc1d_norm_params": NormParams, "cc1d_norm_bwd_params": NormBwdParams, "cc1d_dequantize_params": DequantizeParams}


def put(p, name, t, *axes):
    """A tensor's address and the strides of its leading dimensions."""
    setattr(p, name, _ptr(t))
    for i, a in enumerate(axes):
        setattr(p, "%s_stride_%s" % (name, a), t.stride(i))


def delta_params(q, k, v, g, beta, out, scale=1.0):
    p = DeltaParams()
    p.batch, p.seqlen, p.heads, p.dim_k = q.shape
    p.v_heads, p.dim_v = v.shape[2:]
    p.sequences = p.batch
    p.x_dtype, p.g_dtype, p.beta_dtype, p.scale = DTYPES[q.dtype], DTYPES[g.dtype], DTYPES[beta.dtype], scale
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta), ("out", out)):
        put(p, name, t, "b", "l", "h")
    return p


def declare_mixer(lib):
    size = C.POINTER(C.c_size_t)
    for name, st in (("delta", DeltaParams), ("delta_bwd", DeltaBwdParams), ("delta_step", DeltaStepParams), ("norm", NormParams),
                     ("norm_bwd", NormBwdParams), ("dequantize", DequantizeParams)):
        getattr(lib, "cc1d_validate_" + name).argtypes = [C.POINTER(st)]
    for name, st in (("delta", DeltaParams), ("delta_bwd", DeltaBwdParams), ("norm_bwd", NormBwdParams)):
        getattr(lib, "cc1d_%s_workspace_bytes" % name).argtypes = [C.POINTER(st), size]
    lib.cc1d_delta_saved_bytes.argtypes = [C.POINTER(DeltaParams), size]
    for name, st in (("delta_fwd", DeltaParams), ("delta_bwd", DeltaBwdParams), ("norm_bwd", NormBwdParams)):
        getattr(lib, "cc1d_" + name).argtypes = [C.POINTER(st), vp, C.c_size_t, vp]
    for name, st in (("delta_step", DeltaStepParams), ("norm_fwd", NormParams), ("dequantize_rows", DequantizeParams)):
        getattr(lib, "cc1d_" + name).argtypes = [C.POINTER(st), vp]
    return lib
