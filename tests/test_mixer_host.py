"""Host-only checks of the mixer's operators (no GPU, no kernel launch): the C ABI of include/cc1d_mixer.h exports what it
declares, its structs have the sizes of their ctypes mirror, every validation path returns its status, sizes of workspaces;
the plain statements of the operators against the formulas written out; and no host path in the public functions."""
import ctypes as C
import os
import re
import subprocess
import tempfile

import pytest
import torch

import cabi
import cabi_mixer as mixer

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cc1d_mixer.h")
OK, E_NULL, E_DTYPE, E_SHAPE, E_WS, E_TOO_LARGE, E_HEADS, E_HEAD_DIM, E_ROW = 0, -1, -2, -4, -13, -16, -21, -22, -23


@pytest.fixture(scope="module")
def lib(cc1d_lib):
    return mixer.declare_mixer(cabi.declare(cc1d_lib))


def test_every_declared_symbol_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(cc1d_[a-z_0-9]+)\s*\(", text))
    assert len(names) >= 16 and {"cc1d_delta_fwd", "cc1d_delta_bwd", "cc1d_delta_step", "cc1d_norm_fwd", "cc1d_norm_bwd", "cc1d_dequantize_rows"} <= names
    for n in names:
        assert hasattr(lib, n), n


def test_struct_sizes_match_the_header():
    names = list(mixer.STRUCTS)
    src = '#include <stdio.h>\n#include "cc1d_mixer.h"\nint main(void){' + "".join('printf("%%zu\\n", sizeof(%s));' % n for n in names) + "return 0;}"
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.dirname(HEADER), os.path.join(d, "s.c"), "-o",
                        os.path.join(d, "s")], check=True)
        sizes = [int(v) for v in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True).stdout.split()]
    assert sizes == [C.sizeof(mixer.STRUCTS[n]) for n in names]


def test_strerror_texts(lib):
    assert b"multiple of the number of key heads" in lib.cc1d_strerror(E_HEADS)
    assert b"dim_k <= 256" in lib.cc1d_strerror(E_HEAD_DIM)
    assert b"element size" in lib.cc1d_strerror(E_ROW)


def delta(batch=2, seqlen=100, heads=2, v_heads=4, dim_k=16, dim_v=24, dtype=torch.bfloat16):
    q = torch.zeros(batch, seqlen, heads, dim_k, dtype=dtype)
    v = torch.zeros(batch, seqlen, v_heads, dim_v, dtype=dtype)
    g = torch.zeros(batch, seqlen, v_heads)
    out = torch.empty_like(v)
    return mixer.delta_params(q, q, v, g, g, out), (q, v, g, out)


def test_validate_delta_paths(lib):
    v = lib.cc1d_validate_delta
    assert v(None) == E_NULL
    p, keep = delta()
    assert v(p) == OK
    for field, value, want in (("x_dtype", 7, E_DTYPE), ("g_dtype", -1, E_DTYPE), ("beta_dtype", 3, E_DTYPE), ("batch", -1, E_SHAPE), ("seqlen", -2, E_SHAPE),
                               ("heads", 0, E_SHAPE), ("v_heads", 3, E_HEADS), ("dim_k", 0, E_HEAD_DIM), ("dim_k", 257, E_HEAD_DIM),
                               ("dim_v", 0, E_HEAD_DIM), ("dim_v", 513, E_HEAD_DIM), ("sequences", 3, E_SHAPE), ("q", None, E_NULL), ("k", None, E_NULL),
                               ("v", None, E_NULL), ("g", None, E_NULL), ("beta", None, E_NULL), ("out", None, E_NULL)):
        p, keep = delta()
        setattr(p, field, value)
        assert v(p) == want, (field, value)
    p, keep = delta()
    p.q += 1
    assert v(p) == E_ROW
    p, keep = delta()
    p.saved = 8
    assert v(p) == E_WS
    cu = torch.tensor([0, 40, 100], dtype=torch.int32)
    p, keep = delta(batch=1)
    p.cu_seqlens, p.sequences = cu.data_ptr(), 2
    assert v(p) == OK
    p, keep = delta()                                    # packed sequences come in a batch of one
    p.cu_seqlens, p.sequences = cu.data_ptr(), 2
    assert v(p) == E_SHAPE
    p, keep = delta(batch=1)                             # tokens that belong to no sequence need one that could clear them
    p.cu_seqlens, p.sequences = cu.data_ptr(), 0
    assert v(p) == E_SHAPE
    p.seqlen = 0
    assert v(p) == OK
    p, keep = delta(batch=0)
    p.q = p.k = p.v = p.g = p.beta = p.out = None
    assert v(p) == OK and lib.cc1d_delta_fwd(p, None, 0, None) == OK


def test_workspaces_of_the_gated_delta_rule(lib):
    """Sizes grow with the sequence, short sequences need none, and a missing or small workspace is refused before a launch."""
    n, more, saved = C.c_size_t(), C.c_size_t(), C.c_size_t()
    p, keep = delta(seqlen=1)
    assert lib.cc1d_delta_workspace_bytes(p, C.byref(n)) == OK and n.value == 0
    p, keep = delta(seqlen=640)
    assert lib.cc1d_delta_workspace_bytes(p, C.byref(n)) == OK and n.value > 0
    assert lib.cc1d_delta_fwd(p, None, n, None) == E_WS
    assert lib.cc1d_delta_fwd(p, C.c_void_p(256), n.value - 1, None) == E_WS
    assert lib.cc1d_delta_fwd(p, C.c_void_p(8), n, None) == E_WS
    q, keep2 = delta(seqlen=1280)
    assert lib.cc1d_delta_workspace_bytes(q, C.byref(more)) == OK and more.value > 1.9 * n.value
    # what the backward needs: a state and 64 rows, in fp32, for every chunk and value head
    assert lib.cc1d_delta_saved_bytes(p, C.byref(saved)) == OK
    assert saved.value >= 2 * 10 * 4 * (16 + 64) * 24 * 4
    assert lib.cc1d_delta_workspace_bytes(p, None) == E_NULL


def test_validate_delta_bwd_paths(lib):
    v = lib.cc1d_validate_delta_bwd

    def block():
        p, keep = delta()
        b = mixer.DeltaBwdParams()
        b.fwd = p
        b.fwd.saved, b.fwd.out = 256, None
        for name, t in (("dout", keep[3]), ("dq", keep[0]), ("dk", keep[0]), ("dv", keep[1])):
            mixer.put(b, name, t, "b", "l", "h")
        b.dg = b.dbeta = keep[2].data_ptr()
        return b, keep
    assert v(None) == E_NULL
    b, keep = block()
    assert v(b) == OK
    n = C.c_size_t()
    assert lib.cc1d_delta_bwd_workspace_bytes(b, C.byref(n)) == OK and n.value > 0
    assert lib.cc1d_delta_bwd(b, None, 0, None) == E_WS
    for field in ("dout", "dq", "dk", "dv", "dg", "dbeta"):
        b, keep = block()
        setattr(b, field, None)
        assert v(b) == E_NULL, field
    b, keep = block()
    b.fwd.saved = None
    assert v(b) == E_NULL
    b, keep = block()
    b.dq += 1
    assert v(b) == E_ROW
    b, keep = block()
    b.dout_stride_l = 1 << 24                            # 2^25 bytes between tokens
    assert lib.cc1d_delta_bwd_workspace_bytes(b, C.byref(n)) == E_TOO_LARGE


def test_validate_delta_step_paths(lib):
    v = lib.cc1d_validate_delta_step

    def block():
        q, x, g, s = torch.zeros(2, 1, 2, 16), torch.zeros(2, 1, 4, 24), torch.zeros(2, 1, 4), torch.zeros(2, 4, 16, 24)
        p = mixer.DeltaStepParams()
        p.batch, p.seqlen, p.heads, p.v_heads, p.dim_k, p.dim_v, p.state_slots = 2, 1, 2, 4, 16, 24, 2
        for name, t in (("q", q), ("k", q), ("v", x), ("g", g), ("beta", g), ("out", x)):
            mixer.put(p, name, t, "b", "l", "h")
        mixer.put(p, "state", s, "n", "h", "k")
        return p, (q, x, g, s)
    assert v(None) == E_NULL
    p, keep = block()
    assert v(p) == OK
    for field, value, want in (("state_slots", 3, E_SHAPE), ("state_slots", -1, E_SHAPE), ("v_heads", 5, E_HEADS), ("dim_v", 600, E_HEAD_DIM), ("x_dtype", 9, E_DTYPE),
                               ("state", None, E_NULL), ("out", None, E_NULL), ("beta", None, E_NULL)):
        p, keep = block()
        setattr(p, field, value)
        assert v(p) == want, field
    p, keep = block()
    p.state_indices, p.state_slots = 256, 7              # any number of slots with indices
    assert v(p) == OK
    p, keep = block()
    p.state += 2
    assert v(p) == E_ROW
    p, keep = block()
    p.batch, p.state_slots = 0, 0
    assert lib.cc1d_delta_step(p, None) == OK


def norm(cls=mixer.NormParams, rows=3, dim=16, residual=True):
    x, w = torch.zeros(rows, dim), torch.zeros(dim)
    p = cls()
    p.rows, p.dim, p.eps = rows, dim, 1e-6
    for name in ("x", "y", "h", "residual", "dy", "dh", "dx", "dresidual"):
        if hasattr(p, name) and (residual or name not in ("residual", "h")):
            setattr(p, name, x.data_ptr())
            setattr(p, name + "_stride", dim)
    p.weight = w.data_ptr()
    if hasattr(p, "dweight"):
        p.dweight = w.data_ptr()
    return p, (x, w)


def test_validate_norm_paths(lib):
    v = lib.cc1d_validate_norm
    assert v(None) == E_NULL
    p, keep = norm()
    assert v(p) == OK
    p, keep = norm(residual=False)
    assert v(p) == OK
    for field, value, want in (("x_dtype", 4, E_DTYPE), ("r_dtype", 1, E_DTYPE), ("w_dtype", 2, E_DTYPE), ("rows", -1, E_SHAPE), ("dim", -1, E_SHAPE), ("x", None, E_NULL),
                               ("weight", None, E_NULL), ("y", None, E_NULL), ("h", None, E_NULL), ("residual", None, E_NULL)):
        p, keep = norm()
        setattr(p, field, value)
        assert v(p) == want, field
    p, keep = norm()
    p.y8 = 256                                           # one output, not two
    assert v(p) == E_NULL
    p, keep = norm()
    p.y, p.y8 = None, 256
    assert v(p) == E_NULL                                # and its scales
    p.scales = 256
    assert v(p) == OK
    p, keep = norm()
    p.x += 2
    assert v(p) == E_ROW
    p, keep = norm(rows=0)
    p.x = p.y = p.weight = None
    assert v(p) == OK and lib.cc1d_norm_fwd(p, None) == OK


def test_validate_norm_bwd_and_dequantize_paths(lib):
    v = lib.cc1d_validate_norm_bwd
    n = C.c_size_t()
    p, keep = norm(mixer.NormBwdParams)
    assert v(None) == E_NULL and v(p) == OK
    assert lib.cc1d_norm_bwd_workspace_bytes(p, C.byref(n)) == OK and n.value >= 16 * 4
    assert lib.cc1d_norm_bwd(p, None, 0, None) == E_WS
    for field, value, want in (("h", None, E_NULL), ("dy", None, E_NULL), ("weight", None, E_NULL), ("dweight", None, E_NULL), ("r_dtype", 2, E_DTYPE), ("rows", -1, E_SHAPE)):
        p, keep = norm(mixer.NormBwdParams)
        setattr(p, field, value)
        assert v(p) == want, field
    d = mixer.DequantizeParams()
    d.rows, d.dim, d.y8, d.scales, d.y = 2, 8, 256, 256, 256
    assert lib.cc1d_validate_dequantize(d) == OK and lib.cc1d_validate_dequantize(None) == E_NULL
    d.y += 2
    assert lib.cc1d_validate_dequantize(d) == E_ROW
    d.y = None
    assert lib.cc1d_validate_dequantize(d) == E_NULL
    d.rows = 0
    assert lib.cc1d_dequantize_rows(d, None) == OK


def test_plain_gated_delta_rule_is_the_recurrence(pkg):
    """Every element by loops over scalars' vectors, in 64 bits: 1e-13 of values near one, sums of a few terms."""
    from causal_conv1d.gated_delta_rule import gated_delta_rule_ref
    r = torch.Generator().manual_seed(3)
    B, L, H, G, K, V = 2, 5, 2, 2, 3, 4
    q, k = (torch.randn(B, L, H, K, generator=r, dtype=torch.float64) for _ in range(2))
    v = torch.randn(B, L, H * G, V, generator=r, dtype=torch.float64)
    g, beta = -torch.rand(B, L, H * G, generator=r, dtype=torch.float64), torch.rand(B, L, H * G, generator=r, dtype=torch.float64)
    s0 = torch.randn(B, H * G, K, V, generator=r, dtype=torch.float64)
    for l2norm in (False, True):
        out, final = gated_delta_rule_ref(q, k, v, g, beta, scale=0.7, initial_states=s0, return_final_states=True, qk_l2norm=l2norm)
        for b in range(B):
            for h in range(H * G):
                s = s0[b, h].clone()
                for t in range(L):
                    kt, qt = k[b, t, h // G], q[b, t, h // G]
                    if l2norm:
                        kt, qt = kt / (kt.dot(kt) + 1e-6).sqrt(), qt / (qt.dot(qt) + 1e-6).sqrt()
                    d = g[b, t, h].exp() * s
                    s = d + torch.outer(kt, beta[b, t, h] * (v[b, t, h] - d.T @ kt))
                    assert (out[b, t, h] - 0.7 * (s.T @ qt)).abs().max() < 1e-13
                assert (final[b, h] - s).abs().max() < 1e-13


def test_plain_forms_have_their_gradients(pkg):
    from causal_conv1d.gated_delta_rule import gated_delta_rule_ref
    from causal_conv1d.rms_norm import rms_norm_ref
    r = torch.Generator().manual_seed(4)

    def rand(*shape):
        return torch.randn(*shape, generator=r, dtype=torch.float64).requires_grad_()
    args = rand(1, 3, 1, 2), rand(1, 3, 1, 2), rand(1, 3, 2, 2), rand(1, 3, 2), rand(1, 3, 2), rand(1, 2, 2, 2)
    assert torch.autograd.gradcheck(lambda q, k, v, g, b, s: gated_delta_rule_ref(q, k, v, g, b, initial_states=s, return_final_states=True, qk_l2norm=True), args)
    assert torch.autograd.gradcheck(lambda x, w, h: rms_norm_ref(x, w, residual=h, eps=1e-3), (rand(2, 5), rand(5), rand(2, 5)))


def test_no_host_path(pkg):
    q, v, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    for call in (lambda: pkg.gated_delta_rule_fn(q, q, v, g, g), lambda: pkg.gated_delta_rule_update(q[:, 0], q[:, 0], v[:, 0], g[:, 0], g[:, 0], torch.zeros(1, 2, 8, 8)),
                 lambda: pkg.rms_norm_fn(v, torch.ones(8)), lambda: pkg.rms_norm_quant_fn(v, torch.ones(8))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_shapes_without_a_device(pkg):
    """The ops' shapes and types on the meta device, as torch.compile asks for them."""
    q, v = torch.empty(2, 9, 2, 16, device="meta", dtype=torch.bfloat16), torch.empty(2, 9, 4, 24, device="meta", dtype=torch.bfloat16)
    g = torch.empty(2, 9, 4, device="meta")
    out = torch.ops.DaoAILab._gated_delta_rule_fwd_cpp(q, q, v, g, g, None, None, None, 0.25, False)
    assert out.shape == v.shape and out.dtype == v.dtype
    x, w = torch.empty(3, 5, 16, device="meta", dtype=torch.bfloat16), torch.empty(16, device="meta")
    y, h = torch.ops.DaoAILab._rms_norm_fwd_cpp(x, w, torch.empty(3, 5, 16, device="meta"), 1e-5)
    assert y.shape == x.shape and y.dtype == x.dtype and h.dtype == torch.float32
    y8, scales, _ = torch.ops.DaoAILab._rms_norm_quant_cpp(x, w, None, 1e-5)
    assert y8.shape == x.shape and y8.dtype == torch.float8_e4m3fn and scales.shape == x.shape[:-1]
