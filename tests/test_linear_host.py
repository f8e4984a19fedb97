"""Host-only checks of linear attention and the layer norm (no GPU, no kernel launch): the C ABI's blocks, refusals, workspaces and ways of a
call, the plain statements against the formulas written out, and no host path in the public functions."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import cabi
import cabi_linear as linear
import cabi_mixer as mixer

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cc1d_mixer.h")
OK, E_NULL, E_DTYPE, E_SHAPE, E_WS, E_TOO_LARGE, E_HEADS, E_HEAD_DIM, E_ROW, E_OPTION = 0, -1, -2, -4, -13, -16, -21, -22, -23, -24


@pytest.fixture(scope="module")
def lib(cc1d_lib):
    return linear.declare_linear(mixer.declare_mixer(cabi.declare(cc1d_lib)))


def test_struct_sizes_match_the_header():
    names = list(linear.STRUCTS)
    src = '#include <stdio.h>\n#include "cc1d_mixer.h"\nint main(void){' + "".join('printf("%%zu\\n", sizeof(%s));' % n for n in names) + "return 0;}"
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.dirname(HEADER), os.path.join(d, "s.c"), "-o",
                        os.path.join(d, "s")], check=True)
        sizes = [int(v) for v in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True).stdout.split()]
    assert sizes == [C.sizeof(linear.STRUCTS[n]) for n in names]


def test_strerror_text(lib):
    assert lib.cc1d_strerror(E_OPTION) != lib.cc1d_strerror(-999) and b"option" in lib.cc1d_strerror(E_OPTION).lower()


def block(batch=2, seqlen=100, heads=2, v_heads=4, dim_k=16, dim_v=24, dtype=torch.bfloat16, beta=True):
    q = torch.zeros(batch, seqlen, heads, dim_k, dtype=dtype)
    v = torch.zeros(batch, seqlen, v_heads, dim_v, dtype=dtype)
    g = torch.zeros(batch, seqlen, v_heads)
    out = torch.empty_like(v)
    p = mixer.delta_params(q, q, v, g, g, out)
    if not beta:
        p.beta = None
    return p, (q, v, g, out)


@pytest.mark.parametrize("beta", [True, False])
def test_validate_linear_paths(lib, beta):
    v = lib.cc1d_validate_linear
    assert v(None) == E_NULL
    p, keep = block(beta=beta)
    assert v(p) == OK
    for field, value, want in (("x_dtype", 7, E_DTYPE), ("g_dtype", -1, E_DTYPE), ("batch", -1, E_SHAPE), ("seqlen", -2, E_SHAPE), ("heads", 0, E_SHAPE),
                               ("v_heads", 3, E_HEADS), ("dim_k", 0, E_HEAD_DIM), ("dim_k", 257, E_HEAD_DIM), ("dim_v", 513, E_HEAD_DIM), ("sequences", 3, E_SHAPE),
                               ("q", None, E_NULL), ("k", None, E_NULL), ("v", None, E_NULL), ("g", None, E_NULL), ("out", None, E_NULL), ("qk_l2norm", 1, E_OPTION)):
        p, keep = block(beta=beta)
        setattr(p, field, value)
        assert v(p) == want, (field, value)
        assert lib.cc1d_linear_fwd(p, None, 0, None) == want
    p, keep = block(beta=beta)
    p.q += 1
    assert v(p) == E_ROW
    p, keep = block(beta=beta)
    p.beta_dtype = 5
    assert v(p) == (E_DTYPE if beta else OK)             # nothing reads the type of a beta that is not there
    p, keep = block(batch=0, beta=beta)
    p.q = p.k = p.v = p.g = p.beta = p.out = None
    assert v(p) == OK and lib.cc1d_linear_fwd(p, None, 0, None) == OK


def test_workspaces(lib):
    n, more, saved = C.c_size_t(), C.c_size_t(), C.c_size_t()
    p, keep = block(seqlen=1)
    assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK and n.value == 0
    p, keep = block(seqlen=1024)
    assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK and n.value > 0
    assert lib.cc1d_linear_fwd(p, None, n, None) == E_WS
    assert lib.cc1d_linear_fwd(p, C.c_void_p(256), n.value - 1, None) == E_WS
    assert lib.cc1d_linear_fwd(p, C.c_void_p(8), n, None) == E_WS
    q, keep2 = block(seqlen=2048)
    assert lib.cc1d_linear_workspace_bytes(q, C.byref(more)) == OK and more.value > 1.9 * n.value
    # a state for every 256 tokens and value head, 6 bytes an element
    assert lib.cc1d_linear_saved_bytes(p, C.byref(saved)) == OK
    assert saved.value >= 2 * 4 * 4 * 16 * 24 * 6
    assert lib.cc1d_linear_workspace_bytes(p, None) == E_NULL and lib.cc1d_linear_saved_bytes(p, None) == E_NULL and lib.cc1d_linear_saved_bytes(None, C.byref(n)) == E_NULL


def bwd_block(beta=True, seqlen=100):
    p, keep = block(beta=beta, seqlen=seqlen)
    b = mixer.DeltaBwdParams()
    b.fwd = p
    b.fwd.saved, b.fwd.out = 256, None
    for name, t in (("dout", keep[3]), ("dq", keep[0]), ("dk", keep[0]), ("dv", keep[1])):
        mixer.put(b, name, t, "b", "l", "h")
    b.dg = keep[2].data_ptr()
    b.dbeta = keep[2].data_ptr() if beta else None
    return b, keep


@pytest.mark.parametrize("beta", [True, False])
def test_validate_linear_bwd_paths(lib, beta):
    v = lib.cc1d_validate_linear_bwd
    assert v(None) == E_NULL
    b, keep = bwd_block(beta)
    assert v(b) == OK
    n = C.c_size_t()
    assert lib.cc1d_linear_bwd_workspace_bytes(b, C.byref(n)) == OK and n.value > 0
    assert lib.cc1d_linear_bwd(b, None, 0, None) == E_WS
    for field in ("dout", "dq", "dk", "dv", "dg") + (("dbeta",) if beta else ()):
        b, keep = bwd_block(beta)
        setattr(b, field, None)
        assert v(b) == E_NULL, field
    b, keep = bwd_block(beta)
    b.fwd.saved = None
    assert v(b) == E_NULL
    b, keep = bwd_block(beta)
    b.fwd.qk_l2norm = 1
    assert v(b) == E_OPTION
    for name in ("dout", "dq", "dk", "dv"):
        b, keep = bwd_block(beta)
        setattr(b, name + "_stride_l", 1 << 22)          # 2^23 bytes between tokens
        assert lib.cc1d_linear_bwd_workspace_bytes(b, C.byref(n)) == E_TOO_LARGE, name


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_tokens_far_apart(lib, name):
    """Rows of a segment are reached with 32 bits: tokens 2^23 bytes apart go one by one, without a workspace; a training call, which cannot, is refused."""
    n = C.c_size_t()
    for stride, seqlen, far in (((1 << 22) - 1, 300, False), (1 << 22, 300, True), (-16, 300, True), (1 << 30, 1, False)):
        p, keep = block(seqlen=seqlen)
        setattr(p, name + "_stride_l", stride)
        assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK and (n.value == 0) == (far or seqlen == 1)
        p.saved = 256
        assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == (E_TOO_LARGE if far else OK)


def test_ways_of_a_call(lib):
    """By tokens (no workspace) or by segments, by the number of tokens, of states and the type; packed sequences that are short on average, but may hold a long
    one, each by its own length."""
    n = C.c_size_t()

    def wants(batch, seqlen, v_heads, dim, dtype, sequences=None):
        p, keep = block(batch, seqlen, 1, v_heads, dim, dim, dtype)
        cu = None
        if sequences is not None:
            cu = torch.zeros(sequences + 1, dtype=torch.int32)
            p.cu_seqlens, p.sequences = cu.data_ptr(), sequences
        p.final_states = 256                             # (without states a sequence of one segment needs no workspace either)
        assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK
        return n.value > 0
    b16, f32 = torch.bfloat16, torch.float32
    for args, want in (((1, 15, 4, 64, b16), False), ((1, 16, 4, 64, b16), True), ((1, 21, 4, 64, f32), False), ((1, 22, 4, 64, f32), True),
                       ((16, 49, 64, 128, b16), False), ((16, 50, 64, 128, b16), True), ((16, 169, 64, 128, f32), False), ((16, 170, 64, 128, f32), True),
                       ((32, 5000, 64, 32, f32), False), ((1, 160, 4, 64, b16, 10), True), ((1, 159, 4, 64, b16, 10), False), ((1, 511, 4, 64, b16, 40), False),
                       ((1, 512, 4, 64, b16, 40), True), ((1, 512, 4, 64, f32, 40), True), ((1, 2000, 2048, 32, f32, 40), False)):
        assert wants(*args) == want, args


@pytest.mark.parametrize("beta", [True, False])
def test_validate_linear_step_paths(lib, beta):
    v = lib.cc1d_validate_linear_step

    def step():
        q, x, g, s = torch.zeros(2, 1, 2, 16), torch.zeros(2, 1, 4, 24), torch.zeros(2, 1, 4), torch.zeros(2, 4, 16, 24)
        p = mixer.DeltaStepParams()
        p.batch, p.seqlen, p.heads, p.v_heads, p.dim_k, p.dim_v, p.state_slots = 2, 1, 2, 4, 16, 24, 2
        for name, t in (("q", q), ("k", q), ("v", x), ("g", g), ("out", x)) + ((("beta", g),) if beta else ()):
            mixer.put(p, name, t, "b", "l", "h")
        mixer.put(p, "state", s, "n", "h", "k")
        return p, (q, x, g, s)
    assert v(None) == E_NULL
    p, keep = step()
    assert v(p) == OK
    for field, value, want in (("state_slots", 3, E_SHAPE), ("v_heads", 5, E_HEADS), ("dim_v", 600, E_HEAD_DIM), ("x_dtype", 9, E_DTYPE), ("state", None, E_NULL),
                               ("out", None, E_NULL), ("qk_l2norm", 1, E_OPTION)):
        p, keep = step()
        setattr(p, field, value)
        assert v(p) == want and lib.cc1d_linear_step(p, None) == want, field
    p, keep = step()
    p.batch, p.state_slots = 0, 0
    assert lib.cc1d_linear_step(p, None) == OK


def norm(cls=linear.LayerNormParams, rows=3, dim=16, residual=True):
    x, w = torch.zeros(rows, dim), torch.zeros(dim)
    p = cls()
    p.rows, p.dim = rows, dim
    for name, kind in cls._fields_:
        if name in ("x", "y", "h", "residual", "dy", "dh", "dx", "dresidual") and (residual or name not in ("residual", "h")):
            setattr(p, name, x.data_ptr())
            setattr(p, name + "_stride", dim)
        if name in ("weight", "bias", "dweight", "dbias"):
            setattr(p, name, w.data_ptr())
    if cls is linear.LayerNormBwdParams:
        p.h, p.h_stride, p.stats = x.data_ptr(), dim, x.data_ptr()
    return p, (x, w)


def test_validate_layer_norm_paths(lib):
    v = lib.cc1d_validate_layer_norm
    assert v(None) == E_NULL
    for residual in (True, False):
        p, keep = norm(residual=residual)
        assert v(p) == OK
    for field, value, want in (("x_dtype", 4, E_DTYPE), ("r_dtype", 1, E_DTYPE), ("w_dtype", 2, E_DTYPE), ("rows", -1, E_SHAPE), ("dim", -1, E_SHAPE), ("x", None, E_NULL),
                               ("weight", None, E_NULL), ("y", None, E_NULL), ("h", None, E_NULL), ("residual", None, E_NULL), ("bias", None, OK),
                               ("stats", 4, E_ROW), ("stats", 8, OK), ("dim", 2 ** 31 - 1, E_TOO_LARGE)):
        p, keep = norm()
        setattr(p, field, value)
        assert v(p) == want, field
    p, keep = norm()
    p.bias += 2
    assert v(p) == E_ROW
    p, keep = norm(rows=0)
    p.x = p.y = p.weight = None
    assert v(p) == OK and lib.cc1d_layer_norm_fwd(p, None) == OK


def test_validate_layer_norm_bwd_paths(lib):
    v = lib.cc1d_validate_layer_norm_bwd
    n, one = C.c_size_t(), C.c_size_t()
    p, keep = norm(linear.LayerNormBwdParams)
    assert v(None) == E_NULL and v(p) == OK
    assert lib.cc1d_layer_norm_bwd_workspace_bytes(p, C.byref(n)) == OK and n.value >= 2 * 16 * 4
    assert lib.cc1d_layer_norm_bwd(p, None, 0, None) == E_WS
    p.dbias = None
    assert v(p) == OK and lib.cc1d_layer_norm_bwd_workspace_bytes(p, C.byref(one)) == OK and 2 * one.value == n.value
    for field, value, want in (("h", None, E_NULL), ("dy", None, E_NULL), ("weight", None, E_NULL), ("dweight", None, E_NULL), ("stats", None, E_NULL), ("r_dtype", 2, E_DTYPE),
                               ("rows", -1, E_SHAPE), ("dx", None, OK), ("dresidual", None, OK), ("dh", None, OK), ("dim", 2 ** 26 - 15, E_TOO_LARGE), ("dim", 2 ** 26 - 16, OK)):
        p, keep = norm(linear.LayerNormBwdParams)
        setattr(p, field, value)
        assert v(p) == want, field


@pytest.mark.parametrize("batch,seqlen,sequences", [(2, 100, None), (3, 0, None), (0, 70, None), (2, 257, None), (1, 100, 1), (1, 1000, 7), (1, 5, 90), (1, 0, 4), (1, 0, 0)])
@pytest.mark.parametrize("v_heads,dim_k,dim_v", [(4, 16, 24), (2, 33, 7), (0, 16, 16), (2, 128, 64), (2, 72, 128), (2, 40, 256), (2, 136, 64), (2, 64, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_bytes_of_a_traced_call(lib, pkg, batch, seqlen, sequences, v_heads, dim_k, dim_v, dtype):
    """The shape that the op has on the meta device is what the library asks for."""
    q = torch.empty(batch, seqlen, 2, dim_k, dtype=dtype)
    v = torch.empty(batch, seqlen, v_heads, dim_v, dtype=dtype)
    g = torch.empty(batch, seqlen, v_heads)
    cu = None if sequences is None else torch.zeros(sequences + 1, dtype=torch.int32)
    p = mixer.delta_params(q, q, v, g, g, v)
    if cu is not None:
        p.cu_seqlens, p.sequences = cu.data_ptr(), sequences
    n = C.c_size_t()
    assert lib.cc1d_linear_saved_bytes(p, C.byref(n)) == OK
    meta = [None if t is None else t.to("meta") for t in (q, q, v, g, g, None, cu)]
    out, saved = torch.ops.DaoAILab._linear_attention_fwd_save_cpp(*meta, None, 1.0)
    assert out.shape == v.shape and tuple(saved.shape) == (n.value,)


def test_plain_linear_attention_is_the_recurrence(pkg):
    """Every element by loops over scalars' vectors, in 64 bits: 1e-13 of values near one, sums of a few terms."""
    from causal_conv1d.linear_attention import linear_attention_ref
    r = torch.Generator().manual_seed(3)
    B, L, H, G, K, V = 2, 5, 2, 2, 3, 4
    q, k = (torch.randn(B, L, H, K, generator=r, dtype=torch.float64) for _ in range(2))
    v = torch.randn(B, L, H * G, V, generator=r, dtype=torch.float64)
    g, beta = -torch.rand(B, L, H * G, generator=r, dtype=torch.float64), torch.rand(B, L, H * G, generator=r, dtype=torch.float64)
    s0 = torch.randn(B, H * G, K, V, generator=r, dtype=torch.float64)
    for gates, weights in ((g, beta), (g, None), (g[0, 0], beta)):
        out, final = linear_attention_ref(q, k, v, gates, weights, scale=0.7, initial_states=s0, return_final_states=True)
        for b in range(B):
            for h in range(H * G):
                s = s0[b, h].clone()
                for t in range(L):
                    gt = gates[h] if gates.dim() == 1 else gates[b, t, h]
                    s = gt.exp() * s + torch.outer(k[b, t, h // G], v[b, t, h]) * (1 if weights is None else weights[b, t, h])
                    assert (out[b, t, h] - 0.7 * (s.T @ q[b, t, h // G])).abs().max() < 1e-13
                assert (final[b, h] - s).abs().max() < 1e-13
    assert torch.equal(linear_attention_ref(q, k, v, g, beta), linear_attention_ref(q, k, v, g, beta, scale=K ** -0.5))


def test_plain_layer_norm_is_the_formula(pkg):
    from causal_conv1d.layer_norm import layer_norm_ref
    r = torch.Generator().manual_seed(4)
    x, res, w, b = (torch.randn(*n, generator=r, dtype=torch.float64) for n in ((3, 7), (3, 7), (7,), (7,)))
    y, h = layer_norm_ref(x, w, b, residual=res, eps=1e-3)
    for i in range(3):
        z = x[i] + res[i]
        z0 = z - sum(z) / 7
        want = z0 / (sum(z0 * z0) / 7 + 1e-3).sqrt() * w + b
        assert (y[i] - want).abs().max() < 1e-14 and torch.equal(h[i], z)
    assert (layer_norm_ref(x, w, b) - torch.nn.functional.layer_norm(x, (7,), w, b, 1e-5)).abs().max() < 1e-14


def test_plain_forms_have_their_gradients(pkg):
    from causal_conv1d.layer_norm import layer_norm_ref
    from causal_conv1d.linear_attention import linear_attention_ref
    r = torch.Generator().manual_seed(4)

    def rand(*shape):
        return torch.randn(*shape, generator=r, dtype=torch.float64).requires_grad_()
    args = rand(1, 3, 1, 2), rand(1, 3, 1, 2), rand(1, 3, 2, 2), rand(1, 3, 2), rand(1, 3, 2), rand(1, 2, 2, 2)
    assert torch.autograd.gradcheck(lambda q, k, v, g, b, s: linear_attention_ref(q, k, v, g, b, initial_states=s, return_final_states=True), args)
    assert torch.autograd.gradcheck(lambda x, w, b, h: layer_norm_ref(x, w, b, residual=h, eps=1e-3), (rand(2, 5), rand(5), rand(5), rand(2, 5)))


def test_no_host_path(pkg):
    q, v, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    for call in (lambda: pkg.linear_attention_fn(q, q, v, g), lambda: pkg.linear_attention_fn(q, q, v, g[0, 0], beta=g),
                 lambda: pkg.linear_attention_update(q[:, 0], q[:, 0], v[:, 0], g[:, 0], torch.zeros(1, 2, 8, 8)),
                 lambda: pkg.layer_norm_fn(v, torch.ones(8)), lambda: pkg.layer_norm_fn(v, torch.ones(8), torch.ones(8), residual=v)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_shapes_without_a_device(pkg):
    """The ops' shapes and types on the meta device, as torch.compile asks for them."""
    q, v = torch.empty(2, 9, 2, 16, device="meta", dtype=torch.bfloat16), torch.empty(2, 9, 4, 24, device="meta", dtype=torch.bfloat16)
    g = torch.empty(2, 9, 4, device="meta")
    for beta in (g, None):
        out = torch.ops.DaoAILab._linear_attention_fwd_cpp(q, q, v, g, beta, None, None, None, 0.25)
        assert out.shape == v.shape and out.dtype == v.dtype
    x, w = torch.empty(3, 5, 16, device="meta", dtype=torch.bfloat16), torch.empty(16, device="meta")
    y, h, stats = torch.ops.DaoAILab._layer_norm_fwd_cpp(x, w, w, torch.empty(3, 5, 16, device="meta"), 1e-5, True)
    assert y.shape == x.shape and y.dtype == x.dtype and h.dtype == torch.float32 and stats.numel() == 30
