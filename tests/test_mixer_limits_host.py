"""Host-only: sizes that the norm's kernels could not count in 32 bits are refused before a launch."""
import ctypes as C

import pytest
import torch

import cabi
import cabi_mixer as mixer

OK, E_TOO_LARGE = 0, -16
LAST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib(cc1d_lib):
    return mixer.declare_mixer(cabi.declare(cc1d_lib))


def block(cls, dim, rows=2):
    p = cls()
    p.rows, p.dim = rows, dim
    for name, _ in cls._fields_:
        if name in ("x", "h", "residual", "y", "y8", "scales", "weight", "dy", "dh", "dx", "dresidual", "dweight"):
            setattr(p, name, 256)
    if cls is mixer.NormParams:
        p.y8 = p.scales = None
    return p


def test_rows_of_nearly_2_31_elements(lib):
    """Lanes step along a row by 8192 elements: the last step of a row longer than 2^31 - 1 - 8192 would leave 32 bits, come back
    negative and read in front of the row, without end."""
    n = C.c_size_t()
    for dim, want in ((LAST - 8192, OK), (LAST - 8191, E_TOO_LARGE), (LAST, E_TOO_LARGE)):
        p = block(mixer.NormParams, dim)
        assert lib.cc1d_validate_norm(p) == want, dim
        if want != OK:
            assert lib.cc1d_norm_fwd(p, None) == want
        assert lib.cc1d_validate_dequantize(block(mixer.DequantizeParams, dim)) == OK          # a vector a thread: no steps
        assert lib.cc1d_validate_norm(block(mixer.NormParams, dim, rows=0)) == OK
    for dim, want in ((2 ** 27 - 32, OK), (2 ** 27 - 31, E_TOO_LARGE), (LAST, E_TOO_LARGE)):   # dweight: 1024 threads for 32 columns, fewer than 2^32 in all
        p = block(mixer.NormBwdParams, dim)
        assert lib.cc1d_validate_norm_bwd(p) == want, dim
        if want != OK:
            assert lib.cc1d_norm_bwd_workspace_bytes(p, C.byref(n)) == want and lib.cc1d_norm_bwd(p, None, 0, None) == want


@pytest.mark.parametrize("batch,seqlen,sequences", [(2, 100, None), (1, 64, None), (3, 0, None), (0, 70, None), (2, 1, None), (1, 100, 1), (1, 1000, 7), (1, 64, 3),
                                                    (1, 5, 90), (1, 0, 1), (1, 0, 4), (1, 0, 0)])
@pytest.mark.parametrize("v_heads,dim_k,dim_v", [(4, 16, 24), (2, 33, 7), (0, 16, 16)])
def test_saved_bytes_of_a_traced_call(lib, pkg, batch, seqlen, sequences, v_heads, dim_k, dim_v):
    """The shape that the op has on the meta device is what the library asks for."""
    q = torch.empty(batch, seqlen, 2, dim_k)
    v = torch.empty(batch, seqlen, v_heads, dim_v)
    g = torch.empty(batch, seqlen, v_heads)
    cu = None if sequences is None else torch.zeros(sequences + 1, dtype=torch.int32)
    p = mixer.delta_params(q, q, v, g, g, v)
    if cu is not None:
        p.cu_seqlens, p.sequences = cu.data_ptr(), sequences
    n = C.c_size_t()
    assert lib.cc1d_delta_saved_bytes(p, C.byref(n)) == OK
    meta = [None if t is None else t.to("meta") for t in (q, q, v, g, g, None, cu)]
    out, saved = torch.ops.DaoAILab._gated_delta_rule_fwd_save_cpp(*meta, None, 1.0, False)
    assert out.shape == v.shape and tuple(saved.shape) == (n.value,)


def test_packed_sequences_are_not_all_judged_by_their_average(lib):
    """One long sequence among many short ones goes by chunks, for which there has to be a workspace; the token kernel alone takes
    none, and as long as the longest.  A few tokens, or a uniform batch of short sequences without a long one's worth of tokens, go by tokens."""
    n = C.c_size_t()
    for seqlen, sequences, v_heads, wanted in ((4224, 129, 32, True), (600, 300, 4, True), (255, 64, 32, False), (64, 16, 32, False)):
        q, v, g = torch.empty(1, seqlen, 1, 16), torch.empty(1, seqlen, v_heads, 16), torch.empty(1, seqlen, v_heads)
        p = mixer.delta_params(q.bfloat16(), q.bfloat16(), v.bfloat16(), g, g, v.bfloat16())
        p.x_dtype = 2
        cu = torch.zeros(sequences + 1, dtype=torch.int32)
        p.cu_seqlens, p.sequences = cu.data_ptr(), sequences
        p.heads = 1
        assert lib.cc1d_delta_workspace_bytes(p, C.byref(n)) == OK
        assert (n.value > 0) == wanted, (seqlen, sequences)


def test_one_token_has_no_distance_to_the_next(lib):
    """The stride between tokens is anything where there is one token a sequence: no reason to refuse a training call."""
    n = C.c_size_t()
    for seqlen, want in ((1, OK), (2, E_TOO_LARGE)):
        q, v, g = torch.empty(2, seqlen, 1, 16), torch.empty(2, seqlen, 2, 16), torch.empty(2, seqlen, 2)
        p = mixer.delta_params(q, q, v, g, g, v)
        p.saved = 256
        p.v_stride_l = p.out_stride_l = 1 << 23          # 2^25 bytes
        assert lib.cc1d_delta_workspace_bytes(p, C.byref(n)) == want
        b = mixer.DeltaBwdParams()
        b.fwd = p
        for name, t in (("dout", v), ("dq", q), ("dk", q), ("dv", v)):
            mixer.put(b, name, t, "b", "l", "h")
        b.dg = b.dbeta = g.data_ptr()
        b.dout_stride_l = b.dv_stride_l = 1 << 23
        assert lib.cc1d_delta_bwd_workspace_bytes(b, C.byref(n)) == want


def test_long_sequences_of_float32_among_many_heads(lib):
    """In float32 with many heads a sequence goes by chunks from 160 tokens on; a call that may hold one is looked at from 256 tokens on as well."""
    n = C.c_size_t()
    for seqlen, wanted in ((255, False), (256, True), (364, True)):
        q, v, g = torch.empty(1, seqlen, 1, 16), torch.empty(1, seqlen, 32, 16), torch.empty(1, seqlen, 32)
        p = mixer.delta_params(q, q, v, g, g, v)
        cu = torch.zeros(66, dtype=torch.int32)
        p.cu_seqlens, p.sequences = cu.data_ptr(), 65
        assert lib.cc1d_delta_workspace_bytes(p, C.byref(n)) == OK and (n.value > 0) == wanted, seqlen
