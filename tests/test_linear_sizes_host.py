"""Sizes of linear attention's calls (no GPU, no kernel launch): what goes by tokens because no grid of segments takes it, and what workspaces hold."""
import ctypes as C

import pytest
import torch

import cabi
import cabi_linear as linear
import cabi_mixer as mixer
from test_linear_host import E_TOO_LARGE, OK, block

B16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib(cc1d_lib):
    return linear.declare_linear(mixer.declare_mixer(cabi.declare(cc1d_lib)))


def call(seqlen, v_heads, dim_k, dim_v, dtype=B16, sequences=None, batch=1, heads=1, states=True):
    """A block of these sizes over small tensors: nothing is launched."""
    p, keep = block(1, 2, 1, 1, dim_k, dim_v, dtype)
    p.batch, p.sequences, p.seqlen, p.heads, p.v_heads = batch, batch, seqlen, heads, v_heads
    if sequences is not None:
        cu = torch.zeros(2, dtype=torch.int32)
        p.cu_seqlens, p.sequences, keep = cu.data_ptr(), sequences, keep + (cu,)
    if states:
        p.final_states = 256                             # (without states a sequence of one segment needs no workspace)
    return p, keep


@pytest.mark.parametrize("args,kw", [((60000 * 50, 80, 128, 64), {"sequences": 60000}), ((1 << 22, 160, 32, 32), {}), ((4096, 1200, 16, 16), {"batch": 512}),
                                     ((1 << 22, 200, 64, 64, F32), {"sequences": 20}), ((1 << 22, 300, 32, 32), {"sequences": 1 << 21})])
def test_more_segments_than_a_grid(lib, args, kw):
    """The token kernel takes them, without a workspace; what a backward needs of the forward does not fit, and is refused."""
    n = C.c_size_t(7)
    p, keep = call(*args, **kw)
    assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK and n.value == 0
    p.saved = 256
    assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == E_TOO_LARGE


@pytest.mark.parametrize("dtype,dim", [(B16, 100), (F32, 50), (B16, 511)])
def test_copies_too_wide(lib, dtype, dim):
    """Rows that would have to be copied, 2^23 bytes and more of them to a token."""
    n = C.c_size_t(7)
    heads = (1 << 23) // (max((dim + 7) // 8 * 8, 128) * (2 if dtype == B16 else 4))       # of the wider of k and v
    for v_heads, fits in ((heads - 1, True), (heads + 1, False)):
        p, keep = call(300, v_heads, 128, dim, dtype)
        assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK and (n.value > 0) == fits
        p.saved = 256
        assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == (OK if fits else E_TOO_LARGE)


def test_border_of_a_grid(lib):
    """Slots of 256 tokens times value heads: 2^21 - 8 are too many."""
    n = C.c_size_t()
    for slots, fits in ((2 ** 21 - 9, True), (2 ** 21 - 8, False)):
        p, keep = call(256 * slots, 1, 16, 16)
        assert lib.cc1d_linear_workspace_bytes(p, C.byref(n)) == OK and (n.value > 0) == fits
