"""Sizes of linear attention's calls (no GPU, no kernel launch): what goes by tokens because no grid of segments takes it, and what workspaces hold."""
import ctypes as C

import pytest
import torch

import cabi
import cabi_linear as linear
import cabi_mixer as mixer
from test_linear_host import E_TOO_LARGE, OK, block, bwd_block

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


def sizes(lib, batch, seqlen, sequences, v_heads, dim_k, dim_v, dtype, initial, heads=1):
    """Bytes of `saved`, and of the workspaces of the forward that leaves it and of the backward."""
    p, keep = call(seqlen, v_heads, dim_k, dim_v, dtype, sequences, batch, heads, states=False)
    p.initial_states = 256 if initial else None
    n = [C.c_size_t() for _ in range(3)]
    assert lib.cc1d_linear_saved_bytes(p, C.byref(n[0])) == OK
    p.saved = 256
    assert lib.cc1d_linear_workspace_bytes(p, C.byref(n[1])) == OK
    b, more = bwd_block()
    b.fwd, b.fwd.out = p, None
    b.dinitial_states = 256 if initial else None
    assert lib.cc1d_linear_bwd_workspace_bytes(b, C.byref(n[2])) == OK
    return [v.value for v in n]


@pytest.mark.parametrize("dtype", [B16, F32])
def test_sequences_without_states_take_no_room_for_them(lib, dtype):
    """What the tensors of a training call take bounds what is kept beside them: a state every 256 tokens of 128 x 64 elements, 6 bytes each in `saved`, 4 and at
    most 12 in a workspace, and 20 bytes a token and value head for the gates' sums.  Not a state for each of a thousand sequences of four tokens."""
    state = 128 * 64 * 80
    saved, fwd, bwd = sizes(lib, 1, 4096, 1000, 80, 128, 64, dtype, False)
    assert saved <= 256 + 16 * 6 * state and fwd <= 16 * 10 * state + 2 ** 20 and bwd <= 16 * 16 * state + 4096 * 80 * 20 + 2 ** 22
    saved, fwd, bwd = sizes(lib, 64, 256, None, 80, 128, 64, dtype, False, heads=80)   # one segment each: none at all
    assert saved <= 256 and fwd == 0 and bwd <= 64 * 256 * 80 * 24 + 2 ** 12
    saved, fwd, bwd = sizes(lib, 64, 300, None, 80, 128, 64, dtype, False)             # two: one between them
    assert saved <= 256 + 64 * 6 * state and fwd <= 64 * 10 * state + 2 ** 20


@pytest.mark.parametrize("dtype", [B16, F32])
def test_states_that_are_there_have_room(lib, dtype):
    state = 128 * 64 * 80
    saved, fwd, bwd = sizes(lib, 1, 4096, 1000, 80, 128, 64, dtype, True)
    assert saved >= 1000 * 6 * state and fwd >= 1000 * 4 * state and bwd >= 1000 * 4 * state
    saved, fwd, bwd = sizes(lib, 4, 2048, None, 80, 128, 64, dtype, False)
    assert saved >= 28 * 6 * state and fwd >= 28 * 8 * state and bwd >= 28 * 14 * state


@pytest.mark.parametrize("seqlen,batch,sequences", [(1, 3, None), (256, 2, None), (257, 2, None), (0, 2, None), (700, 1, 5), (256, 1, 2), (0, 1, 3)])
@pytest.mark.parametrize("initial", [True, False])
def test_saved_bytes_of_a_traced_call_with_states(lib, pkg, seqlen, batch, sequences, initial):
    q, v, g = torch.empty(batch, seqlen, 1, 40), torch.empty(batch, seqlen, 2, 72), torch.empty(batch, seqlen, 2)
    cu = None if sequences is None else torch.zeros(sequences + 1, dtype=torch.int32)
    init = torch.empty(sequences or batch, 2, 40, 72) if initial else None
    p = mixer.delta_params(q, q, v, g, g, v)
    if cu is not None:
        p.cu_seqlens, p.sequences = cu.data_ptr(), sequences
    if initial:
        p.initial_states = init.data_ptr()
    n = C.c_size_t()
    assert lib.cc1d_linear_saved_bytes(p, C.byref(n)) == OK
    meta = [None if t is None else t.to("meta") for t in (q, q, v, g, g, init, cu)]
    out, saved = torch.ops.DaoAILab._linear_attention_fwd_save_cpp(*meta, None, 1.0)
    assert tuple(saved.shape) == (n.value,)
