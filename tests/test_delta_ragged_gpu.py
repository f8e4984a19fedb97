"""gated_delta_rule_fn over packed sequences of very unequal lengths, where each goes by tokens or by chunks by its own.  Tolerances are
those of test_gated_delta_rule_gpu.py and test_gated_delta_rule_bwd_gpu.py."""
import pytest
import torch

from test_gated_delta_rule_bwd_gpu import NAMES, gradients, gradients64, near
from test_gated_delta_rule_gpu import close, make, recurrence

RAGGED = {
    "one_long": [1] * 40 + [300] + [1] * 40,
    "edges": [63, 64, 65, 1, 0, 127, 128, 129] + [2] * 60,
    "long_ends": [200] + [0, 1, 3] * 40 + [130],
    "empty_ones": [0] * 100 + [257] + [0] * 70,
    "neighbours": [64, 64, 65, 66, 70] + [1] * 90,
    "many": [1] * 4500 + [150] + [0] * 30 + [70],
}


def check(pkg, dev, lengths, dtype, front, behind, index_dtype, with_states):
    total = front + sum(lengths) + behind
    q, k, v, g, beta, s0 = make(1, total, 1, 2, 40, 24, dtype, dev, sequences=len(lengths), l2norm=True)
    cu = torch.tensor([front] + lengths).cumsum(0).to(index_dtype).to(dev)
    before = s0.clone()
    if with_states:
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s0, return_final_states=True, final_states_out=s0, cu_seqlens=cu, qk_l2norm=True)
    else:
        out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, cu_seqlens=cu, qk_l2norm=True)
    assert not out[:, :front].any() and not out[:, total - behind:].any()
    edges = cu.tolist()
    by_length = {}
    for i, n in enumerate(lengths):
        by_length.setdefault(n, []).append(i)
    for n, which in by_length.items():                   # sequences of a length as one batch
        first = before[which] if with_states else torch.zeros_like(before[which])
        if n == 0:
            assert torch.equal(final[which], first)
            continue
        part = [torch.cat([t[:, edges[i]:edges[i] + n] for i in which]) for t in (q, k, v, g, beta)]
        want, want_final = recurrence(*part, first, True)
        close(torch.cat([out[:, edges[i]:edges[i] + n] for i in which]), want, dtype, 40, "out of length %d" % n)
        close(final[which], want_final, torch.float32, 40, "final of length %d" % n)


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(RAGGED))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("front,behind", [(0, 0), (5, 70)])
def test_each_by_its_own_length(pkg, gpu_device, name, dtype, front, behind):
    check(pkg, gpu_device, RAGGED[name], dtype, front, behind, torch.int32, True)
    check(pkg, gpu_device, RAGGED[name], dtype, front, behind, torch.int64, False)


@pytest.mark.gpu
def test_unequal_short_sequences_by_tokens(pkg, gpu_device):
    """Few tokens: the token kernel alone, with tokens of no sequence in front and behind."""
    check(pkg, gpu_device, [2, 0, 4, 1, 4], torch.bfloat16, 3, 6, torch.int32, True)
    check(pkg, gpu_device, [2, 0, 4, 1, 4], torch.float32, 3, 6, torch.int64, False)


@pytest.mark.gpu
def test_a_sequence_alone_and_among_others(pkg, gpu_device):
    """The long sequence gives the bits that it gives alone, wherever it lies."""
    q, k, v, g, beta, s0 = make(1, 400, 2, 2, 64, 48, torch.bfloat16, gpu_device, l2norm=True)
    want, last = pkg.gated_delta_rule_fn(q[:, 37:337], k[:, 37:337], v[:, 37:337], g[:, 37:337], beta[:, 37:337], initial_states=s0, return_final_states=True, qk_l2norm=True)
    lengths = [1] * 37 + [300] + [1] * 63
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(gpu_device)
    states = torch.randn(101, 4, 64, 48, device=gpu_device)
    states[37] = s0[0]
    out, final = pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=states, return_final_states=True, cu_seqlens=cu, qk_l2norm=True)
    assert torch.equal(out[:, 37:337], want) and torch.equal(final[37], last[0])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["one_long", "edges"])
def test_gradients(pkg, gpu_device, name):
    """More than 64 sequences: the chunk's sequence is found in two steps."""
    lengths = RAGGED[name]
    total = sum(lengths)
    q, k, v, g, beta, s0 = make(1, total, 1, 2, 40, 24, torch.bfloat16, gpu_device, sequences=len(lengths), l2norm=True)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(gpu_device)
    r = torch.Generator().manual_seed(5)
    dout, dfinal = torch.randn(v.shape, generator=r).bfloat16().to(gpu_device), torch.randn(s0.shape, generator=r).to(gpu_device)
    got = gradients(pkg, [q, k, v, g, beta, s0], dout, dfinal, True, cu=cu)
    want = [torch.zeros(t.shape, dtype=torch.float64, device=gpu_device) for t in (q, k, v, g, beta, s0)]
    edges = cu.tolist()
    for n in set(lengths):
        which = [i for i, m in enumerate(lengths) if m == n]
        if n == 0:
            want[5][which] = dfinal[which].double()
            continue
        cut = [torch.cat([t[:, edges[i]:edges[i] + n] for i in which]) for t in (q, k, v, g, beta, dout)]
        for j, d in enumerate(gradients64(cut[:5] + [s0[which]], cut[5], dfinal[which], True)):
            for row, i in enumerate(which):
                if j < 5:
                    want[j][:, edges[i]:edges[i] + n] = d[row:row + 1]
                else:
                    want[5][i] = d[row]
    for label, a, b in zip(NAMES, got, want):
        near(a, b, 40, 24, "d" + label)
