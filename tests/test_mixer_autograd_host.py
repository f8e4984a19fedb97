"""What autograd is told by the mixer's operators, on meta tensors, without a GPU: nothing is cut off or left out without a word."""
import contextlib

import pytest
import torch
from torch._dynamo import compiled_autograd


def _meta(*shape, grad=False, dtype=torch.float32):
    return torch.empty(*shape, device="meta", dtype=dtype, requires_grad=grad)


def _delta(grad=False):
    """q, k, v, g, beta, states"""
    return [_meta(2, 9, 2, 16, grad=grad), _meta(2, 9, 2, 16, grad=grad), _meta(2, 9, 4, 24, grad=grad), _meta(2, 9, 4, grad=grad), _meta(2, 9, 4, grad=grad),
            _meta(2, 4, 16, 24, grad=grad)]


def _norm(grad=False):
    """x, weight, residual"""
    return [_meta(3, 40, grad=grad), _meta(40, grad=grad), _meta(3, 40, grad=grad)]


def _delta_out(pkg, a):
    return pkg.gated_delta_rule_fn(*a[:5], initial_states=a[5], return_final_states=True)


def _norm_out(pkg, a):
    return pkg.rms_norm_fn(a[0], a[1], residual=a[2])


def _python_delta(pkg, a):
    from causal_conv1d.gated_delta_rule import GatedDeltaRuleFn
    return GatedDeltaRuleFn.apply(*a[:5], 0.25, a[5], True, None, False)


def _python_norm(pkg, a):
    from causal_conv1d.rms_norm import RMSNormFn
    return RMSNormFn.apply(*a, 1e-5)


@pytest.mark.parametrize("make,run", [(_delta, _delta_out), (_norm, _norm_out), (_delta, _python_delta), (_norm, _python_norm)])
def test_second_derivatives_are_refused(pkg, make, run, recwarn):
    """A first derivative may be asked for with its graph; differentiating that is an error, not a zero with a warning."""
    leaves = make(grad=True)
    outs = run(pkg, leaves)
    grads = torch.autograd.grad(outs, leaves, [torch.empty_like(t) for t in outs], create_graph=True)
    for g in grads:
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="derivative for .* is not implemented"):
            torch.autograd.grad(g.sum(), leaves, allow_unused=True, retain_graph=True)
    assert not [w for w in recwarn if "autograd kernel was not registered" in str(w.message)]
    plain = torch.autograd.grad(run(pkg, leaves)[0].sum(), leaves[:2])
    assert not any(g.requires_grad for g in plain)


def test_ops_without_a_graph_say_so(pkg):
    """The ops behind the functions, called as they are on tensors that require a gradient."""
    ops = torch.ops.DaoAILab
    q, k, v, g, beta, s = _delta(grad=True)
    x, w, r = _norm(grad=True)
    for outs in (ops._gated_delta_rule_fwd_cpp(q, k, v, g, beta, s, None, None, 0.25, False),
                 ops._gated_delta_rule_fwd_save_cpp(q, k, v, g, beta, s, None, None, 0.25, False)[0], ops._rms_norm_fwd_cpp(x, w, r, 1e-5)[0]):
        with pytest.raises(RuntimeError, match="derivative for .* is not implemented"):
            outs.sum().backward()


@pytest.mark.parametrize("make,run", [(_delta, _delta_out), (_norm, _norm_out), (_delta, _python_delta), (_norm, _python_norm)])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(pkg, make, run, grad):
    """Forward-mode differentiation: of any input, whether it requires a gradient or not, and with gradients off."""
    args = make(grad=grad)
    for i in range(len(args)):
        with torch.autograd.forward_ad.dual_level():
            dual = [torch.autograd.forward_ad.make_dual(t, torch.empty_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="jvp"):
                run(pkg, dual)
            if run in (_delta_out, _norm_out):
                with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                    run(pkg, dual)
    run(pkg, args)


def test_what_has_no_backward_claims_none(pkg, recwarn):
    """The decode step, the output in 8 bits and its reading back: results outside of any graph, through the functions and the ops."""
    ops = torch.ops.DaoAILab
    q, k, v, g, beta, _ = _delta(grad=True)
    state = _meta(2, 4, 16, 24)
    x, w, r = _norm(grad=True)
    y8, scales = _meta(3, 40, dtype=torch.float8_e4m3fn), _meta(3, grad=True)
    for outs in ([pkg.gated_delta_rule_update(q, k, v, g, beta, state)], [ops._gated_delta_rule_update_cpp(q, k, v, g, beta, state, None, 0.25, False)],
                 pkg.rms_norm_quant_fn(x, w, residual=r), ops._rms_norm_quant_cpp(x, w, r, 1e-5), [pkg.dequantize_rows(y8, scales)],
                 [ops._dequantize_rows_cpp(y8, scales, torch.bfloat16)]):
        assert not any(t.requires_grad for t in outs)
    assert not state.requires_grad
    assert not [w for w in recwarn if "autograd kernel was not registered" in str(w.message)]


def test_states_with_a_graph_are_not_written(pkg):
    """What an operator writes in place may not be part of a graph that gradients are recorded for: its gradient would be wrong."""
    q, k, v, g, beta, s = _delta()
    leaf = _meta(2, 4, 16, 24, grad=True)
    for state in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            pkg.gated_delta_rule_update(q, k, v, g, beta, state)
        with pytest.raises(RuntimeError, match="requires a gradient"):
            pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, final_states_out=state)
        with torch.no_grad():
            pkg.gated_delta_rule_update(q, k, v, g, beta, state)
            pkg.gated_delta_rule_fn(q, k, v, g, beta, return_final_states=True, final_states_out=state)


def test_writing_in_place_moves_the_version(pkg):
    """As torch's own operators do: a graph that has saved a state notices that it has changed since."""
    ops = torch.ops.DaoAILab
    q, k, v, g, beta, _ = _delta()
    for write in (lambda s: pkg.gated_delta_rule_update(q, k, v, g, beta, s), lambda s: ops._gated_delta_rule_update_cpp(q, k, v, g, beta, s, None, 0.25, False),
                  lambda s: pkg.gated_delta_rule_fn(q, k, v, g, beta, initial_states=s, return_final_states=True, final_states_out=s),
                  lambda s: ops._gated_delta_rule_fwd_save_cpp(q, k, v, g, beta, None, None, s, 0.25, False)):
        state, w = _meta(2, 4, 16, 24), _meta(2, 4, 16, 24, grad=True)
        out = (state * w).sum()
        before = state._version
        with torch.no_grad():
            write(state)
        assert state._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()
    with torch.inference_mode():
        state = _meta(2, 4, 16, 24)
        pkg.gated_delta_rule_update(q, k, v, g, beta, state)
    with torch.no_grad():
        pkg.gated_delta_rule_update(q, k, v, g, beta, state)                 # (a server's states, made in inference mode)


@pytest.mark.parametrize("make,run", [(_delta, _delta_out), (_norm, _norm_out)])
@pytest.mark.parametrize("compiled", [False, True], ids=["engine", "compiled_autograd"])
def test_every_gradient_arrives(pkg, make, run, compiled):
    leaves = make(grad=True)
    with compiled_autograd._enable(torch.compile(backend="eager")) if compiled else contextlib.nullcontext():
        sum(t.sum() for t in run(pkg, leaves)).backward()
    assert [None if t.grad is None else t.grad.shape for t in leaves] == [t.shape for t in leaves]


def test_final_states_out_that_is_not_asked_for(pkg):
    """Without return_final_states it is left alone, whichever of the two graphs records the call (a scale that is no float: the Python one)."""
    a = _delta(grad=True)
    for scale in (0.25, 1):
        for args in (a, [t.detach() for t in a]):
            s = _meta(2, 4, 16, 24)
            out = pkg.gated_delta_rule_fn(*args[:5], scale=scale, initial_states=args[5], final_states_out=s)
            assert out.shape == a[2].shape and s._version == 0
        with pytest.raises(RuntimeError, match="where gradients are recorded"):
            pkg.gated_delta_rule_fn(*a[:5], scale=scale, return_final_states=True, final_states_out=s)
