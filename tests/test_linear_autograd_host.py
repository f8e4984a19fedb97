"""What autograd and the dispatcher are told by linear attention and the layer norm, on meta tensors, without a GPU."""
import contextlib

import pytest
import torch
from torch._dynamo import compiled_autograd
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode


def _meta(*shape, grad=False, dtype=torch.float32):
    return torch.empty(*shape, device="meta", dtype=dtype, requires_grad=grad)


def _linear(grad=False):
    """q, k, v, g, beta, states"""
    return [_meta(2, 9, 2, 16, grad=grad), _meta(2, 9, 2, 16, grad=grad), _meta(2, 9, 4, 24, grad=grad), _meta(2, 9, 4, grad=grad), _meta(2, 9, 4, grad=grad),
            _meta(2, 4, 16, 24, grad=grad)]


def _norm(grad=False):
    """x, weight, bias, residual"""
    return [_meta(3, 40, grad=grad), _meta(40, grad=grad), _meta(40, grad=grad), _meta(3, 40, grad=grad)]


def _linear_out(pkg, a):
    return pkg.linear_attention_fn(*a[:5], initial_states=a[5], return_final_states=True)


def _constant_decay(pkg, a):
    return pkg.linear_attention_fn(*a[:3], a[3][0, 0], initial_states=a[5], return_final_states=True) + (a[4] * 1,)


def _norm_out(pkg, a):
    return pkg.layer_norm_fn(a[0], a[1], a[2], residual=a[3])


def _python_linear(pkg, a):
    from causal_conv1d.linear_attention import LinearAttentionFn
    return LinearAttentionFn.apply(*a[:5], 0.25, a[5], True, None)


def _python_norm(pkg, a):
    from causal_conv1d.layer_norm import LayerNormFn
    return LayerNormFn.apply(*a, 1e-5)


BOTH = [(_linear, _linear_out), (_norm, _norm_out), (_linear, _python_linear), (_norm, _python_norm)]


@pytest.mark.parametrize("make,run", BOTH)
def test_second_derivatives_are_refused(pkg, make, run, recwarn):
    leaves = make(grad=True)
    outs = run(pkg, leaves)
    grads = torch.autograd.grad(outs, leaves, [torch.empty_like(t) for t in outs], create_graph=True)
    for g in grads:
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="derivative for .* is not implemented"):
            torch.autograd.grad(g.sum(), leaves, allow_unused=True, retain_graph=True)
    assert not [w for w in recwarn if "autograd kernel was not registered" in str(w.message)]


def test_ops_without_a_graph_say_so(pkg):
    ops = torch.ops.DaoAILab
    q, k, v, g, beta, s = _linear(grad=True)
    x, w, b, r = _norm(grad=True)
    for outs in (ops._linear_attention_fwd_cpp(q, k, v, g, beta, s, None, None, 0.25), ops._linear_attention_fwd_save_cpp(q, k, v, g, beta, s, None, None, 0.25)[0],
                 ops._layer_norm_fwd_cpp(x, w, b, r, 1e-5, True)[0]):
        with pytest.raises(RuntimeError, match="derivative for .* is not implemented"):
            outs.sum().backward()


@pytest.mark.parametrize("make,run", BOTH)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(pkg, make, run, grad):
    args = make(grad=grad)
    for i in range(len(args)):
        with torch.autograd.forward_ad.dual_level():
            dual = [torch.autograd.forward_ad.make_dual(t, torch.empty_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="jvp"):
                run(pkg, dual)
            if run in (_linear_out, _norm_out):
                with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                    run(pkg, dual)
    run(pkg, args)


def test_the_step_claims_no_graph(pkg):
    q, k, v, g, beta, _ = _linear(grad=True)
    state = _meta(2, 4, 16, 24)
    for out in (pkg.linear_attention_update(q, k, v, g, state, beta=beta), torch.ops.DaoAILab._linear_attention_update_cpp(q, k, v, g, state, beta, None, 0.25)):
        assert not out.requires_grad and not state.requires_grad and out.shape == v.shape


def test_states_with_a_graph_are_not_written(pkg):
    q, k, v, g, beta, s = _linear()
    leaf = _meta(2, 4, 16, 24, grad=True)
    for state in (leaf, leaf * 2):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            pkg.linear_attention_update(q, k, v, g, state, beta=beta)
        with pytest.raises(RuntimeError, match="requires a gradient"):
            pkg.linear_attention_fn(q, k, v, g, return_final_states=True, final_states_out=state)
        with torch.no_grad():
            pkg.linear_attention_update(q, k, v, g, state)
            pkg.linear_attention_fn(q, k, v, g, return_final_states=True, final_states_out=state)


def test_writing_in_place_moves_the_version(pkg):
    ops = torch.ops.DaoAILab
    q, k, v, g, beta, _ = _linear()
    for write in (lambda s: pkg.linear_attention_update(q, k, v, g, s), lambda s: ops._linear_attention_update_cpp(q, k, v, g, s, beta, None, 0.25),
                  lambda s: pkg.linear_attention_fn(q, k, v, g, initial_states=s, return_final_states=True, final_states_out=s),
                  lambda s: ops._linear_attention_fwd_save_cpp(q, k, v, g, beta, None, None, s, 0.25)):
        state, w = _meta(2, 4, 16, 24), _meta(2, 4, 16, 24, grad=True)
        out = (state * w).sum()
        before = state._version
        with torch.no_grad():
            write(state)
        assert state._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()


@pytest.mark.parametrize("make,run", [(_linear, _linear_out), (_linear, _constant_decay), (_norm, _norm_out)])
@pytest.mark.parametrize("compiled", [False, True], ids=["engine", "compiled_autograd"])
def test_every_gradient_arrives(pkg, make, run, compiled):
    leaves = make(grad=True)
    with compiled_autograd._enable(torch.compile(backend="eager")) if compiled else contextlib.nullcontext():
        sum(t.sum() for t in run(pkg, leaves)).backward()
    assert [None if t.grad is None else t.grad.shape for t in leaves] == [t.shape for t in leaves]


def test_final_states_out_that_is_not_asked_for(pkg):
    a = _linear(grad=True)
    for scale in (0.25, 1):
        for args in (a, [t.detach() for t in a]):
            s = _meta(2, 4, 16, 24)
            out = pkg.linear_attention_fn(*args[:5], scale=scale, initial_states=args[5], final_states_out=s)
            assert out.shape == a[2].shape and s._version == 0
        with pytest.raises(RuntimeError, match="where gradients are recorded"):
            pkg.linear_attention_fn(*a[:5], scale=scale, return_final_states=True, final_states_out=s)


class _Subclass(torch.Tensor):
    pass


class _Functions(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class _Ops(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name)
        return func(*args, **(kwargs or {}))


def test_left_to_the_generic_path(pkg):
    """What the direct calls must not take: subclasses, what is no tensor, wrong numbers of arguments, active modes."""
    import causal_conv1d_cuda as ext
    q, k, v, g, beta, s = _linear()
    x, w, b, r = _norm()
    calls = [(ext._linear_attention_call, [q, k, v, g, beta, 0.25, s, True, None, None], (0, 1, 2, 3, 4, 6)),
             (ext._linear_attention_update_call, [q, k, v, g, s, beta, None, 0.25], (0, 1, 2, 3, 4, 5)), (ext._layer_norm_call, [x, w, b, r, 1e-5], (0, 1, 2, 3))]
    for call, args, tensors in calls:
        assert call(*args) is not NotImplemented
        for i in tensors:
            for other in (args[i].as_subclass(_Subclass), 5):
                a = list(args)
                a[i] = other
                assert call(*a) is NotImplemented
        assert call(*args[:-1]) is NotImplemented
        with _Functions():
            assert call(*args) is NotImplemented
    with _Ops() as ops:
        pkg.linear_attention_fn(q, k, v, g)
        pkg.linear_attention_update(q, k, v, g, s)
        pkg.layer_norm_fn(x, w, b, residual=r)
    for name in ("fwd", "update"):
        assert "DaoAILab::_linear_attention_%s_cpp" % name in ops.names
    assert "DaoAILab::_layer_norm_fwd_cpp" in ops.names
