"""CPU: what the operators on q and k and the 8-bit ones do where a derivative is asked of them that the kernels do not give.  The
launches are replaced (outputs hold whatever their memory holds); nothing touches a device."""
import pytest
import torch
from torch.autograd import forward_ad

from vision_longformer_amd import _lib, act8, rotary


@pytest.fixture
def launched(monkeypatch):
    """names of the entry points that a test reaches"""
    names = []

    def launch(index, fn, *args):
        assert torch._C._get_tracing_state() is None            # (where the launch itself would refuse)
        names.append(fn.__name__)

    monkeypatch.setattr(_lib, "launch", launch)
    monkeypatch.setattr(rotary, "_check", lambda *a: None)
    monkeypatch.setattr(act8, "_check", lambda *a: None)
    monkeypatch.setattr(act8, "_check_packed", lambda *a: None)
    monkeypatch.setattr(rotary, "_PLANS", {})                   # (none of these layouts is kept as checked)
    return names


def qk(**kw):
    q, k = torch.randn(1, 6, 2, 32, **kw), torch.randn(1, 6, 1, 32, **kw)
    return q, k, dict(positions=rotary.grid_positions(2, 3), inv_freq=rotary.rotary_frequencies((8, 8)), sections=(8, 8))


def test_norm_gradient_under_create_graph(launched):
    """the incoming gradient requires none, the norm's gradient depends on q, k and the weights all the same"""
    q, k, turn = qk(requires_grad=True)
    w = torch.ones(32, requires_grad=True)
    yq, yk = rotary.vil_qk_norm_rope(q, k, w, w, **turn)
    grads = torch.autograd.grad(yq.sum() + yk.sum(), (q, k, w), create_graph=True)
    for g, v in zip(grads, (q, k, w)):
        assert g.shape == v.shape
        with pytest.raises(RuntimeError):
            (g.sum() + v.square().sum()).backward(retain_graph=True)
    assert launched == ["vil_qk_rope_fwd", "vil_qk_rope_bwd"]


def test_rotation_gradient_under_create_graph(launched):
    """linear in q: nothing is left out where the incoming gradient is a constant, and where it is not, the call raises"""
    q, _, turn = qk(requires_grad=True)
    y = rotary.vil_rope(q, **turn)
    g, = torch.autograd.grad(y.sum(), q, create_graph=True)
    (g.sum() + q.square().sum()).backward(retain_graph=True)
    assert torch.equal(q.grad, 2 * q.detach())
    g, = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        (g.sum() + q.square().sum()).backward()


@pytest.mark.parametrize("op", ["gelu", "mlp"])
def test_8_bit_gradients_under_create_graph(op, launched):
    """the incoming gradient requires none, the GELU's slope depends on its input all the same"""
    x = torch.randn(4, 32, requires_grad=True)
    leaves = [x]
    if op == "mlp":
        leaves += [torch.randn(s, requires_grad=True) for s in ((64, 32), (64,), (32, 64), (32,))]
    y = act8.vil_gelu_act8(x) if op == "gelu" else act8.vil_mlp_act8(*leaves)
    for g, v in zip(torch.autograd.grad(y.sum(), leaves, create_graph=True), leaves):
        assert g.shape == v.shape
        with pytest.raises(RuntimeError):
            (g.sum() + v.square().sum()).backward(retain_graph=True)
    assert "vil_gelu_act8_fwd" in launched and "vil_gelu_act8_bwd" in launched


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("norm", [True, False])
def test_forward_mode_is_refused(norm, grad, launched):
    """a dual tensor requires no gradient: its tangent must not be dropped for that"""
    q, k, turn = qk()
    fn = rotary.vil_qk_norm_rope if norm else rotary.vil_rope
    with torch.set_grad_enabled(grad):
        for at in (0, 1):
            with forward_ad.dual_level():
                dual = [q, k]
                dual[at] = forward_ad.make_dual(dual[at], torch.ones_like(dual[at]))
                with pytest.raises(NotImplementedError):
                    fn(*dual, **turn)
                if norm:
                    with pytest.raises(NotImplementedError):
                        fn(q, k, forward_ad.make_dual(torch.ones(32), torch.ones(32)), **turn)
                assert fn(q, k, **turn)[at].shape == (q, k)[at].shape                # no tangent: an ordinary call
        n = len(launched)
        fn(q, k, **turn)
        assert len(launched) == n + 1


@pytest.mark.parametrize("norm", [True, False])
def test_a_traced_call_launches(norm, launched):
    """a trace of a call without gradients records the node, not its empty outputs alone"""
    q, k, turn = qk()
    fn = rotary.vil_qk_norm_rope if norm else rotary.vil_rope
    traced = torch.jit.trace(lambda q, k: fn(q, k, **turn), (q, k), check_trace=False)
    n = len(launched)
    yq, yk = traced(q, k)
    assert launched[n:] == ["vil_qk_rope_fwd"] and yq.shape == q.shape and yk.shape == k.shape


@pytest.mark.parametrize("fn", [lambda x: act8.vil_act8_unpack(act8.vil_act8_pack(x)), lambda x: act8.vil_gelu_act8_fwd(x)[0]])
def test_calls_without_a_node_are_not_traced(fn, monkeypatch):
    """(without `launched`: what refuses is the launch)"""
    monkeypatch.setattr(act8, "_check", lambda *a: None)
    monkeypatch.setattr(act8, "_check_packed", lambda *a: None)
    with pytest.raises(RuntimeError, match="no launch"):
        torch.jit.trace(fn, (torch.randn(4, 64),), check_trace=False)


@pytest.mark.parametrize("op", ["gelu", "mlp"])
def test_a_traced_8_bit_node_launches(op, launched):
    ws = [torch.randn(s) for s in ((128, 64), (128,), (64, 128), (64,))]
    traced = torch.jit.trace(act8.vil_gelu_act8 if op == "gelu" else lambda x: act8.vil_mlp_act8(x, *ws), (torch.randn(4, 64),), check_trace=False)
    n = len(launched)
    assert traced(torch.randn(4, 64)).shape == (4, 64) and "vil_gelu_act8_fwd" in launched[n:]


def test_a_failing_call_leaves_the_trace_on(monkeypatch):
    """(the node turns tracing off while it runs)"""
    class Node(torch.autograd.Function):
        @staticmethod
        @_lib.untraced
        def forward(ctx, x):
            assert torch._C._get_tracing_state() is None and type(x.shape[0]) is int
            raise KeyError("no")

    def fn(x):
        on = torch._C._get_tracing_state()
        assert on is not None
        with pytest.raises(KeyError):
            Node.apply(x)
        assert torch._C._get_tracing_state() is not None
        return x + 1

    torch.jit.trace(fn, (torch.ones(3),), check_trace=False)
