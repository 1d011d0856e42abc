"""CPU: vil_rotary_attention_qkv -- what it refuses before anything touches the device."""
import pytest
import torch

from vision_longformer_amd import ops, rotary


def args(nx=14, ny=14, nglo=1, H=2, M=64, **kw):
    """a packed projection with norm and rotation; table, g2l, g2g of the sliding-chunk layers unless given"""
    w = kw.get("w")
    side = 4 * w - 1 if w is not None else 2 * max(nx, ny) - 1
    a = dict(qkv=torch.zeros(2, nglo + nx * ny, 3 * H * M, dtype=torch.bfloat16), bias_table=torch.zeros(side * side, H),
             g2l_bias=torch.zeros(2, H, nglo), g2g_bias=torch.zeros(H, nglo, nglo), nx=nx, ny=ny, nglo=nglo, num_heads=H, norm=True)
    a.update(rotary.GridTurn(M).of(nx, ny, nglo, torch.device("cpu")))
    return {**a, **kw}


def test_windows_have_no_dense_kernels():
    """backend "dense" attends to all tokens and reads a (2 nx - 1)(2 ny - 1) table: with a window it has neither"""
    with pytest.raises(ValueError, match="dense"):
        ops.vil_rotary_attention_qkv(**args(w=4, backend="dense"))
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.vil_rotary_attention_qkv(**args(w=4))


@pytest.mark.parametrize("w", [None, 4])
@pytest.mark.parametrize("which,shape", [("bias_table", (26 * 26, 2)), ("bias_table", (27 * 27, 1)), ("bias_table", (15, 15, 2)),
                                         ("g2l_bias", (2, 2)), ("g2l_bias", (1, 2, 1)), ("g2g_bias", (2, 2, 1)), ("g2g_bias", (1, 1, 1))])
def test_biases_of_another_shape_are_refused(w, which, shape):
    """the kernels read them by address"""
    with pytest.raises(ValueError, match=which):
        ops.vil_rotary_attention_qkv(**args(w=w, **{which: torch.zeros(shape)}))
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.vil_rotary_attention_qkv(**args(w=w, **{which: None}))


@pytest.mark.parametrize("w", [None, 4])
@pytest.mark.parametrize("which", ["bias_table", "g2l_bias", "g2g_bias"])
def test_biases_on_another_device_are_refused(w, which):
    a = args(w=w)
    a[which] = a[which].to("meta")
    with pytest.raises(RuntimeError, match=which + " on meta"):
        ops.vil_rotary_attention_qkv(**a)


@pytest.mark.parametrize("eps", [-1e-6, float("nan")])
def test_eps_is_checked_like_vil_qk_norm_rope_s(eps):
    """a negative one gives NaN where mean(x^2) is smaller"""
    for f in (lambda: ops.vil_rotary_attention_qkv(**args(w=4, eps=eps)), lambda: rotary.vil_qk_norm_rope(torch.zeros(1, 1, 1, 8), eps=eps)):
        with pytest.raises(ValueError, match="eps"):
            f()


@pytest.mark.parametrize("w", [None, 4])
def test_a_second_derivative_is_refused(w, monkeypatch):
    """With the launches replaced, and an incoming gradient that requires none: under create_graph the gradients come back, and a
    penalty on them next to another term raises instead of leaving the attention's part out."""
    def empty_out(q, *rest):
        return torch.zeros_like(q), torch.zeros(1), torch.zeros(1)

    def no_grads(q, k, v, out, dout, lse, lse_g, tab, g2l, g2g, dq, dk, dv, cfg, backend):
        for t in (dq, dk, dv):
            t.zero_()
        return tab, g2l, g2g

    monkeypatch.setattr(ops, "_check_dev", lambda *a: None)
    monkeypatch.setattr(rotary, "_check", lambda *a: None)
    monkeypatch.setattr(rotary, "_PLANS", {})                   # (none of this test's layouts is kept as checked)
    monkeypatch.setattr(rotary, "_bwd", lambda plan, desc, gq, gk, q, k, wq, wk, pos, f, dq, dk, need_wq, need_wk: (
        dq.zero_(), dk.zero_(), torch.zeros_like(wq), torch.zeros_like(wk))[2:])
    monkeypatch.setattr(rotary._lib, "launch", lambda *a: None)
    monkeypatch.setattr(ops, "_full_fwd", empty_out)
    monkeypatch.setattr(ops, "_full_bwd", no_grads)
    a = args(w=w, q_weight=torch.ones(64, requires_grad=True), k_weight=torch.ones(64, requires_grad=True))
    leaves = [a[n].requires_grad_() for n in ("qkv", "bias_table", "g2l_bias", "g2g_bias", "q_weight", "k_weight")]
    out = ops.vil_rotary_attention_qkv(**a)
    grads = torch.autograd.grad(out.float().sum(), leaves, create_graph=True)
    for g, v in zip(grads, leaves):
        assert g.shape == v.shape
        with pytest.raises(RuntimeError):
            (g.float().square().sum() + v.float().square().sum()).backward(retain_graph=True)
