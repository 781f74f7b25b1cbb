"""What the layers do with inputs that plain reverse-mode training does not hand them."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def _inputs(dev="cpu"):
    g = torch.Generator().manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    return dict(x=mk(6, 8), w=mk(8), b=mk(8), wg=mk(5, 8), wu=mk(5, 8), bg=mk(5), bu=mk(5))


def _norm(t):
    from gsr.layers import layer_norm
    return layer_norm(t["x"], t["w"], t["b"])


def _gated(t):
    from gsr.layers import gated_linear
    return gated_linear(t["x"], t["wg"], t["wu"], t["bg"], t["bu"])


@pytest.mark.parametrize("layer,which", [(_norm, k) for k in ("x", "w", "b")] + [(_gated, k) for k in ("x", "wg", "wu", "bg", "bu")])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(layer, which, grad):
    """A tensor with a tangent is refused, whether or not something requires a gradient: the result would
    have none, which reads as a derivative of zero."""
    t = _inputs()
    with fwd.dual_level():
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        if grad:
            t["x"].requires_grad_(True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            layer(t)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            layer(t)


@pytest.mark.parametrize("layer", [_norm, _gated])
def test_functional_jvp_is_refused(layer):
    t = _inputs()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: layer({**t, "x": x}), (t["x"],), (torch.ones_like(t["x"]),))


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [_norm, _gated])
def test_forward_mode_over_a_backward_is_refused(cuda, layer):
    t = _inputs(cuda)
    t["x"].requires_grad_(True)
    y = layer(t)
    plain, = torch.autograd.grad(y, [t["x"]], torch.ones_like(y), retain_graph=True)
    with fwd.dual_level():
        dy = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, [t["x"]], dy, retain_graph=True)
    assert torch.equal(plain, torch.autograd.grad(y, [t["x"]], torch.ones_like(y))[0])
