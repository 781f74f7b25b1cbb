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


def _negated(t):
    """-t as a view that negates when it is read (what autograd makes of an imaginary part's conjugate)."""
    return torch._neg_view(-t)


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [_norm, _gated])
def test_negated_views(cuda, layer):
    """Views that hold their negative give the values they stand for, as inputs and as the output's gradient."""
    t = {k: v.requires_grad_(True) for k, v in _inputs(cuda).items()}
    y = layer(t)
    dy = torch.randn(y.shape, device=cuda)
    want = [y, *(g for g in torch.autograd.grad(y, list(t.values()), dy, allow_unused=True) if g is not None)]
    n = {k: _negated(v.detach()).requires_grad_(True) for k, v in t.items()}
    assert all(v.is_neg() for v in n.values())
    y = layer(n)
    got = [y, *(g for g in torch.autograd.grad(y, list(n.values()), _negated(dy), allow_unused=True) if g is not None)]
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.no_grad():
        assert torch.equal(want[0], layer({k: v.detach() for k, v in n.items()}))


@pytest.mark.gpu
def test_negated_gradient_of_a_step(cuda):
    from gsr.optim import adamw_step
    g = torch.randn(300, device=cuda)
    make = lambda: [torch.ones(300, device=cuda), torch.zeros(300, device=cuda), torch.zeros(300, device=cuda)]  # noqa: E731
    a, b = make(), make()
    adamw_step([a[0]], [g], [a[1]], [a[2]], step=1)
    adamw_step([b[0]], [_negated(g)], [b[1]], [b[2]], step=1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_negated_views_are_not_written():
    from gsr.optim import adamw_step, decode_root
    f = lambda: torch.zeros(4)  # noqa: E731
    for k in range(3):
        written = [f(), f(), f()]
        written[k] = _negated(f())
        with pytest.raises(ValueError, match="negat"):
            adamw_step([written[0]], [f()], [written[1]], [written[2]], step=1)
    e4, u8 = f().to(torch.float8_e4m3fn), f().to(torch.uint8)
    for units in ((_negated(f()[:1]), f()[:1]), (f()[:1], _negated(f()[:1]))):
        with pytest.raises(ValueError, match="negat"):
            adamw_step([f()], [f()], [e4], [u8], step=1, exp_avg_units=[units[0]], exp_avg_root_units=[units[1]])
    with pytest.raises(ValueError, match="negat"):
        adamw_step([f()], [f()], [f()], [f()], step=1, lr=_negated(torch.tensor(1e-3)))
    with pytest.raises(ValueError, match="negat"):
        decode_root(u8, _negated(f()[:1]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,hidden", [(300, 9, 40), (300, 264, 520), (60, 2501, 900), (700, 509, 1363), (2600, 72, 1025)])
def test_saved_tensors_elsewhere(cuda, rows, dim, hidden):
    """What the forward keeps may be moved before the backward (other addresses, rows packed), and a graph
    that is kept may be walked twice: the same bits."""
    from gsr.layers import gated_linear, layer_norm
    g = torch.Generator(device=cuda).manual_seed(rows)
    mk = lambda *s: torch.randn(*s, device=cuda, generator=g).to(torch.bfloat16)  # noqa: E731
    x, w, wg, wu, dh = mk(rows, dim + 5)[:, 3:3 + dim], mk(dim), mk(hidden, dim), mk(hidden, dim), mk(rows, hidden)

    def graph():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, wg, wu)]
        return leaves, gated_linear(layer_norm(leaves[0], leaves[1]), *leaves[2:])
    leaves, h = graph()
    want = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(h, leaves, dh)))
    with torch.autograd.graph.save_on_cpu():
        leaves, h = graph()
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(h, leaves, dh)))
    leaves = [t.detach().requires_grad_(True) for t in (x, w, wg, wu)]
    h = torch.utils.checkpoint.checkpoint(lambda *t: gated_linear(t[0], *t[1:]), leaves[0], *leaves[2:], use_reentrant=False)
    direct = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    for a, b in zip(torch.autograd.grad(h, [leaves[0], *leaves[2:]], dh), torch.autograd.grad(gated_linear(*direct), direct, dh)):
        assert torch.equal(a, b)
