"""Layers at sizes where a count of threads or elements passes 32 bits.

Tolerances: tests/test_layer_norm.py's and tests/test_gated.py's."""
import pytest
import torch

from test_layer_norm import U


@pytest.mark.gpu
def test_layer_norm_of_one_long_row(cuda):
    """One row of 2^27 + 7 columns, backward too.  A lane adds 2^17 values of magnitudes up to 1 before the
    tree: G = 2 (dim / 1024 + 48) u of the magnitudes' mean, as for shorter rows."""
    from gsr.layers import layer_norm
    dim = (1 << 27) + 7
    g = torch.Generator(device=cuda).manual_seed(1)
    mk = lambda: torch.rand(1, dim, device=cuda, generator=g)  # noqa: E731
    x, dy = mk().requires_grad_(True), mk()
    w, b = torch.full((dim,), 0.5, device=cuda, requires_grad=True), torch.zeros(dim, device=cuda, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    xd, dyd = x.detach().double(), dy.double()
    mean = xd.mean()
    rstd = 1 / ((xd - mean).square().mean() + 1e-5).sqrt()
    z = (xd - mean) * rstd
    G = 2 * (48 + dim / 1024) * U
    X = float((1 + xd.abs().mean()) * rstd)
    assert float((y.double() - 0.5 * z).abs().max()) <= G * 0.5 * X
    want = rstd * 0.5 * (dyd - dyd.mean() - z * (dyd * z).mean())
    assert float((dx.double() - want).abs().max()) <= 2 * G * float(rstd) * 0.5 * (2 + 2 * X * X)
    assert torch.equal(db, dy[0])
    assert float((dw.double() - (dyd * z)[0]).abs().max()) <= (G + 65 * U) * X


@pytest.mark.gpu
def test_no_rows_of_a_large_block(cuda):
    """The weights' gradients of no rows are zeros, to the last of 2^31 + 2^15 of them (none of the others are
    asked for; the inputs are not read)."""
    from gsr import _lib
    hidden, dim = (1 << 16) + 1, 1 << 15
    out = torch.full((hidden, dim), 3.0, device=cuda)
    x = out.data_ptr()
    _lib.check(_lib.lib().gsr_gated_bwd(None, 0, dim, dim, _lib.F32, x, x, hidden, None, None, 0, None, hidden, None, None, x, None,
                                        None, None, None, 0, torch.cuda.current_stream().cuda_stream), "gsr_gated_bwd")
    assert not bool(out.any())
