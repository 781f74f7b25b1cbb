"""The gated block's kernels at activations and sizes beside tests/test_gated.py's, with its tolerances."""
import pytest
import torch

from test_gated import NAMES, TYPES, _case, _check, _reference, _run


# 64 x 64 tiles; few rows, without and with kept projections; up to 15 columns, alone and in shares; square tiles that
# compute the projections again and that read them, whole and cut
RELU = [(70, 48, 80), (33, 72, 200), (16, 264, 520), (400, 12, 128), (100, 3, 5000), (4100, 136, 1000), (4100, 264, 1000),
        (100, 4000, 1000), (300, 2056, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", RELU)
def test_relu(cuda, rows, dim, hidden, kind):
    args, dh = _case(rows, dim, hidden, kind, True, rows + dim)
    want, tol = _reference(*args, dh, "relu", TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, "relu"), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [136, 264])
def test_offsets_past_32_bits(cuda, dim):
    """2.3 G outputs (and of the projections that the forward keeps, where dim is 264): the first and last rows
    against the definition, both biases' gradients against sums over all rows."""
    from gsr.layers import gated_linear
    rows, hidden = 280003, 8200
    (_, wg, wu, bg, bu), _ = _case(1, dim, hidden, "bf16", True, 4)
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(rows, dim, device=cuda, generator=g, dtype=torch.bfloat16)
    dh = torch.randn(rows, hidden, device=cuda, generator=g, dtype=torch.bfloat16)
    leaves = [x.requires_grad_(True)] + [t.to(cuda).requires_grad_(True) for t in (wg, wu, bg, bu)]
    h = gated_linear(*leaves)
    dx, *dw = torch.autograd.grad(h, leaves, dh)
    sums = None
    size = 20000
    for at in range(0, rows, size):
        part = slice(at, min(rows, at + size))
        want, tol = _reference(x.detach()[part], *(t.detach() for t in leaves[1:]), dh[part], "silu", torch.bfloat16)
        _check(h[part], want[0], tol[0], f"h from {at}")
        _check(dx[part], want[1], tol[1], f"dx from {at}")
        # (a part's tolerance counts its own rows: the chain over all of them takes as many times as much of c(rows))
        now = [t.clone() for t in (*want[2:], *tol[2:])]
        sums = now if sums is None else [a + b for a, b in zip(sums, now)]
        del want, tol
    for name, got, v, t in zip(NAMES[2:], dw, sums[:4], sums[4:]):
        _check(got, v, t * (rows / size), name)
