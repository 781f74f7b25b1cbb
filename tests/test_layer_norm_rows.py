"""Layer norm over more rows than its launches have places for: workgroups walk the rows, load the next one
ahead, and add dw and db up over all of theirs.  Against the definition in 64 bits, with
tests/test_layer_norm.py's tolerances; every row has a mean and a size of its own, so that one taken for
another shows."""
import pytest
import torch

from test_layer_norm import TYPES, _reference


def _case(rows, dim, kind, device):
    g = torch.Generator(device=device).manual_seed(rows + dim)
    mk = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    t = TYPES[kind]
    x = (mk(rows, dim) * (mk(rows, 1) * 0.5).exp() + mk(rows, 1)).to(t)
    return x, (mk(rows, dim) * (mk(rows, 1) * 0.5).exp()).to(t), (1 + 0.3 * mk(dim)).to(t), (0.3 * mk(dim)).to(t)


def _check(got, want, tol, what):
    half = torch.finfo(got.dtype).eps / 2
    limit = tol + half * want.abs() + torch.finfo(got.dtype).tiny
    bad = ~((got.detach().double() - want).abs() <= limit)
    assert got.shape == want.shape and not bool(bad.any()), f"{what}: {int(bad.sum())} values, first at {bad.nonzero()[0].tolist()}"


# Lanes a row from 1 to a wave, a workgroup of 256 and of 1024, and rows longer than registers hold; a whole number
# of vectors, a last one that begins early, rows shorter than one; rows that do not fill the last round
SHAPES = [(530001, 3), (530001, 7), (270001, 14), (140003, 30), (70001, 60), (35003, 125), (17001, 250), (9001, 500), (9001, 512),
          (8900, 1000), (8900, 1031), (2500, 2048), (2501, 2501), (2499, 4096), (2501, 8190), (2100, 9001), (2101, 16388), (2070, 33001)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_rows_are_walked(cuda, rows, dim, kind):
    from gsr.layers import layer_norm
    x, dy, w, b = _case(rows, dim, kind, cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    want, tol = _reference(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    for name, got, v, t in zip(("y", "dx", "dw", "db"), (y, *grads), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim} {kind}")
    with torch.no_grad():   # (without the statistics)
        assert torch.equal(layer_norm(*leaves), y)


@pytest.mark.gpu
@pytest.mark.parametrize("left,right", [(0, 3), (1, 4)])
def test_walked_rows_of_a_wider_buffer(cuda, left, right):
    """The same bits as packed rows, with NaN around them that no row may read."""
    from gsr.layers import layer_norm
    x, dy, w, b = _case(9001, 253, "bf16", cuda)

    def inside(t):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), device=cuda, dtype=t.dtype)
        wide[:, left:left + t.shape[1]] = t
        return wide[:, left:left + t.shape[1]]

    def run(x, dy):
        leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)]
        y = layer_norm(*leaves)
        return [y, *torch.autograd.grad(y, leaves, dy)]
    assert all(torch.equal(p, q) for p, q in zip(run(x, dy), run(inside(x), inside(dy))))


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """2.4 G elements: the first and last rows against the definition, and dw and db against sums of all."""
    from gsr.layers import layer_norm
    rows, dim = 600011, 4000
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(rows, dim, device=cuda, generator=g, dtype=torch.bfloat16).requires_grad_(True)
    dy = torch.randn(rows, dim, device=cuda, generator=g, dtype=torch.bfloat16)
    w = torch.full((dim,), 1.5, device=cuda, requires_grad=True)
    b = torch.zeros(dim, device=cuda, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    sums = [0.0] * 4
    for at in range(0, rows, 1 << 16):
        part = slice(at, min(rows, at + (1 << 16)))
        want, tol = _reference(x.detach()[part], w.detach(), b.detach(), dy[part], 1e-5)
        _check(y[part], want[0], tol[0], f"y from {at}")
        _check(dx[part], want[1], tol[1], f"dx from {at}")
        sums = [s + v for s, v in zip(sums, (want[2], want[3], tol[2], tol[3]))]
    # (a part's tolerance counts its own rows; the chain over all of them adds rows / 256 u of the magnitudes)
    more = rows / 65536
    _check(dw, sums[0], sums[2] * (1 + more), "dw")
    _check(db, sums[1], sums[3] * (1 + more), "db")
