"""What a gated block's forward leaves for its backward, and how much memory its passes take."""
import pytest
import torch

from test_gated import NAMES, TYPES, _case, _check, _reference, _run


def _kept(rows, dim, hidden, kind):
    from gsr import _lib
    return _lib.lib().gsr_gated_kept(rows, dim, hidden, {"f32": _lib.F32, "bf16": _lib.BF16, "f16": _lib.F16}[kind])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows,dim,hidden", [(16, 50, 45000), (64, 50, 45000), (5, 63, 34000), (40, 9, 300000), (1, 15, 1 << 20)])
def test_nothing_is_kept_that_no_backward_reads(rows, dim, hidden, kind):
    """Up to 64 rows of a short odd length: no product of the backward reads copies of x and the weights."""
    assert _kept(rows, dim, hidden, kind) == 0


def test_copies_are_kept_where_the_backward_reads_them():
    """Odd lengths on square tiles of 128 and more, and few rows whose projections are kept."""
    assert _kept(4100, 129, 1025, "bf16") == (4100 + 2 * 1025) * 136 * 2
    projections = 60 * 5760 * 6
    assert _kept(60, 2699, 5750, "bf16") == projections + (60 + 2 * 5750) * 2704 * 2
    assert _kept(60, 2704, 5750, "bf16") == projections


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", [(16, 50, 45000), (33, 50, 45000), (5, 63, 34000), (40, 9, 240000)])
def test_few_short_odd_rows(cuda, rows, dim, hidden, kind):
    bias = rows % 2 == 1
    act = ("silu", "gelu", "sigmoid")[rows % 3]
    args, dh = _case(rows, dim, hidden, kind, bias, rows + dim)
    dh = dh * 2 ** -5   # (keeps fp16's sums over the hidden columns in range)
    want, tol = _reference(*args, dh, act, TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, act), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind} {act}")


# A backward of up to 15 columns: rows' parts of the weights' gradients, columns' parts of dx
@pytest.mark.parametrize("rows,dim,hidden", [(32768, 15, 65536), (1 << 26, 15, 16), (1 << 20, 15, 1 << 16), (100000, 15, 1 << 20),
                                             (65, 15, 1 << 20), (1 << 24, 1, 1 << 20), (1, 1, 1 << 20), (16000, 8, 12288)])
def test_narrow_workspace_is_bounded(rows, dim, hidden):
    """512 MB for either, or one part of dx, or two of the weights' gradients where those are more."""
    from gsr import _lib
    weights, dx = 2 * hidden * (dim + 4) // 4 * 4 * 4, rows * dim * 4
    got = _lib.lib().gsr_gated_workspace(rows, dim, hidden, _lib.BF16, 1)
    assert got <= max(512 << 20, 2 * weights) + max(512 << 20, dx) + 512


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_narrow_rows_share_their_parts(cuda, kind):
    """So wide a hidden layer that workgroups add several tiles of rows to one part, and columns share dx."""
    rows, dim, hidden = 4210, 15, 65500
    args, dh = _case(rows, dim, hidden, kind, True, 6)
    args, dh = [t.to(cuda) for t in args], (dh * 2 ** -5).to(cuda)
    want, tol = _reference(*args, dh, "silu", TYPES[kind])
    first = _run(cuda, args, dh, "silu")
    for name, got, v, t in zip(NAMES, first, want, tol):
        _check(got, v, t, f"{name} {kind}")
    assert all(torch.equal(a, b) for a, b in zip(first, _run(cuda, args, dh, "silu")))
