"""gsr.layers.layer_norm against its definition in 64 bits.

Tolerances (u = 2^-24, the fp32 half step).  A lane adds up to 32 elements of a row (dim / 1024
more for rows longer than registers hold) before a tree of at most 10 levels, so a sum of n
terms is off by at most (48 + dim/1024) u times the sum of magnitudes; mean and rstd inherit
that, products and quotients add a few u.  With X = (|x| + mean|x|) rstd >= |xhat|:
    y   G (X |w| + |b|)                                  G = 2 (48 + dim/1024) u
    dx  2 G rstd (|w dy| + mean|w dy| + 2 X mean(|w dy| X))
    dw  (G + R) sum_rows |dy| X,  db  R sum_rows |dy|     R = (rows/256 + 64) u
plus half a step of the output's type."""
import pytest
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _reference(x, w, b, dy, eps):
    """(values, tolerances without the last rounding) of y, dx, dw, db in float64."""
    x, dy = x.double(), dy.double()
    rows, dim = x.shape
    w = torch.ones(dim, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(dim, dtype=torch.float64) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    z = (x - mean) * rstd
    wdy = w * dy
    dx = rstd * (wdy - wdy.mean(1, keepdim=True) - z * (wdy * z).mean(1, keepdim=True))
    G, R = 2 * (48 + dim / 1024) * U, (rows / 256 + 64) * U
    X = (x.abs() + x.abs().mean(1, keepdim=True)) * rstd
    a = wdy.abs()
    tol = [G * (X * w.abs() + b.abs()),
           2 * G * rstd * (a + a.mean(1, keepdim=True) + 2 * X * (a * X).mean(1, keepdim=True)),
           (G + R) * (dy.abs() * X).sum(0), R * dy.abs().sum(0)]
    return [z * w + b, dx, (dy * z).sum(0), dy.sum(0)], tol


def _check(got, want, tol, what):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    limit = tol + half * want.abs() + torch.finfo(got.dtype).tiny
    err = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= limit).all()), f"{what}: {float((err / limit).max()):.3g} of the tolerance"


def _case(rows, dim, kind, wkind, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, dim, generator=g) + offset).to(TYPES[kind])
    dy = torch.randn(rows, dim, generator=g).to(TYPES[kind])
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(TYPES[wkind])
    b = (0.3 * torch.randn(dim, generator=g)).to(TYPES[wkind])
    return x, dy, w, b


def _run(cuda, x, dy, w, b, eps=1e-5, view=lambda t: t):
    from gsr.layers import layer_norm
    xl = x.to(cuda).requires_grad_(True)
    wl, bl = (None if t is None else t.to(cuda).requires_grad_(True) for t in (w, b))
    y = layer_norm(view(xl), wl, bl, eps)
    leaves = [t for t in (xl, wl, bl) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy.to(cuda).view(y.shape)))
    return y, grads


SHAPES = [(1, 1), (5, 2), (7, 3), (300, 8), (33, 7), (9, 64), (4, 65), (260, 129), (3, 255), (6, 512), (2, 1000),
          (11, 1031), (5, 2048), (4, 2049), (3, 4100), (2, 8192), (3, 9001), (2, 16384), (2, 33000), (1030, 40),
          (2600, 14)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,wkind", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"),
                                        ("f32", "bf16")])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_forward_backward(cuda, rows, dim, kind, wkind):
    x, dy, w, b = _case(rows, dim, kind, wkind, seed=rows * 131 + dim)
    want, tol = _reference(x, w, b, dy, 1e-5)
    y, grads = _run(cuda, x, dy, w, b)
    for name, got, v, t in zip(("y", "dx", "dw", "db"), [y, *grads], want, tol):
        _check(got, v, t, f"{name} {rows}x{dim} {kind}/{wkind}")
    assert y.dtype == x.dtype and grads[0].dtype == x.dtype and grads[1].dtype == w.dtype


@pytest.mark.gpu
@pytest.mark.parametrize("use_w,use_b", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(cuda, use_w, use_b):
    x, dy, w, b = _case(37, 100, "f32", "f32")
    w, b = (w if use_w else None), (b if use_b else None)
    want, tol = _reference(x, w, b, dy, 1e-5)
    y, grads = _run(cuda, x, dy, w, b)
    _check(y, want[0], tol[0], "y")
    _check(grads[0], want[1], tol[1], "dx")
    if use_w:
        _check(grads[1], want[2], tol[2], "dw")
    if use_b:
        _check(grads[-1], want[3], tol[3], "db")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["pad", "offset", "transposed", "batched", "expanded", "skipped"])
def test_layouts(cuda, kind, layout):
    """Rows of wider buffers, odd starts, transposed and repeated inputs give the plain rows' results."""
    from gsr.layers import layer_norm
    g = torch.Generator().manual_seed(3)
    t = TYPES[kind]
    make = {"pad": lambda: torch.randn(20, 77, generator=g).to(t)[:, :70], "offset": lambda: torch.randn(20, 77, generator=g).to(t)[:, 3:],
            "transposed": lambda: torch.randn(16, 50, generator=g).to(t).T, "batched": lambda: torch.randn(3, 4, 33, generator=g).to(t),
            "expanded": lambda: torch.randn(1, 24, generator=g).to(t).expand(9, 24),
            "skipped": lambda: torch.randn(12, 60, generator=g).to(t)[:, ::2]}
    x = make[layout]()
    dim = x.shape[-1]
    w = torch.randn(dim, generator=g).to(t)
    dy = torch.randn(x.shape, generator=g).to(t)
    xg = x.to(cuda) if layout in ("batched",) else None
    if xg is None:   # keep the strides on the device
        base = {"pad": lambda: x._base.to(cuda)[:, :70], "offset": lambda: x._base.to(cuda)[:, 3:],
                "transposed": lambda: x._base.to(cuda).T, "expanded": lambda: x._base.to(cuda).expand(9, 24),
                "skipped": lambda: x._base.to(cuda)[:, ::2]}
        xg = base[layout]()
    xg = xg.detach().requires_grad_(True)
    y = layer_norm(xg, w.to(cuda))
    # the gradient arrives transposed as well
    dyg = dy.to(cuda).transpose(0, -1).contiguous().transpose(0, -1)
    (dx,) = torch.autograd.grad(y, [xg], dyg)
    want, tol = _reference(x.reshape(-1, dim), w, None, dy.reshape(-1, dim), 1e-5)
    _check(y.reshape(-1, dim), want[0], tol[0], "y")
    _check(dx.reshape(-1, dim), want[1], tol[1], "dx")


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """Central differences of a weighted sum in float64 steps of the fp32 forward: step h = 2^-6 on
    values of size 1 leaves h^2 curvature and u/h rounding, both below 2e-3 of the gradient's size."""
    from gsr.layers import layer_norm
    x, dy, w, b = _case(4, 24, "f32", "f32", seed=5)
    _, grads = _run(cuda, x, dy, w, b)
    h = 2.0 ** -6
    f = lambda x, w, b: float((layer_norm(x.to(cuda), w.to(cuda), b.to(cuda)).double().cpu() * dy.double()).sum())  # noqa: E731
    for which, grad in enumerate(grads):
        args = [x, w, b]
        flat = args[which].reshape(-1)
        for i in range(0, flat.numel(), 7):
            ends = []
            for s in (h, -h):
                moved = flat.clone()
                moved[i] += s
                ends.append(f(*[moved.view_as(a) if k == which else a for k, a in enumerate(args)]))
            slope = (ends[0] - ends[1]) / (2 * h)
            assert abs(slope - float(grad.reshape(-1)[i])) <= 4e-3 * (1 + float(grad.abs().max())), (which, i)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 700, 5000, 40000])
def test_rows_are_independent(cuda, dim):
    """NaN, infinite, huge and constant rows leave the others as they are."""
    x, dy, w, b = _case(8, dim, "f32", "f32", seed=1)
    y0, g0 = _run(cuda, x, dy, w, b)
    x2 = x.clone()
    x2[1, dim // 2] = float("nan")
    x2[3, 0] = float("inf")
    x2[5] = 2.0
    y, g = _run(cuda, x2, dy, w, b)
    for r in (0, 2, 4, 6, 7):
        assert torch.equal(y[r], y0[r]) and torch.equal(g[0][r], g0[0][r])
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().any()) and not bool(y[3].isfinite().all())
    assert torch.equal(y[5].cpu(), b) and bool(g[0][5].isfinite().all())


@pytest.mark.gpu
def test_large_offset(cuda):
    """Rows far from zero: the variance is taken about the mean (E[x^2] - mean^2 would lose it)."""
    x, dy, w, b = _case(6, 512, "f32", "f32", seed=2, offset=1000.0)
    want, tol = _reference(x, w, b, dy, 1e-5)
    y, g = _run(cuda, x, dy, w, b)
    _check(y, want[0], tol[0], "y")
    _check(g[0], want[1], tol[1], "dx")


@pytest.mark.gpu
def test_empty_and_same_bits(cuda):
    from gsr.layers import layer_norm
    w = torch.ones(12, device=cuda, requires_grad=True)
    x = torch.zeros(0, 12, device=cuda, requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert y.shape == (0, 12) and dx.shape == (0, 12) and bool((dw == 0).all())
    x, dy, w, b = _case(3000, 96, "f32", "f32")
    first = _run(cuda, x, dy, w, b)
    for _ in range(3):
        again = _run(cuda, x, dy, w, b)
        assert all(torch.equal(p, q) for p, q in zip([first[0], *first[1]], [again[0], *again[1]]))


@pytest.mark.gpu
def test_side_stream_and_graph(cuda):
    """A call on another stream, and a captured forward and backward replayed with new inputs."""
    from gsr.layers import layer_norm
    x, dy, w, b = (t.to(cuda) for t in _case(513, 200, "bf16", "f32"))

    def both(x):
        leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)]
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = both(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(x)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    buf = x.clone()
    with torch.cuda.stream(s):
        both(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(buf)
    for k in range(4):
        buf.copy_(x * (1 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(both(x * (1 + k)), out)), k


@pytest.mark.gpu
def test_module_matches_torch_checkpoint(cuda):
    from gsr.layers import LayerNorm
    a, b = torch.nn.LayerNorm(48), LayerNorm(48)
    with torch.no_grad():
        a.weight.uniform_(0.5, 1.5)
        a.bias.uniform_(-1, 1)
    b.load_state_dict(a.state_dict())
    x = torch.randn(9, 48)
    want, tol = _reference(x, a.weight.detach(), a.bias.detach(), x, 1e-5)
    _check(b.to(cuda)(x.to(cuda)), want[0], tol[0], "module")


def test_refusals():
    from gsr import _lib
    from gsr.layers import LayerNorm, layer_norm
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        layer_norm(x.double())
    with pytest.raises(ValueError, match="dim"):
        layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="dim"):
        layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match=r"weight must be \[8\]"):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="one type"):
        layer_norm(x, torch.ones(8), torch.zeros(8).half())
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="weight is on"):
        layer_norm(x, torch.ones(8, device="meta"))
    assert "bias=False" in repr(LayerNorm(4, bias=False))
    L = _lib.lib()
    bad = [((-1, 8, 8), b"bad rows"), ((4, 0, 8), b"bad dim"), ((4, 8, 7), b"row stride")]
    for (rows, dim, stride), msg in bad:
        assert L.gsr_layer_norm_fwd(None, rows, dim, stride, 0, None, None, 0, 1e-5, None, None, None) == -1
        assert msg in L.gsr_last_error()
        assert L.gsr_layer_norm_bwd(None, None, rows, dim, stride, stride, 0, None, 0, None, None, None, None, None, 0,
                                    None) == -1
    assert L.gsr_layer_norm_fwd(None, 4, 8, 8, 5, None, None, 0, 1e-5, None, None, None) == -1
    assert b"bad type" in L.gsr_last_error()
    assert L.gsr_layer_norm_fwd(None, 4, 8, 8, 0, None, None, 0, 1e-5, None, None, None) == -1
    assert b"null" in L.gsr_last_error()
    assert L.gsr_layer_norm_bwd(1, 1, 4, 8, 8, 8, 0, None, 0, 1, None, 1, None, None, 0, None) == -1
    assert b"workspace" in L.gsr_last_error()
    assert L.gsr_layer_norm_workspace(1000, 8, 0) > 0 and L.gsr_layer_norm_workspace(0, 8, 0) == 0
