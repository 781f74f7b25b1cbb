"""gsr.layers.gated_linear against its definition in 64 bits.

Tolerances (u = 2^-24; c(n) = (n + 16) u bounds an fp32 sum of n products, whatever its order;
inputs are exact, 16-bit products are exact in fp32).
    eg = c(D) sum|x||wg| + 2u|g|,  eu alike
    h   |u| 1.13 eg + |a| eu + k |a u|,        k = (16 + |g|) u, + 2^-20 in 16 bits (v_exp, v_rcp)
        (below, in 16 bits, eg + 2^-15 |g| and eu + 2^-15 |u|: a forward that keeps its projections
        truncates them to 24 bits, of which 8 are exponent and sign and 16 mantissa's)
    dg  |dh| (|s| eu + |u| e_s),  e_s = eg + k (1 + |g|);  du  |dh| (1.13 eg + k |a|)
        (|act'| <= 1.13 and |act''| <= 1 for the smooth ones; relu's slope is open within eg of 0)
    then half a step of the type where dg, du are rounded for the products (not for the biases)
    dx  sum_h (eg' |wg| + eu' |wu|) + c(2H) sum_h (|dg||wg| + |du||wu|);  dW, db alike over rows
plus half a step of the output's type."""
import pytest
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _act(kind, g):
    if kind == "relu":
        return g.clamp_min(0), (g > 0).double()
    if kind == "gelu":
        area = 0.5 * torch.special.erfc(-g / 2 ** 0.5)
        return g * area, area + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    s = torch.sigmoid(g)
    return (s, s * torch.sigmoid(-g)) if kind == "sigmoid" else (g * s, s + g * s * torch.sigmoid(-g))


def _reference(x, wg, wu, bg, bu, dh, kind, dtype):
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    zero = torch.zeros(wg.shape[0], dtype=torch.float64, device=x.device)
    bg, bu = (zero if b is None else b.double() for b in (bg, bu))
    c = lambda n: (n + 16) * U  # noqa: E731
    short = dtype != torch.float32
    half = torch.finfo(dtype).eps / 2
    g, u = x @ wg.T + bg, x @ wu.T + bu
    a, s = _act(kind, g)
    eg = c(x.shape[1]) * (x.abs() @ wg.abs().T + bg.abs()) + 2 * U * g.abs()
    eu = c(x.shape[1]) * (x.abs() @ wu.abs().T + bu.abs()) + 2 * U * u.abs()
    k = (16 + g.abs()) * U + (2.0 ** -20 if short else 0)
    th = u.abs() * 1.13 * eg + a.abs() * eu + k * (a * u).abs()
    if short:
        eg, eu = eg + 2.0 ** -15 * g.abs(), eu + 2.0 ** -15 * u.abs()
    es = (g.abs() <= eg).double() if kind == "relu" else eg + k * (1 + g.abs())
    dg, du = dh * u * s, dh * a
    tg, tu = dh.abs() * (s.abs() * eu + u.abs() * es) + 4 * U * dg.abs(), dh.abs() * (1.13 * eg + k * a.abs())
    # (fp16 operands below its normal range lose up to half of its smallest step)
    rg, ru = (tg + half * dg.abs() * 1.01, tu + half * du.abs() * 1.01) if short else (tg, tu)
    if dtype == torch.float16:
        rg, ru = rg + 2.0 ** -25, ru + 2.0 ** -25
    cr, ch = c(x.shape[0]), c(2 * wg.shape[0])
    values = [a * u, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dg.sum(0), du.sum(0)]
    tols = [th,
            (rg + ch * dg.abs()) @ wg.abs() + (ru + ch * du.abs()) @ wu.abs(),
            (rg + cr * dg.abs()).T @ x.abs(), (ru + cr * du.abs()).T @ x.abs(),
            (tg + cr * dg.abs()).sum(0), (tu + cr * du.abs()).sum(0)]
    return values, tols


def _check(got, want, tol, what):
    got = got.detach().to(want.device)
    info = torch.finfo(got.dtype)
    limit = tol + info.eps / 2 * want.abs() * 1.01 + info.smallest_normal * info.eps
    err = (got.double() - want).abs()
    assert got.shape == want.shape, what
    assert bool((err <= limit).all()), f"{what}: {float((err / limit).max()):.3g} of the tolerance"


def _case(rows, dim, hidden, kind, bias, seed):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[kind]
    mk = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(t)  # noqa: E731
    return [mk(rows, dim), mk(hidden, dim, scale=dim ** -0.5), mk(hidden, dim, scale=dim ** -0.5),
            mk(hidden, scale=0.3) if bias else None, mk(hidden, scale=0.3) if bias else None], mk(rows, hidden)


def _run(cuda, args, dh, act):
    from gsr.layers import gated_linear
    leaves = [None if t is None else t.to(cuda).requires_grad_(True) for t in args]
    h = gated_linear(*leaves, activation=act)
    return [h, *torch.autograd.grad(h, [t for t in leaves if t is not None], dh.to(cuda))]


NAMES = ("h", "dx", "dwg", "dwu", "dbg", "dbu")
SHAPES = [(1, 1, 1), (1, 8, 128), (2, 3, 5), (17, 8, 128), (64, 64, 64), (65, 33, 130), (130, 200, 65), (777, 129, 75),
          (1, 1000, 300), (16, 264, 520), (33, 72, 200), (300, 96, 256), (520, 512, 384), (1500, 8, 128), (4100, 16, 24),
          (40, 1024, 1030)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", SHAPES)
def test_forward_backward(cuda, rows, dim, hidden, kind):
    bias = (rows + dim) % 2 == 1
    act = ("silu", "gelu", "sigmoid")[(rows + hidden) % 3]
    args, dh = _case(rows, dim, hidden, kind, bias, rows * 7 + dim)
    want, tol = _reference(*args, dh, act, TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, act), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind} {act}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_activations(cuda, kind, act):
    """Every activation over a wide range of arguments, the saturated ends among them."""
    args, dh = _case(70, 48, 80, kind, True, 11)
    args[1] = args[1] * 6
    want, tol = _reference(*args, dh, act, TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, act), want, tol):
        _check(got, v, t, f"{name} {kind} {act}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["pad", "pad8", "offset", "transposed", "batched", "expanded_grad", "weight_view"])
def test_layouts(cuda, kind, layout):
    from gsr.layers import gated_linear
    (x, wg, wu, bg, bu), dh = _case(48, 40, 72, kind, True, 5)
    want, tol = _reference(x, wg, wu, bg, bu, dh, "silu", TYPES[kind])
    xg, wgg, wug, bgg, bug, dhg = (t.to(cuda) for t in (x, wg, wu, bg, bu, dh))

    def inside(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), device=cuda, dtype=t.dtype)
        wide[:, left:left + t.shape[1]] = t
        return wide[:, left:left + t.shape[1]]
    if layout == "pad":
        xg, dhg = inside(xg, 0, 5), inside(dhg, 0, 3)
    elif layout == "pad8":
        xg, dhg = inside(xg, 8, 8), inside(dhg, 8, 16)
    elif layout == "offset":
        xg, dhg = inside(xg, 1, 0), inside(dhg, 3, 0)
    elif layout == "transposed":
        xg, dhg = xg.T.contiguous().T, dhg.T.contiguous().T
    elif layout == "batched":
        xg, dhg = xg.view(4, 12, 40), dhg.view(4, 12, 72)
    elif layout == "expanded_grad":
        dhg = torch.ones((), device=cuda, dtype=x.dtype).expand(48, 72)
        want, tol = _reference(x, wg, wu, bg, bu, torch.ones_like(dh), "silu", TYPES[kind])
    elif layout == "weight_view":
        wgg, wug = inside(wgg, 4, 4), wug.T.contiguous().T
    leaves = [t.detach().requires_grad_(True) for t in (xg, wgg, wug, bgg, bug)]
    h = gated_linear(*leaves)
    out = [h, *torch.autograd.grad(h, leaves, dhg)]
    for name, got, v, t in zip(NAMES, out, want, tol):
        _check(got.reshape(v.shape), v, t, f"{name} {kind} {layout}")


WIDE = [(3, 4096, 8200), (3000, 1100, 4100), (4096, 64, 1024), (4100, 72, 1025), (4097, 65, 1100), (8192, 200, 600), (300, 130, 8256), (4864, 512, 1030),
        (2049, 320, 2000)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", WIDE)
def test_large_cases(cuda, rows, dim, hidden, kind):
    """Tiles of 256 and 128: whole and ragged ones in every direction, cut along K, dims that need padded copies."""
    args, dh = _case(rows, dim, hidden, kind, rows % 2 == 0, rows + dim)
    args[0] = args[0] * 2 ** -3   # (keeps fp16's sums over thousands of rows in range)
    want, tol = _reference(*(None if t is None else t.to(cuda) for t in args), dh.to(cuda), "silu", TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, "silu"), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_largest_tiles(cuda, kind):
    """Enough steps for tiles of 256 in all products, ragged ones, and a last round cut along K; and the same
    backward without what the forward kept, which computes the projections again."""
    from gsr import _lib
    rows, dim, hidden = 8200, 2056, 4104
    args, dh = _case(rows, dim, hidden, kind, True, 77)
    args, dh = [t.to(cuda) for t in args], dh.to(cuda)
    args[0] = args[0] * 2 ** -3
    want, tol = _reference(*args, dh, "silu", TYPES[kind])
    out = _run(cuda, args, dh, "silu")
    for name, got, v, t in zip(NAMES, out, want, tol):
        _check(got, v, t, f"{name} {kind}")
    L, code = _lib.lib(), {"bf16": _lib.BF16, "f16": _lib.F16}[kind]
    assert L.gsr_gated_kept(rows, dim, hidden, code) >= 6 * rows * hidden
    grads = [torch.empty_like(t) for t in args]
    ws = torch.empty(L.gsr_gated_workspace(rows, dim, hidden, code, 1), device=cuda, dtype=torch.uint8)
    x, wg, wu, bg, bu = (t.data_ptr() for t in args)
    _lib.check(L.gsr_gated_bwd(x, rows, dim, dim, code, wg, wu, hidden, bg, bu, 0, dh.data_ptr(), hidden, None,
                               *(g.data_ptr() for g in grads), ws.data_ptr(), ws.numel(),
                               torch.cuda.current_stream().cuda_stream), "gsr_gated_bwd")
    for name, got, v, t in zip(NAMES[1:], grads, want[1:], tol[1:]):
        _check(got, v, t, f"{name} {kind}, computed again")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_large_views(cuda, kind):
    """Large rows at odd addresses and inside wider buffers of NaN: nothing outside is read into a result."""
    from gsr.layers import gated_linear
    (x, wg, wu, _, _), dh = _case(4100, 72, 1032, kind, False, 8)
    leaves = [t.to(cuda).requires_grad_(True) for t in (x, wg, wu)]
    h = gated_linear(*leaves)
    want = [h, *torch.autograd.grad(h, leaves, dh.to(cuda))]
    for left, right in ((0, 8), (8, 0), (1, 2)):
        def inside(t):
            wide = torch.full((t.shape[0] + 1, left + t.shape[1] + right), float("nan"), device=cuda, dtype=t.dtype)
            wide[:-1, left:left + t.shape[1]] = t.to(cuda)
            return wide[:-1, left:left + t.shape[1]]
        leaves = [t.detach().requires_grad_(True) for t in (inside(x), leaves[1], leaves[2])]
        h = gated_linear(*leaves)
        got = [h, *torch.autograd.grad(h, leaves, inside(dh))]
        assert all(torch.equal(a, b) for a, b in zip(want, got)), (left, right)


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """Central differences (h = 2^-5, arguments of size 1): curvature leaves h^2/6 of third derivatives of
    size 1 and rounding 16 u / h of sums of 20 terms, both below 2e-3 of the largest slope."""
    from gsr.layers import gated_linear
    args, dh = _case(5, 7, 20, "f32", True, 3)
    grads = _run(cuda, args, dh, "silu")[1:]
    f = lambda a: float((gated_linear(*[t.to(cuda) for t in a]).double().cpu() * dh.double()).sum())  # noqa: E731
    h = 2.0 ** -5
    for which, grad in enumerate(grads):
        flat = args[which].reshape(-1)
        for i in range(0, flat.numel(), 11):
            ends = []
            for s in (h, -h):
                moved = flat.clone()
                moved[i] += s
                ends.append(f([moved.view_as(a) if k == which else a for k, a in enumerate(args)]))
            slope = (ends[0] - ends[1]) / (2 * h)
            assert abs(slope - float(grad.reshape(-1)[i])) <= 2e-3 * (1 + float(grad.abs().max())), (which, i)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", [(70, 40, 72), (3, 64, 96), (300, 128, 300), (4096, 72, 1024)])
def test_bad_rows_stay_alone(cuda, kind, rows, dim, hidden):
    """A NaN or infinite row reaches its own outputs and input gradient, and no other row's."""
    args, dh = _case(rows, dim, hidden, kind, False, 9)
    first = _run(cuda, args, dh, "silu")
    args[0] = args[0].clone()
    args[0][1, 3] = float("nan")
    args[0][rows - 1, 0] = float("inf")
    again = _run(cuda, args, dh, "silu")
    keep = torch.ones(rows, dtype=torch.bool)
    keep[1] = keep[rows - 1] = False
    for k in (0, 1):
        assert torch.equal(first[k].cpu()[keep], again[k].cpu()[keep])
        assert bool(again[k][1].isnan().all()) and not bool(again[k][rows - 1].isfinite().all())
    assert not bool(again[2].isfinite().any()) or bool(again[2].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_no_rows(cuda, kind):
    args, dh = _case(0, 12, 20, kind, True, 1)
    out = _run(cuda, args, dh, "silu")
    assert out[0].shape == (0, 20) and out[1].shape == (0, 12)
    assert all(bool((g == 0).all()) for g in out[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,hidden,kind", [(600, 200, 136, "bf16"), (2000, 8, 128, "f32"), (1, 512, 640, "bf16"),
                                                  (1024, 512, 512, "bf16"), (1024, 256, 512, "f32"),
                                                  (4200, 136, 1000, "bf16"), (4100, 65, 1030, "f16")])
def test_same_bits_streams_and_graph(cuda, rows, dim, hidden, kind):
    """Repeated calls, a call on another stream and a captured pass replayed with new inputs give the same bits."""
    from gsr.layers import gated_linear
    args, dh = _case(rows, dim, hidden, kind, True, 21)
    x, wg, wu, bg, bu = (t.to(cuda) for t in args)
    dh = dh.to(cuda)

    def both(x):
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
        h = gated_linear(*leaves, activation="gelu")
        return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

    want = both(x)
    assert all(torch.equal(a, b) for a, b in zip(want, both(x)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    buf = x.clone()
    with torch.cuda.stream(side):
        got = both(buf)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(buf)
    for k in range(4):
        new = x * (0.5 + k)
        buf.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(both(new), out)), k


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    """Two passes in flight on two streams keep their own workspaces."""
    from gsr.layers import gated_linear
    jobs = []
    for k in range(2):
        args, dh = _case(900, 256, 320, "bf16", False, 30 + k)
        jobs.append(([t.to(cuda).requires_grad_(True) for t in args[:3]], dh.to(cuda), torch.cuda.Stream()))
    run = lambda leaves, dh: torch.autograd.grad(gated_linear(*leaves), leaves, dh)  # noqa: E731
    want = [run(leaves, dh) for leaves, dh, _ in jobs]
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for _ in range(5):
        for k, (leaves, dh, s) in enumerate(jobs):
            with torch.cuda.stream(s):
                got[k].append(run(leaves, dh))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for r in got[k] for a, b in zip(want[k], r))


@pytest.mark.gpu
def test_some_gradients_only_and_refused_twice(cuda):
    from gsr.layers import gated_linear, layer_norm
    args, dh = _case(50, 24, 40, "f32", True, 2)
    full = _run(cuda, args, dh, "silu")
    for which in range(5):
        leaves = [t.to(cuda).requires_grad_(k == which) for k, t in enumerate(args)]
        h = gated_linear(*leaves)
        (g,) = torch.autograd.grad(h, [leaves[which]], dh.to(cuda))
        assert torch.equal(g, full[1 + which])
    leaves = [t.to(cuda).requires_grad_(True) for t in args]
    for f in (lambda: gated_linear(*leaves), lambda: layer_norm(leaves[0])):
        (g,) = torch.autograd.grad(f().square().sum(), leaves[:1], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiat"):
            torch.autograd.grad(g.sum(), leaves[:1])


@pytest.mark.gpu
def test_head_trains(cuda):
    """The parameter head through the framework's own path: selection, norm, gated block, projection and pose
    to renderer rows, one optimizer step; gradients against the same network in 64 bits."""
    from gsr.head import GatedHead, params_from_volume_3d, select_gaussians
    from gsr.optim import AdamW
    torch.manual_seed(0)
    c, M = 8, 24 ** 3
    head = GatedHead(c, 48).to(cuda)
    volume = torch.randn(c, M, device=cuda)
    grid = (torch.rand(M, 3, device=cuda) - 0.5) * 0.18
    scale = torch.tensor([-5.5], device=cuda)
    opt = AdamW(head.parameters(), lr=1e-3, moment_bits=8)
    out = params_from_volume_3d(volume, head, grid, scale, angle=0.4, p_3d=torch.tensor([0.0, 0.1, 0.0]))
    cot = torch.randn_like(out)
    before = [p.detach().clone() for p in head.parameters()]
    (out * cot).sum().backward()
    assert all(bool(p.grad.isfinite().all()) and bool(p.grad.abs().max() > 0) for p in head.parameters())
    opt.step()
    assert all(not torch.equal(p, q) for p, q in zip(before, head.parameters()))
    # the network alone, against 64 bits
    idx, _ = select_gaussians(volume[0])
    x = volume.index_select(1, idx).T
    for p, q in zip(head.parameters(), before):
        p.data.copy_(q)
        p.grad = None
    net = head(x)
    cot = torch.randn_like(net)
    (net * cot).sum().backward()
    n, gt = head.norm, head.gated
    leaf = {k: p.detach().double().cpu().requires_grad_(True) for k, p in head.named_parameters()}
    xd = x.double().cpu()
    z = torch.nn.functional.layer_norm(xd, (c,), leaf["norm.weight"], leaf["norm.bias"], n.eps)
    hd = torch.nn.functional.silu(z @ leaf["gated.w_gate"].T + leaf["gated.b_gate"]) * (z @ leaf["gated.w_up"].T + leaf["gated.b_up"])
    want = hd @ leaf["out.weight"].T + leaf["out.bias"]
    (want * cot.double().cpu()).sum().backward()
    assert gt.hidden == 48
    # sums of up to 4000 rows of fp32 products of sums of 48: relative to the largest, 4096 u
    assert float((net.detach().double().cpu() - want.detach()).abs().max()) <= 256 * U * float(want.detach().abs().max()) * 4
    for k, p in head.named_parameters():
        assert float((p.grad.double().cpu() - leaf[k].grad).abs().max()) <= 4096 * U * float(leaf[k].grad.abs().max()) + 1e-5, k


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", [(100, 4000, 1000), (70, 1001, 517), (300, 2056, 700), (129, 1024, 64), (500, 1000, 1000),
                                             (65, 4096, 1)])
def test_few_tiles(cuda, rows, dim, hidden, kind):
    """Long rows and few tiles: every product's K in shares, the forward's among them."""
    bias = rows % 2 == 1
    act = ("silu", "gelu", "sigmoid")[hidden % 3]
    args, dh = _case(rows, dim, hidden, kind, bias, rows + dim)
    want, tol = _reference(*args, dh, act, TYPES[kind])
    out = _run(cuda, args, dh, act)
    for name, got, v, t in zip(NAMES, out, want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind} {act}")
    again = [a.clone() if k == 0 else a for k, a in enumerate(args)]
    again[0][3, 5] = float("nan")
    keep = torch.arange(rows) != 3
    bad = _run(cuda, again, dh, act)
    for k in (0, 1):
        assert torch.equal(bad[k].cpu()[keep], out[k].cpu()[keep]) and bool(bad[k][3].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", [(60, 2699, 800), (5, 2501, 900), (17, 2050, 1027), (64, 300, 7001), (1, 4095, 601)])
def test_few_odd_rows(cuda, rows, dim, hidden, kind):
    """Up to 64 rows of odd length: with a backward to follow (kept projections and copies) and without."""
    from gsr.layers import gated_linear
    bias = rows % 2 == 1
    act = ("silu", "gelu", "sigmoid")[rows % 3]
    args, dh = _case(rows, dim, hidden, kind, bias, rows + dim)
    want, tol = _reference(*args, dh, act, TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, act), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind} {act}")
    with torch.no_grad():
        h = gated_linear(*(None if a is None else a.to(cuda) for a in args), activation=act)
    _check(h, want[0], tol[0], f"h alone {rows}x{dim}->{hidden} {kind} {act}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", [(300, 301, 300), (777, 509, 200), (200, 264, 136), (4200, 129, 1000)])
def test_without_what_the_forward_keeps(cuda, rows, dim, hidden, kind):
    """The C ABI's backward where the caller kept nothing: everything is made again."""
    from gsr import _lib
    L, t = _lib.lib(), {"f32": _lib.F32, "bf16": _lib.BF16, "f16": _lib.F16}[kind]
    args, dh = _case(rows, dim, hidden, kind, True, 21)
    want, tol = _reference(*args, dh, "silu", TYPES[kind])
    dev = [v.to(cuda) for v in (*args, dh)]
    out = [torch.full(s, float("nan"), device=cuda, dtype=TYPES[kind])
           for s in ((rows, hidden), (rows, dim), (hidden, dim), (hidden, dim), (hidden,), (hidden,))]
    x, wg, wu, bg, bu, d = (v.data_ptr() for v in dev)
    stream = torch.cuda.current_stream().cuda_stream
    ws = [torch.empty(max(1, L.gsr_gated_workspace(rows, dim, hidden, t, b)), device=cuda, dtype=torch.uint8) for b in (0, 1)]
    _lib.check(L.gsr_gated_fwd(x, rows, dim, dim, t, wg, wu, hidden, bg, bu, 0, out[0].data_ptr(), None, ws[0].data_ptr(),
                               ws[0].numel(), stream), "gsr_gated_fwd")
    _lib.check(L.gsr_gated_bwd(x, rows, dim, dim, t, wg, wu, hidden, bg, bu, 0, d, hidden, None, *(o.data_ptr() for o in out[1:]),
                               ws[1].data_ptr(), ws[1].numel(), stream), "gsr_gated_bwd")
    for name, got, v, lim in zip(NAMES, out, want, tol):
        _check(got, v, lim, f"{name} {rows}x{dim}->{hidden} {kind}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 256])
def test_more_rows_than_a_grid_side(cuda, dim):
    """4.2 million rows (65536 blocks of 64 and more): the first and last ones against the definition, the
    bias gradient against a sum of what the rows give."""
    from gsr.layers import gated_linear
    rows, hidden = 65536 * 64 + 100, 8
    g = torch.Generator(device=cuda).manual_seed(1)
    (_, wg, wu, bg, bu), _ = _case(1, dim, hidden, "bf16", True, 4)
    x = torch.randn(rows, dim, device=cuda, generator=g, dtype=torch.bfloat16)
    dh = torch.randn(rows, hidden, device=cuda, generator=g, dtype=torch.bfloat16)
    leaves = [x.requires_grad_(True)] + [t.to(cuda).requires_grad_(True) for t in (wg, wu, bg, bu)]
    h = gated_linear(*leaves)
    dx, db = torch.autograd.grad(h, [leaves[0], leaves[4]], dh)
    for at in (slice(0, 100), slice(rows - 200, rows)):
        want, tol = _reference(x.detach()[at].cpu(), wg, wu, bg, bu, dh[at].cpu(), "silu", torch.bfloat16)
        _check(h[at], want[0], tol[0], "h")
        _check(dx[at], want[1], tol[1], "dx")
    gate = torch.nn.functional.silu(x.detach().double() @ wg.to(cuda).double().T + bg.to(cuda).double())
    terms = dh.double() * gate
    # (each term is off by at most 2^-12 of |dh| (1 + |gate|), their sum by c(rows) of sum|terms|, then bf16)
    limit = 2.0 ** -12 * (dh.double().abs() * (1 + gate.abs())).sum(0) + (rows + 16) * U * terms.abs().sum(0)
    assert bool(((db.double() - terms.sum(0)).abs() <= limit + 2.0 ** -8 * terms.sum(0).abs()).all())


# dim <= 15: one row, one column; rows that end inside 16 and 64; each width of a step of 4; few rows and many columns
# (dx in shares); more row tiles than workgroups
NARROW = [(1, 15, 2050), (15, 4, 16), (64, 7, 17), (70, 15, 400), (129, 12, 128), (400, 2, 1000), (20000, 1, 7), (33100, 5, 40),
          (40000, 15, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,dim,hidden", NARROW)
def test_narrow(cuda, rows, dim, hidden, kind):
    bias = dim % 2 == 1
    act = ("silu", "gelu", "sigmoid")[rows % 3]
    args, dh = _case(rows, dim, hidden, kind, bias, rows + dim)
    want, tol = _reference(*args, dh, act, TYPES[kind])
    for name, got, v, t in zip(NAMES, _run(cuda, args, dh, act), want, tol):
        _check(got, v, t, f"{name} {rows}x{dim}->{hidden} {kind} {act}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows", [50, 300])
def test_narrow_views_and_parts(cuda, kind, rows):
    """Rows of wider buffers that hold NaN around them, at odd addresses, give the same bits; so does a
    backward pass that is asked for one gradient only."""
    from gsr.layers import gated_linear
    args, dh = _case(rows, 9, 205, kind, True, 3)
    full = _run(cuda, args, dh, "silu")

    def inside(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), device=cuda, dtype=t.dtype)
        wide[:, left:left + t.shape[1]] = t
        return wide[:, left:left + t.shape[1]]
    leaves = [inside(args[0].to(cuda), 1, 2).requires_grad_(True)] + [t.to(cuda).requires_grad_(True) for t in args[1:]]
    h = gated_linear(*leaves)
    for a, b in zip(full, [h, *torch.autograd.grad(h, leaves, inside(dh.to(cuda), 3, 1))]):
        assert torch.equal(a, b)
    for which in range(5):
        leaves = [t.to(cuda).requires_grad_(k == which) for k, t in enumerate(args)]
        (g,) = torch.autograd.grad(gated_linear(*leaves), [leaves[which]], dh.to(cuda))
        assert torch.equal(g, full[1 + which])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows", [40, 300])
def test_narrow_bad_values_stay_alone(cuda, kind, rows):
    """A row of x that is not finite reaches its own dx and no other row's; a weight row that is not
    finite its own gradients and no other weight row's, also where rows end inside a tile."""
    args, dh = _case(rows, 6, 70, kind, True, 9)
    first = _run(cuda, args, dh, "silu")
    bad = [t.clone() for t in args]
    bad[0][1, 3], bad[0][rows - 1, 0] = float("nan"), float("inf")
    again = _run(cuda, bad, dh, "silu")
    keep = torch.ones(rows, dtype=torch.bool)
    keep[1] = keep[rows - 1] = False
    for k in (0, 1):
        assert torch.equal(first[k].cpu()[keep], again[k].cpu()[keep])
        assert bool(again[k][1].isnan().all()) and not bool(again[k][rows - 1].isfinite().all())
    bad = [t.clone() for t in args]
    bad[1][20, 2], bad[4][60] = float("nan"), float("inf")
    again = _run(cuda, bad, dh, "silu")
    keep = torch.ones(70, dtype=torch.bool)
    keep[20] = keep[60] = False
    assert torch.equal(first[0].cpu()[:, keep], again[0].cpu()[:, keep])
    for k in (2, 3, 4, 5):
        assert torch.equal(first[k].cpu()[keep], again[k].cpu()[keep])
    assert bool(again[2][20].isnan().all())


def test_refusals():
    from gsr import _lib
    from gsr.layers import GatedLinear, gated_linear
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear(f(4, 8), f(6, 8), f(6, 8))
    with pytest.raises(ValueError, match="activation"):
        gated_linear(f(4, 8), f(6, 8), f(6, 8), activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        GatedLinear(4, 8, "swish")
    with pytest.raises(ValueError, match=r"\[hidden, 8\]"):
        gated_linear(f(4, 8), f(6, 7), f(6, 7))
    with pytest.raises(ValueError, match=r"\[hidden, 8\]"):
        gated_linear(f(4, 8), f(6, 8), f(5, 8))
    with pytest.raises(ValueError, match=r"\[hidden, 8\]"):
        gated_linear(f(4, 8), f(0, 8), f(0, 8))
    with pytest.raises(ValueError, match="dim >= 1"):
        gated_linear(f(4, 0), f(6, 0), f(6, 0))
    with pytest.raises(ValueError, match="go together"):
        gated_linear(f(4, 8), f(6, 8), f(6, 8), f(6))
    with pytest.raises(ValueError, match="biases must be"):
        gated_linear(f(4, 8), f(6, 8), f(6, 8), f(5), f(5))
    with pytest.raises(ValueError, match="x's type"):
        gated_linear(f(4, 8), f(6, 8), f(6, 8).half())
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        gated_linear(f(4, 8).double(), f(6, 8).double(), f(6, 8).double())
    with pytest.raises(ValueError, match="is on"):
        gated_linear(f(4, 8), torch.zeros(6, 8, device="meta"), f(6, 8))
    with pytest.raises(ValueError, match="2\\^26"):
        gated_linear(f(1, 1).expand(1 << 27, 1), f(1, 1), f(1, 1))
    L = _lib.lib()
    fwd = lambda rows=4, dim=8, stride=8, t=0, hidden=6, act=0: L.gsr_gated_fwd(  # noqa: E731
        None, rows, dim, stride, t, None, None, hidden, None, None, act, None, None, None, 0, None)
    for kw, msg in [(dict(rows=-1), b"bad rows"), (dict(dim=0), b"bad dim"), (dict(hidden=0), b"bad dim"),
                    (dict(stride=7), b"row stride"), (dict(t=3), b"bad type"), (dict(act=4), b"bad activation"),
                    ({}, b"null pointer"), (dict(hidden=1 << 21), b"bad dim")]:
        assert fwd(**kw) == -1 and msg in L.gsr_last_error(), kw
    bwd = lambda ws, n, dh=1: L.gsr_gated_bwd(1, 4, 24, 24, 0, 1, 1, 6, None, None, 0, dh, 6, None, 1, 1, 1, None, None, ws,  # noqa: E731
                                              n, None)
    assert bwd(1, 16) == -1 and b"workspace" in L.gsr_last_error()
    assert bwd(1, 1 << 20, dh=None) == -1 and b"null" in L.gsr_last_error()
    assert L.gsr_gated_workspace(4, 24, 6, 0, 1) >= 4 * 128 * 4 and L.gsr_gated_workspace(4, 24, 6, 7, 1) == 0
    assert L.gsr_gated_workspace(4, 8, 6, 1, 0) == 0 and L.gsr_gated_workspace(0, 8, 6, 1, 1) == 0
