"""gsr.optim's AdamW step against its formula in 64 bits.

Tolerances (u = 2^-24).  m and v are two products and a sum: 3 u of |b1 m| + |(1-b1) g| (both
terms' magnitudes) and 4 u of v.  The step's quotient adds the root's u, the denominator's 2 u and
two more, so p is off by at most u (2 |p| + 12 |step|) plus m's own error over the denominator,
plus half a step of p's type.  An 8-bit moment is off by half a step of its code: e4m3 2^-4
relative and 2^-10 units below its normal range; a root 2^-5 relative, half a unit below 16
units, and a whole unit where a root that is not zero is kept from vanishing; a value next to a
border between codes may take either, which is the same half step (1 + 2^-20)."""
import copy

import pytest
import torch

U = 2.0 ** -24
ARGS = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LEVELS = torch.tensor([float(k) for k in range(16)] + [float((16 + k) << e) for e in range(15) for k in range(16)],
                      dtype=torch.float64)


def _units(n):
    return -(-n // 256)


def _spread(u, n):
    return u.double().repeat_interleave(256)[:n]


def _formula(p, g, m, v, step, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v2 / (1 - b2 ** step)).sqrt() + eps
    delta = lr * m2 / (1 - b1 ** step) / denom
    m_err = 3 * U * (abs(b1) * m.abs() + (1 - b1) * g.abs())
    tol_p = U * (2 * p.abs() + 12 * delta.abs()) + lr / (1 - b1 ** step) * m_err / denom
    return p * (1 - lr * weight_decay) - delta, m2, v2, tol_p, m_err


def _inputs(shape, ptype, gtype, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(2 * torch.randn(shape, generator=g) - 3) * (torch.rand(shape, generator=g) > 0.1)
    p = torch.randn(shape, generator=g).to(TYPES[ptype])
    grad = (torch.randn(shape, generator=g) * size).to(TYPES[gtype])
    m = torch.randn(shape, generator=g) * size * 0.3
    v = torch.rand(shape, generator=g) * size * size
    return p, grad, m, v


def _codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.Size(shape).numel()
    m = (torch.randn(shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    v = torch.randint(0, 256, shape, generator=g).to(torch.uint8)
    mu = torch.rand(_units(n), generator=g) * 1e-4
    vu = torch.rand(_units(n), generator=g) * 1e-7
    return m, v, mu, vu


def _within(err, tol, what):
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max()):.3g} of the tolerance"


SHAPES = [[(1,)], [(255,), (256,), (257,)], [(14, 128), (14,), (3, 5, 7), (2049,)], [(100, 14), (0, 3), (4097,), ()]]


@pytest.mark.gpu
@pytest.mark.parametrize("ptype,gtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("shapes", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("step", [1, 7])
def test_step_32(cuda, shapes, ptype, gtype, step):
    from gsr.optim import adamw_step
    cpu = [_inputs(s, ptype, gtype, 10 * i + step) for i, s in enumerate(shapes)]
    dev = [[t.to(cuda) for t in c] for c in cpu]
    adamw_step(*[list(x) for x in zip(*dev)], step=step, **ARGS)
    for (p, g, m, v), (p2, g2, m2, v2) in zip(cpu, dev):
        wp, wm, wv, tp, tm = _formula(*(t.double() for t in (p, g, m, v)), step, **ARGS)
        half = torch.finfo(p.dtype).eps / 2
        tiny = 1e-40   # products below fp32's normal range
        _within((m2.cpu().double() - wm).abs(), tm + tiny, "m")
        _within((v2.cpu().double() - wv).abs(), 4 * U * wv + tiny, "v")
        _within((p2.cpu().double() - wp).abs(), tp + half * wp.abs() * (1 + 2 ** -7) + torch.finfo(p.dtype).tiny, "p")
        assert torch.equal(g2.cpu(), g)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype,gtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("shapes", SHAPES[:3], ids=["one", "borders", "several"])
def test_step_8(cuda, shapes, ptype, gtype):
    from gsr.optim import adamw_step, decode_root
    step = 5
    for i, shape in enumerate(shapes):
        p, g, _, _ = _inputs(shape, ptype, gtype, i)
        n = p.numel()
        mc, vc, mu, vu = _codes(shape, 50 + i)
        d = [t.to(cuda) for t in (p, g, mc, vc, mu, vu)]
        m = mc.float().double().reshape(-1) * _spread(mu, n)
        v = (LEVELS[vc.reshape(-1).long()] * _spread(vu, n)).square()
        assert torch.allclose(decode_root(d[3], d[5]).cpu().double().reshape(-1), v.sqrt(), rtol=2 * U, atol=0)
        adamw_step([d[0]], [d[1]], [d[2]], [d[3]], exp_avg_units=[d[4]], exp_avg_root_units=[d[5]], step=step, **ARGS)
        wp, wm, wv, tp, tm = _formula(p.double().reshape(-1), g.double().reshape(-1), m, v, step, **ARGS)
        # the stored moments carry a rounding more than fp32 ones: m's and v's units, r * r
        tp, tm = 2 * tp, 2 * tm
        half = torch.finfo(p.dtype).eps / 2
        _within((d[0].cpu().double().reshape(-1) - wp).abs(), tp + half * wp.abs() * (1 + 2 ** -7) + torch.finfo(p.dtype).tiny, "p")
        nmu, nvu = d[4].cpu(), d[5].cpu()
        pad = _units(n) * 256 - n
        top = lambda t: torch.nn.functional.pad(t.abs(), (0, pad)).view(-1, 256).amax(1)  # noqa: E731
        assert torch.allclose(nmu.double(), top(wm) / 448, rtol=16 * U, atol=0)
        assert torch.allclose(nvu.double(), top(wv.sqrt()) / 507904, rtol=16 * U, atol=0)
        got_m = d[2].cpu().float().double().reshape(-1) * _spread(nmu, n)
        _within((got_m - wm).abs(), (1 + 2 ** -20) * (2 ** -4 * wm.abs() + 2 ** -10 * _spread(nmu, n)) + tm, "m")
        got_r, want_r, unit = LEVELS[d[3].cpu().reshape(-1).long()] * _spread(nvu, n), wv.sqrt(), _spread(nvu, n)
        _within((got_r - want_r).abs(), (1 + 2 ** -20) * torch.maximum(2 ** -5 * want_r, unit) + 8 * U * want_r, "root")
        assert bool(((got_r > 0) == (want_r > 0)).all())


def _nearest_root(q):
    """The code whose level is nearest q, ties to the even step."""
    d = (LEVELS[None] - q[:, None]).abs()
    best = d.amin(1, keepdim=True)
    even = (torch.arange(256) % 2 == 0)[None]
    return torch.where(d == best, torch.where(even, 0, 1), 9).argmin(1)


@pytest.mark.gpu
def test_root_codes_are_the_nearest(cuda):
    """Every level, every midpoint and their neighbours, through a step that changes nothing (b2 v alone:
    g = 0 and b2 scaled out by the block's own unit)."""
    from gsr.optim import adamw_step
    q = torch.cat([LEVELS, (LEVELS[1:] + LEVELS[:-1]) / 2]).float()
    # v = b2 v0 + (1 - b2) g^2 with b2 = 0 and g = q exactly representable: root = |q| where q^2 is exact
    q = q[(q.double() ** 2) == (q ** 2).double()]
    blocks = []
    for i in range(0, q.numel(), 255):
        part = q[i:i + 255]
        blocks.append(torch.cat([torch.tensor([507904.0]), part, torch.zeros(255 - part.numel())]))
    g = torch.cat(blocks)
    n = g.numel()
    p, mc, vc = torch.zeros(n, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda)
    mu, vu = torch.zeros(_units(n), device=cuda), torch.zeros(_units(n), device=cuda)
    adamw_step([p], [g.to(cuda)], [mc.view(torch.float8_e4m3fn)], [vc], exp_avg_units=[mu], exp_avg_root_units=[vu],
               step=1, lr=1e-3, betas=(0.9, 0.0), eps=1e-8, weight_decay=0.0)
    assert bool((vu.cpu() - 1).abs().max() <= U)
    want = _nearest_root(g.double())
    want = torch.where((g > 0) & (want == 0), 1, want)
    got = vc.cpu().long()
    near_tie = torch.zeros(n, dtype=torch.bool) if bool((vu.cpu() == 1).all()) else None
    if near_tie is not None:
        assert torch.equal(got, want)
    assert bool(((got - want).abs() <= 1).all())


@pytest.mark.gpu
def test_zero_blocks_and_bad_gradients(cuda):
    """A zero block stays zero; a NaN gradient reaches its own block (8 bits) or element (32) and no other;
    elements behind a tensor's end keep what they hold."""
    from gsr.optim import adamw_step
    n = 700
    big = torch.full((n + 300,), 5.0, device=cuda)
    p = big[:n]
    g = torch.zeros(n, device=cuda)
    g[300] = float("nan")
    codes = torch.full((n + 300,), 7, dtype=torch.uint8, device=cuda)
    codes[:n] = 0
    roots = codes.clone()
    mu, vu = torch.zeros(3, device=cuda), torch.zeros(3, device=cuda)
    adamw_step([p], [g], [codes[:n].view(torch.float8_e4m3fn)], [roots[:n]], exp_avg_units=[mu], exp_avg_root_units=[vu],
               step=1, lr=1e-2, weight_decay=0.0)
    keep = torch.ones(n, dtype=torch.bool)
    keep[300] = False
    assert bool((p.cpu()[keep] == 5).all()) and bool(p[300].isnan()) and bool((big[n:] == 5).all())
    assert bool((codes[n:] == 7).all()) and bool((roots[n:] == 7).all())
    assert bool((codes[:256] == 0).all()) and bool((roots[512:n] == 0).all()) and float(mu[0]) == 0 and float(vu[2]) == 0
    assert bool(mu[1].isnan()) and bool(vu[1].isnan())
    m, v, q = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda), torch.full((n,), 5.0, device=cuda)
    adamw_step([q], [g], [m], [v], step=1, lr=1e-2, weight_decay=0.0)
    assert int(m.isnan().sum()) == 1 and int(v.isnan().sum()) == 1 and int(q.isnan().sum()) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("count", [55, 56, 57, 130])
def test_many_tensors(cuda, count):
    """More tensors than one launch's arguments hold; every one gets the single tensor's bits."""
    from gsr.optim import adamw_step
    cpu = [_inputs((1 + 37 * i % 700,), "f32", "f32", i) for i in range(count)]
    dev = [[t.to(cuda) for t in c] for c in cpu]
    adamw_step(*[list(x) for x in zip(*dev)], step=3, **ARGS)
    for c, d in zip(cpu, dev):
        one = [t.to(cuda) for t in c]
        adamw_step(*[[t] for t in one], step=3, **ARGS)
        assert all(torch.equal(a, b) for a, b in zip(one, d))


@pytest.mark.gpu
def test_misaligned_and_permuted(cuda):
    """Views that start anywhere, transposed parameters, gradients of another layout."""
    from gsr.optim import adamw_step
    p, g, m, v = _inputs((33, 21), "f32", "f32", 4)
    want = [t.to(cuda) for t in (p, g, m, v)]
    adamw_step(*[[t] for t in want], step=2, **ARGS)
    moved = []
    for t in (p, g, m, v):
        buf = torch.zeros(t.numel() + 3, device=cuda)
        buf[3:] = t.reshape(-1).to(cuda)
        moved.append(buf[3:].view(t.shape))
    adamw_step(*[[t] for t in moved], step=2, **ARGS)
    assert all(torch.equal(a, b) for a, b in zip(want, moved))
    turned = [t.T.contiguous().T.to(cuda) for t in (p, m, v)]
    assert not turned[0].is_contiguous()
    adamw_step([turned[0]], [g.to(cuda)], [turned[1]], [turned[2]], step=2, **ARGS)
    assert torch.equal(turned[0], want[0]) and torch.equal(turned[1], want[2]) and torch.equal(turned[2], want[3])


def _model():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(8, 40), torch.nn.ReLU(), torch.nn.Linear(40, 14))


def _train(model, opt, steps, x):
    for k in range(steps):
        opt.zero_grad()
        (model(x) - k).square().mean().backward()
        opt.step()


@pytest.mark.gpu
def test_optimizer_follows_torch(cuda):
    """Ten steps beside torch.optim.AdamW from the same start: each step's p differs by the two sides' own
    rounding, 32 u of |p| + lr a step at most, and gradients of nearby weights by as much again."""
    from gsr.optim import AdamW
    a = _model().to(cuda)
    b = copy.deepcopy(a)
    x = torch.randn(64, 8, generator=torch.Generator().manual_seed(1)).to(cuda)
    _train(a, torch.optim.AdamW(a.parameters(), lr=1e-2, foreach=False), 10, x)
    _train(b, AdamW(b.parameters(), lr=1e-2), 10, x)
    for p, q in zip(a.parameters(), b.parameters()):
        assert float((p - q).abs().max()) <= 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype", ["f32", "bf16"])
def test_state_dict_continues(cuda, bits, ptype):
    """A reloaded optimizer takes the steps that the first would have taken, with its moments' own types."""
    from gsr.optim import AdamW
    a = _model().to(cuda, TYPES[ptype])
    x = torch.randn(32, 8, generator=torch.Generator().manual_seed(1)).to(cuda, TYPES[ptype])
    opt = AdamW(a.parameters(), lr=1e-2, moment_bits=bits)
    _train(a, opt, 3, x)
    b = copy.deepcopy(a)
    again = AdamW(b.parameters(), lr=1e-2, moment_bits=bits)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    _train(a, opt, 3, x)
    _train(b, again, 3, x)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    s = next(iter(again.state.values()))
    assert s["step"] == 6 and s["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="bits"):
        AdamW(b.parameters(), moment_bits=40 - bits).load_state_dict(opt.state_dict())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(cuda, bits):
    """A captured step replayed with new gradients and a new device lr gives the eager steps' bits."""
    from gsr.optim import AdamW
    torch.manual_seed(0)
    start = torch.randn(3000, device=cuda)
    grads = [torch.randn(3000, device=cuda) for _ in range(6)]
    lrs = [1e-2, 1e-2, 5e-3, 5e-3, 1e-3, 1e-3]

    def make():
        p = torch.nn.Parameter(start.clone())
        lr = torch.tensor(lrs[0], device=cuda)
        p.grad = grads[0].clone()
        return p, lr, AdamW([p], lr=lr, moment_bits=bits, capturable=True)

    p, lr, opt = make()
    for g, r in zip(grads, lrs):
        p.grad.copy_(g)
        lr.fill_(r)
        opt.step()
    q, lr2, opt2 = make()
    opt2.step()   # creates the state
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt2.step()
    for g, r in zip(grads[1:], lrs[1:]):
        q.grad.copy_(g)
        lr2.fill_(r)
        graph.replay()
        torch.cuda.synchronize()
        float(q.detach().sum())
    assert torch.equal(p, q)
    assert int(opt2.state[q]["step"]) == 6
    # the device's scalars are the host's: the same steps with host values, lr as the fp32 value it is
    h = torch.nn.Parameter(start.clone())
    opt3 = AdamW([h], lr=1e-2, moment_bits=bits)
    for g, r in zip(grads, lrs):
        opt3.param_groups[0]["lr"] = float(torch.tensor(r))
        h.grad = g
        opt3.step()
    assert torch.equal(h, p)


@pytest.mark.gpu
def test_groups_and_absent_gradients(cuda):
    """Groups with their own lr and moment bits step as optimizers of their own; a parameter without a gradient
    keeps its value and its own step count."""
    from gsr.optim import AdamW
    torch.manual_seed(3)
    start = [torch.randn(300, device=cuda) for _ in range(3)]
    grads = [[torch.randn(300, device=cuda) for _ in range(3)] for _ in range(4)]
    ps = [torch.nn.Parameter(t.clone()) for t in start]
    opt = AdamW([{"params": ps[:1], "lr": 1e-2}, {"params": ps[1:], "moment_bits": 8}], lr=1e-3)
    alone = [torch.nn.Parameter(t.clone()) for t in start]
    single = [AdamW([alone[0]], lr=1e-2), AdamW([alone[1]], lr=1e-3, moment_bits=8), AdamW([alone[2]], lr=1e-3, moment_bits=8)]
    for k, gs in enumerate(grads):
        for i in range(3):
            ps[i].grad = alone[i].grad = None if (i == 2 and k == 1) else gs[i]
        opt.step()
        for o in single:
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, alone))
    assert [opt.state[p]["step"] for p in ps] == [4, 4, 3]


@pytest.mark.gpu
def test_refused_while_capturing(cuda):
    from gsr.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(8, device=cuda))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    assert bool(p.isfinite().all())


def test_refusals():
    from gsr import _lib
    from gsr.optim import AdamW, adamw_step, decode_root
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    one = lambda **kw: adamw_step([f(4)], [f(4)], [f(4)], [f(4)], **{"step": 1, **kw})  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        one()
    with pytest.raises(ValueError, match="step must be at least 1"):
        one(step=0)
    with pytest.raises(ValueError, match="betas"):
        one(betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="lr"):
        one(lr=-1.0)
    with pytest.raises(ValueError, match="lr"):
        one(lr=float("nan"))
    with pytest.raises(ValueError, match="eps"):
        one(eps=-1e-8)
    with pytest.raises(ValueError, match="float32 value"):
        one(lr=torch.tensor(1e-3, dtype=torch.float64))
    with pytest.raises(ValueError, match="int64"):
        one(step=torch.tensor(1.0))
    with pytest.raises(ValueError, match="2 params, but 1 steps"):
        adamw_step([f(4), f(4)], [f(4)] * 2, [f(4), f(4)], [f(4), f(4)], step=[torch.tensor(1)])
    with pytest.raises(ValueError, match="go together"):
        one(exp_avg_units=[f(1)])
    with pytest.raises(ValueError, match="lists of"):
        adamw_step([f(4)], [], [f(4)], [f(4)], step=1)
    with pytest.raises(ValueError, match="exp_avg must be torch.float32"):
        adamw_step([f(4)], [f(4)], [f(4).half()], [f(4)], step=1)
    with pytest.raises(ValueError, match="shape and strides"):
        adamw_step([f(4)], [f(4)], [f(5)], [f(4)], step=1)
    with pytest.raises(ValueError, match="shape and strides"):
        adamw_step([f(4, 3)], [f(4, 3)], [f(3, 4).T], [f(4, 3)], step=1)
    with pytest.raises(ValueError, match="gradient 0"):
        adamw_step([f(4)], [f(1)], [f(4)], [f(4)], step=1)
    with pytest.raises(ValueError, match="fill its memory"):
        adamw_step([f(8)[::2]], [f(4)], [f(4)], [f(4)], step=1)
    with pytest.raises(ValueError, match="fill its memory"):
        adamw_step([f(1).expand(4)], [f(4)], [f(4)], [f(4)], step=1)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        adamw_step([f(4).double()], [f(4)], [f(4)], [f(4)], step=1)
    p, m, v = f(4), f(4), f(4)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([p, p], [f(4)] * 2, [m, f(4)], [v, f(4)], step=1)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([p, f(4)], [f(4)] * 2, [m, m], [v, f(4)], step=1)
    both = f(7)
    with pytest.raises(ValueError, match="overlap"):
        adamw_step([both[:4], both[3:]], [f(4)] * 2, [f(4), f(4)], [f(4), f(4)], step=1)
    e4, u8 = f(300).to(torch.float8_e4m3fn), f(300).to(torch.uint8)
    with pytest.raises(ValueError, match=r"float32 \[2\]"):
        adamw_step([f(300)], [f(300)], [e4], [u8], step=1, exp_avg_units=[f(1)], exp_avg_root_units=[f(2)])
    with pytest.raises(ValueError, match="uint8"):
        decode_root(f(4), f(1))
    with pytest.raises(ValueError, match="units"):
        decode_root(u8, f(1))
    with pytest.raises(RuntimeError, match="CUDA"):
        decode_root(u8, f(2))
    with pytest.raises(ValueError, match="moment_bits"):
        AdamW([f(4).requires_grad_()], moment_bits=16)
    with pytest.raises(ValueError, match="betas"):
        AdamW([f(4).requires_grad_()], betas=(1.0, 0.9))
    opt = AdamW([f(4).requires_grad_()])
    for bad, msg in (({"moment_bits": 16}, "moment_bits"), ({"lr": -1.0}, "lr"), ({"betas": (0.9, 1.5)}, "betas")):
        with pytest.raises(ValueError, match=msg):
            opt.add_param_group({"params": [f(3).requires_grad_()], **bad})
    assert len(opt.param_groups) == 1
    adamw_step([], [], [], [], step=1)
    L = _lib.lib()
    args = _lib.AdamwArgs(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, step=1, bits=32)
    t = _lib.AdamwTensor(n=4)
    import ctypes
    call = lambda t, n=1, pt=0: L.gsr_adamw_step(ctypes.byref(t), n, pt, 0, ctypes.byref(args), None)  # noqa: E731
    assert call(t) == -1 and b"null pointer" in L.gsr_last_error()
    assert call(t, pt=9) == -1 and b"bad type" in L.gsr_last_error()
    assert call(t, n=-1) == -1 and b"bad list" in L.gsr_last_error()
    assert call(_lib.AdamwTensor(n=-4)) == -1 and b"bad length" in L.gsr_last_error()
    args.bits = 16
    assert call(t) == -1 and b"32 or 8" in L.gsr_last_error()
    assert L.gsr_adamw_decode_root(None, None, 4, None, None) == -1


def test_struct_layouts_match_header(tmp_path):
    """The ctypes mirrors of gsr_adamw_tensor and gsr_adamw_args have the C compiler's size and offsets."""
    import ctypes
    import os
    import shutil
    import subprocess
    from gsr import _lib
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    structs = {"gsr_adamw_tensor": _lib.AdamwTensor, "gsr_adamw_args": _lib.AdamwArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "gsr.h"', "int main(void) {",
             'printf("block %d\\n", GSR_ADAMW_BLOCK);']
    for name, py in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join([*lines, "return 0;", "}"]))
    subprocess.run([cc, "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                         text=True).stdout.splitlines())
    assert int(got["block"]) == _lib.ADAMW_BLOCK
    for name, py in structs.items():
        assert int(got[f"{name} size"]) == ctypes.sizeof(py)
        assert all(int(got[f"{name} {f}"]) == getattr(py, f).offset for f, _ in py._fields_)


def test_binding_refuses_another_library(tmp_path):
    """The torch binding fails loudly on a library that is missing or is not libgsr."""
    from gsr import _lib
    native = _lib.native()
    with pytest.raises(RuntimeError, match="cannot load"):
        native.bind(str(tmp_path / "nope.so"))
    with pytest.raises(RuntimeError, match="has no gsr_"):
        native.bind("libc.so.6")
    native.bind(_lib.LIB_PATH)
