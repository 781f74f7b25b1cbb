"""8-bit moments rounded without bias (gsr.optim.adamw_step's moment_rounding, gsr.optim.AdamW).

One step: a rounded value is one of the two codes beside it, so it is off by less than a code's step:
e4m3 2^-3 relative or 2^-9 units, a root 2^-4 relative or a unit (and one unit where it is kept from
vanishing).  Many steps: E[m] and E[v] follow the recursion of unrounded moments.  A step's rounding
has at most the variance of its two neighbours' distance, squared, over 4: (m / 8)^2 / 4 of a mean
(below the normal codes, m times their step, 2^-9 of a unit),
and of a root's square, whose neighbours differ by (17/16)^2 - 1 of the lower one, ((33/256) v)^2 / 4;
it decays with the moment.  The mean of N elements' moments lies within six of its standard
deviations, and fp32's own rounding (8 u a step)."""
import pytest
import torch

from test_adamw import LEVELS, U, _codes, _formula, _inputs, _spread, _units, _within

ARGS = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def _empty(n, cuda):
    """Zero moments of n elements: e4m3 codes, root codes and their units."""
    byte = lambda: torch.zeros(n, dtype=torch.uint8, device=cuda)  # noqa: E731
    unit = lambda: torch.zeros(_units(n), device=cuda)  # noqa: E731
    return byte().view(torch.float8_e4m3fn), byte(), unit(), unit()


def _step(p, g, m, v, mu, vu, **kw):
    from gsr.optim import adamw_step
    adamw_step([p], [g], [m], [v], exp_avg_units=[mu], exp_avg_root_units=[vu], moment_rounding="unbiased", **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype,gtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 4099])
def test_one_step(cuda, n, ptype, gtype):
    step = 5
    p, g, _, _ = _inputs((n,), ptype, gtype, n)
    mc, vc, mu, vu = _codes((n,), 50 + n)
    d = [t.to(cuda) for t in (p, g, mc, vc, mu, vu)]
    m = mc.float().double() * _spread(mu, n)
    v = (LEVELS[vc.long()] * _spread(vu, n)).square()
    _step(*d, step=step, **ARGS)
    wp, wm, wv, tp, tm = _formula(p.double(), g.double(), m, v, step, **ARGS)
    tp, tm = 2 * tp, 2 * tm   # (the stored moments carry a rounding more than fp32 ones)
    half = torch.finfo(p.dtype).eps / 2
    _within((d[0].cpu().double() - wp).abs(), tp + half * wp.abs() * (1 + 2 ** -7) + torch.finfo(p.dtype).tiny, "p")
    nmu, nvu = _spread(d[4].cpu(), n), _spread(d[5].cpu(), n)
    _within((d[2].cpu().float().double() * nmu - wm).abs(), (1 + 2 ** -20) * (2 ** -3 * wm.abs() + 2 ** -9 * nmu) + tm, "m")
    got, want = LEVELS[d[3].cpu().long()] * nvu, wv.sqrt()
    _within((got - want).abs(), (1 + 2 ** -20) * torch.maximum(2 ** -4 * want, nvu) + 8 * U * want, "root")
    assert bool(((got > 0) == (want > 0)).all())


@pytest.mark.gpu
def test_codes_stay_themselves(cuda):
    """Values that are codes keep them at every step count (b1 = b2 = 0: the moments are g and g^2; each block
    holds the largest code, so that its unit is 1)."""
    e4 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    g = torch.where(e4.isnan(), 448.0, e4).to(cuda)
    r = LEVELS.float().to(cuda)
    for step in (1, 2, 3, 1000, 2 ** 33 + 1):
        for values, roots in ((g, False), (r, True)):
            p = torch.zeros(256, device=cuda)
            m, v, mu, vu = _empty(256, cuda)
            _step(p, values, m, v, mu, vu, step=step, lr=1e-3, betas=(0.0, 0.0), weight_decay=0.0)
            if roots:
                assert float(vu) == 1 and torch.equal(v.cpu().long(), torch.arange(256))
            else:
                assert float(mu) == 1 and torch.equal(m.float(), values)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1.5, 3.25, 15.75, 16.5, 17.25, 31.5, 40.0 + 1 / 3, 1000.1, 400000.0])
def test_share_rounded_up(cuda, q):
    """A root of q units becomes the code above with the probability that keeps its square's expectation; a
    mean likewise its own (six standard deviations of 65000 draws)."""
    blocks = 256
    g = torch.full((blocks, 256), q, device=cuda)
    g[:, 0] = 507904.0
    p = torch.zeros(blocks * 256, device=cuda)
    m, v, mu, vu = _empty(p.numel(), cuda)
    _step(p, g.view(-1), m, v, mu, vu, step=11, lr=1e-3, betas=(0.0, 0.0), weight_decay=0.0)
    assert bool((vu == 1).all())
    root = LEVELS[v.cpu().long()].view(blocks, 256)[:, 1:]
    lo = float(LEVELS[LEVELS <= torch.tensor(q).double()].max())
    hi = float(LEVELS[LEVELS > torch.tensor(q).double()].min())
    assert bool(((root == lo) | (root == hi)).all())
    count = root.numel()
    share = (float(torch.tensor(q)) ** 2 - lo * lo) / (hi * hi - lo * lo)
    limit = 6 * (share * (1 - share) / count) ** 0.5 + 2.0 ** -18
    assert abs(float((root == hi).double().mean()) - share) <= limit
    # the same values as means, beside 448 (so that the unit is 1), of both signs
    w = 300.0 * q / 507904.0
    g = torch.full((blocks, 256), w, device=cuda)
    g[:, 0], g[1::2, 1:] = 448.0, -w
    m, v, mu, vu = _empty(p.numel(), cuda)
    _step(p, g.view(-1), m, v, mu, vu, step=11, lr=1e-3, betas=(0.0, 0.0), weight_decay=0.0)
    assert bool((mu == 1).all())
    got = m.float().double().cpu().view(blocks, 256)[:, 1:]
    assert bool((got[0::2] >= 0).all()) and bool((got[1::2] <= 0).all())
    levels = got.abs().unique()
    assert levels.numel() <= 2
    w = float(torch.tensor(w))
    step = 2.0 ** -9 if w < 2.0 ** -6 else 2.0 ** (torch.tensor(w).log2().floor() - 3)
    assert abs(float(got.abs().mean()) - w) <= 6 * float(step) / 2 / got.numel() ** 0.5 + 2.0 ** -18 * float(step)


def _follow(schedule, steps, advance, read, blocks, b1, b2, check):
    """Blocks of one element of gradient 1 and 255 that take the schedule's three; `advance(g, step)` takes a step,
    `read()` gives the decoded m and v; at the steps in `check` the means over the blocks are compared."""
    n = blocks * 256
    kind = (torch.arange(n) % 256 - 1) % 3   # of the 255; element 0 of a block: the largest
    first = torch.arange(n) % 256 == 0
    m, v = [0.0] * 3, [0.0] * 3
    vm, vv = [0.0] * 3, [0.0] * 3
    for t in range(1, steps + 1):
        now = schedule(t)
        g = torch.tensor(now, dtype=torch.float32)[kind]
        advance(torch.where(first, 1.0, g), t)
        for k in range(3):
            x = float(torch.tensor(now[k]))
            m[k], v[k] = b1 * m[k] + (1 - b1) * x, b2 * v[k] + (1 - b2) * x * x
            vm[k] = b1 * b1 * vm[k] * (1 + 1 / 256) + m[k] ** 2 / 256 + abs(m[k]) * 2 ** -9 / 448
            c = (33 / 256) ** 2 / 4
            vv[k] = b2 * b2 * vv[k] * (1 + c) + c * v[k] ** 2
        if t in check:
            gm, gv = read()
            for k in range(3):
                at = (kind == k) & ~first
                count = int(at.sum())
                for name, got, want, var in (("m", gm, m[k], vm[k]), ("v", gv, v[k], vv[k])):
                    off = abs(float(got[at].mean()) - want)
                    assert off <= 6 * (var / count) ** 0.5 + 8 * U * t * abs(want), (name, k, t, off / want)


def _schedule(t):
    return (0.1 if t <= 300 else 0.0), (0.01 if t <= 300 else 0.04), (0.3 if t % 2 else -0.1)


@pytest.mark.gpu
def test_many_steps_follow_the_moments(cuda):
    from gsr.optim import decode_root
    n = 64 * 256
    p = torch.zeros(n, device=cuda)
    m, v, mu, vu = _empty(n, cuda)

    def advance(g, t):
        _step(p, g.to(cuda), m, v, mu, vu, step=t, lr=1e-3, betas=(0.9, 0.99), weight_decay=0.0)

    def read():
        return m.float().double().cpu() * _spread(mu.cpu(), n), decode_root(v, vu).double().cpu().square()
    _follow(_schedule, 600, advance, read, 64, 0.9, 0.99, (1, 2, 50, 300, 310, 320, 600))


@pytest.mark.gpu
def test_optimizer_follows_the_moments(cuda):
    """The optimizer's own 8-bit steps, with changes far below half a code a step (b2 = 0.999)."""
    from gsr.optim import AdamW, decode_root
    n = 64 * 256
    p = torch.nn.Parameter(torch.zeros(n, device=cuda))
    opt = AdamW([p], lr=1e-3, betas=(0.9, 0.999), moment_bits=8)

    def advance(g, t):
        p.grad = g.to(cuda)
        opt.step()

    def read():
        s = opt.state[p]
        return (s["exp_avg"].float().double().cpu() * _spread(s["exp_avg_unit"].cpu(), n),
                decode_root(s["exp_avg_sq"], s["exp_avg_root_unit"]).double().cpu().square())
    _follow(_schedule, 2000, advance, read, 64, 0.9, 0.999, (300, 310, 1000, 2000))


@pytest.mark.gpu
def test_draws_go_by_place_and_step(cuda):
    """The same bits every run and in any list; others at another step count."""
    from gsr.optim import adamw_step
    sizes = [3000, 1, 700, 3000, 2049]
    start = [(_inputs((n,), "f32", "f32", 7), _codes((n,), 8)) for n in sizes]

    def state(k):
        (p, g, _, _), (m, v, mu, vu) = start[k]
        return [t.to(cuda) for t in (p, g, m, v, mu, vu)]

    def step(states, count):
        adamw_step(*[list(x) for x in zip(*[s[:4] for s in states])], exp_avg_units=[s[4] for s in states],
                   exp_avg_root_units=[s[5] for s in states], step=count, moment_rounding="unbiased", **ARGS)
        return [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for s in states for t in s]
    for count in (1, 6):
        alone = [t for k in range(5) for t in step([state(k)], count)]
        assert all(torch.equal(a, b) for a, b in zip(alone, step([state(k) for k in range(5)], count)))
        on_device = torch.tensor(count, device=cuda)
        assert all(torch.equal(a, b) for a, b in zip(alone, step([state(k) for k in range(5)], on_device)))
    a, b = step([state(0)], 6), step([state(0)], 6)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # (the moments before rounding do not know the step count: what differs is the draws)
    c = step([state(0)], 7)
    assert not torch.equal(a[2], c[2]) and not torch.equal(a[3], c[3]) and torch.equal(a[4], c[4])


@pytest.mark.gpu
def test_bad_gradients_stay_in_their_block(cuda):
    n = 700
    p = torch.full((n,), 5.0, device=cuda)
    g = torch.zeros(n, device=cuda)
    g[300] = float("nan")
    m, v, mu, vu = _empty(n, cuda)
    _step(p, g, m, v, mu, vu, step=1, lr=1e-2, weight_decay=0.0)
    keep = torch.arange(n) != 300
    assert bool((p.cpu()[keep] == 5).all()) and bool(p[300].isnan())
    raw = m.view(torch.uint8)
    assert bool((raw[:256] == 0).all()) and bool((v[512:] == 0).all()) and float(mu[0]) == 0 and float(vu[2]) == 0
    assert bool(mu[1].isnan()) and bool(vu[1].isnan())


def test_refusals():
    from gsr import _lib
    from gsr.optim import adamw_step
    f = torch.zeros
    with pytest.raises(ValueError, match="moment_rounding"):
        adamw_step([f(4)], [f(4)], [f(4)], [f(4)], step=1, moment_rounding="up")
    import ctypes
    args = _lib.AdamwArgs(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1, bits=8, rounding=2)
    t = _lib.AdamwTensor(n=4)
    L = _lib.lib()
    assert L.gsr_adamw_step(ctypes.byref(t), 1, 0, 0, ctypes.byref(args), None) == -1
    assert b"bad rounding" in L.gsr_last_error()
