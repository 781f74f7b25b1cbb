"""gsr.optim.AdamW's state between optimizers: what load_state_dict takes, converts and refuses.

Only moves of data, so everything is compared for equality; on the CPU where no step is taken."""
import copy

import pytest
import torch


def _bytes_state(p, seed=0):
    """A state of 8-bit moments for p, codes and units of every size."""
    g = torch.Generator().manual_seed(seed)
    units = -(-p.numel() // 256)
    like = dict(size=p.shape, stride=p.stride())
    m, v = (torch.empty_strided(**like, dtype=torch.uint8) for _ in range(2))
    m.copy_(torch.randint(0, 0x7F, p.shape, generator=g))   # (no NaN codes)
    v.copy_(torch.randint(0, 256, p.shape, generator=g))
    return {"step": 3, "exp_avg": m.view(torch.float8_e4m3fn), "exp_avg_sq": v,
            "exp_avg_unit": torch.rand(units, generator=g), "exp_avg_root_unit": torch.rand(units, generator=g)}


def _saved(p, state, **more):
    """The state_dict of an AdamW over p that holds `state`."""
    from gsr.optim import AdamW
    opt = AdamW([p], **more)
    opt.state[p] = state
    return copy.deepcopy(opt.state_dict())


def _permuted(shape, order):
    """A parameter of `shape` whose dimensions lie in memory in the order given."""
    t = torch.zeros([shape[i] for i in order]).permute([order.index(i) for i in range(len(shape))])
    return torch.nn.Parameter(t)


@pytest.mark.parametrize("shape,order,other", [((64, 32), (0, 1), (1, 0)), ((64, 32), (1, 0), (0, 1)),
                                               ((4, 8, 3, 5), (0, 1, 2, 3), (0, 2, 3, 1)), ((4, 8, 3, 5), (0, 2, 3, 1), (0, 1, 2, 3))])
def test_bytes_keep_their_memory_order(shape, order, other):
    """8-bit moments' units belong to runs of 256 elements in memory order: a parameter of another order
    is refused and nothing is changed, one of the same order takes codes and units as they are."""
    from gsr.optim import AdamW
    source = _permuted(shape, order)
    saved = _saved(source, _bytes_state(source), moment_bits=8)
    same, turned = _permuted(shape, order), _permuted(shape, other)
    opt = AdamW([same], moment_bits=8)
    opt.load_state_dict(copy.deepcopy(saved))
    for name, v in saved["state"][0].items():
        got = opt.state[same][name]
        raw = (lambda t: t.view(torch.uint8)) if name == "exp_avg" else (lambda t: t)
        assert got == v if name == "step" else torch.equal(raw(got), raw(v)) and got.dtype == v.dtype
    opt = AdamW([turned], lr=7e-3, moment_bits=8)
    with pytest.raises(ValueError, match="memory order"):
        opt.load_state_dict(saved)
    assert not opt.state and opt.param_groups[0]["lr"] == 7e-3


def test_bytes_of_one_element_dimensions():
    """Strides of dimensions of one element order nothing."""
    from gsr.optim import AdamW
    a = torch.nn.Parameter(torch.zeros(40, 10).as_strided((40, 1, 10), (10, 3, 1)))
    b = torch.nn.Parameter(torch.zeros(40, 1, 10))
    saved = _saved(a, _bytes_state(a), moment_bits=8)
    opt = AdamW([b], moment_bits=8)
    opt.load_state_dict(saved)
    assert torch.equal(opt.state[b]["exp_avg_sq"], saved["state"][0]["exp_avg_sq"])
    assert opt.state[b]["exp_avg_sq"].stride() == b.stride()


def test_words_change_their_memory_order():
    """32-bit moments follow the parameter into another order: each element keeps its own."""
    from gsr.optim import AdamW
    a, b = _permuted((6, 5), (0, 1)), _permuted((6, 5), (1, 0))
    state = {"step": 2, "exp_avg": torch.randn(6, 5), "exp_avg_sq": torch.rand(6, 5)}
    opt = AdamW([b])
    opt.load_state_dict(_saved(a, state))
    for name in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(opt.state[b][name], state[name]) and opt.state[b][name].stride() == b.stride()


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_of_another_shape(bits):
    """A state of other shapes is refused: it would be repeated over the parameter."""
    from gsr.optim import AdamW
    a, b = torch.nn.Parameter(torch.zeros(1, 300)), torch.nn.Parameter(torch.zeros(7, 300))
    state = _bytes_state(a) if bits == 8 else {"step": 2, "exp_avg": torch.randn(1, 300), "exp_avg_sq": torch.rand(1, 300)}
    opt = AdamW([b], moment_bits=bits)
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(_saved(a, state, moment_bits=bits))
    assert not opt.state


def _torch_checkpoint(dtype=torch.float32, cls=torch.optim.AdamW, **kw):
    g = torch.Generator().manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in ((5, 7), (9,))]
    opt = cls(ps, lr=3e-3, betas=(0.8, 0.95), **kw)
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(dtype)
        opt.step()
    return ps, opt.state_dict()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("capturable", [False, True])
def test_torch_checkpoint_is_taken_whole(dtype, capturable):
    """torch.optim.AdamW's state: its groups' values, its moments in fp32 whatever their type, its step
    counts, and the options that it does not know as this optimizer was made with."""
    from gsr.optim import AdamW
    ps, saved = _torch_checkpoint(dtype)
    saved["param_groups"][0]["capturable"] = capturable
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = AdamW(qs)
    opt.load_state_dict(copy.deepcopy(saved))
    group = opt.param_groups[0]
    assert group["moment_bits"] == 32 and group["capturable"] is capturable
    assert (group["lr"], group["betas"]) == (3e-3, (0.8, 0.95))
    for i, q in enumerate(qs):
        s = opt.state[q]
        assert int(s["step"]) == 3 and (not capturable or s["step"].dtype == torch.int64)
        for k in ("exp_avg", "exp_avg_sq"):
            assert s[k].dtype == torch.float32 and torch.equal(s[k], saved["state"][i][k].float())
        q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="CUDA"):   # (the next step gets as far as the device)
        opt.step()
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))]})
    assert opt.param_groups[1]["moment_bits"] == 32


def test_torch_checkpoint_of_another_step():
    """Groups whose update is another one are refused, and nothing is changed."""
    from gsr.optim import AdamW
    for cls, kw, word in ((torch.optim.AdamW, dict(maximize=True), "maximize"), (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
                          (torch.optim.Adam, dict(weight_decay=0.1), "decoupled")):
        ps, saved = _torch_checkpoint(cls=cls, **kw)
        opt = AdamW(ps, lr=7e-3)
        with pytest.raises(ValueError, match=word):
            opt.load_state_dict(saved)
        assert not opt.state and opt.param_groups[0]["lr"] == 7e-3
    ps, saved = _torch_checkpoint(cls=torch.optim.Adam)   # (no decay: the same step)
    AdamW(ps).load_state_dict(saved)
    for key, bad in (("lr", -1.0), ("betas", (0.9, 1.0)), ("eps", -1.0)):
        ps, saved = _torch_checkpoint()
        saved["param_groups"][0][key] = bad
        opt = AdamW(ps, lr=7e-3)
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(saved)
        assert not opt.state and opt.param_groups[0]["lr"] == 7e-3


def test_step_size_tensor_of_a_checkpoint():
    """A step size saved as a tensor comes back as one fp32 value on the parameters' device."""
    from gsr.optim import AdamW
    ps, saved = _torch_checkpoint()
    saved["param_groups"][0]["lr"] = torch.tensor([2e-3], dtype=torch.float64)
    opt = AdamW(ps)
    opt.load_state_dict(saved)
    lr = opt.param_groups[0]["lr"]
    assert lr.dtype == torch.float32 and lr.device == ps[0].device and float(lr) == float(torch.tensor(2e-3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tensor_lr", [False, True])
def test_torch_checkpoint_continues(cuda, dtype, tensor_lr):
    """Steps after the reload against the recursion in 64 bits from the saved state.  A step's parameter is
    rounded to its type once, half a step of it, and carries fp32's rounding (32 u of |p| and of a
    step's size): added over four steps."""
    from gsr.optim import AdamW
    ps, saved = _torch_checkpoint(dtype)
    if tensor_lr:
        saved["param_groups"][0] |= dict(lr=torch.tensor(3e-3), capturable=True)
    qs = [torch.nn.Parameter(p.detach().to(cuda)) for p in ps]
    opt = AdamW(qs)
    opt.load_state_dict(saved)
    g = torch.Generator().manual_seed(8)
    want = [p.detach().double() for p in ps]
    ms, vs = ([saved["state"][i][k].double() for i in range(2)] for k in ("exp_avg", "exp_avg_sq"))
    off = [torch.zeros(p.shape, dtype=torch.float64) for p in ps]
    b1, b2, lr, eps, wd = 0.8, 0.95, float(torch.tensor(3e-3)) if tensor_lr else 3e-3, 1e-8, 0.01
    for step in range(4, 8):
        for i, q in enumerate(qs):
            grad = torch.randn(q.shape, generator=g).to(dtype)
            q.grad = grad.to(cuda)
            ms[i] = b1 * ms[i] + (1 - b1) * grad.double()
            vs[i] = b2 * vs[i] + (1 - b2) * grad.double() ** 2
            delta = lr / (1 - b1 ** step) * ms[i] / ((vs[i] / (1 - b2 ** step)).sqrt() + eps)
            want[i] = want[i] * (1 - lr * wd) - delta
            off[i] += torch.finfo(dtype).eps / 2 * want[i].abs() * 1.01 + 32 * 2.0 ** -24 * (want[i].abs() + delta.abs() + lr)
        opt.step()
    for q, w, tol in zip(qs, want, off):
        assert bool(((q.detach().cpu().double() - w).abs() <= tol).all())


def test_load_hooks_see_what_is_loaded():
    """A pre-hook's state_dict is the one that is loaded; a post-hook finds the state as it stays."""
    from gsr.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16))
    saved = _saved(p, {"step": 2, "exp_avg": torch.rand(300), "exp_avg_sq": torch.rand(300)})
    opt = AdamW([p])
    seen = {}

    def double(_, sd):
        sd = copy.deepcopy(sd)
        sd["state"][0]["exp_avg"] *= 2
        return sd
    opt.register_load_state_dict_pre_hook(double)
    opt.register_load_state_dict_post_hook(lambda o: seen.update(o.state[p]))
    opt.load_state_dict(saved)
    assert torch.equal(opt.state[p]["exp_avg"], 2 * saved["state"][0]["exp_avg"])
    assert seen["exp_avg"].dtype == torch.float32 and seen["exp_avg"] is opt.state[p]["exp_avg"]
    opt.load_state_dict(saved)   # (once more: the hooks are still the caller's two)
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 1


@pytest.mark.gpu
def test_refused_step_is_not_counted(cuda):
    """A step that is refused (the parameter changed its memory order under its moments) leaves the device's
    step count, the parameter and the moments as they were."""
    from gsr.optim import AdamW
    p = torch.nn.Parameter(torch.randn(6, 5, device=cuda))
    opt = AdamW([p], capturable=True)
    p.grad = torch.randn(6, 5, device=cuda)
    opt.step()
    p.data = p.data.T.contiguous().T
    before = [p.detach().clone(), *(v.clone() for v in opt.state[p].values())]
    with pytest.raises(ValueError, match="strides"):
        opt.step()
    after = [p.detach(), *opt.state[p].values()]
    assert int(opt.state[p]["step"]) == 1 and all(torch.equal(a, b) for a, b in zip(before, after))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_state_of_another_default_type(cuda, bits, default):
    """The state's types do not follow torch's default type; parameters of no and of one element among them."""
    from gsr.optim import AdamW
    ps = [torch.nn.Parameter(torch.ones(s, device=cuda)) for s in ((300,), (0, 3), ())]
    for p in ps:
        p.grad = torch.ones_like(p)
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(default)
        opt = AdamW(ps, moment_bits=bits)
        opt.step()
        opt.step()
    finally:
        torch.set_default_dtype(before)
    assert all(s["exp_avg_unit"].dtype == torch.float32 for s in opt.state.values() if "exp_avg_unit" in s)
    want = 1.0   # (equal gradients: each step is lr, and the decay)
    for _ in range(2):
        want = want * (1 - 1e-3 * 1e-2) - 1e-3
    assert float((ps[0].detach() - want).abs().max()) <= 1e-6 and abs(float(ps[2]) - want) <= 1e-6
