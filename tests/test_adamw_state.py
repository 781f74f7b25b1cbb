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
