"""What ``optim.AdamW`` takes from a checkpoint, and what a copy of the optimizer keeps: looked at on the CPU, where the moments are
left as the load put them into ``state`` (the flat buffers of the kernels are on a device)."""
import copy
import pickle

import pytest
import torch

from crystalframer_amd import optim


class OnTheHost(optim.AdamW):
    def _group_state(self, group):
        return None


TYPES = dict(exp_avg=torch.float32, exp_avg_sq=torch.float32)
TYPES_8 = dict(exp_avg=torch.float8_e4m3fn, exp_avg_sq=torch.uint8, exp_avg_scale=torch.uint8, exp_avg_sq_scale=torch.uint8)


def _optimizer(dtype=torch.bfloat16, **options):
    ps = [torch.nn.Parameter(torch.zeros(n, dtype=dtype)) for n in (5, 70)]
    return ps, OnTheHost(ps + [torch.nn.Parameter(torch.zeros(3, dtype=dtype), requires_grad=False)], **options)


def _checkpoint(opt, types=TYPES, seed=0):
    gen = torch.Generator().manual_seed(seed)
    whole = opt.state_dict()
    state = {}
    for k, n in enumerate((5, 70)):
        state[k] = dict(step=torch.tensor([7]))
        for name, t in types.items():
            size = -(-n // 64) if name.endswith("scale") else n
            bits = torch.randint(1, 100, (size,), generator=gen, dtype=torch.uint8)
            state[k][name] = torch.randn(n, generator=gen) if t == torch.float32 else bits if t == torch.uint8 else bits.view(t)
    whole["state"] = state
    return whole


def _same(a, b):
    return a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("types", [TYPES, TYPES_8], ids=["32", "8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_moments_keep_their_type(dtype, types):
    ps, opt = _optimizer(dtype)
    whole = _checkpoint(opt, types)
    before = copy.deepcopy(whole)
    opt.load_state_dict(whole)
    for k, p in enumerate(ps):
        assert set(opt.state[p]) == {"step", *types}
        for name, t in types.items():
            assert opt.state[p][name].dtype == t and _same(opt.state[p][name], before["state"][k][name])
            assert _same(whole["state"][k][name], before["state"][k][name])          # (the caller's dict is left alone)


def test_a_hook_before_the_load_hands_over_other_moments():
    ps, opt = _optimizer()
    one, other = _checkpoint(opt, seed=1), _checkpoint(opt, seed=2)
    opt.register_load_state_dict_pre_hook(lambda o, state: dict(state, state=other["state"]))
    opt.load_state_dict(one)
    for k, p in enumerate(ps):
        assert _same(opt.state[p]["exp_avg"], other["state"][k]["exp_avg"])
        assert _same(opt.state[p]["exp_avg_sq"], other["state"][k]["exp_avg_sq"])


def test_a_hook_before_the_load_gives_parameters_other_numbers():
    ps, opt = _optimizer()
    whole = _checkpoint(opt)
    numbers = {0: "a", 1: "b", 2: "c"}

    def rename(o, state):
        groups = [dict(g, params=[numbers[i] for i in g["params"]]) for g in state["param_groups"]]
        return dict(state={numbers[i]: s for i, s in state["state"].items()}, param_groups=groups)
    opt.register_load_state_dict_pre_hook(rename)
    opt.load_state_dict(whole)
    for k, p in enumerate(ps):
        assert _same(opt.state[p]["exp_avg"], whole["state"][k]["exp_avg"])


def test_a_hook_after_the_load_changes_the_state():
    ps, opt = _optimizer()
    seen = []

    def after(o):
        seen.append(o.state[ps[1]]["exp_avg"].dtype)
        o.state[ps[1]]["exp_avg"] = torch.full((70,), 0.25)
        o.state[ps[0]]["exp_avg_sq"].fill_(3.0)
    opt.register_load_state_dict_post_hook(after)
    whole = _checkpoint(opt)
    opt.load_state_dict(whole)
    assert seen == [torch.float32]
    assert torch.equal(opt.state[ps[1]]["exp_avg"], torch.full((70,), 0.25))
    assert torch.equal(opt.state[ps[0]]["exp_avg_sq"], torch.full((5,), 3.0))
    assert _same(opt.state[ps[0]]["exp_avg"], whole["state"][0]["exp_avg"])


def test_the_hooks_of_a_load_are_the_callers_alone():
    ps, opt = _optimizer()
    calls = []
    opt.register_load_state_dict_pre_hook(lambda o, state: calls.append("before"))
    opt.register_load_state_dict_post_hook(lambda o: calls.append("after"))
    for _ in range(2):
        opt.load_state_dict(_checkpoint(opt))
    with pytest.raises(ValueError):
        opt.load_state_dict(dict(state={}, param_groups=[]))
    opt = copy.deepcopy(opt)
    opt.load_state_dict(_checkpoint(opt))
    assert calls == ["before", "after"] * 2 + ["before"]


def _pickled(opt):
    return pickle.loads(pickle.dumps(opt))


@pytest.mark.parametrize("copied", [copy.deepcopy, _pickled])
def test_a_copy_clips_as_its_original(copied):
    _, opt = _optimizer(max_grad_norm=0.5)
    opt.grad_norm = torch.tensor(3.0)
    opt.load_state_dict(_checkpoint(opt))
    other = copied(opt)
    assert other.max_grad_norm == 0.5 and float(other.grad_norm) == 3.0
    assert other.param_groups[0]["state_bits"] == 32 and other._flat == {}
    for p, q in zip(opt.param_groups[0]["params"][:2], other.param_groups[0]["params"]):
        assert all(_same(opt.state[p][name], other.state[q][name]) for name in TYPES)
    assert copied(_optimizer()[1]).max_grad_norm is None


def test_a_copy_written_without_the_options():
    _, opt = _optimizer()
    old = opt.__getstate__()
    for name in ("max_grad_norm", "grad_norm"):
        del old[name]
    for group in old["param_groups"]:
        del group["state_bits"]
    new = OnTheHost.__new__(OnTheHost)
    new.__setstate__(old)
    assert new.max_grad_norm is None and new.grad_norm is None and new.param_groups[0]["state_bits"] == 32


@pytest.mark.parametrize("copied", [copy.deepcopy, _pickled])
def test_a_copy_has_its_originals_8_bit_moments(copied):
    _, opt = _optimizer(state_bits=8)
    opt.load_state_dict(_checkpoint(opt, TYPES_8))
    other = copied(opt)
    assert other.param_groups[0]["state_bits"] == 8
    for p, q in zip(opt.param_groups[0]["params"][:2], other.param_groups[0]["params"]):
        assert opt.state[p]["exp_avg"].dtype == torch.float8_e4m3fn
        assert all(_same(opt.state[p][name], other.state[q][name]) for name in TYPES_8)
    whole = opt.state_dict()
    assert whole["state"][1]["exp_avg"].dtype == torch.float8_e4m3fn


def test_entries_that_belong_to_no_parameter():
    """The base class hands them through as they are."""
    ps, opt = _optimizer()
    whole = _checkpoint(opt)
    whole["state"]["note"] = 3
    opt.load_state_dict(whole)
    assert opt.state["note"] == 3 and _same(opt.state[ps[1]]["exp_avg"], whole["state"][1]["exp_avg"])
    assert copy.deepcopy(opt).state["note"] == 3
