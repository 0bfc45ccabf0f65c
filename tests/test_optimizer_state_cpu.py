"""State dicts of the fused optimizer, without a GPU: hooks around loading, and checkpoints whose options the step does
not have."""
import copy

import pytest
import torch

from sv3d import optim


def stepped(cls=torch.optim.Adam, sizes=(3, 3), **kw):
    """A state dict of torch's optimizer after one step."""
    g = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(n, generator=g)) for n in sizes]
    a = cls(params, **kw)
    for p in params:
        p.grad = torch.randn(p.shape, generator=g)
    a.step()
    return a.state_dict()


def fresh(sizes=(3, 3), **kw):
    params = [torch.nn.Parameter(torch.zeros(n)) for n in sizes]
    return params, optim.AdamW(params, **kw)


@pytest.mark.parametrize("in_place", [False, True])
def test_what_a_hook_before_loading_makes_of_the_state_is_loaded(in_place):
    saved = stepped()

    def sevens(_, d):
        if not in_place:
            d = copy.deepcopy(d)
        for state in d["state"].values():
            state["exp_avg"] = torch.full_like(state["exp_avg"], 7.0)
        return None if in_place else d

    params, b = fresh()
    b.register_load_state_dict_pre_hook(sevens)
    b.load_state_dict(copy.deepcopy(saved))
    for i, p in enumerate(params):
        assert bool((b.state[p]["exp_avg"] == 7.0).all())
        assert torch.equal(b.state[p]["exp_avg_sq"], saved["state"][i]["exp_avg_sq"])


def test_a_hook_that_reorders_the_parameters_gives_each_its_own_moments():
    saved = stepped()

    def swapped(_, d):
        return {"state": {0: d["state"][1], 1: d["state"][0]}, "param_groups": d["param_groups"]}

    params, b = fresh()
    b.register_load_state_dict_pre_hook(swapped)
    b.load_state_dict(saved)
    for p, i in zip(params, (1, 0)):
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(b.state[p][name], saved["state"][i][name])


def test_a_hook_that_drops_state_or_sets_options_before_loading():
    saved = stepped(lr=0.5)

    def fewer(_, d):
        d = copy.deepcopy(d)
        del d["state"][1]
        d["param_groups"][0]["lr"] = torch.tensor(0.25, dtype=torch.float64)
        return d

    params, b = fresh()
    b.register_load_state_dict_pre_hook(fewer)
    b.load_state_dict(saved)
    assert torch.equal(b.state[params[0]]["exp_avg"], saved["state"][0]["exp_avg"]) and not b.state.get(params[1])
    lr = b.param_groups[0]["lr"]
    assert lr.dtype == torch.float32 and lr == 0.25


def test_a_hook_after_loading_has_the_last_word():
    params, b = fresh()

    def zeros(o):
        assert all(s["exp_avg"].dtype == torch.float32 for s in o.state.values())
        for s in o.state.values():
            s["exp_avg"] = torch.zeros_like(s["exp_avg"])

    b.register_load_state_dict_post_hook(zeros)
    b.load_state_dict(stepped())
    assert all(not b.state[p]["exp_avg"].any() and b.state[p]["exp_avg_sq"].any() for p in params)


def test_loading_leaves_no_hooks_behind():
    params, b = fresh()
    saved = stepped()
    b.load_state_dict(saved)
    with pytest.raises(ValueError):
        b.load_state_dict(stepped(sizes=(3, 3, 3)))
    c = copy.deepcopy(saved)
    c["state"][0]["exp_avg"] += 1
    b.load_state_dict(c)
    assert torch.equal(b.state[params[0]]["exp_avg"], c["state"][0]["exp_avg"])
    assert not b._optimizer_load_state_dict_pre_hooks and not b._optimizer_load_state_dict_post_hooks


@pytest.mark.parametrize("cls, kw, words", [
    (torch.optim.Adam, dict(amsgrad=True), "amsgrad"),
    (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"),
    (torch.optim.Adam, dict(weight_decay=0.1), "weight_decay"),         # added to the gradient, not taken off the weight
])
def test_a_checkpoint_whose_update_is_another_one_is_refused(cls, kw, words):
    params, b = fresh(lr=0.125)
    b.load_state_dict(stepped())
    before = copy.deepcopy(b.state_dict())
    with pytest.raises(ValueError, match=words):
        b.load_state_dict(stepped(cls, **kw))
    after = b.state_dict()
    assert after["param_groups"] == before["param_groups"]
    for i in (0, 1):
        assert all(torch.equal(after["state"][i][k], v) for k, v in before["state"][i].items())


def test_a_checkpoint_of_the_same_update_is_taken():
    for cls, kw in ((torch.optim.Adam, {}), (torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.AdamW, dict(maximize=True)),
                    (torch.optim.Adam, dict(foreach=True))):
        saved = stepped(cls, **kw)
        params, b = fresh()
        b.load_state_dict(saved)
        assert torch.equal(b.state[params[1]]["exp_avg"], saved["state"][1]["exp_avg"])
        for name in ("weight_decay", "maximize"):
            assert b.param_groups[0][name] == saved["param_groups"][0][name]


def test_options_that_an_old_checkpoint_lacks_are_the_constructors():
    saved = stepped()
    for name in ("maximize", "amsgrad", "decoupled_weight_decay"):
        del saved["param_groups"][0][name]
    params, b = fresh(maximize=True)
    b.load_state_dict(saved)
    assert b.param_groups[0]["maximize"] is True
    p = torch.nn.Parameter(torch.zeros(3, device="meta"))
    c = optim.AdamW([p])
    del saved["param_groups"][0]["params"][1], saved["state"][1]
    c.load_state_dict(saved)
    p.grad = torch.zeros_like(p)
    c.step()
