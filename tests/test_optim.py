"""The optimizer's bookkeeping, on the CPU: nothing is launched."""
import copy

import pytest
import torch

from slim_amd.optim import AdamW


def parameter(n=8, dtype=torch.bfloat16):
    return torch.nn.Parameter(torch.zeros(n, dtype=dtype))


def with_state(opt, value=1.0):
    """`opt` as after five steps, its moments at `value`."""
    for group in opt.param_groups:
        for p in group["params"]:
            opt.state[p] = dict(step=5, exp_avg=torch.full(p.shape, value), exp_avg_sq=torch.full(p.shape, value))
    return opt


def test_load_hooks_decide_what_is_loaded():
    saved = with_state(AdamW([parameter()])).state_dict()
    p = parameter()
    opt, seen = AdamW([p]), []

    def pre(_, state_dict):
        state_dict = copy.deepcopy(state_dict)
        state_dict["state"][0]["exp_avg"] += 6
        state_dict["state"][0]["step"] = torch.tensor(9.0)
        return state_dict

    def post(o):
        seen.append({k: v if k == "step" else v.dtype for k, v in o.state[p].items()})
    hooks = opt.register_load_state_dict_pre_hook(pre), opt.register_load_state_dict_post_hook(post)
    opt.load_state_dict(saved)
    assert bool((opt.state[p]["exp_avg"] == 7).all()) and bool((opt.state[p]["exp_avg_sq"] == 1).all()) and opt.state[p]["step"] == 9
    assert seen == [dict(step=9, exp_avg=torch.float32, exp_avg_sq=torch.float32)]       # (not the parameter's bf16)
    assert bool((saved["state"][0]["exp_avg"] == 1).all())
    for hook in hooks:
        hook.remove()
    opt.load_state_dict(saved)
    assert bool((opt.state[p]["exp_avg"] == 1).all()) and len(seen) == 1
    with pytest.raises(ValueError, match="parameter group"):
        opt.load_state_dict(AdamW([parameter(), parameter()]).state_dict())
    assert bool((opt.state[p]["exp_avg"] == 1).all()) and opt.state[p]["step"] == 5
    assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks       # (none of its own stays)


@pytest.mark.parametrize("cls,kw,refused", [("AdamW", {}, False), ("AdamW", dict(amsgrad=True), True), ("AdamW", dict(maximize=True), True),
                                            ("Adam", dict(weight_decay=0.1), True), ("Adam", {}, False), ("AdamW", dict(fused=True), False)])
def test_states_of_another_update_are_refused(cls, kw, refused):
    """Not continued as if they were plain AdamW's: the sign of the step, or the second moment it divides by, would change."""
    q = parameter(dtype=torch.float32)
    other = getattr(torch.optim, cls)([q], lr=1e-2, **kw)
    q.grad = torch.ones_like(q)
    other.step()
    p = parameter(dtype=torch.float32)
    opt = with_state(AdamW([p]), 3.0)
    if refused:
        with pytest.raises(ValueError, match="another update"):
            opt.load_state_dict(other.state_dict())
        assert opt.state[p]["step"] == 5 and bool((opt.state[p]["exp_avg"] == 3).all())
    else:
        opt.load_state_dict(other.state_dict())
        assert opt.state[p]["step"] == 1 and torch.equal(opt.state[p]["exp_avg"], other.state[q]["exp_avg"])


def test_the_seed_is_saved():
    saved = with_state(AdamW([parameter()], seed=7)).state_dict()
    opt = AdamW([parameter()], seed=8)
    opt.load_state_dict(saved)
    assert [g["seed"] for g in opt.param_groups] == [7] and opt.seed == 7
    q = parameter(dtype=torch.float32)
    opt = AdamW([parameter(dtype=torch.float32)], seed=8)
    opt.load_state_dict(torch.optim.AdamW([q]).state_dict())               # (which has none)
    assert [g["seed"] for g in opt.param_groups] == [8]


@pytest.mark.parametrize("option", [dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=2.0 ** -130), dict(weight_decay=-0.1)])
def test_a_groups_own_options_are_checked(option):
    """As the constructor's are: 16-bit moments were taken for 32-bit ones."""
    with pytest.raises(ValueError):
        AdamW([dict(params=[parameter()], **option)])
    opt = AdamW([parameter()])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[parameter()], **option))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[parameter()], state_bits=8))
    assert opt.param_groups[1]["state_bits"] == 8
