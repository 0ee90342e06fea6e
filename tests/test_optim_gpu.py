"""The optimizer where a step is refused, or resumed."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def AdamW():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd.optim import AdamW as _AdamW
    return _AdamW


def bits(t):
    return t.detach().reshape(-1).view(torch.uint8).clone()


def contents(opt, ps):
    return [[bits(p)] + [v if k == "step" else bits(v) for k, v in sorted(opt.state[p].items())] for p in ps if p in opt.state] + [bits(p) for p in ps]


def same(a, b):
    return len(a) == len(b) and all(same(x, y) if isinstance(x, list) else torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


@pytest.mark.parametrize("damage", ["moment", "betas", "second group's new parameter"])
def test_a_refused_step_changes_nothing(AdamW, damage):
    """The refusal comes from the last of three calls (8-bit moments, 32-bit moments, another group); no parameter, moment or count of
    the others moves, and the step that follows once it is mended is the one that would have been taken."""
    runs = []
    for refused in (False, True):
        g = torch.Generator().manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(n, generator=g).to(DEV).bfloat16()) for n in (5000, 300, 700)]
        late = damage.startswith("second")
        opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:], lr=0.1)], lr=1e-2, state_bits=8, master_weights=True, max_grad_norm=1.0, seed=2)
        for step in range(3):
            for p in ps[:2] if late and step < 2 else ps:
                p.grad = torch.randn(p.shape, generator=g).to(DEV).bfloat16()
            if step == 2 and refused:
                group = opt.param_groups[1]
                if damage == "moment":
                    kept = opt.state[ps[2]]["exp_avg_sq"]
                    opt.state[ps[2]]["exp_avg_sq"] = kept[:-1]
                else:
                    kept = group["betas"]
                    group["betas"] = (0.9, 1.5)
                before, norm = contents(opt, ps), opt.last_norm.clone()
                with pytest.raises(ValueError):
                    opt.step()
                assert same(before, contents(opt, ps)) and torch.equal(opt.last_norm, norm) and (ps[2] in opt.state) != late
                if damage == "moment":
                    opt.state[ps[2]]["exp_avg_sq"] = kept
                else:
                    group["betas"] = kept
            opt.step()
        runs.append(contents(opt, ps))
    assert same(*runs)


def test_a_loaded_run_goes_on_with_its_own_random_bits(AdamW):
    """Saved by an optimizer of seed 4, loaded into one made without: the same codes, bit for bit."""
    runs = []
    for resumed in (False, True):
        g = torch.Generator().manual_seed(5)
        p = torch.nn.Parameter(torch.randn(6000, generator=g).to(DEV))
        opt = AdamW([p], state_bits=8, seed=4)
        for step in range(4):
            if step == 2 and resumed:
                saved = opt.state_dict()
                opt = AdamW([p], state_bits=8)
                opt.load_state_dict(saved)
            p.grad = torch.randn(6000, generator=g).to(DEV)
            opt.step()
        runs.append(contents(opt, [p]))
    assert same(*runs)
