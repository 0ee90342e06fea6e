"""8-bit moments far below the normal range: what is positive stays positive, so that eps = 0 stays a legal choice."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("size", [1e-15, 1e-17, 1e-19, 1e-21])
def test_a_step_without_a_gradient_after_a_small_one(size):
    """eps = 0: one step with gradients of 1e-15 to 1e-20 (second moments from below 2^-100 to subnormal numbers), then one without.  The
    second moves by the ratio of the decayed moments, as with 32 bits; a lost second moment would make it infinite."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd import ops
    n, e = 1300, 2.0 ** -24
    gen = torch.Generator().manual_seed(5)
    g0 = (torch.rand(n, generator=gen) * 9 + 1) * size * torch.randint(0, 2, (n,), generator=gen).mul(2).sub(1)
    p, g = torch.zeros(n, device=DEV), g0.to(DEV)
    cm = torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    cv = torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e5m2)
    s = torch.zeros(3, 2, device=DEV)
    ops.adamw_step([p], [g], [cm], [cv], step=1, lr=1e-2, eps=0.0, scales=[s], seed=1)
    sm, sv = (s[:, k].double().cpu().repeat_interleave(512)[:n] for k in (0, 1))
    m, v = cm.float().double().cpu() * sm, cv.float().double().cpu() * sv
    em = g0.double() * (1 - 0.9)
    ev = ((g0 * g0) * torch.tensor(1 - 0.999)).double()                   # (the formula's fp32 operations)
    # one step of the code's format (2^-3 and 2^-2 of itself, fixed below its normal numbers), and the fp32 product's rounding
    assert bool(((m - em).abs() <= torch.maximum(em.abs() * 2.0 ** -3, sm * 2.0 ** -9) * 1.001 + 1e-44).all())
    assert bool(((v - ev).abs() <= torch.maximum(ev * 2.0 ** -2, sv * 2.0 ** -16) * 1.001).all())
    assert bool(((v > 0) == (ev > 0)).all()) and (size < 1e-20 or bool((ev > 0).all()))
    w = p.double().cpu()
    ops.adamw_step([p], [torch.zeros_like(p)], [cm], [cv], step=2, lr=1e-2, eps=0.0, scales=[s], seed=2)
    live = ev > 0                                                          # (squares that fp32 itself takes for 0 divide by 0, in any width)
    m, v = m[live] * 0.9, v[live] * 0.999
    update = 1e-2 / (1 - 0.9 ** 2) * m / (v / (1 - 0.999 ** 2)).sqrt()
    # decayed moments rounded to multiples of 2^-149 (half of that; in the root half its relative size), the rest as in the normal range
    allowed = update.abs() * (17 * e + 0.5 * 1.01 * 2.0 ** -149 / v) + 2.0 ** -149 / m.abs().clamp(min=1e-300) * update.abs() + 4 * e * (w[live].abs() + update.abs())
    assert bool(((p.double().cpu()[live] - (w[live] - update)).abs() <= allowed).all())
