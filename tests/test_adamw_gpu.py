"""AdamW over many tensors and the global gradient norm: fp32 results against 64 bits with bounds counted from the roundings,
8-bit codes bit for bit against the definition in numpy's fp32."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
SIZES = [1, 3, 255, 511, 512, 513, 1023, 2047, 2048, 2049, 4097, 100003]
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd import ops as _ops
    return _ops


def tensors(sizes, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=g).to(dtype) for n in sizes]
    d = [(torch.randn(n, generator=g) * 1e-2 * torch.exp(torch.randn(n, generator=g))).to(dtype) for n in sizes]
    m = [torch.randn(n, generator=g) * 1e-3 for n in sizes]
    v = [torch.randn(n, generator=g).square() * 1e-5 for n in sizes]
    return p, d, m, v


def to_dev(*lists):
    return [[t.to(DEV) for t in x] for x in lists]


def formula(w, g, m, v, step, clip=1.0, lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1):
    g, m, v, w = g.double() * clip, m.double(), v.double(), w.double()
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    update = lr / (1 - beta1 ** step) * m / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return w * (1 - lr * weight_decay) - update, m, v, update


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("step", [1, 7, 100000])
def test_32_bit_moments(ops, dtype, master, step):
    if master and dtype == torch.float32:
        pytest.skip("fp32 parameters have no master copies")
    p0, g0, m0, v0 = tensors(SIZES, dtype, 1)
    p, g, m, v = to_dev(p0, g0, m0, v0)
    w0 = [t.float() + torch.randn(t.shape) * 1e-3 for t in p0] if master else p0
    w = [t.to(DEV) for t in w0] if master else None
    ops.adamw_step(p, g, m, v, step=step, masters=w, **HYPER)
    e = 2.0 ** -24
    for i in range(len(SIZES)):
        ew, em, ev, update = formula(w0[i], g0[i], m0[i], v0[i], step)
        gd = g0[i].double()
        # beta, 1 - beta as fp32, two products, one sum
        assert bool(((m[i].cpu().double() - em).abs() <= 4 * e * (0.9 * m0[i].double().abs() + 0.1 * gd.abs()) + SMALL[torch.float32]).all())
        assert bool(((v[i].cpu().double() - ev).abs() <= 5 * e * ev + 2 * SMALL[torch.float32]).all())
        # the update: m's error (absolute), v's through the root (2.5), root and reciprocal of one unit in the last place each (2 + 2),
        # their constants and products (6); w * keep and the difference: 3 on |w| and 1 on the result
        merr = 4 * e * (0.9 * m0[i].double().abs() + 0.1 * gd.abs()) / em.abs().clamp(min=1e-300)
        allowed = update.abs() * (13 * e + merr) + 4 * e * (w0[i].double().abs() + update.abs()) + SMALL[torch.float32]
        got = (w if master else p)[i].cpu().double()
        if master:
            assert torch.equal(p[i], w[i].to(dtype))
            assert bool(((got - ew).abs() <= allowed).all())
        else:
            assert bool(((got - ew).abs() <= allowed + (ew.abs() + allowed) * HALF[dtype] * 1.01 + SMALL[dtype]).all())


def random16(n, index, seed):
    M = 0xffffffff
    key = (seed * 0x85ebca6b + index * 0xc2b2ae35 + 0x27d4eb2f) & M
    h = (np.arange(n, dtype=np.uint64) * 0x9e3779b9 + key) & M
    h ^= h >> np.uint64(16)
    h = (h * np.uint64(0x7feb352d)) & M
    h ^= h >> np.uint64(15)
    h = (h * np.uint64(0x846ca68b)) & M
    h ^= h >> np.uint64(16)
    return (h & np.uint64(0xffff)).astype(np.float64), (h >> np.uint64(16)).astype(np.float64)


def blocks(x):
    return np.concatenate([x, np.zeros(-len(x) % 512, x.dtype)]).reshape(-1, 512)


def round_up(x, r16, top, mantissa, exponent, positive):
    """(grid values, scales) of fp32 x: |x| * (top / max) rounded up where its place between two neighbours plus the random
    number passes one."""
    f = np.float32
    a = np.abs(blocks(x)).max(1)
    ok = np.isfinite(a) & (a >= f(2.0 ** -100))
    scale = np.where(ok, (a / f(top)).astype(f), np.where(np.isfinite(a), f(0), f("nan")))
    inv = np.where(ok, f(top) / np.where(ok, a, f(1)), f(0)).astype(f)
    t = np.minimum((np.abs(blocks(np.where(np.isfinite(x), x, f(0)))) * inv[:, None]).astype(f), f(top)).reshape(-1)[:len(x)].astype(np.float64)
    unit = np.exp2(np.floor(np.log2(np.maximum(t, 2.0 ** exponent))) - mantissa)
    # the random number has the weight of the bits below the last kept one; in the range of subnormals those bits are cut at 16
    place = np.where(t >= 2.0 ** exponent, t / unit, np.floor(t / unit * 65536) / 65536)
    q = np.floor(place + r16 / 65536) * unit
    if positive:
        q = np.where((q == 0) & (x > 0), 2.0 ** (exponent - mantissa), q)
    live = np.repeat(ok, 512)[:len(x)]
    return np.where(live, np.sign(x) * q, 0.0), scale


def eight_bit_state(m, v):
    """Codes and scales that represent fp32 moments, by rounding to nearest."""
    out = []
    for a, b in zip(m, v):
        sm = torch.from_numpy(np.abs(blocks(a.numpy())).max(1)) / 448
        sv = torch.from_numpy(np.abs(blocks(b.numpy())).max(1)) / 57344
        n = a.numel()
        cm = (a / sm.repeat_interleave(512)[:n].clamp(min=1e-30)).clamp(-448, 448).to(torch.float8_e4m3fn)
        cv = (b / sv.repeat_interleave(512)[:n].clamp(min=1e-30)).clamp(0, 57344).to(torch.float8_e5m2)
        out.append((cm, cv, torch.stack([sm, sv], 1).contiguous()))
    return [list(x) for x in zip(*out)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("master", [False, True])
def test_8_bit_moments_bit_for_bit(ops, dtype, master):
    if master and dtype == torch.float32:
        pytest.skip("fp32 parameters have no master copies")
    sizes = SIZES + [2000]
    p0, g0, m0, v0 = tensors(sizes, dtype, 2)
    g0[-1] *= 0
    m0[-1] *= 0
    v0[-1] *= 0                                                          # nothing learned yet, no gradient
    g0[4][:] = 0
    m0[5] *= torch.exp(6 * torch.randn(m0[5].shape, generator=torch.Generator().manual_seed(3)))      # far more range than the codes have
    v0[5] *= torch.exp(12 * torch.randn(v0[5].shape, generator=torch.Generator().manual_seed(4)))
    cm0, cv0, s0 = eight_bit_state(m0, v0)
    p, g, cm, cv, s = to_dev(p0, g0, cm0, cv0, s0)
    w0 = [t.float() * 1.001 for t in p0] if master else p0
    w = [t.to(DEV) for t in w0] if master else None
    seed, first = 12345, 3
    ops.adamw_step(p, g, cm, cv, step=9, scales=s, masters=w, seed=seed, first_index=first, **HYPER)
    f = np.float32
    for i, n in enumerate(sizes):
        sm, sv = (np.repeat(s0[i][:, k].numpy(), 512)[:n] for k in (0, 1))
        m_old, v_old = cm0[i].float().numpy() * sm, cv0[i].float().numpy() * sv
        gd = g0[i].float().numpy()
        m_new = m_old * f(0.9) + gd * f(1 - 0.9)
        v_new = v_old * f(0.999) + (gd * gd) * f(1 - 0.999)
        low, high = random16(n, first + i, seed)
        qm, ms = round_up(m_new, low, 448.0, 3, -6, False)
        qv, vs = round_up(v_new, high, 57344.0, 2, -14, True)
        assert np.array_equal(s[i][:, 0].cpu().numpy(), ms) and np.array_equal(s[i][:, 1].cpu().numpy(), vs), i
        assert np.array_equal(cm[i].float().cpu().numpy().astype(np.float64), qm), i
        assert np.array_equal(cv[i].float().cpu().numpy().astype(np.float64), qv), i
        # the parameters move by the moments before they are rounded
        ew, em, ev, update = formula(w0[i], g0[i], torch.from_numpy(m_old), torch.from_numpy(v_old), 9)
        e = 2.0 ** -24
        merr = 4 * e * (0.9 * np.abs(m_old.astype(np.float64)) + 0.1 * np.abs(gd))
        allowed = update.abs() * 13 * e + torch.from_numpy(merr) * (update / em.where(em != 0, torch.ones_like(em))).abs() + 4 * e * (w0[i].double().abs() + update.abs()) + SMALL[torch.float32]
        got = (w if master else p)[i].cpu().double()
        slack = 0 if master else (ew.abs() + allowed) * HALF[dtype] * 1.01 + SMALL[dtype]
        ok = (got - ew).abs() <= allowed + slack
        if dtype == torch.float16 and not master:        # from 65520 on, the middle between fp16's largest number and the next, it is infinity
            ok = ok & got.isfinite() | (got == torch.sign(ew) * float("inf")) & (ew.abs() * (1 + 2.0 ** -20) >= 65520)
        assert bool(ok.all()), i


def test_not_finite_gradients_stay_in_their_block(ops):
    p, g = [torch.ones(2000, device=DEV)], [torch.full((2000,), 0.1, device=DEV)]
    g[0][700], g[0][1999] = float("nan"), float("inf")
    cm, cv = [torch.zeros(2000, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)], [torch.zeros(2000, dtype=torch.uint8, device=DEV).view(torch.float8_e5m2)]
    s = [torch.zeros(4, 2, device=DEV)]
    ops.adamw_step(p, g, cm, cv, step=1, scales=s, seed=1, **HYPER)
    assert s[0].isnan().cpu().tolist() == [[False, False], [True, True], [False, False], [True, True]]
    assert p[0].isnan().nonzero().flatten().cpu().tolist() == [700, 1999]
    g[0][700], g[0][1999] = 0.1, 0.1
    ops.adamw_step(p, g, cm, cv, step=2, scales=s, seed=2, **HYPER)
    assert bool(p[0][512:1024].isnan().all()) and bool(p[0][1536:].isnan().all()) and bool(torch.isfinite(p[0][:512]).all()) and bool(torch.isfinite(p[0][1024:1536]).all())


def test_8_bit_second_moment_follows_small_changes(ops):
    """A constant gradient for 3000 steps from a second moment four times too large: it falls by 0.1 % a step, a thirtieth of what
    rounding to nearest would ever notice.  Rounding up with the right probability keeps the expectation: the mean over n elements
    is within five standard deviations; one element's is below sqrt(step / 2) = sqrt(0.25 / 2) of its value (each rounding adds at
    most step * change to the variance, and the average remembers half its length)."""
    n, steps = 512 * 64, 3000
    p, g = [torch.zeros(n, device=DEV)], [torch.ones(n, device=DEV)]
    cm = [torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)]
    cv = [torch.full((n,), 28672.0, device=DEV).to(torch.float8_e5m2)]
    s = [torch.tensor([[0.0, 4.0 / 28672]], device=DEV).repeat(n // 512, 1)]
    # one element of each block holds the scale: its own second moment does not change
    g[0][::512] = 8.0 ** 0.5
    cv[0].view(torch.uint8)[::512] = torch.tensor([57344.0]).to(torch.float8_e5m2).view(torch.uint8).item()
    for t in range(1, steps + 1):
        ops.adamw_step(p, g, cm, cv, step=t, lr=0.0, scales=s, seed=t)
    v = (cv[0].float().view(-1, 512) * s[0][:, 1:]).double()
    want = 1 + 3 * 0.999 ** steps
    rest = v[:, 1:]
    sd = (0.25 / 2) ** 0.5 * want / rest.numel() ** 0.5
    # the values of a block share the roundings of its scale (fp32, 2^-24 a step)
    assert abs(float(rest.mean()) - want) <= 5 * sd + steps * 2.0 ** -23 * want, (float(rest.mean()), want, sd)
    m = (cm[0].float().view(-1, 512) * s[0][:, :1]).double()[:, 1:]
    assert abs(float(m.mean()) - 1) <= 5 * (0.125 / 2) ** 0.5 / m.numel() ** 0.5 + steps * 2.0 ** -23


@pytest.mark.parametrize("dtype", TYPES)
def test_norm(ops, dtype):
    g = torch.Generator().manual_seed(5)
    for sizes in ([1], [7, 2048, 5000], [3] * 400, [1000003], [0, 5, 0]):
        x = [(torch.randn(n, generator=g) * 10).to(dtype) for n in sizes]
        want = sum(float(t.double().square().sum()) for t in x) ** 0.5
        got = ops.grad_norm([t.to(DEV) for t in x])
        assert got.dtype == torch.float32 and got.dim() == 0
        assert abs(float(got) - want) <= want * 2.0 ** -24 * 1.01, (sizes, float(got), want)
    huge = torch.full((1000,), 3e4 if dtype == torch.float16 else 1e30, dtype=dtype, device=DEV)
    want = float(huge.double().square().sum().sqrt())
    assert abs(float(ops.grad_norm([huge])) - want) <= want * 2.0 ** -24 * 1.01
    huge[3] = float("nan")
    assert bool(ops.grad_norm([huge, huge[:2]]).isnan())
    huge[3] = float("-inf")
    assert bool(ops.grad_norm([huge]).isinf())
    assert float(ops.grad_norm([torch.zeros(0, device=DEV)])) == 0.0
    assert float(ops.grad_norm([torch.zeros(5, 7, device=DEV).t()])) == 0.0


@pytest.mark.parametrize("factor", [0.5, 2.0])
def test_clipping(ops, factor):
    """max_norm below and above the norm; the gradients themselves stay."""
    p0, g0, m0, v0 = tensors(SIZES, torch.float32, 6)
    p, g, m, v = to_dev(p0, g0, m0, v0)
    norm = ops.grad_norm(g)
    limit = float(norm) * factor
    ops.adamw_step(p, g, m, v, step=3, norm=norm, max_norm=limit, **HYPER)
    clip = min(1.0, limit / (float(norm) + 1e-6))
    for i in range(len(SIZES)):
        _, em, ev, _ = formula(p0[i], g0[i], m0[i], v0[i], 3, clip)
        assert torch.equal(g[i].cpu(), g0[i])
        assert bool(((m[i].cpu().double() - em).abs() <= 6 * 2.0 ** -24 * (0.9 * m0[i].double().abs() + 0.1 * clip * g0[i].double().abs()) + 1e-44).all())
        assert bool(((v[i].cpu().double() - ev).abs() <= 9 * 2.0 ** -24 * ev + 1e-44).all())


def test_many_tensors_and_odd_addresses(ops):
    """More tensors than a launch takes, each starting at an odd element of one buffer: the elements between stay."""
    count, n = 150, 700
    for dtype in TYPES:
        buf = torch.full((count * (n + 1) + 1,), 3.0, device=DEV, dtype=dtype)
        views = [buf[i * (n + 1) + 1:(i + 1) * (n + 1)] for i in range(count)]
        g = [torch.randn(n, device=DEV).to(dtype) for _ in range(count)]
        alone = [v.clone() for v in views]
        state = [[torch.zeros(n, device=DEV) for _ in range(count)] for _ in range(4)]
        ops.adamw_step(views, g, state[0], state[1], step=1, **HYPER)
        for i in range(count):
            ops.adamw_step([alone[i]], [g[i]], [state[2][i]], [state[3][i]], step=1, **HYPER)
        assert all(torch.equal(a, b) for a, b in zip(views, alone)) and all(torch.equal(a, b) for k in (0, 1) for a, b in zip(state[k], state[k + 2]))
        keep = torch.arange(buf.numel(), device=DEV) % (n + 1) == 0
        assert bool((buf[keep] == 3.0).all())


def test_captured_and_replayed(ops):
    p0, g0, m0, v0 = tensors([5000, 300], torch.bfloat16, 8)
    cm0, cv0, s0 = eight_bit_state(m0, v0)
    p, g, cm, cv, s = to_dev(p0, g0, cm0, cv0, s0)
    q = [[t.clone() for t in x] for x in (p, cm, cv, s)]
    kw = dict(step=5, seed=3, max_norm=0.1, **HYPER)
    ops.adamw_step([t.clone() for t in p], g, [t.clone() for t in cm], [t.clone() for t in cv], scales=[t.clone() for t in s], norm=ops.grad_norm(g), **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw_step(p, g, cm, cv, scales=s, norm=ops.grad_norm(g), **kw)
    for i in range(4):
        for t in g:
            t.copy_(torch.randn(t.shape, device=DEV) * 1e-2)
        graph.replay()
        torch.cuda.synchronize()
        ops.adamw_step(q[0], g, q[1], q[2], scales=q[3], norm=ops.grad_norm(g), **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p, q[0])) and all(torch.equal(a, b) for a, b in zip(s, q[3]))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for k, x in ((1, cm), (2, cv)) for a, b in zip(x, q[k]))


def test_step_refusals(ops):
    p, f = torch.zeros(8, device=DEV), [torch.zeros(8, device=DEV)]
    for bad in (dict(params=[p], grads=[p.half()]), dict(params=[p], grads=[p[:4]]), dict(params=[p, p], grads=[p]), dict(params=[torch.zeros(4, 2, device=DEV).t()], grads=[p]),
                dict(params=[p], grads=[p], masters=f), dict(params=[p], grads=[p], norm=p[0]), dict(params=[p], grads=[p], scales=[torch.zeros(1, 2, device=DEV)])):
        kw = dict(masters=bad.get("masters"), norm=bad.get("norm"), scales=bad.get("scales"))
        with pytest.raises(ValueError):
            ops.adamw_step(bad["params"], bad["grads"], f, f, step=1, lr=0.1, **kw)
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p, p], [p, p], f * 2, f * 2, step=1, lr=0.1)
    with pytest.raises(TypeError):
        ops.adamw_step([p.double()], [p.double()], f, f, step=1, lr=0.1)
    with pytest.raises(ValueError):
        ops.adamw_step([p], [p], f, f, step=0, lr=0.1)
    ops.adamw_step([], [], [], [], step=1, lr=0.1)
    ops.adamw_step([p[:0]], [p[:0]], [p[:0]], [p[:0]], step=1, lr=0.1)
    before = p._version
    ops.adamw_step([p], [p], f, [torch.zeros(8, device=DEV)], step=1, lr=0.1)
    assert p._version > before                                          # autograd sees the update


# ---- the optimizer --------------------------------------------------------------------------------------------------
def small_model(dtype):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(96, 128), torch.nn.GELU(), torch.nn.Linear(128, 64, bias=False)).to(DEV).to(dtype)


def run_steps(model, opt, steps, seed=1, clip=None):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        for p in model.parameters():
            p.grad = (torch.randn(p.shape, generator=g)).to(DEV).to(p.dtype)
        if clip:
            torch.nn.utils.clip_grad_norm_(model.parameters(), clip)
        opt.step()


def test_optimizer_equals_torchs(ops):
    """fp32: twenty steps with clipping and two parameter groups, against torch's AdamW in 64 bits.  Per step the update's relative
    error is below 40 * 2^-24 (13 of the update, the rest from the moments and the clipping factor), its size below lr * 10."""
    from slim_amd.optim import AdamW
    a, b = small_model(torch.float32), small_model(torch.float32).double()

    def groups(m):
        ps = list(m.parameters())
        return [dict(params=ps[:1], lr=1e-3, weight_decay=0.1), dict(params=ps[1:])]
    x, y = AdamW(groups(a), lr=1e-2, weight_decay=0.0, max_grad_norm=1.0), torch.optim.AdamW(groups(b), lr=1e-2, weight_decay=0.0)
    run_steps(a, x, 20)
    g = torch.Generator().manual_seed(1)
    for _ in range(20):
        for p in b.parameters():
            p.grad = torch.randn(p.shape, generator=g).to(DEV).double()
        torch.nn.utils.clip_grad_norm_(b.parameters(), 1.0)
        y.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert float((p.detach().double() - q.detach()).abs().max()) <= 20 * (1e-1 * 40 * 2.0 ** -24 + float(q.detach().abs().max()) * 4 * 2.0 ** -24)
    assert x.last_norm is not None and float(x.last_norm) > 1


@pytest.mark.parametrize("bits,dtype,master", [(32, torch.float32, False), (32, torch.bfloat16, True), (8, torch.bfloat16, True), (8, torch.float16, False), (8, torch.float32, False)])
def test_optimizer_state_round_trip(ops, bits, dtype, master, tmp_path):
    """A run saved to a file after three steps goes on as the uninterrupted one, bit for bit."""
    from slim_amd.optim import AdamW
    a = small_model(dtype)
    x = AdamW(a.parameters(), lr=1e-2, state_bits=bits, master_weights=master, max_grad_norm=1.0, seed=4)
    run_steps(a, x, 3)
    kinds = {n: {t.dtype for s in x.state.values() for k, t in s.items() if k == n} for n in ("exp_avg", "exp_avg_sq")}
    assert (torch.float8_e4m3fn in kinds["exp_avg"]) == (bits == 8) and torch.float32 in kinds["exp_avg"] or bits == 32      # (the bias stays in 32 bits)
    torch.save(dict(model=a.state_dict(), opt=x.state_dict()), tmp_path / "run.pt")
    run_steps(a, x, 3, seed=2)
    saved = torch.load(tmp_path / "run.pt", weights_only=True)
    b = small_model(dtype)
    b.load_state_dict(saved["model"])
    y = AdamW(b.parameters(), lr=1e-2, state_bits=bits, master_weights=master, max_grad_norm=1.0, seed=4)
    y.load_state_dict(saved["opt"])
    run_steps(b, y, 3, seed=2)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
        for n, t in x.state[p].items():
            u = y.state[q][n]
            assert (t == u) if n == "step" else (t.dtype == u.dtype and torch.equal(t.view(torch.uint8), u.view(torch.uint8))), n


def test_optimizer_master_copies_keep_small_updates(ops):
    """bf16 parameters at 1: updates of 1e-4 are below half a step (2^-9); only the 32-bit copy moves, and then the parameter."""
    from slim_amd.optim import AdamW
    for master, moved in ((False, False), (True, True)):
        p = torch.nn.Parameter(torch.ones(5000, device=DEV, dtype=torch.bfloat16))
        opt = AdamW([p], lr=1e-4, weight_decay=0.0, master_weights=master)
        for _ in range(60):
            p.grad = torch.ones_like(p)
            opt.step()
        assert bool((p < 1).all()) == moved


def test_optimizer_skips_and_refuses(ops):
    from slim_amd.optim import AdamW
    a = small_model(torch.float32)
    ps = list(a.parameters())
    opt = AdamW(ps, lr=0.1)
    ps[0].grad = torch.ones_like(ps[0])
    before = [p.detach().clone() for p in ps]
    opt.step()
    assert not torch.equal(ps[0], before[0]) and all(torch.equal(p, b) for p, b in zip(ps[1:], before[1:])) and ps[1] not in opt.state
    ps[1].grad = torch.ones_like(ps[1])
    assert opt.step(lambda: 5) == 5                                       # parameters at different steps
    assert opt.state[ps[0]]["step"] == 2 and opt.state[ps[1]]["step"] == 1
    ps[0].grad = torch.ones(ps[0].shape, device=DEV).t().contiguous().t()      # a gradient in another order
    opt.step()
    ps[0].grad = torch.ones_like(ps[0]).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    t = torch.nn.Parameter(torch.zeros(4, 6, device=DEV).t())
    t.grad = torch.zeros_like(t)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([t]).step()
    ps[0].grad = torch.ones_like(ps[0])
    opt = AdamW(ps, lr=0.1)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            opt.step()
    copy.deepcopy(opt.state_dict())


def test_norm_of_more_elements_than_a_grid_takes(ops):
    """Nine times 2^34 elements: 18.9 million chunks of 8192, which a workgroup each would be more than a launch's 2^24."""
    g = torch.zeros(2 ** 34, dtype=torch.bfloat16, device=DEV)
    g[0], g[2 ** 33 + 12345], g[-1] = 3.0, 2.0, -5.0
    norm = float(ops.grad_norm([g] * 9))
    assert abs(norm - (9 * 38.0) ** 0.5) <= 2.0 ** -24 * (9 * 38.0) ** 0.5 * 1.01      # exact sums, a root in 64 bits, one rounding


def test_second_moments_below_the_normal_range(ops):
    """eps = 0: what a step does depends on the ratio of the moments alone, down to gradients whose squares are subnormal."""
    n = 517
    gen = torch.Generator().manual_seed(5)
    g0 = (torch.rand(n, generator=gen) * 9 + 1) * 1e-19 * torch.randint(0, 2, (n,), generator=gen).mul(2).sub(1)
    zero = torch.zeros(n)
    p, g, m, v = to_dev([zero], [g0], [zero], [zero])
    ops.adamw_step(p, g, m, v, step=1, lr=1e-2, eps=0.0)
    ew, _, ev, update = formula(zero, g0, zero, zero, 1, eps=0.0, weight_decay=0.0)
    assert float(ev.max()) < 2.0 ** -126
    # the square and its product with 1 - beta2 are each rounded to a multiple of 2^-149: half of that twice, and half its
    # relative size in the root; the rest as in the normal range
    rounding = 2.0 ** -149 / ev.double()
    assert bool(((p[0].cpu().double() - ew).abs() <= update.abs() * (0.5 * rounding * 1.01 + 17 * 2.0 ** -24)).all())


def test_step_refuses_shared_state_and_takes_inference_tensors(ops):
    p, q, m, v, s = (torch.zeros(8, device=DEV) for _ in range(5))
    for lists in (([p, q], [m, m], [v, s]), ([p], [m], [m]), ([p], [p], [v])):
        with pytest.raises(ValueError, match="twice"):
            ops.adamw_step(lists[0], lists[0], lists[1], lists[2], step=1, lr=0.1)
    with pytest.raises(ValueError, match="eps"):
        ops.adamw_step([p], [q], [m], [v], step=1, lr=0.1, eps=2.0 ** -127)
    with torch.inference_mode():
        w = torch.ones(8, device=DEV)
        ops.adamw_step([w, p], [torch.ones(8, device=DEV)] * 2, [m, q], [v, s], step=1, lr=0.1, weight_decay=0.0)
    assert bool((w < 0.91).all()) and bool((p < -0.09).all())
    with torch.no_grad():
        g = torch.ones(8, device=DEV)
        ops.adamw_step([g], [g], [torch.zeros(8, device=DEV)], [torch.zeros(8, device=DEV)], step=1, lr=0.1)     # its own gradient: read first
    assert bool(((g - 0.9).abs() < 1e-6).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_copies(ops, bits):
    """A deep copy goes on exactly as the original does; gradients that are refused leave the step count alone."""
    from slim_amd.optim import AdamW
    a = small_model(torch.float32)
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=3)
    run_steps(a, opt, 3)
    b, twin = copy.deepcopy((a, opt))
    run_steps(a, opt, 3, seed=7)
    run_steps(b, twin, 3, seed=7)
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters())) and torch.equal(opt.last_norm, twin.last_norm)
    p = next(a.parameters())
    opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"][:1]
    with pytest.raises(ValueError):
        opt.step()
    assert opt.state[p]["step"] == 6


def test_optimizer_continues_from_torchs_state(ops):
    from slim_amd.optim import AdamW
    a, b = small_model(torch.float32), small_model(torch.float32)
    x, y = torch.optim.AdamW(a.parameters(), lr=1e-2), torch.optim.AdamW(b.parameters(), lr=1e-2)
    run_steps(a, x, 5)
    run_steps(b, y, 5)
    z = AdamW(b.parameters(), lr=1e-3)
    z.load_state_dict(copy.deepcopy(y.state_dict()))
    run_steps(a, x, 5, seed=2)
    run_steps(b, z, 5, seed=2)
    for p, q in zip(a.parameters(), b.parameters()):
        # five updates of relative error 40 * 2^-24 on either side, each below lr * 10, and the sums' roundings
        assert bool(((p - q).abs() <= 5 * 2 * (40 * 2.0 ** -24 * 0.1 + 4 * 2.0 ** -24 * (p.abs() + 0.1))).all())
        assert z.state[q]["step"] == 10
