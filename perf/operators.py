"""The 8-bit fine-tuning and serving operators as they are measured: what each case stands for, its inputs, the plain form of
the operators in elementary torch operations, and the calls of slim_amd that a user makes instead.

The operators (formulas in 32-bit arithmetic unless said otherwise):

rows    symmetric 8-bit codes of the rows of x [R, K]: a = max |x| of the row, scale = a / 127, code = rint(x * (127 / a)).  A row
        with a < 2^-100 has scale 0 and codes 0; a row that holds an infinity or a NaN has scale NaN and codes 0.  Codes are
        stored with the row length rounded up to a multiple of 128, zeros behind column K.
linear  y = (codes(x) . codes(W)^T) * scale(x) * scale(W) + bias, the sum in whole numbers; x is quantised row by row (per token)
        as above, W [N, K] is kept as codes with one scale per output channel.
grad    dx = (dy * scale(W)) . codes(W), the straight-through gradient of `linear` with respect to x.
adamw   one AdamW update of a list of tensors, after clipping by the global norm of their gradients; moments in 32 bits, or in
        8 bits with scales over blocks of 512 elements (first moment e4m3, second e5m2, stochastically rounded with random bits
        that are a function of seed, tensor and position).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
TINY = 2.0 ** -100
BLOCK = 512
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 5e-5, 0.9, 0.999, 1e-8, 0.01, 1.0


def listed():
    return [
        # decoding one token through an attention projection of the 7B shape: latency
        dict(name="linear token 4096x4096", op="linear", rows=1, n=4096, k=4096, dtype="bf16", bias=False),
        # a decoding batch through the gate projection
        dict(name="linear 13x11008x4096", op="linear", rows=13, n=11008, k=4096, dtype="bf16", bias=False),
        # a short prompt through the 13B shape's down projection, half precision, with a bias
        dict(name="linear 301x5120x13824 fp16", op="linear", rows=301, n=5120, k=13824, dtype="fp16", bias=True),
        # two sequences of 2048 tokens through the gate projection: prefill, or a training forward
        dict(name="linear 4096x11008x4096", op="linear", rows=4096, n=11008, k=4096, dtype="bf16", bias=False),
        # a ragged micro-batch's backward through a layer of no round size, 32-bit gradients
        dict(name="grad 77x1000x776 fp32", op="grad", rows=77, n=1000, k=776, dtype="fp32"),
        # one sequence of 2048 tokens backwards through the down projection
        dict(name="grad 2048x4096x11008", op="grad", rows=2048, n=4096, k=11008, dtype="bf16"),
        # one sequence's activations
        dict(name="rows 2048x4096", op="rows", rows=2048, k=4096, dtype="bf16"),
        # a weight of the 70B shape being packed
        dict(name="rows 28672x8192", op="rows", rows=28672, k=8192, dtype="bf16"),
        # adapters (rank 76) of the attention projections of a 768-wide block: latency
        dict(name="adamw32 8 adapters of 768", op="adamw", bits=32, dtype="fp32", master=False, shape="attention", hidden=768, ffn=0, rank=76),
        # adapters (rank 409) of one 7B-shaped block, bf16 parameters with 32-bit master copies
        dict(name="adamw32 14 adapters of 4096", op="adamw", bits=32, dtype="bf16", master=True, shape="block", hidden=4096, ffn=11008, rank=409),
        # the same adapters with 8-bit moments
        dict(name="adamw8 14 adapters of 4096", op="adamw", bits=8, dtype="bf16", master=False, shape="block", hidden=4096, ffn=11008, rank=409),
        # an embedding table with its 32-bit gradients, 8-bit moments
        dict(name="adamw8 table 32000x4096 fp32", op="adamw", bits=8, dtype="fp32", master=False, shape="table", hidden=4096, ffn=32000, rank=0),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "grad", "rows", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rows":
        k = _spread(rng, 1, 28672)
        return dict(op=op, rows=_spread(rng, 1, min(65536, 28672 * 8192 // 2 // k)), k=k, dtype=dtype)
    if op in ("linear", "grad"):
        n, k = _spread(rng, 16, 14336), _spread(rng, 16, 14336)
        if rng.random() < 0.5:
            n, k = -(-n // 128) * 128, -(-k // 128) * 128
        rows = _spread(rng, 1, 4096)
        most = 4096 * 11008 * 4096 if op == "linear" else 2048 * 4096 * 11008
        case = dict(op=op, rows=max(1, min(rows, most // (n * k))), n=n, k=k, dtype=dtype)
        if op == "linear":
            case["bias"] = rng.random() < 0.5
        return case
    bits = rng.choice([8, 32])
    shape = rng.choice(["attention", "block", "table"])
    hidden = _spread(rng, 32, 4096)
    ffn = 0 if shape == "attention" else _spread(rng, 16, 11008)
    rank = 0 if shape == "table" else max(1, hidden // rng.choice([10, 20, 64]))
    return dict(op=op, bits=bits, dtype=dtype, master=dtype != "fp32" and rng.random() < 0.5, shape=shape, hidden=hidden, ffn=ffn, rank=rank)


def _shapes(case):
    h, f, r = case["hidden"], case["ffn"], case["rank"]
    if case["shape"] == "table":
        return [(f, h)]
    pairs = [(h, h)] * 4 + ([(f, h), (f, h), (h, f)] if case["shape"] == "block" else [])
    return [s for n, k in pairs for s in ((k, r), (r, n))]


def _padded(k):
    return -(-k // 128) * 128


def _activations(g, rows, k, dtype):
    """Token rows as a decoder block sees them: channels of different size, a few of them much larger, and one padded token."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    size = torch.exp(torch.randn(k, generator=g, device="cuda") * 0.5)
    size[torch.randint(0, k, (4,), generator=g, device="cuda")] *= 30
    x *= size
    if rows > 8:
        x[rows // 2] = 0
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        return dict(op="rows", x=_activations(g, case["rows"], case["k"], dtype))
    if case["op"] == "adamw":
        shapes, eight = _shapes(case), case["bits"] == 8

        def randn(size):
            return torch.randn(size, generator=g, device="cuda")
        masters = [randn(s) * 0.02 for s in shapes]
        params = [m.to(dtype) for m in masters]
        # gradients whose rows differ in size, as those of adapters and of rarely seen tokens do
        grads = [(randn(s) * torch.exp(randn((s[0], 1)) - 6)).to(dtype) for s in shapes]
        m = [randn(s) * 1e-3 for s in shapes]
        v = [randn(s).square() * 1e-6 for s in shapes]
        scales = None
        if eight:
            scales = [torch.stack([_block_max(a) / 448.0, _block_max(b) / 57344.0], 1).contiguous() for a, b in zip(m, v)]
            m = [(_blocks(a) / s[:, :1]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(-1)[:a.numel()].view(a.shape) for a, s in zip(m, scales)]
            v = [(_blocks(b) / s[:, 1:]).clamp(2.0 ** -16, 57344.0).to(torch.float8_e5m2).reshape(-1)[:b.numel()].view(b.shape) for b, s in zip(v, scales)]
        return dict(op="adamw", params=params, grads=grads, m=m, v=v, scales=scales, masters=masters if case["master"] else None, step=100, seed=seed & 0xffff)
    n, k = case["n"], case["k"]
    codes = torch.zeros(n, _padded(k), dtype=torch.int8, device="cuda")
    codes[:, :k] = (torch.randn(n, k, generator=g, device="cuda") * 32).round().clamp(-127, 127).to(torch.int8)
    scale = torch.exp(torch.randn(n, generator=g, device="cuda") * 0.3) * (0.02 / 32)
    if case["op"] == "grad":
        dy = (torch.randn(case["rows"], n, generator=g, device="cuda") * torch.exp(torch.randn(case["rows"], 1, generator=g, device="cuda")) * 1e-3).to(dtype)
        # a frozen layer in training keeps its codes in both orders
        codes_t = torch.zeros(k, _padded(n), dtype=torch.int8, device="cuda")
        codes_t[:, :n] = codes[:, :k].t()
        return dict(op="grad", dy=dy, codes=codes, codes_t=codes_t, scale=scale, k=k)
    x = _activations(g, case["rows"], k, dtype)
    bias = torch.randn(n, generator=g, device="cuda").to(dtype) if case["bias"] else None
    return dict(op="linear", x=x, codes=codes, scale=scale, bias=bias)


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _quantise(x):
    """(codes as 32-bit floats [R, K], scale [R]); the two quotients are rounded once from 64 bits."""
    x = x.float()
    a = x.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(a)
    none = bad | (a < TINY)
    r = torch.where(none, 0.0, (torch.full_like(a, 127.0).double() / torch.where(none, 1.0, a).double()).float())
    codes = torch.where(none, 0.0, torch.round(x * r))
    scale = torch.where(bad, math.nan, torch.where(none, 0.0, (a.double() / 127.0).float()))
    return codes, scale.reshape(-1)


def _rows(s):
    codes, scale = _quantise(s["x"])
    out = torch.zeros(codes.shape[0], _padded(codes.shape[1]), dtype=torch.int8, device=codes.device)
    out[:, :codes.shape[1]] = codes.to(torch.int8)
    return out, scale


def _linear(s):
    x = s["x"]
    codes, scale = _quantise(x)
    y = torch.matmul(codes, s["codes"][:, :x.shape[1]].float().t()) * scale[:, None] * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(x.dtype)


def _grad(s):
    dy = s["dy"]
    return torch.matmul(dy.float() * s["scale"], s["codes"][:, :s["k"]].float()).to(dy.dtype)


def _blocks(t):
    """t as rows of BLOCK elements, zeros behind the last."""
    flat = t.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def _block_max(t):
    return _blocks(t.float()).abs().amax(1)


def _random16(n, key, device):
    """Two 16-bit numbers for each position: a multiply-xorshift mix of the position and the key, in wrapping 32-bit integers."""
    def signed(v):
        v &= 0xffffffff
        return v - (1 << 32) if v >= 1 << 31 else v
    h = torch.arange(n, dtype=torch.int32, device=device) * signed(0x9e3779b9) + signed(key)
    h = h ^ ((h >> 16) & 0xffff)
    h = h * signed(0x7feb352d)
    h = h ^ ((h >> 15) & 0x1ffff)
    h = h * signed(0x846ca68b)
    h = h ^ ((h >> 16) & 0xffff)
    return h & 0xffff, (h >> 16) & 0xffff


def _tensor_key(seed, index):
    return (seed * 0x85ebca6b + index * 0xc2b2ae35 + 0x27d4eb2f) & 0xffffffff


def _encode(t, random, mantissa, exponent):
    """Codes of t >= 0 in a format with `mantissa` bits and smallest normal number 2^exponent, rounded up where the random
    number (16 bits) and the bits below the last kept one carry."""
    drop = 23 - mantissa
    bits = t.view(torch.int32)
    normal = ((bits + (random << (drop - 16))) >> drop) - ((exponent + 126) << mantissa)
    small = ((t * 2.0 ** (mantissa - exponent + 16)).clamp(max=2.0 ** 24).to(torch.int32) + random) >> 16
    return torch.where(t >= 2.0 ** exponent, normal, small)


def _requantise(x, random, top, mantissa, exponent):
    """(codes of |x| [n], block scales, where the block has no scale): every block against its largest magnitude."""
    n = x.numel()
    a = _block_max(x)
    bad = ~torch.isfinite(a)
    none = bad | (a < TINY)
    inv = torch.where(none, 0.0, (torch.full_like(a, top).double() / torch.where(none, 1.0, a).double()).float())
    scale = torch.where(bad, math.nan, torch.where(none, 0.0, (a.double() / top).float()))
    t = (_blocks(x.abs()) * inv[:, None]).clamp(max=top).reshape(-1)[:n]
    none = none[:, None].expand(-1, BLOCK).reshape(-1)[:n]
    return torch.where(none, 0, _encode(torch.where(none, 0.0, t), random, mantissa, exponent)), scale, none


def _adamw_one(i, s, coefficient):
    p, g, m, v = s["params"][i], s["grads"][i], s["m"][i], s["v"][i]
    step, eight = s["step"], s["scales"] is not None
    shape, n = p.shape, p.numel()
    if eight:
        scales = s["scales"][i]
        m = (_blocks(m.float()) * scales[:, :1]).reshape(-1)[:n].view(shape)
        v = (_blocks(v.float()) * scales[:, 1:]).reshape(-1)[:n].view(shape)
    g = g.float() * coefficient
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    w = p.float() if s["masters"] is None else s["masters"][i]
    denominator = v.sqrt() / math.sqrt(1 - BETA2 ** step) + EPS
    w = w * (1 - LR * DECAY) - (m / denominator) * (LR / (1 - BETA1 ** step))
    p.copy_(w)
    if s["masters"] is not None:
        s["masters"][i].copy_(w)
    if not eight:
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
        return
    low, high = _random16(n, _tensor_key(s["seed"], i), p.device)
    m, v = m.reshape(-1), v.reshape(-1)
    mc, ms, _ = _requantise(m, low, 448.0, 3, -6)
    vc, vs, none = _requantise(v, high, 57344.0, 2, -14)
    vc = torch.where((v > 0) & ~none, vc.clamp(min=1), vc)      # a positive second moment never becomes zero
    mc = torch.where(m < 0, mc | 128, mc)
    s["m"][i].copy_(mc.to(torch.uint8).view(torch.float8_e4m3fn).view(shape))
    s["v"][i].copy_(vc.to(torch.uint8).view(torch.float8_e5m2).view(shape))
    s["scales"][i].copy_(torch.stack([ms, vs], 1))


def _adamw(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()
    coefficient = (MAX_NORM / (norm.double() + 1e-6)).clamp(max=1.0).float()
    [_adamw_one(i, s, coefficient) for i in range(len(s["params"]))]
    return norm


def run(state):
    s = state
    if s["op"] == "rows":
        if own:
            from slim_amd import ops
            return ops.quantize_rows8(s["x"])
        return _rows(s)
    if s["op"] == "linear":
        if own:
            from slim_amd import ops
            return ops.linear8_forward(s["x"], s["codes"], s["scale"], s["bias"])
        return _linear(s)
    if s["op"] == "grad":
        if own:
            from slim_amd import ops
            return ops.linear8_backward(s["dy"], s["codes_t"], s["scale"])
        return _grad(s)
    s["step"] += 1
    s["seed"] += 1
    if own:
        from slim_amd import ops
        norm = ops.grad_norm(s["grads"])
        ops.adamw_step(s["params"], s["grads"], s["m"], s["v"], step=s["step"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS,
                       weight_decay=DECAY, scales=s["scales"], masters=s["masters"], seed=s["seed"], norm=norm, max_norm=MAX_NORM)
    else:
        norm = _adamw(s)
    out = dict(norm=norm, p=s["params"], m=s["m"], v=s["v"])
    if s["scales"] is not None:
        out["scales"] = s["scales"]
    if s["masters"] is not None:
        out["masters"] = s["masters"]
    return out


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "rows":
        r, k = case["rows"], case["k"]
        return dict(bytes=r * k * (size + 1) + 4 * r, flops=2 * r * k)
    if case["op"] in ("linear", "grad"):
        r, n, k = case["rows"], case["n"], case["k"]
        return dict(bytes=r * (k + n) * size + n * k + 4 * n + (n * size if case.get("bias") else 0), flops=2 * r * n * k)
    count = sum(a * b for a, b in _shapes(case))
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    # the gradient once (its norm has to be known before the update: a second reading is not counted), the parameters both
    # ways (with a master copy they are only written)
    weights = size + 8 if case["master"] else 2 * size
    return dict(bytes=count * (size + moments + weights), flops=16 * count)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _codes64(x):
    """Codes and scales of the rows of x from the definition; codes at a border follow the 32-bit product that defines them."""
    a = x.double().abs().max(dim=1).values
    live = a >= TINY
    r = torch.zeros_like(a)
    r[live] = 127.0 / a[live]
    codes = (x.double() * r.float().double()[:, None]).float().double().round()
    return codes, a / 127.0 * live


def _update64(case, s, i, coefficient):
    count = s["params"][i].numel()

    def spread(scale):
        return scale.double().repeat_interleave(BLOCK)[:count]
    m, v = s["m"][i].reshape(-1).double(), s["v"][i].reshape(-1).double()
    if case["bits"] == 8:
        m, v = m * spread(s["scales"][i][:, 0]), v * spread(s["scales"][i][:, 1])
    g = s["grads"][i].reshape(-1).double() * coefficient
    t = s["step"] + 1
    m += (1 - BETA1) * (g - m)
    v += (1 - BETA2) * (g ** 2 - v)
    w = (s["params"] if s["masters"] is None else s["masters"])[i].reshape(-1).double()
    w = w - LR * DECAY * w - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    return w.view(s["params"][i].shape), m, v


def _grid64(x, bits16, top, mantissa, exponent):
    """(values on the format's grid, block scales): x / scale rounded up with probability equal to its place between neighbours."""
    pad = (-x.numel()) % BLOCK
    scale = torch.cat([x.abs(), x.new_zeros(pad)]).view(-1, BLOCK).max(dim=1).values / top
    t = x.abs() / scale.repeat_interleave(BLOCK)[:x.numel()].clamp(min=1e-300)
    unit = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** exponent))) - mantissa)
    t = torch.floor(t.clamp(max=top) / unit + bits16.double() / 65536) * unit
    return torch.sign(x) * t.clamp(max=top), scale


def _mix64(count, key):
    h = (torch.arange(count, device="cuda") * 0x9e3779b9 + key) % 2 ** 32
    for shift, factor in ((16, 0x7feb352d), (15, 0x846ca68b)):
        h ^= h >> shift
        h = ((h & 0xffff) * factor + (((h >> 16) * factor) % 65536) * 65536) % 2 ** 32
    h ^= h >> 16
    return h % 65536, h // 65536


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        return None, _codes64(s["x"])[1]
    if case["op"] == "linear":
        codes, scale = _codes64(s["x"])
        y = codes @ s["codes"][:, :case["k"]].double().t()
        y *= scale[:, None]
        y *= s["scale"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "grad":
        weight = s["codes"][:, :case["k"]].double() * s["scale"].double()[:, None]
        return s["dy"].double() @ weight
    norm = sum(float((g.double() ** 2).sum()) for g in s["grads"]) ** 0.5
    coefficient = min(1.0, MAX_NORM / (norm + 1e-6))
    out = dict(norm=norm, p=[], m=[], v=[])
    if s["scales"] is not None:
        out["scales"] = []
    for i in range(len(s["params"])):
        w, m, v = _update64(case, s, i, coefficient)
        shape = w.shape
        if s["scales"] is not None:
            low, high = _mix64(m.numel(), _tensor_key(s["seed"] + 1, i))
            m, ms = _grid64(m, low, 448.0, 3, -6)
            positive = v > 0
            v, vs = _grid64(v, high, 57344.0, 2, -14)
            v = torch.where(positive, v.clamp(min=2.0 ** -16), v)
            out["scales"].append(torch.stack([ms, vs], 1))
        out["p"].append(w)
        out["m"].append(m.view(shape))
        out["v"].append(v.view(shape))
    if s["masters"] is not None:
        out["masters"] = out["p"]
    return out
