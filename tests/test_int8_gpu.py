"""Linears in 8-bit integers against their definitions on the CPU: codes and scales bit for bit, products and gradients against
64 bits with bounds counted from the roundings."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative
TINIEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd import ops as _ops
    return _ops


def pad(k):
    return -(-k // 128) * 128


def definition(x):
    """(codes [R, K], scales) of the rows of x on the CPU, in the fp32 operations of the definition (quotients through 64 bits:
    a quotient of two 24-bit numbers rounded to 53 bits and then to 24 is the one rounded once)."""
    x = x.detach().cpu().float()
    a = x.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(a)
    none = bad | (a < 2.0 ** -100)
    safe = torch.where(none, torch.ones_like(a), a).double()
    r = (torch.full_like(safe, 127.0) / safe).float()
    codes = torch.where(none, torch.zeros_like(x), torch.round(x * r))
    scale = torch.where(bad, torch.full_like(a, float("nan")), torch.where(none, torch.zeros_like(a), (safe / 127).float()))
    return codes.to(torch.int8), scale.reshape(-1)


def make_rows(R, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(torch.randn(K, generator=g)) * torch.exp(2 * torch.randn(R, 1, generator=g))
    x = x.to(dtype)
    if R >= 6:
        x[0] = 0
        x[1, K // 2] = float("inf")
        x[2, K - 1] = float("nan")
        x[3] = 2.0 ** -101 if dtype != torch.float16 else 2.0 ** -24      # below the smallest scale, or a subnormal
        x[4] = float("-inf")
    return x


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-1.0), torch.nan_to_num(b, nan=-1.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (7, 3), (6, 127), (9, 128), (5, 129), (8, 512), (6, 513), (7, 1024), (6, 1030), (6, 2048), (3, 2500), (7, 4096),
                                 (6, 8191), (2, 8200), (6, 16384), (6, 16385), (3, 28672), (130, 200)])
def test_rows_equal_the_definition(ops, R, K, dtype):
    x = make_rows(R, K, dtype, R * K)
    codes, scale = ops.quantize_rows8(x.to(DEV))
    want, want_scale = definition(x)
    assert codes.shape == (R, pad(K)) and codes.dtype == torch.int8 and scale.dtype == torch.float32
    assert torch.equal(codes[:, :K].cpu(), want)
    assert not bool(codes[:, K:].any())
    assert same(scale.cpu(), want_scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_views(ops, dtype):
    """Rows that start at odd elements, rows apart, columns apart, empty."""
    big = torch.randn(40, 777, device=DEV).to(dtype)
    for x in (big[3:20, 1:700], big[:, 5:6], big[::3], big[5:6, 7:], big.t(), big[:, ::2], big[7:8]):
        codes, scale = ops.quantize_rows8(x)
        want, want_scale = definition(x)
        assert torch.equal(codes[:, :x.shape[1]].cpu(), want) and same(scale.cpu(), want_scale)
    codes, scale = ops.quantize_rows8(big[:0])
    assert codes.shape == (0, pad(777)) and scale.shape == (0,)


def random_codes(n, k, seed, extremes=False):
    g = torch.Generator().manual_seed(seed)
    c = torch.zeros(n, pad(k), dtype=torch.int8)
    c[:, :k] = torch.randint(-128, 128, (n, k), generator=g).to(torch.int8)
    if extremes:
        c[:, :k] = -128
    return c


def exact_product(a, sa, b, sb, bias):
    p = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    return p if bias is None else p + bias.double()


def bound(p, bias, dtype):
    """float(sum), two products, one addition: 4 roundings of fp32 on |product| + |bias|, then the output's."""
    size = p.abs() if bias is None else (p - bias.double()).abs() + bias.double().abs()
    return size * 4.1 * 2.0 ** -24 + p.abs() * HALF[dtype] * 1.01 + TINIEST[dtype]


def within(out, p, allowed, dtype):
    """|out - p| <= allowed; a result of 65520 or more is fp16's infinity (65504 is its largest number and 65536 would be the next:
    from their middle on rounding to nearest gives infinity), either of the two within the bound around 65520."""
    ok = (out - p).abs() <= allowed
    if dtype == torch.float16:
        ok = ok & out.isfinite() | (out == torch.sign(p) * float("inf")) & (p.abs() * (1 + 2.0 ** -20) >= 65520)
    return bool(ok.all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 64), (2, 129, 130), (15, 17, 300), (16, 256, 128), (17, 64, 1000), (33, 300, 257), (64, 128, 512), (65, 1000, 700),
                                   (100, 96, 2048), (129, 513, 384), (200, 130, 1300), (257, 512, 640), (300, 700, 4096), (520, 1100, 260), (1030, 520, 1500)])
def test_product_against_64_bits(ops, M, N, K, dtype):
    a, b = random_codes(M, K, M + N), random_codes(N, K, M + N + 1)
    g = torch.Generator().manual_seed(K)
    sa, sb = torch.exp(torch.randn(M, generator=g)) * 1e-2, torch.exp(torch.randn(N, generator=g)) * 1e-2
    for bias in (None, torch.randn(N, generator=g).to(dtype)):
        out = ops.gemm8_nt(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), None if bias is None else bias.to(DEV), dtype).cpu().double()
        p = exact_product(a, sa, b, sb, bias)
        assert within(out, p, bound(p, bias, dtype), dtype), float(((out - p).abs() - bound(p, bias, dtype)).max())


# every tile and its neighbours: 256 x 256 alone, with a last round of 192 and of 128 columns, 128 x 256, 128 x 128, 64 x 128, and slices of
# the reduction (4 and 8); ragged in both directions.  The reference product runs on the GPU in 64 bits (whole numbers: exact).
LARGE = [(2500, 4099, 200), (2048, 4095, 500), (6000, 4097, 700), (4100, 4100, 300), (2049, 4097, 500), (513, 5121, 13000), (1111, 2222, 1000), (70, 130, 20000), (300, 201, 13000), (90, 9001, 5000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", LARGE)
def test_large_products_against_64_bits(ops, M, N, K, dtype):
    a, b = random_codes(M, K, 1).to(DEV), random_codes(N, K, 2).to(DEV)
    sa, sb = torch.rand(M, device=DEV) * 1e-2, torch.rand(N, device=DEV) * 1e-2
    bias = torch.randn(N, device=DEV).to(dtype)
    out = ops.gemm8_nt(a, sa, b, sb, bias, dtype).double()
    p = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double() + bias.double()
    assert within(out, p, bound(p, bias, dtype), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(2100, 300, 4101), (4101, 300, 5003), (3100, 200, 4097), (1025, 1000, 2100), (513, 5000, 1100), (40, 20001, 131), (17, 13001, 200)])
def test_large_gradients_against_64_bits(ops, M, N, K, dtype):
    w = random_codes(N, K, 3).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    scale = torch.rand(N, generator=g, device=DEV) * 1e-2
    dy = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    dx = ops.linear8_backward(dy, ops.transpose8(w, K), scale).double()
    exact, allowed = gradient_bound(dy, w[:, :K], scale, dtype)
    assert bool(((dx - exact).abs() <= allowed).all()), float(((dx - exact).abs() / allowed).max())


def test_longest_sum_is_exact(ops):
    """131071 products of -128 by -128: 2^31 - 16384, the largest sum 32 bits have to hold."""
    K = 131071
    a, b = random_codes(3, K, 1, extremes=True).to(DEV), random_codes(130, K, 2, extremes=True).to(DEV)
    one = torch.ones(130, device=DEV)
    out = ops.gemm8_nt(a, one[:3], b, one, None, torch.float32, K=K)
    assert bool((out == float(K * 16384)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 13, 16, 17, 31, 32, 33, 64, 77, 128, 300])
def test_forward_is_rows_then_product(ops, M, dtype):
    """Every number of tokens, whichever kernels serve it: bit for bit the product of the codes."""
    for N, K, seed in ((48, 100, 3), (515, 1024, 4), (1024, 4224, 5)):
        x = make_rows(M, K, dtype, seed).to(DEV)
        codes, scale = ops.quantize_rows8(make_rows(N + 6, K, torch.float32, seed)[6:].to(DEV))
        bias = torch.randn(N, device=DEV).to(dtype)
        y = ops.linear8_forward(x, codes, scale, bias)
        xc, xs = definition(x)
        full = torch.zeros(M, pad(K), dtype=torch.int8)
        full[:, :K] = xc
        want = ops.gemm8_nt(full.to(DEV), xs.to(DEV), codes, scale, bias, dtype)
        assert same(y, want)
        p = exact_product(full, xs, codes.cpu(), scale.cpu(), bias.cpu())
        fine = torch.isfinite(xs)
        assert bool(y.cpu()[~fine].isnan().all())                    # rows with an infinity or a NaN
        assert within(y.cpu().double()[fine], p[fine], bound(p, bias.cpu(), dtype)[fine], dtype)
        if M >= 6:
            assert torch.equal(y[0], bias)                             # a row of zeros


def test_output_rows_apart_and_what_lies_between(ops):
    from slim_amd import _lib
    M, N, K = 19, 70, 200
    a, b = random_codes(M, K, 1).to(DEV), random_codes(N, K, 2).to(DEV)
    sa, sb = torch.rand(M, device=DEV), torch.rand(N, device=DEV)
    out = torch.full((M + 3, 99), 7.0, device=DEV, dtype=torch.bfloat16)
    ws = torch.empty(max(16, _lib.query("slim_gemm8_workspace_bytes", M, N, K)), dtype=torch.uint8, device=DEV)
    _lib.call("slim_gemm8_nt", a.data_ptr(), 256, sa.data_ptr(), b.data_ptr(), 256, sb.data_ptr(), M, N, K, None, 1, out.data_ptr() + 2, 99, ws.data_ptr(),
              ws.numel(), torch.cuda.current_stream().cuda_stream)
    want = ops.gemm8_nt(a, sa, b, sb)
    flat = out.reshape(-1)
    got = torch.as_strided(flat, (M, N), (99, 1), 1)
    assert torch.equal(got, want)
    keep = torch.ones_like(flat, dtype=torch.bool)
    torch.as_strided(keep, (M, N), (99, 1), 1).fill_(False)
    assert bool((flat[keep] == 7.0).all())


def gradient_bound(dy, w, scale, dtype):
    """dy * scale is rounded to a grid of step max / L per row: half a step, plus the roundings of the product with the scale, of
    the reciprocal and of the product with it (three of 2^-24 on at most L steps), each times |code|; then the fp32 operations that join
    the planes and the output's rounding."""
    L = 8355711.0 if dtype == torch.float32 else 32639.0
    v = dy.double() * scale.double()
    step = v.abs().amax(1, keepdim=True) / L
    exact = v @ w.double()
    return exact, step * (0.5 + 3.1 * 2.0 ** -24 * L) * w.double().abs().sum(0) + exact.abs() * (HALF[dtype] * 1.01 + 2.0 ** -22) + (v.abs() @ w.double().abs()) * 2.0 ** -22 + TINIEST[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 129), (5, 128, 64), (16, 130, 128), (17, 1000, 776), (47, 64, 513), (77, 1000, 776), (130, 515, 300), (300, 2000, 1100)])
def test_backward_against_64_bits(ops, M, N, K, dtype):
    w = random_codes(N, K, M * N)
    g = torch.Generator().manual_seed(K)
    scale = torch.exp(torch.randn(N, generator=g) * 0.3) * 1e-2
    dy = (torch.randn(M, N, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(dtype)
    if M > 4:
        dy[1] = 0
    wt = ops.transpose8(w.to(DEV), K)
    assert torch.equal(wt.cpu()[:, :N], w[:, :K].t()) and not bool(wt[:, N:].any())
    dx = ops.linear8_backward(dy.to(DEV), wt, scale.to(DEV)).cpu().double()
    exact, allowed = gradient_bound(dy, w[:, :K], scale, dtype)
    assert bool(((dx - exact).abs() <= allowed).all()), float(((dx - exact).abs() / allowed).max())
    # a row's error in the 2-norm: that of rounding dy * scale, sqrt(N / 12) 2^-15 (2^-23 in fp32) of its norm at most, through the weight
    norm = (dy.double() * scale.double()).norm(dim=1) * torch.linalg.matrix_norm(w.double(), 2)
    grid = (N / 12) ** 0.5 * (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -15)      # (24-bit grid: the product's own rounding as well)
    assert bool(((dx - exact).norm(dim=1) <= norm * (grid + 2.0 ** -20) + exact.norm(dim=1) * 1.01 * HALF[dtype]).all())


def test_backward_rows_that_are_not_finite(ops):
    w = random_codes(64, 100, 1)
    wt, scale = ops.transpose8(w.to(DEV), 100), torch.ones(64, device=DEV)
    dy = torch.ones(40, 64, device=DEV)
    dy[3, 5], dy[17, 0], dy[39, 63] = float("nan"), float("inf"), float("-inf")
    dx = ops.linear8_backward(dy, wt, scale)
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[3, 17, 39]] = True
    assert bool(dx.cpu()[bad].isnan().all()) and bool(torch.isfinite(dx.cpu()[~bad]).all())


def test_gradient_against_differences(ops):
    """With x on its grid and the row's maximum held by a channel that does not move, moving another channel by whole steps
    changes the codes by exactly that: the difference quotient is the straight-through gradient."""
    N, K, M = 24, 40, 3
    g = torch.Generator().manual_seed(1)
    w = random_codes(N, K, 2)
    codes, scale = w.to(DEV), torch.full((N,), 2.0 ** -7, device=DEV)
    step = 2.0 ** -5
    x = torch.randint(-60, 61, (M, K), generator=g).float()
    x[:, 0] = 127
    x = (x * step).to(DEV)
    dy = torch.randint(-100, 101, (M, N), generator=g).float().to(DEV)
    dx = ops.linear8_backward(dy, ops.transpose8(codes, K), scale)
    for k in range(1, K):
        e = torch.zeros(K, device=DEV)
        e[k] = 16 * step
        d = (ops.linear8_forward(x + e, codes, scale) - ops.linear8_forward(x - e, codes, scale)).double() / (32 * step)
        quotient = (d * dy.double()).sum(1)
        # both sides: whole numbers below 2^24 times powers of two, but for the gradient's 24-bit grid
        assert bool(((quotient - dx[:, k].double()).abs() <= gradient_bound(dy.cpu(), w[:, :K], scale.cpu(), torch.float32)[1][:, k].to(DEV)).all())


def test_captured_and_replayed(ops):
    """A captured forward and backward, replayed with new inputs between eager calls of other sizes on the same stream."""
    N, K = 300, 1000
    codes, scale = ops.quantize_rows8(torch.randn(N, K, device=DEV))
    codes_t = ops.transpose8(codes, K)
    for M in (1, 7, 40, 200):
        x, dy = torch.randn(M, K, device=DEV).bfloat16(), torch.randn(M, N, device=DEV).bfloat16()
        ops.linear8_forward(x, codes, scale), ops.linear8_backward(dy, codes_t, scale)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, dx = ops.linear8_forward(x, codes, scale), ops.linear8_backward(dy, codes_t, scale)
        for i in range(4):
            x.copy_(torch.randn(M, K, device=DEV) * (i + 1))
            dy.copy_(torch.randn(M, N, device=DEV))
            graph.replay()
            ops.linear8_forward(torch.randn(M + 50, K, device=DEV), codes, scale)
            torch.cuda.synchronize()
            assert torch.equal(y, ops.linear8_forward(x, codes, scale)) and torch.equal(dx, ops.linear8_backward(dy, codes_t, scale))


def test_two_streams_at_once(ops):
    N, K = 515, 2048
    codes, scale = ops.quantize_rows8(torch.randn(N, K, device=DEV))
    xs = [torch.randn(m, K, device=DEV).half() for m in (1, 9, 70, 260)]
    want = [ops.linear8_forward(x, codes, scale) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(5):
        for i, (st, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(st):
                got[i].append(ops.linear8_forward(x, codes, scale))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)


def test_wrapper_refusals(ops):
    x = torch.randn(4, 100, device=DEV)
    codes, scale = ops.quantize_rows8(torch.randn(10, 100, device=DEV))
    with pytest.raises(ValueError, match="columns"):
        ops.linear8_forward(torch.randn(4, 200, device=DEV), codes, scale)
    with pytest.raises(ValueError, match="10 values"):
        ops.linear8_forward(x, codes, scale[:9])
    with pytest.raises(TypeError, match="bias"):
        ops.linear8_forward(x.bfloat16(), codes, scale, torch.zeros(10, device=DEV))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        ops.linear8_forward(x.double(), codes, scale)
    with pytest.raises(ValueError, match="matrix"):
        ops.quantize_rows8(x[0])
    with pytest.raises(ValueError, match="equally long"):
        ops.gemm8_nt(codes, scale, torch.zeros(3, 256, dtype=torch.int8, device=DEV), scale[:3])
    with pytest.raises(ValueError, match="K must lie"):
        ops.gemm8_nt(codes, scale, codes, scale, K=129)
    with pytest.raises(ValueError, match="too large"):
        ops.gemm8_nt(*(torch.zeros(1, 131072, dtype=torch.int8, device=DEV), scale[:1]) * 2)
    with pytest.raises(ValueError, match="codes_t"):
        ops.linear8_backward(torch.randn(4, 300, device=DEV), codes, scale)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.linear8_forward(x, codes, scale.cpu())
    assert ops.linear8_forward(x[:0], codes, scale).shape == (0, 10)
    assert ops.linear8_backward(torch.randn(0, 10, device=DEV), ops.transpose8(codes, 100), scale).shape == (0, 100)


def test_padded_c_abi_rows_of_codes(ops):
    """Rows of codes further apart than they are long."""
    from slim_amd import _lib
    x = torch.randn(9, 150, device=DEV)
    codes = torch.full((9, 400), 9, dtype=torch.int8, device=DEV)
    scale = torch.empty(9, device=DEV)
    _lib.call("slim_quantize_rows8", x.data_ptr(), 0, 9, 150, 150, codes.data_ptr(), 400, scale.data_ptr(), torch.cuda.current_stream().cuda_stream)
    want, _ = definition(x)
    assert torch.equal(codes[:, :150].cpu(), want) and not bool(codes[:, 150:256].any()) and bool((codes[:, 256:] == 9).all())


# 128 x 256, 64 x 128 with two workgroups a CU, and 128 x 128 and 64 x 128 in slices
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1030, 5000, 300), (600, 9001, 300), (301, 9001, 300), (128, 5121, 13700), (130, 5121, 9000), (500, 2003, 9000)])
def test_more_tiles_against_64_bits(ops, M, N, K, dtype):
    test_large_products_against_64_bits(ops, M, N, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(300, 600, 5000), (301, 2000, 5001), (129, 9001, 1000), (257, 9001, 1100), (600, 1000, 5003)])
def test_more_gradient_tiles_against_64_bits(ops, M, N, K, dtype):
    test_large_gradients_against_64_bits(ops, M, N, K, dtype)


def sampled_rows_equal(ops, y, x, codes, scale, bias, rows):
    """Rows of a product against the exact sums of their codes: the fp32 operations of the definition, so bit for bit."""
    xc, xs = ops.quantize_rows8(x[rows])
    sums = torch.stack([(c[None, :].double() * codes.double()).sum(1) for c in xc]) if codes.numel() < 1 << 24 else torch.cat(
        [torch.stack([(c[None, :].double() * part.double()).sum(1) for c in xc]) for part in codes.split(1 << 10)], 1)
    want = sums.float() * xs[:, None] * scale
    want = (want if bias is None else want + bias.float()).to(y.dtype)
    return same(y[rows], want)


@pytest.mark.parametrize("M,N,K", [(1, 8191, 14336), (1, 8192, 14337), (1, 300, 28672), (1, 300, 28673), (2, 8191, 8192), (2, 8193, 8193), (2, 300, 16384), (2, 300, 16385),
                                   (3, 4096, 1000), (16, 4097, 1000), (17, 4096, 1000), (32, 4097, 1000), (33, 4096, 1000), (33, 4097, 1000), (64, 8192, 500), (64, 8193, 500),
                                   (65, 8192, 500), (5, 260, 131071)])
def test_borders_of_the_kernels_for_few_tokens(ops, M, N, K):
    x = torch.randn(M, K, device=DEV).bfloat16()
    codes, scale = ops.quantize_rows8(torch.randn(N, K, device=DEV))
    bias = torch.randn(N, device=DEV).bfloat16()
    y = ops.linear8_forward(x, codes, scale, bias)
    assert sampled_rows_equal(ops, y, x, codes, scale, bias, list(range(M)) if M < 4 else [0, M // 2, M - 1])


def test_offsets_beyond_32_bits(ops):
    """A result, rows of a 16-bit input, and a weight's codes of more than 2^31 elements each; the last rows, where an offset counts."""
    codes, scale = ops.quantize_rows8(torch.randn(32000, 64, device=DEV))
    x = torch.randn(70001, 64, device=DEV).bfloat16()
    y = ops.linear8_forward(x, codes, scale)
    assert y.numel() > 2 ** 31 and sampled_rows_equal(ops, y, x, codes, scale, None, [0, 67108, 67109, 69999, 70000])
    del y, x
    x = torch.randn(300001, 8192, device=DEV, dtype=torch.bfloat16)
    c, s = ops.quantize_rows8(x)
    want, want_scale = definition(x[-3:])
    assert torch.equal(c[-3:].cpu(), want) and same(s[-3:].cpu(), want_scale)
    del x, c, s
    N, K = 17001, 131071
    codes = torch.randint(-127, 128, (N, pad(K)), dtype=torch.int8, device=DEV)
    codes[:, K:] = 0
    scale = torch.rand(N, device=DEV)
    assert codes.numel() > 2 ** 31
    for M in (1, 5, 70):
        x = torch.randn(M, K, device=DEV).bfloat16()
        y = ops.linear8_forward(x, codes, scale)
        assert sampled_rows_equal(ops, y[:, -600:], x, codes[-600:], scale[-600:], None, [0, M - 1])
        assert sampled_rows_equal(ops, y[:, :600], x, codes[:600], scale[:600], None, [0, M - 1])
    t = ops.transpose8(codes[:, :128 * 7].contiguous(), 128 * 7 - 5)
    assert torch.equal(t[:, :N], codes[:, :128 * 7 - 5].t()) and not bool(t[:, N:].any())


# more 256 x 256 (192 x 256) tiles than CUs: workgroups that take several, with two steps and with one, all tiles whole or not, with and
# without a last round of narrower ones
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(4096, 8192, 256), (4090, 8190, 130), (4096, 8192, 100), (1200, 25500, 260), (2600, 9000, 1100), (8200, 4352, 500)])
def test_workgroups_with_several_tiles(ops, M, N, K, dtype):
    test_large_products_against_64_bits(ops, M, N, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(2048, 256, 8192), (2050, 130, 8190), (2048, 100, 8192), (2100, 700, 9001)])
def test_gradient_workgroups_with_several_tiles(ops, M, N, K, dtype):
    test_large_gradients_against_64_bits(ops, M, N, K, dtype)


def test_several_tiles_captured_and_on_two_streams(ops):
    a, b = random_codes(2600, 1100, 5).to(DEV), random_codes(9000, 1100, 6).to(DEV)
    sa, sb = torch.rand(2600, device=DEV), torch.rand(9000, device=DEV)
    want = ops.gemm8_nt(a, sa, b, sb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gemm8_nt(a, sa, b, sb)
    for i in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.gemm8_nt(a, sa, b, sb))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# small results on wave-private rings: the borders of the smaller and the larger workgroups, reductions of one unit, fewer and more
# than the waves take at once
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(33, 17, 100), (512, 512, 300), (513, 511, 640), (255, 2047, 1700), (257, 2048, 130), (100, 1000, 5000), (1025, 100, 900), (4000, 33, 500)])
def test_small_results_against_64_bits(ops, M, N, K, dtype):
    test_large_products_against_64_bits(ops, M, N, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 100, 17), (128, 300, 1024), (129, 640, 1023), (255, 1700, 1024), (257, 130, 1024), (16, 5000, 4097), (33, 4000, 700), (1025, 900, 100), (4000, 500, 33)])
def test_small_gradients_against_64_bits(ops, M, N, K, dtype):
    test_large_gradients_against_64_bits(ops, M, N, K, dtype)


# one launch for small products: the borders of its rule in rows, channels and reduction, ragged everywhere, views and rows that are not finite
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(3, 1, 1), (16, 16, 128), (17, 33, 129), (300, 50, 511), (512, 512, 512), (513, 512, 512), (64, 2048, 1000), (65, 2048, 1000), (255, 255, 513),
                                   (64, 1024, 2048), (65, 1024, 2047), (7, 200, 1025), (16000, 16, 40)])
def test_one_launch_equals_rows_then_product(ops, M, N, K, dtype):
    x = make_rows(M, K + 3, dtype, 8).to(DEV)[:, 1:K + 1]
    codes, scale = ops.quantize_rows8(torch.randn(N, K, device=DEV))
    bias = torch.randn(N, device=DEV).to(dtype)
    xc, xs = ops.quantize_rows8(x)
    assert same(ops.linear8_forward(x, codes, scale, bias), ops.gemm8_nt(xc, xs, codes, scale, bias, dtype, K=K))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (16, 128, 16), (17, 129, 33), (300, 511, 50), (128, 512, 1024), (129, 513, 100), (256, 1024, 256), (257, 1000, 256), (512, 1024, 256), (8, 1023, 4096)])
def test_gradients_in_one_launch(ops, M, N, K, dtype):
    """Against 64 bits, and row by row the same as of a taller gradient, which takes other kernels."""
    test_large_gradients_against_64_bits(ops, M, N, K, dtype)
    w, scale = ops.quantize_rows8(torch.randn(N, K, device=DEV))
    t = ops.transpose8(w, K)
    dy = make_rows(9000, N, dtype, 9).to(DEV)
    if K >= 16:
        assert same(ops.linear8_backward(dy, t, scale)[:M], ops.linear8_backward(dy[:M], t, scale))
