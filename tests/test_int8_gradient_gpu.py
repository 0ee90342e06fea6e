"""The gradient of the 8-bit linears where the elements of a row of dy differ by orders of magnitude: every element counts with its own
precision, so that a column of dx whose codes are zero at the large elements keeps the bits of the small ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative
TINIEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
FLOOR = {torch.float32: 2.0 ** -61, torch.bfloat16: 2.0 ** -50, torch.float16: 2.0 ** -50}
# one launch (either length), and the tiles: few rows, more, many; rows kept in registers and rows read twice
SHAPES = [(5, 200, 300), (33, 1000, 260), (20, 4100, 130), (3, 17000, 200), (200, 2000, 1500), (900, 1300, 4000), (2050, 600, 7000)]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from slim_amd import ops as _ops
    return _ops


def half_zero_codes(ops, N, K, seed):
    """(codes, their transposed copy): half of them zero, as a pruned weight has them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randint(-127, 128, (N, K), generator=g, device=DEV) * torch.randint(0, 2, (N, K), generator=g, device=DEV)
    codes = torch.zeros(N, -(-K // 128) * 128, dtype=torch.int8, device=DEV)
    codes[:, :K] = w.to(torch.int8)
    return codes[:, :K], ops.transpose8(codes, K)


def documented(v, w, dtype):
    """(dx in 64 bits, the header's bound and the output's rounding).  v: dy * scale, an fp32 product (one rounding, 2^-24)."""
    N = v.shape[1]
    exact, size = v @ w.double(), v.abs() @ w.double().abs()
    allowed = ((N + 8) * 2.0 ** -23 + 2.0 ** -24) * size + FLOOR[dtype] * v.abs().amax(1, keepdim=True) * w.double().abs().sum(0)
    return exact, allowed * (1 + HALF[dtype]) + exact.abs() * HALF[dtype] * 1.01 + TINIEST[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_small_elements_beside_large_ones(ops, M, N, K, dtype):
    w, wt = half_zero_codes(ops, N, K, N)
    g = torch.Generator(device=DEV).manual_seed(K)
    scale = torch.exp(torch.randn(N, generator=g, device=DEV)) * 1e-3
    for ratio in (1e3, 1e5) if dtype == torch.float16 else (1e3, 1e5, 1e8, 1e11):
        dy = torch.randn(M, N, generator=g, device=DEV) * (0.1 if dtype == torch.float16 else 1.0)
        dy[:, N // 3] = ratio * (0.1 if dtype == torch.float16 else 1.0)
        dy = dy.to(dtype)
        dx = ops.linear8_backward(dy, wt, scale).double()
        v = dy.double() * scale.double()
        exact, allowed = documented(v, w, dtype)
        assert bool(((dx - exact).abs() <= allowed).all()), (ratio, float(((dx - exact).abs() / allowed).max()))
        # the columns that the large element does not reach: as precise as if it were not there, but for the second plane's floor
        blind = w[N // 3] == 0
        error, norm = (dx - exact)[:, blind].norm(dim=1), exact[:, blind].norm(dim=1)
        # every result's rounding to its type, dy * scale's to 2^-23, and sums in fp32 of terms N^0.5 times the result: all far below 2^-14
        assert bool((error <= norm * (HALF[dtype] * 1.01 + 2.0 ** -14) + (K ** 0.5) * TINIEST[dtype]).all()), (ratio, float((error / norm).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SHAPES[:2] + SHAPES[4:5])
@pytest.mark.parametrize("exponent", [-126, -110, -99, 60, 110])
def test_rows_of_any_size(ops, M, N, K, dtype, exponent):
    """Rows far below and far above 1 (rows below 2^-100 were once taken for zero).  Powers of two: dy * scale is exact."""
    w, wt = half_zero_codes(ops, N, K, 3)
    g = torch.Generator(device=DEV).manual_seed(4)
    scale = torch.ones(N, device=DEV)
    dy = (torch.randint(-64, 65, (M, N), generator=g, device=DEV).float() * 2.0 ** exponent).to(dtype)
    dx = ops.linear8_backward(dy, wt, scale).double()
    exact, allowed = documented(dy.double(), w, dtype)
    # the largest sums, up to 64 * 127 * N * 2^110 > 2^128, pass the type's largest number: infinity from half a step beyond it on (either
    # of the two within the bound around that border, to which a part in 2^20 of itself is added)
    border = 2.0 ** 128 * (1 - HALF[dtype] / 2)
    ok = dx.isfinite() & ((dx - exact).abs() <= allowed) | (dx == torch.sign(exact) * float("inf")) & (exact.abs() * (1 + 2.0 ** -20) >= border)
    assert bool(dx.any()) and bool(ok.all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K", [(600, 300), (1025, 300), (3000, 1500), (5000, 260)])
def test_a_rows_gradient_does_not_depend_on_the_others(ops, N, K, dtype):
    """The same bits alone, among few and among many, whichever kernels serve them."""
    w, wt = half_zero_codes(ops, N, K, 5)
    dy = (torch.randn(4100, N, device=DEV) * torch.exp(3 * torch.randn(4100, N, device=DEV))).to(dtype)
    scale = torch.rand(N, device=DEV) * 1e-3
    dx = ops.linear8_backward(dy, wt, scale)
    for a, b in ((0, 1), (17, 40), (100, 333), (4099, 4100), (1000, 2200)):
        # (rows in which fp16 holds an infinity, from 65520 on, are NaN on both sides)
        x, y = dx[a:b], ops.linear8_backward(dy[a:b], wt, scale)
        same = (x == y) | x.isnan() & y.isnan()
        assert bool(same.all()), (a, b)


def test_gradient_is_that_of_differences_of_the_dense_product(ops):
    """In 64 bits on the CPU: the loss (x @ W.T * dy).sum() moved along single inputs, W the weight that the codes stand for.  The
    loss is linear in x, so the quotient is the gradient up to the 64-bit sums' rounding."""
    M, N, K = 4, 60, 50
    w, wt = half_zero_codes(ops, N, K, 6)
    g = torch.Generator().manual_seed(7)
    scale = torch.rand(N, generator=g) * 1e-2
    dy, x = torch.randn(M, N, generator=g), torch.randn(M, K, generator=g).double()
    dx = ops.linear8_backward(dy.to(DEV), wt, scale.to(DEV)).cpu().double()
    W = w.cpu().double() * scale.double()[:, None]
    _, allowed = documented(dy.double() * scale.double(), w.cpu(), torch.float32)

    def loss(x):
        return ((x @ W.t()) * dy.double()).sum(1)
    for k in range(K):
        e = torch.zeros(K, dtype=torch.float64)
        e[k] = 0.5
        quotient = loss(x + e) - loss(x - e)
        assert bool(((quotient - dx[:, k]).abs() <= allowed[:, k] + 1e-9).all())


def close(ops, dx, dy, wt, scale, N, rows, cols=slice(None)):
    """Rows and columns of a gradient against 64 bits, within the header's bound."""
    w = wt[cols, :N].t()
    exact, allowed = documented(dy[rows].double() * scale.double(), w, dy.dtype)
    return bool(((dx[rows][:, cols].double() - exact).abs() <= allowed).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K", [(700, 300), (1500, 300)])
def test_gradients_of_views(ops, N, K, dtype):
    """Rows that start at odd elements, rows and columns apart, one row for all (what a sum sends back), transposed; one launch and two."""
    w, wt = half_zero_codes(ops, N, K, 8)
    scale = torch.rand(N, device=DEV) * 1e-2
    big = torch.randn(60, 2 * N + 9, device=DEV).to(dtype)
    for dy in (big[3:40, 1:N + 1], big[::3, 7:N + 7], big[:, :2 * N:2], big[5:6, 2:N + 2], big[1:2, :N].expand(33, N), big.t()[:N].t(), big[:N, :40].t()[:, :1].expand(40, N)):
        assert dy.shape[1] == N and close(ops, ops.linear8_backward(dy, wt, scale), dy, wt, scale, N, slice(None))


@pytest.mark.parametrize("M,N,K", [(19, 200, 70), (19, 1200, 70), (300, 1300, 2101), (2000, 1100, 5003)])
def test_gradient_rows_apart_and_what_lies_between(ops, M, N, K):
    """Through the C entry: results at an odd element, rows apart; nothing beside them is written."""
    from slim_amd import _lib
    w, wt = half_zero_codes(ops, N, K, 9)
    scale, dy = torch.rand(N, device=DEV) * 1e-2, torch.randn(M, N, device=DEV).bfloat16()
    ld = K + 29
    out = torch.full((M * ld + 40,), 7.0, device=DEV, dtype=torch.bfloat16)
    need = _lib.query("slim_linear8_backward_workspace_bytes", M, N, K, 1)
    ws = torch.full((need + 256,), 85, dtype=torch.uint8, device=DEV)
    _lib.call("slim_linear8_backward", dy.data_ptr(), 1, N, M, N, wt.data_ptr(), scale.data_ptr(), K, out.data_ptr() + 2, ld, ws.data_ptr() if need else None, need,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(torch.as_strided(out, (M, K), (ld, 1), 1), ops.linear8_backward(dy, wt, scale))
    torch.as_strided(out, (M, K), (ld, 1), 1).fill_(7.0)
    assert bool((out == 7.0).all()) and bool((ws[need:] == 85).all())


@pytest.mark.parametrize("M,N,K", [(40, 300, 500), (40, 1500, 500), (400, 1200, 2500), (1500, 2000, 4000)])
def test_captured_and_on_several_streams(ops, M, N, K):
    w, wt = half_zero_codes(ops, N, K, 10)
    scale = torch.rand(N, device=DEV) * 1e-2
    dy = torch.randn(M, N, device=DEV).bfloat16()
    ops.linear8_backward(dy, wt, scale)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                      # (two graphs that live at once, each with its workspace)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dx = ops.linear8_backward(dy, wt, scale)
        graphs.append((graph, dx))
    for i in range(4):
        dy.copy_(torch.randn(M, N, device=DEV) * 10.0 ** i)
        for graph, _ in graphs:
            graph.replay()
        ops.linear8_backward(torch.randn(M + 5, N, device=DEV), wt, scale)
        torch.cuda.synchronize()
        want = ops.linear8_backward(dy, wt, scale)
        assert all(torch.equal(dx, want) for _, dx in graphs)
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.linear8_backward(dy, wt, scale))
    torch.cuda.synchronize()
    assert all(torch.equal(dx, want) for dx in outs)


def test_gradient_offsets_beyond_32_bits(ops):
    """A result, the planes of the rows, and transposed codes of more than 2^31 elements each."""
    for M, N, K in ((70001, 1100, 32000), (1000001, 2048, 24)):
        w, wt = half_zero_codes(ops, N, K, 11)
        scale, dy = torch.rand(N, device=DEV) * 1e-2, torch.randn(M, N, device=DEV, dtype=torch.bfloat16)
        dx = ops.linear8_backward(dy, wt, scale)
        assert M * K > 2 ** 31 or 2 * M * N > 2 ** 31
        assert close(ops, dx, dy, wt, scale, N, [0, 1, M // 2, M - 17, M - 1])
        del dx, dy, w, wt
    N, K = 131071, 17001
    wt = torch.randint(-127, 128, (K, 131072), dtype=torch.int8, device=DEV)
    wt[:, N:] = 0
    scale = torch.rand(N, device=DEV) * 1e-2
    assert wt.numel() > 2 ** 31
    for dtype, M in ((torch.bfloat16, 5), (torch.float32, 300)):
        dy = torch.randn(M, N, device=DEV).to(dtype)
        dx = ops.linear8_backward(dy, wt, scale)
        for cols in (slice(0, 300), slice(K - 300, K)):
            assert close(ops, dx, dy, wt, scale, N, [0, M - 1], cols)
