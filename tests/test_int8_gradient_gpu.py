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
