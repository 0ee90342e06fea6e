"""Int8Linear as a module, on the CPU: the product itself is replaced by one that reads the values alone, as the kernels do."""
import pytest
import torch

from slim_amd import ops, packed
from slim_amd.packed import Int8Linear

N, K = 6, 10


def values_only(x, codes, scale, bias=None):
    """What linear8_forward sees of its input: raw memory, without derivatives."""
    y = torch.from_numpy(x.detach().numpy().copy()) @ (codes[:, :x.shape[1]].float() * scale[:, None]).t()
    return y if bias is None else y + bias


@pytest.fixture
def layer(monkeypatch):
    monkeypatch.setattr(ops, "linear8_forward", values_only)
    codes = torch.zeros(N, 128, dtype=torch.int8)
    codes[:, :K] = torch.randint(-127, 128, (N, K), generator=torch.Generator().manual_seed(0)).to(torch.int8)
    return Int8Linear.from_tensors(dict(codes=codes, scale=torch.rand(N) + 0.1), N, K, "cpu")


def test_forward_mode_derivatives_are_refused(layer):
    """Not dropped: nn.Linear, which the module replaces, gives a tangent."""
    x, t = torch.randn(3, K), torch.randn(3, K)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            layer(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            layer(dual)
        assert layer(x).shape == (3, N)                    # (an input without a tangent is served)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(layer, (x,), (t,))
    assert torch.allclose(layer(x), x @ layer.dense_weight().t(), atol=1e-5)
