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


def test_hooks_of_the_linear_carry_over(layer):
    """Forward hooks and pre-hooks of either signature, those of the adapters' mask among them; not those whose work is done here."""
    from slim_amd.fine_tune import disable_linear_layer_grads
    from slim_amd.quantization.quantization import attach_input_quantization_hooks
    model = torch.nn.Module()
    model.model = torch.nn.Module()
    model.model.layers = torch.nn.ModuleList([torch.nn.Sequential(torch.nn.Linear(K, N), torch.nn.Linear(K, N))])
    adapted, plain = model.model.layers[0]
    adapted.lora_left = torch.nn.Parameter(torch.ones(K, 2))
    adapted.lora_right = torch.nn.Parameter(torch.ones(2, N))
    adapted.lora_left_mask = torch.zeros(K, 2, dtype=torch.bool)
    adapted.lora_left_mask[3] = True
    attach_input_quantization_hooks(model)
    disable_linear_layer_grads(model)
    seen = []
    adapted.register_forward_pre_hook(lambda module, args: seen.append("pre"))
    adapted.register_forward_pre_hook(lambda module, args, kwargs: seen.append(("pre", dict(kwargs))), with_kwargs=True)
    adapted.register_forward_hook(lambda module, args, out: seen.append("post"))
    adapted.register_forward_hook(lambda module, args, kwargs, out: out + 1, with_kwargs=True)
    adapted.register_full_backward_hook(lambda module, grad_in, grad_out: seen.append("backward"))
    adapted.register_forward_hook(lambda module, args, out: seen.append("always"), always_call=True)
    x = torch.randn(3, K)
    before = layer(x)
    layer.lora_left, layer.lora_left_mask = adapted.lora_left, adapted.lora_left_mask
    layer._take_hooks(adapted)
    with torch.no_grad():
        y = layer(x)
    assert seen == ["pre", ("pre", {}), "post", "always"] and torch.equal(y, before + 1)
    assert bool((layer.lora_left[3] == 0).all()) and bool((layer.lora_left[:3] == 1).all())
    with pytest.raises(ValueError, match="channels"):
        layer(x[:, 1:])
    assert seen[4:] == ["pre", ("pre", {}), "always"]
    assert len(layer._backward_hooks) == 1 and layer._is_full_backward_hook
    other = Int8Linear.from_tensors(dict(codes=layer.codes, scale=layer.scale), N, K, "cpu")
    other._take_hooks(plain)                                 # an input quantiser and the mask of a trained weight: neither is called
    assert torch.equal(other(x), before) and len(plain._forward_pre_hooks) == 2 and not other._forward_pre_hooks


def decoder(*linears):
    model = torch.nn.Module()
    model.model = torch.nn.Module()
    model.model.layers = torch.nn.ModuleList([torch.nn.Sequential(*linears)])
    return model


def test_files_hold_one_known_kind(layer, tmp_path):
    """A model of both kinds is not saved, a file of another format not loaded; the kind that a file names is what it becomes."""
    from safetensors.torch import save_file
    from slim_amd.packed import PackedLinear, load_packed, save_packed
    mixed = PackedLinear()
    mixed.sf = torch.ones(1)
    mixed.vals = mixed.meta = torch.zeros(8, dtype=torch.uint8)
    mixed.bias = mixed.LeffT = mixed.ReffT = mixed.qL = mixed.qR = None
    mixed.out_features, mixed.in_features, mixed.rank, mixed.a_div, mixed.qblock = 2, 16, 0, 1.0, 0
    with pytest.raises(ValueError, match="one kind"):
        save_packed(decoder(layer, mixed), str(tmp_path / "both"))
    assert not (tmp_path / "both").exists()
    save_file({"0.0.codes": layer.codes}, str(tmp_path / "foreign"), metadata={"format": "another/1", "layers": "{}"})
    with pytest.raises(ValueError, match="not a"):
        load_packed(decoder(torch.nn.Linear(K, N)), str(tmp_path / "foreign"), device="cpu")
    save_packed(decoder(layer), str(tmp_path / "int8"))
    model = decoder(torch.nn.Linear(K, N))
    assert load_packed(model, str(tmp_path / "int8"), device="cpu") == 1
    loaded = model.model.layers[0][0]
    x = torch.randn(3, K)
    assert isinstance(loaded, Int8Linear) and torch.equal(loaded.codes, layer.codes) and torch.equal(loaded(x), layer(x))
