"""Int8Linear on the GPU: what it takes over from the linear it replaces, and its files."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def test_pruned_adapters_stay_pruned_when_packed_late():
    """Packed after the adapters' masks were set up for training, in a training loop of one's own."""
    from slim_amd.fine_tune import disable_linear_layer_grads
    from slim_amd.packed import Int8Linear, pack_model
    from slim_amd.prune import add_lora_hook
    model = torch.nn.Module()
    model.model = torch.nn.Module()
    model.model.layers = torch.nn.ModuleList([torch.nn.Sequential(torch.nn.Linear(64, 32))])
    model = model.to(DEV).bfloat16()
    lin = model.model.layers[0][0]
    lin.lora_left = torch.nn.Parameter(torch.randn(64, 8, device=DEV).bfloat16())
    lin.lora_right = torch.nn.Parameter(torch.randn(8, 32, device=DEV).bfloat16())
    lin.lora_rank = torch.tensor(8)
    lin.lora_left_mask = torch.rand(64, 8, device=DEV) < 0.5
    lin.lora_left.data[lin.lora_left_mask] = 0
    lin.register_forward_hook(add_lora_hook)
    disable_linear_layer_grads(model)
    pack_model(model, form="int8")
    m = model.model.layers[0][0]
    assert isinstance(m, Int8Linear)
    opt = torch.optim.SGD([m.lora_left, m.lora_right], lr=0.1)
    for _ in range(3):
        opt.zero_grad()
        m(torch.randn(5, 64, device=DEV).bfloat16()).float().square().sum().backward()
        opt.step()
    with torch.no_grad():
        m(torch.randn(5, 64, device=DEV).bfloat16())
    assert not bool(m.lora_left[m.lora_left_mask].any()) and bool(m.lora_left[~m.lora_left_mask].all())


def test_transposed_codes_follow_the_codes_and_can_be_given_back():
    from slim_amd.packed import Int8Linear
    torch.manual_seed(0)
    m = Int8Linear(torch.nn.Linear(300, 200, bias=False).to(DEV))
    x, dy = torch.randn(7, 300, device=DEV, requires_grad=True), torch.randn(7, 200, device=DEV)

    def check():
        (dx,) = torch.autograd.grad(m(x), [x], dy)
        exact = dy.double() @ m.dense_weight().double()
        # sums of 200 fp32 products (each rounded, and the weight's too): 2^-23 for each at most
        size = dy.double().abs() @ m.dense_weight().double().abs()
        assert bool(((dx.double() - exact).abs() <= 210 * 2.0 ** -23 * size).all())
    check()
    kept = m.transposed()
    assert m.transposed() is kept
    m.codes.neg_()                                            # changed in place
    check()
    m.codes = m.codes.flip(0).contiguous()                    # replaced
    check()
    del kept
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    m.drop_transposed()
    assert before - torch.cuda.memory_allocated() >= 300 * 256
    check()
    with torch.inference_mode():
        n = Int8Linear(torch.nn.Linear(300, 200, bias=False).to(DEV))
    m.codes, m.scale = n.codes, n.scale
    check()
