"""The 8-bit operators together, as a user has them: a compressed model whose linears run in 8-bit integers, its adapters
fine-tuned with 8-bit moments, saved, loaded and decoded token by token."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def compressed_linear(N, K, dtype=torch.bfloat16, bits=8, rank=16, bias=True):
    from slim_amd import ops
    from slim_amd.prune import add_lora_hook
    torch.manual_seed(N + K)
    lin = torch.nn.Linear(K, N, bias=bias).to(dtype).to(DEV)
    if bits:
        sf = torch.tensor([[2.0 ** (bits - 1) / 0.11]], device=DEV)
        c = torch.round(lin.weight.data.float() * sf).clamp(-2 ** (bits - 1), 2 ** (bits - 1) - 1)
        lin.weight.data = (c / sf).to(dtype)
        lin.scaling_factor = sf
    lin.lora_left = torch.nn.Parameter((torch.randn(K, rank, device=DEV) * 0.05).to(dtype))
    lin.lora_right = torch.nn.Parameter((torch.randn(rank, N, device=DEV) * 0.05).to(dtype))
    lin.lora_rank = torch.tensor(rank)
    lin.register_forward_hook(add_lora_hook)
    return lin, ops


def test_codes_of_a_compressed_weight_are_kept(gpu):
    from slim_amd.packed import Int8Linear
    for bits in (4, 8):
        lin, _ = compressed_linear(100, 300, bits=bits)
        m = Int8Linear(lin)
        assert torch.equal(m.dense_weight().bfloat16(), lin.weight.data)
    lin, ops = compressed_linear(100, 300, bits=0)
    m = Int8Linear(lin)
    codes, scale = ops.quantize_rows8(lin.weight.data)
    assert torch.equal(m.codes, codes) and torch.equal(m.scale, scale)


def test_layer_forward_and_gradients(gpu):
    """The layer with its adapter hook: the output is that of the quantised input and the dense weight of the codes; gradients of
    the input (both paths) and of the adapters against 64 bits."""
    from slim_amd.packed import Int8Linear
    N, K, r = 200, 300, 16
    lin, ops = compressed_linear(N, K)
    m = Int8Linear(lin)
    x = torch.randn(2, 37, K, device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn(2, 37, N, device=DEV).bfloat16()
    y = m(x)
    y.backward(dy)
    xc, xs = ops.quantize_rows8(x.detach().reshape(-1, K))
    xq = xc[:, :K].double() * xs.double()[:, None]
    L, R = m.lora_left.detach().double() / r ** 0.5, m.lora_right.detach().double() / r ** 0.5
    W, xd, d = m.dense_weight().double(), x.detach().double().reshape(-1, K), dy.double().reshape(-1, N)
    want = xq @ W.t() + lin.bias.double() + xd @ L @ R
    # roundings to bf16 on the way, 2^-8 each: base product, x L, the two adapters, their product, the sum
    size = (xq @ W.t()).abs() + lin.bias.double().abs() + xd.abs() @ L.abs() @ R.abs()
    assert bool(((y.detach().double().reshape(-1, N) - want).abs() <= 6 * 2.0 ** -8 * size).all())
    dx = d @ W + d @ R.t() @ L.t()
    size = d.abs() @ W.abs() + d.abs() @ R.abs().t() @ L.abs().t()
    assert bool(((x.grad.double().reshape(-1, K) - dx).abs() <= 6 * 2.0 ** -8 * size).all())
    for got, want, size in ((m.lora_left.grad, xd.t() @ (d @ R.t()) / r ** 0.5, xd.abs().t() @ (d.abs() @ R.abs().t()) / r ** 0.5),
                            (m.lora_right.grad, (xd @ L).t() @ d / r ** 0.5, (xd.abs() @ L.abs()).t() @ d.abs() / r ** 0.5)):
        assert bool(((got.double() - want).abs() <= 6 * 2.0 ** -8 * size).all())
    with torch.no_grad():
        assert torch.equal(m(x), y)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert m(x.detach().float()).dtype == torch.bfloat16
    with pytest.raises(ValueError, match="channels"):
        m(x[..., :-1])
    assert m(x[:, :0]).shape == (2, 0, N)


def test_captured_training_step_of_a_layer(gpu):
    """Forward and backward captured once the transposed codes are there; refused before."""
    from slim_amd.packed import Int8Linear
    lin, _ = compressed_linear(128, 256)
    m = Int8Linear(lin)
    x = torch.randn(5, 256, device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn(5, 128, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            m.transposed()
    m.transposed()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(m(x), [x], dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dx,) = torch.autograd.grad(m(x), [x], dy)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(5, 256, device=DEV))
        dy.copy_(torch.randn(5, 128, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, torch.autograd.grad(m(x), [x], dy)[0])


@pytest.mark.parametrize("optimizer", ["adamw_slim", "adamw_8bit", "adamw_bnb_8bit"])
def test_compress_pack_fine_tune_save_and_decode(gpu, optimizer, tmp_path):
    from transformers import LlamaConfig, LlamaForCausalLM
    import slim.fine_tune as F
    import slim.prune as P
    from slim.lora import quantize_lora
    from slim_amd.data import get_synthetic
    from slim_amd.optim import AdamW
    from slim_amd.packed import Int8Linear, load_packed, pack_model, save_packed
    from test_finetune import learnable_blocks
    torch.manual_seed(0)
    vocab, seq = 256, 32
    config = LlamaConfig(vocab_size=vocab, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=4,
                         max_position_embeddings=seq)
    m = LlamaForCausalLM(config).to(torch.bfloat16).cuda().eval()
    calib, _ = get_synthetic(8, 0, seq, vocab)
    saved = P.get_loaders, P.KEEP_ON_DEVICE
    P.get_loaders, P.KEEP_ON_DEVICE = (lambda *a, **k: (calib, None)), True
    try:
        P.prune_and_quantize(m, None, bitwidth=8, slim_quant=True, prune_method="wanda", sparsity_ratio=0.5, sparsity_type="2:4", quantize_weight=True, nsamples=8,
                             lora_rank=0.1, slim_lora=True, quantize_lora=optimizer == "adamw_8bit", lora_tile_size=256 if optimizer == "adamw_8bit" else None)
    finally:
        P.get_loaders, P.KEEP_ON_DEVICE = saved
    if optimizer == "adamw_8bit":
        quantize_lora(m, bitwidth=8, lora_tile_size=256)
    weights = {n: mod.weight.data.clone() for n, mod in m.named_modules() if hasattr(mod, "lora_left")}
    dense, packed = pack_model(m, form="int8")
    layers = {n: mod for n, mod in m.named_modules() if isinstance(mod, Int8Linear)}
    assert len(layers) == len(weights) == 14
    assert dense == sum(2 * w.numel() for w in weights.values())
    assert packed == sum(mod.codes.numel() + 4 * mod.out_features + 2 * (mod.lora_left.numel() + mod.lora_right.numel()) for mod in layers.values())
    for n, mod in layers.items():                                        # every weight lay on its 8-bit grid
        assert torch.equal(mod.dense_weight().bfloat16(), weights[n]), n
    before = {n: (mod.codes.clone(), mod.lora_left.data.clone(), mod.lora_right.data.clone()) for n, mod in layers.items()}
    train, evalb = learnable_blocks(32, seq, vocab), learnable_blocks(4, seq, vocab, seed=4)
    made = []
    saved = F.get_token_blocks, F.LEARNING_RATE, F.make_optimizer
    F.get_token_blocks = lambda *a, **k: (train, evalb)
    F.LEARNING_RATE = 1e-3
    F.make_optimizer = lambda *a: made.append(saved[2](*a)) or made[-1]
    try:
        F.fine_tune(m, None, global_batch_size=8, local_batch_size=4, optimizer=optimizer)
    finally:
        F.get_token_blocks, F.LEARNING_RATE, F.make_optimizer = saved
    assert isinstance(made[0], AdamW) and F.LAST_LOG[-1][0] == 4
    kinds = {t.dtype for s in made[0].state.values() for k, t in s.items() if k == "exp_avg"}
    assert (torch.float8_e4m3fn in kinds) == (optimizer != "adamw_slim")
    for n, mod in layers.items():
        c, l, r = before[n]
        assert torch.equal(mod.codes, c) and mod.scale.dtype == torch.float32
        assert not torch.equal(mod.lora_left.data, l) and not torch.equal(mod.lora_right.data, r), n
        assert bool(torch.isfinite(mod.lora_left.data.float()).all())
    # written and read back: the same logits, token by token with a cache and at once
    save_packed(m, str(tmp_path / "int8.safetensors"))
    torch.manual_seed(1)
    m2 = LlamaForCausalLM(config).to(torch.bfloat16).cuda().eval()
    m2.load_state_dict({k: v for k, v in m.state_dict().items() if "lora" not in k}, strict=False)
    assert load_packed(m2, str(tmp_path / "int8.safetensors")) == 14
    ids = evalb[:2].cuda()
    with torch.no_grad():
        whole = m(input_ids=ids).logits
        assert torch.equal(m2(input_ids=ids).logits, whole)
        m.config.use_cache = True
        cache, rows = None, []
        for t in range(6):
            out = m(input_ids=ids[:, t:t + 1], past_key_values=cache, use_cache=True)
            cache = out.past_key_values
            rows.append(out.logits[:, 0])
    assert bool(torch.isfinite(whole.float()).all())
    stepwise = torch.stack(rows, 1).float()
    # the same tokens in other batches: only roundings to bf16 (and the codes they tip) differ
    assert float((stepwise - whole[:, :6].float()).norm() / whole[:, :6].float().norm()) < 0.05


def test_files_of_the_other_kind_are_refused(gpu, tmp_path):
    from slim_amd.packed import save_packed, load_packed

    class Block(torch.nn.Module):
        pass
    model = torch.nn.Module()
    model.model = torch.nn.Module()
    model.model.layers = torch.nn.ModuleList([Block()])
    with pytest.raises(ValueError, match="no PackedLinear or Int8Linear"):
        save_packed(model, str(tmp_path / "x"))


def test_autocast_decides_the_type(gpu):
    """As for nn.Linear: under autocast the input of any 16- or 32-bit type is taken in autocast's type."""
    from slim_amd.packed import Int8Linear
    lin, _ = compressed_linear(100, 300)
    del lin.lora_left, lin.lora_right
    lin._forward_hooks.clear()
    m = Int8Linear(lin)
    x = torch.randn(5, 300, device=DEV)
    for to in (torch.bfloat16, torch.float16):
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            with torch.autocast("cuda", dtype=to):
                y = m(x.to(dtype))
            assert y.dtype == to and torch.equal(y, m(x.to(dtype).to(to)))
