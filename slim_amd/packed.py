"""Inference from packed storage: a compressed nn.Linear (2:4 sparse 4-bit weight + low-rank adapters, as
slim.prune.prune_and_quantize / slim.lora.quantize_lora leave it) is replaced by a module that keeps the
weight at 0.375 byte per element and runs Linear + adapter hook (reference slim/prune.py:303-321) as two
fused launches.  The reference itself only emulates this forward with dense bf16 tensors.

Int8Linear is the 8-bit counterpart, for linears with any pattern of zeros: the weight as int8 codes with one scale per
output channel, the input quantised token by token, the product in whole numbers (the reference emulates it with fake-quantised
bf16 tensors, slim/quantization/quantization.py:219-263, :266-304).  Its adapters stay what they were, and it passes gradients
to its input, so the adapters can be fine-tuned over the frozen 8-bit weight (slim_amd.fine_tune)."""
import math

import torch

from . import ops
from .utils import get_layers_list, find_layers


# From this many rows on, the forward expands the packed weight into a transient dense bf16 tensor (one streaming
# kernel, 2 B written per element) and multiplies with the library GEMM (hipBLASLt through torch.matmul).  Off by
# default: the library's own large-batch kernel (128 x 256 tile, sparse MFMA) is level with or ahead of the dense
# emulated forward from 512 rows on, and the expansion costs 0.1 ms per call on top of the dense product (28672 x 8192:
# 0.75 x the emulated forward at 512-1024 rows).  Storage stays packed either way.
LARGE_BATCH = int(__import__("os").environ.get("SLIM_PACKED_LARGE_BATCH", str(1 << 30)))
# Keep 4-bit group-quantised adapters as codes + scales for the small-batch path (0.5 instead of 2 bytes per
# adapter element in HBM).  Off by default: rebuilding bf16(code / 7 * alpha) in registers costs more VALU time
# than the bytes save on MI355X (28672 x 8192, rank 1024, batch 1: 81 us against 63 us with bf16 operands), so it
# is a memory-footprint option, not a speed one.
Q4_ADAPTERS = __import__("os").environ.get("SLIM_PACKED_Q4_ADAPTERS", "0") == "1"


class PackedLinear(torch.nn.Module):
    """Drop-in for a compressed nn.Linear (inference only).

    Built from the attributes the compression leaves on the layer: weight.data (dequantised values),
    scaling_factor, and optionally lora_left [K, r], lora_right [r, N], lora_rank, lora_quantizer.
    """

    def __init__(self, lin=None):
        super().__init__()
        self._ws = None
        if lin is None:              # filled by from_tensors
            return
        W = lin.weight.data
        if not W.is_cuda or W.dtype != torch.bfloat16:
            raise RuntimeError("PackedLinear needs a bf16 weight on the GPU (slim_amd has no CPU path)")
        sf = getattr(lin, "scaling_factor", None)
        if sf is None:
            raise ValueError("the layer has no scaling_factor: it was not quantised by prune_and_quantize")
        self.out_features, self.in_features = W.shape
        self.sf = sf.detach().to(torch.float32).reshape(1).contiguous()
        self.vals, self.meta = ops.pack24(W.contiguous(), self.sf)
        self.bias = None if lin.bias is None else lin.bias.data.to(torch.bfloat16).contiguous()
        self.rank = 0
        self.a_div = 1.0
        self.LeffT = self.ReffT = None
        self.qL = self.qR = None       # 4-bit adapter operands of the small-batch path
        self.qblock = 0
        if hasattr(lin, "lora_left"):
            r = int(lin.lora_rank)
            sqrt_r = torch.sqrt(lin.lora_rank)        # on the device the reference computes it on (lora_rank's own)
            L, R = lin.lora_left.data, lin.lora_right.data
            q = getattr(lin, "lora_quantizer", None)
            if q is not None:
                # QuantizedMatmul re-quantises the stored adapters on every call (quantization.py:313-317)
                # and the hook divides the activations by sqrt(rank) (prune.py:305-312)
                if not q.block_quantization:
                    raise NotImplementedError("PackedLinear supports group-quantised adapters only")
                L, aL, cL = ops.group_fake_quant(L.contiguous(), q.block_dim, q.num_bits, want_codes=True)
                R, aR, cR = ops.group_fake_quant(R.contiguous(), q.block_dim, q.num_bits, want_codes=True)
                self.a_div = float(sqrt_r)
                if Q4_ADAPTERS and q.num_bits == 4 and q.block_dim % 32 == 0:
                    # codes and scales themselves, laid out for the small-batch kernel (0.5 byte per element)
                    self.qblock = int(q.block_dim)
                    self.qL = ops.pack_q4_operand(cL.t().contiguous(), aL.t().contiguous(), -(-r // 128) * 128)
                    self.qR = ops.pack_q4_operand(cR.t().contiguous(), aR.t().contiguous())
            else:
                # prune.py:317-321 divides the adapters by sqrt(rank) on every call
                sqrt_r = sqrt_r if sqrt_r.dim() == 0 and not sqrt_r.is_cuda else sqrt_r.to(W.device)
                L, R = L / sqrt_r, R / sqrt_r
            r8, r128 = -(-r // 8) * 8, -(-r // 128) * 128
            self.LeffT = torch.zeros(r128, self.in_features, dtype=torch.bfloat16, device=W.device)
            self.LeffT[:r] = L.t()
            self.ReffT = torch.zeros(self.out_features, r8, dtype=torch.bfloat16, device=W.device)
            self.ReffT[:, :r] = R.t()
            self.rank = r
        for hook_id, hook in lin._forward_pre_hooks.items():      # input fake-quantisation hooks carry over
            self._forward_pre_hooks[hook_id] = hook

    TENSORS = ("vals", "meta", "sf", "bias", "LeffT", "ReffT", "qL_codes", "qL_alpha", "qR_codes", "qR_alpha")

    @classmethod
    def from_tensors(cls, tensors, out_features, in_features, rank, a_div, device, qblock=0):
        """Rebuild from the tensors `state()` returns (a checkpoint written by save_packed)."""
        self = cls()
        self.out_features, self.in_features, self.rank, self.a_div = int(out_features), int(in_features), int(rank), float(a_div)
        self.qblock = int(qblock)
        got = {k: (None if tensors.get(k) is None else tensors[k].to(device).contiguous()) for k in cls.TENSORS}
        for k in ("vals", "meta", "sf", "bias", "LeffT", "ReffT"):
            setattr(self, k, got[k])
        self.qL = (got["qL_codes"], got["qL_alpha"]) if got["qL_codes"] is not None else None
        self.qR = (got["qR_codes"], got["qR_alpha"]) if got["qR_codes"] is not None else None
        if self.vals.numel() * 4 != self.out_features * self.in_features or self.meta.numel() * 8 != self.vals.numel() * 4:
            raise ValueError("packed tensors do not match the recorded shape")
        return self

    def state(self):
        out = {k: getattr(self, k) for k in ("vals", "meta", "sf", "bias", "LeffT", "ReffT") if getattr(self, k) is not None}
        if self.qL is not None:
            out.update(qL_codes=self.qL[0], qL_alpha=self.qL[1], qR_codes=self.qR[0], qR_alpha=self.qR[1])
        return out

    def packed_bytes(self):
        """Bytes the small-batch forward streams: packed weight + adapters (4-bit when quantised, else bf16)."""
        n = self.vals.numel() + self.meta.numel()
        if self.qL is not None:
            n += sum(t.numel() * t.element_size() for t in self.qL + self.qR)
        elif self.rank:
            n += 2 * (self.LeffT.numel() + self.ReffT.numel())
        return n

    def dense_weight(self):
        """The dequantised bf16 weight (what the reference keeps in weight.data)."""
        return ops.unpack24(self.vals, self.meta, self.sf, self.out_features, self.in_features)

    def forward(self, x):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1])
        if x2.dtype != torch.bfloat16:
            x2 = x2.to(torch.bfloat16)
        if x2.shape[0] >= LARGE_BATCH:
            y = self._forward_expanded(x2)
        elif self.qL is not None and x2.shape[0] <= 16:
            y = ops.linear24_forward_q4(x2.contiguous(), self.vals, self.meta, self.sf, self.out_features, self.bias,
                                        self.qL, self.qR, self.rank, self.qblock, self.a_div)
        else:
            y = ops.linear24_forward(x2.contiguous(), self.vals, self.meta, self.sf, self.out_features, self.bias,
                                     self.LeffT, self.ReffT, self.rank, self.a_div)
        return y.reshape(*shape[:-1], self.out_features)

    def _forward_expanded(self, x2):
        """Large batches: transient dense weight + library GEMMs, adapter terms as in prune.py:303-321."""
        y = torch.nn.functional.linear(x2, self.dense_weight(), self.bias)
        if self.rank:
            r = self.rank
            xs = x2 if self.a_div == 1.0 else x2 / self.a_div
            t = torch.matmul(xs, self.LeffT[:r].t())
            if self.a_div != 1.0:
                t = t / self.a_div
            y += torch.matmul(t, self.ReffT[:, :r].t())
        return y

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, rank={self.rank}, packed 2:4 int4"


class _Int8Product(torch.autograd.Function):
    """The product of Int8Linear; its gradient passes the quantisation of the input straight through (as the reference's
    QuantizedMatmul does with the weight's, quantization.py:322-328).  The weight and bias are frozen."""

    @staticmethod
    def forward(ctx, x, module):
        ctx.module = module
        return module.product(x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return ops.linear8_backward(dy, ctx.module.transposed(), ctx.module.scale), None


class Int8Linear(torch.nn.Module):
    """Drop-in for an nn.Linear in 8-bit integers, for inference and for fine-tuning adapters over it.

    A weight that lies on a per-tensor grid of at most 8 bits (what prune_and_quantize leaves: values code / scaling_factor) keeps
    its codes exactly; any other weight is quantised here, one scale per output channel (ops.quantize_rows8).  The activation
    is quantised token by token on every call.  Adapters (lora_left, lora_right, lora_rank, lora_quantizer, lora_left_mask) and
    hooks of the linear carry over, but for input fake-quantisation (the input is quantised here) and the mask of a trained
    weight (fine_tune; the codes are frozen).
    Derivatives are backward-mode: a forward-mode dual tensor is refused.
    As with PackedLinear the tensors are plain attributes: `model.to(dtype)` does not change them."""

    TENSORS = ("codes", "scale", "bias", "lora_left", "lora_right", "lora_left_mask")

    def __init__(self, lin=None):
        super().__init__()
        self._codes_t = None
        if lin is None:              # filled by from_tensors
            return
        W = lin.weight.data
        if not W.is_cuda:
            raise RuntimeError("Int8Linear needs a weight on the GPU (slim_amd has no CPU path)")
        self.out_features, self.in_features = W.shape
        self.codes, self.scale = self._codes_of(W, getattr(lin, "scaling_factor", None))
        self.bias = None if lin.bias is None else lin.bias.data.contiguous()
        for name in ("lora_left", "lora_right", "lora_rank", "lora_quantizer", "lora_left_mask"):
            if hasattr(lin, name):
                setattr(self, name, getattr(lin, name))
        self._take_hooks(lin)

    def _take_hooks(self, lin):
        """The linear's hooks with their marks, but for those that the module itself makes needless (input fake-quantisation, the mask
        of a trained weight)."""
        for name in ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks", "_forward_pre_hooks_with_kwargs",
                     "_backward_hooks", "_backward_pre_hooks"):
            getattr(self, name).update(getattr(lin, name))
        self._is_full_backward_hook = lin._is_full_backward_hook
        for hook_id, hook in list(self._forward_pre_hooks.items()):
            if getattr(hook, "needless_in_int8", False):
                del self._forward_pre_hooks[hook_id]
                self._forward_pre_hooks_with_kwargs.pop(hook_id, None)

    @staticmethod
    def _codes_of(W, sf):
        """(codes, scale): the grid of a per-tensor scaling factor where every value lies on it (one synchronisation), else
        quantised rows."""
        if sf is not None and sf.numel() == 1:
            sf = sf.detach().to(device=W.device, dtype=torch.float32).reshape(())
            c = torch.round(W.float() * sf)
            if bool(((c / sf).to(W.dtype) == W).all() & (c.amin() >= -128) & (c.amax() <= 127)):
                codes = torch.zeros(W.shape[0], -(-W.shape[1] // 128) * 128, dtype=torch.int8, device=W.device)
                codes[:, :W.shape[1]] = c.to(torch.int8)
                return codes, (1.0 / sf).expand(W.shape[0]).contiguous()
        return ops.quantize_rows8(W)

    @classmethod
    def from_tensors(cls, tensors, out_features, in_features, device, rank=None, quantizer=None):
        """Rebuild from the tensors `state()` returns (a checkpoint written by save_packed)."""
        from .prune import add_lora_hook
        from .quantization.quantization import Quantizer
        self = cls()
        self.out_features, self.in_features = int(out_features), int(in_features)
        got = {k: (None if tensors.get(k) is None else tensors[k].to(device).contiguous()) for k in cls.TENSORS}
        self.codes, self.scale, self.bias = got["codes"], got["scale"], got["bias"]
        if tuple(self.codes.shape) != (self.out_features, -(-self.in_features // 128) * 128) or self.scale.numel() != self.out_features:
            raise ValueError("8-bit tensors do not match the recorded shape")
        if got["lora_left"] is not None:
            self.lora_left, self.lora_right = torch.nn.Parameter(got["lora_left"]), torch.nn.Parameter(got["lora_right"])
            self.lora_rank = torch.tensor(rank)
            if got["lora_left_mask"] is not None:
                self.lora_left_mask = got["lora_left_mask"]
            if quantizer is not None:
                self.lora_quantizer = Quantizer("weight", **quantizer)
            self.register_forward_hook(add_lora_hook)
        return self

    def state(self):
        return {k: getattr(self, k).data for k in self.TENSORS if getattr(self, k, None) is not None}

    def info(self):
        """What from_tensors needs beside the tensors (plain values)."""
        out = dict(out_features=self.out_features, in_features=self.in_features)
        if hasattr(self, "lora_left"):
            out["rank"] = int(self.lora_rank)
            q = getattr(self, "lora_quantizer", None)
            if q is not None:
                out["quantizer"] = dict(num_bits=q.num_bits, slim_quant=q.slim_quant, block_quantization=q.block_quantization, block_dim=q.block_dim)
        return out

    def packed_bytes(self):
        """Bytes of codes and scales, and of the adapters where there are any."""
        return sum(t.numel() * t.element_size() for k, t in self.state().items() if k != "lora_left_mask")

    def dense_weight(self):
        """The weight the codes stand for, fp32 [N, K]."""
        return self.codes[:, :self.in_features].float() * self.scale[:, None]

    def transposed(self):
        """The codes in the order of the backward pass, laid out on its first use and kept until drop_transposed(), or until the codes are
        replaced or changed in place: a second byte per weight element, which packed_bytes does not count."""
        version = None if self.codes.is_inference() else self.codes._version
        if self._codes_t is None or self._codes_t[0] is not self.codes or self._codes_t[1] != version:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Int8Linear: the first backward pass lays out the transposed codes and cannot be captured; run one eagerly, "
                                   "or call transposed() before the capture")
            self._codes_t = self.codes, version, ops.transpose8(self.codes, self.in_features)
            torch.cuda.current_stream(self.codes.device).synchronize()       # (whatever stream uses them next)
        return self._codes_t[2]

    def drop_transposed(self):
        """Give the memory of transposed() back, after training; a later backward pass lays it out again.  (Not while a captured
        backward pass is still to be replayed: it reads that memory.)"""
        self._codes_t = None

    def product(self, x2):
        bias = self.bias
        if bias is not None and bias.dtype != x2.dtype:
            bias = bias.to(x2.dtype)
        return ops.linear8_forward(x2, self.codes, self.scale, bias)

    def forward(self, x):
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Int8Linear: the input has {x.shape[-1]} channels, the weight {self.in_features}")
        if torch.is_autocast_enabled("cuda") and x.dtype in (torch.float32, torch.bfloat16, torch.float16):
            x = x.to(torch.get_autocast_dtype("cuda"))
        x2 = x.reshape(-1, self.in_features)
        if torch.autograd.forward_ad.unpack_dual(x2).tangent is not None:
            raise NotImplementedError("Int8Linear has no forward-mode derivative (backward mode only)")
        y = _Int8Product.apply(x2, self) if torch.is_grad_enabled() and x2.requires_grad else self.product(x2)
        return y.reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, int8"


def pack_model(model, form="2:4"):
    """Replace every Linear of the decoder blocks in place: by a PackedLinear (form "2:4": compressed to 2:4 int4), or by
    an Int8Linear (form "int8": any weight).  Returns (dense bytes, packed bytes) of the replaced layers."""
    kinds = {"2:4": PackedLinear, "int8": Int8Linear}
    if form not in kinds:
        raise ValueError(f"form must be one of {sorted(kinds)}, got {form!r}")
    dense = packed = 0
    for layer in get_layers_list(model):
        subset = find_layers(layer)
        for name, lin in subset.items():
            parent = layer
            parts = name.split(".")
            for p in parts[:-1]:
                parent = getattr(parent, p)
            pl = kinds[form](lin)
            setattr(parent, parts[-1], pl)
            dense += lin.weight.numel() * 2
            packed += pl.packed_bytes()
    return dense, packed


FORMAT = "slim_amd.packed24/1"
FORMAT_INT8 = "slim_amd.int8/1"


def _packed_modules(model, kind=PackedLinear):
    for i, layer in enumerate(get_layers_list(model)):
        for name, mod in layer.named_modules():
            if isinstance(mod, kind):
                yield f"{i}.{name}", layer, name, mod


def save_packed(model, path):
    """Write every PackedLinear of `model` to one safetensors file: per layer `<block>.<name>.{vals,meta,sf,bias,
    LeffT,ReffT}` plus the shapes, rank and activation divisor in the file's metadata; or every Int8Linear:
    `<block>.<name>.{codes,scale,bias,lora_left,lora_right,lora_left_mask}`.  A model that holds both is refused.  The rest of
    the model (embeddings, norms, head) is not touched -- save it the usual way."""
    import json
    from safetensors.torch import save_file
    tensors, index = {}, {}
    for key, _, _, mod in _packed_modules(model):
        for k, t in mod.state().items():
            tensors[f"{key}.{k}"] = t.detach().cpu().contiguous()
        index[key] = dict(out_features=mod.out_features, in_features=mod.in_features, rank=mod.rank, a_div=mod.a_div,
                          qblock=mod.qblock)
    int8 = list(_packed_modules(model, Int8Linear))
    if index and int8:
        raise ValueError("the model holds both PackedLinear and Int8Linear layers; a file holds one kind")
    for key, _, _, mod in int8:
        for k, t in mod.state().items():
            tensors[f"{key}.{k}"] = t.detach().cpu().contiguous()
        index[key] = mod.info()
    if not index:
        raise ValueError("the model holds no PackedLinear or Int8Linear; call pack_model first")
    save_file(tensors, path, metadata={"format": FORMAT_INT8 if int8 else FORMAT, "layers": json.dumps(index)})
    return index


def load_packed(model, path, device="cuda"):
    """Replace the linears named in a save_packed file by PackedLinear (or Int8Linear) modules built from it (the model
    needs the right architecture, not the right weights).  Returns the number of layers replaced."""
    import json
    from safetensors import safe_open
    with safe_open(path, framework="pt", device="cpu") as f:
        meta = f.metadata() or {}
        kind = {FORMAT: PackedLinear, FORMAT_INT8: Int8Linear}.get(meta.get("format"))
        if kind is None:
            raise ValueError(f"{path} is not a {FORMAT} or {FORMAT_INT8} file")
        index = json.loads(meta["layers"])
        names = set(f.keys())
        layers = get_layers_list(model)
        for key, info in index.items():
            block, name = key.split(".", 1)
            tensors = {k: f.get_tensor(f"{key}.{k}") for k in kind.TENSORS if f"{key}.{k}" in names}
            parent = layers[int(block)]
            parts = name.split(".")
            for p in parts[:-1]:
                parent = getattr(parent, p)
            setattr(parent, parts[-1], kind.from_tensors(tensors, device=device, **info))
    return len(index)
