"""Refusals of the 8-bit linears and of the AdamW kernels, on the CPU: nothing is launched for them."""
import ctypes

import pytest
import torch

from slim_amd import _lib, ops


def rc_of(name, *args):
    rc = getattr(_lib.load(), name)(*args)
    return rc, _lib.load().slim_last_error().decode()


def test_sizes():
    lib = _lib.load()
    assert [lib.slim_rows8_ld(k) for k in (1, 127, 128, 129, 4096, 0, -3)] == [128, 128, 128, 256, 4096, 0, 0]
    assert [lib.slim_adamw_blocks(n) for n in (1, 512, 513, 0)] == [1, 1, 2, 0]
    assert lib.slim_linear8_workspace_bytes(5, 64, 2200) >= 5 * 2304 + 5 * 4 and lib.slim_linear8_workspace_bytes(0, 64, 100) == 0
    assert lib.slim_linear8_workspace_bytes(1, 64, 100) == lib.slim_linear8_workspace_bytes(5, 64, 100) == 0      # one launch, tokens quantised on the way
    assert lib.slim_linear8_backward_workspace_bytes(5, 64, 100, 1) == lib.slim_linear8_backward_workspace_bytes(5, 64, 100, 0) == 0
    assert lib.slim_linear8_backward_workspace_bytes(5, 1100, 100, 1) >= 2 * 16 * 1152 + 5 * 4
    assert lib.slim_linear8_backward_workspace_bytes(5, 1100, 100, 0) >= 3 * 16 * 1152 + 5 * 4
    assert lib.slim_linear8_backward_workspace_bytes(5, 64, 100, 7) == 0
    assert lib.slim_grad_norm_workspace_bytes(1) > 0 and lib.slim_grad_norm_workspace_bytes(0) == 0


P = 1 << 20        # (an address that nothing reads: every call below is refused before a launch)


@pytest.mark.parametrize("name,args", [
    ("slim_quantize_rows8", (None, 1, 4, 8, 8, P, 128, P, None)),
    ("slim_quantize_rows8", (P, 3, 4, 8, 8, P, 128, P, None)),
    ("slim_quantize_rows8", (P, 1, 0, 8, 8, P, 128, P, None)),
    ("slim_quantize_rows8", (P, 1, 4, 8, 7, P, 128, P, None)),
    ("slim_quantize_rows8", (P, 1, 4, 129, 129, P, 128, P, None)),
    ("slim_quantize_rows8", (P, 1, 4, 8, 8, P + 1, 128, P, None)),
    ("slim_quantize_rows8", (P, 1, 1 << 24, 8, 8, P, 128, P, None)),
    ("slim_transpose8", (P, 4, 8, 8, P, 128, None)),
    ("slim_transpose8", (P, 4, 8, 7, 2 * P, 128, None)),
    ("slim_transpose8", (P, 129, 8, 128, 2 * P, 128, None)),
    ("slim_gemm8_nt", (P, 128, P, P, 128, P, 4, 4, 129, None, 1, P, 4, None, 0, None)),
    ("slim_gemm8_nt", (P, 128, P, P, 128, P, 4, 4, 128, None, 1, P, 3, None, 0, None)),
    ("slim_gemm8_nt", (P, 128, P, P, 128, P, 4, 4, 128, None, 9, P, 4, None, 0, None)),
    ("slim_gemm8_nt", (P, 1 << 18, P, P, 1 << 18, P, 4, 4, 131072, None, 1, P, 4, None, 0, None)),
    ("slim_gemm8_nt", (P, 136, P, P, 128, P, 4, 4, 128, None, 1, P, 4, None, 0, None)),
    ("slim_linear8_forward", (P, 1, 2176, 4, 2176, P, P, 4, None, P, 4, P, 16, None)),
    ("slim_linear8_forward", (P, 1, 128, 4, 128, None, P, 4, None, P, 4, P, 1 << 20, None)),
    ("slim_linear8_backward", (P, 1, 1152, 4, 1152, P, P, 128, P, 128, P, 16, None)),
    ("slim_linear8_backward", (P, 1, 4, 4, 131072, P, P, 128, P, 128, P, 1 << 40, None)),
    ("slim_linear8_backward", (P, 5, 4, 4, 4, P, P, 128, P, 128, P, 1 << 20, None)),
])
def test_invalid_arguments_are_refused(name, args):
    rc, msg = rc_of(name, *args)
    assert rc == _lib.ERR_INVALID and name in msg, (rc, msg)


def step_args(count=1, dtype=1, numel=4, params=P, masters=None, scales=None, step=1, lr=1e-3, beta1=0.9, norm=None, max_norm=0.0, m=P):
    def arr(v):
        return (ctypes.c_void_p * max(count, 1))(*[v] * max(count, 1))
    keep = [arr(params), arr(P), arr(m), arr(P), None if scales is None else arr(scales), None if masters is None else arr(masters),
            (ctypes.c_int64 * max(count, 1))(*[numel] * max(count, 1))]
    a = [None if k is None else ctypes.addressof(k) for k in keep]
    return keep, (*a, count, dtype, 0, step, lr, beta1, 0.999, 1e-8, 0.0, norm, max_norm, 0, None)


@pytest.mark.parametrize("kw", [dict(count=0), dict(dtype=4), dict(numel=0), dict(numel=1 << 50), dict(params=None), dict(params=P + 1), dict(dtype=0, masters=P),
                                dict(step=0), dict(lr=-1.0), dict(beta1=1.0), dict(norm=P, max_norm=0.0), dict(m=P + 2), dict(scales=P + 2)])
def test_invalid_steps_are_refused(kw):
    keep, args = step_args(**kw)
    rc, msg = rc_of("slim_adamw_step", *args)
    assert rc == _lib.ERR_INVALID and "slim_adamw_step" in msg, (rc, msg)


def test_invalid_norms_are_refused():
    ptr, n = (ctypes.c_void_p * 1)(P), (ctypes.c_int64 * 1)(4)
    for args in [(None, ctypes.addressof(n), 1, 1, P, P, 1 << 20, None), (ctypes.addressof(ptr), ctypes.addressof(n), 1, 8, P, P, 1 << 20, None),
                 (ctypes.addressof(ptr), ctypes.addressof(n), 1, 1, P, P, 8, None), (ctypes.addressof(ptr), ctypes.addressof(n), 0, 1, P, P, 1 << 20, None)]:
        rc, msg = rc_of("slim_grad_norm", *args)
        assert rc == _lib.ERR_INVALID and "slim_grad_norm" in msg


def test_cpu_tensors_are_refused():
    x, c, s = torch.zeros(4, 8), torch.zeros(4, 128, dtype=torch.int8), torch.ones(4)
    for call in (lambda: ops.quantize_rows8(x), lambda: ops.transpose8(c, 8), lambda: ops.gemm8_nt(c, s, c, s), lambda: ops.linear8_forward(x, c, s),
                 lambda: ops.linear8_backward(x, c, s), lambda: ops.grad_norm([x]), lambda: ops.adamw_step([x], [x], [x], [x], step=1, lr=0.1)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="at least one tensor"):
        ops.grad_norm([])


def test_optimizer_arguments():
    from slim_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(state_bits=4), dict(max_grad_norm=0.0), dict(eps=-1e-8), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    opt = AdamW([p])
    opt.step()                       # no gradient: nothing to do
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()


def test_pack_model_refuses_unknown_forms():
    from slim_amd.packed import pack_model
    with pytest.raises(ValueError, match="form must be"):
        pack_model(None, form="int3")
