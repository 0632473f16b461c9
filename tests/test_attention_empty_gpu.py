"""Extents of zero through the attention training operators: what has no entries is returned without entries,
a sum over nothing is zero, and a query that sees no key has O = 0 and lse = -inf."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def tables(rows, R):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def dirty(n):
    """The allocator's next block of n floats holds NaN."""
    torch.full((n,), math.nan, device="cuda")
    torch.cuda.synchronize()


@pytest.mark.parametrize("D,R", [(64, 64), (66, 50)])
def test_weight_gradient_of_no_key_heads_is_zero(cuda_device, D, R):
    from kernelcodegen_b200 import ops

    cos, sin = tables(5, R)
    q, dq_out = make((2, 3, 5, D), 1), make((2, 3, 5, D), 2)
    k = torch.empty((2, 0, 5, D), device="cuda", dtype=torch.bfloat16)
    w = make((D,), 3)
    want = ops.qk_norm_rope_backward(dq_out, None, q, None, cos, sin, q_weight=w)
    for q_weight in (w, None):
        dirty(D)
        dq, dk, dwq, dwk = ops.qk_norm_rope_backward(dq_out, k, q, k, cos, sin, q_weight=q_weight, k_weight=w)
        assert dk.shape == k.shape and dwk.shape == (D,) and (dwk == 0).all()
        if q_weight is not None:
            assert torch.equal(dq, want[0]) and torch.equal(dwq, want[2])
    assert ops.last_device_status() == 0


def test_weight_gradient_of_no_key_heads_through_the_c_entry(cuda_device):
    from kernelcodegen_b200 import capi, ops

    lib, D, S, H = capi.load(), 64, 5, 3
    cos, sin = tables(S, D)
    q, dy = make((1, H, S, D), 1), make((1, H, S, D), 2)
    dq, dw = torch.empty_like(q), torch.full((D,), math.nan, device="cuda")
    d = capi.RopeDesc()
    d.B, d.S, d.H, d.Hk, d.D, d.R = 1, S, H, 0, D, D
    d.dtype, d.dtype_w, d.pos_bits, d.table_rows, d.eps = capi.KCG_BF16, capi.KCG_F32, 32, S, 1e-6
    for name in ("q", "q_out", "d_q"):
        setattr(d, name, (ctypes.c_int64 * 3)(H * S * D, S * D, D))
    ws = torch.empty(lib.kcg_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(d)), device="cuda", dtype=torch.uint8)
    st = lib.kcg_qk_norm_rope_bwd_launch(ctypes.byref(d), dy.data_ptr(), None, q.data_ptr(), None, None, None, cos.data_ptr(),
                                         sin.data_ptr(), None, dq.data_ptr(), None, None, dw.data_ptr(), ws.data_ptr(), ws.numel(),
                                         torch.cuda.current_stream().cuda_stream)
    assert st == capi.KCG_OK and (dw == 0).all()
    assert torch.equal(dq, ops.qk_norm_rope_backward(dy, None, q, None, cos, sin)[0])
