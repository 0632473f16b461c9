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


def test_norm_and_rotation_of_no_query_heads(cuda_device):
    """The keys of a step whose queries live elsewhere."""
    from kernelcodegen_b200 import ops

    D = 64
    cos, sin = tables(9, D)
    q = torch.empty((2, 0, 5, D), device="cuda", dtype=torch.bfloat16)
    k, dk_out, w = make((2, 3, 5, D), 1), make((2, 3, 5, D), 2), make((D,), 3)
    at = torch.tensor([[0, 3, 8, 1, 2], [4, 4, 4, 7, 0]], device="cuda")
    kw = dict(positions=at, eps=1e-5, interleaved=True)
    want, _ = ops.qk_norm_rope(k, None, cos, sin, q_weight=w, **kw)
    into = torch.empty_like(k)
    y, yk = ops.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w, k_out=into, **kw)
    assert y.shape == q.shape and yk.data_ptr() == into.data_ptr() and torch.equal(yk, want)
    back = ops.qk_norm_rope_backward(dk_out, None, k, None, cos, sin, q_weight=w, **kw)
    dirty(D)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(q, dk_out, q, k, cos, sin, q_weight=w, k_weight=w, **kw)
    assert dq.shape == q.shape and (dwq == 0).all()
    assert torch.equal(dk, back[0]) and torch.equal(dwk, back[2])
    assert ops.last_device_status() == 0


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv", [(0, 4, 2, 5, 7), (2, 0, 2, 5, 7), (2, 4, 2, 0, 7), (2, 4, 2, 5, 0), (2, 4, 2, 0, 0), (2, 0, 0, 5, 7)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_nothing(cuda_device, B, H, Hkv, Sq, Skv, causal):
    from kernelcodegen_b200 import ops

    D = 64
    q, k, v, dout = make((B, H, Sq, D), 1), make((B, Hkv, Skv, D), 2), make((B, Hkv, Skv, D), 3), make((B, H, Sq, D), 4)
    room = torch.full((B, Sq, H + 1, D), 7.0, device="cuda", dtype=torch.bfloat16)
    for given in (None, room[:, :, :H].transpose(1, 2)):
        dirty(max(1, B * H * Sq))
        out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=causal, out=given)
        assert out.shape == q.shape and lse.shape == q.shape[:3] and lse.dtype == torch.float32
        assert (out == 0).all() and (lse == -math.inf).all()
    assert (room[:, :, H] == 7).all()
    dq, dk, dv = ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=causal)
    for g, t in ((dq, q), (dk, k), (dv, v)):
        assert g.shape == t.shape and g.dtype == t.dtype and (g == 0).all()
    assert ops.last_device_status() == 0


def test_attention_of_nothing_is_checked_like_any_other(cuda_device):
    from kernelcodegen_b200 import capi, ops

    q, k = make((2, 4, 0, 64), 1), make((2, 2, 7, 64), 2)
    lse = torch.empty((2, 4, 0), device="cuda")
    with pytest.raises(TypeError):
        ops.fmha_with_lse(q.float(), k.float(), k.float())
    with pytest.raises(capi.KcgError) as e:
        ops.fmha_with_lse(q, k, k, scale=0.0)
    assert e.value.status == capi.KCG_BAD_ARGUMENT
    with pytest.raises(capi.KcgError) as e:
        ops.fmha_with_lse(*(torch.empty((1, 2, 0, 96), device="cuda", dtype=torch.bfloat16),) * 3)
    assert e.value.status == capi.KCG_BAD_SHAPE
    with pytest.raises(ValueError):
        ops.fmha_backward(q, q, k, k, q, lse, dk=make((2, 2, 6, 64), 1))
    with pytest.raises(ValueError):          # three query heads of two key/value heads
        ops.fmha_with_lse(q[:, :3], k, k)
