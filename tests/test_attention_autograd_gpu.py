"""The attention training operators as autograd functions, in the pairing that their documentation gives: autograd's
gradients are those of the functions called by hand, and a plain formula's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def tables(rows, R):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal):
        from kernelcodegen_b200 import ops

        out, lse = ops.fmha_with_lse(q, k, v, scale=scale, causal=causal)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.args = dict(scale=scale, causal=causal)
        return out

    @staticmethod
    def backward(ctx, dout):
        from kernelcodegen_b200 import ops

        if not dout.stride(3) == 1 or 0 in dout.stride():
            dout = dout.contiguous()
        return (*ops.fmha_backward(dout, *ctx.saved_tensors, **ctx.args), None, None)


class NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, wq, wk):
        from kernelcodegen_b200 import ops

        ctx.save_for_backward(q, k, cos, sin, wq, wk)
        return ops.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk)

    @staticmethod
    def backward(ctx, dq, dk):
        from kernelcodegen_b200 import ops

        q, k, cos, sin, wq, wk = ctx.saved_tensors
        dq, dk, dwq, dwk = ops.qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=wq, k_weight=wk)
        return dq, dk, None, None, dwq.to(wq.dtype), dwk.to(wk.dtype)


@pytest.mark.parametrize("expanded", [False, True])
def test_the_pairing_for_autograd(cuda_device, expanded):
    """The gradients that autograd returns are those of the functions called by hand."""
    from kernelcodegen_b200 import ops

    B, S, H, Hkv, D = 2, 150, 4, 2, 64
    x, wq, wk = make((B, S, H + 2 * Hkv, D), 1), make((D,), 2), make((D,), 3)
    cos, sin = tables(S, D)
    leaves = [t.clone().requires_grad_() for t in (x, wq, wk)]
    q, k, v = (t.transpose(1, 2) for t in leaves[0].split([H, Hkv, Hkv], dim=2))
    out = Attention.apply(*NormRope.apply(q, k, cos, sin, *leaves[1:]), v, 0.125, True)
    dout = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(out.shape) if expanded else make(out.shape, 5)
    if expanded:
        out.sum().backward()
    else:
        out.backward(dout)
    q, k, v = (t.transpose(1, 2) for t in x.split([H, Hkv, Hkv], dim=2))
    qr, kr = ops.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk)
    o, lse = ops.fmha_with_lse(qr, kr, v, scale=0.125, causal=True)
    dqr, dkr, dv = ops.fmha_backward(dout.contiguous(), qr, kr, v, o, lse, scale=0.125, causal=True)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(dqr, dkr, q, k, cos, sin, q_weight=wq, k_weight=wk)
    assert torch.equal(out, o)
    assert torch.equal(leaves[0].grad, torch.cat([t.transpose(1, 2) for t in (dq, dk, dv)], 2))
    assert torch.equal(leaves[1].grad, dwq.to(wq.dtype)) and torch.equal(leaves[2].grad, dwk.to(wk.dtype))


def test_the_functions_alone_record_no_history(cuda_device):
    from kernelcodegen_b200 import ops

    q, k = make((1, 2, 40, 64), 1).requires_grad_(), make((1, 1, 40, 64), 2)
    cos, sin = tables(40, 64)
    out, lse = ops.fmha_with_lse(q, k, k)
    rotated, _ = ops.qk_norm_rope(q, k, cos, sin)
    assert not (out.requires_grad or lse.requires_grad or rotated.requires_grad)
