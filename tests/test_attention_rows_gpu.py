"""A whole layer through the attention training operators, row by row: no row of a result is lost, stale or in
another's place, the last, ragged rows of a tile among them.

The chain is that of test_attention_block_gpu.py.  What bf16 between the operators does to a result, in its 2-norm
and in units of u^2 / 3 (a rounding is at most u = 2^-8 relative and u / sqrt(3) in the mean square, independent from
entry to entry): its own rounding 1; that of the gradient that it is computed from 1; P or dS as an operand 1; q and k
rounded, which moves a score by (|q||k| scale / sqrt(D) = 1 here) sqrt(2) u / sqrt(3), and P by as much of itself, 2;
O rounded, which moves delta by at most |dO||O| / sqrt(D) u / sqrt(3), where |dP - delta| is about |dO||v| / sqrt(D) and
|O| <= |v|, 1.  Together 6 / 3 u^2, so 1.42 u.  A whole tensor may be off by 2.5 times that, 3.5 u = 1.4e-2; one row (all
heads of a token) by 5 times that, 7 u = 2.7e-2.  A row that is lost or stale is off by 1 and more.  In the rows of dQ
that see fewer than 8 keys P may be near 1, where dP - delta is a difference of nearly equal numbers: those are
bounded in the whole tensor only."""
import math

import pytest
import torch

from test_attention_block_gpu import U, attention, layer, make, norm_rope, tables

pytestmark = pytest.mark.gpu


def off(got, want, dims):
    return (got.double() - want).square().sum(dims).sqrt() / want.square().sum(dims).sqrt()


@pytest.mark.parametrize("B,S,H,Hkv,D", [(2, 200, 4, 2, 128), (1, 333, 8, 4, 64), (1, 1030, 4, 4, 128), (2, 257, 8, 4, 64)])
def test_every_row_of_a_layer(cuda_device, B, S, H, Hkv, D):
    from kernelcodegen_b200 import ops

    x, wq, wk = make((B, S, H + 2 * Hkv, D), 1), make((D,), 2) * 0.2 + 1, make((D,), 3) * 0.2 + 1
    dout = make((B, S, H, D), 4).transpose(1, 2)
    cos, sin = tables(S, D)
    scale = D ** -0.5
    grad = torch.full_like(x, math.nan)
    out, dwq, dwk = layer(x, wq, wk, dout, H, Hkv, cos, sin, scale, grad)
    assert ops.last_device_status() == 0
    leaves = [t.double().requires_grad_() for t in (x, wq, wk)]
    q, k, v = (t.transpose(1, 2) for t in leaves[0].split([H, Hkv, Hkv], dim=2))
    qr, kr = (norm_rope(t, w, cos.double(), sin.double(), 1e-5) for t, w in ((q, leaves[1]), (k, leaves[2])))
    want = attention(qr, kr, v, scale, True)
    want.backward(dout.double())
    assert off(out, want.detach(), (0, 1, 2, 3)) <= 3.5 * U
    assert off(out, want.detach(), (1, 3)).max() <= 7 * U
    dx = leaves[0].grad
    for name, part in (("dq", slice(0, H)), ("dk", slice(H, H + Hkv)), ("dv", slice(H + Hkv, None))):
        got, ref = grad[:, :, part], dx[:, :, part]
        whole, rows = off(got, ref, (0, 1, 2, 3)).item(), off(got, ref, (2, 3))
        assert whole <= 3.5 * U, (name, whole)
        rows = rows[:, 7:] if name == "dq" else rows
        assert rows.max() <= 7 * U, (name, rows.max().item(), rows.argmax().item())
    for got, ref in ((dwq, leaves[1].grad), (dwk, leaves[2].grad)):
        assert off(got, ref, 0) <= 3.5 * U
