"""The attention training operators in a row, as a layer runs them: packed projection -> norm and rotation of
queries and keys -> attention -> gradients back into the packed projection; and the decoding step that
appends a token's key to a cache and attends to it.  Against the same chain in 64 bits.

Tolerances: every tensor that passes from one operator to the next is rounded to bf16, u = 2^-8 relative,
independently from entry to entry.  In the 2-norm over a tensor such a rounding is at most u of it, and a
rounding of the queries or keys moves the scores by u |scale q.k| ~ u |z|, hence P by u |z| relative,
|z| <= 6 in the tests; forward roundings: q, k, P, O (1 + 1 + 6 + 6 of them), backward the same ones again,
plus dO.O - delta, dS, and the gradients of the rotated rows: 32 u in all, of each result's own 2-norm and of
the value it is a difference of (dS has two terms of the size of P dP: twice that)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def tables(rows, R):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def norm_rope(x, w, c, s, eps):
    n = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    a, b = n.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attention(q, k, v, scale, causal):
    k, v = (t.repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v))
    z = q @ k.transpose(2, 3) * scale
    if causal:
        S, T = z.shape[-2:]
        z = z.masked_fill(torch.arange(T, device=z.device) > torch.arange(S, device=z.device)[:, None] + T - S, -math.inf)
    return torch.softmax(z, -1) @ v


def close(got, want, what):
    off = (got.double() - want).norm() / want.norm()
    assert off <= 32 * U, f"{what}: {off.item()} of its norm"


def layer(x, wq, wk, dout, H, Hkv, cos, sin, scale, grad):
    """Forward and backward through the operators; the gradient of x goes into `grad` (x's shape)."""
    from kernelcodegen_b200 import ops

    heads = [H, Hkv, Hkv]
    q, k, v = (t.transpose(1, 2) for t in x.split(heads, dim=2))
    dq, dk, dv = (t.transpose(1, 2) for t in grad.split(heads, dim=2))
    qr, kr = ops.qk_norm_rope(q, k, cos, sin, q_weight=wq, k_weight=wk, eps=1e-5)
    out, lse = ops.fmha_with_lse(qr, kr, v, scale=scale, causal=True)
    ops.fmha_backward(dout, qr, kr, v, out, lse, scale=scale, causal=True, dq=dq, dk=dk, dv=dv)
    _, _, dwq, dwk = ops.qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=wq, k_weight=wk, eps=1e-5, dq=dq, dk=dk)
    return out, dwq, dwk


@pytest.mark.parametrize("B,S,H,Hkv,D", [(2, 200, 4, 2, 128), (1, 333, 6, 1, 64), (3, 1, 2, 2, 64), (1, 1030, 4, 4, 128)])
def test_a_layer_forward_and_backward(cuda_device, B, S, H, Hkv, D):
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
    close(out, want.detach(), "out")
    if S == 1:      # one key: P is 1, and nothing depends on queries and keys
        v_grad = leaves[0].grad[:, :, H + Hkv:]
        close(grad[:, :, H + Hkv:], v_grad, "dv")
        # dS = P (dP - delta), both D products of about 1 with O = v rounded nowhere: at most D 2^-23 |dO|.|v|
        assert (grad[:, :, :H + Hkv].abs().amax() <= 1e-2) and (dwq.abs().amax() <= 1e-1)
        return
    for name, got, w in (("dq", grad[:, :, :H], leaves[0].grad[:, :, :H]), ("dk", grad[:, :, H:H + Hkv], leaves[0].grad[:, :, H:H + Hkv]),
                         ("dv", grad[:, :, H + Hkv:], leaves[0].grad[:, :, H + Hkv:]), ("dwq", dwq, leaves[1].grad), ("dwk", dwk, leaves[2].grad)):
        close(got, w, name)


def test_a_layer_captured(cuda_device):
    """The whole chain in one graph, replayed with new inputs: the bits of a plain run."""
    B, S, H, Hkv, D = 2, 150, 4, 2, 128
    x, wq, wk = make((B, S, H + 2 * Hkv, D), 1), make((D,), 2), make((D,), 3)
    dout = make((B, H, S, D), 4)
    cos, sin = tables(S, D)
    grad, plain = torch.zeros_like(x), torch.zeros_like(x)
    args = (x, wq, wk, dout, H, Hkv, cos, sin, 0.09)
    layer(*args, grad)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = layer(*args, grad)
    for seed in (10, 20):
        x.copy_(make(x.shape, seed))
        dout.copy_(make(dout.shape, seed + 1))
        graph.replay()
        want = layer(*args, plain)
        torch.cuda.synchronize()
        assert torch.equal(grad, plain)
        for a, b in zip(result, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("D,Hkv", [(64, 1), (128, 2)])
def test_decoding_into_a_cache(cuda_device, D, Hkv):
    """One token at a time: its rotated key is written into its place of the cache, and attention reads the
    filled part of the cache; what lies behind is left alone."""
    from kernelcodegen_b200 import ops

    B, H, room, start = 3, 4, 140, 126
    cos, sin = tables(room, D)
    keys, values = make((B, Hkv, room, D), 1), make((B, Hkv, room, D), 2)
    kept = keys.clone()
    for pos in range(start, start + 4):
        x = make((B, 1, H + 2 * Hkv, D), 10 + pos)
        q, k, v = (t.transpose(1, 2) for t in x.split([H, Hkv, Hkv], dim=2))
        at = torch.full((B, 1), pos, dtype=torch.int32, device="cuda")
        qr, _ = ops.qk_norm_rope(q, k, cos, sin, positions=at, k_out=keys[:, :, pos:pos + 1])
        values[:, :, pos:pos + 1] = v
        out, lse = ops.fmha_with_lse(qr, keys[:, :, :pos + 1], values[:, :, :pos + 1], scale=D ** -0.5)
        c, s = cos.double()[pos], sin.double()[pos]
        close(keys[:, :, pos:pos + 1], norm_rope(k.double(), 1, c, s, 1e-6), "key")
        close(out, attention(norm_rope(q.double(), 1, c, s, 1e-6), keys[:, :, :pos + 1].double(), values[:, :, :pos + 1].double(), D ** -0.5, False), "out")
    assert torch.equal(keys[:, :, :start], kept[:, :, :start]) and torch.equal(keys[:, :, start + 4:], kept[:, :, start + 4:])
    assert ops.last_device_status() == 0


def test_stores_stay_inside_their_buffers(cuda_device):
    """The same tests of views, pieces and layers under the bounds-checking build, where a store outside its
    buffer is skipped and sets the status word that they read."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    from kernelcodegen_b200 import build

    build.build_bounds()
    here = Path(__file__).resolve().parent
    files = [str(here / f) for f in ("test_attention_train_gpu.py", "test_qk_norm_rope_gpu.py", "test_attention_block_gpu.py")]
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-k", "views or pieces or forward_and or cache", *files],
                         env=dict(os.environ, KCG_DEBUG_BOUNDS="1"), capture_output=True, text=True, timeout=600, cwd=here.parent)
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-1000:]
