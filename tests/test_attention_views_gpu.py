"""Views that the attention training operators take side by side in one buffer, and those that they refuse with a
reason: expanded ones (stride 0), which autograd hands out."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def tables(rows, R):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


@pytest.mark.parametrize("layout", ["heads of a token in a row", "q, k, v of a head in a row", "tensors in a row", "batches interleaved"])
def test_everything_in_one_buffer(cuda_device, layout):
    """Inputs, output and gradients interleaved in one allocation: the bits of separate tensors."""
    from kernelcodegen_b200 import ops

    B, H, S, D = 2, 3, 70, 64
    n = 8                                   # q, k, v, out, dout, dq, dk, dv
    if layout == "heads of a token in a row":
        views = torch.zeros((B, S, n, H, D), device="cuda", dtype=torch.bfloat16).permute(2, 0, 3, 1, 4)
    elif layout == "q, k, v of a head in a row":
        views = torch.zeros((B, S, H, n, D), device="cuda", dtype=torch.bfloat16).permute(3, 0, 2, 1, 4)
    elif layout == "tensors in a row":
        views = torch.zeros((n, B, H, S, D), device="cuda", dtype=torch.bfloat16)
    else:
        views = torch.zeros((B, n, H, S, D), device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    q, k, v, out, dout, dq, dk, dv = views.unbind(0)
    flat = [make((B, H, S, D), s) for s in range(4)]
    for view, t in zip((q, k, v, dout), flat):
        view.copy_(t)
    _, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=True, out=out)
    ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=True, dq=dq, dk=dk, dv=dv)
    out2, lse2 = ops.fmha_with_lse(*flat[:3], scale=0.1, causal=True)
    grads = ops.fmha_backward(flat[3], *flat[:3], out2, lse2, scale=0.1, causal=True)
    for a, b in zip((out, lse, dq, dk, dv), (out2, lse2, *grads)):
        assert torch.equal(a, b)
    for view, t in zip((q, k, v, dout), flat):
        assert torch.equal(view, t)
    cos, sin = tables(S, D)
    want = ops.qk_norm_rope(flat[0], flat[1], cos, sin)
    ops.qk_norm_rope(q, k, cos, sin, q_out=dq, k_out=dk)
    assert torch.equal(dq, want[0]) and torch.equal(dk, want[1])
    grads = ops.qk_norm_rope_backward(flat[3], flat[2], flat[0], flat[1], cos, sin)
    ops.qk_norm_rope_backward(dout, v, q, k, cos, sin, dq=dq, dk=dk)
    assert torch.equal(dq, grads[0]) and torch.equal(dk, grads[1])
    ops.qk_norm_rope_backward(dout, v, q, k, cos, sin, dq=dout, dk=v)          # over the gradients that came in
    assert torch.equal(dout, grads[0]) and torch.equal(v, grads[1])
    assert torch.equal(q, flat[0]) and torch.equal(k, flat[1])
    assert ops.last_device_status() == 0


def test_one_place_of_a_cache_to_another(cuda_device):
    """A key read from one place of a cache and written to another, and over itself."""
    from kernelcodegen_b200 import ops

    cache = make((2, 3, 20, 64), 1)
    keep, q = cache.clone(), make((2, 4, 1, 64), 2)
    cos, sin = tables(20, 64)
    at = torch.tensor([7], device="cuda")
    _, want = ops.qk_norm_rope(q, keep[:, :, 4:5].contiguous(), cos, sin, positions=at)
    for to in (5, 3, 19, 4):
        ops.qk_norm_rope(q, cache[:, :, 4:5], cos, sin, positions=at, k_out=cache[:, :, to:to + 1])
        assert torch.equal(cache[:, :, to:to + 1], want)
    rest = [i for i in range(20) if i not in (3, 4, 5, 19)]
    assert torch.equal(cache[:, :, rest], keep[:, :, rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,R", [(128, 128), (96, 38)])
def test_gradients_over_the_inputs(cuda_device, dtype, D, R):
    """dq and dk written over q and k themselves, rows of a packed projection and of their own."""
    from kernelcodegen_b200 import ops

    B, S, H, Hk = 2, 531, 7, 3
    x, w = make((B, S, H + 2 * Hk, D), 1, dtype), make((D,), 2, dtype)
    q, k, v = (t.transpose(1, 2) for t in x.split([H, Hk, Hk], dim=2))
    cos, sin = tables(S, R)
    dyq, dyk, keep = make(q.shape, 3, dtype), make(k.shape, 4, dtype), v.clone()
    want = ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, q_weight=w, k_weight=w)
    flat = [q.contiguous(), k.contiguous()]
    for a, b in (flat, (q, k)):
        got = ops.qk_norm_rope_backward(dyq, dyk, a, b, cos, sin, q_weight=w, k_weight=w, dq=a, dk=b)
        for g, t in zip(got, want):
            assert torch.equal(g, t)
    assert torch.equal(v, keep) and ops.last_device_status() == 0


def test_expanded_tensors_are_refused_by_name(cuda_device):
    from kernelcodegen_b200 import ops

    q, k = make((2, 4, 64, 64), 1), make((2, 2, 64, 64), 2)
    out, lse = ops.fmha_with_lse(q, k, k)
    row = make((2, 4, 1, 64), 3)
    with pytest.raises(ValueError, match="dout.*stride 0.*contiguous"):
        ops.fmha_backward(row.expand(q.shape), q, k, k, out, lse)
    with pytest.raises(ValueError, match="dout.*stride 0.*contiguous"):         # what out.sum().backward() hands out
        ops.fmha_backward(torch.ones((), device="cuda", dtype=torch.bfloat16).expand(q.shape), q, k, k, out, lse)
    with pytest.raises(ValueError, match="K.*stride 0.*contiguous"):
        ops.fmha_with_lse(q, k[:, :1].expand(2, 4, 64, 64), k.repeat(1, 2, 1, 1))
    with pytest.raises(ValueError, match="V.*stride 0.*contiguous"):
        ops.fmha_with_lse(q, k, k[:1].expand(2, 2, 64, 64))
    # an extent of one has no stride to speak of
    one = make((1, 1, 1, 64), 4)
    a, b = ops.fmha_with_lse(one.as_strided((1, 1, 1, 64), (0, 0, 0, 1)), one, one)
    assert torch.equal(a, one) and torch.isfinite(b).all()
    # norm and rotation read expanded rows
    cos, sin = tables(64, 64)
    y, _ = ops.qk_norm_rope(row.expand(q.shape), None, cos, sin)
    assert torch.equal(y, ops.qk_norm_rope(row.expand(q.shape).contiguous(), None, cos, sin)[0])
    dy, _, _, _ = ops.qk_norm_rope_backward(row.expand(q.shape), None, q, None, cos, sin)
    assert torch.equal(dy, ops.qk_norm_rope_backward(row.expand(q.shape).contiguous(), None, q, None, cos, sin)[0])
