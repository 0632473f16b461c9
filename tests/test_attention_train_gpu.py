"""`ops.fmha_with_lse` and `ops.fmha_backward` against the formulas in 64 bits.

The bounds are worked out entry by entry from the roundings the kernels make (u = 2^-8, half a step of
bf16; e = 2^-23, a truncating 32-bit addition):
  scores      D products of bf16 are exact in 32 bits, their sum is off by at most D e (|q|.|k|)
  P           relative: that times scale, plus 6e-6 (2^x to 2.9e-6, lse and the scaled score rounded)
  dP, delta   D e (|dO|.|v|), D e (|dO|.|O|)
  P, dS       rounded to bf16 where they enter a product: u relative
  sums        n e times the sum of magnitudes, n terms
  results     rounded to bf16: u relative
  underflow   2^x gives 0 below 2^-126 and the products may drop operands below it, so every P and dS
              that enters a sum may lack up to 2^-126 (times what multiplies P in dS), and every result
The inputs of the backward pass are `out` and `lse` themselves, so nothing of the forward pass's
rounding enters the comparison."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, E, TINY = 2.0 ** -8, 2.0 ** -23, 2.0 ** -126


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def packed(B, H, Hkv, S, D, seed):
    """q, k, v as the heads of one projection."""
    x = make((B, S, H + 2 * Hkv, D), seed)
    return [t.transpose(1, 2) for t in x.split([H, Hkv, Hkv], dim=2)]


def repeat(t, H):
    return t.double().repeat_interleave(H // t.shape[1], dim=1)


def hidden(Sq, Skv):
    return torch.arange(Skv, device="cuda")[None, :] > torch.arange(Sq, device="cuda")[:, None] + (Skv - Sq)


def scores(q, k, scale, causal):
    qd, kd = q.double(), repeat(k, q.shape[1])
    z = qd @ kd.transpose(2, 3) * scale
    rel = qd.abs() @ kd.abs().transpose(2, 3) * scale * q.shape[3] * E
    if causal:
        z = z.masked_fill(hidden(q.shape[2], k.shape[2]), -math.inf)
    return z, rel


def check(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got[torch.isfinite(want)]).all(), f"{what}: not finite"
    over = ((got - want).abs() - bound).nan_to_num(nan=0.0)
    assert (over <= 0).all(), f"{what}: off by {(got - want).abs().max().item()}, {over.max().item()} over the bound"


def check_forward(q, k, v, scale, causal, out, lse):
    z, rel = scores(q, k, scale, causal)
    want_lse = torch.logsumexp(z, -1)
    empty = want_lse == -math.inf
    assert (lse[empty] == -math.inf).all()
    rel = torch.where(z == -math.inf, torch.zeros_like(z), rel)
    n = k.shape[2]
    err_lse = rel.amax(-1) + 6e-6 + n * E + want_lse.abs() * E
    check(torch.where(empty, 0, lse.double()), torch.where(empty, 0, want_lse), torch.where(empty, 0, err_lse), "lse")
    p = torch.exp(z - torch.where(empty, 0, want_lse)[..., None])
    vd = repeat(v, q.shape[1])
    want = p @ vd
    mags = p @ vd.abs()
    bound = (U + n * E + 6e-6) * mags + 2 * (p * rel) @ vd.abs() + err_lse.nan_to_num(posinf=0)[..., None] * mags + U * want.abs()
    check(out, want, bound * 1.01, "out")       # 1 %: products of the errors above


def check_backward(dout, q, k, v, out, lse, scale, causal, grads):
    H, D, n, m = q.shape[1], q.shape[3], k.shape[2], q.shape[2]
    z, rel = scores(q, k, scale, causal)
    at = lse.double()[..., None]
    p = torch.where(z == -math.inf, torch.zeros_like(z), torch.exp(z - at))
    g, o, vd, kd, qd = dout.double(), out.double(), repeat(v, H), repeat(k, H), q.double()
    dp, delta = g @ vd.transpose(2, 3), (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    relp = rel + 6e-6 + (at.abs() * E).nan_to_num(posinf=0)
    err_ds = p * (g.abs() @ vd.abs().transpose(2, 3) + (g * o).abs().sum(-1, keepdim=True)) * D * E + (relp + U) * ds.abs()
    err_ds = err_ds + TINY * (1 + dp.abs() + delta.abs())
    err_p = (relp + U) * p + TINY
    ha = H // k.shape[1] * m          # terms of dk and dv
    fold = lambda t: t.view(t.shape[0], k.shape[1], -1, *t.shape[2:]).sum(2)  # noqa: E731
    want = [ds @ kd * scale, fold(ds.transpose(2, 3) @ qd) * scale, fold(p.transpose(2, 3) @ g)]
    bound = [(err_ds + n * E * ds.abs()) @ kd.abs() * scale,
             fold((err_ds + ha * E * ds.abs()).transpose(2, 3) @ qd.abs()) * scale,
             fold((err_p + ha * E * p).transpose(2, 3) @ g.abs())]
    for name, got, w, b in zip(("dq", "dk", "dv"), grads, want, bound):
        check(got, w, 1.01 * b + U * w.abs() + TINY, name)


SHAPES = [  # B, H, Hkv, Sq, Skv, D
    (1, 1, 1, 128, 128, 64), (1, 2, 2, 256, 256, 128), (2, 3, 3, 200, 200, 64), (1, 2, 2, 200, 328, 128),
    (1, 1, 1, 1, 17, 64), (1, 2, 1, 384, 130, 128), (2, 4, 2, 1, 1, 128), (1, 6, 2, 129, 127, 64), (3, 7, 1, 65, 300, 128),
    (2, 8, 2, 513, 513, 128), (1, 5, 5, 1025, 1025, 64), (1, 2, 2, 333, 1777, 128), (1, 1, 1, 2, 1500, 64),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", SHAPES)
def test_forward_and_gradients(cuda_device, B, H, Hkv, Sq, Skv, D, causal):
    from kernelcodegen_b200 import ops

    q, k, v = make((B, H, Sq, D), 1), make((B, Hkv, Skv, D), 2), make((B, Hkv, Skv, D), 3)
    scale = D ** -0.5
    out, lse = ops.fmha_with_lse(q, k, v, scale=scale, causal=causal)
    check_forward(q, k, v, scale, causal, out, lse)
    dout = make((B, H, Sq, D), 4)
    grads = ops.fmha_backward(dout, q, k, v, out, lse, scale=scale, causal=causal)
    assert ops.last_device_status() == 0
    check_backward(dout, q, k, v, out, lse, scale, causal, grads)


@pytest.mark.parametrize("B,H,Hkv,S,D,causal", [(2, 4, 2, 300, 128, True), (2, 3, 1, 129, 64, False), (1, 8, 8, 257, 64, True)])
def test_views_of_a_packed_projection_and_into_one(cuda_device, B, H, Hkv, S, D, causal):
    """Heads of a packed projection in, O as [B, S, H, D] and the gradients as the heads of a packed
    gradient out: the same bits as with contiguous tensors, and nothing written beside the rows."""
    from kernelcodegen_b200 import ops

    q, k, v = packed(B, H, Hkv, S, D, 5)
    dout = make((B, S, H, D), 6).transpose(1, 2)
    scale = D ** -0.5
    room = torch.full((B, S + 1, H, D), 7.0, device="cuda", dtype=torch.bfloat16)
    out, lse = ops.fmha_with_lse(q, k, v, scale=scale, causal=causal, out=room[:, :S].transpose(1, 2))
    heads = H + 2 * Hkv
    grad = torch.full((B, S + 1, heads + 1, D), 7.0, device="cuda", dtype=torch.bfloat16)
    dq, dk, dv, _ = (t.transpose(1, 2) for t in grad[:, :S].split([H, Hkv, Hkv, 1], dim=2))
    ops.fmha_backward(dout, q, k, v, out, lse, scale=scale, causal=causal, dq=dq, dk=dk, dv=dv)
    flat = [t.contiguous() for t in (q, k, v)]
    out2, lse2 = ops.fmha_with_lse(*flat, scale=scale, causal=causal)
    grads = ops.fmha_backward(dout.contiguous(), *flat, out2, lse2, scale=scale, causal=causal)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    for a, b in zip((dq, dk, dv), grads):
        assert torch.equal(a, b)
    assert (room[:, S] == 7).all() and (grad[:, S] == 7).all() and (grad[:, :, heads] == 7).all()
    check_backward(dout, q, k, v, out, lse, scale, causal, grads)
    assert ops.last_device_status() == 0


def test_forward_agrees_with_fmha(cuda_device):
    """Head dimension 128 takes the same exponentials with and without the statistics."""
    from kernelcodegen_b200 import ops

    q, k, v = (make((2, 4, 700, 128), s) for s in (1, 2, 3))
    out, _ = ops.fmha_with_lse(q, k, v, scale=0.09, causal=True)
    assert torch.equal(out, ops.fmha(q, k, v, scale=0.09, causal=True))


def test_gradients_against_differences(cuda_device):
    """Directional derivatives of sum(O * dO), O in 64 bits, against the returned gradients."""
    from kernelcodegen_b200 import ops

    B, H, Hkv, S, D, scale = 1, 4, 2, 96, 64, 0.125
    q, k, v, dout = make((B, H, S, D), 1), make((B, Hkv, S, D), 2), make((B, Hkv, S, D), 3), make((B, H, S, D), 4)
    out, lse = ops.fmha_with_lse(q, k, v, scale=scale, causal=True)
    grads = ops.fmha_backward(dout, q, k, v, out, lse, scale=scale, causal=True)

    def value(q, k, v):
        z = (q @ k.repeat_interleave(H // Hkv, 1).transpose(2, 3) * scale).masked_fill(hidden(S, S), -math.inf)
        return ((torch.softmax(z, -1) @ v.repeat_interleave(H // Hkv, 1)) * dout.double()).sum()

    xs = [t.double() for t in (q, k, v)]
    for i, g in enumerate(grads):
        step = make(g.shape, 10 + i, torch.float32).double()
        h = 1e-4
        hi, lo = ([x + (s * h * step if j == i else 0) for j, x in enumerate(xs)] for s in (1, -1))
        want = (value(*hi) - value(*lo)) / (2 * h)
        got = (g.double() * step).sum()
        # every entry of g is off by about u of its size, independently: the sum by u times the 2-norm,
        # four times that for the tail; `out` rounded to bf16 moves delta by as much again
        assert (got - want).abs() <= 8 * U * (g.double() * step).norm(), (i, got.item(), want.item())


@pytest.mark.parametrize("D", [64, 128])
def test_queries_without_a_visible_key(cuda_device, D):
    """Causal with fewer keys than queries: the first rows are empty. Their O and dq are zero, and
    whatever their dout holds leaves the other gradients alone."""
    from kernelcodegen_b200 import ops

    q, k, v = make((1, 2, 400, D), 1), make((1, 2, 130, D), 2), make((1, 2, 130, D), 3)
    out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=True)
    assert (lse[:, :, :270] == -math.inf).all() and (out[:, :, :270] == 0).all()
    a, b = make((1, 2, 400, D), 4), make((1, 2, 400, D), 4)
    b[:, :, :270] = 1e30
    one, two = (ops.fmha_backward(t, q, k, v, out, lse, scale=0.1, causal=True) for t in (a, b))
    assert (one[0][:, :, :270] == 0).all()
    for x, y in zip(one, two):
        assert torch.equal(x, y)
    check_backward(a, q, k, v, out, lse, 0.1, True, one)


@pytest.mark.parametrize("spread", [4.0, 40.0, 400.0])
def test_wide_logits(cuda_device, spread):
    """Scores far below the row's largest, whole rows dominated by one key, and large lse."""
    from kernelcodegen_b200 import ops

    B, H, S, D = 1, 2, 300, 64
    q = torch.zeros((B, H, S, D))
    q[..., 0] = 1.0
    k = torch.randn((B, H, S, D), generator=torch.Generator().manual_seed(31)) * 0.01
    k[..., 0] = -torch.rand((B, H, S), generator=torch.Generator().manual_seed(32)) * spread + spread / 2
    q, k = q.bfloat16().cuda(), k.bfloat16().cuda()
    v, dout = make((B, H, S, D), 33), make((B, H, S, D), 34)
    for causal in (False, True):
        out, lse = ops.fmha_with_lse(q, k, v, causal=causal)
        check_forward(q, k, v, 1.0, causal, out, lse)
        check_backward(dout, q, k, v, out, lse, 1.0, causal, ops.fmha_backward(dout, q, k, v, out, lse, causal=causal))


def test_rows_further_apart_than_32_bits(cuda_device):
    """Batches 2^31 elements apart, in inputs, output and gradients."""
    from kernelcodegen_b200 import ops

    B, H, Hkv, S, D = 2, 3, 1, 140, 64
    room = torch.empty(2 ** 31 + 8 * H * S * D, device="cuda", dtype=torch.bfloat16)

    def place(heads, at):
        return room.as_strided((B, heads, S, D), (2 ** 31, S * D, D, 1), at * H * S * D)

    flat = [make((B, h, S, D), s) for s, h in enumerate((H, Hkv, Hkv, H))]
    q, k, v, dout = far = [place(t.shape[1], i) for i, t in enumerate(flat)]
    for a, b in zip(far, flat):
        a.copy_(b)
    out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=True, out=place(H, 4))
    grads = ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=True, dq=place(H, 5), dk=place(Hkv, 6), dv=place(Hkv, 7))
    out2, lse2 = ops.fmha_with_lse(*flat[:3], scale=0.1, causal=True)
    grads2 = ops.fmha_backward(flat[3], *flat[:3], out2, lse2, scale=0.1, causal=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    for a, b in zip(grads, grads2):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D,causal", [(1, 8, 1, 700, 700, 128, True), (1, 2, 2, 100, 3000, 64, False), (1, 6, 2, 2000, 90, 64, True)])
def test_items_in_pieces_into_a_packed_gradient(cuda_device, B, H, Hkv, Sq, Skv, D, causal):
    """Few items with long streams (each is cut, its pieces added up): the same bits on every call, views as
    outputs, nothing written past their rows."""
    from kernelcodegen_b200 import ops

    q, k, v, dout = make((B, H, Sq, D), 1), make((B, Hkv, Skv, D), 2), make((B, Hkv, Skv, D), 3), make((B, H, Sq, D), 4)
    out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=causal)
    first = ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=causal)
    check_backward(dout, q, k, v, out, lse, 0.1, causal, first)
    gq = torch.full((B, Sq + 1, H, D), 7.0, device="cuda", dtype=torch.bfloat16)
    gkv = torch.full((B, Skv + 1, 2 * Hkv, D), 7.0, device="cuda", dtype=torch.bfloat16)
    dq = gq[:, :Sq].transpose(1, 2)
    dk, dv = (t.transpose(1, 2) for t in gkv[:, :Skv].split([Hkv, Hkv], dim=2))
    ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=causal, dq=dq, dk=dk, dv=dv)
    for a, b in zip(first, (dq, dk, dv)):
        assert torch.equal(a, b)
    assert (gq[:, Sq] == 7).all() and (gkv[:, Skv] == 7).all()
    assert ops.last_device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_is_not_hidden(cuda_device, D):
    """A NaN in a query, a visible key or a value reaches the outputs that are made of it."""
    from kernelcodegen_b200 import ops

    base = [make((1, 2, 300, D), s) for s in (1, 2, 3)]
    for which in range(3):
        x = [t.clone() for t in base]
        x[which][0, 1, 290, 5] = math.nan
        out, lse = ops.fmha_with_lse(*x, scale=0.1)
        rows = slice(290, 291) if which == 0 else slice(None)
        at = out[0, 1, rows, 5] if which == 2 else out[0, 1, rows]
        assert at.isnan().all()
        assert which == 2 or lse[0, 1, rows].isnan().all()
        assert torch.isfinite(out[0, 0]).all()


def test_the_same_bits_every_time_and_on_another_stream(cuda_device):
    from kernelcodegen_b200 import ops

    q, k, v, dout = make((2, 8, 700, 128), 1), make((2, 2, 700, 128), 2), make((2, 2, 700, 128), 3), make((2, 8, 700, 128), 4)
    out, lse = ops.fmha_with_lse(q, k, v, scale=0.09, causal=True)
    first = ops.fmha_backward(dout, q, k, v, out, lse, scale=0.09, causal=True)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for _ in range(4):
        for s in side:      # two calls at once
            with torch.cuda.stream(s):
                results.append(ops.fmha_backward(dout, q, k, v, out, lse, scale=0.09, causal=True))
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


def test_captured_and_replayed(cuda_device):
    """Two graphs, replayed in turn with new inputs: each has its own scratch."""
    from kernelcodegen_b200 import ops

    graphs = []
    for S, D in ((260, 64), (131, 128)):
        q, k, v, dout = make((1, 4, S, D), 1), make((1, 2, S, D), 2), make((1, 2, S, D), 3), make((1, 4, S, D), 4)

        def step(q=q, k=k, v=v, dout=dout):
            out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=True)
            return ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=True)

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            result = step()
        graphs.append((g, (q, k, v, dout), result, step))
    for round_ in range(3):
        for g, inputs, _, _ in graphs:
            for i, t in enumerate(inputs):
                t.copy_(make(t.shape, 100 * round_ + i))
            g.replay()
        torch.cuda.synchronize()
        for _, _, result, step in graphs:
            for a, b in zip(result, step()):
                assert torch.equal(a, b)


def test_refusals(cuda_device):
    from kernelcodegen_b200 import capi, ops

    q = make((1, 4, 64, 64), 1)
    k = make((1, 2, 64, 64), 2)
    out, lse = ops.fmha_with_lse(q, k, k)
    with pytest.raises(TypeError):
        ops.fmha_with_lse(q.float(), k.float(), k.float())
    with pytest.raises(ValueError):
        ops.fmha_with_lse(q, make((1, 3, 64, 64), 2), make((1, 3, 64, 64), 2))
    with pytest.raises(capi.KcgError) as e:
        ops.fmha_with_lse(*(make((1, 2, 64, 96), 1),) * 3)
    assert e.value.status == capi.KCG_BAD_SHAPE
    with pytest.raises(capi.KcgError) as e:
        ops.fmha_with_lse(q, k, k, scale=0.0)
    assert e.value.status == capi.KCG_BAD_ARGUMENT
    with pytest.raises(ValueError):          # an expanded gradient: no entry has memory of its own
        ops.fmha_backward(torch.ones((), device="cuda", dtype=torch.bfloat16).expand(q.shape), q, k, k, out, lse)
    with pytest.raises(capi.KcgError) as e:  # rows that are not 16-byte aligned
        ops.fmha_with_lse(make((1, 4, 64, 68), 1)[..., :64], k, k)
    assert e.value.status == capi.KCG_BAD_ALIGN
    with pytest.raises(capi.KcgError) as e:  # heads that share one row of memory: the sum would be lost
        ops.fmha_backward(q, q, k, k, out, lse, dk=make((1, 1, 64, 64), 1).expand(1, 2, 64, 64))
    assert e.value.status == capi.KCG_BAD_SHAPE
    with pytest.raises(ValueError):
        ops.fmha_backward(q, q, k, k, out, lse.transpose(1, 2).contiguous())
    for given in (dict(dq=q), dict(dk=k), dict(dv=k), dict(dq=out)):     # over an input
        with pytest.raises(capi.KcgError) as e:
            ops.fmha_backward(q.clone(), q, k, k, out, lse, **given)
        assert e.value.status == capi.KCG_BAD_ARGUMENT
    same = torch.empty_like(k)
    with pytest.raises(capi.KcgError) as e:
        ops.fmha_backward(q, q, k, k, out, lse, dk=same, dv=same)
    assert e.value.status == capi.KCG_BAD_ARGUMENT
    with pytest.raises(capi.KcgError) as e:
        ops.fmha_with_lse(q, k, k, out=q)
    assert e.value.status == capi.KCG_BAD_ARGUMENT
