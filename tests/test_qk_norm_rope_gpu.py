"""`ops.qk_norm_rope` and its gradients against the formulas in 64 bits.

Bounds, entry by entry, in steps of 32-bit rounding e = 2^-24 (half a step) and of the type's own
u (bf16 2^-8, fp32 e): the mean square is off by at most (D + 2) e relative, its inverse root by half of
that and 3 e; every product and sum after it adds e of the magnitudes involved.  16 e covers those, D e
the sums over a row, and the number of rows times e the sums over rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def tables(rows, R):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def turn(x, c, s, R, interleaved, back=False):
    """The rotation of the first R entries, and the same with every term's magnitude."""
    i = torch.arange(R // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    if back:
        s = -s
    y, mag = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    mag[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    mag[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, mag


def angles(cos, sin, positions, B, S):
    at = positions if positions is not None else torch.arange(S, device="cuda")
    at = at.long().expand(B, S)
    return cos.double()[at][:, None], sin.double()[at][:, None]


def check(got, want, bound, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound).all(), f"{what}: off by {off.max().item()}, {(off - bound).max().item()} over the bound"


def forward(x, w, c, s, R, eps, interleaved):
    xd = x.double()
    D = x.shape[-1]
    n = xd * (xd.square().mean(-1, keepdim=True) + eps).rsqrt() * (1 if w is None else w.double())
    y, mag = turn(n, c, s, R, interleaved)
    return y, mag * (D + 16) * E + HALF[x.dtype] * y.abs()


def backward(dy, x, w, c, s, R, eps, interleaved):
    xd, D = x.double(), x.shape[-1]
    r = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
    g, gm = turn(dy.double(), c, s, R, interleaved, back=True)
    xh, wd = xd * r, (1 if w is None else w.double())
    m = (g * wd * xh).mean(-1, keepdim=True)
    dx = r * (g * wd - xh * m)
    mags = r * ((gm * wd).abs() + xh.abs() * (gm * wd * xh).abs().mean(-1, keepdim=True))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    dw = (g * xh).sum((0, 1, 2))
    return dx, mags * (2 * D + 16) * E + HALF[x.dtype] * dx.abs(), dw, (gm * xh.abs()).sum((0, 1, 2)) * (rows + D + 16) * E


CASES = [  # B, S, H, Hk, D, R, interleaved
    (2, 37, 4, 2, 128, 128, False), (1, 1, 8, 2, 128, 128, False), (3, 130, 5, 1, 64, 64, True), (2, 65, 3, 3, 128, 64, False),
    (1, 200, 16, 4, 256, 256, False), (2, 33, 4, 4, 256, 128, True), (1, 77, 12, 4, 80, 32, True), (1, 77, 12, 4, 80, 32, False),
    (2, 19, 3, 1, 96, 38, False), (2, 19, 3, 1, 96, 38, True), (1, 9, 2, 1, 192, 76, False), (2, 5, 1, 1, 2, 2, False),
    (1, 11, 3, 2, 66, 50, False), (1, 700, 9, 2, 32, 16, False), (64, 1, 10, 5, 192, 192, False), (1, 40, 2, 2, 16, 16, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hk,D,R,interleaved", CASES)
def test_forward_and_gradients(cuda_device, B, S, H, Hk, D, R, interleaved, dtype):
    from kernelcodegen_b200 import ops

    q, k = make((B, H, S, D), 1, dtype), make((B, Hk, S, D), 2, dtype)
    wq, wk = make((D,), 3, dtype), make((D,), 4, dtype)
    cos, sin = tables(S + 50, R)
    positions = torch.randint(0, S + 50, (B, S), generator=torch.Generator().manual_seed(5)).int().cuda()
    kw = dict(q_weight=wq, k_weight=wk, positions=positions, eps=1e-5, interleaved=interleaved)
    c, s = angles(cos, sin, positions, B, S)
    yq, yk = ops.qk_norm_rope(q, k, cos, sin, **kw)
    for name, got, x, w in (("q", yq, q, wq), ("k", yk, k, wk)):
        check(got, *forward(x, w, c, s, R, 1e-5, interleaved), name)
    dyq, dyk = make((B, H, S, D), 6, dtype), make((B, Hk, S, D), 7, dtype)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, **kw)
    assert dwq.dtype == dwk.dtype == torch.float32
    for name, got, gw, dy, x, w in (("q", dq, dwq, dyq, q, wq), ("k", dk, dwk, dyk, k, wk)):
        dx, bound, dw, wbound = backward(dy, x, w, c, s, R, 1e-5, interleaved)
        check(got, dx, bound, "d" + name)
        check(gw, dw, wbound, f"d{name}_weight")
    assert ops.last_device_status() == 0


@pytest.mark.parametrize("positions", ["none", "row64", "all64", "one"])
def test_positions_and_weights(cuda_device, positions):
    """No positions, int64 ones, one row for all sequences, one position for all tokens; no weights, or
    32-bit ones beside bf16 rows; queries alone."""
    from kernelcodegen_b200 import ops

    B, S, H, D, R = 2, 50, 4, 64, 64
    q = make((B, H, S, D), 1, torch.bfloat16)
    cos, sin = tables(90, R)
    at = {"none": None, "row64": torch.arange(7, 7 + S).cuda(), "all64": (torch.arange(B * S).view(B, S) % 90).cuda(),
          "one": torch.tensor([3], device="cuda").expand(B, S)}[positions]
    c, s = angles(cos, sin, at, B, S)
    for w in (None, make((D,), 3, torch.float32)):
        y, none = ops.qk_norm_rope(q, None, cos, sin, q_weight=w, positions=at)
        assert none is None
        check(y, *forward(q, w, c, s, R, 1e-6, False), "q")
        dy = make(q.shape, 9, torch.bfloat16)
        dq, dk, dw, dkw = ops.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w, positions=at)
        assert dk is None and dkw is None and (dw is None) == (w is None)
        dx, bound, dwant, wbound = backward(dy, q, w, c, s, R, 1e-6, False)
        check(dq, dx, bound, "dq")
        if w is not None:
            check(dw, dwant, wbound, "dw")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,R", [(128, 128), (96, 38), (50, 50)])
def test_views_in_place_and_into_a_cache(cuda_device, dtype, D, R):
    from kernelcodegen_b200 import ops

    B, S, H, Hk = 2, 21, 6, 2
    x = make((B, S, H + 2 * Hk, D), 1, dtype)
    q, k, v = (t.transpose(1, 2) for t in x.split([H, Hk, Hk], dim=2))
    cos, sin = tables(64, R)
    want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), cos, sin)
    cache = torch.full((B, Hk, 40, D), 7.0, device="cuda", dtype=dtype)
    got = ops.qk_norm_rope(q, k, cos, sin, k_out=cache[:, :, 5:5 + S])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert (cache[:, :, :5] == 7).all() and (cache[:, :, 5 + S:] == 7).all()
    dyq, dyk = make(q.shape, 2, dtype), make(k.shape, 3, dtype)
    grads = ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin)
    dx = torch.full_like(x, 7.0)
    dq, dk, dv = (t.transpose(1, 2) for t in dx.split([H, Hk, Hk], dim=2))
    ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, dq=dq, dk=dk)
    assert torch.equal(dq, grads[0]) and torch.equal(dk, grads[1]) and (dv == 7).all()
    again = [dyq.clone(), dyk.clone()]
    ops.qk_norm_rope_backward(*again, q, k, cos, sin, dq=again[0], dk=again[1])
    assert torch.equal(again[0], grads[0]) and torch.equal(again[1], grads[1])
    vv = v.clone()
    ops.qk_norm_rope(q, k, cos, sin, q_out=q, k_out=k)       # over the projection itself
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, vv)
    assert ops.last_device_status() == 0


def test_gradients_against_differences(cuda_device):
    from kernelcodegen_b200 import ops

    B, S, H, Hk, D, R = 2, 9, 3, 1, 24, 16
    q, k = make((B, H, S, D), 1, torch.float32), make((B, Hk, S, D), 2, torch.float32)
    wq, wk = make((D,), 3, torch.float32), make((D,), 4, torch.float32)
    cos, sin = tables(S, R)
    dyq, dyk = make(q.shape, 5, torch.float32), make(k.shape, 6, torch.float32)
    c, s = angles(cos, sin, None, B, S)
    for interleaved in (False, True):
        grads = ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, q_weight=wq, k_weight=wk, interleaved=interleaved)

        def value(q, k, wq, wk):
            total = 0
            for x, w, dy in ((q, wq, dyq), (k, wk, dyk)):
                n = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
                total = total + (turn(n, c, s, R, interleaved)[0] * dy.double()).sum()
            return total

        xs = [t.double() for t in (q, k, wq, wk)]
        for i, g in enumerate(grads):
            step = make(g.shape, 20 + i, torch.float32).double()
            hi, lo = ([x + (sign * 1e-5 * step if j == i else 0) for j, x in enumerate(xs)] for sign in (1, -1))
            want = (value(*hi) - value(*lo)) / 2e-5
            # 32-bit entries, each off by some hundred e; the difference quotient by about 1e-10 of the values
            assert abs((g.double() * step).sum() - want) <= 1e-4 * (g.double() * step).abs().sum(), i


def test_rows_of_zeros_and_extremes(cuda_device):
    from kernelcodegen_b200 import ops

    cos, sin = tables(8, 64)
    q = make((1, 2, 8, 64), 1, torch.float32)
    q[0, 0, 1] = 0
    q[0, 0, 2] *= 1e-15
    q[0, 0, 3] *= 1e15
    c, s = angles(cos, sin, None, 1, 8)
    y, _ = ops.qk_norm_rope(q, None, cos, sin)
    check(y, *forward(q, None, c, s, 64, 1e-6, False), "q")
    dy = make(q.shape, 2, torch.float32)
    dq = ops.qk_norm_rope_backward(dy, None, q, None, cos, sin)[0]
    dx, bound, _, _ = backward(dy, q, None, c, s, 64, 1e-6, False)
    check(dq, dx, bound, "dq")


def test_out_of_memory_is_torch_s_error(cuda_device):
    """An output of 512 GB cannot be had: the caller sees what any allocation would raise."""
    from kernelcodegen_b200 import ops

    q = torch.ones((1, 1, 1, 256), device="cuda", dtype=torch.bfloat16).expand(1, 1024, 2 ** 20, 256)
    cos, sin = tables(4, 256)
    with pytest.raises(torch.OutOfMemoryError):
        ops.qk_norm_rope(q, None, cos, sin, positions=torch.zeros((1,), device="cuda", dtype=torch.int32).expand(2 ** 20))


def test_eps_of_zero(cuda_device):
    """No row is zero, so nothing is infinite: rows that a group of lanes has nothing to do for included."""
    from kernelcodegen_b200 import ops

    for S, H, D, R, dtype in ((5, 3, 64, 64, torch.bfloat16), (5, 3, 64, 64, torch.float32), (5, 3, 66, 50, torch.bfloat16), (13001, 3, 64, 64, torch.bfloat16)):
        q, w = make((1, H, S, D), 1, dtype), make((D,), 2, dtype)
        cos, sin = tables(S, R)
        c, s = angles(cos, sin, None, 1, S)
        y, _ = ops.qk_norm_rope(q, None, cos, sin, q_weight=w, eps=0.0)
        check(y, *forward(q, w, c, s, R, 0.0, False), "q")
        dy = make(q.shape, 3, dtype)
        dq, _, dw, _ = ops.qk_norm_rope_backward(dy, None, q, None, cos, sin, q_weight=w, eps=0.0)
        dx, bound, dwant, wbound = backward(dy, q, w, c, s, R, 0.0, False)
        check(dq, dx, bound, "dq")
        check(dw, dwant, wbound, "dw")


def test_rows_further_apart_than_32_bits(cuda_device):
    from kernelcodegen_b200 import ops

    S, H, D = 70, 3, 64
    room = torch.empty(2 ** 31 + 4 * H * S * D, device="cuda", dtype=torch.bfloat16)
    q, y, dy, dq = (room.as_strided((2, H, S, D), (2 ** 31, D, H * D, 1), i * H * S * D) for i in range(4))
    q.copy_(make((2, H, S, D), 1, torch.bfloat16))
    dy.copy_(make((2, H, S, D), 2, torch.bfloat16))
    cos, sin = tables(S, D)
    ops.qk_norm_rope(q, None, cos, sin, q_out=y)
    assert torch.equal(y, ops.qk_norm_rope(q.contiguous(), None, cos, sin)[0])
    ops.qk_norm_rope_backward(dy, None, q, None, cos, sin, dq=dq)
    assert torch.equal(dq, ops.qk_norm_rope_backward(dy.contiguous(), None, q.contiguous(), None, cos, sin)[0])


@pytest.mark.parametrize("D,R", [(64, 32), (64, 18)])
def test_a_position_outside_the_tables_is_reported(cuda_device, D, R):
    """Its rotated entries are NaN, the others and the other rows are what they should be."""
    from kernelcodegen_b200 import ops

    cos, sin = tables(10, R)
    q = make((1, 3, 4, D), 1, torch.float32)
    good = torch.tensor([0, 3, 9, 2], dtype=torch.int32, device="cuda")
    for outside in (-1, 10, 2 ** 31 - 1, -2 ** 31):
        bad = good.clone()
        bad[1] = outside
        want, _ = ops.qk_norm_rope(q, None, cos, sin, positions=good)
        assert ops.last_device_status() == 0
        got, _ = ops.qk_norm_rope(q, None, cos, sin, positions=bad)
        assert ops.last_device_status() == 11 and ops.last_device_status() == 0
        assert got[:, :, 1, :R].isnan().all() and torch.equal(got[:, :, 1, R:], want[:, :, 1, R:])
        keep = [0, 2, 3]
        assert torch.equal(got[:, :, keep], want[:, :, keep])


def test_streams_and_graphs(cuda_device):
    from kernelcodegen_b200 import ops

    q, k = make((2, 8, 300, 128), 1, torch.bfloat16), make((2, 2, 300, 128), 2, torch.bfloat16)
    w = make((128,), 3, torch.bfloat16)
    cos, sin = tables(300, 128)
    dyq, dyk = make(q.shape, 4, torch.bfloat16), make(k.shape, 5, torch.bfloat16)

    def step():
        return (*ops.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w),
                *ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, q_weight=w, k_weight=w))

    first = step()
    torch.cuda.synchronize()
    results = []
    for s in [torch.cuda.Stream(), torch.cuda.Stream()] * 3:
        with torch.cuda.stream(s):
            results.append(step())
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        captured = step()
    g.replay()
    torch.cuda.synchronize()
    for r in (*results, captured):
        for a, b in zip(first, r):
            assert torch.equal(a, b)


def test_empty(cuda_device):
    from kernelcodegen_b200 import ops

    cos, sin = tables(4, 64)
    q = torch.empty((0, 2, 3, 64), device="cuda")
    w = torch.ones(64, device="cuda")
    y, _ = ops.qk_norm_rope(q, None, cos, sin, q_weight=w)
    assert y.shape == q.shape
    dq, _, dw, _ = ops.qk_norm_rope_backward(q, None, q, None, cos, sin, q_weight=w)
    assert dq.shape == q.shape and (dw == 0).all()


def test_refusals(cuda_device):
    from kernelcodegen_b200 import capi, ops

    cos, sin = tables(8, 64)
    q = make((1, 2, 8, 64), 1, torch.float32)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q.half(), None, cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(make((1, 2, 9, 64), 1, torch.float32), None, cos, sin)     # more tokens than table rows
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q[..., :32], None, cos, sin)                                 # R > D
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, None, cos, sin, q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q, None, cos, sin, positions=torch.zeros(8, device="cuda"))
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q, None, cos.double(), sin.double())
    with pytest.raises(capi.KcgError) as e:
        ops.qk_norm_rope(make((1, 2, 8, 320), 1, torch.float32), None, cos, sin)
    assert e.value.status == capi.KCG_BAD_SHAPE
    with pytest.raises(capi.KcgError) as e:
        ops.qk_norm_rope(q, None, cos, sin, eps=-1.0)
    assert e.value.status == capi.KCG_BAD_ARGUMENT
    with pytest.raises(capi.KcgError) as e:
        ops.qk_norm_rope(q, None, cos, sin, q_out=q[:, :1].expand(1, 2, 8, 64))
    assert e.value.status == capi.KCG_BAD_SHAPE
