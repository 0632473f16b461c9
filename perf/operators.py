"""Cases of the attention training operators: attention with its row statistics, its gradients, and the
per-head norm and rotation of queries and keys that comes before it (forward and backward).

Every case is computed in plain torch operations in 32 bits, or by the framework's operators (`own`).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the forward pass of a training step on a packed qkv projection, shared K/V heads, odd length
        dict(name="fwd_packed_gqa_s1500_d128", op="fwd", B=2, H=32, Hkv=8, Sq=1500, Skv=1500, D=128, causal=True, packed=True),
        # the benchmark's attention shape (batch 4, 16 heads, 1024 tokens, head dimension 64), full attention
        dict(name="fwd_b4_h16_s1024_d64", op="fwd", B=4, H=16, Hkv=16, Sq=1024, Skv=1024, D=64, causal=False, packed=False),
        # gradients of one short sequence on few heads: launch latency counts
        dict(name="bwd_short_h4_s128_d64", op="bwd", B=1, H=4, Hkv=4, Sq=128, Skv=128, D=64, causal=True, packed=False),
        # the benchmark's attention shape again, its gradients
        dict(name="bwd_b4_h16_s1024_d64", op="bwd", B=4, H=16, Hkv=16, Sq=1024, Skv=1024, D=64, causal=False, packed=False),
        # an ordinary training step: packed projection, shared K/V heads, a length that ends inside a tile
        dict(name="bwd_packed_gqa_s1500_d128", op="bwd", B=2, H=32, Hkv=8, Sq=1500, Skv=1500, D=128, causal=True, packed=True),
        # cross attention: other lengths on the two sides, both ragged
        dict(name="bwd_cross_333x1777_d128", op="bwd", B=4, H=16, Hkv=16, Sq=333, Skv=1777, D=128, causal=False, packed=False),
        # a long sequence: the benchmark's causal shape, one sequence of it
        dict(name="bwd_h32_s8192_d128", op="bwd", B=1, H=32, Hkv=32, Sq=8192, Skv=8192, D=128, causal=True, packed=False),
        # serving: one new token for each of 32 sequences, each at a position of its own
        dict(name="rope_decode_b32", op="rope", B=32, S=1, H=32, Hkv=8, D=128, R=128, dtype="bf16", interleaved=False, packed=True, table=8192),
        # a training step's queries and keys out of the packed projection
        dict(name="rope_packed_b4_s4096", op="rope", B=4, S=4096, H=32, Hkv=8, D=128, R=128, dtype="bf16", interleaved=False, packed=True, table=4096),
        # 32-bit, an odd length, a head dimension that is no power of two, part of it rotated, neighbouring pairs
        dict(name="rope_f32_d80_r32_s777", op="rope", B=3, S=777, H=12, Hkv=4, D=80, R=32, dtype="f32", interleaved=True, packed=False, table=2048),
        # the gradients of the training step's queries, keys and norm weights
        dict(name="rope_bwd_packed_b4_s4096", op="rope_bwd", B=4, S=4096, H=32, Hkv=8, D=128, R=128, dtype="bf16", interleaved=False, packed=True, table=4096),
        # a small 32-bit one
        dict(name="rope_bwd_f32_d64_s333", op="rope_bwd", B=2, S=333, H=16, Hkv=4, D=64, R=64, dtype="f32", interleaved=False, packed=False, table=512),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["fwd", "bwd", "bwd", "rope", "rope_bwd"])
    if op in ("fwd", "bwd"):
        D = rng.choice([64, 128])
        Hkv = rng.choice([1, 2, 3, 4, 8, 16])
        H = Hkv * rng.choice([1, 1, 2, 4, 7])
        causal = rng.random() < 0.6
        packed = rng.random() < 0.5
        # with one key the probabilities are one whatever the scores: the gradients of q and k are zero but for rounding
        low = 1 if op == "fwd" else 2
        Sq = _spread(rng, low, 6000)
        Skv = Sq if packed or rng.random() < 0.5 else _spread(rng, low, 6000)
        B = _spread(rng, 1, 8)
        over = lambda: B * H * Sq * Skv > 32 * 8192 * 8192 // 2 or B * (H + Hkv) * (Sq + Skv) > 2 * 32 * 2 * 8192  # noqa: E731
        while over() and B > 1:
            B -= 1
        while over():
            Sq, Skv = (Sq + 1) // 2, (Skv + 1) // 2
        return dict(op=op, B=B, H=H, Hkv=Hkv, Sq=Sq, Skv=Skv, D=D, causal=causal, packed=packed)
    D = rng.choice([64, 80, 96, 128, 128, 192, 256])
    R = rng.choice([D, D, D // 2, 2 * (D // 5)])
    Hkv = rng.choice([1, 2, 4, 5, 8])
    H = Hkv * rng.choice([1, 2, 4, 8])
    S = 1 if rng.random() < 0.2 else _spread(rng, 2, 8192)
    B = _spread(rng, 1, 64)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    while B * S * (H + Hkv) * D * (4 if dtype == "f32" else 2) > 4 * 4096 * 40 * 128 * 2 and B > 1:
        B -= 1
    while B * S * (H + Hkv) * D * (4 if dtype == "f32" else 2) > 4 * 4096 * 40 * 128 * 2:
        S = (S + 1) // 2
    return dict(op=op, B=B, S=S, H=H, Hkv=Hkv, D=D, R=R, dtype=dtype, interleaved=rng.random() < 0.4,
                packed=rng.random() < 0.5, table=S + _spread(rng, 1, 4096))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _heads(gen, B, H, S, D, dtype, packed, extra=()):
    """[B, H, S, D] tensors of H and of each of `extra` heads: views of one packed projection, or each on its own."""
    counts = [H, *extra]
    if packed:
        width = sum(counts) * D
        whole = _randn(gen, B, S, width).to(dtype).view(B, S, sum(counts), D)
        return list(t.transpose(1, 2) for t in whole.split(counts, dim=2))
    return [_randn(gen, B, n, S, D).to(dtype) for n in counts]


def prepare(case, seed):
    gen = _gen(seed)
    if case["op"] in ("fwd", "bwd"):
        B, H, Hkv, Sq, Skv, D = (case[n] for n in ("B", "H", "Hkv", "Sq", "Skv", "D"))
        if case["packed"]:
            q, k, v = _heads(gen, B, H, Sq, D, torch.bfloat16, True, (Hkv, Hkv))
        else:
            q, = _heads(gen, B, H, Sq, D, torch.bfloat16, False)
            k, v = _heads(gen, B, Hkv, Skv, D, torch.bfloat16, False, (Hkv,))
        state = dict(case=case, q=q, k=k, v=v, scale=D ** -0.5)
        if case["op"] == "bwd":
            # what the forward pass left, and the gradient that comes back through the next layer
            out, lse = _attention(q, k, v, state["scale"], case["causal"])
            state |= dict(out=out, lse=lse, dout=_randn(gen, B, H, Sq, D).to(torch.bfloat16))
        return state
    B, S, H, Hkv, D, R = (case[n] for n in ("B", "S", "H", "Hkv", "D", "R"))
    dtype = DTYPES[case["dtype"]]
    # a packed projection holds the values too, which this pass leaves alone
    q, k = _heads(gen, B, H, S, D, dtype, case["packed"], (Hkv, Hkv) if case["packed"] else (Hkv,))[:2]
    weights = [(1 + 0.2 * _randn(gen, D)).to(dtype) for _ in range(2)]
    angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    first = torch.randint(0, case["table"] - S + 1, (B, 1), generator=gen, device="cuda", dtype=torch.int32)
    state = dict(case=case, q=q, k=k, q_weight=weights[0], k_weight=weights[1], cos=angle.cos().float(), sin=angle.sin().float(),
                 positions=first + torch.arange(S, device="cuda", dtype=torch.int32), eps=1e-6)
    if case["op"] == "rope_bwd":
        state |= dict(dq=_randn(gen, B, H, S, D).to(dtype), dk=_randn(gen, B, Hkv, S, D).to(dtype))
    return state


def _hidden(Sq, Skv, device):
    """[Sq, Skv], true where the causal mask hides the key; the last query sees every key."""
    return torch.arange(Skv, device=device)[None, :] > torch.arange(Sq, device=device)[:, None] + (Skv - Sq)


def _scores(q, k, scale, causal):
    """[B, Hkv, H / Hkv, Sq, Skv] in 32 bits, -inf where hidden."""
    B, H, Sq, D = q.shape
    Hkv, Skv = k.shape[1:3]
    s = (q.float().reshape(B, Hkv, -1, D) @ k.float().transpose(2, 3)).view(B, Hkv, H // Hkv, Sq, Skv).mul_(scale)
    return s.masked_fill_(_hidden(Sq, Skv, q.device), -math.inf) if causal else s


def _attention(q, k, v, scale, causal):
    B, H, Sq, D = q.shape
    Hkv, Skv = k.shape[1:3]
    s = _scores(q, k, scale, causal)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, Hkv, -1, Skv) @ v.float()).view(total.shape[:-1] + (D,)) / torch.where(total == 0, torch.ones_like(total), total)
    return out.view(B, H, Sq, D).to(q.dtype), (total.log() + top).view(B, H, Sq)


def _attention_backward(dout, q, k, v, out, lse, scale, causal):
    B, H, Sq, D = q.shape
    Hkv, Skv = k.shape[1:3]
    g = H // Hkv
    at = lse.view(B, Hkv, g, Sq, 1)
    p = _scores(q, k, scale, causal).sub_(torch.where(at == -math.inf, torch.zeros_like(at), at)).exp_()
    do = dout.float().reshape(B, Hkv, g * Sq, D)
    delta = (dout.float() * out.float()).sum(-1).view(B, Hkv, g, Sq, 1)
    dv = p.view(B, Hkv, g * Sq, Skv).transpose(2, 3) @ do
    ds = (do @ v.float().transpose(2, 3)).view(B, Hkv, g, Sq, Skv).sub_(delta).mul_(p).view(B, Hkv, g * Sq, Skv)
    dq = (ds @ k.float()).mul_(scale).view(B, H, Sq, D)
    dk = (ds.transpose(2, 3) @ q.float().reshape(B, Hkv, g * Sq, D)).mul_(scale)
    return dq.to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


def _pairs(x, R, interleaved):
    """The two members of each rotated pair, and the rest."""
    rot, rest = x[..., :R], x[..., R:]
    return (rot[..., 0::2], rot[..., 1::2], rest) if interleaved else (rot[..., :R // 2], rot[..., R // 2:], rest)


def _join(a, b, rest, interleaved):
    rot = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((rot, rest), -1)


def _norm_rope(x, w, c, s, R, eps, interleaved):
    x = x.float()
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()
    a, b, rest = _pairs(n, R, interleaved)
    return _join(a * c - b * s, b * c + a * s, rest, interleaved)


def _norm_rope_backward(dy, x, w, c, s, R, eps, interleaved):
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    a, b, rest = _pairs(dy.float(), R, interleaved)
    g = _join(a * c + b * s, b * c - a * s, rest, interleaved)
    xh = x * r
    gw = g * w.float()
    return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (g * xh).sum((0, 1, 2))


def run(state):
    case = state["case"]
    if case["op"] == "fwd":
        args = (state["q"], state["k"], state["v"])
        if own:
            from kernelcodegen_b200 import ops
            return ops.fmha_with_lse(*args, scale=state["scale"], causal=case["causal"])
        return _attention(*args, state["scale"], case["causal"])
    if case["op"] == "bwd":
        args = tuple(state[n] for n in ("dout", "q", "k", "v", "out", "lse"))
        if own:
            from kernelcodegen_b200 import ops
            return ops.fmha_backward(*args, scale=state["scale"], causal=case["causal"])
        return _attention_backward(*args, state["scale"], case["causal"])
    R, style = case["R"], case["interleaved"]
    if own:
        from kernelcodegen_b200 import ops
        kw = dict(q_weight=state["q_weight"], k_weight=state["k_weight"], positions=state["positions"], eps=state["eps"], interleaved=style)
        if case["op"] == "rope":
            return ops.qk_norm_rope(state["q"], state["k"], state["cos"], state["sin"], **kw)
        return ops.qk_norm_rope_backward(state["dq"], state["dk"], state["q"], state["k"], state["cos"], state["sin"], **kw)
    at = state["positions"].long()
    c, s = state["cos"][at][:, None], state["sin"][at][:, None]
    if case["op"] == "rope":
        return tuple(_norm_rope(state[n], state[n + "_weight"], c, s, R, state["eps"], style).to(state[n].dtype) for n in "qk")
    (dq, dqw), (dk, dkw) = (_norm_rope_backward(state["d" + n], state[n], state[n + "_weight"], c, s, R, state["eps"], style) for n in "qk")
    return dq.to(state["q"].dtype), dk.to(state["k"].dtype), dqw, dkw


def _visible(Sq, Skv, causal):
    """How many (query, key) pairs the mask leaves."""
    if not causal:
        return Sq * Skv
    first, last = Skv - Sq + 1, Skv      # keys of the first and of the last query
    low = max(first, 1)
    return (low + last) * (last - low + 1) // 2


def work(case):
    if case["op"] in ("fwd", "bwd"):
        B, H, Hkv, Sq, Skv, D = (case[n] for n in ("B", "H", "Hkv", "Sq", "Skv", "D"))
        q, kv, lse = B * H * Sq * D * 2, B * Hkv * Skv * D * 2, B * H * Sq * 4
        pairs = B * H * _visible(Sq, Skv, case["causal"])
        if case["op"] == "fwd":
            return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * D * pairs}
        return {"bytes": 4 * q + 4 * kv + lse, "flops": 10 * D * pairs}
    B, S, H, Hkv, D, R = (case[n] for n in ("B", "S", "H", "Hkv", "D", "R"))
    size = 4 if case["dtype"] == "f32" else 2
    x = B * S * (H + Hkv) * D
    # one row of each table for a position, and the position; the weights and their gradients
    small = min(B * S, case["table"]) * R * 4 + B * S * 4 + 2 * D * size
    if case["op"] == "rope":
        return {"bytes": 2 * x * size + small, "flops": 8 * x}
    return {"bytes": 3 * x * size + small + 2 * D * 4, "flops": 16 * x}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("fwd", "bwd"):
        return _exact_attention(state)
    D, R, eps = case["D"], case["R"], state["eps"]
    # the rotation as a matrix for each position: x -> M x, so that its gradient is M^T dy
    at = state["positions"].flatten().long()
    c, s = state["cos"][at].double(), state["sin"][at].double()
    idx = torch.arange(R // 2, device="cuda")
    i, j = (2 * idx, 2 * idx + 1) if case["interleaved"] else (idx, idx + R // 2)
    results, sums = [], []
    for n in "qk":
        x = state[n].double().transpose(1, 2).flatten(0, 1)           # [tokens, heads, D]
        w = state[n + "_weight"].double()
        r = (x.pow(2).sum(-1, keepdim=True) / D + eps).pow(-0.5)
        if case["op"] == "rope":
            y = x * r * w
            z = y.clone()
            z[..., i] = y[..., i] * c[:, None] - y[..., j] * s[:, None]
            z[..., j] = y[..., i] * s[:, None] + y[..., j] * c[:, None]
        else:
            y = state["d" + n].double().transpose(1, 2).flatten(0, 1)
            g = y.clone()
            g[..., i] = y[..., i] * c[:, None] + y[..., j] * s[:, None]
            g[..., j] = y[..., j] * c[:, None] - y[..., i] * s[:, None]
            sums.append((g * x * r).sum((0, 1)))
            # d/dx of x r w with r = (x.x / D + eps)^-1/2 : r w g - x r^3 (x . w g) / D
            z = r * w * g - x * r.pow(3) * (x * w * g).sum(-1, keepdim=True) / D
        results.append(z.unflatten(0, (case["B"], case["S"])).transpose(1, 2))
    return (*results, *sums)


def _exact_attention(state):
    case, scale = state["case"], state["scale"]
    q, k, v = state["q"], state["k"], state["v"]
    (B, H, Sq, D), (Hkv, Skv) = q.shape, k.shape[1:3]
    bwd = case["op"] == "bwd"
    like = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    first, lse = like(B, H, Sq, D), like(B, H, Sq)
    dk, dv = like(B, Hkv, Skv, D), like(B, Hkv, Skv, D)
    keep = ~_hidden(Sq, Skv, "cuda") if case["causal"] else None
    for b in range(B):
        for h in range(H):
            kh = h * Hkv // H
            qd, kd, vd = q[b, h].double(), k[b, kh].double(), v[b, kh].double()
            z = torch.einsum("id,jd->ij", qd, kd) * scale
            if keep is not None:
                z = torch.where(keep, z, torch.full_like(z, -math.inf))
            if not bwd:
                lse[b, h] = torch.logsumexp(z, -1)
                first[b, h] = torch.nan_to_num(torch.exp(z - lse[b, h][:, None])) @ vd
                continue
            at = state["lse"][b, h].double()[:, None]
            p = torch.where(z == -math.inf, torch.zeros_like(z), torch.exp(z - at))
            g, o = state["dout"][b, h].double(), state["out"][b, h].double()
            ds = p * (torch.einsum("id,jd->ij", g, vd) - (g * o).sum(-1, keepdim=True))
            first[b, h] = torch.einsum("ij,jd->id", ds, kd) * scale
            dk[b, kh] += torch.einsum("ij,id->jd", ds, qd) * scale
            dv[b, kh] += torch.einsum("ij,id->jd", p, g)
    return (first, dk, dv) if bwd else (first, lse)
