"""`ops.qk_norm_rope` and its gradients where a group of lanes takes many runs of heads, one after another: tokens
and heads beyond what the SMs hold at once, queries and keys in the same group, a last run that is shorter.

The formulas in 64 bits and the bounds are those of test_qk_norm_rope_gpu.py."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_qk_norm_rope_gpu import angles, backward, check, forward, make, tables

pytestmark = pytest.mark.gpu

# B, S, H, Hk, D, R.  By the rules of launch_rope on 148 SMs every group of lanes gets 1.3 to 48 runs, and the runs of
# 2, 4 or 8 query heads that it chooses leave a shorter one at the end.
VECTORS = [(2, 9000, 11, 3, 128, 128), (1, 20011, 5, 1, 64, 32), (3, 4001, 13, 7, 256, 256), (1, 6007, 9, 9, 80, 64)]
PAIRS = [(3, 14003, 11, 3, 66, 50), (2, 4003, 13, 1, 130, 130), (4, 9001, 9, 5, 34, 10)]
CASES = [(*c, il) for c in VECTORS + PAIRS for il in (False, True)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hk,D,R,interleaved", CASES)
def test_many_runs_forward_and_gradients(cuda_device, B, S, H, Hk, D, R, interleaved, dtype):
    from kernelcodegen_b200 import ops

    q, k = make((B, H, S, D), 1, dtype), make((B, Hk, S, D), 2, dtype)
    wq, wk = make((D,), 3, dtype), make((D,), 4, dtype)
    cos, sin = tables(S + 50, R)
    positions = torch.randint(0, S + 50, (B, S), generator=torch.Generator().manual_seed(5)).cuda()
    kw = dict(q_weight=wq, k_weight=wk, positions=positions, eps=1e-5, interleaved=interleaved)
    c, s = angles(cos, sin, positions, B, S)
    yq, yk = ops.qk_norm_rope(q, k, cos, sin, **kw)
    for name, got, x, w in (("q", yq, q, wq), ("k", yk, k, wk)):
        check(got, *forward(x, w, c, s, R, 1e-5, interleaved), name)
    dyq, dyk = make((B, H, S, D), 6, dtype), make((B, Hk, S, D), 7, dtype)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, **kw)
    for name, got, gw, dy, x, w in (("q", dq, dwq, dyq, q, wq), ("k", dk, dwk, dyk, k, wk)):
        dx, bound, dw, wbound = backward(dy, x, w, c, s, R, 1e-5, interleaved)
        check(got, dx, bound, "d" + name)
        check(gw, dw, wbound, f"d{name}_weight")
    # the same bits in place
    a, b, da, db = q.clone(), k.clone(), dyq.clone(), dyk.clone()
    ops.qk_norm_rope(a, b, cos, sin, q_out=a, k_out=b, **kw)
    assert torch.equal(a, yq) and torch.equal(b, yk)
    again = ops.qk_norm_rope_backward(da, db, q, k, cos, sin, dq=da, dk=db, **kw)
    for x, y in zip(again, (dq, dk, dwq, dwk)):
        assert torch.equal(x, y)
    assert ops.last_device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_runs_out_of_a_packed_projection_and_into_one(cuda_device, dtype):
    from kernelcodegen_b200 import ops

    B, S, H, Hk, D = 2, 7001, 11, 3, 64
    for R in (64, 38):
        x = make((B, S, H + 2 * Hk, D), 1, dtype)
        q, k, _ = (t.transpose(1, 2) for t in x.split([H, Hk, Hk], dim=2))
        cos, sin = tables(S, R)
        dyq, dyk = make((B, S, H, D), 2, dtype).transpose(1, 2), make((B, Hk, S, D), 3, dtype)
        dx = torch.full((B, S + 1, H + 2 * Hk, D), 7.0, device="cuda", dtype=dtype)
        dq, dk, dv = (t.transpose(1, 2) for t in dx[:, :S].split([H, Hk, Hk], dim=2))
        ops.qk_norm_rope_backward(dyq, dyk, q, k, cos, sin, dq=dq, dk=dk)
        want = ops.qk_norm_rope_backward(dyq.contiguous(), dyk, q.contiguous(), k.contiguous(), cos, sin)
        assert torch.equal(dq, want[0]) and torch.equal(dk, want[1])
        assert (dv == 7).all() and (dx[:, S] == 7).all()


def test_many_runs_stay_inside_their_buffers(cuda_device):
    """The same under the bounds-checking build, where an access outside its buffer is skipped and sets the
    status word that the tests read."""
    from kernelcodegen_b200 import build

    build.build_bounds()
    here = Path(__file__).resolve()
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-k", "forward_and or packed", str(here)],
                         env=dict(os.environ, KCG_DEBUG_BOUNDS="1"), capture_output=True, text=True, timeout=600, cwd=here.parents[1])
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-1000:]
