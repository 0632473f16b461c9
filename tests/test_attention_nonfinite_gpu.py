"""Scores that overflow 32 bits or are NaN: every result that is made of one is NaN, none that is not.

The exponentials of a tile are shared between two instructions by column, so the bad score is put into every
column of a tile in turn."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def overflowing(H, S, D, big_q=1e25, big_k=1e20):
    """Head h: the score of every query with key h is past the largest 32-bit number; all entries are finite."""
    q, k, v = make((1, H, S, D), 1), make((1, H, S, D), 2), make((1, H, S, D), 3)
    q[..., 0], k[..., 0] = big_q, 0
    at = torch.arange(H)
    k[0, at, at, 0] = big_k
    return q, k, v


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_an_infinite_score_is_not_hidden(cuda_device, D, causal):
    from kernelcodegen_b200 import ops

    S = H = 200
    q, k, v = overflowing(H, S, D)
    out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=causal)
    sees = torch.ones((H, S), dtype=torch.bool, device="cuda")
    if causal:
        sees = torch.arange(S, device="cuda")[None, :] >= torch.arange(H, device="cuda")[:, None]
    assert lse[0][sees].isnan().all() and out[0][sees].isnan().all()
    assert torch.isfinite(lse[0][~sees]).all() and torch.isfinite(out[0][~sees]).all()
    assert ops.last_device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_a_score_that_overflows_when_scaled(cuda_device, D):
    """q.k fits 32 bits, scale q.k does not."""
    from kernelcodegen_b200 import ops

    q, k, v = overflowing(130, 130, D, big_q=1e19, big_k=1e19)
    out, lse = ops.fmha_with_lse(q, k, v, scale=10.0)
    assert lse.isnan().all() and out.isnan().all()


@pytest.mark.parametrize("D", [64, 128])
def test_infinite_scores_in_a_later_block(cuda_device, D):
    from kernelcodegen_b200 import ops

    q, k, v = (make((1, 2, 400, D), s) for s in (1, 2, 3))
    q[..., 0], k[..., 0] = 1e25, 0
    for at in (0, 127, 128, 300, 399):
        x = k.clone()
        x[0, 1, at, 0] = 1e20
        out, lse = ops.fmha_with_lse(q, x, v, scale=0.1)
        assert lse[0, 1].isnan().all() and out[0, 1].isnan().all()
        assert torch.isfinite(lse[0, 0]).all() and torch.isfinite(out[0, 0]).all()
