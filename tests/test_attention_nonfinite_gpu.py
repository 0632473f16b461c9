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


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_gradients_of_a_bad_score(cuda_device, D, bad):
    """A query whose scores are NaN, or overflow, gets a NaN gradient and gives one to every key that it sees,
    even if its own dout is zero (0 * NaN is NaN in every step of the formula)."""
    from kernelcodegen_b200 import ops

    S = 200
    for row in (*range(0, 34, 3), 63, 64, 100, 127, 128, 199):
        q, k, v, dout = (make((1, 2, S, D), s) for s in (1, 2, 3, 4))
        if bad == "nan":
            q[0, 1, row, 5] = math.nan
        else:
            q[..., 0], k[..., 0] = 0, 1e20
            q[0, 1, row, 0] = 1e25
        dout[0, 1, row] = 0
        out, lse = ops.fmha_with_lse(q, k, v, scale=0.1, causal=True)
        assert lse[0, 1, row].isnan()
        dq, dk, dv = ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1, causal=True)
        assert dq[0, 1, row].isnan().all(), row
        assert dk[0, 1, :row + 1].isnan().all() and dv[0, 1, :row + 1].isnan().all(), row
        for t in (dq, dk, dv):
            assert torch.isfinite(t[0, 0]).all()
    assert ops.last_device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_of_a_bad_score_with_few_keys(cuda_device, D):
    """One and two keys: all of a query's probabilities come from the same kind of instruction."""
    from kernelcodegen_b200 import ops

    for Skv in (1, 2, 3, 5):
        q, dout = make((1, 1, 3, D), 1), make((1, 1, 3, D), 4)
        k, v = make((1, 1, Skv, D), 2), make((1, 1, Skv, D), 3)
        q[0, 0, 1, 5] = math.nan
        dout[0, 0, 1] = 0
        out, lse = ops.fmha_with_lse(q, k, v, scale=0.1)
        dq, dk, dv = ops.fmha_backward(dout, q, k, v, out, lse, scale=0.1)
        assert dq[0, 0, 1].isnan().all() and dk.isnan().all() and dv.isnan().all()
        assert torch.isfinite(dq[0, 0, [0, 2]]).all()
