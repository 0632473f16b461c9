"""Outputs that overlap an input or another output are refused before anything is launched: equal pointers, views
shifted against one another, heads of one packed buffer that share some.  (Views side by side in one buffer are
used by the GPU tests.)  The pointers are never dereferenced."""
import ctypes

import pytest

from kernelcodegen_b200 import capi

AT, FAR = 0x10000, 1 << 32
B, H, HKV, S, D = 2, 4, 2, 64, 64
SIZE = 2                                  # bytes of bf16
ROW, HEAD = D * SIZE, S * D * SIZE        # of a contiguous tensor


def strides(heads):
    return (ctypes.c_int64 * 3)(heads * S * D, S * D, D)


def packed(total):
    return (ctypes.c_int64 * 3)(S * total * D, D, total * D)


def attn():
    d = capi.AttnDesc()
    d.B, d.H, d.Hkv, d.Sq, d.Skv, d.D, d.dtype, d.scale = B, H, HKV, S, S, D, capi.KCG_BF16, 1.0
    for name in ("q", "o", "d_o", "d_q"):
        setattr(d, name, strides(H))
    for name in ("k", "v", "d_k", "d_v"):
        setattr(d, name, strides(HKV))
    return d


def apart(n):
    return [AT + i * FAR for i in range(n)]


def forward(lib, d, ptrs):
    return lib.kcg_fmha_fwd_lse_launch(ctypes.byref(d), *ptrs, None)


def backward(lib, d, ptrs):
    return lib.kcg_fmha_bwd_launch(ctypes.byref(d), *ptrs, AT + 20 * FAR, 1 << 30, None)


SHIFTS = [0, ROW, HEAD, (H - 1) * HEAD, -ROW, -HEAD]


@pytest.mark.parametrize("shift", SHIFTS)
def test_forward_output_over_an_input(native_lib, shift):
    for i in range(3):
        ptrs = apart(5)
        ptrs[3] = ptrs[i] + min(shift, HEAD)
        assert forward(native_lib, attn(), ptrs) == capi.KCG_BAD_ARGUMENT


def test_forward_statistics_over_a_tensor(native_lib):
    for i in range(4):
        for shift in (0, 512, -512):      # lse is B * H * S * 4 = 2048 bytes
            ptrs = apart(5)
            ptrs[4] = ptrs[i] + shift
            assert forward(native_lib, attn(), ptrs) == capi.KCG_BAD_ARGUMENT


def test_forward_output_in_the_heads_of_a_packed_projection(native_lib):
    """Heads 0..3 are Q, 4..5 K, 6..7 V: an output that starts at any head from 0 to 7 meets one of them."""
    total = H + 2 * HKV
    for at in range(total):
        d = attn()
        for name in "qkvo":
            setattr(d, name, packed(total))
        assert forward(native_lib, d, [AT, AT + H * ROW, AT + (H + HKV) * ROW, AT + at * ROW, FAR]) == capi.KCG_BAD_ARGUMENT


@pytest.mark.parametrize("shift", SHIFTS)
def test_gradients_over_inputs_and_one_another(native_lib, shift):
    for out in (6, 7, 8):                 # dO, Q, K, V, O, lse, dQ, dK, dV
        for other in (0, 1, 2, 3, 4, 6, 7, 8):
            if out == other:
                continue
            ptrs = apart(9)
            ptrs[out] = ptrs[other] + max(-HEAD, min(shift, HEAD))
            assert backward(native_lib, attn(), ptrs) == capi.KCG_BAD_ARGUMENT, (out, other)
        ptrs = apart(9)
        ptrs[out] = ptrs[5]               # over lse
        assert backward(native_lib, attn(), ptrs) == capi.KCG_BAD_ARGUMENT


def test_gradients_that_share_heads_of_a_packed_gradient(native_lib):
    total = H + 2 * HKV
    for heads in ((0, H - 1, H + HKV), (0, H, H + 1), (2, 1, H + HKV), (0, H, H)):
        d = attn()
        for name in ("d_q", "d_k", "d_v"):
            setattr(d, name, packed(total))
        grads = [AT + 30 * FAR + h * ROW for h in heads]
        assert backward(native_lib, d, [*apart(6), *grads]) == capi.KCG_BAD_ARGUMENT, heads


def rope(dt=capi.KCG_BF16):
    d = capi.RopeDesc()
    d.B, d.S, d.H, d.Hk, d.D, d.R = B, S, H, HKV, D, D
    d.dtype, d.dtype_w, d.pos_bits, d.table_rows, d.eps = dt, capi.KCG_F32, 32, S, 1e-6
    for name in ("q", "q_out", "d_q"):
        setattr(d, name, strides(H))
    for name in ("k", "k_out", "d_k"):
        setattr(d, name, strides(HKV))
    return d


def rope_forward(lib, d, q, k, q_out, k_out):
    return lib.kcg_qk_norm_rope_launch(ctypes.byref(d), q, k, None, None, AT + 40 * FAR, AT + 41 * FAR, None, q_out, k_out, None)


def rope_backward(lib, d, dq_out, dk_out, q, k, dq, dk):
    return lib.kcg_qk_norm_rope_bwd_launch(ctypes.byref(d), dq_out, dk_out, q, k, None, None, AT + 40 * FAR, AT + 41 * FAR, None, dq, dk,
                                           None, None, None, 0, None)


def test_rotation_over_an_input_that_is_not_the_same_view(native_lib):
    q, k, qo, ko = apart(4)
    cases = [(q, k, k, ko), (q, k, qo, q), (q, k, qo, qo), (q, k, q + ROW, ko), (q, k, qo, k - ROW), (q, k, qo, q + HEAD), (q, k, q, q)]
    for case in cases:
        assert rope_forward(native_lib, rope(), *case) == capi.KCG_BAD_ARGUMENT, case
    d = rope()                            # over its own input, read with other strides
    d.q = (ctypes.c_int64 * 3)(H * S * D, D, H * D)
    assert rope_forward(native_lib, d, q, k, q, ko) == capi.KCG_BAD_ARGUMENT


def test_rotation_gradients_over_an_input_that_is_not_the_same_view(native_lib):
    dyq, dyk, q, k, dq, dk = apart(6)
    cases = [(dyk, dk), (k, dk), (dq, q), (dq, dyq), (dq, dq), (q + ROW, dk), (dyq - HEAD, dk), (dq, dyk + HEAD)]
    for case in cases:
        assert rope_backward(native_lib, rope(), dyq, dyk, q, k, *case) == capi.KCG_BAD_ARGUMENT, case
    d = rope()
    d.q_out = (ctypes.c_int64 * 3)(H * S * D, D, H * D)
    assert rope_backward(native_lib, d, dyq, dyk, q, k, dyq, dk) == capi.KCG_BAD_ARGUMENT


def test_views_overlap_against_their_bytes(tmp_path):
    """Random views: none is called overlapping that is not; heads and tokens of one buffer: every answer is right."""
    import shutil
    import subprocess
    from pathlib import Path

    exe = tmp_path / "overlap"
    source = Path(__file__).resolve().parent / "cpp" / "head_view_overlap.cc"
    subprocess.run([shutil.which("g++") or "g++", "-std=c++17", "-O2", str(source), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    (yes, no, _, wrong), (yes2, no2, untold2, wrong2) = (map(int, line.split()) for line in lines[:2])
    assert min(yes, no, yes2, no2) > 1000
    assert wrong == wrong2 == untold2 == 0
