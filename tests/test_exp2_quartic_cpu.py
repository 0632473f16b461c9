"""The quartic that the attention training kernels use for a share of their exponentials (ex2_quartic2 in
kernelcodegen_b200/csrc/ptx.cuh), restated in numpy float32: the error bound its comment states."""
import re
from pathlib import Path

import numpy as np

PTX = Path(__file__).resolve().parents[1] / "kernelcodegen_b200" / "csrc" / "ptx.cuh"


def coefficients():
    text = PTX.read_text()
    body = text[text.index("float2 ex2_quartic2(float2 x)"):]
    c = [np.float32(v) for v in re.findall(r"make_float2\((0\.\d+)f,", body[:body.index("return r;")])]
    assert len(c) == 5
    return c


def ex2_quartic(x):
    c = coefficients()
    x = np.asarray(x, dtype=np.float32)
    magic = np.float32(12582912.0)
    t = (x + magic).astype(np.float32)
    f = (x - (t - magic)).astype(np.float32)
    p = (f * c[0] + c[1]).astype(np.float32)
    for k in c[2:]:
        p = (p * f + k).astype(np.float32)
    return (p.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(np.float32)


def test_relative_error():
    f = np.linspace(-0.5, 0.5, 200001)
    assert np.abs(np.polyval([float(v) for v in coefficients()], f) / np.exp2(f) - 1.0).max() < 2.7e-6
    x = np.linspace(-125.0, 8.0, 400001, dtype=np.float32)
    assert np.abs(ex2_quartic(x).astype(np.float64) / np.exp2(x.astype(np.float64)) - 1.0).max() < 2.7e-6 + 4 * 2.0 ** -24


def test_clamped_argument_gives_a_tiny_normal_number():
    got = ex2_quartic(np.array([-125.0], dtype=np.float32))[0]
    assert 0.0 < got < 1e-37
