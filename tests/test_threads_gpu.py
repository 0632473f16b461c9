"""Calls from threads that have not used CUDA before, as autograd's workers are: the first call of a thread may be
one of this library's.  Every tensor exists already, so nothing else brings the thread to the device."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def calls():
    from kernelcodegen_b200 import ops

    q, k, dout = make((1, 4, 130, 64), 1), make((1, 2, 130, 64), 2), make((1, 4, 130, 64), 3)
    out, lse = ops.fmha_with_lse(q, k, k, scale=0.1, causal=True)
    angle = torch.rand((130, 32)).cuda()
    cos, sin = angle.cos(), angle.sin()
    into = [torch.empty_like(t) for t in (q, k, k)]
    yield "fmha_with_lse", lambda: ops.fmha_with_lse(q, k, k, scale=0.1, causal=True, out=into[0])
    yield "fmha_backward", lambda: ops.fmha_backward(dout, q, k, k, out, lse, scale=0.1, causal=True, dq=into[0], dk=into[1], dv=into[2])
    yield "qk_norm_rope", lambda: ops.qk_norm_rope(q, k, cos, sin, q_out=into[0], k_out=into[1])
    yield "qk_norm_rope_backward", lambda: ops.qk_norm_rope_backward(dout, k, q, k, cos, sin, dq=into[0], dk=into[1])
    h, h_out = make((1, 2, 130, 64), 4), torch.empty((1, 2, 130, 64), device="cuda", dtype=torch.bfloat16)
    yield "fmha", lambda: ops.fmha(h, h, h, out=h_out)
    a, c = make((256, 256), 5), torch.empty((256, 256), device="cuda", dtype=torch.bfloat16)
    yield "matmul", lambda: ops.matmul(a, a, out=c)


@pytest.mark.parametrize("which", range(6))
def test_first_call_of_a_thread(cuda_device, which):
    name, call = list(calls())[which]

    def results():
        got = call()
        return [t.clone() for t in (got if isinstance(got, tuple) else (got,)) if t is not None]

    want = results()
    torch.cuda.synchronize()
    got, errors = [], []

    def work():
        try:
            call()
            got.extend(results())
            torch.cuda.synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not errors, (name, errors)
    assert len(got) == len(want)
    for x, y in zip(got, want):
        assert torch.equal(x, y), name
