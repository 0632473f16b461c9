"""Child process of tests/test_attention_bounds_gpu.py: runs with KCG_DEBUG_BOUNDS=1, so that `capi.load()` picks
the bounds-checking build.  Caps the extents that the kernels check against, on buffers that are in fact large
enough: what lies beyond the cap is skipped and reported.  Prints one JSON line."""
import ctypes
import json
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from kernelcodegen_b200 import capi, ops  # noqa: E402


def make(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def strides(heads, S, D):
    return (ctypes.c_int64 * 3)(heads * S * D, S * D, D)


def nan(n):
    return torch.full((n,), math.nan, device="cuda")


class Attention:
    """Buffers of one call through the C entries, the workspace among them."""

    def __init__(self, lib, B, H, Hkv, Sq, Skv, D):
        self.lib, d = lib, capi.AttnDesc()
        d.B, d.H, d.Hkv, d.Sq, d.Skv, d.D, d.dtype, d.scale = B, H, Hkv, Sq, Skv, D, capi.KCG_BF16, 0.1
        for name in ("q", "o", "d_o", "d_q"):
            setattr(d, name, strides(H, Sq, D))
        for name in ("k", "v", "d_k", "d_v"):
            setattr(d, name, strides(Hkv, Skv, D))
        self.d = d
        self.q, self.dout = make((B, H, Sq, D), 1), make((B, H, Sq, D), 2)
        self.k, self.v = make((B, Hkv, Skv, D), 3), make((B, Hkv, Skv, D), 4)
        self.out, self.lse = torch.zeros_like(self.q), nan(B * H * Sq)
        self.grads = [torch.zeros_like(t) for t in (self.q, self.k, self.v)]
        self.ws = nan(lib.kcg_fmha_bwd_workspace_bytes(ctypes.byref(d)) // 4)

    def forward(self):
        st = self.lib.kcg_fmha_fwd_lse_launch(ctypes.byref(self.d), *(t.data_ptr() for t in (self.q, self.k, self.v, self.out, self.lse)),
                                              torch.cuda.current_stream().cuda_stream)
        return st, ops.last_device_status()

    def backward(self):
        st = self.lib.kcg_fmha_bwd_launch(ctypes.byref(self.d), *(t.data_ptr() for t in (self.dout, self.q, self.k, self.v, self.out, self.lse, *self.grads, self.ws)),
                                          self.ws.numel() * 4, torch.cuda.current_stream().cuda_stream)
        return st, ops.last_device_status()


def rotation(lib, S, D, R, w):
    """The weight gradient of one head of as many tokens as one CTA takes (64 in vectors of 4 lanes a row, 16 in
    pairs): one row of partial sums."""
    d = capi.RopeDesc()
    d.B, d.S, d.H, d.Hk, d.D, d.R = 1, S, 1, 0, D, R
    d.dtype, d.dtype_w, d.pos_bits, d.table_rows, d.eps = capi.KCG_BF16, capi.KCG_BF16, 32, S, 1e-6
    for name in ("q", "q_out", "d_q"):
        setattr(d, name, strides(1, S, D))
    q, dy = make((1, 1, S, D), 1), make((1, 1, S, D), 2)
    angle = torch.arange(S)[:, None] * 10.0 ** -torch.arange(R // 2)
    cos, sin = angle.cos().cuda(), angle.sin().cuda()
    dq, dw, ws = torch.zeros_like(q), nan(D), nan(lib.kcg_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(d)) // 4)
    st = lib.kcg_qk_norm_rope_bwd_launch(ctypes.byref(d), dy.data_ptr(), None, q.data_ptr(), None, w.data_ptr(), None, cos.data_ptr(), sin.data_ptr(),
                                         None, dq.data_ptr(), None, dw.data_ptr(), None, ws.data_ptr(), ws.numel() * 4,
                                         torch.cuda.current_stream().cuda_stream)
    return st, ops.last_device_status(), dw, ws


def main():
    lib = capi.load()
    out = {"enabled": int(lib.kcg_debug_bounds_enabled())}
    limit, detail = lib.kcg_debug_set_extent_limit, (ctypes.c_uint64 * 2)()

    # row statistics: 200 rows of 4 bytes, capped after 100
    a = Attention(lib, 1, 1, 1, 200, 200, 64)
    plain = a.forward()
    want = a.lse.clone()
    a.lse.fill_(math.nan)
    limit(400)
    capped = a.forward()
    limit(0)
    out["lse"] = {"plain": plain, "capped": capped, "kept": bool(torch.equal(a.lse[:100], want[:100])), "untouched": bool(a.lse[100:].isnan().all())}

    # -lse and -delta by row, padded to 128 rows a head: more bytes than the one-row tensors
    a = Attention(lib, 1, 4, 4, 1, 1, 64)
    a.forward()
    plain = a.backward()
    a.ws.fill_(math.nan)
    limit(1024)                            # the tensors have 512 bytes, the statistics 2048 each
    capped = a.backward()
    lib.kcg_debug_bounds_detail(detail)
    limit(0)
    stats = a.ws[:1024].view(2, 512)
    out["stat"] = {"plain": plain, "capped": capped, "extent": int(detail[1]), "kept": bool(not stats[:, :256].isnan().any()),
                   "untouched": bool(stats[:, 256:].isnan().all())}

    # pieces of dK and dV (8 of 32 query heads' one tile each), and of dQ (6 for each query tile): more bytes
    # than any tensor and than the statistics
    for what, shape in (("pieces", (1, 32, 1, 1, 90, 64)), ("pieces_q", (1, 8, 1, 100, 3000, 64))):
        a = Attention(lib, *shape)
        a.forward()
        plain = a.backward()
        grads = [t.clone() for t in a.grads]
        cap = max(*(t.numel() * 2 for t in a.grads), shape[1] * 128 * 4)
        limit(cap)
        capped = a.backward()
        lib.kcg_debug_bounds_detail(detail)
        limit(0)
        after = a.backward()
        out[what] = {"plain": plain, "capped": capped, "extent": int(detail[1]), "cap": cap, "after": after, "bytes": a.ws.numel() * 4,
                     "same": all(bool(torch.equal(x, y)) for x, y in zip(grads, a.grads))}

    # partial weight gradients and their sum: D of 4 bytes, capped after 32
    for what, S, D, R in (("dw", 60, 64, 64), ("dw_pairs", 16, 66, 38)):
        w = torch.ones(D, device="cuda", dtype=torch.bfloat16)
        st, status, want, _ = rotation(lib, S, D, R, w)
        limit(128)
        st2, status2, dw, ws = rotation(lib, S, D, R, w)
        limit(0)
        out[what] = {"plain": (st, status), "capped": (st2, status2), "kept": bool(torch.equal(dw[:32], want[:32]) and not ws[:32].isnan().any()),
                     "untouched": bool(dw[32:].isnan().all() and ws[32:].isnan().all())}
    print(json.dumps(out))


if __name__ == "__main__":
    main()
