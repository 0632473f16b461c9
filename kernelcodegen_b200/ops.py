"""Operator-level entry points on torch CUDA tensors.

Names follow the reference's Frontend operators (include/Frontend/Operators.h:73-98):
`matmul` (+ fused `relu`, the `@fuse_matmul_relu` graph of README.md:9-26 with the ReLU of
src/Frontend/Operators.cc:232-244 folded into the epilogue) and `fmha`
(BatchedMatmul(Q, K^T) -> Softmax -> BatchedMatmul(P, V), test/test.cc:88-90).

torch is used for device memory and streams only; the arithmetic is done by the hand-written
sm_100a kernels behind the C-ABI.  Nothing here falls back to torch math.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import capi

_PRECISIONS = {"3xtf32": capi.KCG_PREC_3XTF32, "tf32": capi.KCG_PREC_TF32, "bf16": capi.KCG_PREC_BF16}
_workspaces: dict = {}


def _dtype_code(dt: torch.dtype) -> int:
    if dt == torch.float32:
        return capi.KCG_F32
    if dt == torch.bfloat16:
        return capi.KCG_BF16
    raise TypeError(f"unsupported dtype {dt}: the kernels take float32 or bfloat16")


def _workspace(device: torch.device, nbytes: int) -> Optional[torch.Tensor]:
    """Grow-only scratch buffer per (device, stream)."""
    if nbytes == 0:
        return None
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _workspaces[key] = buf
    return buf


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError("kernelcodegen_b200 operators need CUDA tensors; there is no CPU path")
        if t.device != dev:
            raise RuntimeError("all tensors must live on the same device")
    return dev


def matmul(a: torch.Tensor, b: torch.Tensor, *, relu: bool = False, precision: Optional[str] = None,
           out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
           b_col_major: bool = False, tile_n: int = 0, stages: int = 0, group_m: int = 0,
           cta_group: int = 0, peers: Sequence[int] = (), mc: int = 0, done_flags: Sequence[int] = (),
           done_value: int = 0) -> torch.Tensor:
    """C = A . B (optionally ReLU'd).  A is [M, K] row-major; B is [K, N] row-major, or
    [N, K] when `b_col_major` (the reference's Layout::colMajor).  fp32 inputs use the
    3xTF32 path unless `precision="tf32"`; bf16 inputs use the bf16 path.
    `peers` are raw device pointers of other ranks' C buffers that also receive every tile;
    `mc` is the multicast address of `out` (every tile is then stored once and delivered to all
    ranks by the switch); `done_flags` are the words that receive `done_value` when the launch,
    and all its stores, have completed (see `peer.SymmetricMatrix`)."""
    dev = _require_cuda(a, b)
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("matmul takes 2-D tensors")
    M, K = a.shape
    if b_col_major:
        N, Kb = b.shape
    else:
        Kb, N = b.shape
    if K != Kb:
        raise ValueError(f"inner dimensions differ: A is {tuple(a.shape)}, B is {tuple(b.shape)}")
    if a.dtype != b.dtype:
        raise TypeError("A and B must have the same dtype")
    if a.stride(1) != 1 or b.stride(1) != 1:
        raise ValueError("A and B must be row-contiguous (stride 1 in the last dimension)")
    if precision is None:
        precision = "bf16" if a.dtype == torch.bfloat16 else "3xtf32"
    if precision not in _PRECISIONS:
        raise ValueError(f"precision must be one of {sorted(_PRECISIONS)}")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else a.dtype
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=dev)
    elif out.shape != (M, N) or out.stride(1) != 1 or out.device != dev:
        raise ValueError("out has the wrong shape, stride or device")
    d = capi.GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = a.stride(0), b.stride(0), out.stride(0)
    d.dtype_in, d.dtype_out = _dtype_code(a.dtype), _dtype_code(out.dtype)
    d.precision = _PRECISIONS[precision]
    d.epilogue = capi.KCG_EPI_RELU if relu else capi.KCG_EPI_NONE
    d.b_layout = capi.KCG_COL_MAJOR if b_col_major else capi.KCG_ROW_MAJOR
    d.tile_n, d.stages, d.group_m = tile_n, stages, group_m
    d.cta_group = cta_group
    d.n_peers = len(peers)
    for i, p in enumerate(peers):
        d.peer_c[i] = p
    d.mc_c = mc or None
    d.n_done_flags = len(done_flags)
    d.done_value = done_value & 0xFFFFFFFF
    for i, p in enumerate(done_flags):
        d.done_flags[i] = p
    lib = capi.load()
    with torch.cuda.device(dev):
        ws_bytes = lib.kcg_gemm_workspace_bytes(ctypes.byref(d))
        ws = _workspace(dev, ws_bytes)
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.kcg_gemm_launch(ctypes.byref(d), a.data_ptr(), b.data_ptr(), out.data_ptr(),
                                 ws.data_ptr() if ws is not None else None, ws_bytes, stream)
    capi.check(st, "kcg_gemm_launch")
    return out


def matmul_host(a_host: torch.Tensor, b_host: Optional[torch.Tensor], c_host: torch.Tensor, a_dev: torch.Tensor,
                b_dev: torch.Tensor, c_dev: torch.Tensor, *, relu: bool = False, precision: Optional[str] = None,
                b_col_major: bool = False, chunks: int = 0, peers: Sequence[int] = ()) -> torch.Tensor:
    """c_host = A . B from HOST arrays (pin them for the copies to overlap), staged through the
    caller's device arrays of the same shapes: row chunks of A and column chunks of B are copied
    while the kernel already runs on the tiles that have arrived, and finished strips of C return
    to the host meanwhile (`kcg_gemm_host_staged`).  `b_host=None`: B is already in `b_dev`.
    Asynchronous: synchronise the current stream before reading `c_host`."""
    dev = _require_cuda(a_dev, b_dev, c_dev)
    for h, t in ((a_host, a_dev), (b_host, b_dev), (c_host, c_dev)):
        if h is None and t is b_dev:
            continue
        if h.is_cuda or h.shape != t.shape or h.dtype != t.dtype or h.stride() != t.stride():
            raise ValueError("host and device arrays must match in shape, dtype and strides")
        if h.dim() != 2 or h.stride(1) != 1:
            raise ValueError("2-D row-contiguous arrays expected")
    M, K = a_dev.shape
    N = b_dev.shape[0] if b_col_major else b_dev.shape[1]
    if (b_dev.shape[1] if b_col_major else b_dev.shape[0]) != K or c_dev.shape != (M, N):
        raise ValueError("shapes do not form a product")
    if precision is None:
        precision = "bf16" if a_dev.dtype == torch.bfloat16 else "3xtf32"
    d = capi.GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.lda, d.ldb, d.ldc = a_dev.stride(0), b_dev.stride(0), c_dev.stride(0)
    d.dtype_in, d.dtype_out = _dtype_code(a_dev.dtype), _dtype_code(c_dev.dtype)
    d.precision = _PRECISIONS[precision]
    d.epilogue = capi.KCG_EPI_RELU if relu else capi.KCG_EPI_NONE
    d.b_layout = capi.KCG_COL_MAJOR if b_col_major else capi.KCG_ROW_MAJOR
    d.n_peers = len(peers)
    for i, p in enumerate(peers):
        d.peer_c[i] = p
    lib = capi.load()
    with torch.cuda.device(dev):
        ws_bytes = lib.kcg_gemm_workspace_bytes(ctypes.byref(d))
        ws = _workspace(dev, ws_bytes)
        st = lib.kcg_gemm_host_staged(ctypes.byref(d), a_host.data_ptr(),
                                      b_host.data_ptr() if b_host is not None else None, c_host.data_ptr(),
                                      a_dev.data_ptr(), b_dev.data_ptr(), c_dev.data_ptr(),
                                      ws.data_ptr() if ws is not None else None, ws_bytes, chunks,
                                      torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_gemm_host_staged")
    return c_host


def matmul_relu(a: torch.Tensor, b: torch.Tensor, **kw) -> torch.Tensor:
    """The `@fuse_matmul_relu` operator: max(0, A . B)."""
    return matmul(a, b, relu=True, **kw)


def fmha(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float = 1.0, causal: bool = False,
         out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """O = softmax(scale * Q K^T [causal]) V over [B, H, S, D] tensors.
    scale=1, causal=False is exactly the reference's three-operator graph."""
    dev = _require_cuda(q, k, v)
    if q.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("expected Q [B,H,Sq,D] and K, V [B,H,Skv,D]")
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        raise ValueError("Q, K, V must be contiguous [B,H,S,D]")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("Q, K, V must share a dtype")
    B, H, Sq, D = q.shape
    Skv = k.shape[2]
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else q.dtype
    if out is None:
        out = torch.empty((B, H, Sq, D), dtype=out_dtype, device=dev)
    elif out.shape != q.shape or not out.is_contiguous() or out.device != dev:
        raise ValueError("out has the wrong shape, stride or device")
    d = capi.FmhaDesc()
    d.B, d.H, d.Sq, d.Skv, d.D = B, H, Sq, Skv, D
    d.dtype_in, d.dtype_out = _dtype_code(q.dtype), _dtype_code(out.dtype)
    d.causal = 1 if causal else 0
    d.scale = float(scale)
    lib = capi.load()
    with torch.cuda.device(dev):
        ws_bytes = lib.kcg_fmha_workspace_bytes(ctypes.byref(d))
        ws = _workspace(dev, ws_bytes)
        stream = torch.cuda.current_stream(dev).cuda_stream
        st = lib.kcg_fmha_fwd_launch(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                     ws.data_ptr() if ws is not None else None, ws_bytes, stream)
    capi.check(st, "kcg_fmha_fwd_launch")
    return out


def _strides(t: torch.Tensor):
    """Batch, head and row stride of a [B, H, S, D] view, as the C-ABI takes them."""
    return (ctypes.c_int64 * 3)(*t.stride()[:3])


def _check_heads(name: str, t: torch.Tensor, shape: Sequence[int], dtype: torch.dtype, dev: torch.device) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != dev:
        raise RuntimeError("all tensors must live on the same device")
    if t.shape[3] != 1 and t.stride(3) != 1:
        raise ValueError(f"{name} must have stride 1 in the last dimension")


def _attn_desc(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, causal: bool) -> "capi.AttnDesc":
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("expected Q [B,H,Sq,D] and K, V [B,Hkv,Skv,D]")
    if q.dtype != torch.bfloat16 or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("Q, K, V must be bfloat16: the gradients' contractions have no float32 form")
    for name, t in (("Q", q), ("K", k), ("V", v)):
        _check_heads(name, t, t.shape, q.dtype, q.device)
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError("the number of query heads must be a multiple of the number of key/value heads")
    d = capi.AttnDesc()
    d.B, d.H, d.Sq, d.D = q.shape
    d.Hkv, d.Skv = k.shape[1:3]
    d.dtype = capi.KCG_BF16
    d.causal = 1 if causal else 0
    d.scale = float(scale)
    d.q, d.k, d.v = _strides(q), _strides(k), _strides(v)
    return d


def fmha_with_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float = 1.0, causal: bool = False,
                  out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`fmha` for a forward pass that will be differentiated: (O, lse), lse[b, h, i] = log sum_j
    exp(scale q_i.k_j) in float32 [B, H, Sq] (-inf, and O = 0, for a query that sees no key).
    bfloat16 [B, H, S, D] views with any strides that are multiples of 16 bytes and stride 1 in the
    last dimension (heads of a packed projection: `x.view(B, S, heads, D).transpose(1, 2)`); K and V may
    have fewer heads, Hkv | H, and query head h then reads head h // (H // Hkv).  D is 64 or 128.
    O is contiguous unless `out` is given."""
    dev = _require_cuda(q, k, v)
    d = _attn_desc(q, k, v, scale, causal)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _check_heads("out", out, q.shape, q.dtype, dev)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev)
    d.o = _strides(out)
    with torch.cuda.device(dev):
        st = capi.load().kcg_fmha_fwd_lse_launch(ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                                 lse.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_fmha_fwd_lse_launch")
    return out, lse


def fmha_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                  lse: torch.Tensor, *, scale: float = 1.0, causal: bool = False, dq: Optional[torch.Tensor] = None,
                  dk: Optional[torch.Tensor] = None, dv: Optional[torch.Tensor] = None
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dQ, dK, dV) of `fmha_with_lse`, from the gradient of its O and the `out` and `lse` it returned
    (call with the same scale and causal).  Views as there; the gradients are contiguous unless dq, dk or
    dv is given, e.g. as the heads of a packed gradient.  Outputs must not overlap one another or an
    input.  The same bits on every call: nothing is added up in an order that can change."""
    dev = _require_cuda(dout, q, k, v, out, lse)
    d = _attn_desc(q, k, v, scale, causal)
    _check_heads("dout", dout, q.shape, q.dtype, dev)
    _check_heads("out", out, q.shape, q.dtype, dev)
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be the contiguous float32 [B,H,Sq] tensor of fmha_with_lse")
    grads = []
    for name, g, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
        if g is None:
            g = torch.empty(like.shape, dtype=like.dtype, device=dev)
        else:
            _check_heads(name, g, like.shape, like.dtype, dev)
        grads.append(g)
    dq, dk, dv = grads
    d.o, d.d_o, d.d_q, d.d_k, d.d_v = (_strides(t) for t in (out, dout, dq, dk, dv))
    lib = capi.load()
    with torch.cuda.device(dev):
        # a buffer of this call alone, from the stream's allocator: two captured graphs never share it
        ws_bytes = lib.kcg_fmha_bwd_workspace_bytes(ctypes.byref(d))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        st = lib.kcg_fmha_bwd_launch(ctypes.byref(d), dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                     out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                     ws.data_ptr(), ws_bytes, torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_fmha_bwd_launch")
    return dq, dk, dv


def _rope_desc(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    """Checks what both directions of qk_norm_rope take and fills the descriptor's shared part."""
    dev = q.device
    if q.dim() != 4:
        raise ValueError("expected queries (and keys) as [B, heads, S, D]")
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {q.dtype}: the kernels take float32 or bfloat16")
    B, H, S, D = q.shape
    _check_heads("q", q, q.shape, q.dtype, dev)
    if k is not None:
        if k.dim() != 4:
            raise ValueError("expected queries (and keys) as [B, heads, S, D]")
        _check_heads("k", k, (B, k.shape[1], S, D), q.dtype, dev)
    elif k_weight is not None:
        raise ValueError("k_weight without keys")
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > D:
        raise ValueError("cos and sin must be [positions, R / 2] with R <= D")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous float32 table")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (D,) or not w.is_contiguous() or w.dtype != weights[0].dtype or w.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("the weights must be contiguous [D] tensors, both float32 or both bfloat16")
    d = capi.RopeDesc()
    d.B, d.S, d.H, d.Hk, d.D, d.R = B, S, H, k.shape[1] if k is not None else 0, D, 2 * cos.shape[1]
    d.dtype = _dtype_code(q.dtype)
    d.dtype_w = _dtype_code(weights[0].dtype) if weights else capi.KCG_F32
    d.interleaved = 1 if interleaved else 0
    d.table_rows = cos.shape[0]
    d.eps = float(eps)
    d.pos_bits = 32
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be int32 or int64")
        if tuple(positions.shape) not in ((S,), (B, S)):
            raise ValueError(f"positions must be [{S}] or [{B}, {S}]")
        d.pos_bits = 64 if positions.dtype == torch.int64 else 32
        d.pos = (ctypes.c_int64 * 2)(positions.stride(0) if positions.dim() == 2 else 0, positions.stride(-1))
    elif S > cos.shape[0]:
        raise ValueError("more tokens than rows of the tables")
    _require_cuda(*[t for t in (q, k, cos, sin, *weights, positions) if t is not None])
    d.q = _strides(q)
    if k is not None:
        d.k = _strides(k)
    return d


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _like(name: str, given: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    if given is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _check_heads(name, given, like.shape, like.dtype, like.device)
    return given


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None
                 ) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """What attention wants done to queries and keys first, in one pass: every head row x becomes
    x / sqrt(mean(x^2) + eps) * weight (weight [D], ones when None), and the pairs (a, b) of its first
    R entries are rotated to (a cos - b sin, b cos + a sin).  q is a [B, H, S, D] view, k a [B, Hk, S, D]
    one or None, float32 or bfloat16, any strides but 1 in the last dimension; D even, at most 256.
    cos, sin: float32 [positions, R / 2] tables; pairs are (i, i + R/2), or (2i, 2i + 1) if `interleaved`.
    positions: int32 or int64 [S] or [B, S], None for 0..S-1; a position outside the tables makes the
    row's rotated entries NaN and sets `last_device_status()` to 11.
    The outputs are contiguous [B, heads, S, D] unless q_out / k_out is given (a slice of a key cache, or
    the input itself)."""
    d = _rope_desc(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    q_out = _like("q_out", q_out, q)
    d.q_out = _strides(q_out)
    if k is not None:
        k_out = _like("k_out", k_out, k)
        d.k_out = _strides(k_out)
    elif k_out is not None:
        raise ValueError("k_out without keys")
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return q_out, k_out
    dev = q.device
    with torch.cuda.device(dev):
        st = capi.load().kcg_qk_norm_rope_launch(ctypes.byref(d), q.data_ptr(), _ptr(k), _ptr(q_weight), _ptr(k_weight),
                                                 cos.data_ptr(), sin.data_ptr(), _ptr(positions), q_out.data_ptr(),
                                                 _ptr(k_out), torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_qk_norm_rope_launch")
    return q_out, k_out


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: Optional[torch.Tensor], q: torch.Tensor, k: Optional[torch.Tensor],
                          cos: torch.Tensor, sin: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                          eps: float = 1e-6, interleaved: bool = False, dq: Optional[torch.Tensor] = None,
                          dk: Optional[torch.Tensor] = None
                          ) -> tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dq, dk, dq_weight, dk_weight) of `qk_norm_rope` for the gradients of its outputs and the inputs
    it was called with.  The weights' gradients are float32 [D], summed over batch, heads and tokens in a
    fixed order (None for a weight that is None).  dq and dk are contiguous unless given; they may be
    dq_out and dk_out themselves."""
    d = _rope_desc(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    dev = q.device
    if (dk_out is None) != (k is None) or (k is None and dk is not None):
        raise ValueError("keys and their gradients go together")
    _check_heads("dq_out", dq_out, q.shape, q.dtype, dev)
    dq = _like("dq", dq, q)
    d.q_out, d.d_q = _strides(dq_out), _strides(dq)
    if k is not None:
        _check_heads("dk_out", dk_out, k.shape, k.dtype, dev)
        dk = _like("dk", dk, k)
        d.k_out, d.d_k = _strides(dk_out), _strides(dk)
    new = torch.zeros if q.numel() == 0 else torch.empty
    dqw, dkw = (new(q.shape[3], dtype=torch.float32, device=dev) if w is not None else None for w in (q_weight, k_weight))
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return dq, dk, dqw, dkw
    lib = capi.load()
    with torch.cuda.device(dev):
        # a buffer of this call alone, from the stream's allocator: two captured graphs never share it
        ws_bytes = lib.kcg_qk_norm_rope_bwd_workspace_bytes(ctypes.byref(d)) if dqw is not None or dkw is not None else 0
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        st = lib.kcg_qk_norm_rope_bwd_launch(ctypes.byref(d), dq_out.data_ptr(), _ptr(dk_out), q.data_ptr(), _ptr(k),
                                             _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), _ptr(positions),
                                             dq.data_ptr(), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(ws), ws_bytes,
                                             torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_qk_norm_rope_bwd_launch")
    return dq, dk, dqw, dkw


def softmax(x: torch.Tensor, *, inplace: bool = False) -> torch.Tensor:
    """Last-axis softmax of an fp32 tensor (the reference's standalone Softmax operator)."""
    dev = _require_cuda(x)
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise TypeError("softmax takes a contiguous float32 tensor")
    y = x if inplace else torch.empty_like(x)
    cols = x.shape[-1]
    rows = x.numel() // cols
    with torch.cuda.device(dev):
        st = capi.load().kcg_softmax_launch(rows, cols, x.data_ptr(), y.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_softmax_launch")
    return y


def transpose(x: torch.Tensor) -> torch.Tensor:
    """y[..., j, i] = x[..., i, j] as a new contiguous tensor (the reference's Transpose operator,
    which it declares without a body); leading dimensions are batch dimensions."""
    dev = _require_cuda(x)
    if x.dim() < 2 or not x.is_contiguous():
        raise ValueError("transpose takes a contiguous tensor of at least 2 dimensions")
    rows, cols = x.shape[-2:]
    batch = x.numel() // max(1, rows * cols)
    y = torch.empty(x.shape[:-2] + (cols, rows), dtype=x.dtype, device=dev)
    if x.numel() == 0:
        return y
    with torch.cuda.device(dev):
        st = capi.load().kcg_transpose_launch(batch, rows, cols, _dtype_code(x.dtype), x.data_ptr(), y.data_ptr(),
                                              torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_transpose_launch")
    return y


def batched_matmul(a: torch.Tensor, b: torch.Tensor, *, b_col_major: bool = False, precision: Optional[str] = None,
                   relu: bool = False) -> torch.Tensor:
    """C[..., m, n] = A[..., m, k] . B[..., k, n]  (B[..., n, k] when `b_col_major`): the
    reference's standalone BatchedMatmul operator; leading dimensions are batch dimensions."""
    dev = _require_cuda(a, b)
    if a.dim() < 2 or a.dim() != b.dim() or a.shape[:-2] != b.shape[:-2]:
        raise ValueError("A and B need equal batch dimensions")
    if not (a.is_contiguous() and b.is_contiguous()) or a.dtype != b.dtype:
        raise ValueError("A and B must be contiguous and share a dtype")
    m, k = a.shape[-2:]
    n, kb = (b.shape[-2], b.shape[-1]) if b_col_major else (b.shape[-1], b.shape[-2])
    if k != kb:
        raise ValueError("inner dimensions differ")
    batch = 1
    for s_ in a.shape[:-2]:
        batch *= s_
    out = torch.empty(a.shape[:-2] + (m, n), dtype=a.dtype, device=dev)
    if precision is None:
        precision = "bf16" if a.dtype == torch.bfloat16 else "3xtf32"
    d = capi.GemmDesc()
    d.M, d.N, d.K = m, n, k
    d.lda, d.ldb, d.ldc = k, (k if b_col_major else n), n
    d.dtype_in = d.dtype_out = _dtype_code(a.dtype)
    d.precision = _PRECISIONS[precision]
    d.epilogue = capi.KCG_EPI_RELU if relu else capi.KCG_EPI_NONE
    d.b_layout = capi.KCG_COL_MAJOR if b_col_major else capi.KCG_ROW_MAJOR
    lib = capi.load()
    with torch.cuda.device(dev):
        ws_bytes = lib.kcg_batched_gemm_workspace_bytes(ctypes.byref(d), batch, m * k, k * n)
        ws = _workspace(dev, ws_bytes)
        st = lib.kcg_batched_gemm_launch(ctypes.byref(d), batch, m * k, k * n, m * n, a.data_ptr(), b.data_ptr(),
                                         out.data_ptr(), ws.data_ptr() if ws is not None else None, ws_bytes,
                                         torch.cuda.current_stream(dev).cuda_stream)
    capi.check(st, "kcg_batched_gemm_launch")
    return out


def peer_wait(flags_ptr: int, n: int, stride_words: int, value: int, device: torch.device, max_polls: int = 0) -> None:
    """Queues, on the current stream, a bounded device-side wait until the `n` flag words at
    `flags_ptr` (stride in 32-bit words) have reached `value`."""
    with torch.cuda.device(device):
        st = capi.load().kcg_peer_wait_launch(flags_ptr, n, stride_words, value & 0xFFFFFFFF, max_polls,
                                              torch.cuda.current_stream(device).cuda_stream)
    capi.check(st, "kcg_peer_wait_launch")


def peer_wait_status() -> None:
    """Synchronises and raises KcgError(KCG_PEER_TIMEOUT / KCG_DEVICE_TIMEOUT) if a bounded wait ran out."""
    capi.check(capi.load().kcg_peer_wait_status(), "kcg_peer_wait_status")


def last_device_status() -> int:
    """0, or the code of the bounded device-side wait that ran out (synchronises)."""
    return int(capi.load().kcg_last_device_status())


def launch_count() -> int:
    return int(capi.load().kcg_launch_count())
