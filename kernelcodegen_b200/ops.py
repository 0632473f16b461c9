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
import struct
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


# The operators below are called once per layer of a step, on short sequences too, where the host's part of a
# call is most of its time: every property of a tensor is read once, and a descriptor is packed whole.
_ATTN_PACK = struct.Struct("@8ifi24q")
_ROPE_PACK = struct.Struct("@10iqfi20q")
_POSITION_BITS = {torch.int32: 32, torch.int64: 64}
_NO_STRIDES = (0, 0, 0)
# the handle alone: torch.cuda.current_stream(dev).cuda_stream builds an object for it, 2 us of a 12 us call
_raw_stream = torch._C._cuda_getCurrentRawStream


def _launch(dev: torch.device, fn, *args) -> int:
    """fn(*args, stream) with `dev` current, on its current stream."""
    index = dev.index
    if torch.cuda.current_device() == index:
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(dev):
        return fn(*args, _raw_stream(index))


def _view(name: str, t: torch.Tensor, shape, dtype: torch.dtype, dev: torch.device):
    """Batch, head and row stride of a [B, H, S, D] view, as the C-ABI takes them, of the tensor that is
    expected."""
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != dev:
        raise RuntimeError("all tensors must live on the same device")
    sb, sh, sr, sd = t.stride()
    if sd != 1 and shape[3] != 1:
        raise ValueError(f"{name} must have stride 1 in the last dimension")
    return sb, sh, sr


def _output(name: str, given: Optional[torch.Tensor], shape, dtype: torch.dtype, dev: torch.device):
    """An output [B, H, S, D] and its strides: a new contiguous tensor, or the one given."""
    if given is not None:
        return given, _view(name, given, shape, dtype, dev)
    _, H, S, D = shape
    strides = (H * S * D, S * D, D)
    # (empty_strided takes half the host time of empty)
    return torch.empty_strided(shape, (*strides, 1), dtype=dtype, device=dev), strides


def _attn_views(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
    """Checks Q, K and V of an attention call; (device, their shapes, their strides)."""
    dev = q.device
    if not q.is_cuda:
        raise RuntimeError("kernelcodegen_b200 operators need CUDA tensors; there is no CPU path")
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 4 or len(k_shape) != 4 or k_shape != v.shape or q_shape[0] != k_shape[0] or q_shape[3] != k_shape[3]:
        raise ValueError("expected Q [B,H,Sq,D] and K, V [B,Hkv,Skv,D]")
    if not q.dtype is k.dtype is v.dtype is torch.bfloat16:
        raise TypeError("Q, K, V must be bfloat16: the gradients' contractions have no float32 form")
    if k_shape[1] == 0 or q_shape[1] % k_shape[1]:
        raise ValueError("the number of query heads must be a multiple of the number of key/value heads")
    bf16 = torch.bfloat16
    return dev, q_shape, k_shape, (*_view("Q", q, q_shape, bf16, dev), *_view("K", k, k_shape, bf16, dev),
                                   *_view("V", v, k_shape, bf16, dev))


def _attn_desc(q_shape, k_shape, causal: bool, scale: float, strides) -> "capi.AttnDesc":
    B, H, Sq, D = q_shape
    return capi.AttnDesc.from_buffer_copy(_ATTN_PACK.pack(B, H, k_shape[1], Sq, k_shape[2], D, capi.KCG_BF16,
                                                          1 if causal else 0, scale, 0, *strides))


def fmha_with_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float = 1.0, causal: bool = False,
                  out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """`fmha` for a forward pass that will be differentiated: (O, lse), lse[b, h, i] = log sum_j
    exp(scale q_i.k_j) in float32 [B, H, Sq] (-inf, and O = 0, for a query that sees no key).
    bfloat16 [B, H, S, D] views with any strides that are multiples of 16 bytes and stride 1 in the
    last dimension (heads of a packed projection: `x.view(B, S, heads, D).transpose(1, 2)`); K and V may
    have fewer heads, Hkv | H, and query head h then reads head h // (H // Hkv).  D is 64 or 128.
    O is contiguous unless `out` is given."""
    dev, q_shape, k_shape, strides = _attn_views(q, k, v)
    out, o = _output("out", out, q_shape, torch.bfloat16, dev)
    B, H, Sq, _ = q_shape
    lse = torch.empty_strided((B, H, Sq), (H * Sq, Sq, 1), dtype=torch.float32, device=dev)
    d = _attn_desc(q_shape, k_shape, causal, scale, (*strides, *o, *_NO_STRIDES * 4))
    st = _launch(dev, capi.load().kcg_fmha_fwd_lse_launch, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                 lse.data_ptr())
    if st:
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
    dev, q_shape, k_shape, strides = _attn_views(q, k, v)
    bf16 = torch.bfloat16
    g = _view("dout", dout, q_shape, bf16, dev)
    o = _view("out", out, q_shape, bf16, dev)
    if lse.shape != q_shape[:3] or lse.dtype is not torch.float32 or lse.device != dev or not lse.is_contiguous():
        raise ValueError("lse must be the contiguous float32 [B,H,Sq] tensor of fmha_with_lse")
    dq, sq = _output("dq", dq, q_shape, bf16, dev)
    dk, sk = _output("dk", dk, k_shape, bf16, dev)
    dv, sv = _output("dv", dv, k_shape, bf16, dev)
    d = _attn_desc(q_shape, k_shape, causal, scale, (*strides, *o, *g, *sq, *sk, *sv))
    lib = capi.load()
    # a buffer of this call alone, from the stream's allocator: two captured graphs never share it
    ws_bytes = lib.kcg_fmha_bwd_workspace_bytes(d)
    ws = torch.empty_strided((ws_bytes,), (1,), dtype=torch.uint8, device=dev)
    st = _launch(dev, lib.kcg_fmha_bwd_launch, d, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                 lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes)
    if st:
        capi.check(st, "kcg_fmha_bwd_launch")
    return dq, dk, dv


def _rope_views(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    """Checks what both directions of qk_norm_rope take; (device, shapes of q and k, the descriptor up to
    the strides, strides of q and k, pointers of weights, tables and positions)."""
    q_shape, dtype, dev = q.shape, q.dtype, q.device
    if len(q_shape) != 4:
        raise ValueError("expected queries (and keys) as [B, heads, S, D]")
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"unsupported dtype {dtype}: the kernels take float32 or bfloat16")
    if not q.is_cuda:
        raise RuntimeError("kernelcodegen_b200 operators need CUDA tensors; there is no CPU path")
    B, H, S, D = q_shape
    strides, k_shape = _view("q", q, q_shape, dtype, dev), None
    if k is not None:
        k_shape = k.shape
        if len(k_shape) != 4 or k_shape[0] != B or k_shape[2] != S or k_shape[3] != D:
            raise ValueError(f"k has shape {tuple(k_shape)}, expected [{B}, heads, {S}, {D}]")
        strides += _view("k", k, k_shape, dtype, dev)
    else:
        if k_weight is not None:
            raise ValueError("k_weight without keys")
        strides += _NO_STRIDES
    t_shape = cos.shape
    if len(t_shape) != 2 or t_shape != sin.shape or 2 * t_shape[1] > D:
        raise ValueError("cos and sin must be [positions, R / 2] with R <= D")
    for t in (cos, sin):
        if t.dtype is not torch.float32 or not t.is_contiguous():
            raise TypeError("cos and sin must be contiguous float32 tables")
        if t.device != dev:
            raise RuntimeError("all tensors must live on the same device")
    w_dtype = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w_dtype is None:
            w_dtype = w.dtype
        if w.shape != (D,) or w.dtype is not w_dtype or not w.is_contiguous():
            raise ValueError("the weights must be contiguous [D] tensors of one type")
        if w.device != dev:
            raise RuntimeError("all tensors must live on the same device")
    pos_bits, pos = 32, (0, 0)
    if positions is not None:
        pos_bits = _POSITION_BITS.get(positions.dtype)
        if pos_bits is None:
            raise TypeError("positions must be int32 or int64")
        p_shape = positions.shape
        if p_shape == (B, S):
            pos = positions.stride()
        elif p_shape == (S,):
            pos = (0, positions.stride(0))
        else:
            raise ValueError(f"positions must be [{S}] or [{B}, {S}]")
        if positions.device != dev:
            raise RuntimeError("all tensors must live on the same device")
    elif S > t_shape[0]:
        raise ValueError("more tokens than rows of the tables")
    head = (B, S, H, k_shape[1] if k is not None else 0, D, 2 * t_shape[1], _dtype_code(dtype),
            capi.KCG_F32 if w_dtype is None else _dtype_code(w_dtype), 1 if interleaved else 0, pos_bits, t_shape[0], eps, 0, *pos)
    return dev, q_shape, k_shape, head, strides, (_ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), _ptr(positions))


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


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
    dev, q_shape, k_shape, head, strides, ptrs = _rope_views(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    dtype = q.dtype
    q_out, yq = _output("q_out", q_out, q_shape, dtype, dev)
    yk = _NO_STRIDES
    if k is not None:
        k_out, yk = _output("k_out", k_out, k_shape, dtype, dev)
    elif k_out is not None:
        raise ValueError("k_out without keys")
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return q_out, k_out
    d = capi.RopeDesc.from_buffer_copy(_ROPE_PACK.pack(*head, *strides, *yq, *yk, *_NO_STRIDES * 2))
    st = _launch(dev, capi.load().kcg_qk_norm_rope_launch, d, q.data_ptr(), _ptr(k), *ptrs, q_out.data_ptr(), _ptr(k_out))
    if st:
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
    dev, q_shape, k_shape, head, strides, ptrs = _rope_views(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    dtype = q.dtype
    if (dk_out is None) != (k is None) or (k is None and dk is not None):
        raise ValueError("keys and their gradients go together")
    gq, gk, sk = _view("dq_out", dq_out, q_shape, dtype, dev), _NO_STRIDES, _NO_STRIDES
    dq, sq = _output("dq", dq, q_shape, dtype, dev)
    if k is not None:
        gk = _view("dk_out", dk_out, k_shape, dtype, dev)
        dk, sk = _output("dk", dk, k_shape, dtype, dev)
    empty = q.numel() == 0 and (k is None or k.numel() == 0)
    dqw, dkw = (torch.empty_strided((q_shape[3],), (1,), dtype=torch.float32, device=dev) if w is not None else None
                for w in (q_weight, k_weight))
    if empty:
        for w in (dqw, dkw):
            if w is not None:
                w.zero_()
        return dq, dk, dqw, dkw
    d = capi.RopeDesc.from_buffer_copy(_ROPE_PACK.pack(*head, *strides, *gq, *gk, *sq, *sk))
    lib = capi.load()
    # a buffer of this call alone, from the stream's allocator: two captured graphs never share it
    ws_bytes = lib.kcg_qk_norm_rope_bwd_workspace_bytes(d) if dqw is not None or dkw is not None else 0
    ws = torch.empty_strided((ws_bytes,), (1,), dtype=torch.uint8, device=dev) if ws_bytes else None
    st = _launch(dev, lib.kcg_qk_norm_rope_bwd_launch, d, dq_out.data_ptr(), _ptr(dk_out), q.data_ptr(), _ptr(k), *ptrs,
                 dq.data_ptr(), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(ws), ws_bytes)
    if st:
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
