"""Tensor-level wrappers of the C ABI: allocate outputs and workspaces with torch (device
memory and streams only), pass raw pointers, launch on torch's current stream, raise on a
nonzero status.  No arithmetic happens here."""

from __future__ import annotations

import ctypes
import functools
import inspect

import torch

from . import _lib
from ._lib import (DTYPE_CODE, NF4Attn, NF4Grad, NF4Lora, NF4LoraJob, NF4PagedKV, check, load,
                   stream_of)
from .quant_state import weight_array, weight_desc

GEMM_DTYPES = (torch.float16, torch.bfloat16)

# tilings of the tiled GEMMs (NF4_TILE_* of the C header)
TILE_256, TILE_128, TILE_128_KSPLIT2 = 0, 1, 3


def _code(dtype: torch.dtype, allowed=GEMM_DTYPES) -> int:
    if dtype not in allowed:
        raise TypeError(f"dtype {dtype} is not supported here (expected one of {allowed})")
    return DTYPE_CODE[dtype]


def _descs(weights):
    """[(packed, quant_state), ...] -> ctypes array of descriptors."""
    return weight_array([weight_desc(p, qs) for p, qs in weights])


def _check_device(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("the NF4 kernels run on the GPU: every tensor must be on a cuda device")


def dequant(weights, dtype=torch.float16, out: torch.Tensor | None = None) -> torch.Tensor:
    """Stacked [sum rows, cols] dequantized weight(s) (nf4_dequant_multi)."""
    packed0 = weights[0][0]
    _check_device(packed0)
    rows = sum(int(qs.shape[0]) for _, qs in weights)
    cols = int(weights[0][1].shape[1])
    if out is None:
        out = torch.empty((rows, cols), dtype=dtype, device=packed0.device)
    arr = _descs(weights)
    st = load().nf4_dequant_multi(arr, len(weights), out.data_ptr(),
                                  _code(dtype, (torch.float16, torch.bfloat16, torch.float32)),
                                  stream_of(out))
    check(st, "nf4_dequant_multi")
    return out


def dequant_batch(weights, dtype=torch.float16, outs=None) -> list:
    """Each weight dequantized into its own [rows, cols] tensor, all in one launch
    (nf4_dequant_batch, at most 8 weights)."""
    packed0 = weights[0][0]
    _check_device(packed0)
    if outs is None:
        outs = [torch.empty(tuple(int(d) for d in qs.shape), dtype=dtype, device=packed0.device)
                for _, qs in weights]
    arr = _descs(weights)
    ptrs = (ctypes.c_void_p * len(outs))(*[o.data_ptr() for o in outs])
    st = load().nf4_dequant_batch(arr, len(weights), ptrs,
                                  _code(dtype, (torch.float16, torch.bfloat16, torch.float32)),
                                  stream_of(outs[0]))
    check(st, "nf4_dequant_batch")
    return outs


class DequantTable:
    """Any number of weights dequantized by one launch (nf4_dequant_table): the descriptor
    table is packed once on the host and kept in device memory; `run()` launches on torch's
    current stream.  `outs` default to fresh [rows, cols] tensors; the weights and outputs must
    stay alive (and in place) as long as the table is used - this object keeps references."""

    def __init__(self, weights, dtype=torch.float16, outs=None):
        packed0 = weights[0][0]
        _check_device(packed0)
        if outs is None:
            outs = [torch.empty(tuple(int(d) for d in qs.shape), dtype=dtype,
                                device=packed0.device) for _, qs in weights]
        self.weights, self.outs, self.dtype = list(weights), list(outs), dtype
        self._code = _code(dtype, (torch.float16, torch.bfloat16, torch.float32))
        arr = _descs(weights)
        lib = load()
        nbytes = lib.nf4_dequant_table_bytes(arr, len(weights))
        host = torch.empty(max(nbytes, 16), dtype=torch.uint8)
        ptrs = (ctypes.c_void_p * len(outs))(*[o.data_ptr() for o in outs])
        blocks = ctypes.c_int64(0)
        check(lib.nf4_dequant_table_pack(arr, len(weights), ptrs, self._code, host.data_ptr(),
                                         nbytes, ctypes.byref(blocks)), "nf4_dequant_table_pack")
        self.blocks = int(blocks.value)
        self.table = host.to(packed0.device)
        self.refs = [w for pair in weights for w in pair]

    def run(self):
        check(load().nf4_dequant_table(self.table.data_ptr(), len(self.weights), self.blocks,
                                       self._code, stream_of(self.table)), "nf4_dequant_table")
        return self.outs


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    if nbytes == 0:
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _lora_array(loras):
    if not loras:
        return None, 0
    arr = (NF4Lora * len(loras))(*loras)
    return arr, len(loras)


def linear_fwd(x: torch.Tensor, weights, bias: torch.Tensor | None = None, loras=(),
               out: torch.Tensor | None = None, tile: int | None = None,
               splits: int = 1) -> torch.Tensor:
    """Y[M, sum rows] = x[M, K] @ W_stack^T (+ bias) (+ LoRA terms).  `loras`: NF4Lora structs
    whose pointers stay alive for the call (make_lora's structs hold their tensors; a struct
    built otherwise needs the caller to keep them).  `tile` (TILE_*) and `splits` pin the
    tiling; None lets the library choose."""
    _check_device(x, bias)
    dt = _code(x.dtype)
    m, k = x.shape
    n = sum(int(qs.shape[0]) for _, qs in weights)
    if out is None:
        out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    arr = _descs(weights)
    lib = load()
    if tile is None:
        ws_bytes = lib.nf4_linear_fwd_workspace(m, arr, len(weights), dt)
    else:
        ws_bytes = 4 * splits * m * n if splits > 1 else 0
    ws = _workspace(ws_bytes, x.device)
    larr, nl = _lora_array(loras)
    args = (x.data_ptr() if m else None, m, x.stride(0), arr, len(weights),
            bias.data_ptr() if bias is not None else None, larr, nl, out.data_ptr(),
            out.stride(0), dt, ws.data_ptr() if ws is not None else None, ws_bytes, stream_of(x))
    if tile is None:
        check(lib.nf4_linear_fwd(*args), "nf4_linear_fwd")
    else:
        check(lib.nf4_linear_fwd_tiled(*args, int(tile), int(splits)), "nf4_linear_fwd_tiled")
    return out


def linear_dx(dy: torch.Tensor, weights, loras=(), out: torch.Tensor | None = None,
              accumulate: bool = False, tile: int | None = None,
              splits: int = 1) -> torch.Tensor:
    """dX[M, K] (+)= dY[M, sum rows] @ W_stack (+ LoRA terms); `tile` / `splits` as in
    linear_fwd."""
    _check_device(dy)
    dt = _code(dy.dtype)
    m = dy.shape[0]
    k = int(weights[0][1].shape[1])
    if out is None:
        out = torch.empty((m, k), dtype=dy.dtype, device=dy.device)
        accumulate = False
    offs = _offsets(weights)
    if tile is None and len(weights) > 1 and any(o % 8 for o in offs):
        return _linear_dx_by_segment(dy, weights, loras, out, accumulate, offs)
    arr = _descs(weights)
    lib = load()
    if tile is None:
        ws_bytes = lib.nf4_linear_dx_workspace(m, arr, len(weights), dt)
    else:
        ws_bytes = 4 * splits * m * k if splits > 1 else 0
    ws = _workspace(ws_bytes, dy.device)
    larr, nl = _lora_array(loras)
    args = (dy.data_ptr() if m else None, m, dy.stride(0), arr, len(weights), larr, nl,
            out.data_ptr(), out.stride(0), int(accumulate), dt,
            ws.data_ptr() if ws is not None else None, ws_bytes, stream_of(dy))
    if tile is None:
        check(lib.nf4_linear_dx(*args), "nf4_linear_dx")
    else:
        check(lib.nf4_linear_dx_tiled(*args, int(tile), int(splits)), "nf4_linear_dx_tiled")
    return out


def _offsets(weights):
    offs, o = [], 0
    for _, qs in weights:
        offs.append(o)
        o += int(qs.shape[0])
    return offs


def _linear_dx_by_segment(dy, weights, loras, out, accumulate, offs):
    """linear_dx over stacked segments of which one starts off a multiple of 8 dY columns: the
    stacked launch reads each segment's dY columns as 16-byte chunks, so each segment runs as
    its own launch over its dY columns (copied when they are not 16-byte aligned), the first
    writing dX and the others adding to it; a LoRA struct goes with its segment's launch."""
    by_seg = {}
    for lo in loras:
        by_seg.setdefault(int(lo.seg), []).append(lo)
    for i, (w, off) in enumerate(zip(weights, offs)):
        rows = int(w[1].shape[0])
        dy_s = dy[:, off: off + rows]
        if dy_s.data_ptr() % 16 or dy_s.stride(0) % 8:  # to rows of a multiple of 8 values
            pad = torch.empty((dy.shape[0], -(-rows // 8) * 8), dtype=dy.dtype, device=dy.device)
            pad[:, :rows].copy_(dy_s)
            dy_s = pad[:, :rows]
        seg_loras = [NF4Lora(seg=0, rank=lo.rank, scale=lo.scale, t=lo.t, b=lo.b, a=lo.a, da=lo.da)
                     for lo in by_seg.get(i, [])]
        linear_dx(dy_s, [w], seg_loras, out=out, accumulate=accumulate or i > 0)
    return out


def lora_xa(xd: torch.Tensor, a: torch.Tensor) -> torch.Tensor:
    """t[M, r] = xd[M, K] @ A[r, K]^T."""
    _check_device(xd, a)
    m, k = xd.shape
    r = a.shape[0]
    t = torch.empty((m, r), dtype=xd.dtype, device=xd.device)
    st = load().nf4_lora_xa(xd.data_ptr(), m, k, xd.stride(0), a.data_ptr(), r, t.data_ptr(),
                            _code(xd.dtype), stream_of(xd))
    check(st, "nf4_lora_xa")
    return t


def lora_da(dy: torch.Tensor, b: torch.Tensor, scale: float) -> torch.Tensor:
    """da[M, r] = scale * dY[M, N] @ B[N, r]  (dY may be a column slice: rows stride(0) apart)."""
    _check_device(dy, b)
    m, n = dy.shape
    r = b.shape[1]
    da = torch.empty((m, r), dtype=dy.dtype, device=dy.device)
    st = load().nf4_lora_da(dy.data_ptr(), m, n, dy.stride(0), b.data_ptr(), r, float(scale),
                            da.data_ptr(), _code(dy.dtype), stream_of(dy))
    check(st, "nf4_lora_da")
    return da


def lora_wgrad(u: torch.Tensor, v: torch.Tensor, scale: float, transpose_out: bool) -> torch.Tensor:
    """scale * U[M, P]^T @ V[M, r] in fp32: [P, r], or [r, P] when transpose_out."""
    _check_device(u, v)
    m, p = u.shape
    r = v.shape[1]
    out = torch.empty((r, p) if transpose_out else (p, r), dtype=torch.float32, device=u.device)
    lib = load()
    ws_bytes = lib.nf4_lora_wgrad_workspace(m, p, r)
    ws = _workspace(ws_bytes, u.device)
    st = lib.nf4_lora_wgrad(u.data_ptr() if m else None, m, p, u.stride(0),
                            v.data_ptr() if m else None, r, float(scale), out.data_ptr(),
                            int(transpose_out), _code(u.dtype),
                            ws.data_ptr() if ws is not None else None, ws_bytes, stream_of(u))
    check(st, "nf4_lora_wgrad")
    return out


def _pair(gate, up):
    if tuple(gate[1].shape) != tuple(up[1].shape):
        raise ValueError("gate and up weights must have the same shape")
    return _descs([gate, up])


def linear_swiglu_fwd(x: torch.Tensor, gate, up, out: torch.Tensor | None = None,
                      tile: int | None = None) -> torch.Tensor:
    """H[M, I] = silu(x @ Wg^T) * (x @ Wu^T), the SwiGLU step in the gate|up GEMM's epilogue.
    `gate`, `up`: (packed, quant_state) pairs of equal shape [I, K]; `tile` pins the tiling."""
    _check_device(x)
    m = x.shape[0]
    inter = int(gate[1].shape[0])
    if out is None:
        out = torch.empty((m, inter), dtype=x.dtype, device=x.device)
    arr = _pair(gate, up)
    if tile is not None:
        st = load().nf4_linear_swiglu_tiled(x.data_ptr() if m else None, m, x.stride(0), arr,
                                            out.data_ptr(), out.stride(0), None, 0,
                                            _code(x.dtype), stream_of(x), 0, int(tile))
        check(st, "nf4_linear_swiglu_tiled")
        return out
    st = load().nf4_linear_swiglu_fwd(x.data_ptr() if m else None, m, x.stride(0), arr,
                                      out.data_ptr(), out.stride(0), _code(x.dtype), stream_of(x))
    check(st, "nf4_linear_swiglu_fwd")
    return out


def linear_swiglu_bwd(x: torch.Tensor, gate, up, d_hidden: torch.Tensor,
                      out: torch.Tensor | None = None, tile: int | None = None) -> torch.Tensor:
    """dGU[M, 2I] (dgate | dup) from d_hidden [M, I] and gate/up recomputed from x inside the
    GEMM; the input of linear_dx over the stacked (gate, up) pair."""
    _check_device(x, d_hidden)
    m = x.shape[0]
    inter = int(gate[1].shape[0])
    if tuple(d_hidden.shape) != (m, inter) or d_hidden.stride(1) != 1:
        raise ValueError("d_hidden must be a row-contiguous [M, I] tensor")
    if out is None:
        out = torch.empty((m, 2 * inter), dtype=x.dtype, device=x.device)
    arr = _pair(gate, up)
    if tile is not None:
        st = load().nf4_linear_swiglu_tiled(x.data_ptr() if m else None, m, x.stride(0), arr,
                                            out.data_ptr(), out.stride(0), d_hidden.data_ptr(),
                                            d_hidden.stride(0), _code(x.dtype), stream_of(x), 1,
                                            int(tile))
        check(st, "nf4_linear_swiglu_tiled")
        return out
    st = load().nf4_linear_swiglu_bwd(x.data_ptr() if m else None, m, x.stride(0), arr,
                                      d_hidden.data_ptr(), d_hidden.stride(0), out.data_ptr(),
                                      out.stride(0), _code(x.dtype), stream_of(x))
    check(st, "nf4_linear_swiglu_bwd")
    return out


def swiglu_fwd(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for two [M, I] views with equal row stride (e.g. halves of gate|up)."""
    _check_device(gate, up)
    rows, cols = gate.shape
    if up.stride(0) != gate.stride(0) or gate.stride(1) != 1 or up.stride(1) != 1:
        raise ValueError("gate and up must be row-contiguous views with one row stride")
    out = torch.empty((rows, cols), dtype=gate.dtype, device=gate.device)
    st = load().nf4_swiglu_fwd(gate.data_ptr(), up.data_ptr(), gate.stride(0), out.data_ptr(),
                               out.stride(0), rows, cols, _code(gate.dtype), stream_of(gate))
    check(st, "nf4_swiglu_fwd")
    return out


def swiglu_bwd(grad: torch.Tensor, gate: torch.Tensor, up: torch.Tensor,
               dgate: torch.Tensor, dup: torch.Tensor) -> None:
    """dgate, dup (row-strided like gate/up; may be gate/up themselves) from grad [M, I]."""
    _check_device(grad, gate, up)
    rows, cols = gate.shape
    st = load().nf4_swiglu_bwd(grad.data_ptr(), grad.stride(0), gate.data_ptr(), up.data_ptr(),
                               gate.stride(0), dgate.data_ptr(), dup.data_ptr(), rows, cols,
                               _code(gate.dtype), stream_of(gate))
    check(st, "nf4_swiglu_bwd")


def bias_grad(dy: torch.Tensor) -> torch.Tensor:
    """Column sums of dY [M, N] in fp32."""
    _check_device(dy)
    m, n = dy.shape
    out = torch.empty(n, dtype=torch.float32, device=dy.device)
    st = load().nf4_bias_grad(dy.data_ptr() if m else None, m, n, dy.stride(0), out.data_ptr(),
                              _code(dy.dtype), stream_of(dy))
    check(st, "nf4_bias_grad")
    return out


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(t, cols):
    if t is not None and (t.dim() != 2 or t.shape[1] != cols or not t.is_contiguous()):
        raise ValueError("norm operands are contiguous [rows, cols] tensors")


def _gemm_dtype(x, *others, dtype=None):
    """The GEMM dtype of a norm call: `dtype`, else the first 16-bit operand's, else x's."""
    if dtype is None:
        for t in (*others, x):
            if t is not None and t.dtype in (torch.float16, torch.bfloat16):
                dtype = t.dtype
                break
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("the norm kernels compute float16 or bfloat16 outputs")
    if x.dtype not in (dtype, torch.float32):
        raise ValueError("the residual stream x is float32 or the GEMM dtype")
    return dtype


def _as_u8(keep):
    keep = keep.contiguous()
    return keep.view(torch.uint8) if keep.dtype == torch.bool else keep.to(torch.uint8)


def add_rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, d: torch.Tensor | None = None,
                dtype=None, keep_q: torch.Tensor | None = None, keep_v: torch.Tensor | None = None,
                rows: torch.Tensor | None = None, packed: torch.Tensor | None = None,
                scale_q: float = 1.0, scale_v: float = 1.0):
    """RMSNorm of the residual stream x (+ d) (layer.py:92-132, 683-715): returns (y, rstd), y in
    the GEMM dtype (`dtype`, default d's or x's) and rstd fp32 [rows].  x is fp32 or the GEMM
    dtype, d the GEMM dtype.  With LoRA dropout also the dropout inputs y * keep * scale:
      keep_q, keep_v (bool or 0/1 uint8 [*, cols], read at row rows[r], or r when rows is None)
        -> (y, rstd, oq, ov, packed), packed the masks 8 per byte ([rows, 2 * cols / 8] uint8,
           q's bytes then v's; bit k of byte j = element 8 j + k);
      packed -> (y, rstd, oq, ov)."""
    _check_device(x, d, w, keep_q, keep_v, rows, packed)
    dtype = _gemm_dtype(x, d, dtype=dtype)
    n, cols = x.shape
    _rows(x, cols)
    _rows(d, cols)
    y = torch.empty((n, cols), dtype=dtype, device=x.device)
    rstd = torch.empty(n, dtype=torch.float32, device=x.device)
    w = w.to(torch.float32).contiguous()
    mode, oq, ov, kq, kv = 0, None, None, None, None
    if keep_q is not None:
        if keep_v is None or packed is not None:
            raise ValueError("give keep_q and keep_v (mode 1) or packed (mode 2)")
        kq, kv = _as_u8(keep_q), _as_u8(keep_v)
        if kq.shape[-1] != cols or kv.shape != kq.shape:
            raise ValueError("keep masks are [*, cols]")
        if rows is not None:
            rows = rows.to(torch.int64).contiguous()
            if rows.numel() != n:
                raise ValueError("rows holds one mask row per token")
        elif kq.shape[0] < n:
            raise ValueError("keep masks need a row per token")
        packed = torch.empty((n, 2 * (cols // 8)), dtype=torch.uint8, device=x.device)
        mode = 1
    elif packed is not None:
        if tuple(packed.shape) != (n, 2 * (cols // 8)) or packed.dtype != torch.uint8:
            raise ValueError("packed masks are uint8 [rows, 2 * cols / 8]")
        packed = packed.contiguous()
        mode = 2
    if mode:
        oq, ov = torch.empty_like(y), torch.empty_like(y)
    keep_rows = int(kq.shape[0]) if kq is not None else 0
    st = load().nf4_add_rmsnorm(_p(x), DTYPE_CODE[x.dtype], _p(d), _p(w), _p(y), _p(rstd), _p(kq),
                                _p(kv), _p(rows) if mode == 1 else None, keep_rows, _p(packed),
                                mode,
                                float(scale_q), float(scale_v), _p(oq), _p(ov), n, cols,
                                float(eps), _code(dtype), stream_of(x))
    check(st, "nf4_add_rmsnorm")
    if mode == 1:
        return y, rstd, oq, ov, packed
    if mode == 2:
        return y, rstd, oq, ov
    return y, rstd


def rmsnorm_bwd(x: torch.Tensor, w: torch.Tensor, rstd: torch.Tensor, dy=None, d=None, dres=None,
                dq=None, dv=None, packed=None, scale_q: float = 1.0, scale_v: float = 1.0,
                dtype=None) -> torch.Tensor:
    """dX of add_rmsnorm (layer.py:135-164, 718-730) from the output's gradient dy and LoRA's
    dropout branches dq, dv (masked with the packed keep bits of the forward), plus the
    residual gradient dres; dX and dres in x's dtype (fp32 for an fp32 residual stream), the
    other gradients in the GEMM dtype."""
    _check_device(x, w, rstd, dy, d, dres, dq, dv, packed)
    dtype = _gemm_dtype(x, dy, dq, d, dtype=dtype)
    n, cols = x.shape
    for t in (x, dy, d, dres, dq, dv):
        _rows(t, cols)
    if dres is not None and dres.dtype != x.dtype:
        raise ValueError("dres has the residual stream's dtype")
    if (dq is None) != (dv is None) or (dq is not None and packed is None):
        raise ValueError("dq and dv come together, with the packed masks")
    if packed is not None:
        if tuple(packed.shape) != (n, 2 * (cols // 8)) or packed.dtype != torch.uint8:
            raise ValueError("packed masks are uint8 [rows, 2 * cols / 8]")
        packed = packed.contiguous()
    dx = torch.empty_like(x)
    w = w.to(torch.float32).contiguous()
    st = load().nf4_rmsnorm_bwd(_p(dy), _p(dq), _p(dv), _p(packed), float(scale_q),
                                float(scale_v), _p(x), DTYPE_CODE[x.dtype], _p(d), _p(w), _p(rstd),
                                _p(dres), _p(dx), n, cols, _code(dtype), stream_of(x))
    check(st, "nf4_rmsnorm_bwd")
    return dx


def qkv_rope(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, n_heads: int, n_kv: int,
             head_dim: int, caches: bool = True):
    """(q, k, v[, k_cache, v_cache]) from the finished q|k|v projection [tokens, ...]: rotary
    embedding on q and k, k and v expanded to [tokens, n_heads, head_dim]."""
    _check_device(qkv, cos, sin)
    tokens = qkv.shape[0]
    if qkv.stride(1) != 1:
        raise ValueError("qkv rows must be contiguous")
    cos, sin = cos.to(torch.float32).contiguous(), sin.to(torch.float32).contiguous()
    e = lambda h: torch.empty(tokens, h, head_dim, dtype=qkv.dtype, device=qkv.device)  # noqa: E731
    q, k, v = e(n_heads), e(n_heads), e(n_heads)
    kc, vc = (e(n_kv), e(n_kv)) if caches else (None, None)
    st = load().nf4_qkv_rope(_p(qkv), qkv.stride(0), _p(cos), _p(sin), _p(q), _p(k), _p(v), _p(kc),
                             _p(vc), tokens, n_heads, n_kv, head_dim, _code(qkv.dtype),
                             stream_of(qkv))
    check(st, "nf4_qkv_rope")
    return (q, k, v, kc, vc) if caches else (q, k, v)


def qkv_rope_bwd(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, n_kv: int) -> torch.Tensor:
    """d(q|k|v) [tokens, (n_heads + 2 n_kv) head_dim] from the gradients of qkv_rope's q, k, v
    ([tokens, n_heads, head_dim] each)."""
    _check_device(dq, dk, dv, cos, sin)
    tokens, n_heads, head_dim = dq.shape
    for t in (dq, dk, dv):
        if tuple(t.shape) != (tokens, n_heads, head_dim) or not t.is_contiguous():
            raise ValueError("dq, dk, dv are contiguous [tokens, n_heads, head_dim] tensors")
    cos, sin = cos.to(torch.float32).contiguous(), sin.to(torch.float32).contiguous()
    out = torch.empty(tokens, (n_heads + 2 * n_kv) * head_dim, dtype=dq.dtype, device=dq.device)
    st = load().nf4_qkv_rope_bwd(_p(dq), _p(dk), _p(dv), _p(cos), _p(sin), _p(out), out.stride(0),
                                 tokens, n_heads, n_kv, head_dim, _code(dq.dtype), stream_of(dq))
    check(st, "nf4_qkv_rope_bwd")
    return out


def _on_its_device(fn):
    """Runs a call (or method) with the device of its first parameter (a tensor, or a list of them) as the
    current one: launches go to the current device, and the handle of another's default stream is none of
    its own.  Calls without such a tensor are refused by `fn` itself."""
    names = list(inspect.signature(fn).parameters)
    at = int(names[0] == "self")

    @functools.wraps(fn)
    def call(*args, **kw):
        if _devices() < 2:
            return fn(*args, **kw)
        t = args[at] if len(args) > at else kw.get(names[at])
        if isinstance(t, (list, tuple)):
            t = t[0] if t else None
        if not getattr(t, "is_cuda", False) or t.get_device() == torch.cuda.current_device():
            return fn(*args, **kw)
        with torch.cuda.device(t.get_device()):
            return fn(*args, **kw)

    return call


@functools.lru_cache(maxsize=None)
def _devices() -> int:
    return torch.cuda.device_count()


@_on_its_device
def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, heads: int, head_dim: int,
         inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """The first `heads` heads of every row of x [tokens, *] rotated as qkv_rope does (cos, sin
    [tokens, head_dim]), or by the transposed rotation (`inverse`: gradients), into `out`
    [tokens, >= heads head_dim] (a new [tokens, heads head_dim] tensor; may be x itself)."""
    _check_device(x, cos, sin, out)
    tokens, cols = x.shape[0], heads * head_dim
    if out is None:
        out = torch.empty((tokens, cols), dtype=x.dtype, device=x.device)
    for t in (x, out):
        if t.dim() != 2 or t.shape[0] != tokens or t.shape[1] < cols or t.stride(1) != 1 \
                or t.dtype != x.dtype or t.device != x.device:
            raise ValueError("x and out are row-contiguous [tokens, >= heads * head_dim] tensors of "
                             "one dtype and device")
    if tuple(cos.shape) != (tokens, head_dim) or cos.shape != sin.shape or \
            not x.device == cos.device == sin.device:
        raise ValueError("cos and sin are [tokens, head_dim] on x's device")
    cos, sin = cos.to(torch.float32).contiguous(), sin.to(torch.float32).contiguous()
    st = load().nf4_rope(x.data_ptr(), x.stride(0), cos.data_ptr(), sin.data_ptr(), out.data_ptr(),
                         out.stride(0), tokens, heads, head_dim, int(inverse), _code(x.dtype),
                         stream_of(x))
    check(st, "nf4_rope")
    return out


def make_lora(seg: int, rank: int, scale: float, t=None, b=None, a=None, da=None) -> NF4Lora:
    """The adapter struct of segment `seg`.  It holds raw pointers, so it also keeps references
    to its tensors: a temporary passed here (t=lora_xa(...)) stays allocated while the struct
    lives, instead of returning to torch's cache where the call's own output could reuse it."""
    lo = NF4Lora(seg=seg, rank=rank, scale=float(scale),
                 t=t.data_ptr() if t is not None else None,
                 b=b.data_ptr() if b is not None else None,
                 a=a.data_ptr() if a is not None else None,
                 da=da.data_ptr() if da is not None else None)
    lo._tensors = (t, b, a, da)
    return lo


__all__ = ["dequant", "linear_fwd", "linear_dx", "lora_xa", "lora_da", "lora_wgrad",
           "swiglu_fwd", "swiglu_bwd", "bias_grad", "make_lora", "GEMM_DTYPES", "_lib"]


def lora_job(inp: torch.Tensor, w: torch.Tensor, out: torch.Tensor, scale: float = 1.0,
             transpose_out: bool = False) -> NF4LoraJob:
    """One job of the multi LoRA launches: `inp` [M, cols] (any row stride), `w` the small
    operand, `out` the result.  Like make_lora's struct, the job holds references to its
    tensors, so a temporary passed here stays allocated while the job lives."""
    _check_device(inp, w, out)
    job = NF4LoraJob(in_=inp.data_ptr(), ld=inp.stride(0), cols=inp.shape[1], w=w.data_ptr(),
                     out=out.data_ptr(), scale=float(scale), transpose_out=int(transpose_out))
    job._tensors = (inp, w, out)
    return job


def _jobs(jobs):
    return (NF4LoraJob * len(jobs))(*jobs), len(jobs)


def lora_xa_multi(jobs, m: int, rank: int, dtype, stream_tensor: torch.Tensor):
    """t_j = in_j @ A_j^T for every job, one launch."""
    arr, n = _jobs(jobs)
    check(load().nf4_lora_xa_multi(arr, n, m, rank, _code(dtype), stream_of(stream_tensor)),
          "nf4_lora_xa_multi")


def lora_da_multi(jobs, m: int, rank: int, dtype, stream_tensor: torch.Tensor):
    """da_j = scale_j * in_j @ B_j for every job, one launch."""
    arr, n = _jobs(jobs)
    check(load().nf4_lora_da_multi(arr, n, m, rank, _code(dtype), stream_of(stream_tensor)),
          "nf4_lora_da_multi")


def lora_ax_multi(jobs, m: int, rank: int, dtype, stream_tensor: torch.Tensor):
    """out_j = scale_j * da_j @ A_j ([M, K]) for every job (lora_ax_job), one launch."""
    arr, n = _jobs(jobs)
    check(load().nf4_lora_ax_multi(arr, n, m, rank, _code(dtype), stream_of(stream_tensor)),
          "nf4_lora_ax_multi")


def lora_ax_job(da: torch.Tensor, a: torch.Tensor, out: torch.Tensor, scale: float = 1.0):
    """A job of lora_ax_multi: da [M, rank] (any row stride), A [rank, K] contiguous, out
    [M, K] contiguous."""
    _check_device(da, a, out)
    if not a.is_contiguous() or not out.is_contiguous() or da.stride(-1) != 1:
        raise ValueError("lora_ax: A and out contiguous, da rows contiguous")
    if out.shape[1] != a.shape[1] or da.shape[1] != a.shape[0] or out.shape[0] != da.shape[0]:
        raise ValueError("lora_ax: da [M, r], A [r, K], out [M, K]")
    return NF4LoraJob(in_=da.data_ptr(), ld=da.stride(0), cols=a.shape[1], w=a.data_ptr(),
                      out=out.data_ptr(), scale=float(scale), transpose_out=0)


def lora_wgrad_multi(jobs, m: int, rank: int, dtype, stream_tensor: torch.Tensor):
    """out_j = scale_j * in_j^T @ V_j (fp32) for every job: one launch over M when the rows
    allow it, else row-chunk partials and a final pass through the workspace."""
    arr, n = _jobs(jobs)
    lib = load()
    nbytes = lib.nf4_lora_wgrad_multi_workspace(arr, n, m, rank)
    ws = _workspace(nbytes, stream_tensor.device)
    check(lib.nf4_lora_wgrad_multi(arr, n, m, rank, _code(dtype),
                                   ws.data_ptr() if ws is not None else None, nbytes,
                                   stream_of(stream_tensor)), "nf4_lora_wgrad_multi")


# ------------------------------------------------- int8 input gradients (off the parity path)

def int8_colscale(weights, dtype=torch.float16) -> torch.Tensor:
    """fp32 [cols]: max(largest |W[:, c]|, 1e-20) / 127 over the stacked weights, W rounded to
    `dtype` (the fixed column scales of the transposed int8 weights)."""
    arr = _descs(weights)
    lib = load()
    dev = weights[0][0].device
    cols = int(weights[0][1].shape[1])
    out = torch.empty(cols, dtype=torch.float32, device=dev)
    nb = lib.nf4_int8_colscale_workspace(arr, len(weights))
    ws = _workspace(nb, dev)
    check(lib.nf4_int8_colscale(arr, len(weights), out.data_ptr(), _code(dtype),
                                ws.data_ptr() if ws is not None else None, nb, stream_of(out)),
          "nf4_int8_colscale")
    return out


def int8_weight_t(weights, scale: torch.Tensor) -> torch.Tensor:
    """int8 [cols, sum rows]: the stacked weights transposed, divided by the column scales."""
    arr = _descs(weights)
    rows = sum(int(qs.shape[0]) for _, qs in weights)
    cols = int(weights[0][1].shape[1])
    q = torch.empty((cols, rows), dtype=torch.int8, device=scale.device)
    check(load().nf4_int8_weight_t(arr, len(weights), scale.data_ptr(), q.data_ptr(), rows,
                                   stream_of(q)), "nf4_int8_weight_t")
    return q


def int8_weight_rows(weights):
    """(int8 [sum rows, cols], fp32 [sum rows]): the stacked weights with one scale per row."""
    arr = _descs(weights)
    rows = sum(int(qs.shape[0]) for _, qs in weights)
    cols = int(weights[0][1].shape[1])
    dev = weights[0][0].device
    q = torch.empty((rows, cols), dtype=torch.int8, device=dev)
    s = torch.empty(rows, dtype=torch.float32, device=dev)
    check(load().nf4_int8_weight_rows(arr, len(weights), q.data_ptr(), cols, s.data_ptr(),
                                      stream_of(q)), "nf4_int8_weight_rows")
    return q, s


def int8_rows(x: torch.Tensor):
    """(int8 [M, N], fp32 [M]): one int8 row per row of x with scale largest |x| / 127."""
    _check_device(x)
    m, n = x.shape
    q = torch.empty((m, n), dtype=torch.int8, device=x.device)
    s = torch.empty(m, dtype=torch.float32, device=x.device)
    code = _code(x.dtype, (torch.float16, torch.bfloat16, torch.float32))
    check(load().nf4_int8_rows(x.data_ptr() if m else None, m, n, x.stride(0), q.data_ptr(), n,
                               s.data_ptr(), code, stream_of(x)), "nf4_int8_rows")
    return q, s


def int8_gemm(a: torch.Tensor, b: torch.Tensor, sa: torch.Tensor | None = None,
              sb: torch.Tensor | None = None, out_dtype=None) -> torch.Tensor:
    """a [M, K] . b [N, K]^T over int8: int32 sums (out_dtype None) or
    round(fp32(C) * sa[m] * sb[n]) in out_dtype (float16 / bfloat16)."""
    _check_device(a, b)
    m, k = a.shape
    n = b.shape[0]
    lib = load()
    if out_dtype is None:
        out = torch.empty((m, n), dtype=torch.int32, device=a.device)
        code = _lib.NF4_I32
    else:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
        code = _code(out_dtype)
    nb = lib.nf4_int8_gemm_workspace(m, n, k)
    ws = _workspace(nb, a.device)
    check(lib.nf4_int8_gemm(a.data_ptr(), m, a.stride(0), b.data_ptr(), n, b.stride(0), k,
                            sa.data_ptr() if sa is not None else None,
                            sb.data_ptr() if sb is not None else None, out.data_ptr(),
                            out.stride(0), code, ws.data_ptr() if ws is not None else None, nb,
                            stream_of(a)), "nf4_int8_gemm")
    return out


def int8_swiglu_bwd(acc: torch.Tensor, sd: torch.Tensor, cs: torch.Tensor,
                    gu: torch.Tensor):
    """(int8 [M, 2I], fp32 [M]): SwiGLU backward of the int32 sums acc [M, I] (scaled by
    sd[m] cs[j]) with the saved gate | up [M, 2I], requantized with one scale per row."""
    _check_device(acc, sd, cs, gu)
    m, inter = acc.shape
    q = torch.empty((m, 2 * inter), dtype=torch.int8, device=acc.device)
    sq = torch.empty(m, dtype=torch.float32, device=acc.device)
    check(load().nf4_int8_swiglu_bwd(acc.data_ptr(), m, inter, acc.stride(0), sd.data_ptr(),
                                     cs.data_ptr(), gu.data_ptr(), gu.stride(0), q.data_ptr(),
                                     2 * inter, sq.data_ptr(), _code(gu.dtype), stream_of(acc)),
          "nf4_int8_swiglu_bwd")
    return q, sq


# ------------------------------------------------- serving: a paged cache, attention over it

class PagedKV:
    """One layer's paged key/value cache and the step's sequences, as the paged calls take them.

    `k_pages`, `v_pages`: [pages, page_size, n_kv, head_dim] float16 or bfloat16 views of one
    layout (any order of the first three dimensions in memory: head-major pages come as
    `pages.transpose(1, 2)`); `table`: int32 [batch, width], the page of every page_size
    positions of a sequence (an entry outside the cache, -1 say, names no page: appends there are
    dropped, its keys are not seen); `lens`: int32 [batch], each sequence's length with the
    step's own tokens.  The layout is checked and packed once; the tensors' contents are read on
    the device by every call, so a program updates `table` and `lens` in place between steps (a
    captured graph then replays with the new lengths).  Layers of a model share `table` and
    `lens`."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor):
        _check_device(k_pages, v_pages, table, lens)
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError("k_pages and v_pages are [pages, page_size, n_kv, head_dim] of one dtype")
        # (a dimension of size one has no stride that matters)
        strides, v_strides = ([st if n > 1 else 0 for n, st in zip(t.shape, t.stride())]
                              for t in (k_pages, v_pages))
        if strides != v_strides or k_pages.stride(3) != 1:
            raise ValueError("k_pages and v_pages share their strides, head_dim contiguous")
        if table.dim() != 2 or table.dtype != torch.int32 or table.stride(1) != 1:
            raise ValueError("table is an int32 [batch, width] tensor with contiguous rows")
        if lens.dtype != torch.int32 or tuple(lens.shape) != (table.shape[0],) \
                or not lens.is_contiguous():
            raise ValueError("lens is a contiguous int32 [batch] tensor")
        if len({t.device for t in (k_pages, v_pages, table, lens)}) != 1:
            raise ValueError("the cache, its table and lens are on one device")
        self.k_pages, self.v_pages, self.table, self.lens = k_pages, v_pages, table, lens
        self.dtype, self.code = k_pages.dtype, _code(k_pages.dtype)
        self.batch, self.width = (int(d) for d in table.shape)
        pages, self.page_size, self.n_kv, self.head_dim = (int(d) for d in k_pages.shape)
        # (one row's stride says nothing; rows that overlap are no rows of `width` entries)
        ld_table = int(table.stride(0)) if self.batch > 1 else self.width
        if ld_table < self.width:
            raise ValueError("the table's rows are at least its width apart (a row that all sequences "
                             "share is copied for each: row.repeat(batch, 1))")
        self.desc = NF4PagedKV(
            k_pages.data_ptr(), v_pages.data_ptr(), *strides[:3], table.data_ptr(), ld_table, lens.data_ptr(), pages,
            self.page_size, self.width, self.batch, self.n_kv, self.head_dim)
        self.ref = ctypes.byref(self.desc)
        self.index = k_pages.get_device()


def _check_cu(cu_q, cache: PagedKV):
    if cu_q is None:
        return None
    if cu_q.get_device() != cache.index or cu_q.dtype != torch.int32 \
            or tuple(cu_q.shape) != (cache.batch + 1,) or not cu_q.is_contiguous():
        raise ValueError("cu_q is a contiguous int32 [batch + 1] tensor on the cache's device")
    return cu_q.data_ptr()


def paged_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, cache: PagedKV,
                 cu_q: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotated q [tokens, n_heads, head_dim] of a step's q|k|v projection (`qkv`
    [tokens, (n_heads + 2 n_kv) head_dim], rows any multiple of 8 apart); its rotated k and its v
    go to the cache, the i-th of a sequence's n tokens to position lens - n + i.  `cos`, `sin`:
    fp32 [positions, head_dim / 2] (rope_table); `cu_q`: int32 offsets of the sequences' tokens,
    None when each brings tokens / batch."""
    dim, kv = cache.head_dim, cache.n_kv
    if qkv.dim() != 2 or qkv.dtype != cache.dtype or qkv.stride(1) != 1:
        raise ValueError("qkv is a row-contiguous [tokens, (n_heads + 2 n_kv) head_dim] tensor of "
                         "the cache's dtype")
    if not qkv.get_device() == cos.get_device() == sin.get_device() == cache.index:
        raise ValueError("qkv, cos and sin are on the cache's device")
    tokens, cols = qkv.shape
    heads = cols // dim - 2 * kv
    if heads < 1 or heads % kv or cols % dim:
        raise ValueError("qkv has (n_heads + 2 n_kv) head_dim columns, n_heads a multiple of the "
                         "cache's n_kv")
    rope = cos.shape
    if len(rope) != 2 or rope[1] * 2 != dim or rope != sin.shape or cos.dtype != torch.float32 \
            or sin.dtype != torch.float32 or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin are contiguous fp32 [positions, head_dim / 2] tables")
    if out is None:
        out = qkv.new_empty((tokens, heads, dim))
    else:
        _check_out(out, (tokens, heads, dim), qkv)
    st = load().nf4_paged_append(cache.ref, qkv.data_ptr(), qkv.stride(0) if tokens > 1 else cols,
                                 cos.data_ptr(), sin.data_ptr(), rope[0],
                                 None if cu_q is None else _check_cu(cu_q, cache), out.data_ptr(),
                                 tokens, heads, cache.code, stream_of(qkv))
    if st:
        check(st, "nf4_paged_append")
    return out


def _check_out(out, shape, like):
    if tuple(out.shape) != shape or out.dtype != like.dtype or out.device != like.device \
            or not out.is_contiguous():
        raise ValueError(f"out is a contiguous {list(shape)} tensor of the input's dtype")


def _attention(q, cache, shared, cu_q, scale, window, sinks, max_q, max_len, out, lse):
    if q.dim() != 3 or q.dtype != cache.dtype or q.shape[2] != cache.head_dim or q.stride(2) != 1:
        raise ValueError("q is [tokens, n_heads, head_dim] of the cache's dtype, head_dim contiguous")
    if q.get_device() != cache.index:
        raise ValueError("q is on the cache's device")
    tokens, heads, dim = q.shape
    if heads < 1 or heads % cache.n_kv:
        raise ValueError("n_heads is a multiple of the cache's n_kv")
    if out is None:
        out = q.new_empty((tokens, heads, dim))
    else:
        _check_out(out, (tokens, heads, dim), q)
    stats = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if lse else None
    lib = load()
    cu = None if cu_q is None else _check_cu(cu_q, cache)
    window, sinks, max_q, max_len = window or 0, sinks or 0, max_q or 0, max_len or 0
    nbytes = lib.nf4_paged_attn_workspace(cache.ref, cu, tokens, heads, window, sinks, shared,
                                          max_q, max_len)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    st = lib.nf4_paged_attn(cache.ref, q.data_ptr(), q.stride(0) if tokens > 1 else 0,
                            q.stride(1) if heads > 1 else 0, cu, out.data_ptr(), _p(stats),
                            tokens, heads, dim ** -0.5 if scale is None else scale,
                            window, sinks, shared, max_q, max_len, cache.code, _p(ws), nbytes,
                            stream_of(q))
    if st:
        check(st, "nf4_paged_attn")
    return (out, stats) if lse else out


def paged_attention(q: torch.Tensor, cache: PagedKV, cu_q: torch.Tensor | None = None,
                    scale: float | None = None, window: int = 0, sinks: int = 0, max_q: int = 0,
                    max_len: int = 0, out: torch.Tensor | None = None, lse: bool = False):
    """Causal attention of a step's queries over the cache: out [tokens, n_heads, head_dim] (and
    with `lse` the fp32 log-sum-exp [tokens, n_heads]).  The i-th of a sequence's n tokens is at
    position p = lens - n + i and sees key j <= p where window == 0, j > p - window or j < sinks;
    a query that sees nothing gives zeros and -inf.  `scale`: head_dim ** -0.5 by default.
    `max_q`, `max_len`: the longest run of new tokens and the longest length, as far as the host
    knows them; they only choose the launch shape (unknown: from the tensors' shapes), and a
    sequence beyond them is still right."""
    return _attention(q, cache, 0, cu_q, scale, window, sinks, max_q, max_len, out, lse)


def shared_prefix_attention(q: torch.Tensor, cache: PagedKV, shared: int,
                            cu_q: torch.Tensor | None = None, scale: float | None = None,
                            window: int = 0, sinks: int = 0, max_q: int = 0, max_len: int = 0,
                            out: torch.Tensor | None = None, lse: bool = False):
    """paged_attention for a batch whose sequences start with the same `shared` positions: their
    keys are read once for all sequences, through the first row of the cache's table (which must
    name their pages); every other position is the sequence's own, as in paged_attention."""
    return _attention(q, cache, int(shared), cu_q, scale, window, sinks, max_q, max_len, out, lse)


def rope_table(positions: int, head_dim: int, base: float, device):
    """(cos, sin) fp32 [positions, head_dim / 2] of paged_append: angles
    position * base ** (-2 i / head_dim), formed in 64 bits, so that far positions are as exact
    as near ones."""
    inv = base ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return ang.cos().float().to(device), ang.sin().float().to(device)


# ------------------------------- training: attention of a packed batch, dropout without masks

def _empty(like):
    """A contiguous tensor like this one (1.2 us of the host's; new_empty 1.6, torch.empty 2.1)."""
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def _attn_desc(q, k, v, cu_seqlens, scale, window, max_len):
    shape, kv_shape, dtype, dev = q.shape, k.shape, q.dtype, q.get_device()
    if len(shape) != 3 or len(kv_shape) != 3 or kv_shape != v.shape or shape[0] != kv_shape[0] \
            or shape[2] != kv_shape[2]:
        raise ValueError("q is [tokens, n_heads, head_dim], k and v [tokens, n_kv, head_dim]")
    if not dtype == k.dtype == v.dtype:
        raise ValueError("q, k and v have one dtype")
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if not qs[2] == ks[2] == vs[2] == 1:
        raise ValueError("q, k and v have head_dim contiguous")
    if dev < 0 or not dev == k.get_device() == v.get_device():
        raise ValueError("q, k and v are on one cuda device")
    tokens, heads, dim = shape
    n_kv = kv_shape[1]
    if heads < 1 or n_kv < 1 or heads % n_kv:
        raise ValueError("n_heads is a multiple of n_kv")
    cu, batch = None, 1
    if cu_seqlens is not None:
        offsets = cu_seqlens.shape
        if cu_seqlens.get_device() != dev or cu_seqlens.dtype != torch.int32 \
                or len(offsets) != 1 or offsets[0] < 1 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens is a contiguous int32 [batch + 1] tensor on q's device")
        cu, batch = cu_seqlens.data_ptr(), offsets[0] - 1
    return NF4Attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
                   cu, tokens, window or 0, max_len or 0, batch, heads, n_kv, dim,
                   dim ** -0.5 if scale is None else scale, _code(dtype))


@_on_its_device
def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  cu_seqlens: torch.Tensor | None = None, scale: float | None = None,
                  window: int = 0, max_len: int = 0, out: torch.Tensor | None = None):
    """Causal attention of a packed batch: (out [tokens, n_heads, head_dim], stats fp32
    [tokens, n_heads, 2]) of q [tokens, n_heads, head_dim], k and v [tokens, n_kv, head_dim] (any
    strides of whole 16 bytes, head_dim contiguous: columns of the projection's output as they are).  `cu_seqlens`:
    int32 offsets of the sequences on the device (None: one sequence); row i of one sees its rows
    j <= i where window == 0 or j > i - window.  stats are (m, l): with t = scale log2(e) q.k, m =
    max t and l = sum 2^(t - m); a row behind the last sequence gives zeros and (0, 0).  `max_len`:
    the longest sequence as the host knows it; it only chooses the launch shape."""
    desc = _attn_desc(q, k, v, cu_seqlens, scale, window, max_len)
    tokens, heads, dim = q.shape
    if out is None:
        out = _empty(q)
    else:
        _check_out(out, (tokens, heads, dim), q)
    stats = q.new_empty(tokens, heads, 2, dtype=torch.float32)
    lib, ref = load(), ctypes.byref(desc)
    nbytes = lib.nf4_attn_fwd_workspace(ref)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    st = lib.nf4_attn_fwd(ref, out.data_ptr(), stats.data_ptr(), _p(ws), nbytes, stream_of(q))
    if st:
        check(st, "nf4_attn_fwd")
    return out, stats


def _grad(t, shape, like, what):
    if t.shape != shape or t.dtype != like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{what} is a {list(shape)} tensor of q's dtype, head_dim contiguous")
    tok, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{what} is a {list(shape)} tensor of q's dtype, head_dim contiguous")
    return NF4Grad(t.data_ptr(), tok, head)


@_on_its_device
def attention_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  out: torch.Tensor, stats: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                  scale: float | None = None, window: int = 0, max_len: int = 0, grads=None):
    """(dq, dk, dv) of attention_fwd from the output's gradient, with the forward pass's `out` and
    `stats` and its other arguments.  dk and dv are summed over the query heads that share a head.
    `grads`: (dq, dk, dv) tensors to write, of any strides (column slices of one buffer), none of
    them an input.  Rows of no sequence get zeros."""
    desc = _attn_desc(q, k, v, cu_seqlens, scale, window, max_len)
    shape, kv_shape = q.shape, k.shape
    args = [_grad(dout, shape, q, "dout")]
    if grads is None:
        dq, dk, dv = grads = _empty(q), _empty(k), _empty(v)
        dim, row = shape[2], kv_shape[1] * shape[2]
        args += (NF4Grad(dq.data_ptr(), shape[1] * dim, dim), NF4Grad(dk.data_ptr(), row, dim),
                 NF4Grad(dv.data_ptr(), row, dim))
    else:
        args += [_grad(t, sh, q, name) for t, sh, name in
                 zip(grads, (shape, kv_shape, kv_shape), ("dq", "dk", "dv"))]
    _check_out(out, shape, q)
    if stats.shape != (*shape[:2], 2) or stats.dtype != torch.float32 \
            or stats.get_device() != q.get_device() or not stats.is_contiguous():
        raise ValueError("stats is the forward pass's fp32 [tokens, n_heads, 2] tensor")
    lib, ref = load(), ctypes.byref(desc)
    nbytes = lib.nf4_attn_bwd_workspace(ref)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    st = lib.nf4_attn_bwd(ref, out.data_ptr(), stats.data_ptr(), *map(ctypes.byref, args), _p(ws),
                          nbytes, stream_of(q))
    if st:
        check(st, "nf4_attn_bwd")
    return tuple(grads)


def _rows_of(t, shape, dtype, index):
    if t.shape != shape or t.dtype != dtype or t.get_device() != index \
            or (t.stride(1) != 1 and shape[1] > 1):
        raise ValueError(f"dropout's tensors are row-contiguous {list(shape)} tensors of one dtype "
                         "and device")


_SITES = range(9)  # (array types are made once: ctypes looks them up by name otherwise)
_PTR_ARRAYS = [ctypes.c_void_p * n for n in _SITES]
_LD_ARRAYS = [ctypes.c_int64 * n for n in _SITES]
_SITE_ARRAYS = [ctypes.c_uint32 * n for n in _SITES]


def _drop_args(tensors, seed, sites, index):
    """(pointers, row strides, site numbers) of the sites' tensors as ctypes arrays, n."""
    if index < 0 or seed.get_device() != index or seed.dtype != torch.int64 \
            or seed.shape != (2,) or not seed.is_contiguous():
        raise ValueError("seed is an int64 [2] tensor (seed, step) on the tensors' cuda device")
    n = len(sites)
    if not 1 <= n <= 8:
        raise ValueError("dropout takes 1 to 8 sites")
    if min(sites) < 0 or max(sites) >> 32:
        raise ValueError("a site is a number of 32 bits")
    return (_PTR_ARRAYS[n](*[t.data_ptr() for t in tensors]),
            _LD_ARRAYS[n](*[t.stride(0) for t in tensors]), _SITE_ARRAYS[n](*sites), n)


@_on_its_device
def dropout(x: torch.Tensor, p: float, seed: torch.Tensor, sites, outs=None) -> list:
    """Dropout without a stored mask: for every site a tensor like x [rows, cols] that holds
    x * 65536 / (65536 - T) where the site keeps the element and 0 where it does not, T =
    floor(65536 p + 1/2).  What is kept is a function of the element's place, the site's number and
    `seed`, an int64 [2] tensor (seed, step) on the device: dropout_bwd with the same ones has the
    same mask.  A program gives every adapter of a model its own site and every step its own `step`
    (seed[1] += 1; a captured graph reads it at each replay)."""
    if x.dim() != 2:
        raise ValueError("x is [rows, cols]")
    shape, dtype, index = x.shape, x.dtype, x.get_device()
    dt = _code(dtype)
    if x.stride(1) != 1 and shape[1] > 1:
        _rows_of(x, shape, dtype, index)  # (refuses)
    if outs is None:
        outs = [_empty(x) for _ in sites]
    else:
        if len(outs) != len(sites):
            raise ValueError("an output for every site")
        for t in outs:
            _rows_of(t, shape, dtype, index)
    ptrs, lds, where, n = _drop_args(outs, seed, sites, index)
    st = load().nf4_dropout(x.data_ptr(), x.stride(0), ptrs, lds, shape[0], shape[1], p,
                            seed.data_ptr(), where, n, dt, stream_of(x))
    if st:
        check(st, "nf4_dropout")
    return outs


@_on_its_device
def dropout_bwd(grads, p: float, seed: torch.Tensor, sites, base: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """dx of dropout: base (None: zeros) plus every site's gradient times its mask and scale, summed
    in fp32 in this order and rounded once.  `out` may be `base`."""
    if not grads or len(grads) != len(sites) or grads[0].dim() != 2:
        raise ValueError("a [rows, cols] gradient for every site")
    g = grads[0]
    shape, dtype, index = g.shape, g.dtype, g.get_device()
    dt = _code(dtype)
    for t in grads:
        _rows_of(t, shape, dtype, index)
    if base is not None:
        _rows_of(base, shape, dtype, index)
    if out is None:
        out = _empty(g)
    elif out is not base:
        _rows_of(out, shape, dtype, index)
    ptrs, lds, where, n = _drop_args(grads, seed, sites, index)
    st = load().nf4_dropout_bwd(ptrs, lds, _p(base), 0 if base is None else base.stride(0),
                                out.data_ptr(), out.stride(0), shape[0], shape[1], p,
                                seed.data_ptr(), where, n, dt, stream_of(g))
    if st:
        check(st, "nf4_dropout_bwd")
    return out
