"""Tensor-level wrappers over the C ABI: torch owns memory and streams, the
library owns every kernel.  Each wrapper validates dtype/device/contiguity,
passes raw pointers plus the current CUDA stream, and raises on any error code.
"""
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import EPI_BIAS, EPI_GELU, EPI_RAW, EPI_RESIDUAL  # noqa: F401  (re-exported)

_status_words = {}


# The current stream of a device, as a pointer; a torch built without CUDA lacks the short way, and imports this module too.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _stream() -> int:
    return _raw_stream(torch.cuda.current_device())


def _same_device(index: Optional[int], name: str) -> None:
    """Every launch goes to the *current* device and its current stream (the C side reads the current
    device for its architecture check and SM count), so a tensor living on another GPU would hand that
    GPU's pointers to a kernel running here.  Reject it before anything is enqueued."""
    cur = torch.cuda.current_device()
    if index is not None and index != cur:
        raise RuntimeError(f"{name} is on cuda:{index} but the current device is cuda:{cur}; "
                           f"call torch.cuda.set_device({index}) (or use `with torch.cuda.device({index})`) first")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 word that kernels write when a bounded wait expires."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _status_words.get(idx)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
        _status_words[idx] = w
    return w


def check_status(device: Optional[torch.device] = None) -> None:
    """Synchronise and raise if any kernel on ``device`` reported a device-side timeout."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    w = status_word(device)
    v = int(w.item())
    if v != 0:
        w.zero_()
        code = _lib.load().samb_decode_status(v)
        raise RuntimeError(f"device status 0x{v & 0xffffffff:08x}: {_lib.error_string(code)}")


def _need(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name}: expected a CUDA tensor (there is no CPU path)")
    if t.dtype != dtype:
        raise RuntimeError(f"{name}: expected {dtype}, got {t.dtype}")
    _same_device(t.device.index, name)


def _rows2d(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 2 or t.stride(1) != 1:
        raise RuntimeError(f"{name}: expected a 2-D tensor with unit inner stride")
    return t


def window_rows(rows: int, grid: int, window: int) -> int:
    """Number of rows of the zero-padded window-partitioned layout."""
    if window == 0:
        return rows
    nw = -(-grid // window)
    return rows // (grid * grid) * nw * nw * window * window


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-6, grid: int = 0,
              window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Row LayerNorm of ``x [rows, C]`` (bf16); with ``window > 0`` the result is in the
    zero-padded window order (see ``samb_layernorm_bf16``)."""
    _need(x, torch.bfloat16, "x"); _need(gamma, torch.float32, "gamma"); _need(beta, torch.float32, "beta")
    x = _rows2d(x, "x")
    if not x.is_contiguous():
        raise RuntimeError("x must be contiguous")
    rows, C = x.shape
    orow = window_rows(rows, grid, window)
    if out is None:
        out = torch.empty(orow, C, dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.load().samb_layernorm_bf16(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), out.data_ptr(), rows, C,
                                               eps, grid, window, _stream()), "samb_layernorm_bf16")
    return out


def layernorm_quant_i8(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-6, grid: int = 0,
                       window: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    _need(x, torch.bfloat16, "x"); _need(gamma, torch.float32, "gamma"); _need(beta, torch.float32, "beta")
    x = _rows2d(x, "x")
    if not x.is_contiguous():
        raise RuntimeError("x must be contiguous")
    rows, C = x.shape
    orow = window_rows(rows, grid, window)
    yq = torch.empty(orow, C, dtype=torch.int8, device=x.device)
    scale = torch.empty(orow, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().samb_layernorm_quant_i8(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), yq.data_ptr(),
                                                   scale.data_ptr(), rows, C, eps, grid, window, _stream()),
               "samb_layernorm_quant_i8")
    return yq, scale


def quant_rows_i8(x: torch.Tensor, gelu: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-row symmetric int8 quantisation of bf16 rows; ``gelu`` applies the exact GELU (rounded to bf16) first."""
    _need(x, torch.bfloat16, "x")
    x = _rows2d(x, "x")
    if not x.is_contiguous():
        raise RuntimeError("x must be contiguous")
    rows, C = x.shape
    yq = torch.empty(rows, C, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    fn = _lib.load().samb_gelu_quant_rows_i8 if gelu else _lib.load().samb_quant_rows_i8
    _lib.check(fn(x.data_ptr(), yq.data_ptr(), scale.data_ptr(), rows, C, _stream()),
               "samb_gelu_quant_rows_i8" if gelu else "samb_quant_rows_i8")
    return yq, scale


def gemm_bf16(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, gelu: bool = False, raw: bool = False,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``epilogue(a [M,K] @ w [N,K]^T)``; residual ``[R, N]`` with ``M % R == 0`` is broadcast over
    row blocks.  ``raw`` returns the fp32 accumulator."""
    _need(a, torch.bfloat16, "a"); _need(w, torch.bfloat16, "w")
    a, w = _rows2d(a, "a"), _rows2d(w, "w")
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise RuntimeError("gemm_bf16: inner dimensions differ")
    epi = 0
    if raw:
        epi = EPI_RAW
    else:
        if bias is not None:
            _need(bias, torch.float32, "bias"); epi |= EPI_BIAS
        if gelu:
            epi |= EPI_GELU
        if residual is not None:
            _need(residual, torch.bfloat16, "residual"); residual = _rows2d(residual, "residual"); epi |= EPI_RESIDUAL
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32 if raw else torch.bfloat16, device=a.device)
    out = _rows2d(out, "out")
    st = status_word(a.device)
    _lib.check(_lib.load().samb_gemm_bf16(
        a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0), _ptr(bias), _ptr(residual),
        residual.stride(0) if residual is not None else 0, residual.shape[0] if residual is not None else 0,
        out.data_ptr(), out.stride(0), M, N, K, epi, st.data_ptr(), _stream()), "samb_gemm_bf16")
    return out


def gemm_i8(aq: torch.Tensor, a_scale: Optional[torch.Tensor], wq: torch.Tensor, w_scale: Optional[torch.Tensor],
            bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, gelu: bool = False,
            raw: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int8 x int8 -> int32 GEMM with the dequantising epilogue; ``raw`` returns the int32 accumulator."""
    _need(aq, torch.int8, "aq"); _need(wq, torch.int8, "wq")
    aq, wq = _rows2d(aq, "aq"), _rows2d(wq, "wq")
    M, K = aq.shape
    N = wq.shape[0]
    if wq.shape[1] != K:
        raise RuntimeError("gemm_i8: inner dimensions differ")
    epi = 0
    if raw:
        epi = EPI_RAW
    else:
        _need(a_scale, torch.float32, "a_scale"); _need(w_scale, torch.float32, "w_scale")
        if bias is not None:
            _need(bias, torch.float32, "bias"); epi |= EPI_BIAS
        if gelu:
            epi |= EPI_GELU
        if residual is not None:
            _need(residual, torch.bfloat16, "residual"); residual = _rows2d(residual, "residual"); epi |= EPI_RESIDUAL
    if out is None:
        out = torch.empty(M, N, dtype=torch.int32 if raw else torch.bfloat16, device=aq.device)
    st = status_word(aq.device)
    _lib.check(_lib.load().samb_gemm_i8(
        aq.data_ptr(), aq.stride(0), _ptr(a_scale), wq.data_ptr(), wq.stride(0), _ptr(w_scale), _ptr(bias),
        _ptr(residual), residual.stride(0) if residual is not None else 0,
        residual.shape[0] if residual is not None else 0, out.data_ptr(), out.stride(0), M, N, K, epi,
        st.data_ptr(), _stream()), "samb_gemm_i8")
    return out


def gemm_i8_requant(aq: torch.Tensor, a_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                    bias: Optional[torch.Tensor] = None, gelu: bool = False, out: Optional[torch.Tensor] = None,
                    meta: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """int8 Linear (+ bias, + GELU) whose output is also quantised per row for the next int8 Linear: returns
    ``(yq int8 [M, N], y_scale [M], out bf16 [M, N])``.  The row maxima come out of the GEMM epilogue (atomic
    maxima into a scratch array of M floats), so no pass over ``out`` reduces anything.  With ``meta`` the weight
    is the 2:4-compressed pair ``(wq = wc [N, K/2], meta)`` of ``pack_sp24``."""
    _need(aq, torch.int8, "aq"); _need(wq, torch.int8, "wq")
    _need(a_scale, torch.float32, "a_scale"); _need(w_scale, torch.float32, "w_scale")
    aq, wq = _rows2d(aq, "aq"), _rows2d(wq, "wq")
    M, K = aq.shape
    N = wq.shape[0]
    if wq.shape[1] * (2 if meta is not None else 1) != K:
        raise RuntimeError("gemm_i8_requant: inner dimensions differ")
    epi = 0
    if bias is not None:
        _need(bias, torch.float32, "bias"); epi |= EPI_BIAS
    if gelu:
        epi |= EPI_GELU
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=aq.device)
    yq = torch.empty(M, N, dtype=torch.int8, device=aq.device)
    y_scale = torch.empty(M, dtype=torch.float32, device=aq.device)
    scratch = torch.empty(M, dtype=torch.float32, device=aq.device)
    st = status_word(aq.device)
    if meta is not None:
        _need(meta, torch.uint8, "meta")
        _lib.check(_lib.load().samb_gemm_i8_sp24_requant(
            aq.data_ptr(), aq.stride(0), a_scale.data_ptr(), wq.data_ptr(), wq.stride(0), meta.data_ptr(),
            w_scale.data_ptr(), _ptr(bias), out.data_ptr(), out.stride(0), yq.data_ptr(), y_scale.data_ptr(),
            scratch.data_ptr(), M, N, K, epi, st.data_ptr(), _stream()), "samb_gemm_i8_sp24_requant")
        return yq, y_scale, out
    _lib.check(_lib.load().samb_gemm_i8_requant(
        aq.data_ptr(), aq.stride(0), a_scale.data_ptr(), wq.data_ptr(), wq.stride(0), w_scale.data_ptr(), _ptr(bias),
        out.data_ptr(), out.stride(0), yq.data_ptr(), y_scale.data_ptr(), scratch.data_ptr(), M, N, K, epi,
        st.data_ptr(), _stream()), "samb_gemm_i8_requant")
    return yq, y_scale, out


def pack_sp24(wq: torch.Tensor):
    """Compress a 2:4-sparse int8 weight ``wq [N, K]`` for ``gemm_i8_sp24``: returns ``(wc [N, K/2] int8,
    meta uint8)``.  A group of four with more than two non-zeros is reported by ``check_status``."""
    _need(wq, torch.int8, "wq")
    wq = _rows2d(wq, "wq")
    N, K = wq.shape
    lib = _lib.load()
    wc = torch.zeros(N, K // 2, dtype=torch.int8, device=wq.device)
    meta = torch.empty(max(int(lib.samb_sp24_meta_bytes(N, K)), 16), dtype=torch.uint8, device=wq.device)
    st = status_word(wq.device)
    _lib.check(lib.samb_pack_sp24(wq.data_ptr(), wq.stride(0), N, K, wc.data_ptr(), wc.stride(0), meta.data_ptr(),
                                  st.data_ptr(), _stream()), "samb_pack_sp24")
    return wc, meta


def gemm_i8_sp24(xq: torch.Tensor, x_scale: Optional[torch.Tensor], wc: torch.Tensor, meta: torch.Tensor,
                 w_scale: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None, gelu: bool = False, raw: bool = False,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gemm_i8`` with the weight given as ``pack_sp24`` output (sparse tensor-core path)."""
    _need(xq, torch.int8, "xq"); _need(wc, torch.int8, "wc"); _need(meta, torch.uint8, "meta")
    xq, wc = _rows2d(xq, "xq"), _rows2d(wc, "wc")
    T, K = xq.shape
    N = wc.shape[0]
    if wc.shape[1] * 2 != K:
        raise RuntimeError("gemm_i8_sp24: inner dimensions differ")
    epi = 0
    if raw:
        epi = EPI_RAW
    else:
        _need(x_scale, torch.float32, "x_scale"); _need(w_scale, torch.float32, "w_scale")
        if bias is not None:
            _need(bias, torch.float32, "bias"); epi |= EPI_BIAS
        if gelu:
            epi |= EPI_GELU
        if residual is not None:
            _need(residual, torch.bfloat16, "residual"); residual = _rows2d(residual, "residual"); epi |= EPI_RESIDUAL
    if out is None:
        out = torch.empty(T, N, dtype=torch.int32 if raw else torch.bfloat16, device=xq.device)
    st = status_word(xq.device)
    _lib.check(_lib.load().samb_gemm_i8_sp24(
        xq.data_ptr(), xq.stride(0), _ptr(x_scale), wc.data_ptr(), wc.stride(0), meta.data_ptr(), _ptr(w_scale),
        _ptr(bias), _ptr(residual), residual.stride(0) if residual is not None else 0,
        residual.shape[0] if residual is not None else 0, out.data_ptr(), out.stride(0), T, N, K, epi,
        st.data_ptr(), _stream()), "samb_gemm_i8_sp24")
    return out


def layernorm2d(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, hw: int, eps: float = 1e-6,
                to_nchw: bool = False) -> torch.Tensor:
    """Channel LayerNorm of token rows ``x [tokens, C]``; ``to_nchw`` stores ``[tokens/hw, C, hw]``."""
    _need(x, torch.bfloat16, "x"); _need(gamma, torch.float32, "gamma"); _need(beta, torch.float32, "beta")
    x = _rows2d(x, "x")
    if not x.is_contiguous():
        raise RuntimeError("x must be contiguous")
    tokens, C = x.shape
    out = torch.empty((tokens // hw, C, hw) if to_nchw else (tokens, C), dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.load().samb_layernorm2d_nchw(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), out.data_ptr(),
                                                 tokens, C, hw, eps, int(to_nchw), _stream()), "samb_layernorm2d_nchw")
    return out


def selftest_bounded_wait(limit_polls: int = 20000) -> int:
    """Run the give-up path of the bounded barrier wait; returns the raw status word."""
    w = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check(_lib.load().samb_selftest_bounded_wait(w.data_ptr(), limit_polls, _stream()),
               "samb_selftest_bounded_wait")
    return int(w.item())


def attn_relpos_global(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rel_h: torch.Tensor,
                       rel_w: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Global-block attention with rel-pos bias: q, k, v ``[B,H,N,d]``, rel_h ``[B,H,N,N/64]``,
    rel_w ``[B,H,N,64]`` (all contiguous, all bfloat16 or all float16) -> ``[B,H,N,d]`` of the same type."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"q must be bfloat16 or float16, got {q.dtype}")
    for name, t in (("q", q), ("k", k), ("v", v), ("rel_h", rel_h), ("rel_w", rel_w)):
        _need(t, q.dtype, name)
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    B, H, N, d = q.shape
    if rel_h.shape != (B, H, N, N // 64) or rel_w.shape != (B, H, N, 64):
        raise RuntimeError("rel_h / rel_w shapes do not match q")
    o = torch.empty_like(q)
    st = status_word(q.device)
    lib = _lib.load()
    fn = lib.samb_attn_relpos_global_f16 if q.dtype == torch.float16 else lib.samb_attn_relpos_global
    _lib.check(fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), rel_h.data_ptr(), rel_w.data_ptr(), o.data_ptr(), B, H, N, d,
                  float(scale if scale is not None else d ** -0.5), st.data_ptr(), _stream()), "samb_attn_relpos_global")
    return o


def attn_relpos_global_qkv(qkv: torch.Tensor, tab: torch.Tensor, t_head_stride: int, t_w_off: int, B: int, H: int,
                           N: int, d: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Global-block attention over the head-major ``qkv [3H, B*N, d]`` buffer with the bias taken from
    the table products ``tab [B*N, ldt]``; returns ``[B*N, H*d]``."""
    _need(qkv, torch.bfloat16, "qkv"); _need(tab, torch.bfloat16, "tab")
    if not qkv.is_contiguous() or qkv.shape != (3 * H, B * N, d):
        raise RuntimeError("qkv must be contiguous [3H, B*N, d]")
    tab = _rows2d(tab, "tab")
    if out is None:
        out = torch.empty(B * N, H * d, dtype=torch.bfloat16, device=qkv.device)
    st = status_word(qkv.device)
    _lib.check(_lib.load().samb_attn_relpos_global_qkv(
        qkv.data_ptr(), tab.data_ptr(), tab.stride(0), t_head_stride, t_w_off, out.data_ptr(), out.stride(0), B, H, N,
        d, float(d ** -0.5), st.data_ptr(), _stream()), "samb_attn_relpos_global_qkv")
    return out


def attn_relpos_global_tables(qkv: torch.Tensor, tables: torch.Tensor, B: int, H: int, N: int, d: int,
                              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Global-block attention over the head-major ``qkv [3H, B*N, d]`` buffer with the rel-pos bias computed inside
    the kernel from ``tables [256, d]`` (rel_pos_h from row 0, rel_pos_w from row 128); returns ``[B*N, H*d]``."""
    _need(qkv, torch.bfloat16, "qkv"); _need(tables, torch.bfloat16, "tables")
    if not qkv.is_contiguous() or qkv.shape != (3 * H, B * N, d):
        raise RuntimeError("qkv must be contiguous [3H, B*N, d]")
    if not tables.is_contiguous() or tables.shape != (256, d):
        raise RuntimeError("tables must be contiguous [256, d]")
    if out is None:
        out = torch.empty(B * N, H * d, dtype=torch.bfloat16, device=qkv.device)
    st = status_word(qkv.device)
    _lib.check(_lib.load().samb_attn_relpos_global_tables(
        qkv.data_ptr(), tables.data_ptr(), out.data_ptr(), out.stride(0), B, H, N, d, float(d ** -0.5), st.data_ptr(),
        _stream()), "samb_attn_relpos_global_tables")
    return out


def attn_relpos_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rel_h: torch.Tensor,
                       rel_w: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Windowed attention with rel-pos bias: q, k, v ``[B,H,196,d]``, rel_h / rel_w ``[B,H,196,14]`` (all bfloat16 or
    all float16) -> ``[B,H,196,d]`` of the same type."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"q must be bfloat16 or float16, got {q.dtype}")
    for name, t in (("q", q), ("k", k), ("v", v), ("rel_h", rel_h), ("rel_w", rel_w)):
        _need(t, q.dtype, name)
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    B, H, N, d = q.shape
    ws = int(round(N ** 0.5))
    if ws * ws != N or rel_h.shape != (B, H, N, ws) or rel_w.shape != (B, H, N, ws):
        raise RuntimeError("rel_h / rel_w shapes do not match q")
    o = torch.empty_like(q)
    st = status_word(q.device)
    lib = _lib.load()
    fn = lib.samb_attn_relpos_window_f16 if q.dtype == torch.float16 else lib.samb_attn_relpos_window
    _lib.check(fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), rel_h.data_ptr(), rel_w.data_ptr(), o.data_ptr(), B, H, ws, d,
                  float(scale if scale is not None else d ** -0.5), st.data_ptr(), _stream()), "samb_attn_relpos_window")
    return o


def attn_relpos_window_qkv(qkv: torch.Tensor, tab: torch.Tensor, t_head_stride: int, t_w_off: int, B: int, H: int,
                           grid: int, window: int, d: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Windowed attention over the window-ordered head-major ``qkv [3H, B*nw*nw*window^2, d]``; returns
    raster-order ``[B*grid*grid, H*d]`` (pad tokens dropped)."""
    _need(qkv, torch.bfloat16, "qkv"); _need(tab, torch.bfloat16, "tab")
    rows = window_rows(B * grid * grid, grid, window)
    if not qkv.is_contiguous() or qkv.shape != (3 * H, rows, d):
        raise RuntimeError("qkv must be contiguous [3H, B*nw*nw*window^2, d]")
    tab = _rows2d(tab, "tab")
    if out is None:
        out = torch.empty(B * grid * grid, H * d, dtype=torch.bfloat16, device=qkv.device)
    st = status_word(qkv.device)
    _lib.check(_lib.load().samb_attn_relpos_window_qkv(
        qkv.data_ptr(), tab.data_ptr(), tab.stride(0), t_head_stride, t_w_off, out.data_ptr(), out.stride(0), B, H,
        grid, window, d, float(d ** -0.5), st.data_ptr(), _stream()), "samb_attn_relpos_window_qkv")
    return out


def attn_relpos_window_raster(qkv: torch.Tensor, qkv_bias: torch.Tensor, tab: torch.Tensor, t_head_stride: int,
                              t_w_off: int, B: int, H: int, grid: int, window: int, d: int,
                              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Windowed attention over raster-order head-major ``qkv [3H, B*grid*grid, d]`` (no padded copy of the
    tokens); ``qkv_bias`` is the projection bias as bf16 ``[3H*d]`` (the keys / values of the zero-padded
    tokens of border windows).  Returns raster-order ``[B*grid*grid, H*d]``."""
    _need(qkv, torch.bfloat16, "qkv"); _need(tab, torch.bfloat16, "tab"); _need(qkv_bias, torch.bfloat16, "qkv_bias")
    if not qkv.is_contiguous() or qkv.shape != (3 * H, B * grid * grid, d):
        raise RuntimeError("qkv must be contiguous [3H, B*grid*grid, d]")
    if not qkv_bias.is_contiguous() or qkv_bias.numel() != 3 * H * d:
        raise RuntimeError("qkv_bias must be contiguous [3H*d]")
    tab = _rows2d(tab, "tab")
    if out is None:
        out = torch.empty(B * grid * grid, H * d, dtype=torch.bfloat16, device=qkv.device)
    st = status_word(qkv.device)
    _lib.check(_lib.load().samb_attn_relpos_window_raster(
        qkv.data_ptr(), qkv_bias.data_ptr(), tab.data_ptr(), tab.stride(0), t_head_stride, t_w_off, out.data_ptr(),
        out.stride(0), B, H, grid, window, d, float(d ** -0.5), st.data_ptr(), _stream()),
        "samb_attn_relpos_window_raster")
    return out


def attn_relpos_window_tables(qkv: torch.Tensor, qkv_bias: torch.Tensor, tables: torch.Tensor, B: int, H: int,
                              grid: int, window: int, d: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``attn_relpos_window_raster`` with the rel-pos bias computed inside the kernel from ``tables [64, d]``
    (rel_pos_h from row 0, rel_pos_w from row 32).  Returns raster-order ``[B*grid*grid, H*d]``."""
    _need(qkv, torch.bfloat16, "qkv"); _need(tables, torch.bfloat16, "tables"); _need(qkv_bias, torch.bfloat16, "qkv_bias")
    if not qkv.is_contiguous() or qkv.shape != (3 * H, B * grid * grid, d):
        raise RuntimeError("qkv must be contiguous [3H, B*grid*grid, d]")
    if not qkv_bias.is_contiguous() or qkv_bias.numel() != 3 * H * d:
        raise RuntimeError("qkv_bias must be contiguous [3H*d]")
    if not tables.is_contiguous() or tables.shape != (64, d):
        raise RuntimeError("tables must be contiguous [64, d]")
    if out is None:
        out = torch.empty(B * grid * grid, H * d, dtype=torch.bfloat16, device=qkv.device)
    st = status_word(qkv.device)
    _lib.check(_lib.load().samb_attn_relpos_window_tables(
        qkv.data_ptr(), qkv_bias.data_ptr(), tables.data_ptr(), out.data_ptr(), out.stride(0), B, H, grid, window, d,
        float(d ** -0.5), st.data_ptr(), _stream()), "samb_attn_relpos_window_tables")
    return out


def gemm_heads(a: torch.Tensor, a_scale: Optional[torch.Tensor], w: torch.Tensor, w_scale: Optional[torch.Tensor],
               bias: Optional[torch.Tensor], head_dim: int) -> torch.Tensor:
    """qkv projection with a head-major result ``[N/head_dim, M, head_dim]`` (bf16).  ``a``/``w`` are bf16,
    or int8 with their row scales."""
    a, w = _rows2d(a, "a"), _rows2d(w, "w")
    M, K = a.shape
    N = w.shape[0]
    if bias is not None:
        _need(bias, torch.float32, "bias")
    out = torch.empty(N // head_dim, M, head_dim, dtype=torch.bfloat16, device=a.device)
    st = status_word(a.device)
    if a.dtype == torch.int8:
        _need(w, torch.int8, "w"); _need(a_scale, torch.float32, "a_scale"); _need(w_scale, torch.float32, "w_scale")
        _lib.check(_lib.load().samb_gemm_i8_heads(a.data_ptr(), a.stride(0), a_scale.data_ptr(), w.data_ptr(), w.stride(0),
                                                  w_scale.data_ptr(), _ptr(bias), out.data_ptr(), M, N, K, head_dim,
                                                  st.data_ptr(), _stream()), "samb_gemm_i8_heads")
    else:
        _need(a, torch.bfloat16, "a"); _need(w, torch.bfloat16, "w")
        _lib.check(_lib.load().samb_gemm_bf16_heads(a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0), _ptr(bias),
                                                    out.data_ptr(), M, N, K, head_dim, st.data_ptr(), _stream()),
                   "samb_gemm_bf16_heads")
    return out


def relpos_table_products(qkv_hm: torch.Tensor, tables: torch.Tensor, col_scale: torch.Tensor, H: int,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``tab[t, h*T + m] = (q_h[t] . tables[m]) * col_scale[m]`` for the H query planes of the head-major
    ``qkv_hm [3H, rows, d]``; ``T = tables.shape[0]``."""
    _need(qkv_hm, torch.bfloat16, "qkv_hm"); _need(tables, torch.bfloat16, "tables"); _need(col_scale, torch.float32, "col_scale")
    if qkv_hm.dim() != 3 or not qkv_hm.is_contiguous() or qkv_hm.shape[0] != 3 * H:
        raise RuntimeError("qkv_hm must be a contiguous [3H, rows, d] tensor")
    _, rows, d = qkv_hm.shape
    T = tables.shape[0]
    if not tables.is_contiguous() or tables.shape != (T, d) or col_scale.shape != (T,):
        raise RuntimeError("tables must be contiguous [T, d] with a [T] scale")
    if out is None:
        out = torch.empty(rows, H * T, dtype=torch.bfloat16, device=qkv_hm.device)
    st = status_word(qkv_hm.device)
    _lib.check(_lib.load().samb_relpos_table_products(
        qkv_hm.data_ptr(), tables.data_ptr(), col_scale.data_ptr(), out.data_ptr(), out.stride(0), rows, H, d, T,
        st.data_ptr(), _stream()), "samb_relpos_table_products")
    return out


def patch_rows(x: torch.Tensor, patch: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """NCHW image batch ``[B,Cin,S,S]`` (bf16) -> patch rows ``[B*(S/patch)^2, Cin*patch*patch]``."""
    _need(x, torch.bfloat16, "x")
    if x.dim() != 4 or not x.is_contiguous() or x.shape[2] != x.shape[3] or x.shape[2] % patch:
        raise RuntimeError("x must be a contiguous square NCHW batch whose side is a multiple of the patch size")
    B, Cin, S, _ = x.shape
    grid = S // patch
    if out is None:
        out = torch.empty(B * grid * grid, Cin * patch * patch, dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.load().samb_patch_rows(x.data_ptr(), out.data_ptr(), B, Cin, grid, patch, _stream()), "samb_patch_rows")
    return out


def patch_rows_u8(x: torch.Tensor, patch: int, mean, std, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """uint8 NCHW image batch ``[B,3,S,S]`` -> normalised bf16 patch rows ``[B*(S/patch)^2, 3*patch*patch]``
    (``(x - mean[c]) / std[c]``, then the gather of ``patch_rows``) in one pass."""
    import ctypes
    _need(x, torch.uint8, "x")
    if x.dim() != 4 or not x.is_contiguous() or x.shape[1] != 3 or x.shape[2] != x.shape[3] or x.shape[2] % patch:
        raise RuntimeError("x must be a contiguous square [B,3,S,S] uint8 batch whose side is a multiple of the patch size")
    B, Cin, S, _ = x.shape
    grid = S // patch
    if out is None:
        out = torch.empty(B * grid * grid, Cin * patch * patch, dtype=torch.bfloat16, device=x.device)
    m = (ctypes.c_float * 3)(*[float(v) for v in mean])
    s = (ctypes.c_float * 3)(*[float(v) for v in std])
    _lib.check(_lib.load().samb_patch_rows_u8(x.data_ptr(), out.data_ptr(), B, Cin, grid, patch, m, s, _stream()),
               "samb_patch_rows_u8")
    return out


def conv3x3_rows(x: torch.Tensor, grid: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Token rows ``[tokens, C]`` -> 3x3 neighbourhood rows ``[tokens, 9*C]`` (zero padding 1)."""
    _need(x, torch.bfloat16, "x")
    x = _rows2d(x, "x")
    if not x.is_contiguous():
        raise RuntimeError("x must be contiguous")
    tokens, C = x.shape
    if out is None:
        out = torch.empty(tokens, 9 * C, dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.load().samb_conv3x3_rows(x.data_ptr(), out.data_ptr(), tokens, grid, C, _stream()), "samb_conv3x3_rows")
    return out


def normalize_u8(x: torch.Tensor, mean, std, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """uint8 ``[B,3,H,W]`` -> bf16 ``(x - mean[c]) / std[c]``."""
    import ctypes
    _need(x, torch.uint8, "x")
    if x.dim() != 4 or not x.is_contiguous():
        raise RuntimeError("x must be a contiguous [B,3,H,W] uint8 tensor")
    B, C, H, W = x.shape
    if out is None:
        out = torch.empty(B, C, H, W, dtype=torch.bfloat16, device=x.device)
    m = (ctypes.c_float * 3)(*[float(v) for v in mean])
    s = (ctypes.c_float * 3)(*[float(v) for v in std])
    _lib.check(_lib.load().samb_normalize_u8(x.data_ptr(), out.data_ptr(), B, C, H, W, m, s, _stream()), "samb_normalize_u8")
    return out


# ---------------------------------------------------------------------------------------------------------------
# Operators of transformer blocks beside the reference's own kind: norms around a block, rotary positions, a mixture
# of experts.  16-bit tensors are bfloat16 or float16.
# An ``out`` is memory of its own or the operand itself that the docstring allows; any other overlap is refused.
# ---------------------------------------------------------------------------------------------------------------
_F32, _F16, _BF16, _I32 = torch.float32, torch.float16, torch.bfloat16, torch.int32


def _here(t: torch.Tensor, dtype: torch.dtype, dev: int, name: str) -> None:
    """``_need`` against a device number that the caller has asked for once."""
    if t.dtype is not dtype or t.get_device() != dev:
        _need(t, dtype, name)


def _half(t: torch.Tensor, name: str) -> Tuple[torch.dtype, int]:
    """Type and device of a bfloat16 or float16 tensor on the current device."""
    dtype = t.dtype
    if dtype is not _BF16 and dtype is not _F16:
        raise RuntimeError(f"{name}: expected bfloat16 or float16, got {dtype}")
    dev = t.get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        _need(t, dtype, name)
    return dtype, dev


def _vector(t: torch.Tensor, name: str, dev: int, shape: Tuple[int, ...]) -> int:
    """Pointer of a contiguous fp32 tensor of this shape."""
    if t.dtype is _F32 and t.get_device() == dev and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    _need(t, _F32, name)
    raise RuntimeError(f"{name}: expected a contiguous float32 tensor of shape {list(shape)}, got {list(t.shape)}")


def _indexes(t: torch.Tensor, name: str, dev: int, n: int) -> int:
    if t.dtype is _I32 and t.get_device() == dev and t.shape == (n,) and t.is_contiguous():
        return t.data_ptr()
    _need(t, _I32, name)
    raise RuntimeError(f"{name}: expected a contiguous int32 tensor of {n} elements, got {list(t.shape)}")


def _matrix(t: torch.Tensor, name: str) -> int:
    """Leading dimension of a row-major matrix; a single row has none of its own."""
    if t.dim() == 2:
        rows, cols = t.shape
        ld, inner = t.stride()
        if inner == 1 or cols <= 1:
            return ld if rows > 1 else cols
    raise RuntimeError(f"{name}: expected a 2-D tensor with unit inner stride")


def _like(t: torch.Tensor, dtype: torch.dtype, dev: int, shape, name: str) -> int:
    """Leading dimension of a matrix that has to have this type and shape."""
    if t.dtype is not dtype or t.get_device() != dev:
        _need(t, dtype, name)
    if t.shape != shape:
        raise RuntimeError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")
    ld, inner = t.stride()
    rows, cols = shape
    if inner != 1 and cols > 1:
        raise RuntimeError(f"{name}: expected unit inner stride")
    return ld if rows > 1 else cols


def _status(t: torch.Tensor, dev: int) -> int:
    """Pointer of the device's status word.  It outlives the call, so a capture must not be what allocates it."""
    w = _status_words.get(dev)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("make one call on this device before capturing it into a graph")
        w = status_word(t.device)
    return w.data_ptr()


def _norm_args(h, dtype, dev, residual, post, pre, gate, out):
    """Arguments of the block norms up to the gate, the output and its leading dimension."""
    ldh = _matrix(h, "h")
    shape = h.shape
    rows, C = shape
    vec = (C,)
    pr = pgg = pgb = pqg = pqb = pg = None
    ldr = gates = 0
    if residual is not None:
        ldr = _like(residual, dtype, dev, shape, "residual")
        pr = residual.data_ptr()
    if post is not None:
        gain, offset = post
        pgg = _vector(gain, "post gain", dev, vec)
        if offset is not None:
            pgb = _vector(offset, "post offset", dev, vec)
    if pre is not None:
        gain, offset = pre
        pqg = _vector(gain, "pre gain", dev, vec)
        if offset is not None:
            pqb = _vector(offset, "pre offset", dev, vec)
    if gate is not None:
        gates = gate.shape[0] if gate.dim() == 2 else 1
        pg = _vector(gate, "gate", dev, (gates, C) if gate.dim() == 2 else vec)
        if gates == 0 or rows % gates:
            raise RuntimeError(f"gate: {gates} vectors do not divide {rows} rows")
    if out is None:
        out, ldx = torch.empty_like(h), C                 # rows of unit inner stride: a dense copy is row-major
    else:
        ldx = _like(out, dtype, dev, shape, "out")
    return (h.data_ptr(), ldh, pr, ldr, pgg, pgb, pqg, pqb, pg, gates), out, ldx


def block_norm(h: torch.Tensor, residual: Optional[torch.Tensor] = None, post=None, pre=None,
               gate: Optional[torch.Tensor] = None, res_scale: float = 1.0, eps: float = 1e-6, rms: bool = False,
               out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The norms before and after a residual addition in one pass: ``x = res_scale * residual + gate * post(h)`` and
    ``y = pre(x)`` over rows ``[rows, C]`` (C a multiple of 8 up to 8192); returns ``(x, y)``, y being None without
    ``pre``.  ``post`` / ``pre`` are ``(gain, offset or None)`` in fp32, LayerNorm or with ``rms`` root-mean-square
    norms; ``gate`` is fp32 ``[C]``, or ``[G, C]`` with one vector for each of G equal blocks of rows.  ``out`` (x) may
    be ``residual`` or ``h``."""
    dtype, dev = _half(h, "h")
    args, x, ldx = _norm_args(h, dtype, dev, residual, post, pre, gate, out)
    y = torch.empty_like(h) if pre is not None else None
    rows, C = h.shape
    _lib.check(_lib.load().samb_block_norm(*args, res_scale, eps, dtype is _F16, rms, x.data_ptr(), ldx,
                                           None if y is None else y.data_ptr(), rows, C, _raw_stream(dev)),
               "samb_block_norm")
    return x, y


def block_norm_quant_i8(h: torch.Tensor, residual: Optional[torch.Tensor], post, pre, gate: Optional[torch.Tensor] = None,
                        res_scale: float = 1.0, eps: float = 1e-6, rms: bool = False,
                        out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``block_norm`` (bf16) whose y leaves quantised per row for an int8 Linear: returns ``(x, yq, y_scale)``, the
    values ``quant_rows_i8`` gives on y."""
    _need(h, torch.bfloat16, "h")
    if pre is None:
        raise RuntimeError("block_norm_quant_i8 needs the norm whose output it quantises")
    dev = h.get_device()
    args, x, ldx = _norm_args(h, _BF16, dev, residual, post, pre, gate, out)
    rows, C = h.shape
    yq = torch.empty(rows, C, dtype=torch.int8, device=h.device)
    scale = torch.empty(rows, dtype=_F32, device=h.device)
    _lib.check(_lib.load().samb_block_norm_quant_i8(*args, res_scale, eps, rms, x.data_ptr(), ldx, yq.data_ptr(),
                                                    scale.data_ptr(), rows, C, _raw_stream(dev)), "samb_block_norm_quant_i8")
    return x, yq, scale


def rotary_freqs(rot: int, base: float = 10000.0, axes: int = 1, scaling: Optional[str] = None, factor: float = 1.0,
                 trained: int = 4096, device=None) -> Tuple[torch.Tensor, float]:
    """Angular frequencies (float64 ``[rot / 2]``, radians a position) and the factor on the rotation for ``rotary``:
    ``base ** (-i / n)`` for the n pairs of each axis.  ``scaling`` stretches them by ``factor`` for positions beyond
    the ``trained`` length: ``"linear"`` divides every frequency, ``"base"`` raises the base so that the slowest pair
    is stretched by the factor and the fastest not at all, ``"parts"`` keeps pairs of more than 32 turns over the
    trained length, divides those of less than one, ramps in between and scales the rotation by
    ``0.1 ln(factor) + 1`` (the YaRN rule)."""
    if rot <= 0 or axes not in (1, 2) or rot % (2 * axes):
        raise RuntimeError(f"rotary_freqs: {rot} rotated elements do not make pairs on {axes} axes")
    if scaling not in (None, "linear", "base", "parts"):
        raise RuntimeError(f"rotary_freqs: unknown scaling {scaling!r}")
    if not (base > 0 and factor >= 1 and trained > 0):
        raise RuntimeError("rotary_freqs: base and trained must be positive and factor at least 1")
    n = rot // 2 // axes
    i = torch.arange(n, dtype=torch.float64)
    if scaling == "base" and n > 1:
        base = base * factor ** (n / (n - 1))
    f = base ** (-i / n)
    mscale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        keep = ((trained * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
        mscale = 0.1 * math.log(factor) + 1.0
    return f.repeat(axes).to(device or torch.device("cuda", torch.cuda.current_device())), mscale


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool = False,
           mscale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions on ``x [planes, rows, d]`` (any plane and row strides that are multiples of 8: the q and k planes
    ``qkv[:2 * H]`` of ``gemm_heads``, or a ``[rows, heads, d]`` tensor seen as ``x.transpose(0, 1)``).  Pairs are
    neighbours (``interleaved``) or half the rotated width apart; the first ``2 * len(freqs)`` elements of a row turn,
    the rest is copied.  ``positions`` int32 / int64: ``[P]``, or ``[P, 2]`` for a raster (first half of the pairs by the
    first coordinate); row r uses entry ``r % P``.  ``freqs`` float64, see ``rotary_freqs``.  ``out`` may be ``x``;
    a new result has the order of x's axes, and rows padded to a multiple of 8 where d is none."""
    dtype, dev = _half(x, "x")
    _here(freqs, torch.float64, dev, "freqs")
    pt = positions.dtype
    if pt is not torch.int64 and pt is not _I32:
        raise RuntimeError(f"positions: expected int32 or int64, got {pt}")
    _here(positions, pt, dev, "positions")
    if x.dim() != 3:
        raise RuntimeError("x: expected a [planes, rows, d] tensor")
    planes, rows, d = x.shape
    ps, rs, es = x.stride()
    axes = positions.dim()
    if axes not in (1, 2) or not positions.is_contiguous() or (axes == 2 and positions.shape[1] != 2):
        raise RuntimeError("positions: expected a contiguous [P] or [P, 2] tensor")
    period = positions.shape[0]
    if rows and (period == 0 or rows % period):
        raise RuntimeError(f"positions: {period} entries do not divide {rows} rows")
    if freqs.dim() != 1 or not freqs.is_contiguous():
        raise RuntimeError("freqs: expected a contiguous 1-D tensor")
    if out is None:
        if d % 8 == 0:
            out = torch.empty_like(x)                     # laid out like x where x has no gaps
        elif ps < rs:                                     # rows start at multiples of 8, as those of x
            out = torch.empty(rows, planes, -(-d // 8) * 8, dtype=dtype, device=x.device)[..., :d].transpose(0, 1)
        else:
            out = torch.empty(planes, rows, -(-d // 8) * 8, dtype=dtype, device=x.device)[..., :d]
    else:
        _here(out, dtype, dev, "out")
        if out.shape != x.shape:
            raise RuntimeError("out must have the shape of x")
    ops_, ors, oes = out.stride()
    if d > 1 and (es != 1 or oes != 1):
        raise RuntimeError("x and out: expected unit inner stride")
    if planes <= 1:                                       # strides of a single plane or row mean nothing
        ps = ops_ = 0
    if rows <= 1:
        rs = ors = 0
    _lib.check(_lib.load().samb_rotary(
        x.data_ptr(), ps, rs, positions.data_ptr(), pt is torch.int64, period, axes, freqs.data_ptr(), 2 * freqs.shape[0],
        interleaved, mscale, out.data_ptr(), ops_, ors, planes, rows, d, dtype is _F16, _raw_stream(dev)), "samb_rotary")
    return out


class Routing(NamedTuple):
    """What ``route_topk`` found: ``ids`` and ``weights`` ``[T, k]``, ``slots [T, k]`` (place of each choice in the order
    by expert, -1: none), ``rows [T * k]`` (token in each place, -1 behind the last), ``offsets [E + 1]``."""
    ids: torch.Tensor
    weights: torch.Tensor
    slots: torch.Tensor
    rows: torch.Tensor
    offsets: torch.Tensor


def route_topk(logits: torch.Tensor, k: int, bias: Optional[torch.Tensor] = None, sigmoid: bool = False,
               renorm: bool = True, scale: float = 1.0) -> Routing:
    """Router of a mixture of experts over fp32 ``logits [T, E]`` (E up to 512, k up to 8): every token's k largest
    logits (plus ``bias [E]``, which decides the choice only; ties to the lower index), their softmax or sigmoid
    weights (the bias is added to the logit: one trained on top of the sigmoid or softmax orders experts differently), and the order of the choices by expert for ``gemm_grouped`` and ``combine_topk``.  An expert at -inf or NaN
    is never chosen: a token with nobody left (a padded one) gets id -1, weight 0 and no place."""
    dev = logits.get_device()
    if logits.dtype is not _F32 or dev < 0 or dev != torch.cuda.current_device():
        _need(logits, _F32, "logits")
    ld = _matrix(logits, "logits")
    T, E = logits.shape
    if not 1 <= k <= min(8, E):
        raise RuntimeError(f"k: {k} is not between 1 and 8 and at most the number of experts ({E})")
    lib = _lib.load()
    n = T * k
    pbias = None if bias is None else _vector(bias, "bias", dev, (E,))
    room = lib.samb_route_scratch_bytes(T, E) // 4
    # one allocation for the whole numbers: ids, slots, rows, offsets and the scratch
    buf = torch.empty(3 * n + E + 1 + room, dtype=_I32, device=logits.device)
    weights = torch.empty(T, k, dtype=_F32, device=logits.device)
    at = buf.data_ptr()
    _lib.check(lib.samb_route_topk(
        logits.data_ptr(), ld, pbias, T, E, k, sigmoid, renorm, scale, at, weights.data_ptr(), at + 4 * n, at + 8 * n,
        at + 12 * n, at + 4 * (3 * n + E + 1), _raw_stream(dev)), "samb_route_topk")
    return Routing(buf.as_strided((T, k), (k, 1), 0), weights, buf.as_strided((T, k), (k, 1), n),
                   buf.as_strided((n,), (1,), 2 * n), buf.as_strided((E + 1,), (1,), 3 * n))


def _grouped(kind, a, a_scale, w, w_scale, offsets, rows, bias, gelu, out, dtype, dev):
    int8 = dtype is torch.int8
    odt = _BF16 if int8 else dtype
    lda = _matrix(a, "a")
    _here(w, dtype, dev, "w")
    if w.dim() != 3:
        raise RuntimeError("w: expected an [experts, N, K] tensor")
    E, N, K = w.shape
    ws, ldw, es = w.stride()
    if es != 1 and K > 1:
        raise RuntimeError("w: expected unit inner stride")
    M, ka = a.shape
    if ka != K:
        raise RuntimeError(f"{kind}: inner dimensions differ")
    lib = _lib.load()
    prow = pbias = psc = None
    S, epi = M, EPI_GELU if gelu else 0
    if rows is not None:
        S = rows.shape[0]
        prow = _indexes(rows, "rows", dev, S)
        room = lib.samb_gemm_grouped_scratch_bytes(S, E, N, K, int8)
        if room:                                          # room to put the rows of a large product in order
            scratch = torch.empty(room, dtype=torch.uint8, device=a.device)
            psc = scratch.data_ptr()
    if bias is not None:
        pbias = _vector(bias, "bias", dev, (E, N))
        epi |= EPI_BIAS
    poff = _indexes(offsets, "offsets", dev, E + 1)
    if out is None:
        out, ldo = torch.empty(S, N, dtype=odt, device=a.device), N
    else:
        ldo = _like(out, odt, dev, (S, N), "out")
    if N <= 1:
        ldw = K
    if E <= 1:
        ws = 0
    st = _status(a, dev)
    if int8:
        _lib.check(lib.samb_gemm_i8_grouped(
            a.data_ptr(), lda, M, _vector(a_scale, "a_scale", dev, (M,)), prow, w.data_ptr(), ldw, ws,
            _vector(w_scale, "w_scale", dev, (E, N)), pbias, poff, out.data_ptr(), ldo, S, E, N, K, epi, psc, st,
            _raw_stream(dev)), "samb_gemm_i8_grouped")
    else:
        _lib.check(lib.samb_gemm_grouped(
            a.data_ptr(), lda, M, prow, w.data_ptr(), ldw, ws, pbias, poff, out.data_ptr(), ldo, S, E, N, K,
            dtype is _F16, epi, psc, st, _raw_stream(dev)), "samb_gemm_grouped")
    return out


def gemm_grouped(a: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, rows: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, gelu: bool = False,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Products grouped by expert: ``out[s] = act(a[rows[s]] @ w[e]^T + bias[e])`` for ``offsets[e] <= s < offsets[e + 1]``
    (without ``rows``: ``a[s]``), with ``a [M, K]`` and ``w [E, N, K]`` bfloat16 or float16, int32 ``offsets [E + 1]`` and
    ``rows [S]`` as ``route_topk`` gives them.  Rows of ``out [S, N]`` behind the last expert's are left as they were
    (unspecified in a new ``out``); an index outside ``a`` (of one row at least) stands for a row of zeros."""
    dtype, dev = _half(a, "a")
    return _grouped("gemm_grouped", a, None, w, None, offsets, rows, bias, gelu, out, dtype, dev)


def gemm_i8_grouped(aq: torch.Tensor, a_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                    offsets: torch.Tensor, rows: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                    gelu: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gemm_grouped`` on int8 ``aq [M, K]`` with row scales ``a_scale [M]`` (gathered with the rows) and ``wq [E, N, K]``
    with ``w_scale [E, N]``: exact int32 accumulation, bf16 out."""
    _need(aq, torch.int8, "aq")
    if a_scale is None or w_scale is None:
        raise RuntimeError("gemm_i8_grouped needs both scales")
    return _grouped("gemm_i8_grouped", aq, a_scale, wq, w_scale, offsets, rows, bias, gelu, out, torch.int8,
                    aq.get_device())


def combine_topk(x: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Weighted sum of the experts' rows back in token order: ``out[t] = residual[t] + sum_j weights[t, j] *
    x[slots[t, j]]`` with ``x [S, C]`` bfloat16 or float16, ``slots`` / ``weights`` ``[T, k]`` of ``route_topk`` (k up to 8);
    a slot of -1 adds nothing.  ``out`` may be ``residual``."""
    dtype, dev = _half(x, "x")
    ldx = _matrix(x, "x")
    S, C = x.shape
    _here(slots, _I32, dev, "slots")
    if slots.dim() != 2 or not slots.is_contiguous():
        raise RuntimeError("slots: expected a contiguous [T, k] tensor")
    T, k = slots.shape
    pr, ldr = None, 0
    if residual is not None:
        ldr = _like(residual, dtype, dev, (T, C), "residual")
        pr = residual.data_ptr()
    if out is None:
        out = torch.empty(T, C, dtype=dtype, device=x.device) if residual is None else torch.empty_like(residual)
        ldo = C
    else:
        ldo = _like(out, dtype, dev, (T, C), "out")
    _lib.check(_lib.load().samb_combine_topk(
        x.data_ptr(), ldx, S, slots.data_ptr(), _vector(weights, "weights", dev, (T, k)), pr, ldr, out.data_ptr(), ldo,
        T, k, C, dtype is _F16, _raw_stream(dev)), "samb_combine_topk")
    return out
