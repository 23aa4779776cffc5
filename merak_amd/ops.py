"""Tensor-level wrappers over the C ABI: shape/dtype/device checks, output
allocation through PyTorch's caching allocator, and the current HIP stream.

PyTorch is plumbing here (device memory and streams); every FLOP and every
byte moved happens inside ``libmerak_tp_gfx950.so``.  CPU tensors are rejected:
there is no fallback path.
"""
from __future__ import annotations

import threading
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import (EPI_BIAS, EPI_BIAS_GELU, EPI_GELU, EPI_NONE, EPI_SWIGLU,
                   MTP_BF16, MTP_F16, MTP_F32)

_DTYPES = {torch.float32: MTP_F32, torch.bfloat16: MTP_BF16, torch.float16: MTP_F16}
_arch_ok = {}


def _dt(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"merak_amd kernels take float32, bfloat16 or float16 tensors, got {t.dtype}") from None


def _require_gpu(*ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                "merak_amd kernels run on an MI355X (gfx950) device only; got a tensor on "
                f"{t.device}. There is no CPU fallback.")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    if idx not in _arch_ok:
        with torch.cuda.device(idx):
            arch = _lib.device_arch()
        if arch != "gfx950":
            raise RuntimeError(f"merak_amd kernels are built for gfx950 only; device {idx} is {arch}")
        _arch_ok[idx] = True
    return dev


def _public_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the handle without the Stream object around it: 1.8 us of a small launch; a torch without this name has the other way
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _stream(dev: torch.device) -> int:
    return _raw_stream(dev.index)


class _Here:
    """Stands in for ``torch.cuda.device(dev)`` where dev is the current device already: entering and leaving that
    takes as long as a small launch."""

    def __enter__(self):
        pass

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _device(dev: torch.device):
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


# --------------------------------------------------------------------------- linear
_linear_ws_cache = {}
_linear_ws_lock = threading.Lock()   # forward runs on the caller's thread, backward on autograd's worker thread


def linear_workspace(dev: torch.device, nbytes: Optional[int] = None) -> torch.Tensor:
    """Scratch of the linear products for the current stream of `dev` (16-bit: stream-K, tiles whose k range
    several workgroups share meet there; fp32: the slices of a product that is cut along k), at least `nbytes`
    long (default: the 16-bit path's full size).  One buffer per (device, stream), allocated when a product first
    asks for scratch and grown when a later one asks for more: launches on one stream are ordered, so they may
    share it.  ``release_workspaces()`` drops them all."""
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    key = (idx, torch.cuda.current_stream(dev).cuda_stream)
    if nbytes is None:
        nbytes = _lib.lib().mtp_linear_workspace_bytes()
    with _linear_ws_lock:
        ws = _linear_ws_cache.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = torch.empty(int(nbytes), dtype=torch.uint8, device=dev)
            _linear_ws_cache[key] = ws
    return ws


def release_workspaces() -> None:
    """Forget the cached scratch buffers of the linear products (they are allocated again on demand)."""
    with _linear_ws_lock:
        _linear_ws_cache.clear()


def _ws_args(kind: int, M: int, N: int, K: int, t: torch.Tensor, dev: torch.device):
    """(pointer, bytes) of the scratch for product `kind` (0 forward, 1 input gradient, 2 weight gradient, 3 both
    gradients) of a layer with M tokens, N output and K input features on tensors like t; (None, 0) for the shapes
    that never use scratch, which then allocate nothing."""
    need = _lib.lib().mtp_linear_workspace_need(kind, M, N, K, _dt(t))
    if need <= 0:
        return None, 0
    ws = linear_workspace(dev, need)
    return ws.data_ptr(), ws.numel()


def linear_fwd(x2d: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], epilogue: int = EPI_NONE,
               want_pre: bool = True, lead: Optional[Tuple[int, ...]] = None
               ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(y, act) = epilogue(x2d @ w.T + bias).  x2d [M,K], w [N,K] contiguous, same dtype.  lead: leading
    dimensions (product M) to allocate the outputs with, so that a caller whose input was [*lead, K] gets
    [*lead, N] tensors that own their storage instead of views of [M, N] ones."""
    dev = _require_gpu(x2d, w, bias)
    if x2d.dim() != 2 or w.dim() != 2:
        raise ValueError(f"linear_fwd: x must be [M, K] and weight [N, K], got {tuple(x2d.shape)} and {tuple(w.shape)}")
    M, K = x2d.shape
    N, K2 = w.shape
    if K != K2:
        raise ValueError(f"linear_fwd: x is [*, {K}] but weight is [{N}, {K2}]")
    if w.dtype != x2d.dtype or (bias is not None and bias.dtype != x2d.dtype):
        raise TypeError("linear_fwd: x, weight and bias must share one dtype")
    if bias is not None and (bias.numel() != N or not bias.is_contiguous()):
        raise ValueError(f"linear_fwd: bias must be a contiguous [{N}] tensor, got {tuple(bias.shape)}")
    if epilogue == EPI_SWIGLU and N % 2:
        raise ValueError(f"linear_fwd: SwiGLU needs an even number of weight rows, got {N}")
    x2d, w = _contig(x2d), _contig(w)
    has_act = epilogue in (EPI_BIAS_GELU, EPI_SWIGLU, EPI_GELU)
    rows = (M,) if lead is None else tuple(lead)
    if lead is not None:
        prod = 1
        for d in rows:
            prod *= d
        if prod != M:
            raise ValueError(f"linear_fwd: leading dimensions {rows} do not hold {M} rows")
    y = torch.empty(rows + (N,), dtype=x2d.dtype, device=dev) if (want_pre or not has_act) else None
    act = None
    if has_act:
        act = torch.empty(rows + (N // 2 if epilogue == EPI_SWIGLU else N,), dtype=x2d.dtype, device=dev)
    with torch.cuda.device(dev):
        wsp, wsb = _ws_args(0, M, N, K, x2d, dev)
        rc = _lib.lib().mtp_linear_fwd_ws(_p(x2d), _p(w), _p(bias), _p(y), _p(act), wsp, wsb, M, N, K, _dt(x2d),
                                          epilogue, _stream(dev))
        if rc == -2 and y is None:
            # shapes served by the general kernel need the pre-activation buffer for SwiGLU
            y = torch.empty((M, N), dtype=x2d.dtype, device=dev)
            rc = _lib.lib().mtp_linear_fwd_ws(_p(x2d), _p(w), _p(bias), _p(y), _p(act), wsp, wsb, M, N, K, _dt(x2d),
                                              epilogue, _stream(dev))
            y = None
        _lib.check(rc, "mtp_linear_fwd")
    return y, act


def linear_dgrad(dy2d: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    dev = _require_gpu(dy2d, w)
    if dy2d.dim() != 2 or w.dim() != 2:
        raise ValueError(f"linear_dgrad: dy must be [M, N] and weight [N, K], got {tuple(dy2d.shape)} and {tuple(w.shape)}")
    M, N = dy2d.shape
    N2, K = w.shape
    if N != N2 or dy2d.dtype != w.dtype:
        raise ValueError("linear_dgrad: dy/weight mismatch")
    dy2d, w = _contig(dy2d), _contig(w)
    dx = torch.empty((M, K), dtype=dy2d.dtype, device=dev)
    with torch.cuda.device(dev):
        wsp, wsb = _ws_args(1, M, N, K, dy2d, dev)
        _lib.check(_lib.lib().mtp_linear_dgrad_ws(_p(dy2d), _p(w), _p(dx), wsp, wsb, M, N, K, _dt(dy2d), _stream(dev)),
                   "mtp_linear_dgrad")
    return dx


def linear_wgrad(dy2d: torch.Tensor, x2d: torch.Tensor, want_db: bool, out_dtype: Optional[torch.dtype] = None,
                 dw: Optional[torch.Tensor] = None, db: Optional[torch.Tensor] = None,
                 accumulate: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    dev = _require_gpu(dy2d, x2d, dw, db)
    if dy2d.dim() != 2 or x2d.dim() != 2:
        raise ValueError(f"linear_wgrad: dy must be [M, N] and x [M, K], got {tuple(dy2d.shape)} and {tuple(x2d.shape)}")
    M, N = dy2d.shape
    M2, K = x2d.shape
    if M != M2 or dy2d.dtype != x2d.dtype:
        raise ValueError("linear_wgrad: dy/x mismatch")
    dy2d, x2d = _contig(dy2d), _contig(x2d)
    out_dtype = out_dtype or (dw.dtype if dw is not None else dy2d.dtype)
    if dw is None:
        if accumulate:
            raise ValueError("linear_wgrad: accumulate needs an existing dw")
        dw = torch.empty((N, K), dtype=out_dtype, device=dev)
    if want_db and db is None:
        if accumulate:
            raise ValueError("linear_wgrad: accumulate needs an existing db")
        db = torch.empty((N,), dtype=out_dtype, device=dev)
    if dw.shape != (N, K) or not dw.is_contiguous() or dw.dtype != out_dtype:
        raise ValueError("linear_wgrad: dw must be a contiguous [N,K] tensor of the output dtype")
    if want_db and (db.numel() != N or not db.is_contiguous() or db.dtype != out_dtype):
        raise ValueError("linear_wgrad: db must be a contiguous [N] tensor of the output dtype")
    with torch.cuda.device(dev):
        wsp, wsb = _ws_args(2, M, N, K, dy2d, dev)
        _lib.check(_lib.lib().mtp_linear_wgrad_ws(_p(dy2d), _p(x2d), _p(dw), _p(db) if want_db else None, wsp, wsb, M, N,
                                                  K, _dt(dy2d), _DTYPES[out_dtype], int(accumulate), _stream(dev)),
                   "mtp_linear_wgrad")
    return dw, (db if want_db else None)


def linear_bwd(dy2d: torch.Tensor, x2d: torch.Tensor, w: torch.Tensor, want_db: bool,
               out_dtype: Optional[torch.dtype] = None, dw: Optional[torch.Tensor] = None,
               db: Optional[torch.Tensor] = None, accumulate: bool = False):
    """(dx, dw, db) = (dy w, dy^T x, sum of dy's rows): linear_dgrad and linear_wgrad of one layer as one call, and
    as one launch where the tiles of the two products together fill fewer rounds of workgroups than apart."""
    dev = _require_gpu(dy2d, x2d, w, dw, db)
    if dy2d.dim() != 2 or x2d.dim() != 2 or w.dim() != 2:
        raise ValueError("linear_bwd: dy [M, N], x [M, K] and weight [N, K] must be 2-d")
    M, N = dy2d.shape
    K = x2d.shape[1]
    if x2d.shape[0] != M or tuple(w.shape) != (N, K):
        raise ValueError(f"linear_bwd: shapes dy {tuple(dy2d.shape)}, x {tuple(x2d.shape)}, weight {tuple(w.shape)}")
    if not (dy2d.dtype == x2d.dtype == w.dtype):
        raise TypeError("linear_bwd: dy, x and weight must share a dtype")
    out_dtype = out_dtype or (dw.dtype if dw is not None else dy2d.dtype)
    if accumulate and dw is None:
        raise ValueError("linear_bwd: accumulate needs the gradient buffers")
    dy2d, x2d, w = _contig(dy2d), _contig(x2d), _contig(w)
    dx = torch.empty((M, K), dtype=dy2d.dtype, device=dev)
    if dw is None:
        dw = torch.empty((N, K), dtype=out_dtype, device=dev)
    if want_db and db is None:
        db = torch.empty((N,), dtype=out_dtype, device=dev)
    if tuple(dw.shape) != (N, K) or dw.dtype != out_dtype or not dw.is_contiguous():
        raise ValueError("linear_bwd: dw must be a contiguous [N, K] tensor of out_dtype")
    if want_db and (tuple(db.shape) != (N,) or db.dtype != out_dtype or not db.is_contiguous()):
        raise ValueError("linear_bwd: db must be a contiguous [N] tensor of out_dtype")
    with torch.cuda.device(dev):
        wsp, wsb = _ws_args(3, M, N, K, dy2d, dev)
        _lib.check(_lib.lib().mtp_linear_bwd_ws(_p(dy2d), _p(x2d), _p(w), _p(dx), _p(dw), _p(db) if want_db else None,
                                                wsp, wsb, M, N, K, _dt(dy2d), _DTYPES[out_dtype], int(accumulate),
                                                _stream(dev)), "mtp_linear_bwd")
    return dx, dw, (db if want_db else None)


def colsum(dy2d: torch.Tensor, db: torch.Tensor, accumulate: bool = False) -> torch.Tensor:
    """db (+)= dy2d.sum(0): the bias gradient alone, for a layer whose weight takes none."""
    dev = _require_gpu(dy2d, db)
    if dy2d.dim() != 2 or db.numel() != dy2d.shape[1] or not db.is_contiguous():
        raise ValueError(f"colsum: dy must be [M, N] and db a contiguous [N], got {tuple(dy2d.shape)} and {tuple(db.shape)}")
    if db.dtype not in (dy2d.dtype, torch.float32):
        raise TypeError("colsum: db must have dy's dtype or float32")
    dy2d = _contig(dy2d)
    M, N = dy2d.shape
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_linear_bias_grad(_p(dy2d), _p(db), M, N, _dt(dy2d), _DTYPES[db.dtype], int(accumulate),
                                                   _stream(dev)), "mtp_linear_bias_grad")
    return db


def activation_bwd(dact: torch.Tensor, y: torch.Tensor, epilogue: int) -> torch.Tensor:
    dev = _require_gpu(dact, y)
    if y.dim() != 2 or dact.dim() != 2 or dact.dtype != y.dtype:
        raise ValueError("activation_bwd: dact and y must be 2-D tensors of one dtype")
    M, N = y.shape
    if tuple(dact.shape) != (M, N // 2 if epilogue == EPI_SWIGLU else N):
        raise ValueError(f"activation_bwd: dact {tuple(dact.shape)} does not match y {tuple(y.shape)} for epilogue {epilogue}")
    dact, y = _contig(dact), _contig(y)
    dy = torch.empty_like(y)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_activation_bwd(_p(dact), _p(y), _p(dy), M, N, _dt(y), epilogue, _stream(dev)),
                   "mtp_activation_bwd")
    return dy


# --------------------------------------------------------------------------- embedding
def embedding_gather(ids: torch.Tensor, table: torch.Tensor, vocab_start: int, vocab_end: int,
                     oob_count: Optional[torch.Tensor] = None) -> torch.Tensor:
    dev = _require_gpu(ids, table, oob_count)
    if ids.dtype != torch.int64:
        raise TypeError(f"embedding ids must be int64, got {ids.dtype}")
    if table.dim() != 2 or not table.is_contiguous():
        raise ValueError("embedding table must be a contiguous [rows, dim] tensor")
    if table.shape[0] != vocab_end - vocab_start:
        raise ValueError("embedding table rows do not match the vocab range")
    flat = _contig(ids).view(-1)
    out = torch.empty((flat.numel(), table.shape[1]), dtype=table.dtype, device=dev)
    row_bytes = table.shape[1] * table.element_size()
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_embedding_gather(_p(flat), _p(table), _p(out), flat.numel(), row_bytes, vocab_start,
                                                   vocab_end, _p(oob_count), _stream(dev)), "mtp_embedding_gather")
    return out.view(*ids.shape, table.shape[1])


def embedding_bwd(ids: torch.Tensor, dout: torch.Tensor, rows: int, vocab_start: int, vocab_end: int,
                  out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Dense gradient [rows, dim] of the lookup, reproducible bit for bit.

    ``out`` given: the gradient is added onto it (e.g. the tied LM head's weight gradient);
    otherwise a zero-filled table of ``dtype`` (default: dout's) is created."""
    dev = _require_gpu(ids, dout, out)
    flat = _contig(ids).view(-1)
    dim = dout.shape[-1]
    d2 = _contig(dout).view(-1, dim)
    if flat.dtype != torch.int64:
        raise TypeError(f"embedding ids must be int64, got {flat.dtype}")
    if d2.shape[0] != flat.numel():
        raise ValueError(f"embedding_bwd: {d2.shape[0]} gradient rows for {flat.numel()} ids")
    if rows != vocab_end - vocab_start:
        raise ValueError("embedding_bwd: table rows do not match the vocab range")
    if out is None:
        out = torch.zeros((rows, dim), dtype=dtype or d2.dtype, device=dev)
    elif tuple(out.shape) != (rows, dim) or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{rows}, {dim}] tensor")
    lib = _lib.lib()
    ws = torch.empty((max(int(lib.mtp_embedding_bwd_workspace_bytes(flat.numel(), dim)), 16),), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.mtp_embedding_bwd(_p(flat), _p(d2), _p(out), _p(ws), ws.numel(), flat.numel(), dim, _dt(d2),
                                         _dt(out), vocab_start, vocab_end, _stream(dev)), "mtp_embedding_bwd")
    return out


# --------------------------------------------------------------------------- cross entropy
def vocab_ce_fwd(logits2d: torch.Tensor, target1d: torch.Tensor, vocab_start: int):
    """-> (loss, row_max, row_sumexp, pred), all fp32 [n_rows]."""
    dev = _require_gpu(logits2d, target1d)
    if target1d.dtype != torch.int64:
        raise TypeError(f"cross-entropy targets must be int64, got {target1d.dtype}")
    if not logits2d.is_contiguous():
        raise ValueError("vocab_parallel_cross_entropy needs contiguous logits")
    n, v = logits2d.shape
    if target1d.numel() != n:
        raise ValueError(f"target has {target1d.numel()} entries for {n} logits rows")
    target1d = _contig(target1d)
    out = torch.empty((4, n), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_vocab_ce_fwd(_p(logits2d), _p(target1d), _p(out[0]), _p(out[1]), _p(out[2]),
                                               _p(out[3]), n, v, vocab_start, _dt(logits2d), _stream(dev)),
                   "mtp_vocab_ce_fwd")
    return out[0], out[1], out[2], out[3]


def vocab_ce_bwd_(logits2d: torch.Tensor, target1d: torch.Tensor, row_max: Optional[torch.Tensor],
                  row_sumexp: Optional[torch.Tensor], grad_out: Optional[torch.Tensor], vocab_start: int) -> torch.Tensor:
    """In place: logits2d <- (softmax - onehot) * grad_out.  Returns logits2d.

    row_max = row_sumexp = None: logits2d already holds the softmax."""
    dev = _require_gpu(logits2d, target1d, row_max, row_sumexp, grad_out)
    if target1d.dtype != torch.int64:
        raise TypeError(f"cross-entropy targets must be int64, got {target1d.dtype}")
    if not logits2d.is_contiguous():
        raise ValueError("vocab_parallel_cross_entropy needs contiguous logits")
    n, v = logits2d.shape
    if target1d.numel() != n:
        raise ValueError(f"target has {target1d.numel()} entries for {n} logits rows")
    for name, t in (("row_max", row_max), ("row_sumexp", row_sumexp)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous()):
            raise ValueError(f"vocab_ce_bwd_: {name} must be contiguous fp32 [{n}]")
    if grad_out is not None:
        grad_out = _contig(grad_out.to(torch.float32))
        if grad_out.numel() != n:
            raise ValueError(f"grad_out has {grad_out.numel()} entries for {n} logits rows")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_vocab_ce_bwd(_p(logits2d), _p(_contig(target1d)), _p(row_max), _p(row_sumexp),
                                               _p(grad_out), n, v, vocab_start, _dt(logits2d), _stream(dev)),
                   "mtp_vocab_ce_bwd")
    return logits2d


def vocab_ce_fused_max_vocab(dtype: torch.dtype) -> int:
    """Longest row the one-launch forward+backward kernel keeps in registers."""
    return int(_lib.lib().mtp_vocab_ce_fwd_bwd_max_vocab(_DTYPES[dtype]))


def vocab_ce_fwd_bwd_(logits2d: torch.Tensor, target1d: torch.Tensor, vocab_start: int,
                      grad_rows: Optional[torch.Tensor] = None, grad_scale: float = 1.0):
    """One launch: -> (loss, row_max, row_sumexp, pred) and, in place,
    logits2d <- (softmax - onehot) * grad_rows[i] * grad_scale."""
    dev = _require_gpu(logits2d, target1d, grad_rows)
    if target1d.dtype != torch.int64:
        raise TypeError(f"cross-entropy targets must be int64, got {target1d.dtype}")
    if not logits2d.is_contiguous():
        raise ValueError("vocab_parallel_cross_entropy needs contiguous logits")
    n, v = logits2d.shape
    if target1d.numel() != n:
        raise ValueError(f"target has {target1d.numel()} entries for {n} logits rows")
    if grad_rows is not None:
        grad_rows = _contig(grad_rows.to(torch.float32))
        if grad_rows.numel() != n:
            raise ValueError(f"grad_rows has {grad_rows.numel()} entries for {n} logits rows")
    target1d = _contig(target1d)
    out = torch.empty((4, n), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_vocab_ce_fwd_bwd(_p(logits2d), _p(target1d), _p(grad_rows), float(grad_scale),
                                                   _p(out[0]), _p(out[1]), _p(out[2]), _p(out[3]), n, v,
                                                   vocab_start, _dt(logits2d), _stream(dev)),
                   "mtp_vocab_ce_fwd_bwd")
    return out[0], out[1], out[2], out[3]


def vocab_ce_rescale_(grad2d: torch.Tensor, grad_rows: torch.Tensor, assumed: float) -> torch.Tensor:
    """In place: rows of grad2d whose grad_rows[i] differs from ``assumed`` are scaled by grad_rows[i]/assumed."""
    dev = _require_gpu(grad2d, grad_rows)
    n, v = grad2d.shape
    grad_rows = _contig(grad_rows.to(torch.float32))
    if grad_rows.numel() != n:
        raise ValueError(f"grad_rows has {grad_rows.numel()} entries for {n} rows")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_vocab_ce_rescale(_p(grad2d), _p(grad_rows), float(assumed), n, v, _dt(grad2d),
                                                   _stream(dev)), "mtp_vocab_ce_rescale")
    return grad2d


# --------------------------------------------------------------------------- decode
def gemv_workspace(B: int, N: int, K: int, epilogue: int, device) -> Optional[torch.Tensor]:
    """Zero-filled scratch for ``gemv(..., workspace=)`` or None when this shape runs without one.  One
    workspace serves any number of launches, of any shapes, that do not overlap: take the largest need (the
    counters every launch leaves zero sit in its first 8 KiB whatever the shape)."""
    need = int(_lib.lib().mtp_gemv_workspace_bytes(B, N, K, epilogue))
    return torch.zeros((need,), dtype=torch.uint8, device=device) if need else None


def _decode_dtype(what: str, *ts: torch.Tensor) -> torch.dtype:
    dt = ts[0].dtype
    if dt not in (torch.bfloat16, torch.float16) or any(t.dtype != dt for t in ts if t is not None):
        raise TypeError(f"{what} takes bfloat16 or float16 tensors of one dtype, got {[t.dtype for t in ts if t is not None]}")
    return dt


def _gemv_shapes(what: str, x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor]):
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"{what}: x must be [B, K] and weight [N, K], got {tuple(x.shape)} and {tuple(w.shape)}")
    if bias is not None and (bias.numel() != w.shape[0] or not bias.is_contiguous()):
        raise ValueError(f"{what}: bias must be a contiguous [{w.shape[0]}] tensor, got {tuple(bias.shape)}")
    return x.shape[0], w.shape[0], x.shape[1]


def gemv(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, epilogue: int = EPI_NONE,
         workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    dev = _require_gpu(x, w, bias, workspace)
    dt = _decode_dtype("gemv", x, w, bias)
    B, N, K = _gemv_shapes("gemv", x, w, bias)
    x, w = _contig(x), _contig(w)
    y = torch.empty((B, N // 2 if epilogue == EPI_SWIGLU else N), dtype=dt, device=dev)
    wbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_gemv_ws(_p(x), _p(w), _p(bias), _p(y), _p(workspace), wbytes, B, N, K, epilogue,
                                          _DTYPES[dt], _stream(dev)), "mtp_gemv")
    return y


def gemv_pair(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, bias1: Optional[torch.Tensor] = None,
              bias2: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """``(x @ w1.T (+ bias1), swiglu(x @ w2.T (+ bias2)))``: two products over the same rows in one call (one
    launch above 16 rows, the two launches of ``gemv`` otherwise)."""
    dev = _require_gpu(x, w1, w2, bias1, bias2, workspace)
    dt = _decode_dtype("gemv_pair", x, w1, bias1)
    _decode_dtype("gemv_pair", x, w2, bias2)
    B, N1, K = _gemv_shapes("gemv_pair", x, w1, bias1)
    _, N2, K2 = _gemv_shapes("gemv_pair", x, w2, bias2)
    if K2 != K or N2 % 2:
        raise ValueError(f"gemv_pair: second weight must be [2 * I, {K}], got {tuple(w2.shape)}")
    x, w1, w2 = _contig(x), _contig(w1), _contig(w2)
    y1 = torch.empty((B, N1), dtype=dt, device=dev)
    act2 = torch.empty((B, N2 // 2), dtype=dt, device=dev)
    wbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_gemv_pair(_p(x), _p(w1), _p(bias1), _p(y1), N1, _p(w2), _p(bias2), _p(act2), N2,
                                            _p(workspace), wbytes, B, K, _DTYPES[dt], _stream(dev)), "mtp_gemv_pair")
    return y1, act2


def gemv_norm_fits(B: int, K: int) -> bool:
    """Whether ``gemv_fused`` can take the RMSNorm of a [B, K] input inside the product (B K <= 8 x 4096, K % 512 == 0, K <= 8192)."""
    return bool(_lib.lib().mtp_gemv_norm_fits(B, K))


def gemv_fused(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, epilogue: int = EPI_NONE,
               norm_weight: Optional[torch.Tensor] = None, sumsq_in: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None, want_sumsq: bool = False,
               workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """``gemv`` with a decoder block's surroundings folded in.

    ``norm_weight`` + ``sumsq_in`` (fp32 [B, K/16]): the product is taken with ``RMSNorm(x)``;
    ``residual`` ([B, N]): ``y = dtype(dtype(x W^T + bias) + residual)`` (``out`` may be ``residual``);
    ``want_sumsq``: also returns fp32 [B, ceil(N/16)] sums of squares of ``y``, the next norm's ``sumsq_in``.
    Returns ``y`` or ``(y, sumsq)``."""
    dev = _require_gpu(x, w, bias, workspace, norm_weight, sumsq_in, residual, out)
    dt = _decode_dtype("gemv_fused", x, w, bias)
    B, N, K = _gemv_shapes("gemv_fused", x, w, bias)
    x, w = _contig(x), _contig(w)
    n_out = N // 2 if epilogue == EPI_SWIGLU else N
    if norm_weight is not None:
        if sumsq_in is None or sumsq_in.dtype != torch.float32 or tuple(sumsq_in.shape) != (B, K // 16) \
                or not sumsq_in.is_contiguous():
            raise ValueError(f"gemv_fused: sumsq_in must be contiguous fp32 [{B}, {K // 16}]")
        if norm_weight.dtype != dt or norm_weight.numel() != K or not norm_weight.is_contiguous():
            raise ValueError(f"gemv_fused: norm_weight must be contiguous {dt} [{K}]")
    if residual is not None and (residual.dtype != dt or tuple(residual.shape) != (B, n_out) or not residual.is_contiguous()):
        raise ValueError(f"gemv_fused: residual must be contiguous {dt} [{B}, {n_out}]")
    if out is None:
        out = torch.empty((B, n_out), dtype=dt, device=dev)
    elif out.dtype != dt or tuple(out.shape) != (B, n_out) or not out.is_contiguous():
        raise ValueError(f"gemv_fused: out must be contiguous {dt} [{B}, {n_out}]")
    sumsq = torch.empty((B, (N + 15) // 16), dtype=torch.float32, device=dev) if want_sumsq else None
    wbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_gemv_fused(_p(x), _p(w), _p(bias), _p(out), _p(norm_weight), _p(sumsq_in), float(eps),
                                             _p(residual), _p(sumsq), _p(workspace), wbytes, B, N, K, epilogue,
                                             _DTYPES[dt], _stream(dev)), "mtp_gemv_fused")
    return (out, sumsq) if want_sumsq else out


def argmax_workspace(B: int, N: int, K: int, dev: torch.device) -> torch.Tensor:
    """Scratch for ``gemv_argmax`` on shapes up to [B, K] x [N, K] (nothing in it needs clearing)."""
    need = _lib.lib().mtp_gemv_argmax_workspace_bytes(B, N, K)
    return torch.empty((max(int(need), 8),), dtype=torch.uint8, device=dev)


def gemv_argmax(x: torch.Tensor, w: torch.Tensor, workspace: Optional[torch.Tensor] = None):
    """-> (idx int64 [B], maxval fp32 [B]) without materialising the logits."""
    dev = _require_gpu(x, w, workspace)
    dt = _decode_dtype("gemv_argmax", x, w)
    B, N, K = _gemv_shapes("gemv_argmax", x, w, None)
    x, w = _contig(x), _contig(w)
    need = _lib.lib().mtp_gemv_argmax_workspace_bytes(B, N, K)
    if workspace is None:
        workspace = argmax_workspace(B, N, K, dev)
    idx = torch.empty((B,), dtype=torch.int64, device=dev)
    val = torch.empty((B,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_gemv_argmax(_p(x), _p(w), _p(idx), _p(val), _p(workspace),
                                              workspace.numel() * workspace.element_size(), B, N, K,
                                              _DTYPES[dt], _stream(dev)), "mtp_gemv_argmax")
    return idx, val


def argmax_rows(logits: torch.Tensor) -> torch.Tensor:
    dev = _require_gpu(logits)
    l2 = _contig(logits).view(-1, logits.shape[-1])
    idx = torch.empty((l2.shape[0],), dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_argmax_rows(_p(l2), _p(idx), l2.shape[0], l2.shape[1], _dt(l2), _stream(dev)),
                   "mtp_argmax_rows")
    return idx.view(logits.shape[:-1])


def sample_top_k_top_p(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0, top_p: float = 0.0,
                       uniforms: Optional[torch.Tensor] = None, want_filtered: bool = False,
                       workspace: Optional[torch.Tensor] = None):
    """-> (tokens int64 [B] or None, filtered fp32 [B, V] or None).

    tokens are drawn when ``uniforms`` (fp32 [B], values in [0, 1)) is given."""
    dev = _require_gpu(logits, uniforms, workspace)
    if logits.dim() != 2:
        raise ValueError("sample_top_k_top_p takes [B, V] logits")
    logits = _contig(logits)
    B, V = logits.shape
    tokens = filtered = None
    if uniforms is not None:
        uniforms = _contig(uniforms.to(torch.float32)).view(-1)
        if uniforms.numel() != B:
            raise ValueError(f"uniforms has {uniforms.numel()} entries for {B} rows")
        tokens = torch.empty((B,), dtype=torch.int64, device=dev)
    if want_filtered:
        filtered = torch.empty((B, V), dtype=torch.float32, device=dev)
    if tokens is None and filtered is None:
        raise ValueError("nothing to compute: give uniforms and/or want_filtered=True")
    lib = _lib.lib()
    need = int(lib.mtp_sample_workspace_bytes(B))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty((max(need, 8),), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.mtp_sample_top_k_top_p(_p(logits), _dt(logits), B, V, float(temperature), int(top_k),
                                              float(top_p), _p(uniforms), _p(tokens), _p(filtered), _p(workspace),
                                              workspace.numel() * workspace.element_size(), _stream(dev)),
                   "mtp_sample_top_k_top_p")
    return tokens, filtered


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
            want_residual: bool = False):
    """-> y, or (y, h) with ``want_residual``: h = x (+ residual), y = weight * (h * rsqrt(mean(h^2) + eps))."""
    dev = _require_gpu(x, weight, residual)
    x = _contig(x)
    dim = x.shape[-1]
    if weight.shape != (dim,) or weight.dtype != x.dtype:
        raise ValueError(f"rmsnorm: weight {tuple(weight.shape)} {weight.dtype} for rows of {dim} {x.dtype}")
    if residual is not None:
        residual = _contig(residual)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError("rmsnorm: residual must match x")
    y = torch.empty_like(x)
    h = torch.empty_like(x) if want_residual else None
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_rmsnorm(_p(x), _p(residual), _p(_contig(weight)), _p(y), _p(h), x.numel() // dim, dim,
                                          float(eps), _dt(x), _stream(dev)), "mtp_rmsnorm")
    return (y, h) if want_residual else y


def rope_kv_append(qkv: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                   k_cache: torch.Tensor, v_cache: torch.Tensor, n_q_heads: int) -> torch.Tensor:
    """Rotates the new q and k heads of ``qkv`` [B, (n_q + 2 n_kv) * 128], writes k and v into row
    ``positions[b]`` of the caches [B, n_kv, max_len, 128] and returns the rotated q [B, n_q, 128]."""
    dev = _require_gpu(qkv, cos_table, sin_table, positions, k_cache, v_cache)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("rope_kv_append: caches must be contiguous [B, n_kv_heads, max_len, head_dim] of one shape")
    B, n_kv, max_len, hd = k_cache.shape
    qkv = _contig(qkv)
    if qkv.shape != (B, (n_q_heads + 2 * n_kv) * hd):
        raise ValueError(f"rope_kv_append: qkv {tuple(qkv.shape)} for {n_q_heads}+2*{n_kv} heads of {hd}")
    if cos_table.shape != sin_table.shape or cos_table.dim() != 2 or cos_table.shape[1] != hd:
        raise ValueError("rope_kv_append: cos / sin tables must be [max_positions, head_dim]")
    for t in (cos_table, sin_table, k_cache, v_cache):
        if t.dtype != qkv.dtype:
            raise ValueError("rope_kv_append: all tensors must share the dtype of qkv")
    if positions.dtype != torch.int64 or positions.numel() != B:
        raise ValueError("rope_kv_append: positions must be int64 [B]")
    q = torch.empty((B, n_q_heads, hd), dtype=qkv.dtype, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_rope_kv_append(_p(qkv), _p(_contig(cos_table)), _p(_contig(sin_table)),
                                                 _p(_contig(positions)), _p(q), _p(k_cache), _p(v_cache), B,
                                                 n_q_heads, n_kv, hd, max_len, cos_table.shape[0], _dt(qkv),
                                                 _stream(dev)), "mtp_rope_kv_append")
    return q


def attn_decode_workspace_bytes(B: int, n_q_heads: int, n_kv_heads: int, len_bound: int) -> int:
    return int(_lib.lib().mtp_attn_decode_workspace_bytes(B, n_q_heads, n_kv_heads, len_bound))


def attn_workspace(B: int, n_q_heads: int, n_kv_heads: int, len_bound: int, device) -> torch.Tensor:
    """Zero-filled scratch for ``attn_decode`` / ``attn_decode_append`` (the kernels need its head zero before
    the first use and leave it zero)."""
    return torch.zeros((max(attn_decode_workspace_bytes(B, n_q_heads, n_kv_heads, len_bound), 16),), dtype=torch.uint8,
                       device=device)


def _attn_workspace(workspace, B, n_q, n_kv, len_bound, dev):
    need = attn_decode_workspace_bytes(B, n_q, n_kv, len_bound)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = attn_workspace(B, n_q, n_kv, len_bound, dev)
    return workspace


def attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                scale: Optional[float] = None, len_bound: Optional[int] = None,
                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new position per row over the first ``lens[b]`` cached tokens.
    q [B, n_q, 128], caches [B, n_kv, max_len, 128] -> [B, n_q, 128]."""
    dev = _require_gpu(q, k_cache, v_cache, lens, workspace)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("attn_decode: caches must be contiguous [B, n_kv_heads, max_len, head_dim] of one shape")
    B, n_kv, max_len, hd = k_cache.shape
    q = _contig(q)
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != hd:
        raise ValueError(f"attn_decode: q {tuple(q.shape)} against caches {tuple(k_cache.shape)}")
    if not (q.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError("attn_decode: q and the caches must share a dtype")
    if lens.dtype != torch.int64 or lens.numel() != B:
        raise ValueError("attn_decode: lens must be int64 [B]")
    n_q = q.shape[1]
    len_bound = max_len if len_bound is None else int(len_bound)
    scale = hd ** -0.5 if scale is None else float(scale)
    lib = _lib.lib()
    workspace = _attn_workspace(workspace, B, n_q, n_kv, len_bound, dev)
    out = torch.empty_like(q)
    wbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        _lib.check(lib.mtp_attn_decode(_p(q), _p(k_cache), _p(v_cache), _p(_contig(lens)), _p(out), _p(workspace),
                                       wbytes, B, n_q, n_kv, hd, max_len, len_bound, scale, _dt(q), _stream(dev)),
                   "mtp_attn_decode")
    return out


def attn_decode_append(qkv: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, n_q_heads: int, scale: Optional[float] = None,
                       len_bound: Optional[int] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rope_kv_append`` then ``attn_decode`` over ``positions + 1`` tokens, as one launch.
    ``workspace``: from ``attn_workspace`` (zero-filled once, reusable)."""
    dev = _require_gpu(qkv, cos_table, sin_table, positions, k_cache, v_cache, workspace)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("attn_decode_append: caches must be contiguous [B, n_kv_heads, max_len, head_dim] of one shape")
    B, n_kv, max_len, hd = k_cache.shape
    qkv = _contig(qkv)
    if qkv.shape != (B, (n_q_heads + 2 * n_kv) * hd):
        raise ValueError(f"attn_decode_append: qkv {tuple(qkv.shape)} for {n_q_heads}+2*{n_kv} heads of {hd}")
    if cos_table.shape != sin_table.shape or cos_table.dim() != 2 or cos_table.shape[1] != hd:
        raise ValueError("attn_decode_append: cos / sin tables must be [max_positions, head_dim]")
    for t in (cos_table, sin_table, k_cache, v_cache):
        if t.dtype != qkv.dtype:
            raise ValueError("attn_decode_append: all tensors must share the dtype of qkv")
    if positions.dtype != torch.int64 or positions.numel() != B:
        raise ValueError("attn_decode_append: positions must be int64 [B]")
    len_bound = max_len if len_bound is None else int(len_bound)
    scale = hd ** -0.5 if scale is None else float(scale)
    workspace = _attn_workspace(workspace, B, n_q_heads, n_kv, len_bound, dev)
    out = torch.empty((B, n_q_heads, hd), dtype=qkv.dtype, device=dev)
    wbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mtp_attn_decode_append(_p(qkv), _p(_contig(cos_table)), _p(_contig(sin_table)),
                                                     _p(_contig(positions)), _p(k_cache), _p(v_cache), _p(out),
                                                     _p(workspace), wbytes, B, n_q_heads, n_kv, hd, max_len,
                                                     cos_table.shape[0], len_bound, scale, _dt(qkv), _stream(dev)),
                   "mtp_attn_decode_append")
    return out


# --------------------------------------------------------------------------- paged key/value cache
class PagedPlan(NamedTuple):
    """What ``paged_plan`` hands out for one step (all on the device)."""
    slots: torch.Tensor        # int64 [tokens]: cache slot of each new token, -1: none
    positions: torch.Tensor    # int64 [tokens]: its position in its request, -1: none
    cu: torch.Tensor           # int64 [requests + 1]: where each request's tokens start
    kv_lens: torch.Tensor      # int64 [requests]: tokens cached after the step, 0 for a refused request
    granted: torch.Tensor      # bool [requests]: False: refused, nothing of it has changed
    held: torch.Tensor         # int32 [requests]: pages each request holds after the step
    free_count: torch.Tensor   # int32 [1]: pages left on the free list


def _index(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, shape: Tuple[int, ...]) -> torch.Tensor:
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{what}: {name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    return _contig(t)


def _own(what: str, name: str, t: torch.Tensor) -> torch.Tensor:
    """A tensor that the call writes into: it must be the caller's memory as it is."""
    if not t.is_contiguous():
        raise ValueError(f"{what}: {name} is written in place and must be contiguous")
    return t


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and on a 16-byte boundary (a slice of a larger tensor may start anywhere)."""
    if t is None:
        return None
    t = _contig(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


def paged_plan(lens: torch.Tensor, new_lens: torch.Tensor, held: torch.Tensor, block_tables: torch.Tensor,
               free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int, tokens: int) -> PagedPlan:
    """Pages, slots and positions of the ``new_lens[r]`` tokens that arrive for each request, one launch.

    ``block_tables`` int32 [requests, max_pages] gets the new pages behind the ``held[r]`` ones (in place); they come
    from the top of ``free_pages`` int32, of which ``free_count`` int32 [1] are free.  ``tokens``: length of the
    per-token outputs, at least the new tokens of all requests.  The caller goes on with the returned ``held`` and
    ``free_count``, and with ``lens + new_lens`` where ``granted``."""
    dev = _require_gpu(lens, new_lens, held, block_tables, free_pages, free_count)
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32:
        raise ValueError("paged_plan: block_tables must be int32 [requests, max_pages]")
    R, max_pages = block_tables.shape
    lens = _index("paged_plan", "lens", lens, torch.int64, (R,))
    new_lens = _index("paged_plan", "new_lens", new_lens, torch.int64, (R,))
    held = _index("paged_plan", "held", held, torch.int32, (R,))
    free_pages = _index("paged_plan", "free_pages", free_pages, torch.int32, (free_pages.numel(),))
    free_count = _index("paged_plan", "free_count", free_count, torch.int32, (1,))
    _own("paged_plan", "block_tables", block_tables)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"paged_plan: tokens={tokens}")
    # two allocations for seven small results: the allocator costs more than the kernel
    wide = torch.empty((2 * tokens + 2 * R + 1,), dtype=torch.int64, device=dev)
    narrow = torch.empty((2 * R + 1,), dtype=torch.int32, device=dev)
    new_held, count, flags = narrow.split((R, 1, R))
    plan = PagedPlan(*wide.split((tokens, tokens, R + 1, R)), flags.view(torch.bool)[:R], new_held, count)
    with _device(dev):
        _lib.check(_lib.lib().mtp_paged_plan(_p(lens), _p(new_lens), _p(held), _p(block_tables), _p(free_pages),
                                             _p(free_count), _p(plan.slots), _p(plan.positions), _p(plan.cu),
                                             _p(plan.kv_lens), _p(plan.granted), _p(plan.held), _p(plan.free_count), R,
                                             max_pages, int(page_size), free_pages.numel(), tokens, _stream(dev)),
                   "mtp_paged_plan")
    return plan


def paged_release(finished: torch.Tensor, held: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor) -> None:
    """Pages of the requests with ``finished[r]`` (bool [requests]) go back on the free list; ``held``, ``free_pages``
    and ``free_count`` are updated in place."""
    dev = _require_gpu(finished, held, block_tables, free_pages, free_count)
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32:
        raise ValueError("paged_release: block_tables must be int32 [requests, max_pages]")
    R, max_pages = block_tables.shape
    finished = _index("paged_release", "finished", finished, torch.bool, (R,))
    for name, t, n in (("held", held, R), ("free_pages", free_pages, free_pages.numel()), ("free_count", free_count, 1)):
        _index("paged_release", name, _own("paged_release", name, t), torch.int32, (n,))
    with _device(dev):
        _lib.check(_lib.lib().mtp_paged_release(_p(finished), _p(held), _p(_contig(block_tables)), _p(free_pages),
                                                _p(free_count), R, max_pages, free_pages.numel(), _stream(dev)),
                   "mtp_paged_release")


def _rotary_args(what: str, qkv, cos_table, sin_table, positions, n_q_heads, n_kv_heads, q_weight, k_weight):
    """Checks shared by the three forms -> (qkv, cos, sin, positions, q_weight, k_weight, T, head_dim)."""
    if cos_table.dim() != 2 or cos_table.shape != sin_table.shape or cos_table.dtype != sin_table.dtype:
        raise ValueError(f"{what}: cos / sin tables must be [max_positions, head_dim] of one type")
    hd = cos_table.shape[1]
    if cos_table.dtype not in (torch.float32, qkv.dtype):
        raise TypeError(f"{what}: tables must be float32 or of the type of qkv, got {cos_table.dtype}")
    if qkv.dim() != 2 or n_q_heads <= 0 or n_kv_heads <= 0 or qkv.shape[1] != (n_q_heads + 2 * n_kv_heads) * hd:
        raise ValueError(f"{what}: qkv {tuple(qkv.shape)} for {n_q_heads}+2*{n_kv_heads} heads of {hd}")
    T = qkv.shape[0]
    positions = _index(what, "positions", positions, torch.int64, (T,))
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (hd,) or w.dtype != qkv.dtype):
            raise ValueError(f"{what}: norm weight {tuple(w.shape)} {w.dtype} for heads of {hd} {qkv.dtype}")
    return (_aligned(qkv), _aligned(cos_table), _aligned(sin_table), positions, _aligned(q_weight), _aligned(k_weight), T,
            hd)


def _kv_heads(what: str, qkv: torch.Tensor, cos_table: torch.Tensor, n_q_heads: int) -> int:
    if qkv.dim() != 2 or cos_table.dim() != 2 or cos_table.shape[1] == 0:
        raise ValueError(f"{what}: qkv must be [T, heads * head_dim] and the tables [max_positions, head_dim]")
    rest = qkv.shape[1] // cos_table.shape[1] - n_q_heads
    if rest <= 0 or rest % 2:
        raise ValueError(f"{what}: qkv {tuple(qkv.shape)} is not {n_q_heads} query heads and as many key as value heads of "
                         f"{cos_table.shape[1]}")
    return rest // 2


def qk_norm_rope(qkv: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                 n_q_heads: int, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (q [T, n_q, head_dim], k [T, n_kv, head_dim]): RMSNorm of each query and key head of ``qkv``
    [T, (n_q + 2 n_kv) * head_dim] with ``q_weight`` / ``k_weight`` [head_dim] (None: no norm), then the rotary embedding
    at ``positions`` int64 [T].  fp32 inside, rounded once.  ``mpu.qk_norm_rotary`` is the form with a gradient."""
    dev = _require_gpu(qkv, cos_table, sin_table, positions, q_weight, k_weight)
    n_kv = _kv_heads("qk_norm_rope", qkv, cos_table, n_q_heads)
    qkv, cos, sin, positions, qw, kw, T, hd = _rotary_args("qk_norm_rope", qkv, cos_table, sin_table, positions, n_q_heads,
                                                           n_kv, q_weight, k_weight)
    q = torch.empty((T, n_q_heads, hd), dtype=qkv.dtype, device=dev)
    k = torch.empty((T, n_kv, hd), dtype=qkv.dtype, device=dev)
    with _device(dev):
        _lib.check(_lib.lib().mtp_qk_norm_rope(_p(qkv), _p(cos), _p(sin), _dt(cos), _p(positions), _p(qw), _p(kw), _p(q),
                                               _p(k), T, n_q_heads, n_kv, hd, cos.shape[0], float(eps), _dt(qkv),
                                               _stream(dev)), "mtp_qk_norm_rope")
    return q, k


def qk_norm_rope_bwd(dq: Optional[torch.Tensor], dk: Optional[torch.Tensor], dv: Optional[torch.Tensor], qkv: torch.Tensor,
                     cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                     q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     n_q_heads: Optional[int] = None, want_dw: bool = True):
    """-> (dqkv, dq_weight or None, dk_weight or None).  ``dq`` [T, n_q, head_dim], ``dk`` and ``dv`` [T, n_kv, head_dim]
    (None: no gradient); ``dv`` is copied into the values' place of ``dqkv``.  ``n_q_heads`` is needed without ``dq``."""
    dev = _require_gpu(qkv, dq, dk, dv, cos_table, sin_table, positions, q_weight, k_weight)
    if n_q_heads is None:
        if dq is None or dq.dim() != 3:
            raise ValueError("qk_norm_rope_bwd: n_q_heads is needed without dq [T, n_q, head_dim]")
        n_q_heads = dq.shape[1]
    n_kv = _kv_heads("qk_norm_rope_bwd", qkv, cos_table, n_q_heads)
    qkv, cos, sin, positions, qw, kw, T, hd = _rotary_args("qk_norm_rope_bwd", qkv, cos_table, sin_table, positions,
                                                           n_q_heads, n_kv, q_weight, k_weight)
    for name, g, n in (("dq", dq, n_q_heads), ("dk", dk, n_kv), ("dv", dv, n_kv)):
        if g is not None and (g.shape != (T, n, hd) or g.dtype != qkv.dtype):
            raise ValueError(f"qk_norm_rope_bwd: {name} must be {qkv.dtype} {[T, n, hd]}, got {g.dtype} {list(g.shape)}")
    dq, dk, dv = _aligned(dq), _aligned(dk), _aligned(dv)
    dqkv = torch.empty_like(qkv)
    dqw = torch.empty_like(qw) if want_dw and qw is not None else None
    dkw = torch.empty_like(kw) if want_dw and kw is not None else None
    if T == 0:
        return dqkv, None if dqw is None else dqw.zero_(), None if dkw is None else dkw.zero_()
    lib = _lib.lib()
    ws = None
    if dqw is not None or dkw is not None:
        need = lib.mtp_qk_norm_rope_bwd_workspace_bytes(T, n_q_heads, n_kv, hd)
        ws = torch.empty((max(int(need), 4),), dtype=torch.uint8, device=dev)
    with _device(dev):
        _lib.check(lib.mtp_qk_norm_rope_bwd(_p(dq), _p(dk), _p(dv), _p(qkv), _p(cos), _p(sin), _dt(cos), _p(positions),
                                            _p(qw), _p(kw), _p(dqkv), _p(dqw), _p(dkw), _p(ws),
                                            0 if ws is None else ws.numel(), T, n_q_heads, n_kv, hd, cos.shape[0],
                                            float(eps), _dt(qkv), _stream(dev)), "mtp_qk_norm_rope_bwd")
    return dqkv, dqw, dkw


def _pages(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{what}: caches must be contiguous [n_pages, n_kv_heads, page_size, head_dim] of one shape")
    return k_cache.shape


def qk_norm_rope_append(qkv: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                        slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, n_q_heads: int,
                        q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                        eps: float = 1e-6) -> torch.Tensor:
    """``qk_norm_rope`` for serving: returns q [T, n_q, head_dim] and writes the keys and the values of each row to
    ``slots[t]`` of the caches [n_pages, n_kv, page_size, head_dim] (-1: nowhere; no slot twice, or parts of either row
    stay)."""
    dev = _require_gpu(qkv, cos_table, sin_table, positions, slots, k_cache, v_cache, q_weight, k_weight)
    n_pages, n_kv, page_size, hd = _pages("qk_norm_rope_append", k_cache, v_cache)
    if cos_table.dim() != 2 or cos_table.shape[1] != hd or k_cache.dtype != qkv.dtype or v_cache.dtype != qkv.dtype:
        raise ValueError("qk_norm_rope_append: caches and tables must match the heads and the type of qkv")
    qkv, cos, sin, positions, qw, kw, T, hd = _rotary_args("qk_norm_rope_append", qkv, cos_table, sin_table, positions,
                                                           n_q_heads, n_kv, q_weight, k_weight)
    slots = _index("qk_norm_rope_append", "slots", slots, torch.int64, (T,))
    q = torch.empty((T, n_q_heads, hd), dtype=qkv.dtype, device=dev)
    with _device(dev):
        _lib.check(_lib.lib().mtp_qk_norm_rope_append(_p(qkv), _p(cos), _p(sin), _dt(cos), _p(positions), _p(slots), _p(qw),
                                                      _p(kw), _p(q), _p(k_cache), _p(v_cache), T, n_q_heads, n_kv, hd,
                                                      cos.shape[0], n_pages, page_size, float(eps), _dt(qkv),
                                                      _stream(dev)), "mtp_qk_norm_rope_append")
    return q


def attn_paged_workspace(device) -> torch.Tensor:
    """Scratch for ``attn_paged``, any shape (the kernels need its head zero before the first use and leave it zero).
    Launches that may overlap in time need one each."""
    ws = torch.empty((int(_lib.lib().mtp_attn_paged_workspace_bytes()),), dtype=torch.uint8, device=device)
    ws[:4096].zero_()
    return ws


def attn_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
               cu: torch.Tensor, kv_lens: torch.Tensor, scale: Optional[float] = None, max_new: Optional[int] = None,
               len_bound: Optional[int] = None, workspace: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of each request's new tokens over its pages, any mix of single tokens, drafts and
    prompts.  q [T, n_q, head_dim]; rows cu[r] .. cu[r+1]-1 are request r's, whose last one is token kv_lens[r] - 1 of
    the pages that row r of ``block_tables`` names.  ``max_new``: upper bound of a request's new tokens known on the host
    (it chooses the kernel; a request that passes it is still computed).  ``len_bound`` is taken as by ``attn_decode`` and
    has no effect: the work is laid out from the lengths on the device.  Rows of no request are left as they were in
    ``out`` (unspecified in a new tensor).  ``workspace``: from ``attn_paged_workspace``."""
    dev = _require_gpu(q, k_cache, v_cache, block_tables, cu, kv_lens, workspace, out)
    n_pages, n_kv, page_size, hd = _pages("attn_paged", k_cache, v_cache)
    if q.dim() != 3 or q.shape[2] != hd or q.shape[1] % n_kv or q.shape[1] == 0:
        raise ValueError(f"attn_paged: q {tuple(q.shape)} against caches {tuple(k_cache.shape)}")
    if not (q.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError("attn_paged: q and the caches must share a dtype")
    if block_tables.dim() != 2 or block_tables.dtype != torch.int32:
        raise ValueError("attn_paged: block_tables must be int32 [requests, max_pages]")
    R, max_pages = block_tables.shape
    cu = _index("attn_paged", "cu", cu, torch.int64, (R + 1,))
    kv_lens = _index("attn_paged", "kv_lens", kv_lens, torch.int64, (R,))
    q, block_tables = _aligned(q), _contig(block_tables)
    T, n_q = q.shape[:2]
    max_new = T if max_new is None else int(max_new)
    len_bound = max_pages * page_size if len_bound is None else int(len_bound)
    scale = hd ** -0.5 if scale is None else float(scale)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("attn_paged: out must be a contiguous, 16-byte aligned tensor like q")
    if workspace is None:
        workspace = attn_paged_workspace(dev)
    _own("attn_paged", "workspace", workspace)
    with _device(dev):
        _lib.check(_lib.lib().mtp_attn_paged(_p(q), _p(k_cache), _p(v_cache), _p(block_tables), _p(cu), _p(kv_lens), _p(out),
                                             _p(workspace), workspace.numel() * workspace.element_size(), T, R, n_q, n_kv,
                                             hd, n_pages, page_size, max_pages, max_new, len_bound, scale, _dt(q),
                                             _stream(dev)), "mtp_attn_paged")
    return out


def verify_draft(draft_tokens: torch.Tensor, target_probs: torch.Tensor, draft_probs: Optional[torch.Tensor],
                 uniforms: torch.Tensor, draft_lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (tokens int64 [R, K + 1], accepted int64 [R]): the accepted drafts of each request, the token drawn after them,
    then -1.  ``draft_tokens`` int64 [R, K]; ``target_probs`` [R, K + 1, V]; ``draft_probs`` [R, K, V] of the same type,
    or None where the drafts were certain; ``uniforms`` fp32 [R, K + 1] in [0, 1): one per draft, the last for the drawn
    token; ``draft_lens`` int64 [R] limits the drafts of a request."""
    dev = _require_gpu(draft_tokens, target_probs, draft_probs, uniforms, draft_lens)
    if draft_tokens.dim() != 2 or target_probs.dim() != 3:
        raise ValueError("verify_draft: draft_tokens must be [R, K] and target_probs [R, K + 1, V]")
    R, K = draft_tokens.shape
    V = target_probs.shape[2]
    draft_tokens = _index("verify_draft", "draft_tokens", draft_tokens, torch.int64, (R, K))
    uniforms = _index("verify_draft", "uniforms", uniforms, torch.float32, (R, K + 1))
    if target_probs.shape != (R, K + 1, V):
        raise ValueError(f"verify_draft: target_probs {tuple(target_probs.shape)} for {R} requests of {K} drafts")
    if draft_probs is not None and (draft_probs.shape != (R, K, V) or draft_probs.dtype != target_probs.dtype):
        raise ValueError("verify_draft: draft_probs must be [R, K, V] of the type of target_probs")
    if draft_lens is not None:
        draft_lens = _index("verify_draft", "draft_lens", draft_lens, torch.int64, (R,))
    target_probs = _contig(target_probs)
    draft_probs = None if draft_probs is None else _contig(draft_probs)
    tokens = torch.empty((R, K + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty((R,), dtype=torch.int64, device=dev)
    lib = _lib.lib()
    need = int(lib.mtp_verify_draft_workspace_bytes(R, V))
    ws = torch.empty((max(need, 8),), dtype=torch.uint8, device=dev)
    with _device(dev):
        _lib.check(lib.mtp_verify_draft(_p(draft_tokens), _p(draft_lens), _p(target_probs), _p(draft_probs), _p(uniforms),
                                        _p(tokens), _p(accepted), _p(ws), ws.numel(), R, K, V, _dt(target_probs),
                                        _stream(dev)), "mtp_verify_draft")
    return tokens, accepted
