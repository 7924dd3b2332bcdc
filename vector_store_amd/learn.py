"""ctypes binding of libvs_learn.so (include/vs_learn.h): learning the vectors an index serves.

    lookup(rows, ids)                     rows read by number                      lookup_grad: their gradient
    softmax_loss(queries, rows, labels)   cross entropy of every query's scores    softmax_loss_grad: the gradients of
                                          against ALL rows                         the queries and of the rows

`rows` is a table (a 2-D torch tensor on the GPU: f32, f16 or bf16) or a HipUsearchIndex, whose members are numbered by slot
(`HipUsearchIndex.slots(keys)`); an index stores what it stores, so its gradients say how its members would have to move.
Work is enqueued on the current torch stream of the tensors' device and nothing is synchronised: calls can be captured into a
HIP graph.  Scratch is allocated per call from torch's caching allocator.  Wrong arguments raise VsError."""
from __future__ import annotations

import contextlib
import ctypes as C
import os

import torch

from . import index as _ix
from .index import COS, IP, HipUsearchIndex, VsError  # noqa: F401

_HERE = os.path.dirname(os.path.abspath(__file__))
_lib = None
_SCALAR = {torch.float32: _ix.F32, torch.float16: _ix.F16, torch.bfloat16: _ix.BF16}
_DTYPE = {v: k for k, v in _SCALAR.items()}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}


class _Rows(C.Structure):
    _fields_ = [("index", C.c_void_p), ("d_data", C.c_void_p), ("scalar", C.c_int), ("rows", C.c_size_t), ("dim", C.c_size_t), ("stride", C.c_size_t)]


class _Softmax(C.Structure):
    _fields_ = [("d_queries", C.c_void_p), ("scalar", C.c_int), ("n", C.c_size_t), ("stride", C.c_size_t), ("d_labels", C.c_void_p),
                ("label_bytes", C.c_size_t), ("scale", C.c_float), ("metric", C.c_int)]


def lib():
    global _lib
    if _lib is None:
        _ix.lib()
        path = os.path.join(os.environ.get("VS_LIB_DIR") or _HERE, "libvs_learn.so")
        if not os.path.exists(path):
            raise VsError(-6, f"{path} is missing: run `python -c 'import __graft_entry__ as g; g.build()'`")
        L = C.CDLL(path)
        vp, sz, f32, i = C.c_void_p, C.c_size_t, C.c_float, C.c_int
        rows, soft = C.POINTER(_Rows), C.POINTER(_Softmax)
        L.vs_lookup_device.argtypes = [rows, vp, sz, sz, f32, vp, i, sz, vp]
        L.vs_lookup_grad_work.argtypes = [sz, sz, sz]
        L.vs_lookup_grad_work.restype = sz
        L.vs_lookup_grad_device.argtypes = [vp, i, sz, vp, sz, sz, sz, sz, f32, i, vp, i, sz, vp, sz, vp]
        L.vs_softmax_loss_work.argtypes = [rows, soft]
        L.vs_softmax_loss_work.restype = sz
        L.vs_softmax_loss_device.argtypes = [rows, soft, vp, vp, vp, sz, vp]
        L.vs_softmax_loss_grad_work.argtypes = [rows, soft, i, i]
        L.vs_softmax_loss_grad_work.restype = sz
        L.vs_softmax_loss_grad_device.argtypes = [rows, soft, vp, vp, vp, sz, vp, sz, vp, sz, vp]
        L.vs_learn_last_error.restype = C.c_char_p
        _lib = L
    return _lib


def _check(rc: int):
    if rc != 0:
        raise VsError(rc, lib().vs_learn_last_error().decode())


def _need(cond: bool, what: str, code: int = -1):
    if not cond:
        raise VsError(code, what)


def _matrix(t, what: str, dtypes=_SCALAR):
    """A 2-D tensor whose rows are contiguous and do not overlap; anything else is copied."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{what}: a tensor on the GPU is needed")
    _need(t.dim() == 2, f"{what}: two dimensions are needed, got {t.dim()}")
    _need(t.dtype in dtypes, f"{what}: f32, f16 or bf16 is needed, got {t.dtype}", -7)
    t = t.detach()
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ids(t, device, what: str):
    _need(isinstance(t, torch.Tensor) and t.device == device, f"{what}: a tensor on {device} is needed")
    _need(t.dtype in _ID_BYTES, f"{what}: int32 or int64 is needed, got {t.dtype}")
    return t.detach().contiguous()


class _Source:
    """The rows of a call: vs_rows, and what the caller's tensors must agree with."""

    def __init__(self, rows):
        if isinstance(rows, HipUsearchIndex):
            v = rows.rows()
            _need(v["quantization"] in _DTYPE, "rows of an index: f32, f16 or bf16 storage is needed", -7)
            self.count, self.dim, self.dtype = v["slots"], rows.dim, _DTYPE[v["quantization"]]
            self.device = torch.device("cuda", v["device"])
            self.keep = rows
            self.c = _Rows(rows.h, None, 0, 0, 0, 0)
        else:
            t = _matrix(rows, "rows")
            self.count, self.dim, self.dtype, self.device = t.shape[0], t.shape[1], t.dtype, t.device
            self.keep = t
            self.c = _Rows(None, t.data_ptr(), _SCALAR[t.dtype], t.shape[0], t.shape[1], _stride(t))


def _on(device):
    """The tensors' device as the current one (a context only where it is not)."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _work(nbytes: int, device):
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def lookup(rows, ids, scale: float = 1.0, dtype=None):
    """scale * rows[ids], of shape ids.shape + (dim,); a row of zeros where an id is outside [0, rows) (or names a removed member)."""
    s = _Source(rows)
    flat = _ids(ids, s.device, "ids").reshape(-1)
    dtype = dtype or s.dtype
    _need(dtype in _SCALAR, f"dtype: f32, f16 or bf16 is needed, got {dtype}", -7)
    with _on(s.device):
        out = torch.empty((flat.numel(), s.dim), dtype=dtype, device=s.device)
        _check(lib().vs_lookup_device(C.byref(s.c), flat.data_ptr(), _ID_BYTES[flat.dtype], flat.numel(), scale, out.data_ptr(), _SCALAR[dtype], s.dim,
                                      _stream(s.device)))
    return out.view(*ids.shape, s.dim)


def lookup_grad(grad, ids, size: int, scale: float = 1.0, dtype=None, into=None):
    """Gradient of `lookup` with respect to a table of `size` rows: row v is scale * the sum of grad[t] over the t with ids[t] == v, in the
    order of t.  grad: ids.shape + (dim,).  `into`: a (size, dim) tensor the sums are added to instead (rows nobody read are left alone)."""
    _need(isinstance(grad, torch.Tensor) and grad.dim() >= 1 and isinstance(ids, torch.Tensor) and tuple(grad.shape[:-1]) == tuple(ids.shape),
          "grad: ids.shape + (dim,) is needed")
    g = _matrix(grad if grad.dim() == 2 else grad.reshape(ids.numel(), grad.shape[-1]), "grad")
    flat = _ids(ids, g.device, "ids").reshape(-1)
    _need(size >= 0, "size must not be negative")
    dim = g.shape[1]
    with _on(g.device):
        if into is not None:
            _need(isinstance(into, torch.Tensor) and into.device == g.device and into.dtype in _SCALAR and tuple(into.shape) == (size, dim),
                  "into: a (size, dim) tensor beside grad is needed")
            _need((dim <= 1 or into.stride(1) == 1) and (size <= 1 or into.stride(0) >= dim), "into: contiguous rows that do not overlap are needed")
            _need(dtype is None or dtype == into.dtype, "dtype: into has another")
            _need(into.numel() == 0 or into.data_ptr() != g.data_ptr(), "into: memory apart from grad's is needed")
            out = into
        else:
            dtype = dtype or g.dtype
            _need(dtype in _SCALAR, f"dtype: f32, f16 or bf16 is needed, got {dtype}", -7)
            out = torch.empty((size, dim), dtype=dtype, device=g.device)
        n = lib().vs_lookup_grad_work(flat.numel(), size, dim)
        w = _work(n, g.device)
        _check(lib().vs_lookup_grad_device(g.data_ptr(), _SCALAR[g.dtype], _stride(g), flat.data_ptr(), _ID_BYTES[flat.dtype], flat.numel(), size, dim,
                                           scale, int(into is not None), out.data_ptr(), _SCALAR[out.dtype], _stride(out), w.data_ptr(), n, _stream(g.device)))
    return out


def _softmax(queries, s: _Source, labels, scale: float, metric):
    q = _matrix(queries, "queries")
    _need(q.device == s.device, f"queries: a tensor on {s.device} is needed")
    _need(q.shape[1] == s.dim, f"wrong embedding dimension: got {q.shape[1]}, the rows have {s.dim}", -2)
    y = _ids(labels, s.device, "labels")
    _need(tuple(y.shape) == (q.shape[0],), "labels: one per query is needed")
    if metric is None:
        metric = s.keep.metric if isinstance(s.keep, HipUsearchIndex) else IP
    return q, y, _Softmax(q.data_ptr(), _SCALAR[q.dtype], q.shape[0], _stride(q), y.data_ptr(), _ID_BYTES[y.dtype], scale, metric)


def softmax_loss(queries, rows, labels, scale: float = 1.0, metric=None):
    """(loss, lse), f32, one per query: lse = log sum_j exp(scale * <query, row j>) over all rows, loss = lse - scale * <query, row label>.
    metric COS: cosines instead of inner products.  A label outside [0, rows) marks padding: loss 0.  (IP unless `rows` is an index: its own.)"""
    s = _Source(rows)
    q, y, c = _softmax(queries, s, labels, scale, metric)
    with _on(s.device):
        loss = torch.empty(q.shape[0], dtype=torch.float32, device=s.device)
        lse = torch.empty_like(loss)
        n = lib().vs_softmax_loss_work(C.byref(s.c), C.byref(c))
        w = _work(n, s.device)
        _check(lib().vs_softmax_loss_device(C.byref(s.c), C.byref(c), loss.data_ptr(), lse.data_ptr(), w.data_ptr(), n, _stream(s.device)))
    return loss, lse


def softmax_loss_grad(queries, rows, labels, lse, grad_loss, scale: float = 1.0, metric=None, grad_queries: bool = True, grad_rows: bool = True):
    """Gradients of (grad_loss * loss).sum() with respect to the queries and to the rows (None where not asked for), in their types.
    `lse` is softmax_loss's; queries, rows, labels, scale and metric must be what it was computed from."""
    s = _Source(rows)
    q, y, c = _softmax(queries, s, labels, scale, metric)
    for t, what in ((lse, "lse"), (grad_loss, "grad_loss")):
        _need(isinstance(t, torch.Tensor) and t.device == s.device and t.dtype == torch.float32 and tuple(t.shape) == (q.shape[0],),
              f"{what}: one f32 per query is needed")
    lse, grad_loss = lse.detach().contiguous(), grad_loss.detach().contiguous()
    with _on(s.device):
        gq = torch.empty((q.shape[0], s.dim), dtype=q.dtype, device=s.device) if grad_queries else None
        gw = torch.empty((s.count, s.dim), dtype=s.dtype, device=s.device) if grad_rows else None
        n = lib().vs_softmax_loss_grad_work(C.byref(s.c), C.byref(c), int(grad_queries), int(grad_rows))
        w = _work(n, s.device)
        if (gq is not None and gq.numel()) or (gw is not None and gw.numel()):
            _check(lib().vs_softmax_loss_grad_device(C.byref(s.c), C.byref(c), lse.data_ptr(), grad_loss.data_ptr(), gq.data_ptr() if gq is not None else None,
                                                     s.dim, gw.data_ptr() if gw is not None else None, s.dim, w.data_ptr(), n, _stream(s.device)))
    return gq, gw
