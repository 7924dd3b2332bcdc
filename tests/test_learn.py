"""What the learning operators refuse, and what their library exports: no GPU work is started by any of these."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

import vector_store_amd as vs
from vector_store_amd import learn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, DIMENSION, UNSUPPORTED = -1, -2, -7


def test_exports_what_the_header_declares():
    text = open(os.path.join(ROOT, "include", "vs_learn.h")).read()
    want = set(re.findall(r"^VS_API [^;(]*?\b(vs_[a-z0-9_]+)\(", text, flags=re.M))
    out = subprocess.check_output(["nm", "-D", "--defined-only", os.path.join(ROOT, "vector_store_amd", "libvs_learn.so")], text=True)
    have = {ln.split()[-1] for ln in out.splitlines() if " T " in ln}
    assert len(want) == 8 and {x for x in have if x.startswith("vs_")} == want


def rows(data=4096, scalar=vs.F32, n=10, dim=8, stride=8, index=None):
    return learn._Rows(index, data, scalar, n, dim, stride)


def soft(q=4096, scalar=vs.F32, n=4, stride=8, labels=4096, label_bytes=8, scale=1.0, metric=vs.IP):
    return learn._Softmax(q, scalar, n, stride, labels, label_bytes, scale, metric)


BAD_ROWS = [(dict(scalar=vs.I8), UNSUPPORTED), (dict(scalar=vs.B1), UNSUPPORTED), (dict(scalar=9), UNSUPPORTED), (dict(data=None), INVALID), (dict(stride=7), INVALID),
            (dict(dim=0), INVALID), (dict(n=2 ** 31), UNSUPPORTED), (dict(dim=2 ** 17, stride=2 ** 17), UNSUPPORTED), (dict(stride=2 ** 21), UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_ROWS)
def test_bad_rows(kw, code):
    L = learn.lib()
    r, s = rows(**kw), soft(stride=max(8, kw.get("dim", 8)))
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), 4096, 4096, 4096, 1 << 40, None) == code
    assert L.vs_softmax_loss_grad_device(C.byref(r), C.byref(s), 4096, 4096, 4096, 1 << 18, 4096, 1 << 18, 4096, 1 << 40, None) == code
    assert L.vs_lookup_device(C.byref(r), 4096, 8, 3, 1.0, 4096, vs.F32, 1 << 18, None) == code
    assert L.vs_learn_last_error()
    assert L.vs_softmax_loss_work(C.byref(r), C.byref(s)) == 0


BAD_QUERIES = [(dict(scalar=vs.I8), UNSUPPORTED), (dict(q=None), INVALID), (dict(labels=None), INVALID), (dict(stride=7), INVALID), (dict(label_bytes=2), INVALID),
               (dict(metric=vs.L2SQ), INVALID), (dict(metric=vs.HAMMING), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
               (dict(n=2 ** 20 + 1), UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_QUERIES)
def test_bad_queries(kw, code):
    L = learn.lib()
    r, s = rows(), soft(**kw)
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), 4096, 4096, 4096, 1 << 40, None) == code
    assert L.vs_softmax_loss_grad_device(C.byref(r), C.byref(s), 4096, 4096, 4096, 8, 4096, 8, 4096, 1 << 40, None) == code


def test_bad_outputs_and_scratch():
    L = learn.lib()
    r, s = rows(), soft()
    work = L.vs_softmax_loss_work(C.byref(r), C.byref(s))
    assert work > 0
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), None, 4096, 4096, work, None) == INVALID
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), 4096, None, 4096, work, None) == INVALID
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), 4096, 4096, 4096, work - 1, None) == INVALID
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), 4096, 4096, None, work, None) == INVALID
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(s), 4096, 4096, 4096 + 128, work, None) == INVALID
    assert L.vs_softmax_loss_device(None, C.byref(s), 4096, 4096, 4096, work, None) == INVALID
    assert L.vs_softmax_loss_device(C.byref(r), None, 4096, 4096, 4096, work, None) == INVALID
    gwork = L.vs_softmax_loss_grad_work(C.byref(r), C.byref(s), 1, 1)
    for lse, g, gq, qs, gw, ws, wk, nb in ((None, 4096, 4096, 8, 4096, 8, 4096, gwork), (4096, None, 4096, 8, 4096, 8, 4096, gwork), (4096, 4096, 4096, 7, 4096, 8, 4096, gwork),
                                           (4096, 4096, 4096, 8, 4096, 7, 4096, gwork), (4096, 4096, 4096, 8, 4096, 8, 4096, gwork - 1), (4096, 4096, 4096, 8, 4096, 8, None, gwork)):
        assert L.vs_softmax_loss_grad_device(C.byref(r), C.byref(s), lse, g, gq, qs, gw, ws, wk, nb, None) == INVALID
    assert L.vs_softmax_loss_grad_device(C.byref(r), C.byref(s), 4096, 4096, None, 0, None, 0, None, 0, None) == 0  # nothing asked for
    empty = soft(n=0, q=None, labels=None)
    assert L.vs_softmax_loss_device(C.byref(r), C.byref(empty), None, None, None, 0, None) == 0


def test_bad_lookups():
    L = learn.lib()
    r = rows()
    for ids, b, out, sc, st, code in ((None, 8, 4096, vs.F32, 8, INVALID), (4096, 3, 4096, vs.F32, 8, INVALID), (4096, 8, None, vs.F32, 8, INVALID), (4096, 8, 4096, vs.I8, 8, UNSUPPORTED),
                                      (4096, 8, 4096, vs.F32, 7, INVALID)):
        assert L.vs_lookup_device(C.byref(r), ids, b, 5, 1.0, out, sc, st, None) == code
    assert L.vs_lookup_device(C.byref(r), None, 8, 0, 1.0, None, vs.F32, 8, None) == 0
    w = L.vs_lookup_grad_work(5, 10, 8)

    def grad(g=4096, gs=vs.F32, gst=8, ids=4096, b=8, n=5, v=10, d=8, out=4096, os_=vs.F32, ost=8, wk=4096, nb=w):
        return L.vs_lookup_grad_device(g, gs, gst, ids, b, n, v, d, 1.0, 0, out, os_, ost, wk, nb, None)

    for kw in (dict(g=None), dict(gst=7), dict(ids=None), dict(b=1), dict(d=0), dict(out=None), dict(ost=7), dict(wk=None), dict(nb=w - 1), dict(wk=4097)):
        assert grad(**kw) == INVALID, kw
    for kw in (dict(gs=vs.B1), dict(os_=7), dict(n=2 ** 30), dict(v=2 ** 31), dict(d=2 ** 17, gst=2 ** 17, ost=2 ** 17)):
        assert grad(**kw) == UNSUPPORTED, kw
    assert grad(v=0, out=None) == 0


def test_tensors_that_are_not_on_the_gpu_are_refused():
    t, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: learn.lookup(t, i), lambda: learn.lookup_grad(t, i, 10), lambda: learn.softmax_loss(t, t, i), lambda: learn.lookup(None, i),
                 lambda: learn.softmax_loss_grad(t, t, i, torch.zeros(4), torch.zeros(4)), lambda: learn.lookup_grad(t, i[:3], 10)):
        with pytest.raises(vs.VsError):
            call()
