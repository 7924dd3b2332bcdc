"""The learning operators (include/vs_learn.h, vector_store_amd.learn) against plain float64 statements of their formulas.

Tolerances are worst-case bounds counted in roundings, half a step each: U = 2^-24 (f32), 2^-8 (bf16), 2^-11 (f16); a number split into two f16
keeps 2^-22 of itself.  A score z = s <q, w> of D terms summed in f32 is off by at most
    s |q| |w| (3 * 2^-22 + 3 (D + 64) * 2^-24)         (two splits and the dropped lo * lo; three products of D terms)
and what is built from it by the sums written out in the helpers below."""
import numpy as np
import pytest
import torch

import vector_store_amd as vs
from vector_store_amd import learn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -126, F16: 2.0 ** -25, BF16: 2.0 ** -126}  # half of the smallest step (f32 / bf16: below the smallest normal)


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def case(n, v, d, tq, tw, seed=0, pad=True):
    g = gen(seed)
    w = (torch.randn(v, d, generator=g, device=DEV) * (torch.rand(v, 1, generator=g, device=DEV) + 0.5) / d ** 0.5).to(tw)
    y = torch.randint(v, (n,), generator=g, device=DEV)
    q = (0.7 * w[y].float() + 0.7 * torch.randn(n, d, generator=g, device=DEV) / d ** 0.5).to(tq)
    if pad and n > 2:
        y[torch.randperm(n, generator=g, device=DEV)[: max(1, n // 20)]] = -1
    gl = torch.rand(n, generator=g, device=DEV) + 0.1
    return q, w, y, gl


def unit(x):
    n = x.norm(dim=1, keepdim=True)
    return torch.where(n > 0, x / n.clamp(min=1e-300), torch.zeros_like(x)), n


def reference(q, w, y, gl, scale, cos, dead=None):
    """loss, lse, dq, dw in float64, and the error bounds of each."""
    d = q.shape[1]
    q, w, gl = q.double(), w.double(), gl.double()
    (qu, nq), (wu, nw) = (unit(q), unit(w)) if cos else ((q, 1.0), (w, 1.0))
    z = scale * qu @ wu.t()
    ez = abs(scale) * (3 * 2.0 ** -22 + 3 * (d + 64) * 2.0 ** -24 + (4 * 2.0 ** -24 if cos else 0)) * qu.norm(dim=1, keepdim=True) * wu.norm(dim=1)[None, :]
    if dead is not None:
        z[:, dead] = -float("inf")
    on = (y >= 0) & (y < w.shape[0])
    if dead is not None:
        on &= ~dead[y.clamp(0, w.shape[0] - 1)]
    at = y.clamp(0, max(w.shape[0] - 1, 0))
    lse = torch.logsumexp(z, dim=1)
    zy = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(on, lse - zy, torch.zeros_like(lse))
    top = ez.max(dim=1).values
    zmax = z.masked_fill(torch.isinf(z), 0).abs().max(dim=1).values
    # the sum of v terms in f32 (blocks of 16 in a lane, then joins): well below 64 roundings of a positive sum; exp2 and log2: a few steps
    e_lse = top + 2.0 ** -24 * (80 + 4 * (zmax + lse.masked_fill(torch.isinf(lse), 0).abs()))
    e_loss = 2 * top + 2.0 ** -24 * (80 + 8 * (zmax + lse.masked_fill(torch.isinf(lse), 0).abs()))
    p = torch.softmax(z, dim=1)
    c = p.clone()
    r = torch.arange(len(y), device=y.device)[on]
    c[r, y[r]] -= 1
    c = torch.where(on[:, None], c * gl[:, None], torch.zeros_like(c))
    m = p
    m[r, y[r]] += 1
    m = torch.where(on[:, None], m * gl.abs()[:, None], torch.zeros_like(m))  # what |c| is bounded by, before cancellation
    ep = 2 * (top + e_lse)[:, None].clamp(max=1)  # relative error of a probability
    fq, fw = (1 / nq, 1 / nw) if cos else (1.0, 1.0)
    dq, dw = scale * (c @ wu), scale * (c.t() @ qu)
    bq, bw = abs(scale) * (m @ wu.abs()), abs(scale) * (m.t() @ qu.abs())                   # sums of magnitudes
    every = torch.where(on, gl.abs(), torch.zeros_like(gl))
    floor = (abs(scale) * every[:, None] * wu.abs().sum(0) * fq, abs(scale) * (every @ qu.abs())[None, :] * (fw if cos else 1.0))  # ... if every p were 1
    floor = tuple(torch.nan_to_num(x, 0.0, 0.0, 0.0) * (2 if cos else 1) for x in floor)
    eq, ew = abs(scale) * ((m * ep) @ wu.abs()), abs(scale) * ((m * ep).t() @ qu.abs())     # ... times the probabilities' errors
    if cos:
        dq, dw = (dq - qu * (qu * dq).sum(1, keepdim=True)) * fq, (dw - wu * (wu * dw).sum(1, keepdim=True)) * fw
        (dq, dw) = (torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (dq, dw))
        along = lambda u, b, f: torch.nan_to_num((b + u.abs() * (u.abs() * b).sum(1, keepdim=True)) * f, 0.0, 0.0, 0.0)  # noqa: E731
        bq, eq, bw, ew = along(qu, bq, fq), along(qu, eq, fq), along(wu, bw, fw), along(wu, ew, fw)
    return loss, lse, dq, dw, e_loss, e_lse, (bq, eq, floor[0]), (bw, ew, floor[1])


def grad_bound(b, e, want, dtype, terms, floor):
    """one rounding of the probability and one of each operand (two f16 where the result is f32), the f32 sum, the result's own rounding.
    A probability is held as p * m * 2^15 (1/2 <= m < 1) in f16, whose steps do not get smaller than 2^-24: half a step is 2^-25 * 2^-15 / m <=
    2^-39 of the loss's gradient, whatever p is, and `floor` is what p = 1 everywhere would add up to."""
    u = 4 * 2.0 ** -22 if dtype == F32 else 3 * U[dtype]
    return b * (u + min(terms, 4096) * 2.0 ** -24) + e + want.abs() * U[dtype] + 4 * TINY[dtype] + floor * 2.0 ** -39


def close(got, want, bound, what):
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() or not torch.isfinite(want).all(), what
    bad = ~(err <= bound)
    bad &= ~((got.double() == want))  # (equal infinities)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((err / bound)[bad].max()):.3g} x"


def check(q, w, y, gl, scale, metric, rows=None, dead=None):
    cos = metric == learn.COS
    loss, lse, dq, dw, e_loss, e_lse, bq, bw = reference(q, w, y, gl, scale, cos, dead)
    src = w if rows is None else rows
    m = None if rows is not None else metric
    l1, s1 = learn.softmax_loss(q, src, y, scale, m)
    close(s1, lse, e_lse, "lse")
    close(l1, loss, e_loss, "loss")
    g1, g2 = learn.softmax_loss_grad(q, src, y, s1, gl, scale, m)
    close(g1, dq, grad_bound(bq[0], bq[1], dq, q.dtype, w.shape[0], bq[2]), "dq")
    close(g2, dw, grad_bound(bw[0], bw[1], dw, w.dtype, q.shape[0], bw[2]), "dw")
    a, none = learn.softmax_loss_grad(q, src, y, s1, gl, scale, m, grad_rows=False)
    assert none is None
    none, b = learn.softmax_loss_grad(q, src, y, s1, gl, scale, m, grad_queries=False)
    assert none is None
    if q.dtype == w.dtype:  # the same kernels on the same numbers: the same bits
        assert torch.equal(a, g1) and torch.equal(b, g2)
    else:
        close(a, dq, grad_bound(bq[0], bq[1], dq, q.dtype, w.shape[0], bq[2]), "dq alone")
        close(b, dw, grad_bound(bw[0], bw[1], dw, w.dtype, q.shape[0], bw[2]), "dw alone")
    return l1, s1, g1, g2


SIZES = [(1, 1, 1), (1, 300, 64), (3, 2, 5), (5, 255, 7), (63, 257, 96), (65, 1000, 100), (129, 4099, 64), (300, 3001, 384), (257, 20011, 72), (20, 70003, 128)]
PAIRS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F16)]


@pytest.mark.parametrize("metric", [learn.IP, learn.COS], ids=["ip", "cos"])
@pytest.mark.parametrize("tq,tw", PAIRS, ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("n,v,d", SIZES)
def test_loss_and_gradients(n, v, d, tq, tw, metric):
    q, w, y, gl = case(n, v, d, tq, tw, seed=n + v + d)
    check(q, w, y, gl, 8.0, metric)


@pytest.mark.parametrize("tq,tw", [(BF16, BF16), (F32, F32)], ids=["bf16", "f32"])
def test_large_tiles_and_pieces(tq, tw):
    """enough of everything for the large tiles, several pieces of the table and slices of k, no multiple of any"""
    q, w, y, gl = case(1030, 70_001 if tw == F32 else 140_001, 200, tq, tw, seed=3)
    check(q, w, y, gl, 8.0, learn.IP)


@pytest.mark.parametrize("metric", [learn.IP, learn.COS], ids=["ip", "cos"])
@pytest.mark.parametrize("v,d", [(515, 1), (4099, 4), (3001, 33), (70_003, 100), (20_011, 128), (1000, 516)])
@pytest.mark.parametrize("n", [1, 2, 31, 64, 65, 128, 129])
def test_few_f32_queries(n, v, d, metric):
    """around the numbers of queries up to which f32 is multiplied as f32: rows in place and re-laid, depths that are no multiple of a step"""
    q, w, y, gl = case(n, v, d, F32, F32, seed=40 + n + d)
    check(q, w, y, gl, 8.0, metric)


@pytest.mark.parametrize("metric", [learn.IP, learn.COS], ids=["ip", "cos"])
@pytest.mark.parametrize("v,d", [(515, 1), (4099, 8), (3001, 33), (20_011, 128), (1000, 520)])
@pytest.mark.parametrize("n", [1, 64, 65, 256, 257])
def test_few_bf16_queries(n, v, d, metric):
    """around the number of queries up to which the probabilities of bf16 queries and rows are two bf16"""
    q, w, y, gl = case(n, v, d, BF16, BF16, seed=50 + n + d)
    check(q, w, y, gl, 8.0, metric)


def test_few_bf16_queries_of_wide_ranges():
    q, w, y, gl = case(50, 700, 96, BF16, BF16, seed=51)
    gl = gl * torch.logspace(-12, 12, 50, device=DEV)
    few = (q.float() * torch.logspace(-8, 0, 50, device=DEV)[:, None]).to(BF16)
    check(few, (w.float() * torch.logspace(-6, 0, 700, device=DEV)[:, None]).to(BF16), y, gl, 8.0, learn.IP)
    check(few, (w.float() * torch.logspace(-9, 9, 700, device=DEV)[:, None]).to(BF16), y, gl, 8.0, learn.COS)


def test_few_f32_queries_of_wide_ranges_and_padding():
    q, w, y, gl = case(50, 700, 96, F32, F32, seed=41)
    gl = gl * torch.logspace(-12, 12, 50, device=DEV)
    q2 = q * torch.logspace(-15, 15, 50, device=DEV)[:, None]
    check(q * torch.logspace(-8, 0, 50, device=DEV)[:, None], w * torch.logspace(-6, 0, 700, device=DEV)[:, None], y, gl, 8.0, learn.IP)
    check(q2, w * torch.logspace(-15, 15, 700, device=DEV)[:, None], y, gl, 8.0, learn.COS)
    for metric in (learn.IP, learn.COS):
        q, w, y, gl = case(50, 515, 100, F32, F32, seed=42, pad=False)
        y[::7] = -1
        y[3] = 515
        off = (y < 0) | (y >= 515)
        l0, s0 = learn.softmax_loss(q, w, y, 8.0, metric)
        a0, b0 = learn.softmax_loss_grad(q, w, y, s0, gl, 8.0, metric)
        for junk in (float("nan"), float("inf"), torch.finfo(F32).max, 0.0):
            dirty, gl2 = q.clone(), gl.clone()
            dirty[off], gl2[off] = junk, float("nan")
            l1, s1 = learn.softmax_loss(dirty, w, y, 8.0, metric)
            a1, b1 = learn.softmax_loss_grad(dirty, w, y, s1, gl2, 8.0, metric)
            assert (l1[off] == 0).all() and (a1[off] == 0).all(), metric
            assert torch.equal(l1, l0) and torch.equal(s1[~off], s0[~off]) and torch.equal(a1, a0) and torch.equal(b1, b0), metric


@pytest.mark.parametrize("t", [F32, BF16], ids=["f32", "bf16"])
def test_few_queries_over_several_pieces(t):
    """more rows than one piece holds (2^20), re-laid and in place"""
    for d, metric in ((5, learn.IP), (8, learn.COS)):
        q, w, y, gl = case(3, 1_100_003, d, t, t, seed=44, pad=False)
        y[1] = 1_100_002
        check(q, w, y, gl, 8.0, metric)


@pytest.mark.parametrize("metric", [vs.IP, vs.COS], ids=["ip", "cos"])
def test_few_f32_queries_of_an_index(metric):
    ix, keys, base = build(F32, metric, 1500, 100, 1)
    slots = torch.from_numpy(ix.slots(keys)).to(DEV)
    stored = learn.lookup(ix, torch.arange(1500, device=DEV))
    g = gen(43)
    y = torch.randint(1500, (33,), generator=g, device=DEV)
    q = stored[y] + 0.05 * torch.randn(33, 100, generator=g, device=DEV)
    gl = torch.rand(33, generator=g, device=DEV)
    check(q, stored, y, gl, 8.0, metric, rows=ix)
    for k in keys[::5]:
        assert ix.remove(int(k))
    dead = torch.zeros(1500, dtype=torch.bool, device=DEV)
    dead[slots[::5]] = True
    _, _, _, dw = check(q, stored, y, gl, 8.0, metric, rows=ix, dead=dead)
    assert (dw[dead] == 0).all()


def test_widest_rows_and_one_query_over_many():
    q, w, y, gl = case(2, 513, 4096, F32, F32, seed=4, pad=False)
    check(q, w, y, gl, 4.0, learn.COS)
    q, w, y, gl = case(1, 300_000, 33, BF16, BF16, seed=5)
    check(q, w, y, gl, 8.0, learn.IP)


def test_offsets_beyond_32_bits():
    """a table of more than 4 GiB: scores, labels, lookups and gradients at its far end"""
    v, d = 3_000_000, 768
    g = gen(6)
    w = torch.empty((v, d), dtype=BF16, device=DEV)
    for a in range(0, v, 500_000):
        w[a:a + 500_000] = torch.randn(500_000, d, generator=g, device=DEV) / d ** 0.5
    y = torch.tensor([v - 1, 5, 2_999_000], device=DEV)
    q = w[y].clone()
    loss, lse = learn.softmax_loss(q, w, y, 12.0)
    z = torch.cat([12.0 * q.double() @ w[a:a + 250_000].double().t() for a in range(0, v, 250_000)], dim=1)
    want = torch.logsumexp(z, dim=1)
    bound = 12 * float(q.double().norm(dim=1).max() * 1.2) * (3 * 2.0 ** -22 + 3 * (d + 64) * 2.0 ** -24) + 2.0 ** -24 * (80 + 8 * 40)
    assert (lse.double() - want).abs().max() <= bound
    assert (loss.double() - (want - z.gather(1, y[:, None])[:, 0])).abs().max() <= 2 * bound
    gl = torch.ones(3, device=DEV)
    gq, gw = learn.softmax_loss_grad(q, w, y, lse, gl, 12.0)
    p = torch.softmax(z, dim=1)
    p[torch.arange(3), y] -= 1
    for j in (0, 5, 1_500_001, 2_999_000, v - 2, v - 1):
        exact = 12.0 * p[:, j] @ q.double()
        m = 12.0 * p[:, j].abs() @ q.double().abs()
        assert ((gw[j].double() - exact).abs() <= m * (3 * U[BF16] + 8 * bound) + exact.abs() * U[BF16] + 1e-30).all(), j
    del gw, p, z
    assert torch.equal(learn.lookup(w, y), w[y])
    grad = torch.randn(3, d, generator=g, device=DEV).to(BF16)
    back = learn.lookup_grad(grad, y, v)
    assert torch.equal(back[y], grad) and int((back != 0).any(dim=1).sum()) == 3


def test_padding_reaches_nobody():
    """queries without a label hold NaN, infinities and the type's extremes: their loss is 0, their gradients 0, and no other value changes"""
    for t in (F32, F16, BF16):
        for metric in (learn.IP, learn.COS):
            q, w, y, gl = case(70, 515, 100, t, t, seed=7, pad=False)
            y[::7] = -1
            y[3] = 515
            y[4] = -(2 ** 40)
            off = (y < 0) | (y >= 515)
            l0, s0 = learn.softmax_loss(q, w, y, 8.0, metric)
            a0, b0 = learn.softmax_loss_grad(q, w, y, s0, gl, 8.0, metric)
            dirty = q.clone()
            junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(t).max, torch.finfo(t).min, 0.0], device=DEV).to(t)
            dirty[off] = junk[torch.arange(int(off.sum()), device=DEV) % 6][:, None].expand(-1, 100)
            gl2 = torch.where(off, torch.full_like(gl, float("nan")), gl)
            l1, s1 = learn.softmax_loss(dirty, w, y, 8.0, metric)
            a1, b1 = learn.softmax_loss_grad(dirty, w, y, s1, gl2, 8.0, metric)
            assert (l1[off] == 0).all() and (a1[off] == 0).all(), (t, metric)
            assert torch.equal(l1, l0) and torch.equal(s1[~off], s0[~off]) and torch.equal(a1, a0) and torch.equal(b1, b0), (t, metric)


def test_nothing_to_learn_from():
    q = torch.randn(5, 64, device=DEV)
    y = torch.zeros(5, dtype=torch.int64, device=DEV)
    empty = torch.empty((0, 64), device=DEV)
    loss, lse = learn.softmax_loss(q, empty, y)
    assert (loss == 0).all() and (lse == -float("inf")).all()
    gq, gw = learn.softmax_loss_grad(q, empty, y, lse, torch.ones(5, device=DEV))
    assert (gq == 0).all() and gw.shape == (0, 64)
    w = torch.randn(9, 64, device=DEV)
    loss, lse = learn.softmax_loss(q[:0], w, y[:0])
    assert loss.shape == (0,) and lse.shape == (0,)
    gq, gw = learn.softmax_loss_grad(q[:0], w, y[:0], lse, loss)
    assert gq.shape == (0, 64) and (gw == 0).all() and gw.shape == (9, 64)
    # every label ignored
    loss, lse = learn.softmax_loss(q, w, y - 1)
    gq, gw = learn.softmax_loss_grad(q, w, y - 1, lse, torch.ones(5, device=DEV))
    assert (loss == 0).all() and (gq == 0).all() and (gw == 0).all()
    # zero vectors under the cosine have no direction: their scores and gradients are 0
    w[3] = 0
    q[1] = 0
    loss, lse = learn.softmax_loss(q, w, y, 3.0, learn.COS)
    assert abs(float(lse[1]) - np.log(9)) < 1e-6
    gq, gw = learn.softmax_loss_grad(q, w, y, lse, torch.ones(5, device=DEV), 3.0, learn.COS)
    assert (gq[1] == 0).all() and (gw[3] == 0).all() and torch.isfinite(gw).all()


def test_wide_ranges():
    """rows and loss gradients of very different magnitude keep their own relative accuracy; large scores do not overflow"""
    q, w, y, gl = case(90, 700, 96, F32, F32, seed=8)
    gl = gl * torch.logspace(-12, 12, 90, device=DEV)
    w2 = w * torch.logspace(-6, 0, 700, device=DEV)[:, None]
    q2 = q * torch.logspace(-8, 0, 90, device=DEV)[:, None]
    check(q2, w2, y, gl, 8.0, learn.IP)
    check(q2, w * torch.logspace(-15, 15, 700, device=DEV)[:, None], y, gl, 8.0, learn.COS)
    # (f16 inner product: a query's loss gradient may be far below the largest; its own row of dq keeps its accuracy)
    h, v16, y, g16 = case(40, 300, 64, F16, F16, seed=9)
    check(h, v16, y, g16 * torch.logspace(-4, 0, 40, device=DEV), 8.0, learn.IP)
    loss, lse = learn.softmax_loss(q, w, y[:1].expand(90).contiguous(), 1e6)
    want = torch.logsumexp(1e6 * q.double() @ w.double().t(), dim=1)
    assert ((lse.double() - want).abs() <= 1e6 * 2 * (3 * 2.0 ** -22 + 480 * 2.0 ** -24) * (q.double().norm(dim=1) * 1.6) + 1).all()


@pytest.mark.parametrize("scale", [0.0, -6.0, 1e-30, 40.0])
def test_scales(scale):
    """scores turned around, flattened to nothing, and stretched until one member holds nearly all"""
    for t in (BF16, F32, F16):
        for metric in (learn.IP, learn.COS):
            q, w, y, gl = case(150, 1300, 72, t, t, seed=30)
            check(q, w, y, gl, scale, metric)


def test_only_the_label_or_one_row():
    """a table of one row: the loss is 0 and nothing moves; every query labelled with the same row"""
    q, w, y, gl = case(100, 1, 64, F32, F32, seed=31, pad=False)
    loss, lse = learn.softmax_loss(q, w, y, 3.0)
    gq, gw = learn.softmax_loss_grad(q, w, y, lse, gl, 3.0)
    assert (loss == 0).all()
    # p - 1 is off by the rounding of lse: half a step of at most 16, times log2(e), twice
    assert gq.abs().max() <= 3 * 1.1 * 4 * 2.0 ** -21 * 2 and gw.abs().max() <= 3 * 110 * 4 * 2.0 ** -21 * 2
    q, w, y, gl = case(200, 900, 96, BF16, BF16, seed=32)
    y[:] = 17
    check(q, w, y, gl, 8.0, learn.IP)


def test_strides_alignment_and_id_types():
    """views with a row stride, rows that start off a 16-byte line, 32-bit labels: the values of contiguous copies, bit for bit"""
    for t in (BF16, F32, F16):
        g = gen(10)
        big = torch.randn(400, 150, generator=g, device=DEV).to(t)
        w, wv = big[:, :96].contiguous(), big[:, :96]
        odd = big[:, 1:97]
        qb = torch.randn(70, 200, generator=g, device=DEV).to(t)
        y = torch.randint(400, (70,), generator=g, device=DEV)
        gl = torch.rand(70, generator=g, device=DEV)
        for a, b, aq, bq in ((w, wv, qb[:, :96].contiguous(), qb[:, :96]), (odd.contiguous(), odd, qb[:, 3:99].contiguous(), qb[:, 3:99]),
                             (big[::2, :96].contiguous(), big[::2, :96], qb[:, 8:104].contiguous(), qb[:, 8:104])):
            yy = y % a.shape[0]
            l0, s0 = learn.softmax_loss(aq, a, yy, 2.0)
            l1, s1 = learn.softmax_loss(bq, b, yy.int(), 2.0)
            assert torch.equal(l0, l1) and torch.equal(s0, s1)
            for x, z in zip(learn.softmax_loss_grad(aq, a, yy, s0, gl, 2.0), learn.softmax_loss_grad(bq, b, yy.int(), s1, gl, 2.0)):
                assert torch.equal(x, z)
            assert torch.equal(learn.lookup(a, yy, 3.0), learn.lookup(b, yy.int(), 3.0))
            assert torch.equal(learn.lookup_grad(aq, yy, 400), learn.lookup_grad(bq, yy.int(), 400))
        # a transposed table and a broadcast query are copied first
        tr = big[:96].t()
        l0, _ = learn.softmax_loss(qb[:, :96].contiguous(), tr.contiguous(), y % 150, 2.0)
        l1, _ = learn.softmax_loss(qb[:, :96], tr, y % 150, 2.0)
        assert torch.equal(l0, l1)
        one = qb[:1, :96].expand(70, 96)
        assert torch.equal(learn.softmax_loss(one, w, y)[0], learn.softmax_loss(one.contiguous(), w, y)[0])


def test_same_bits_again():
    for t in (BF16, F32, F16):
        q, w, y, gl = case(300, 9001, 200, t, t, seed=11)
        first = None
        for _ in range(3):
            l, s = learn.softmax_loss(q, w, y, 8.0)
            out = (l, s) + learn.softmax_loss_grad(q, w, y, s, gl, 8.0) + (learn.lookup_grad(q, y % 17, 9001),)
            first = first or out
            assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_against_differences():
    """the gradients predict how the loss itself changes: central differences along random directions, f32.
    The difference quotient is off by (error of two losses) / 2h and by h^2 / 6 times the third derivative of the loss along the direction,
    at most (2 scale |dir| r)^3 with r the largest vector."""
    q, w, y, gl = case(40, 500, 64, F32, F32, seed=12)
    scale, h = 4.0, 2.0 ** -6
    for metric in (learn.IP, learn.COS):
        _, s = learn.softmax_loss(q, w, y, scale, metric)
        gq, gw = learn.softmax_loss_grad(q, w, y, s, gl, scale, metric)
        g = gen(13)
        for _ in range(4):
            dq = torch.randn(q.shape, generator=g, device=DEV)
            dq /= dq.norm(dim=1, keepdim=True)
            dw = torch.randn(w.shape, generator=g, device=DEV)
            dw /= dw.norm(dim=1, keepdim=True)
            tot = lambda a, b: (learn.softmax_loss(a, b, y, scale, metric)[0].double() * gl.double()).sum()  # noqa: E731
            for grad, lo, hi, dirn in ((gq, (q - h * dq, w), (q + h * dq, w), dq), (gw, (q, w - h * dw), (q, w + h * dw), dw)):
                got = float((tot(*hi) - tot(*lo)) / (2 * h))
                want = float((grad.double() * dirn.double()).sum())
                r = 2.0 if metric == learn.IP else 4.0  # (cosine: the normalisation's own derivatives, vectors of length >= 1/2)
                noise = float(gl.sum()) * 1e-5 / (2 * h)
                assert abs(got - want) <= noise + h * h / 6 * float(gl.sum()) * (2 * scale * r) ** 3 / 40 + 1e-3 * abs(want), (metric, got, want)


# ---------------------------------------------------------------------------------------------------- lookups
@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (7, 3, 5), (16, 1000, 128), (1000, 77, 100), (4097, 5000, 768), (70_001, 300, 33)])
def test_lookup_and_gradient(n, v, d, t):
    g = gen(n + v)
    w = torch.randn(v, d, generator=g, device=DEV).to(t)
    ids = (torch.rand(n, generator=g, device=DEV, dtype=torch.float64) ** 4 * (v + 1)).long() - 1  # -1 among them; the first rows often
    ids[-1] = v + 5
    ok = (ids >= 0) & (ids < v)
    for scale in (1.0, 0.3):
        for out in (t, F32):
            got = learn.lookup(w, ids, scale, out)
            want = torch.where(ok[:, None], w[ids.clamp(0, v - 1)].double() * scale, torch.zeros((), dtype=torch.float64, device=DEV))
            close(got, want, want.abs() * (U[out] + 2 * U[F32]) + TINY[out], "lookup")
        grad = torch.randn(n, d, generator=g, device=DEV).to(t)
        want = torch.zeros(v, d, dtype=torch.float64, device=DEV).index_put_((ids[ok],), grad[ok].double() * scale, accumulate=True)
        mag = torch.zeros(v, d, dtype=torch.float64, device=DEV).index_put_((ids[ok],), grad[ok].double().abs() * abs(scale), accumulate=True)
        cnt = torch.bincount(ids[ok], minlength=v)[:, None].double()
        bound = mag * (cnt + 4) * U[F32]
        for out in (t, F32):
            got = learn.lookup_grad(grad, ids, v, scale, out)
            close(got, want, bound + want.abs() * U[out] + TINY[out], "lookup gradient")
        into = torch.randn(v, d, generator=g, device=DEV).to(t)
        before = into.clone()
        back = learn.lookup_grad(grad, ids, v, scale, into=into)
        assert back is into
        assert torch.equal(into[cnt[:, 0] == 0], before[cnt[:, 0] == 0])
        close(into, want + before.double(), bound + (want.abs() + before.double().abs()) * (U[t] + 2 * U[F32]) + TINY[t], "added gradient")


@pytest.mark.parametrize("n,v,d", [(1_300_000, 5000, 8), (5000, 3_000_000, 16), (4096, 10, 24), (4097, 2, 1), (200_000, 100_000, 520)])
def test_many_ids_and_many_rows(n, v, d):
    """long lists (several waves' worth of counts, long runs of one id), row numbers of more than two digits of the sort"""
    g = gen(n)
    ids = torch.where(torch.rand(n, generator=g, device=DEV) < 0.3, torch.zeros((), dtype=torch.int64, device=DEV), torch.randint(v, (n,), generator=g, device=DEV))
    ids[::1001] = -1
    grad = torch.randint(-3, 4, (n, d), generator=g, device=DEV).float()  # whole numbers: every sum below 2^24 is exact in any order
    got = learn.lookup_grad(grad, ids, v)
    ok = ids >= 0
    want = torch.zeros(v, d, dtype=torch.float64, device=DEV).index_put_((ids[ok],), grad[ok].double(), accumulate=True)
    assert want.abs().max() < 2 ** 24 and torch.equal(got.double(), want)


def test_lookup_shapes_and_untouched_neighbours():
    w = torch.randn(50, 12, device=DEV)
    ids = torch.randint(50, (3, 4, 5), device=DEV)
    assert learn.lookup(w, ids).shape == (3, 4, 5, 12) and torch.equal(learn.lookup(w, ids), w[ids])
    assert learn.lookup(w, ids[:0]).shape == (0, 4, 5, 12)
    grad = torch.randn(3, 4, 5, 12, device=DEV)
    want = torch.zeros(50, 12, device=DEV, dtype=torch.float64).index_put_((ids.reshape(-1),), grad.reshape(-1, 12).double(), accumulate=True)
    got = learn.lookup_grad(grad, ids, 50)
    assert (got.double() - want).abs().max() <= 60 * 5 * 2.0 ** -24
    assert (learn.lookup_grad(grad[:0], ids[:0], 50) == 0).all()
    assert learn.lookup_grad(grad, ids, 0).shape == (0, 12)
    # a strided target: the columns between its rows stay as they are
    frame = torch.full((50, 20), 7.0, device=DEV)
    learn.lookup_grad(grad, ids, 50, into=frame[:, 4:16])
    assert (frame[:, :4] == 7).all() and (frame[:, 16:] == 7).all()
    assert ((frame[:, 4:16] - 7).double() - want).abs().max() <= 60 * 12 * 2.0 ** -23
    # one row read by everybody
    many = torch.zeros(100_000, dtype=torch.int32, device=DEV)
    ones = torch.ones(100_000, 12, device=DEV)
    assert (learn.lookup_grad(ones, many, 3)[0] == 100_000).all()


def test_a_gradient_is_not_added_onto_itself():
    x = torch.ones(7, 4, device=DEV)
    with pytest.raises(vs.VsError):
        learn.lookup_grad(x, torch.arange(7, device=DEV), 7, into=x)
    assert (x == 1).all()


# ---------------------------------------------------------------------------------------------------- members of an index
def build(t, metric, n, d, seed):
    g = np.random.default_rng(seed)
    ix = vs.HipUsearchIndex(d, metric, quantization={F32: vs.F32, F16: vs.F16, BF16: vs.BF16}[t])
    ix.reserve(n + 10)
    base = (g.standard_normal((n, d)) / np.sqrt(d)).astype(np.float32)
    keys = np.arange(n, dtype=np.uint64) * 3 + 100
    ix.add_batch(keys, base)
    return ix, keys, base


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("metric", [vs.IP, vs.COS], ids=["ip", "cos"])
def test_members_of_an_index(t, metric):
    ix, keys, base = build(t, metric, 1500, 100, 1)
    slots = ix.slots(keys)
    assert sorted(slots.tolist()) == list(range(1500)) and ix.slots([1, 2]).tolist() == [-1, -1]
    stored = learn.lookup(ix, torch.from_numpy(np.arange(1500)).to(DEV))
    assert stored.dtype == t and torch.equal(stored[torch.from_numpy(slots).to(DEV)], torch.from_numpy(base).to(DEV).to(t))
    g = gen(2)
    y = torch.randint(1500, (66,), generator=g, device=DEV)
    q = (stored[y].float() + 0.05 * torch.randn(66, 100, generator=g, device=DEV)).to(t)
    gl = torch.rand(66, generator=g, device=DEV)
    check(q, stored, y, gl, 8.0, metric, rows=ix)
    # removed members: out of the loss, no gradient, no label, read as zeros
    gone = keys[::5]
    for k in gone:
        assert ix.remove(int(k))
    dead = torch.zeros(1500, dtype=torch.bool, device=DEV)
    dead[torch.from_numpy(slots[::5]).to(DEV)] = True
    assert (ix.slots(gone) == -1).all()
    _, _, _, dw = check(q, stored, y, gl, 8.0, metric, rows=ix, dead=dead)
    assert (dw[dead] == 0).all()
    read = learn.lookup(ix, torch.arange(1500, device=DEV))
    assert (read[dead] == 0).all() and torch.equal(read[~dead], stored[~dead])


def test_members_added_and_updated_one_by_one():
    """single adds and updates are staged: a call sees them all"""
    ix, keys, base = build(F32, vs.IP, 300, 24, 4)
    extra = np.random.default_rng(5).standard_normal((6, 24)).astype(np.float32)
    for j in range(5):
        ix.add(10_000 + j, extra[j])
    assert ix.remove(int(keys[7]))
    ix.add(int(keys[7]), extra[5])
    slots = torch.from_numpy(ix.slots([10_000, 10_001, 10_002, 10_003, 10_004, int(keys[7]), int(keys[8])])).to(DEV)
    want = torch.from_numpy(np.concatenate([extra, base[8:9]])).to(DEV)
    assert torch.equal(learn.lookup(ix, slots), want)
    loss, lse = learn.softmax_loss(want, ix, slots)
    members = torch.from_numpy(np.concatenate([np.delete(base, 7, 0), extra])).to(DEV).double()
    z = want.double() @ members.t()
    # a score is off by |q| |w| (3 * 2^-22 + 3 (D + 64) * 2^-24), the sum and lse's rounding by 2^-24 (80 + 8 |z|), as in `reference`
    e = float(want.norm(dim=1).max() * members.norm(dim=1).max()) * (3 * 2.0 ** -22 + 3 * (24 + 64) * 2.0 ** -24) + 2.0 ** -24 * (80 + 8 * float(z.abs().max()))
    want_lse = torch.logsumexp(z, dim=1)
    assert (lse.double() - want_lse).abs().max() <= e
    assert (loss.double() - (want_lse - (want.double() ** 2).sum(1))).abs().max() <= 2 * e


def test_index_types_and_metrics_that_are_refused():
    for kw in (dict(quantization=vs.I8), dict(quantization=vs.B1)):
        ix = vs.HipUsearchIndex(64, vs.COS, **kw)
        ix.reserve(10)
        with pytest.raises(vs.VsError):
            learn.lookup(ix, torch.zeros(1, dtype=torch.int64, device=DEV))
    ix, _, _ = build(F32, vs.L2SQ, 20, 64, 3)
    q, y = torch.randn(2, 64, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(vs.VsError):
        learn.softmax_loss(q, ix, y)
    with pytest.raises(vs.VsError):
        learn.softmax_loss(q, ix, y, metric=learn.IP)
    assert learn.lookup(ix, y).shape == (2, 64)  # (reading rows needs no metric)
    empty = vs.HipUsearchIndex(64, vs.IP)
    loss, lse = learn.softmax_loss(q, empty, y)
    assert (loss == 0).all() and (lse == -float("inf")).all()


# ---------------------------------------------------------------------------------------------------- streams, graphs, a run of it all
def test_another_stream_and_two_calls_at_once():
    q, w, y, gl = case(200, 5000, 96, BF16, BF16, seed=14)
    l0, s0 = learn.softmax_loss(q, w, y, 8.0)
    a0, b0 = learn.softmax_loss_grad(q, w, y, s0, gl, 8.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for st in streams:
        with torch.cuda.stream(st):
            l, s = learn.softmax_loss(q, w, y, 8.0)
            out.append((l, s) + learn.softmax_loss_grad(q, w, y, s, gl, 8.0))
    torch.cuda.synchronize()
    for o in out:
        assert all(torch.equal(x, z) for x, z in zip(o, (l0, s0, a0, b0)))


def test_called_from_several_threads():
    import threading
    q, w, y, gl = case(130, 2500, 64, F32, F32, seed=17)
    ids = torch.randint(2500, (700,), device=DEV)
    want = learn.softmax_loss(q, w, y, 8.0)
    want = want + learn.softmax_loss_grad(q, w, y, want[1], gl, 8.0) + (learn.lookup_grad(w[ids], ids, 2500),)
    torch.cuda.synchronize()
    bad = []

    def run():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                l = learn.softmax_loss(q, w, y, 8.0)
                got = l + learn.softmax_loss_grad(q, w, y, l[1], gl, 8.0) + (learn.lookup_grad(w[ids], ids, 2500),)
                torch.cuda.current_stream().synchronize()
                bad.extend(0 for a, b in zip(got, want) if not torch.equal(a, b))

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_captured_and_replayed():
    for t in (BF16, F32):
        q, w, y, gl = case(150, 3000, 96, t, t, seed=15)
        ids = torch.randint(3000, (500,), device=DEV)

        def step():
            l, s = learn.softmax_loss(q, w, y, 8.0)
            a, b = learn.softmax_loss_grad(q, w, y, s, gl, 8.0)
            r = learn.lookup(w, ids, 0.5)
            learn.lookup_grad(r, ids, 3000, 0.5, into=b)
            return l, s, a, b, r

        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            step()
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = step()
        graph2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph2, stream=st):
            out2 = step()
        for rep in range(4):
            q2, w2, y2, gl2 = case(150, 3000, 96, t, t, seed=20 + rep)
            q.copy_(q2), w.copy_(w2), y.copy_(y2), gl.copy_(gl2)
            graph.replay()
            torch.cuda.synchronize()
            first = [x.clone() for x in out]
            want = step()
            torch.cuda.synchronize()
            graph2.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, z) for x, z in zip(first, want)) and all(torch.equal(x, z) for x, z in zip(out2, want)), rep


def test_few_f32_queries_captured_and_on_another_stream():
    for metric in (learn.IP, learn.COS):
        q, w, y, gl = case(20, 3000, 96, F32, F32, seed=18)

        def step():
            l, s = learn.softmax_loss(q, w, y, 8.0, metric)
            return (l, s) + learn.softmax_loss_grad(q, w, y, s, gl, 8.0, metric)

        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            other = step()
        st.synchronize()
        assert all(torch.equal(x, z) for x, z in zip(other, step()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = step()
        for rep in range(3):
            q2, w2, y2, gl2 = case(20, 3000, 96, F32, F32, seed=60 + rep)
            q.copy_(q2), w.copy_(w2), y.copy_(y2), gl.copy_(gl2)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, z) for x, z in zip(out, step())), rep


def test_learn_then_index_then_search():
    """a run of them together: vectors of items are learned so that the mean of a user's items finds the next item; the learned table is put
    into an index, whose exact search and whose own loss agree with the table's."""
    g = gen(16)
    v, d, n, ctx = 600, 64, 256, 4
    group = torch.arange(v, device=DEV) % 30  # items of a group follow each other
    w = torch.randn(v, d, generator=g, device=DEV) / d ** 0.5
    for step in range(3):
        first = torch.randint(v, (n,), generator=g, device=DEV)
        items = (first[:, None] + 30 * torch.randint(20, (n, ctx), generator=g, device=DEV)) % v
        label = (first + 30 * torch.randint(20, (n,), generator=g, device=DEV)) % v
        assert (group[items] == group[label][:, None]).all()
        gl = torch.full((n,), 1.0 / n, device=DEV)
        q = learn.lookup(w, items, 1.0 / ctx).sum(dim=1)
        loss, lse = learn.softmax_loss(q, w, label, 4.0)
        gq, gw = learn.softmax_loss_grad(q, w, label, lse, gl, 4.0)
        learn.lookup_grad(gq[:, None, :].expand(n, ctx, d).reshape(n, ctx, d), items, v, 1.0 / ctx, into=gw)
        leaf = w.double().requires_grad_(True)  # the same step in float64, through autograd on the CPU's formula
        qq = leaf[items].mean(dim=1)
        ref = torch.nn.functional.cross_entropy(4.0 * qq @ leaf.t(), label)
        ref.backward()
        assert abs(float((loss * gl).sum()) - float(ref.detach())) <= 1e-5
        # bound: 4 |v| * (2^-20 relative error of what enters) per sum of n * ctx terms of magnitude gl * 4 * |q|
        assert (gw.double() - leaf.grad).abs().max() <= 4 * 2.0 ** -18
        w = w - 5.0 * gw
    ix = vs.HipUsearchIndex(d, vs.IP)
    ix.reserve(v)
    keys = np.arange(v, dtype=np.uint64)
    torch.cuda.synchronize()
    ix.add_batch_device(keys, w.contiguous().data_ptr(), v, d)
    k, dist, found = ix.exact_search_batch(q.cpu().numpy(), 5)
    top = (q.double() @ w.double().t()).topk(5, dim=1)
    assert (found == 5).all() and np.abs((1 - dist) - top.values.cpu().numpy()).max() <= 1e-4
    l_ix, s_ix = learn.softmax_loss(q, ix, torch.from_numpy(ix.slots(label.cpu().numpy().astype(np.uint64))).to(DEV), 4.0)
    l_w, s_w = learn.softmax_loss(q, w, label, 4.0)
    assert (l_ix - l_w).abs().max() <= 1e-5 and (s_ix - s_w).abs().max() <= 1e-5
