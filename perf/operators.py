"""Workloads of the learning operators (vector_store_amd.learn): vectors read by row number, the softmax loss of
queries over all rows of a table, and the gradients of both.  `run` computes a case in plain torch operations in
32 bits, or (where `own` is true) through the package's calls.

    loss_i = log(sum_j exp z_ij) - z_i,label      z_ij = scale * <q_i, w_j>   (cosine: of the normalised vectors)
    out_t  = scale * w[id_t]
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the vectors of one answer (top-16 of a 10k x 128 index) read back by row number: a call's latency
        {"name": "lookup_answer", "kind": "lookup", "n": 16, "rows": 10_000, "dim": 128, "dtype": "f32"},
        # the positives of a large training batch out of a million bf16 vectors, an odd count
        {"name": "lookup_batch", "kind": "lookup", "n": 40_001, "rows": 1_000_000, "dim": 768, "dtype": "bf16"},
        # gradient of a small step's lookups
        {"name": "lookup_grad_small", "kind": "lookup_grad", "n": 1_000, "rows": 10_000, "dim": 128, "dtype": "f32"},
        # gradient of 128k lookups whose popularity is skewed (a few rows are read thousands of times)
        {"name": "lookup_grad_batch", "kind": "lookup_grad", "n": 131_072, "rows": 262_144, "dim": 768, "dtype": "bf16"},
        # odd sizes and f16 storage
        {"name": "lookup_grad_odd", "kind": "lookup_grad", "n": 30_011, "rows": 50_021, "dim": 1536, "dtype": "f16"},
        # how probable is this answer: one query against a million members
        {"name": "loss_one", "kind": "loss", "n": 1, "rows": 1_000_000, "dim": 768, "dtype": "bf16", "cosine": False},
        # validation loss of a batch of queries over the whole index
        {"name": "loss_batch", "kind": "loss", "n": 256, "rows": 1_000_000, "dim": 768, "dtype": "bf16", "cosine": False},
        # the small index in the storage type most indexes have, cosine
        {"name": "loss_small", "kind": "loss", "n": 33, "rows": 10_000, "dim": 128, "dtype": "f32", "cosine": True},
        # training steps: loss and the gradients of queries and rows; a small one ...
        {"name": "step_small", "kind": "step", "n": 64, "rows": 10_000, "dim": 128, "dtype": "f32", "cosine": False},
        # ... the bulk of a training run ...
        {"name": "step_large", "kind": "step", "n": 4_096, "rows": 131_072, "dim": 768, "dtype": "bf16", "cosine": False},
        # ... f32 vectors under cosine, nothing a multiple of a tile ...
        {"name": "step_f32_cosine", "kind": "step", "n": 777, "rows": 50_021, "dim": 1536, "dtype": "f32", "cosine": True},
        # ... and f16 with a scaled loss
        {"name": "step_f16", "kind": "step", "n": 300, "rows": 100_003, "dim": 384, "dtype": "f16", "cosine": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "lookup_grad", "loss", "step"])
    case = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"])}
    dim = rng.choice([128, 384, 768, 1024, 1536, _log(rng, 16, 1536)])
    if kind in ("lookup", "lookup_grad"):
        top = 1_000_000 if kind == "lookup" else 262_144
        case.update(n=_log(rng, 1, 40_001 if kind == "lookup" else 131_072), rows=_log(rng, 1_000, top), dim=dim)
        # no more bytes than the largest listed case
        limit = (262_144 + 131_072) * 768 * 2
        while (case["n"] + (case["rows"] if kind == "lookup_grad" else case["n"])) * dim * BYTES[case["dtype"]] > limit:
            case["rows"], case["n"] = max(1_000, case["rows"] // 2), max(1, case["n"] // 2)
    else:
        case.update(n=_log(rng, 1, 4_096 if kind == "step" else 256), rows=_log(rng, 1_000, 1_000_000 if kind == "loss" else 131_072), dim=dim,
                    cosine=rng.random() < 0.4)
        limit = 777 * 50_021 * 1536 if case["dtype"] != "bf16" else (4_096 * 131_072 * 768 if kind == "step" else 256 * 1_000_000 * 768)
        while case["n"] * case["rows"] * dim > limit:
            case["rows"], case["n"] = max(1_000, case["rows"] * 2 // 3), max(1, case["n"] * 2 // 3)
    return case


def _randn(g, n, dim, dtype, rms):
    return (torch.randn((n, dim), generator=g, device="cuda", dtype=torch.float32) * rms).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, rows, dim, dtype = case["n"], case["rows"], case["dim"], DTYPES[case["dtype"]]
    kind = case["kind"]
    s = {"kind": kind, "rows": rows, "dim": dim, "dtype": dtype}
    if kind in ("lookup", "lookup_grad"):
        # popularity falls as a power of the rank (u^4 * rows: one read in six goes to a thousandth of the rows)
        u = torch.rand((n,), generator=g, device="cuda", dtype=torch.float64)
        perm = torch.randperm(rows, generator=g, device="cuda")
        ids = perm[(u.pow(4) * rows).long().clamp_(max=rows - 1)]
        pad = torch.rand((n,), generator=g, device="cuda") < 0.02  # padding of ragged batches
        s["ids"] = torch.where(pad, torch.full_like(ids, -1), ids)
        s["scale"] = math.sqrt(dim) / 4
        if kind == "lookup":
            s["table"] = _randn(g, rows, dim, dtype, 1 / math.sqrt(dim))
        else:
            s["grad"] = _randn(g, n, dim, dtype, 1e-2)
        return s
    # rows of about unit norm; a query lies near the member it is labelled with, so that the label is likely but not certain
    norms = torch.rand((rows, 1), generator=g, device="cuda") * 0.4 + 0.8
    table = torch.randn((rows, dim), generator=g, device="cuda", dtype=torch.float32)
    table = (table.mul_(norms / math.sqrt(dim))).to(dtype)
    labels = torch.randint(rows, (n,), generator=g, device="cuda")
    noise = torch.randn((n, dim), generator=g, device="cuda", dtype=torch.float32) / math.sqrt(dim)
    s["queries"] = (0.7 * table[labels].float() + 0.7 * noise).to(dtype)
    s["table"] = table
    if n > 1:
        pad = torch.rand((n,), generator=g, device="cuda") < 0.03
        labels = torch.where(pad, torch.full_like(labels, -1), labels)
    s["labels"] = labels
    s["cosine"] = case["cosine"]
    s["scale"] = 20.0
    if kind == "step":
        valid = max(1, int((labels >= 0).sum()))
        loss_scale = 512.0 if dtype == torch.float16 else 1.0
        s["grad_loss"] = torch.full((n,), loss_scale / valid, device="cuda", dtype=torch.float32)
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from vector_store_amd import learn

    if s["kind"] == "lookup":
        return learn.lookup(s["table"], s["ids"], s["scale"])
    if s["kind"] == "lookup_grad":
        return learn.lookup_grad(s["grad"], s["ids"], s["rows"], s["scale"])
    metric = learn.COS if s["cosine"] else learn.IP
    loss, lse = learn.softmax_loss(s["queries"], s["table"], s["labels"], s["scale"], metric)
    if s["kind"] == "loss":
        return loss, lse
    dq, dw = learn.softmax_loss_grad(s["queries"], s["table"], s["labels"], lse, s["grad_loss"], s["scale"], metric)
    return loss, lse, dq, dw


def _plain(s):
    dtype = s["dtype"]
    if s["kind"] == "lookup":
        out = s["table"][s["ids"].clamp(min=0)].float() * s["scale"]
        return torch.where((s["ids"] >= 0)[:, None], out, torch.zeros_like(out)).to(dtype)
    if s["kind"] == "lookup_grad":
        keep = s["ids"] >= 0
        g = torch.where(keep[:, None], s["grad"].float() * s["scale"], torch.zeros((), device="cuda"))
        out = torch.zeros((s["rows"], s["dim"]), dtype=torch.float32, device="cuda")
        out.index_add_(0, s["ids"].clamp(min=0), g)
        return out.to(dtype)
    q, w = s["queries"].float(), s["table"].float()
    if s["cosine"]:
        fq, fw = _inverse_norm(q), _inverse_norm(w)
        q, w = q * fq, w * fw
    z = (q @ w.t()) * s["scale"]
    top = z.max(dim=1, keepdim=True).values
    lse = (torch.log(torch.exp(z - top).sum(dim=1, keepdim=True)) + top)
    keep = s["labels"] >= 0
    safe = s["labels"].clamp(min=0)
    at = z.gather(1, safe[:, None])[:, 0]
    loss = torch.where(keep, lse[:, 0] - at, torch.zeros_like(at))
    if s["kind"] == "loss":
        return loss, lse[:, 0]
    c = torch.exp(z - lse)
    c[torch.arange(len(safe), device=c.device), safe] -= 1.0
    c *= torch.where(keep, s["grad_loss"], torch.zeros_like(s["grad_loss"]))[:, None] * s["scale"]
    dq, dw = c @ w, c.t() @ q
    if s["cosine"]:  # through the normalisation: what lies along the vector itself is lost
        dq = (dq - q * (q * dq).sum(dim=1, keepdim=True)) * fq
        dw = (dw - w * (w * dw).sum(dim=1, keepdim=True)) * fw
    return loss, lse[:, 0], dq.to(dtype), dw.to(dtype)


def _inverse_norm(x):
    n = (x * x).sum(dim=1, keepdim=True).sqrt()
    return torch.where(n > 0, 1.0 / n, torch.zeros_like(n))


def work(case):
    n, rows, dim, e = case["n"], case["rows"], case["dim"], BYTES[case["dtype"]]
    kind = case["kind"]
    if kind == "lookup":
        return {"bytes": n * (2 * dim * e + 8), "flops": n * dim}
    if kind == "lookup_grad":
        return {"bytes": (n + rows) * dim * e + 8 * n, "flops": 2 * n * dim}
    if kind == "loss":
        return {"bytes": (n + rows) * dim * e + 16 * n, "flops": 2 * n * rows * dim}
    return {"bytes": 2 * (n + rows) * dim * e + 20 * n, "flops": 6 * n * rows * dim}


def exact(case, seed):
    s = prepare(case, seed)
    ids = s["ids"] if "ids" in s else s["labels"]
    if s["kind"] == "lookup":
        out = torch.zeros((case["n"], case["dim"]), dtype=torch.float64, device="cuda")
        out[ids >= 0] = s["table"][ids[ids >= 0]].double() * s["scale"]
        return out
    if s["kind"] == "lookup_grad":
        out = torch.zeros((case["rows"], case["dim"]), dtype=torch.float64, device="cuda")
        out.index_put_((ids[ids >= 0],), s["grad"][ids >= 0].double() * s["scale"], accumulate=True)
        return out
    w = s["table"].double()
    nw = w.norm(dim=1)
    loss, lse, dq = [], [], []
    dw = torch.zeros_like(w) if s["kind"] == "step" else None
    step = max(1, (1 << 28) // case["rows"])  # queries at a time: at most 2 GiB of scores
    for a in range(0, case["n"], step):
        q = s["queries"][a:a + step].double()
        y = ids[a:a + step]
        nq = q.norm(dim=1)
        z = s["scale"] * torch.mm(q, w.t())
        if s["cosine"]:
            z = z / nq[:, None] / nw[None, :]
        l = torch.logsumexp(z, dim=1)
        r = torch.arange(len(y), device=y.device)[y >= 0]
        e = torch.zeros_like(l)
        e[r] = l[r] - z[r, y[r]]
        loss.append(e)
        lse.append(l)
        if dw is None:
            continue
        p = torch.softmax(z, dim=1)
        p[r, y[r]] -= 1.0
        p *= (s["grad_loss"][a:a + step].double() * (y >= 0))[:, None]
        if s["cosine"]:
            t = p * z  # sum over j (over i) of p z: the part of the gradient along q_i (along w_j)
            p = s["scale"] * p / nq[:, None] / nw[None, :]
            dq.append(torch.mm(p, w) - q * (t.sum(dim=1) / nq.pow(2))[:, None])
            dw += torch.mm(p.t(), q) - w * (t.sum(dim=0) / nw.pow(2))[:, None]
        else:
            dq.append(s["scale"] * torch.mm(p, w))
            dw += s["scale"] * torch.mm(p.t(), q)
    if dw is None:
        return torch.cat(loss), torch.cat(lse)
    return torch.cat(loss), torch.cat(lse), torch.cat(dq), dw
