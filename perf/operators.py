"""The softmax head over a large vocabulary, with its gradient, and the global
gradient norm with clipping: the operators on device tensors, each in a plain
form and through the package's entry points.

A case is a dict of plain values.  op "loss" or "grad" (the softmax head):

    rows, width, vocab   sizes of hidden (rows x width) and weight (vocab x width)
    dtype                "bf16", "fp16" or "fp32"
    left_out             share of each 512-row sequence without a label (a prompt)
    weighted             rows have weights
    softcap, z_loss      0 for none
    grad_scale           the loss scale of a float16 run

op "norm" or "clip" (gradients of many tensors):

    tensors   "adapters", "ragged" or "block": how shapes follow from the sizes
    count, width, vocab, dtype
    inv_scale, max_norm  max_norm below the norm clips

Sizes are generic: widths and vocabularies of small to large language models.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SEQ = 512


def _head(name, op, rows, width, vocab, dtype, left_out=0.0, weighted=False, softcap=0.0,
          z_loss=0.0, grad_scale=1.0):
    c = dict(op=op, rows=rows, width=width, vocab=vocab, dtype=dtype, left_out=left_out,
             weighted=weighted, softcap=softcap, z_loss=z_loss, grad_scale=grad_scale)
    return dict(c, name=name) if name else c


def _many(name, op, tensors, count, width, vocab, dtype, inv_scale=1.0, max_norm=1.0):
    c = dict(op=op, tensors=tensors, count=count, width=width, vocab=vocab, dtype=dtype,
             inv_scale=inv_scale, max_norm=max_norm)
    return dict(c, name=name) if name else c


def listed():
    return [
        # The log-probability of one token while text is scored as it arrives.
        _head("score_1", "loss", 1, 2048, 32000, "bf16"),
        # A small batch of candidate tokens; an odd vocabulary, a capped model.
        _head("score_13", "loss", 13, 2560, 50257, "fp16", softcap=30.0),
        # Perplexity of a short text in full precision.
        _head("eval_fp32", "loss", 700, 1024, 30011, "fp32"),
        # Evaluation of long texts with a large vocabulary.
        _head("eval_large", "loss", 4096, 4096, 131072, "bf16"),
        # A training step of a small model in full precision; prompts carry no loss.
        _head("train_small", "grad", 128, 512, 4099, "fp32", left_out=0.25, weighted=True),
        # A float16 run with its loss scale, a capped output and the z-loss.
        _head("train_capped", "grad", 1500, 2048, 32003, "fp16", softcap=30.0, z_loss=1e-4,
              grad_scale=1024.0),
        # A head on features of an odd width (embeddings with columns added).
        _head("train_odd", "grad", 2047, 1001, 50257, "bf16", weighted=True),
        # The training step of a large model; a quarter of the rows are prompts.
        _head("train_large", "grad", 8192, 4096, 131072, "bf16", left_out=0.25),
        # The gradients of low-rank adapters: many small tensors.
        _many("norm_adapters", "norm", "adapters", 192, 1024, 0, "fp32"),
        # Tensors of any size, scaled gradients.
        _many("norm_ragged", "norm", "ragged", 61, 700, 0, "fp16", inv_scale=1.0 / 1024),
        # Two blocks of a transformer; norms in full precision.
        _many("clip_blocks", "clip", "block", 2, 2560, 0, "bf16", max_norm=1.0),
        # A wide block and the vocabulary's weight.
        _many("clip_large", "clip", "block", 1, 8192, 131072, "bf16", inv_scale=0.5, max_norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "grad", "grad", "norm", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("loss", "grad"):
        while True:
            rows = _log_int(rng, 1, 8192)
            width = _log_int(rng, 64, 8192)
            if rng.random() < 0.75:
                width = (width + 63) // 64 * 64
            vocab = _log_int(rng, 1000, 200000)
            if rows * width * vocab <= (1 << 39 if dtype != "fp32" else 1 << 37):
                break
        return _head(None, op, rows, width, vocab, dtype,
                     left_out=rng.choice([0.0, 0.0, 0.3, 0.6]) if rows >= 64 else 0.0,
                     weighted=rng.random() < 0.3, softcap=rng.choice([0.0, 0.0, 30.0]),
                     z_loss=rng.choice([0.0, 1e-4]),
                     grad_scale=4096.0 if dtype == "fp16" and op == "grad" else 1.0)
    kind = rng.choice(["adapters", "ragged", "block"])
    count = {"adapters": _log_int(rng, 8, 400), "ragged": _log_int(rng, 2, 400),
             "block": rng.randint(1, 3)}[kind]
    if op == "clip":
        count = min(count, 60)
    width = _log_int(rng, 64, 4096)
    return _many(None, op, kind, count, width, 0, dtype,
                 inv_scale=rng.choice([1.0, 1.0 / 128]), max_norm=rng.choice([0.1, 1.0, 1e9]))


def _left_out(case):
    """Which rows have no label: the first part of each sequence."""
    part = int(_SEQ * case["left_out"]) if case["rows"] >= _SEQ else int(
        case["rows"] * case["left_out"])
    return [i % _SEQ < part for i in range(case["rows"])]


def _shapes(case):
    """[(rows, cols or None, full precision)] of the case's tensors."""
    d = case["width"]
    if case["tensors"] == "adapters":
        return [((16, d) if i % 2 else (d, 16), False) for i in range(case["count"])]
    if case["tensors"] == "ragged":
        rng = random.Random(case["count"] * 7919 + d)
        return [((int(math.exp(rng.uniform(0.0, math.log(d * d)))),), False)
                for _ in range(case["count"])]
    out = []
    for _ in range(case["count"]):
        out += [((d, d), False)] * 4 + [((4 * d, d), False), ((d, 4 * d), False), ((d,), True),
                                        ((d,), True)]
    if case["vocab"]:
        out.append(((case["vocab"], d), False))
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = "cuda"
    dtype = _DTYPES[case["dtype"]]
    if case["op"] in ("loss", "grad"):
        n, d, v = case["rows"], case["width"], case["vocab"]
        # Scores of standard deviation 2 (5 under a cap); the label's score is
        # raised by up to 12, so that rows range from surprising to certain.
        # Labels are spread over the vocabulary's logarithm, as words are.
        spread = 5.0 if case["softcap"] else 2.0
        weight = torch.randn(v, d, generator=g, device=dev).mul_(spread / math.sqrt(d)).to(dtype)
        hidden = torch.randn(n, d, generator=g, device=dev)
        u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
        labels = (float(v) ** u).long().clamp_(1, v) - 1
        raised = torch.rand(n, 1, generator=g, device=dev) * (12.0 / spread ** 2)
        hidden = (hidden + raised * weight[labels].float()).to(dtype)
        labels[torch.tensor(_left_out(case), device=dev)] = -100
        row_weight = 0.25 + torch.rand(n, generator=g, device=dev) if case["weighted"] else None
        return dict(case, hidden=hidden, weight=weight, labels=labels, row_weight=row_weight)
    grads = []
    for shape, full in _shapes(case):
        t = torch.randn(*shape, generator=g, device=dev) * (0.01 / case["inv_scale"])
        grads.append(t if full else t.to(dtype))
    out = [torch.empty_like(t) for t in grads] if case["op"] == "clip" else None
    return dict(case, grads=grads, out=out)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bsscl-gbm_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import bsscl_gbm
    return bsscl_gbm


def _run_own(s):
    pkg = _package()
    if s["op"] == "loss":
        r = pkg.linear_softmax_loss(s["hidden"], s["weight"], s["labels"],
                                    row_weight=s["row_weight"], softcap=s["softcap"],
                                    z_loss=s["z_loss"])
        return {"loss": r.loss, "row_loss": r.row_loss, "lse": r.lse}
    if s["op"] == "grad":
        r = pkg.linear_softmax_grad(s["hidden"], s["weight"], s["labels"],
                                    row_weight=s["row_weight"], softcap=s["softcap"],
                                    z_loss=s["z_loss"], grad_scale=s["grad_scale"])
        return {"loss": r.loss, "row_loss": r.row_loss, "lse": r.lse, "d_hidden": r.d_hidden,
                "d_weight": r.d_weight}
    if s["op"] == "norm":
        return {"norm": pkg.grad_norm(s["grads"], inv_scale=s["inv_scale"])}
    norm = pkg.clip_grads(s["grads"], s["max_norm"], inv_scale=s["inv_scale"], out=s["out"])
    return {"norm": norm, "out": s["out"]}


def _run_head(s):
    h, w, y, cap = s["hidden"].float(), s["weight"].float(), s["labels"], s["softcap"]
    counts = (y >= 0) & (y < w.shape[0])
    at = torch.where(counts, y, torch.zeros_like(y))[:, None]
    z = h @ w.t()
    if cap:
        z = cap * torch.tanh(z / cap)
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    zero = torch.zeros_like(lse)
    row_loss = torch.where(counts[:, None], lse - z.gather(1, at) + s["z_loss"] * lse * lse, zero)
    u = torch.ones_like(lse) if s["row_weight"] is None else s["row_weight"].float()[:, None]
    u = torch.where(counts[:, None], u, zero)
    u = u / u.sum()
    out = {"loss": (u * row_loss).sum(), "row_loss": row_loss[:, 0],
           "lse": torch.where(counts[:, None], lse, zero)[:, 0]}
    if s["op"] == "grad":
        u = u * s["grad_scale"]
        ds = torch.exp(z - lse) * (u * (1.0 + 2.0 * s["z_loss"] * lse))
        # The label's p - 1 as an expm1 of its own: their difference would
        # lose the small values of rows that are nearly certain.
        zy = z.gather(1, at) - lse
        ds.scatter_(1, at, u * (torch.expm1(zy) + 2.0 * s["z_loss"] * lse * torch.exp(zy)))
        if cap:
            ds = ds * (1.0 - (z / cap) * (z / cap))
        out["d_hidden"] = (ds @ w).to(s["hidden"].dtype)
        out["d_weight"] = (ds.t() @ h).to(s["weight"].dtype)
    return out


def _run_many(s):
    squares = torch.stack([t.double().square().sum() for t in s["grads"]])
    norm = torch.sqrt(squares.sum()) * abs(s["inv_scale"])
    if s["op"] == "norm":
        return {"norm": norm.float()}
    factor = (torch.clamp(s["max_norm"] / norm, max=1.0) * s["inv_scale"]).float()
    return {"norm": norm.float(), "out": [(t.float() * factor).to(t.dtype) for t in s["grads"]]}


def run(state):
    if own:
        return _run_own(state)
    return _run_head(state) if state["op"] in ("loss", "grad") else _run_many(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("loss", "grad"):
        n, d, v = case["rows"], case["width"], case["vocab"]
        used = n - sum(_left_out(case))
        once = (used * d + v * d) * size + 8 * n + 8 * n + 4 + (4 * n if case["weighted"] else 0)
        if case["op"] == "loss":
            return {"bytes": once, "flops": 2 * used * d * v}
        return {"bytes": once + (n * d + v * d) * size, "flops": 6 * used * d * v}
    total = values = 0
    for shape, full in _shapes(case):
        values += math.prod(shape)
        total += math.prod(shape) * (4 if full else size)
    if case["op"] == "norm":
        return {"bytes": total + 4, "flops": 2 * values}
    return {"bytes": 2 * total + 4, "flops": 3 * values}


def exact(case, seed):
    """The definition in float64, some rows at a time."""
    s = prepare(case, seed)
    if case["op"] in ("norm", "clip"):
        sq = sum(float(torch.linalg.vector_norm(t.double())) ** 2 for t in s["grads"])
        norm = abs(case["inv_scale"]) * math.sqrt(sq)
        if case["op"] == "norm":
            return {"norm": torch.tensor(norm, dtype=torch.float64)}
        f = case["inv_scale"] * (case["max_norm"] / norm if norm > case["max_norm"] else 1.0)
        return {"norm": torch.tensor(norm, dtype=torch.float64),
                "out": [t.double() * f for t in s["grads"]]}
    w = s["weight"].double()
    n, d, v = case["rows"], case["width"], case["vocab"]
    y, cap, zeta = s["labels"], case["softcap"], case["z_loss"]
    rows = [i for i, out in enumerate(_left_out(case)) if not out]
    if s["row_weight"] is None:
        share = torch.full((n,), 1.0 / len(rows), dtype=torch.float64, device=y.device)
    else:
        share = s["row_weight"].double() / s["row_weight"].double()[rows].sum()
    out = {k: torch.zeros(n, dtype=torch.float64, device=y.device) for k in ("row_loss", "lse")}
    grad = case["op"] == "grad"
    d_hidden = torch.zeros(n, d, dtype=torch.float64, device=y.device) if grad else None
    d_weight = torch.zeros(v, d, dtype=torch.float64, device=y.device) if grad else None
    for a in range(0, len(rows), 2048):
        at = torch.tensor(rows[a:a + 2048], device=y.device)
        h = s["hidden"][at].double()
        z = torch.mm(h, w.t())
        slope = None
        if cap:
            t = torch.tanh(z / cap)
            z, slope = cap * t, 1.0 - t * t
        log_p = torch.log_softmax(z, dim=1)
        k = torch.arange(len(at), device=y.device)
        lse = z[:, 0] - log_p[:, 0]
        out["lse"][at] = lse
        out["row_loss"][at] = zeta * lse ** 2 - log_p[k, y[at]]
        if grad:
            ds = log_p.exp()
            ds += (2.0 * zeta * lse)[:, None] * ds
            ds[k, y[at]] -= 1.0
            if cap:
                ds *= slope
            ds *= (case["grad_scale"] * share[at])[:, None]
            d_hidden[at] = torch.mm(ds, w)
            d_weight += torch.mm(ds.t(), h)
    out["loss"] = (share * out["row_loss"]).sum()
    if grad:
        out.update(d_hidden=d_hidden, d_weight=d_weight)
    return out
