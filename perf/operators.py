"""The class-head operators as a user calls them, beside their plain forms: what is timed, on which sizes.

A class head scores n rows of d features against V classes, z = x w^T (+ bias). Three operators:
``loss`` (softmax cross entropy with its gradients), ``distill`` (a teacher's top logits as the target, with
gradients) and ``topk`` (the k largest scores of a row, their classes and the log of the sum of all exponentials).
"""
import math

import torch

own = False

IGNORE = -100


def listed():
    return [
        # a training step of a language-model-sized head: the matrix products decide
        dict(name="loss_large", op="loss", dtype="bf16", n=8192, d=4096, V=131072, bias=False, ignored=0.0, weighted=False,
             base=False, dx=True, dw=True),
        # a fine-tuning batch: bias, a third of the rows ignored (prompt and padding), row weights, an odd class count
        dict(name="loss_masked", op="loss", dtype="bf16", n=2040, d=1024, V=50021, bias=True, ignored=0.35, weighted=True,
             base=False, dx=True, dw=True),
        # multiclass linear on dense rows, full batch: weights' gradient only, the last class fixed at 0
        dict(name="loss_dense_fp32", op="loss", dtype="fp32", n=20000, d=520, V=1008, bias=False, ignored=0.0, weighted=True,
             base=True, dx=False, dw=True),
        # a small step, where launches count
        dict(name="loss_small", op="loss", dtype="fp32", n=96, d=200, V=331, bias=True, ignored=0.0, weighted=False,
             base=False, dx=True, dw=True),
        # evaluation of a held-out set: no gradients
        dict(name="loss_eval", op="loss", dtype="bf16", n=4100, d=2048, V=32003, bias=False, ignored=0.1, weighted=False,
             base=False, dx=False, dw=False),
        # a student's step on a teacher's 64 best classes with the teacher's own normaliser, temperature 2
        dict(name="distill_large", op="distill", dtype="bf16", n=4096, d=2048, V=65536, k=64, T=2.0, bias=False, ragged=False,
             tail=True, dx=True, dw=True),
        # short ragged lists (some empty) renormalised, fp32, odd sizes
        dict(name="distill_ragged", op="distill", dtype="fp32", n=777, d=1000, V=5003, k=10, T=1.0, bias=True, ragged=True,
             tail=False, dx=True, dw=True),
        # one row answered: the weights are read once
        dict(name="topk_one", op="topk", dtype="bf16", n=1, d=4096, V=131072, k=16, T=1.0, bias=False),
        # a batch of rows answered
        dict(name="topk_batch", op="topk", dtype="bf16", n=48, d=2048, V=50021, k=40, T=1.0, bias=True),
        # a teacher writes down its top logits for a whole batch
        dict(name="topk_teacher", op="topk", dtype="bf16", n=4096, d=1024, V=65536, k=64, T=2.0, bias=False),
        # a few fp32 rows of an ordinary classifier: launches count
        dict(name="topk_small", op="topk", dtype="fp32", n=7, d=333, V=2003, k=5, T=1.0, bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "distill", "topk"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    most = 2e12 if op == "topk" else 8e12 if dtype == "bf16" else 1e12  # n d V products
    while True:
        n, d, V = _log(rng, 1, 8192), _log(rng, 16, 4096), _log(rng, 128, 131072)
        if rng.random() < 0.4:  # widths of real layers
            d = max(16, d // 64 * 64)
        if 2.0 * n * d * V <= most:
            break
    c = dict(op=op, dtype=dtype, n=n, d=d, V=V, bias=rng.random() < 0.5)
    if op == "loss":
        grads = rng.choice([(True, True), (True, True), (False, True), (True, False), (False, False)])
        c.update(ignored=rng.choice([0.0, 0.3]), weighted=rng.random() < 0.5, base=rng.random() < 0.25, dx=grads[0], dw=grads[1])
    elif op == "distill":
        c.update(k=_log(rng, 1, 128), T=rng.choice([1.0, 2.0, 3.5]), ragged=rng.random() < 0.5, tail=rng.random() < 0.5, dx=True, dw=True)
    else:
        c.update(k=_log(rng, 1, 128), T=rng.choice([1.0, 2.0]))
    return c


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    n, d, V = case["n"], case["d"], case["V"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    # scores of unrelated classes have a deviation of 2; a row points to its own class more or less clearly, as in a
    # half-trained model, and frequent classes come first
    w = (randn(V, d) * (2.0 / math.sqrt(d))).to(dt)
    own_class = (rand(n).pow(3) * V).long().clamp(max=V - 1)
    x = (randn(n, d) + (4.0 * rand(n, 1)) * w[own_class].float()).to(dt)
    s = {"case": dict(case), "x": x, "w": w, "bias": (randn(V) * 0.5).to(dt) if case["bias"] else None}
    if case["op"] == "loss":
        labels = own_class
        if case["base"]:
            labels = torch.where(rand(n) < 0.01, torch.full_like(labels, V), labels)
        if case["ignored"] > 0:
            labels = torch.where(rand(n) < case["ignored"], torch.full_like(labels, IGNORE), labels)
        s["labels"] = labels
        s["weight"] = 0.5 + rand(n) if case["weighted"] else None
    elif case["op"] == "distill":
        k = case["k"]
        idx = ((torch.arange(k, device=dev) + rand(n, k)) * (V / k)).long().clamp(max=V - 1)  # distinct classes
        idx = idx.gather(1, rand(n, k).argsort(1))
        idx[:, 0] = torch.where((idx[:, 1:] == own_class[:, None]).any(1), idx[:, 0], own_class)
        logits = (randn(n, k) * 2.0 + 6.0).sort(1, descending=True).values
        if case["ragged"]:  # lists shorter than k, some empty
            length = (rand(n, 1) * (k + 1)).long()
            idx = torch.where(torch.arange(k, device=dev)[None, :] < length, idx, torch.full_like(idx, -1))
        s["top_idx"], s["top_logits"] = idx, logits
        s["top_lse"] = torch.logsumexp(logits / case["T"], 1) + 0.3 * rand(n) if case["tail"] else None
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    if op == "loss":
        return _plain_loss(state)
    if op == "distill":
        return _plain_distill(state)
    return _plain_topk(state)


def _run_own(op, s):
    from ytk_learn_amd.ops import head

    c = s["case"]
    if op == "loss":
        r = head.softmax_head_loss(s["x"], s["w"], s["labels"], bias=s["bias"], weight=s["weight"], ignore_index=IGNORE,
                                   base_class=c["base"], want_dx=c["dx"], want_dw=c["dw"])
        return {"loss": r.loss, "lse": r.lse, "dx": r.dx, "dw": r.dw, "db": r.db}
    if op == "distill":
        r = head.distill_head_loss(s["x"], s["w"], s["top_idx"], s["top_logits"], bias=s["bias"], temperature=c["T"],
                                   top_lse=s["top_lse"], want_dx=c["dx"], want_dw=c["dw"])
        return {"loss": r.loss, "lse": r.lse, "dx": r.dx, "dw": r.dw, "db": r.db}
    values, classes, lse = head.head_topk(s["x"], s["w"], c["k"], bias=s["bias"], temperature=c["T"])
    return {"values": values, "classes": classes, "lse": lse}


# ------------------------------------------------------------------ plain forms
def _scores(s, dtype):
    z = s["x"].to(dtype) @ s["w"].to(dtype).t()
    return z if s["bias"] is None else z + s["bias"].to(dtype)


def _lse(z):
    m = z.amax(1, keepdim=True)
    return (m + (z - m).exp().sum(1, keepdim=True).log()).squeeze(1)


def _grads(s, D):
    c, x, w = s["case"], s["x"], s["w"]
    return {"dx": (D @ w.float()).to(x.dtype) if c["dx"] else None,
            "dw": (D.t() @ x.float()).to(w.dtype) if c["dw"] else None,
            "db": D.sum(0).to(w.dtype) if c["dw"] and s["bias"] is not None else None}


def _plain_loss(s):
    c, labels = s["case"], s["labels"]
    V = c["V"]
    z = _scores(s, torch.float32)
    if c["base"]:
        z = torch.cat([z, z.new_zeros(z.shape[0], 1)], 1)
    lse = _lse(z)
    valid = labels != IGNORE
    y = torch.where(valid, labels, torch.zeros_like(labels))
    g = valid.float() if s["weight"] is None else s["weight"] * valid
    loss = torch.where(valid, g * (lse - z.gather(1, y[:, None]).squeeze(1)), torch.zeros_like(lse))
    if not (c["dx"] or c["dw"]):
        return {"loss": loss, "lse": lse, "dx": None, "dw": None, "db": None}
    D = (z - lse[:, None]).exp()
    D = (D.scatter_add(1, y[:, None], -torch.ones_like(D[:, :1])) * g[:, None])[:, :V]
    return {"loss": loss, "lse": lse, **_grads(s, D)}


def _plain_distill(s):
    c, idx = s["case"], s["top_idx"]
    T = c["T"]
    z = _scores(s, torch.float32) / T
    lse = _lse(z)
    there = idx >= 0
    t = torch.where(there, s["top_logits"].float() / T, torch.full_like(s["top_logits"], -math.inf))
    if s["top_lse"] is None:
        m = t.amax(1, keepdim=True).clamp(min=-1e30)
        e = (t - m).exp()
        total = e.sum(1, keepdim=True).clamp(min=1e-30)
        q, logq = e / total, t - m - total.log()
    else:
        logq = t - s["top_lse"][:, None]
        q = logq.exp()
    logq = torch.where(there, logq, torch.zeros_like(logq))
    at = idx.clamp(min=0)
    logp = z.gather(1, at) - lse[:, None]
    loss = T * T * torch.where(there, q * (logq - logp), torch.zeros_like(q)).sum(1)
    D = T * ((z - lse[:, None]).exp() * q.sum(1, keepdim=True)).scatter_add(1, at, -q)
    return {"loss": loss, "lse": lse, **_grads(s, D)}


def _plain_topk(s):
    # 64 bits: the order of neighbouring scores is an output, and 32-bit sums swap near ties
    c = s["case"]
    z = _scores(s, torch.float64) / c["T"]
    lse = _lse(z).float()
    values, classes = torch.topk(z, min(c["k"] + 8, c["V"]), dim=1)
    classes, order = classes.sort(1)  # equal scores: the lowest class first
    values, order = values.gather(1, order).sort(dim=1, descending=True, stable=True)
    classes = classes.gather(1, order)
    return {"values": values[:, :c["k"]].float(), "classes": classes[:, :c["k"]], "lse": lse}


# ------------------------------------------------------------------ work and the definition in 64 bits
def work(case):
    n, d, V = case["n"], case["d"], case["V"]
    e = 2 if case["dtype"] == "bf16" else 4
    bias = V * e if case["bias"] else 0
    read, written, products = (n * d + V * d) * e + bias, n * 4, 1
    if case["op"] == "topk":
        written += n * case["k"] * 12
    else:
        written += n * 4
        read += n * 8 + (n * 4 if case.get("weighted") else 0) if case["op"] == "loss" else n * case["k"] * 12
        written += (n * d * e if case["dx"] else 0) + ((V * d * e + bias) if case["dw"] else 0)
        products += int(case["dx"]) + int(case["dw"])
    return {"bytes": read + written, "flops": 2.0 * n * d * V * products}


def exact(case, seed):
    s = prepare(case, seed)
    x, w = s["x"].double(), s["w"].double()
    z = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
    if case["op"] == "topk":
        z /= case["T"]
        v, i = z.sort(dim=1, descending=True, stable=True)
        return {"values": v[:, :case["k"]].contiguous(), "classes": None, "lse": torch.logsumexp(z, 1)}
    n = x.shape[0]
    if case["op"] == "loss":
        T, labels = 1.0, s["labels"]
        if case["base"]:
            z = torch.nn.functional.pad(z, (0, 1))
        keep = (labels != IGNORE).double()
        gain = keep if s["weight"] is None else keep * s["weight"].double()
        idx, q = labels.clamp(min=0)[:, None], keep[:, None]
    else:
        T = case["T"]
        z /= T
        gain = torch.ones(n, dtype=torch.float64, device=x.device)
        idx = s["top_idx"].clamp(min=0)
        t = (s["top_logits"].double() / T).masked_fill(s["top_idx"] < 0, -math.inf)
        norm = torch.logsumexp(t, 1) if s["top_lse"] is None else s["top_lse"].double()
        q = (t - norm[:, None]).exp().masked_fill(s["top_idx"] < 0, 0.0)
    lse = torch.logsumexp(z, 1)
    z -= lse[:, None]
    loss = gain * T * T * (torch.xlogy(q, q) - q * z.gather(1, idx)).sum(1)
    out = {"loss": loss, "lse": lse, "dx": None, "dw": None, "db": None}
    if case["dx"] or case["dw"]:
        D = z.exp_().mul_(q.sum(1, keepdim=True)).scatter_add_(1, idx, -q).mul_(T * gain[:, None])[:, :case["V"]]
        out["dx"] = D @ w if case["dx"] else None
        out["dw"] = D.t() @ x if case["dw"] else None
        out["db"] = D.sum(0) if case["dw"] and s["bias"] is not None else None
    return out
