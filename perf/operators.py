"""Workloads of the distillation operators: top logits of a teacher, and the loss on them with its gradient.

A semantic scene renders class (or codebook) scores per pixel and trains them against a 2-D teacher of which each view keeps
the k largest logits of every pixel. ``top`` makes those targets, ``loss`` is the loss alone (validation) and ``train`` the loss
with the gradient of the student's logits. The row counts are pixels of this repository's image sizes, or a batch of rows; the
class counts run from a handful of labels over codebooks to vocabularies of open labels.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
MOST = 520_000_000  # logits of the largest case


def _case(name, op, rows, classes, k, dtype, temperature=1.0, rest=False, weights=False, ragged=False, pad=0):
    return {"name": name, "op": op, "rows": rows, "classes": classes, "k": k, "dtype": dtype, "temperature": temperature,
            "rest": rest, "weights": weights, "ragged": ragged, "pad": pad}


def listed():
    return [
        # a handful of picked pixels with few labels: the call's latency
        _case("top_tiny", "top", 5, 19, 3, "fp32"),
        # one pixel queried against a large open vocabulary
        _case("top_one_long_row", "top", 1, 100_003, 50, "bf16"),
        # a 256 x 256 view of a teacher with an odd number of labels
        _case("top_view_256", "top", 256 * 256, 133, 5, "fp32", temperature=2.0),
        # a 1080p view of a teacher's label scores, stored as k of them
        _case("top_view_1080p", "top", 1080 * 1920, 150, 8, "fp16"),
        # an 800 x 800 view scored against a codebook of features
        _case("top_codebook_800", "top", 800 * 800, 512, 16, "bf16"),
        # a batch of rows over a large vocabulary, many kept
        _case("top_vocabulary", "top", 2048, 128_000, 64, "fp32"),
        # the validation loss of an 840 x 1297 view
        _case("loss_view_840", "loss", 840 * 1297, 101, 10, "fp16", rest=True),
        # a few rows over an odd vocabulary whose logits are a slice of a padded product
        _case("loss_few_long_rows", "loss", 33, 65_537, 20, "fp32", temperature=1.5, pad=127),
        # seven rows of three labels: the training call's latency
        _case("train_tiny", "train", 7, 3, 2, "fp32"),
        # a 1080p training view with a pixel mask and confidences, the teacher's remaining mass as one class
        _case("train_view_1080p", "train", 1080 * 1920, 150, 8, "fp32", rest=True, weights=True, ragged=True),
        # an 800 x 800 view against a codebook with one code for "none"
        _case("train_codebook_800", "train", 800 * 800, 513, 16, "bf16", temperature=2.0),
        # a batch of rows over a large vocabulary
        _case("train_vocabulary", "train", 4000, 128_000, 32, "bf16", temperature=2.0, rest=True),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["top", "loss", "train"])
    classes = _spread(rng, 2, 140_000)
    rows = _spread(rng, 1, min(1080 * 1920, (260_000_000 if op == "top" else MOST) // (classes + 64)))
    k = min(classes, _spread(rng, 1, 64))
    distils = op != "top"
    return _case("", op, rows, classes, k, rng.choice(["fp32", "bf16", "fp16"]), temperature=rng.choice([1.0, 1.0, 0.5, 2.0, 3.0]),
                 rest=distils and rng.random() < 0.5, weights=distils and rng.random() < 0.4, ragged=distils and rng.random() < 0.4,
                 pad=rng.choice([0, 0, 0, 1, 8, 61]))


def _logits(g, rows, classes, pad, dtype):
    """Scores with a spread of 2.5 and, in each row, a few classes that stand out."""
    wide = torch.empty(rows, classes + pad, device="cuda", dtype=dtype)
    step = max(1, 100_000_000 // (classes + pad))
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = torch.randn(n, classes + pad, device="cuda", generator=g) * 2.5
        for _ in range(3):
            at = torch.randint(0, classes, (n, 1), device="cuda", generator=g)
            x.scatter_add_(1, at, torch.rand(n, 1, device="cuda", generator=g) * 9.0)
        wide[r : r + n] = x.to(dtype)
    return wide


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, classes, k, dtype = case["rows"], case["classes"], case["k"], DTYPES[case["dtype"]]
    state = {"op": case["op"], "k": k, "temperature": case["temperature"], "lse": None, "weights": None}
    teacher = _logits(g, rows, classes, case["pad"], dtype)
    if case["op"] == "top":
        return {**state, "logits": teacher[:, :classes]}
    student = _logits(g, rows, classes, case["pad"], dtype)
    step = max(1, 100_000_000 // classes)
    values = torch.empty(rows, k, device="cuda", dtype=dtype)
    ids = torch.empty(rows, k, device="cuda", dtype=torch.int32)
    lse = torch.empty(rows, device="cuda")
    for r in range(0, rows, step):  # the student has learned a part of what the teacher says
        t = teacher[r : r + step, :classes].float()
        top = t.topk(k, dim=1)
        values[r : r + step], ids[r : r + step] = top.values.to(dtype), top.indices.to(torch.int32)
        lse[r : r + step] = torch.logsumexp(t / case["temperature"], 1)
        s = student[r : r + step, :classes]
        s.copy_((0.5 * s.float() + 0.6 * t).to(dtype))
    if case["ragged"]:  # pixels where fewer classes were kept, some with none
        kept = torch.randint(0, k + 1, (rows, 1), device="cuda", generator=g)
        ids[torch.arange(k, device="cuda") >= kept] = -1
    if case["weights"]:  # three pixels in ten are masked, the others have a confidence
        w = torch.rand(rows, device="cuda", generator=g)
        state["weights"] = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.3, torch.zeros_like(w), w)
    if case["op"] == "train":
        student = student.requires_grad_()
    return {**state, "logits": student[:, :classes], "values": values, "ids": ids, "lse": lse if case["rest"] else None}


def _own(state):
    import splax_b200 as sx

    if state["op"] == "top":
        return list(sx.top_logits(state["logits"], state["k"], temperature=state["temperature"]))
    args = (state["logits"], state["values"], state["ids"], state["lse"])
    more = {"temperature": state["temperature"], "weights": state["weights"]}
    if state["op"] == "loss":
        with torch.no_grad():
            return [sx.distill_loss(*args, **more)]
    loss = sx.distill_loss(*args, **more)
    return [loss.detach(), torch.autograd.grad(loss, state["logits"])[0]]


def _top(state):
    z = state["logits"]
    values, ids = torch.sort(z, dim=1, descending=True, stable=True)
    s = z.float() / state["temperature"]
    m = s.amax(1, keepdim=True)
    lse = (s - m).exp().sum(1).log() + m[:, 0]
    return [values[:, : state["k"]].contiguous(), ids[:, : state["k"]].to(torch.int32), lse]


def _log_sum_exp(x):
    """Over the last axis, with -inf for a row of nothing but -inf."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    return (x - m).exp().sum(-1).log() + m[..., 0]


def _distil(state):
    """The formulas as they stand: entries and the other classes apart, one array operation after another."""
    with torch.no_grad():
        z, ids, tau = state["logits"], state["ids"], state["temperature"]
        rows, classes = z.shape
        s = z.float() / tau
        a = state["values"].float() / tau
        valid = (ids >= 0) & (ids < classes)
        a = torch.where(valid, a, torch.full_like(a, -math.inf))
        at = torch.where(valid, ids, torch.zeros_like(ids)).long()
        norm = _log_sum_exp(a) if state["lse"] is None else state["lse"]
        in_use = norm > -math.inf
        if state["weights"] is not None:
            in_use = in_use & (state["weights"] != 0)
        log_p = a - torch.where(norm > -math.inf, norm, torch.zeros_like(norm))[:, None]
        p = log_p.exp()
        mass = p.sum(1)
        named = torch.zeros(rows, classes, device=z.device, dtype=torch.int32)
        named.scatter_add_(1, at, valid.to(torch.int32))
        named = named > 0
        lse = _log_sum_exp(s)
        others = _log_sum_exp(torch.where(named, torch.full_like(s, -math.inf), s))
        some = others > -math.inf
        if state["lse"] is None:
            rho = torch.zeros_like(mass)
        else:
            rho = torch.where(some, (1 - mass).clamp_min(0), torch.zeros_like(mass))
        each = p * (log_p - s.gather(1, at) + lse[:, None])
        row = torch.where(p > 0, each, torch.zeros_like(p)).sum(1)
        rest = rho * (rho.log() - others + lse)
        row = row + torch.where(rho > 0, rest, torch.zeros_like(rest))
        w = torch.ones_like(row) if state["weights"] is None else state["weights"]
        row = torch.where(in_use, w * row, torch.zeros_like(row))
        loss = (row.double().sum() * (tau * tau / rows)).float()
        if state["op"] == "loss":
            return [loss]
        others = torch.where(some, others, torch.zeros_like(others))
        other = ((mass + rho) * (others - lse).exp() - rho)[:, None] * (s - others[:, None]).exp()
        grad = torch.where(named, (mass + rho)[:, None] * (s - lse[:, None]).exp(), other)
        grad.scatter_add_(1, at, torch.where(valid, -p, torch.zeros_like(p)))
        grad = grad * (w * tau / rows)[:, None]
        grad = torch.where(in_use[:, None], grad, torch.zeros_like(grad))
        return [loss, grad.to(z.dtype)]


def run(state):
    if own:
        return _own(state)
    return _top(state) if state["op"] == "top" else _distil(state)


def work(case):
    rows, classes, k = case["rows"], case["classes"], case["k"]
    size = 4 if case["dtype"] == "fp32" else 2
    logits, kept = rows * classes * size, rows * k * (size + 4)
    if case["op"] == "top":
        return {"bytes": logits + kept + 4 * rows, "flops": 4 * rows * classes}
    extra = 4 * rows * (int(case["rest"]) + int(case["weights"]))
    if case["op"] == "loss":
        return {"bytes": logits + kept + extra + 4, "flops": 4 * rows * classes}
    return {"bytes": 2 * logits + kept + extra + 4, "flops": 6 * rows * classes}


def exact(case, seed):
    """From the definitions in 64 bits: the k largest by taking the first maximum k times; the loss as the divergence between two
    distributions over the named classes and, where it counts, one class for all others; its gradient by differentiating that."""
    state = prepare(case, seed)
    z, k, tau = state["logits"].detach(), case["k"], case["temperature"]
    rows, classes = z.shape
    step = max(1, 60_000_000 // classes)
    out = []
    for r in range(0, rows, step):
        x = z[r : r + step].double()
        if case["op"] == "top":
            lse = torch.logsumexp(x / tau, 1)
            values, ids = [], []
            for _ in range(k):
                best, at = x.max(1, keepdim=True)
                # the lowest of the classes that hold the maximum
                place = torch.arange(classes, device=x.device)
                at = torch.where(x == best, place, classes).amin(1, keepdim=True)
                values.append(best)
                ids.append(at)
                x.scatter_(1, at, -math.inf)
            out.append([torch.cat(values, 1), torch.cat(ids, 1).to(torch.int32), lse])
            continue
        with torch.enable_grad():
            x = x.requires_grad_(case["op"] == "train")
            log_q = torch.log_softmax(x / tau, 1)
            v, ids = state["values"][r : r + step].double() / tau, state["ids"][r : r + step].long()
            valid = ids >= 0
            ids = ids.clamp_min(0)
            # the teacher's distribution over the named classes, zero elsewhere
            t = torch.where(valid, v, -math.inf)
            if state["lse"] is None:
                live = valid.any(1)
                p = torch.where(valid, torch.softmax(torch.where(live[:, None], t, 0.0), 1), 0.0)
            else:
                live = torch.ones_like(valid[:, 0])
                p = torch.exp(t - state["lse"][r : r + step, None].double())
            positive = torch.where(p > 0, p, 1.0)
            terms = torch.where(p > 0, p * (positive.log() - log_q.gather(1, ids)), 0.0)
            row = terms.sum(1)
            if state["lse"] is not None:
                outside = torch.ones_like(x, dtype=torch.bool)
                outside.scatter_(1, ids, torch.zeros_like(valid))
                first_free = ~((ids == 0) & valid).any(1)  # empty entries were put at class 0
                outside[:, 0] = first_free
                rest = (1.0 - p.sum(1)).clamp_min(0.0)
                some = outside.any(1) & (rest > 0)
                log_rest = torch.logsumexp(torch.where(outside | ~some[:, None], log_q, -math.inf), 1)
                row = row + torch.where(some, rest * (torch.where(some, rest, 1.0).log() - log_rest), 0.0)
            w = torch.ones_like(row) if state["weights"] is None else state["weights"][r : r + step].double()
            loss = (torch.where(live, row, 0.0) * w).sum() * (tau * tau / rows)
            grad = torch.autograd.grad(loss, x)[0] if case["op"] == "train" else None
        out.append([loss.detach(), grad])
        del x, log_q
    if case["op"] == "top":
        return [torch.cat(part) for part in zip(*out)]
    loss = torch.stack([o[0] for o in out]).sum()
    return [loss] if case["op"] == "loss" else [loss, torch.cat([o[1] for o in out])]
