"""Cases of the 8-bit linear layer, the teacher's top logits and the distillation loss.

``listed()`` names the cases, ``draw()`` gives further ones of the same ranges, ``prepare()`` makes
a case's inputs from a seed, ``run()`` makes one pass (the plain torch form, or the framework's
calls where ``own`` is set), ``exact()`` gives the outputs in 64 bits from the definitions, and
``work()`` the bytes and operations of a pass.

The definitions, for a row x of K values, a weight row w_n, and logits z of V classes:

* int8 linear: s = max(max|x| / 127, 2^-126) in fp32, q = x / s rounded half to even, and
  y_n = s * s_n * sum_k q_k w_nk (+ b_n), then max(., 0) where a ReLU is asked for.
* top logits: the k largest of z in falling order (equal ones: lowest index first), their indices,
  and log sum_i exp(z_i / T).
* distillation: p_j = softmax over the named teacher logits t_j / T, or exp(t_j / T - lse) where the
  teacher's normaliser is given; q = softmax(z / T);
  KD = sum_j p_j (log p_j - log q_{c_j}) + r (log r - log q_rest), r = 1 - sum_j p_j and q_rest the
  sum of q outside the named classes (the last term only with the normaliser);
  loss = (1 - h) T^2 KD + h (-log softmax(z)_y), averaged over the rows whose y is a class.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
TINY = 2.0 ** -126


# ----------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a square layer: a pass is the weight's bytes, and the calls' latency
        _linear("int8 one token", 1, 4096, 4096, "bf16"),
        # a served batch of single tokens through a wide layer with a bias
        _linear("int8 served batch", 24, 8192, 8192, "bf16", bias=True),
        # ResNet-50's classifier (2048 -> 1000) at batch 256 in the fp32 of the layer path
        _linear("int8 classifier", 256, 2048, 1000, "fp32", bias=True),
        # two layers on one quantised input, MLP-like with a ReLU; no size is a multiple of a tile
        _linear("int8 shared input", 1777, 5000, 5000, "fp16", bias=True, relu=True, products=2),
        # the tokens of a long batch: the matrix units' rate
        _linear("int8 many tokens", 8192, 8192, 8192, "bf16"),
        # a ResNet-50 teacher's answers for a batch of 256 images
        _top("top of a classifier", 256, 1000, 10, "fp32", 2.0),
        # one token's answer over a large vocabulary
        _top("top of one token", 1, 131072, 50, "fp16", 1.0),
        # the teacher's answers for a batch of tokens
        _top("top of many tokens", 4096, 131072, 64, "bf16", 1.0),
        # an image classifier learns from a teacher and from its labels
        _distill("distill a classifier", 256, 1000, 10, "fp32", 4.0, hard=0.1),
        # ragged sizes: odd vocabulary, padded tokens, some rows that the teacher says nothing about
        _distill("distill ragged", 1023, 50001, 33, "fp16", 2.0, hard=0.5, padded=0.25),
        # a validation pass: each token's loss, no gradient
        _distill("distill evaluation", 2048, 65536, 32, "bf16", 1.0, tail=True, grad=False, per_token=True),
        # a training step's loss and gradient over a large vocabulary
        _distill("distill many tokens", 4096, 131072, 64, "bf16", 1.0, tail=True),
    ]


def _linear(name, tokens, inner, outer, dtype, bias=False, relu=False, products=1):
    return {"name": name, "op": "linear", "tokens": tokens, "inner": inner, "outer": outer, "dtype": dtype,
            "bias": bias, "relu": relu, "products": products}


def _top(name, rows, classes, k, dtype, temperature):
    return {"name": name, "op": "top", "rows": rows, "classes": classes, "k": k, "dtype": dtype,
            "temperature": temperature}


def _distill(name, rows, classes, k, dtype, temperature, tail=False, hard=0.0, padded=0.0, grad=True, per_token=False):
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "k": k, "dtype": dtype,
            "temperature": temperature, "tail": tail, "hard": hard, "padded": padded, "grad": grad,
            "per_token": per_token}


def _spread(rng, low, high):
    """A whole number of [low, high], evenly spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "top", "distill"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op == "linear":
        products = rng.choice([1, 1, 2])
        inner, outer = _spread(rng, 64, 8192), _spread(rng, 10, 8192)
        if rng.random() < 0.5:  # half of the layers have rows of whole 16-byte pieces
            inner, outer = (inner + 15) // 16 * 16, (outer + 15) // 16 * 16
        c = _linear("", _spread(rng, 1, 8192 // products), inner, outer, dtype, rng.random() < 0.5, rng.random() < 0.3,
                    products)
    else:
        classes = _spread(rng, 10, 131072)
        rows = _spread(rng, 1, min(4096, (1 << 30) // (classes * SIZE[dtype])))
        k = _spread(rng, 1, min(classes, 128))
        temperature = rng.choice([1.0, 1.0, 2.0, 4.0, 0.7])
        if op == "top":
            c = _top("", rows, classes, k, dtype, temperature)
        else:
            c = _distill("", rows, classes, k, dtype, temperature, rng.random() < 0.5, rng.choice([0.0, 0.3, 0.5]),
                         rng.choice([0.0, 0.0, 0.2]), rng.random() < 0.8, rng.random() < 0.3)
    del c["name"]
    return c


def work(case):
    if case["op"] == "linear":
        m, k, n, p = case["tokens"], case["inner"], case["outer"], case["products"]
        b = SIZE[case["dtype"]]
        return {"bytes": m * k * b + p * (n * k + 4 * n + (4 * n if case["bias"] else 0) + m * n * b),
                "flops": 2 * p * m * k * n}
    r, v, k, b = case["rows"], case["classes"], case["k"], SIZE[case["dtype"]]
    if case["op"] == "top":
        return {"bytes": r * v * b + r * (k * (b + 4) + 4), "flops": 4 * r * v}
    named = r * (k * (b + 4) + (4 if case["tail"] else 0) + 8) + 4 * (r if case["per_token"] else 1)
    return {"bytes": r * v * b * (2 if case["grad"] else 1) + named, "flops": (8 if case["grad"] else 4) * r * v}


# ---------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        # activations: a few channels are much larger than the rest
        x = normal(m, k) * torch.exp(0.6 * normal(k))
        layers = []
        for _ in range(case["products"]):
            w = normal(n, k) / math.sqrt(k)
            scale = w.abs().amax(1) / 127
            layers.append(((w / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale,
                           normal(n) if case["bias"] else None))
        return {"case": case, "x": x.to(dtype), "layers": layers}
    r, v, k = case["rows"], case["classes"], case["k"]
    # a teacher's logits: most classes far below a few likely ones
    teacher = 2.5 * normal(r, v)
    teacher.scatter_add_(1, torch.randint(v, (r, 4), generator=g, device="cuda"), 6 + 2 * normal(r, 4))
    if case["op"] == "top":
        return {"case": case, "logits": teacher.to(dtype)}
    t = case["temperature"]
    answer = teacher.to(dtype)
    values, index = teacher.topk(k, dim=1)
    values = answer.gather(1, index)
    lse = torch.logsumexp(answer.float() / t, 1) if case["tail"] else None
    logits = teacher.mul_(0.6).add_(normal(r, v)).to(dtype)  # a student that has learned a part of it
    target = None
    if case["hard"] > 0 or case["padded"] > 0:
        target = torch.randint(v, (r,), generator=g, device="cuda")
        target = torch.where(torch.rand(r, generator=g, device="cuda") < 0.5, index[:, 0], target)
        target[torch.rand(r, generator=g, device="cuda") < case["padded"]] = -100
    index = index.to(torch.int32)
    if case["padded"] > 0:  # shorter lists, and rows with none
        length = torch.randint(0, k + 1, (r, 1), generator=g, device="cuda")
        index[torch.arange(k, device="cuda") >= length] = -1
    weight = torch.rand(r, generator=g, device="cuda") if case["per_token"] else None
    return {"case": case, "logits": logits.requires_grad_(case["grad"]), "values": values, "index": index,
            "lse": lse, "target": target, "weight": weight}


# ------------------------------------------------------------------------------------------ runs
def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "linear":
        return _plain_linear(state, case)
    if case["op"] == "top":
        return _plain_top(state, case)
    return _plain_distill(state, case)


def _own(state, case):
    from mxddp import ops

    if case["op"] == "linear":
        x = state["x"]
        if case["products"] == 1:
            (w, scale, bias), = state["layers"]
            return ops.linear_int8(x, w, scale, bias, relu=case["relu"])
        q, s = ops.quantize_rows(x)
        return [ops.linear_int8(q, w, scale, bias, relu=case["relu"], x_scale=s, out_dtype=x.dtype)
                for w, scale, bias in state["layers"]]
    if case["op"] == "top":
        return list(ops.top_logits(state["logits"], case["k"], temperature=case["temperature"]))
    loss = ops.distill_loss(state["logits"], state["values"], state["index"], target=state["target"],
                            top_lse=state["lse"], temperature=case["temperature"], hard_weight=case["hard"],
                            reduction="none" if case["per_token"] else "mean")
    if not case["grad"]:
        return loss
    grad, = torch.autograd.grad(loss, state["logits"], state["weight"])
    return [loss, grad]


def _plain_linear(state, case):
    x = state["x"]
    top = x.abs().amax(1, keepdim=True).double()
    s = (top / 127).float().clamp_min(TINY)
    # in 64 bits: a quotient next to a half has to round as the exact one does
    q = (x.double() / s.double()).round().float()
    out = []
    for w, scale, bias in state["layers"]:
        y = (q @ w.float().t()) * s * scale
        if bias is not None:
            y = y + bias
        if case["relu"]:
            y = y.clamp_min(0)
        out.append(y.to(x.dtype))
    return out[0] if len(out) == 1 else out


def _plain_top(state, case):
    z, k = state["logits"], case["k"]
    values, index = torch.sort(z, dim=1, descending=True, stable=True)
    scaled = z.float() / case["temperature"]
    top = scaled.amax(1, keepdim=True)
    lse = (scaled - top).exp().sum(1).log() + top[:, 0]
    return [values[:, :k].contiguous(), index[:, :k].to(torch.int32), lse]


def _log_total(z, t):
    """log sum exp(z / t) of each row, the sum in 64 bits; -inf for a row of -inf."""
    most = z.amax(1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    return ((z - most) / t).exp().sum(1, keepdim=True, dtype=torch.float64).log() + most.double() / t


def _plain_distill(state, case):
    logits, target = state["logits"], state["target"]
    t, h = case["temperature"], case["hard"]
    z = logits.detach().float()
    r, v = z.shape
    used = state["index"] >= 0
    at = torch.where(used, state["index"], v).long()  # unused entries point behind the last class
    # the teacher's probabilities, in 64 bits as all that is summed over a row: what they leave to
    # the other classes, and the loss itself, are small differences
    scaled = torch.where(used, state["values"].double() / t, -math.inf)
    norm = state["lse"][:, None].double() if state["lse"] is not None else _log_total(scaled, 1.0)
    logp = scaled - norm
    p = torch.where(used, logp.exp(), 0.0)
    # the student's, at the temperature
    logz = _log_total(z, t)
    logq = torch.where(used, z.gather(1, at.clamp_max(v - 1)).double() / t - logz, 0.0)
    kd = torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    grad = (z / t - logz.float()).exp()
    if state["lse"] is not None:
        rest = (1 - p.sum(1, keepdim=True)).clamp_min(0)
        inside = torch.zeros(r, v + 1, dtype=torch.bool, device=z.device).scatter_(1, at, True)[:, :v]
        log_out = _log_total(torch.where(inside, -math.inf, z), t)
        has = (rest > 0) & (log_out > -math.inf)
        kd = kd + torch.where(has, rest * (rest.log() - (log_out - logz)), 0.0)[:, 0]
        share = torch.where(has, rest.log() - log_out, -math.inf).float()
        grad = grad - torch.where(inside, 0.0, (z / t + share).exp())
    else:
        # a row that the teacher says nothing about has no such term
        grad = grad * used.any(1, keepdim=True)
    grad = torch.cat([grad, grad[:, :1]], 1).scatter_add_(1, at, -p.float())[:, :v] * ((1 - h) * t)
    loss = (1 - h) * t * t * kd
    counted = used.any(1)
    if target is not None:
        counted = (target >= 0) & (target < v)
        if h > 0:
            y = torch.where(counted, target, 0)[:, None]
            logz = _log_total(z, 1.0)
            loss = loss + h * (logz - z.gather(1, y))[:, 0]
            grad = grad + h * (z - logz.float()).exp()
            grad.scatter_add_(1, y, torch.full_like(y, -h, dtype=torch.float32))
    loss = torch.where(counted, loss, 0.0)
    if case["per_token"]:
        share = torch.where(counted, state["weight"], 0.0)
    else:
        share = counted.float() / counted.sum().clamp_min(1)
        loss = loss.sum() / counted.sum().clamp_min(1)
    loss = loss.float()
    if not case["grad"]:
        return loss
    return [loss, torch.where(counted[:, None], grad * share[:, None], 0.0).to(logits.dtype)]


# ---------------------------------------------------------------------------------------- exact
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(state, case)
    rows = max(1, (1 << 26) // case["classes"])
    if case["op"] == "top":
        parts = [_exact_top(z, case) for z in state["logits"].split(rows)]
        return [torch.cat(p) for p in zip(*parts)]
    return _exact_distill(state, case, rows)


def _exact_linear(state, case):
    x = state["x"].double()
    s = torch.maximum(x.abs().max(1).values / 127, torch.tensor(TINY, device="cuda", dtype=torch.float64))
    s = s.float().double()
    d = x / s[:, None]
    low = d.floor()
    up = (d - low > 0.5) | ((d - low == 0.5) & (low.remainder(2) == 1))
    q = low + up.double()
    out = []
    for w, scale, bias in state["layers"]:
        y = torch.mm(q, w.double().t().contiguous())
        y = y * torch.outer(s, scale.double())
        y = y if bias is None else y + bias.double()
        out.append(y.relu() if case["relu"] else y)
    return out[0] if len(out) == 1 else out


def _exact_top(z, case):
    z = z.double()
    order = torch.argsort(-z, dim=1, stable=True)[:, :case["k"]]
    return z.gather(1, order), order.to(torch.int32), torch.logsumexp(z / case["temperature"], 1)


def _exact_distill(state, case, rows):
    """Row by row from the definition: log-probabilities over (named classes, all others), the
    gradient by differentiating the definition's sum."""
    n = case["rows"]
    target = state["target"]
    ok = (state["index"] >= 0).any(1) if target is None else (target >= 0) & (target < case["classes"])
    count = max(1, int(ok.sum()))
    losses, grads = [], []
    for i in range(0, n, rows):
        j = slice(i, i + rows)
        z = state["logits"].detach()[j].double().requires_grad_(case["grad"])
        row = _exact_rows(z, state["values"][j].double(), state["index"][j].long(),
                          None if target is None else target[j], None if state["lse"] is None else state["lse"][j].double(),
                          case)
        row = torch.where(ok[j], row, torch.zeros_like(row))
        losses.append(row.detach())
        if case["grad"]:
            share = state["weight"][j].double() if case["per_token"] else torch.full_like(row, 1 / count)
            g, = torch.autograd.grad(row, z, share)
            grads.append(torch.where(ok[j, None], g, torch.zeros_like(g)).to(torch.float64))
    loss = torch.cat(losses)
    loss = loss if case["per_token"] else loss.sum() / count
    return [loss, torch.cat(grads)] if case["grad"] else loss


def _exact_rows(z, values, index, target, lse, case):
    t, h = case["temperature"], case["hard"]
    used = index >= 0
    pad = torch.cat([z / t, torch.zeros_like(z[:, :1])], 1)  # one more column that unused entries point to
    at = torch.where(used, index, z.shape[1])
    total = torch.logsumexp(pad[:, :-1], 1, keepdim=True)
    u = values / t
    if lse is None:
        floor = torch.where(used, u, torch.full_like(u, -math.inf))
        norm = torch.logsumexp(floor, 1, keepdim=True)
        norm = torch.where(norm == -math.inf, torch.zeros_like(norm), norm)
    else:
        norm = lse[:, None]
    p = torch.where(used, (u - norm).exp(), torch.zeros_like(u))
    kd = (p * torch.where(used, u - norm - (pad.gather(1, at) - total), torch.zeros_like(u))).sum(1)
    if lse is not None:
        inside = torch.zeros_like(pad, dtype=torch.bool).scatter(1, at, True)[:, :-1]
        rest = (1 - p.sum(1)).clamp_min(0)
        has = (rest > 0) & ~inside.all(1)
        safe = torch.where(has, rest, torch.ones_like(rest))
        other = torch.logsumexp(torch.where(inside & has[:, None], torch.full_like(z, -math.inf), pad[:, :-1]), 1)
        kd = kd + torch.where(has, safe * (safe.log() - (other - total[:, 0])), torch.zeros_like(kd))
    loss = (1 - h) * t * t * kd
    if h > 0:
        y = torch.where((target >= 0) & (target < z.shape[1]), target, 0)[:, None]
        loss = loss + h * (torch.logsumexp(z, 1) - z.gather(1, y)[:, 0])
    return loss
