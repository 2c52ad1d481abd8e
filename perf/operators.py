"""Measured cases of the losses of a large-vocabulary head: the cross entropy of the last layer's product, which keeps no
logits, and the distillation from a teacher's largest logits; each forward and with its gradient.

`own` false: the plain form, in elementary torch operations.  `own` true: the framework's operators."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # scoring one token against a vocabulary: latency and one pass over W
        {"name": "ce token bf16", "op": "ce", "n": 1, "d": 1024, "v": 32000, "dtype": "bfloat16", "grad": False, "ignored": 0.0, "weighted": False},
        # a small classifier trained in the framework's own type, no size a power of two
        {"name": "ce small f32", "op": "ce", "n": 200, "d": 520, "v": 1003, "dtype": "float32", "grad": True, "ignored": 0.0, "weighted": False},
        # perplexity of a batch, no gradient
        {"name": "ce eval f16", "op": "ce", "n": 2048, "d": 1024, "v": 32768, "dtype": "float16", "grad": False, "ignored": 0.0, "weighted": False},
        # an ordinary training step
        {"name": "ce train bf16", "op": "ce", "n": 4096, "d": 2048, "v": 32000, "dtype": "bfloat16", "grad": True, "ignored": 0.0, "weighted": False},
        # a padded batch: a third of the rows carries no target; ragged sizes, one weight a token
        {"name": "ce padded bf16", "op": "ce", "n": 3001, "d": 1000, "v": 49999, "dtype": "bfloat16", "grad": True, "ignored": 0.33, "weighted": True},
        # the framework's own type at a training size
        {"name": "ce train f32", "op": "ce", "n": 1024, "d": 1024, "v": 16384, "dtype": "float32", "grad": True, "ignored": 0.0, "weighted": False},
        # rows that start at odd addresses
        {"name": "ce odd f16", "op": "ce", "n": 777, "d": 1001, "v": 30011, "dtype": "float16", "grad": True, "ignored": 0.1, "weighted": True},
        # the largest: a long batch on a large vocabulary
        {"name": "ce large bf16", "op": "ce", "n": 8192, "d": 4096, "v": 131072, "dtype": "bfloat16", "grad": True, "ignored": 0.0, "weighted": False},
        # one token's distillation loss
        {"name": "kd token f32", "op": "kd", "n": 1, "v": 32000, "k": 8, "dtype": "float32", "grad": False, "ragged": False, "temperature": 1.0},
        # validation on the teacher's list
        {"name": "kd eval f16", "op": "kd", "n": 2048, "v": 32000, "k": 20, "dtype": "float16", "grad": False, "ragged": False, "temperature": 2.0},
        # lists of different lengths, an odd vocabulary
        {"name": "kd ragged f32", "op": "kd", "n": 512, "v": 50021, "k": 100, "dtype": "float32", "grad": True, "ragged": True, "temperature": 2.0},
        # a training step on a large vocabulary
        {"name": "kd train bf16", "op": "kd", "n": 4096, "v": 131072, "k": 64, "dtype": "bfloat16", "grad": True, "ragged": False, "temperature": 1.0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(sorted(TYPES))
    grad = rng.random() < 0.6
    if rng.random() < 0.6:
        # f32 has 512 times less work at most: its plain products are as slow, and users of it have smaller heads
        most = 8192 * 4096 * 131072 // (512 if dtype == "float32" else 8)
        d, v = _spread(rng, 64, 4096), _spread(rng, 500, 131072)
        if rng.random() < 0.5:
            d = -(-d // 8) * 8
        n = _spread(rng, 1, max(1, min(8192, most // (d * v))))
        return {"op": "ce", "n": n, "d": d, "v": v, "dtype": dtype, "grad": grad, "ignored": rng.choice([0.0, 0.0, 0.25]), "weighted": rng.random() < 0.3}
    v = _spread(rng, 500, 131072)
    n = _spread(rng, 1, min(8192, 4096 * 131072 // (2 * v)))
    return {"op": "kd", "n": n, "v": v, "k": _spread(rng, 1, 128), "dtype": dtype, "grad": grad, "ragged": rng.random() < 0.3,
            "temperature": rng.choice([1.0, 1.0, 2.0, 4.0])}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, n, v = TYPES[case["dtype"]], case["n"], case["v"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "ce":
        # hidden states after a norm, and a head whose logits have a deviation of 1.5
        x = normal(n, case["d"]).to(dtype)
        w = (normal(v, case["d"]) * (1.5 / math.sqrt(case["d"]))).to(dtype)
        target = torch.randint(0, v, (n,), generator=gen, device=dev)
        ignored = torch.rand(n, generator=gen, device=dev) < case["ignored"]
        target = torch.where(ignored, torch.full_like(target, -100), target)
        g = torch.full((n,), 1.0, device=dev) / (~ignored).sum().clamp(min=1)
        if case["weighted"]:
            g = g * torch.rand(n, generator=gen, device=dev)
        if case["grad"]:
            x.requires_grad_()
            w.requires_grad_()
        return {"case": case, "x": x, "w": w, "target": target, "g": g}
    logits = (normal(n, v) * 2.5).to(dtype)
    k = min(case["k"], v)
    # a row's entries are distinct places; the teacher's logits come in falling order
    places = torch.randperm(v, generator=gen, device=dev)[:k]
    indices = (torch.randint(0, v, (n, 1), generator=gen, device=dev) + places) % v
    teacher = (normal(n, k) * 3).sort(dim=1, descending=True).values.to(dtype)
    if case["ragged"]:
        lengths = torch.randint(0, k + 1, (n, 1), generator=gen, device=dev)
        indices = torch.where(torch.arange(k, device=dev) < lengths, indices, torch.full_like(indices, -1))
    g = torch.full((n,), 1.0 / n, device=dev)
    if case["grad"]:
        logits.requires_grad_()
    return {"case": case, "logits": logits, "indices": indices, "teacher": teacher, "g": g}


def _plain_ce(state):
    with torch.no_grad():
        case, target = state["case"], state["target"]
        x, w = state["x"].float(), state["w"].float()
        z = x @ w.t()
        kept = target != -100
        at = torch.where(kept, target, torch.zeros_like(target))[:, None]
        top = z.amax(dim=1, keepdim=True)
        p = torch.exp(z - top)
        total = p.sum(dim=1, keepdim=True)
        loss = torch.where(kept, (top - z.gather(1, at) + torch.log(total))[:, 0], torch.zeros_like(total[:, 0]))
        if not case["grad"]:
            return {"loss": loss}
        del z
        p = p.div_(total)
        p.scatter_add_(1, at, torch.full_like(total, -1.0))
        p = p.mul_(torch.where(kept, state["g"], torch.zeros_like(state["g"]))[:, None])
        return {"loss": loss, "dx": (p @ w).to(state["x"].dtype), "dw": (p.t() @ x).to(state["w"].dtype)}


def _plain_kd(state):
    with torch.no_grad():
        case, indices, t = state["case"], state["indices"], state["case"]["temperature"]
        z = state["logits"].float() / t
        top = z.amax(dim=1, keepdim=True)
        p = torch.exp(z - top)
        total = p.sum(dim=1, keepdim=True)
        there = indices >= 0
        at = torch.where(there, indices, torch.zeros_like(indices))
        s = torch.where(there, state["teacher"].float() / t, torch.full_like(at, -math.inf, dtype=torch.float32))
        best = s.amax(dim=1, keepdim=True)
        some = best > -math.inf
        s = s - torch.where(some, best, torch.zeros_like(best))
        e = torch.exp(s)
        weight = e.sum(dim=1, keepdim=True)
        weight = torch.where(some, weight, torch.ones_like(weight))
        q = e / weight
        term = q * (s - torch.log(weight) - (z.gather(1, at) - top - torch.log(total)))
        loss = t * t * torch.where(q > 0, term, torch.zeros_like(term)).sum(dim=1)
        if not case["grad"]:
            return {"loss": loss}
        del z
        p = p.div_(total)
        p.scatter_add_(1, at, -q)
        p = p.mul_(torch.where(some, t * state["g"][:, None], torch.zeros_like(best)))
        return {"loss": loss, "dlogits": p.to(state["logits"].dtype)}


def _own_ce(state):
    import tensorcomprehensions_b200 as tc

    loss = tc.linear_cross_entropy(state["x"], state["w"], state["target"], ignore_index=-100)
    if not state["case"]["grad"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (state["x"], state["w"]), state["g"])
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def _own_kd(state):
    import tensorcomprehensions_b200 as tc

    loss = tc.topk_distillation(state["logits"], state["indices"], state["teacher"], temperature=state["case"]["temperature"])
    if not state["case"]["grad"]:
        return {"loss": loss}
    (dlogits,) = torch.autograd.grad(loss, (state["logits"],), state["g"])
    return {"loss": loss.detach(), "dlogits": dlogits}


def run(state):
    if state["case"]["op"] == "ce":
        return _own_ce(state) if own else _plain_ce(state)
    return _own_kd(state) if own else _plain_kd(state)


def work(case):
    n, v, size = case["n"], case["v"], TYPES[case["dtype"]].itemsize
    if case["op"] == "ce":
        d = case["d"]
        moved = (n + v) * d * size + 8 * n + 4 * n
        # the gradient's two products; getting the logits back a second time is this form's own cost
        return {"bytes": moved + ((n + v) * d * size + 4 * n if case["grad"] else 0), "flops": 2 * n * d * v * (3 if case["grad"] else 1)}
    k = min(case["k"], v)
    moved = n * v * size + n * k * (8 + size) + 4 * n
    return {"bytes": moved + (n * v * size + 4 * n if case["grad"] else 0), "flops": n * v * (6 if case["grad"] else 4)}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ce":
            return _exact_ce(case, state)
        return _exact_kd(case, state)


def _exact_ce(case, state):
    x, w, target = state["x"].detach().double(), state["w"].detach().double(), state["target"]
    n, v = case["n"], case["v"]
    loss = torch.zeros(n, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    rows = max(1, (1 << 28) // v)
    for a in range(0, n, rows):
        # log p of some rows over the whole vocabulary, by the definition
        logp = torch.log_softmax(x[a:a + rows] @ w.t(), dim=1)
        hot = torch.nonzero(target[a:a + rows] >= 0)[:, 0]
        loss[a + hot] = -logp[hot, target[a + hot]]
        if case["grad"]:
            share = torch.zeros_like(logp)
            share[hot] = torch.exp(logp[hot]) * state["g"].double()[a + hot, None]
            share[hot, target[a + hot]] -= state["g"].double()[a + hot]
            dx[a:a + rows] = share @ w
            dw += share.t() @ x[a:a + rows]
    return {"loss": loss, "dx": dx, "dw": dw} if case["grad"] else {"loss": loss}


def _exact_kd(case, state):
    t, indices = case["temperature"], state["indices"]
    n, v = case["n"], case["v"]
    loss = torch.zeros(n, dtype=torch.float64, device=indices.device)
    grad = torch.zeros(n, v, dtype=torch.float64, device=indices.device) if case["grad"] else None
    rows = max(1, (1 << 28) // v)
    for a in range(0, n, rows):
        logp = torch.log_softmax(state["logits"][a:a + rows].detach().double() / t, dim=1)
        kept = indices[a:a + rows] >= 0
        some = kept.any(dim=1)
        # the teacher's distribution spread over the vocabulary; nothing where a row has no entry
        logq = torch.log_softmax((state["teacher"][a:a + rows].double() / t).masked_fill(~kept, -math.inf), dim=1)
        q = torch.exp(logq).masked_fill(~(kept & some[:, None]), 0.0)
        at = indices[a:a + rows].clamp(min=0)
        gap = (logq - logp.gather(1, at)).masked_fill(q == 0, 0.0)
        loss[a:a + rows] = t * t * (q * gap).sum(dim=1)
        if case["grad"]:
            spread = torch.zeros_like(logp).scatter_add_(1, at, q)
            scale = t * state["g"].double()[a:a + rows, None] * some[:, None]
            grad[a:a + rows] = scale * (torch.exp(logp) - spread)
    return {"loss": loss, "dlogits": grad} if case["grad"] else {"loss": loss}
