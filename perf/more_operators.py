"""The operators that need the top of a row of logits, as timed cases.

Each case is a dict of plain values; "kind" picks one operator:

  sample  logits.sample_logits: a token for every row, drawn with given random numbers after temperature, top-k, top-p
          and min-p, and the logarithm of its probability
  top     distill.top_logits: the k largest logits of every row with their ids, and the row's log-sum-exp: what is kept
          of a teacher, or answered as log-probabilities
  kl      distill.top_kl_loss: the KL of a student from such a record, its gradient, and the product of its second
          derivative with a direction (the Hutchinson probe's)

run() computes them by elementary torch operations where `own` is false, and by the package's calls where it is true.
exact() computes them in float64 from the definitions.

Sizes are those of this repository's models (vocabularies of 32000 and 50257, micro-batches of 2 x 2048 tokens, probes
of 1024) and of a large vocabulary of 131072; batches are those of a few users, of a server and of a rollout.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # four users, the usual settings of a chat: the smallest call, all latency
        {"name": "sample chat", "kind": "sample", "batch": 4, "vocab": 32000, "dtype": "bf16", "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "each": False, "masked": False},
        # a server's batch, every user with settings of their own (some greedy), tokens that a grammar forbids, a
        # sequence that has nothing to say
        {"name": "sample serve f32", "kind": "sample", "batch": 48, "vocab": 50257, "dtype": "f32", "temperature": 1.0,
         "top_k": 200, "top_p": 0.9, "min_p": 0.02, "each": True, "masked": True},
        # answers for a policy to learn from: the whole distribution, with the probability each was drawn with
        {"name": "sample rollout", "kind": "sample", "batch": 1024, "vocab": 32000, "dtype": "bf16",
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "each": False, "masked": False},
        # a nucleus of a large vocabulary
        {"name": "sample nucleus f32", "kind": "sample", "batch": 256, "vocab": 131072, "dtype": "f32",
         "temperature": 0.9, "top_k": 0, "top_p": 0.92, "min_p": 0.0, "each": False, "masked": False},
        # log-probabilities beside the answers of a small batch
        {"name": "top answers", "kind": "top", "rows": 16, "vocab": 32000, "dtype": "bf16", "k": 20,
         "temperature": 1.0},
        # a teacher's micro-batch recorded for distillation
        {"name": "top record", "kind": "top", "rows": 4096, "vocab": 32000, "dtype": "bf16", "k": 64,
         "temperature": 2.0},
        # a long record of a large vocabulary in float32
        {"name": "top long f32", "kind": "top", "rows": 509, "vocab": 131072, "dtype": "f32", "k": 500,
         "temperature": 2.0},
        # evaluation of a student on a short text, top entries alone: the smallest loss
        {"name": "kl evaluate", "kind": "kl", "batch": 1, "seq": 65, "shifted": True, "vocab": 32000, "dtype": "bf16",
         "k": 16, "rest": False, "padded": False, "prompt": 0.0, "temperature": 2.0, "order": "loss"},
        # a training micro-batch, the other tokens' probability as one more outcome
        {"name": "kl train", "kind": "kl", "batch": 2, "seq": 2048, "shifted": False, "vocab": 32000, "dtype": "bf16",
         "k": 64, "rest": True, "padded": False, "prompt": 0.0, "temperature": 2.0, "order": "grad"},
        # GPT-2's odd vocabulary in float32: rows of a shifted view, prompts left out, records of unequal length
        {"name": "kl shifted f32", "kind": "kl", "batch": 2, "seq": 1024, "shifted": True, "vocab": 50257,
         "dtype": "f32", "k": 20, "rest": False, "padded": True, "prompt": 0.3, "temperature": 1.0, "order": "grad"},
        # the Hutchinson probe of 1024 tokens: the gradient's own derivative along a direction
        {"name": "kl probe", "kind": "kl", "batch": 1, "seq": 1024, "shifted": False, "vocab": 32000, "dtype": "bf16",
         "k": 64, "rest": True, "padded": False, "prompt": 0.0, "temperature": 2.0, "order": "hvp"},
        # a large vocabulary with long records of unequal length, prompts left out
        {"name": "kl large", "kind": "kl", "batch": 2, "seq": 1024, "shifted": False, "vocab": 131072, "dtype": "bf16",
         "k": 250, "rest": True, "padded": True, "prompt": 0.2, "temperature": 2.0, "order": "grad"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _vocab(rng):
    return rng.choice([32000, 50257, 131072, _log_int(rng, 300, 140000), _log_int(rng, 20000, 140000)])


def _draw_sample(rng):
    k = rng.choice([0, 1, _log_int(rng, 2, 1000), _log_int(rng, 20, 200), _log_int(rng, 1000, 8000)])
    return {"kind": "sample", "batch": _log_int(rng, 1, 1024), "vocab": _vocab(rng),
            "dtype": rng.choice(["bf16", "f32"]), "temperature": rng.choice([1.0, round(rng.uniform(0.2, 2.0), 2)]),
            "top_k": k, "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
            "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)]), "each": rng.random() < 0.3,
            "masked": rng.random() < 0.4}


def _draw_top(rng):
    v = _vocab(rng)
    return {"kind": "top", "rows": _log_int(rng, 1, 4096), "vocab": v, "dtype": rng.choice(["bf16", "f32"]),
            "k": min(v, rng.choice([1, _log_int(rng, 2, 128), _log_int(rng, 2, 1024)])),
            "temperature": rng.choice([1.0, 2.0])}


def _draw_kl(rng):
    v = _vocab(rng)
    return {"kind": "kl", "batch": rng.choice([1, 2, 4]), "seq": _log_int(rng, 2, 2048),
            "shifted": rng.random() < 0.5, "vocab": v, "dtype": rng.choice(["bf16", "f32"]),
            "k": min(v // 2, rng.choice([1, _log_int(rng, 2, 128), _log_int(rng, 2, 1024)])),
            "rest": rng.random() < 0.5, "padded": rng.random() < 0.5, "prompt": rng.choice([0.0, 0.25, 0.5]),
            "temperature": rng.choice([1.0, 2.0, 4.0]), "order": rng.choice(["loss", "grad", "grad", "hvp"])}


def draw(rng):
    kind, make = rng.choices([("sample", _draw_sample), ("top", _draw_top), ("kl", _draw_kl)], [35, 25, 40])[0]
    most = {}  # the largest listed case of the kind bounds the drawn ones, in bytes and in operations
    for c in listed():
        if c["kind"] == kind:
            for k, v in work(c).items():
                most[k] = max(most.get(k, 0), v)
    while True:
        case = make(rng)
        if all(v <= most[k] for k, v in work(case).items()):
            return case


# ---------------------------------------------------------------------------
# sizes that follow from a case
# ---------------------------------------------------------------------------
def _tokens(case):
    """kl: tokens of a sequence that have a target (a shifted view leaves out the last)."""
    return case["seq"] - 1 if case["shifted"] else case["seq"]


def _prompt(case):
    return int(_tokens(case) * case["prompt"])


def work(case):
    size = DT[case["dtype"]].itemsize
    if case["kind"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * size + case["batch"] * (4 + 8 + 4 + 16 * case["each"]), "flops": 4 * n}
    if case["kind"] == "top":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (case["k"] * (size + 4) + 4), "flops": 4 * n}
    rows = case["batch"] * _tokens(case)
    live = case["batch"] * (_tokens(case) - _prompt(case))  # rows of a prompt are not looked at
    V, K = case["vocab"], case["k"]
    lists = live * (K * (size + 4) + 4 * case["rest"]) + 4 * rows * (case["prompt"] > 0) + 4
    # the loss reads the logits; the gradient is written as well, every row of it; so is the second derivative's
    # product, which reads its direction too
    passes = {"loss": live, "grad": live + rows, "hvp": 2 * live + 2 * rows}[case["order"]]
    flops = {"loss": 4, "grad": 8, "hvp": 16}[case["order"]]
    return {"bytes": passes * V * size + lists, "flops": flops * live * V}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device=DEV)


def _distinct(g, shape, n, V):
    """n ids for each of `shape` that differ, anywhere in the vocabulary."""
    first = torch.randint(0, V, (*shape, 1), generator=g, device=DEV)
    step = torch.randint(1, max(2, V // n), (*shape, 1), generator=g, device=DEV)
    return (first + step * torch.arange(n, device=DEV)) % V


def _model_logits(g, rows, V, dtype):
    """A model's logits: a broad bulk, and some tokens far above it, more so in rows where the model is sure."""
    x = torch.randn(rows, V, generator=g, device=DEV) * 2.0
    n = min(48, V)
    at = _distinct(g, (rows,), n, V)
    lift = _rand(g, rows, n) * (4.0 + 10.0 * _rand(g, rows, 1))
    return x.scatter_(1, at, x.gather(1, at) + lift).to(dtype)


def _sample_inputs(case, seed):
    g = _gen(seed)
    B, V = case["batch"], case["vocab"]
    t = {"logits": _model_logits(g, B, V, DT[case["dtype"]]), "uniform": _rand(g, B)}
    if case["masked"]:
        t["logits"].masked_fill_(_rand(g, B, V) < 0.3, -math.inf)
        if B > 2:
            t["logits"][B // 2] = -math.inf
    for name in ("temperature", "top_k", "top_p", "min_p"):
        t[name] = case[name]
    if case["each"]:
        t["temperature"] = case["temperature"] * (0.5 + _rand(g, B))
        t["temperature"][::7] = 0.0
        t["top_k"] = torch.randint(0, 2 * case["top_k"] + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        t["top_p"] = (case["top_p"] + 0.2 * (_rand(g, B) - 0.5)).clamp_(max=1.0)
        t["min_p"] = case["min_p"] * 2.0 * _rand(g, B)
    return t


def _top_inputs(case, seed):
    return _model_logits(_gen(seed), case["rows"], case["vocab"], DT[case["dtype"]])


def _kl_inputs(case, seed):
    g = _gen(seed)
    dt, B, S, V, K = DT[case["dtype"]], case["batch"], case["seq"], case["vocab"], case["k"]
    n, T = _tokens(case), case["temperature"]
    t = {}
    ids = _distinct(g, (B, n), K, V)
    # logits that fall from the first entry to the last
    fall = torch.cumsum(_rand(g, B, n, K) * 8.0 / K ** 0.5, -1)
    values = (14.0 + 4.0 * _rand(g, B, n, 1) - fall).to(dt)
    t["lse"] = None
    if case["rest"]:  # the other tokens hold up to a third of the teacher's probability
        t["lse"] = torch.logsumexp(values.double() / T, -1) - torch.log1p(-0.33 * _rand(g, B, n).double())
        t["lse"] = t["lse"].float()
    logits = torch.randn(B, S, V, generator=g, device=DEV) * 2.0
    near = values.float() + torch.randn(B, n, K, generator=g, device=DEV)
    logits[:, :n].scatter_(2, ids, near)
    t["logits"] = logits.to(dt)[:, :n]
    if case["padded"]:  # records end where the teacher's probability is covered, one of them at once
        length = torch.randint(1, K + 1, (B, n, 1), generator=g, device=DEV)
        length[0, 0] = 0
        past = torch.arange(K, device=DEV) >= length
        ids = ids.masked_fill(past, -1)
    t["values"], t["ids"] = values, ids.int()
    t["weights"] = None
    if case["prompt"] > 0:
        t["weights"] = (torch.arange(n, device=DEV) >= _prompt(case)).float().expand(B, n).contiguous()
    if case["order"] == "hvp":
        t["along"] = torch.randn(B, n, V, generator=g, device=DEV).to(dt)
    return t


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------
def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "sample":
        state.update(_sample_inputs(case, seed))
    elif case["kind"] == "top":
        state["logits"] = _top_inputs(case, seed)
    else:
        state.update(_kl_inputs(case, seed))
        if own and case["order"] != "loss":
            state["logits"].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"sample": _run_sample, "top": _run_top, "kl": _run_kl}[state["case"]["kind"]](state)


def _column(x, dtype, B):
    if isinstance(x, torch.Tensor):
        return x.to(dtype)[:, None]
    return torch.full((B, 1), x, dtype=torch.float32, device=DEV).to(dtype)


def _run_sample(state):
    x, u = state["logits"], state["uniform"]
    if own:
        from sparseforge_amd.logits import sample_logits

        return sample_logits(x, u, temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                             min_p=state["min_p"], logprobs=True)
    B, V = x.shape
    temperature, p, least = (_column(state[n], torch.float64, B) for n in ("temperature", "top_p", "min_p"))
    k = _column(state["top_k"], torch.int64, B)
    sorted_, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    top = sorted_[:, :1].double()
    none = top == -math.inf
    d = sorted_.double() - top.masked_fill(none, 0.0)
    w = torch.where(temperature > 0, d / temperature.clamp_min(1e-30), torch.where(d < 0, -math.inf, d)).exp_()
    rank = torch.arange(V, device=DEV)[None]
    kept = (rank < k.masked_fill(k <= 0, V)) & ((temperature > 0) | (rank == 0))
    w.masked_fill_(~kept, 0.0)
    before = torch.cumsum(w, -1)
    total = before[:, -1:].clone()
    before = torch.cat([torch.zeros_like(total), before[:, :-1]], -1)
    kept &= ((p >= 1.0) | (before < p * total) | (rank == 0)) & (w >= least)
    w.masked_fill_(~kept, 0.0)
    w = torch.zeros_like(w).scatter_(1, ids, w)  # in the order of the ids
    c = torch.cumsum(w, -1)
    total = c[:, -1:].clone()
    drawn = (c <= u.double()[:, None] * total).sum(-1, keepdim=True).clamp_(max=V - 1)
    logprob = (w.gather(1, drawn) / total).log().float()[:, 0]
    none = none[:, 0]
    return drawn[:, 0].masked_fill(none, -1), logprob.masked_fill(none, -math.inf)


def _run_top(state):
    case, x = state["case"], state["logits"]
    if own:
        from sparseforge_amd.distill import top_logits

        top = top_logits(x, case["k"], case["temperature"])
        return top.values, top.ids, top.lse
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    k = case["k"]
    a = x.float() / case["temperature"]
    m = a.amax(-1, keepdim=True)
    lse = m + (a - m).exp().sum(-1, keepdim=True).log()
    return values[:, :k].clone(), ids[:, :k].int(), lse[:, 0]


def _run_kl(state):
    case, s = state["case"], state["logits"]
    T = case["temperature"]
    if own:
        from sparseforge_amd.distill import TopLogits, top_kl_loss

        teacher = TopLogits(state["values"], state["ids"], state["lse"], T)
        loss = top_kl_loss(s, teacher, T, weights=state["weights"])
        if case["order"] == "loss":
            return (loss,)
        if case["order"] == "grad":
            return loss, torch.autograd.grad(loss, s)[0]
        g, = torch.autograd.grad(loss, s, create_graph=True)
        h, = torch.autograd.grad(g, s, state["along"])
        return loss, g.detach(), h
    B, n, V = s.shape
    s = s.reshape(B * n, V)
    ids, values = state["ids"].view(B * n, -1).long(), state["values"].view(B * n, -1)
    real = ids >= 0
    ids = ids.clamp_min(0)
    # the teacher's few entries in float64: what they leave to the other tokens is a small difference
    b = (values.double() / T).masked_fill(~real, -math.inf)
    if state["lse"] is not None:
        p = (b - state["lse"].view(-1, 1).double()).exp()
        r = (1.0 - p.sum(-1)).clamp_min(0.0)
    else:
        top = b.amax(-1, keepdim=True)
        p = (b - top.masked_fill(top == -math.inf, 0.0)).exp()
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        r = torch.zeros(B * n, dtype=torch.float64, device=DEV)
    P = p.sum(-1) + r
    a = s.float() / T
    m = a.amax(-1, keepdim=True)
    e = (a - m).exp()
    total = e.sum(-1, keepdim=True)
    listed_ = torch.zeros(B * n, V, dtype=torch.bool, device=DEV)
    row = torch.arange(B * n, device=DEV)[:, None].expand_as(ids)[real]
    listed_[row, ids[real]] = True
    rest = e.masked_fill(listed_, 0.0).sum(-1, keepdim=True)
    log_q = a.gather(1, ids) - m - total.log()
    loss = torch.where(p > 0, p * (p.log() - log_q.double()), 0.0).sum(-1)
    loss = loss + torch.where(r > 0, r * (r.log() - (rest / total).log()[:, 0].double()), 0.0)
    w = state["weights"].view(-1).double() if state["weights"] is not None else torch.ones_like(loss)
    share = w / w.sum().clamp_min(1e-300)
    out = [(T * T * (share * loss.masked_fill(w == 0, 0.0)).sum()).float()]
    if case["order"] == "loss":
        return tuple(out)
    q = e / total
    rho = (e / rest).masked_fill_(listed_, 0.0)
    P, r, scale = P.float()[:, None], r.float()[:, None], (T * share).float()[:, None]
    g = P * q - r * rho
    g.scatter_add_(1, ids, -p.float())
    out.append((scale * g).masked_fill_(scale == 0, 0.0).view(B, n, V).to(s.dtype))
    if case["order"] == "hvp":
        u = state["along"].view(B * n, V).float()
        h = P * q * (u - (u * q).sum(-1, keepdim=True)) - r * rho * (u - (u * rho).sum(-1, keepdim=True))
        out.append((scale / T * h).masked_fill_(scale == 0, 0.0).view(B, n, V).to(s.dtype))
    return tuple(out)


# ---------------------------------------------------------------------------
# the definitions in float64
# ---------------------------------------------------------------------------
def exact(case, seed):
    return {"sample": _exact_sample, "top": _exact_top, "kl": _exact_kl}[case["kind"]](case, seed)


def _exact_sample(case, seed):
    t = _sample_inputs(case, seed)
    B, V = case["batch"], case["vocab"]

    def at(name, b):
        return float(t[name][b]) if isinstance(t[name], torch.Tensor) else float(torch.tensor(t[name]))

    tokens, logprobs = [], []
    for b in range(B):
        x = t["logits"][b].double()
        T, k, p, least = at("temperature", b), int(at("top_k", b)), at("top_p", b), at("min_p", b)
        if not bool((x > -math.inf).any()):
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        order = torch.argsort(-x, stable=True)[:k if 0 < k < V else V]
        if T == 0.0:
            order, T = order[:1], 1.0
        prob = torch.softmax(x[order] / T, 0)
        count = len(order)
        if p < 1.0:  # the fewest tokens that hold p, the first of them in any case
            held = torch.cumsum(prob, 0)
            count = max(1, min(count, int(torch.searchsorted(held, torch.tensor([p], dtype=held.dtype, device=DEV)))
                               + 1))
        count = min(count, int((prob >= least * prob[0]).sum()))
        order = order[:count].sort().values
        prob = torch.softmax(x[order] / T, 0)
        held = torch.cumsum(prob, 0)
        i = int(torch.searchsorted(held, t["uniform"][b:b + 1].double() * held[-1], right=True))
        i = min(i, count - 1)
        tokens.append(int(order[i]))
        logprobs.append(float(prob[i].log()))
    return (torch.tensor(tokens, device=DEV), torch.tensor(logprobs, dtype=torch.float64, device=DEV))


def _exact_top(case, seed):
    x = _top_inputs(case, seed).double()
    k = case["k"]
    ids = torch.empty(case["rows"], k, dtype=torch.int64, device=DEV)
    for at in range(0, case["rows"], 64):
        ids[at:at + 64] = torch.argsort(-x[at:at + 64], dim=-1, stable=True)[:, :k]
    return x.gather(1, ids), ids.int(), torch.logsumexp(x / case["temperature"], -1)


def _exact_kl(case, seed):
    """A definition to differentiate: cross-entropies of the listed tokens and of the rest taken together."""
    t = _kl_inputs(case, seed)
    T, order = case["temperature"], case["order"]
    B, n, V = t["logits"].shape
    w = t["weights"].double() if t["weights"] is not None else torch.ones(B, n, dtype=torch.float64, device=DEV)
    loss, grads, products = torch.zeros((), dtype=torch.float64, device=DEV), [], []
    step = max(1, (1 << 25) // V)
    for b in range(B):
        for i in range(0, n, step):
            rows = slice(i, min(n, i + step))
            s = t["logits"][b, rows].double().requires_grad_(order != "loss")
            part = (_kl_rows(s / T, t["values"][b, rows].double() / T, t["ids"][b, rows].long(),
                             t["lse"][b, rows].double() if t["lse"] is not None else None)
                    * w[b, rows]).sum() * (T * T) / w.sum()
            loss += part.detach()
            if order == "loss":
                continue
            g, = torch.autograd.grad(part, s, create_graph=order == "hvp")
            grads.append(g.detach())
            if order == "hvp":
                products.append(torch.autograd.grad(g, s, t["along"][b, rows].double())[0])
    out = [loss]
    for parts in (grads, products):
        if parts:
            out.append(torch.cat(parts).view(B, n, V))
    return tuple(out)


def _kl_rows(a, b, ids, lse):
    log_q = torch.log_softmax(a, -1)
    real = ids >= 0
    spare = a.shape[1]  # padding goes to a column past the vocabulary
    flags = torch.zeros(a.shape[0], spare + 1, dtype=torch.bool, device=a.device)
    flags.scatter_(1, torch.where(real, ids, spare), True)
    b = b.masked_fill(~real, -math.inf)
    log_p = b - (lse[:, None] if lse is not None else torch.logsumexp(b, -1, keepdim=True))
    log_p = log_p.masked_fill(~real, 0.0)
    p = log_p.exp().masked_fill(~real, 0.0)
    loss = (p * (log_p - log_q.gather(1, ids.clamp_min(0)))).sum(-1)
    if lse is not None:
        r = (1.0 - p.sum(-1)).clamp_min(0.0)
        log_rest = torch.logsumexp(log_q.masked_fill(flags[:, :spare], -math.inf), -1)
        loss = loss + torch.where(r > 0, r * (r.clamp_min(1e-300).log() - log_rest), 0.0)
    return loss
