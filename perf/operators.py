"""The workloads on which the token-scoring operators are measured.

Three operators, each with the calls a training or serving program makes of it:

* ``statistics``: log-probability of given tokens, entropy and the top alternatives of rows of logits
  (``ops.token_statistics``), with the gradient where the case trains;
* ``distillation``: the KL divergence from a teacher's recorded top alternatives to a student's logits and
  its gradient (``ops.distillation_loss``);
* ``head``: the same statistics straight from hidden states and the LM head's weight
  (``ops.linear_token_statistics``), with both gradients where the case trains.

A case is a dict: ``op``, ``rows``, ``vocab``, ``dtype`` and ``temperature``, and what its operator adds.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}

# The largest of each, in logits (rows x vocab) and in multiply-adds of the LM head's products.
_MOST_LOGITS = 4096 * 151936
_MOST_PRODUCT = 4096 * 2048 * 151936


def _statistics(name, rows, vocab, dtype, temperature, top, targets, ignored=0, masked=0, pitch=0, grad=False):
    return {"name": name, "op": "statistics", "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top": top, "targets": targets, "ignored": ignored, "masked": masked,
            "pitch": pitch or vocab, "grad": grad}


def _distillation(name, rows, vocab, dtype, temperature, top, tail, ignored=0, grad=True):
    return {"name": name, "op": "distillation", "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top": top, "tail": tail, "ignored": ignored, "grad": grad}


def _head(name, rows, vocab, hidden, temperature, ignored=0, grad=False):
    return {"name": name, "op": "head", "rows": rows, "vocab": vocab, "hidden": hidden, "dtype": "bf16",
            "temperature": temperature, "ignored": ignored, "grad": grad}


def listed():
    return [
        # one step of one request: the sampled token's log-probability, the entropy and 20 alternatives
        _statistics("decode one token", 1, 151936, "bf16", 0.7, 20, True),
        # one step of a rollout group whose logits the sampler holds in 32 bits, with masked-out padding
        _statistics("decode a group, f32", 64, 129280, "f32", 1.0, 5, True, masked=120),
        # teacher-forced scoring of padded responses: a third of the positions are prompt or padding
        _statistics("score responses", 3001, 151936, "bf16", 0.7, 0, True, ignored=1000),
        # a teacher's records for distillation: 64 alternatives of every position
        _statistics("record a teacher", 4096, 151936, "bf16", 1.0, 64, False),
        # the policy step with an entropy bonus, on logits cut to the tokeniser's odd vocabulary
        _statistics("policy step, odd vocabulary", 2047, 151669, "bf16", 1.0, 0, True, ignored=400, pitch=151936,
                    grad=True),
        # the training loop of a small model: launch latency only
        _distillation("distil a small model", 6, 512, "f32", 1.0, 8, True, ignored=1),
        # a distillation step at the length of the training configurations
        _distillation("distil a sequence", 4096, 151936, "bf16", 1.0, 64, True),
        # 32-bit logits, renormalised alternatives, part of the rows without a teacher
        _distillation("distil, f32 renormalised", 1500, 129280, "f32", 2.0, 20, False, ignored=300),
        # the loss alone on held-out text
        _distillation("distillation evaluation", 2000, 151936, "bf16", 1.0, 32, True, grad=False),
        # one step of a rollout group from its hidden states: the weight's traffic is all there is
        _head("head, decode a group", 16, 151936, 2048, 1.0),
        # scoring one training sequence from its hidden states
        _head("head, score a sequence", 4096, 151936, 2048, 0.7, ignored=1024),
        # the policy step from the hidden states: gradients of these and of the weight
        _head("head, policy step", 1023, 129280, 5120, 1.0, ignored=100, grad=True),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["statistics", "statistics", "distillation", "distillation", "head"])
    temperature = rng.choice([0.6, 0.7, 1.0, 1.0, 1.3, 2.0])
    if op == "head":
        hidden = 8 * _spread(rng, 8, 640)
        vocab = _spread(rng, 32, 151936)
        grad = rng.random() < 0.5
        rows = _spread(rng, 1, min(4096, max(1, _MOST_PRODUCT // (hidden * vocab * (3 if grad else 1)))))
        return {k: v for k, v in _head("", rows, vocab, hidden, temperature, rng.randrange(rows // 3 + 1),
                                       grad).items() if k != "name"}
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    most = _MOST_LOGITS // (2 if dtype == "f32" else 1)
    vocab = _spread(rng, 32, 151936)
    rows = _spread(rng, 1, min(4096, max(1, most // vocab)))
    ignored = rng.randrange(rows // 3 + 1)
    grad = rng.random() < 0.6
    if op == "distillation":
        case = _distillation("", rows, vocab, dtype, temperature, min(vocab // 2, _spread(rng, 1, 64)),
                             rng.random() < 0.5, ignored, grad)
    else:
        top = rng.choice([0, 1, 5, 20, 64])
        case = _statistics("", rows, vocab, dtype, temperature, min(top, vocab // 2), True if grad else rng.random() < 0.7,
                           ignored, rng.choice([0, 0, min(7, vocab // 8)]),
                           vocab + rng.choice([0, 0, 0, 1, 8, 64 - vocab % 64]), grad)
        if not case["targets"]:
            case["ignored"] = 0
    return {k: v for k, v in case.items() if k != "name"}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(case, g):
    """Rows of logits as a language model gives them: a broad bulk, and some tens of tokens far above it."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, case.get("pitch", vocab), device="cuda", generator=g)
    x = x.mul_(2.0)
    # distinct tokens, one of each of 40 (or `vocab`) stretches of the vocabulary, rotated by row
    count = min(40, vocab)
    likely = torch.randint(0, vocab // count, (rows, count), device="cuda", generator=g)
    likely = likely + torch.arange(count, device="cuda") * (vocab // count)
    likely = (likely + torch.randint(0, vocab, (rows, 1), device="cuda", generator=g)) % vocab
    x.scatter_(1, likely, 4 + 6 * torch.rand(likely.shape, device="cuda", generator=g))
    if case.get("masked"):
        x[:, vocab - case["masked"]:vocab] = float("-inf")
    return x.to(_TYPES[case["dtype"]])[:, :vocab], likely[:, 0]


def _targets(case, likely, g):
    """Half of the tokens are likely ones; `ignored` of the rows, spread over them, have none (-100)."""
    rows = case["rows"]
    anywhere = torch.randint(0, case["vocab"] - case.get("masked", 0), (rows,), device="cuda", generator=g)
    likely = torch.minimum(likely, torch.full_like(likely, case["vocab"] - case.get("masked", 0) - 1))
    t = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.5, likely, anywhere)
    t[torch.randperm(rows, device="cuda", generator=g)[:case["ignored"]]] = -100
    return t


def _teacher(case, logits, g):
    """A teacher near the student: its top alternatives and their log-probabilities at the temperature;
    some rows have fewer, and `ignored` of them none (id -1)."""
    rows, top = case["rows"], case["top"]
    t = torch.randn(logits.shape, device="cuda", generator=g).mul_(0.7).add_(logits).div_(case["temperature"])
    values, ids = t.topk(top, dim=1)
    values = values - t.logsumexp(dim=1, keepdim=True)
    count = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.2,
                        torch.randint(1, top + 1, (rows,), device="cuda", generator=g), top)
    count[torch.randperm(rows, device="cuda", generator=g)[:case["ignored"]]] = 0
    absent = torch.arange(top, device="cuda") >= count[:, None]
    return ids.masked_fill(absent, -1), values.masked_fill(absent, float("-inf"))


def prepare(case, seed):
    g = _generator(seed)
    rows, state = case["rows"], {"case": case}
    if case["op"] == "head":
        state["hidden"] = torch.randn(rows, case["hidden"], device="cuda", generator=g).to(torch.bfloat16)
        state["weight"] = torch.randn(case["vocab"], case["hidden"], device="cuda", generator=g).mul_(
            2.5 / math.sqrt(case["hidden"])).to(torch.bfloat16)
        state["targets"] = _targets(case, torch.randint(0, case["vocab"], (rows,), device="cuda", generator=g), g)
    else:
        logits, likely = _logits(case, g)
        state["logits"] = logits
        if case["op"] == "distillation":
            state["ids"], state["teacher"] = _teacher(case, logits, g)
            state["weights"] = torch.rand(rows, device="cuda", generator=g) / rows
        elif case["targets"]:
            state["targets"] = _targets(case, likely, g)
    if case["op"] != "distillation" and case["grad"]:
        # what a policy gradient with an entropy bonus hands back for each row
        state["g"] = torch.randn(rows, device="cuda", generator=g)
        state["h"] = torch.rand(rows, device="cuda", generator=g) * 0.2
    if case["grad"]:
        for name in ("logits", "hidden", "weight"):
            if name in state:
                state[name].requires_grad_()
    return state


# -- the plain forms ------------------------------------------------------------------------------
def _alternatives(x, lp, skip, top):
    """The `top` largest of each row, ties to the lowest index, by a whole-number key of value and index."""
    bits = (x + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    key = key + torch.arange(x.shape[1] - 1, -1, -1, device=x.device)
    ids = x.shape[1] - 1 - (key.topk(top, dim=1).values & 0xFFFFFFFF)
    values = lp.gather(1, ids)
    absent = skip[:, None] | (x.gather(1, ids) == float("-inf"))
    return ids.masked_fill(absent, -1), values.masked_fill(absent, float("-inf"))


def _plain_rows(x, targets, temperature, top):
    """Statistics of 32-bit logits, and what their gradient needs: (log_probs, entropy, ids, values, p, lp)."""
    y = x / temperature
    y = y - y.amax(dim=1, keepdim=True)
    e = y.exp()
    total = e.sum(dim=1, keepdim=True)
    lp, p = y - total.log(), e / total
    plogp = torch.where(p > 0, p * lp, 0.0)
    skip = torch.zeros(len(x), dtype=torch.bool, device=x.device) if targets is None else targets == -100
    entropy = torch.where(skip, 0.0, -plogp.sum(dim=1))
    log_probs = None
    if targets is not None:
        log_probs = torch.where(skip, 0.0, lp.gather(1, targets.clamp(min=0)[:, None])[:, 0])
    ids = values = None
    if top:
        ids, values = _alternatives(x, lp, skip, top)
    return log_probs, entropy, ids, values, p, lp, skip


def _plain_gradient(p, lp, entropy, targets, skip, g, h, temperature):
    d = -p * (g[:, None] + h[:, None] * (torch.where(p > 0, lp, 0.0) + entropy[:, None]))
    d.scatter_add_(1, targets.clamp(min=0)[:, None], g[:, None])
    return torch.where(skip[:, None], 0.0, d / temperature)


def _plain_statistics(state):
    case = state["case"]
    x, targets = state["logits"].detach().float(), state.get("targets")
    log_probs, entropy, ids, values, p, lp, skip = _plain_rows(x, targets, case["temperature"], case["top"])
    out = {"entropy": entropy}
    if targets is not None:
        out["log_probs"] = log_probs
    if case["top"]:
        out["top_ids"], out["top_log_probs"] = ids, values
    if case["grad"]:
        out["dlogits"] = _plain_gradient(p, lp, entropy, targets, skip, state["g"], state["h"],
                                         case["temperature"]).to(state["logits"].dtype)
    return out


def _plain_distillation(state):
    case = state["case"]
    ids, t, w = state["ids"], state["teacher"].float(), state["weights"]
    y = state["logits"].detach().float() / case["temperature"]
    there, at = ids >= 0, ids.clamp(min=0)
    any_ = there.any(dim=1)
    q = torch.where(there, t, float("-inf")).exp()
    rest = torch.zeros_like(w)
    if case["tail"]:
        rest = torch.where(any_, (1 - q.sum(dim=1)).clamp(min=0), 0.0)
    else:
        q = q / torch.where(any_, q.sum(dim=1), 1.0)[:, None]
    y = y - y.amax(dim=1, keepdim=True)
    # the logits outside the alternatives: absent places point at a column of their own
    outside = torch.cat((y, y.new_zeros(len(y), 1)), dim=1)
    outside.scatter_(1, torch.where(there, at, y.shape[1]), float("-inf"))
    outside = outside[:, :-1]
    e, e_out = y.exp(), outside.exp()
    total, total_out = e.sum(dim=1), e_out.sum(dim=1)
    lp = y.gather(1, at) - total.log()[:, None]
    rows = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(dim=1)
    rows = rows + torch.where(rest > 0, rest * (rest.log() - (total_out / total).log()), 0.0)
    rows = torch.where(any_, rows, 0.0)
    out = {"rows": rows, "total": (w * rows).sum()}
    if case["grad"]:
        whole = q.sum(dim=1) + rest
        d = whole[:, None] * e / total[:, None]
        d = d - torch.where(rest > 0, rest / total_out, 0.0)[:, None] * e_out
        d = d.scatter_add_(1, at, -torch.where(there, q, 0.0))
        d = d * (w / case["temperature"])[:, None]
        out["dlogits"] = torch.where(any_[:, None], d, 0.0).to(state["logits"].dtype)
    return out


def _plain_head(state):
    case, targets = state["case"], state["targets"]
    hidden, weight = state["hidden"].detach().float(), state["weight"].detach().float()
    log_probs, entropy, _, _, p, lp, skip = _plain_rows(hidden @ weight.t(), targets, case["temperature"], 0)
    out = {"log_probs": log_probs, "entropy": entropy}
    if case["grad"]:
        d = _plain_gradient(p, lp, entropy, targets, skip, state["g"], state["h"], case["temperature"])
        out["dhidden"] = (d @ weight).to(torch.bfloat16)
        out["dweight"] = (d.t() @ hidden).to(torch.bfloat16)
    return out


# -- the framework's operators --------------------------------------------------------------------
def _own_statistics(state):
    from tiny_dsv41_b200 import ops

    case = state["case"]
    s = ops.token_statistics(state["logits"], state.get("targets"), temperature=case["temperature"], top=case["top"])
    out = {"entropy": s.entropy.detach()}
    if s.log_probs is not None:
        out["log_probs"] = s.log_probs.detach()
    if case["top"]:
        out["top_ids"], out["top_log_probs"] = s.top_ids, s.top_log_probs.detach()
    if case["grad"]:
        out["dlogits"], = torch.autograd.grad((s.log_probs, s.entropy), state["logits"], (state["g"], state["h"]))
    return out


def _own_distillation(state):
    from tiny_dsv41_b200 import ops

    case = state["case"]
    loss = ops.distillation_loss(state["logits"], state["ids"], state["teacher"], state["weights"],
                                 temperature=case["temperature"], tail=case["tail"])
    out = {"rows": loss.rows, "total": loss.total.detach()}
    if case["grad"]:
        out["dlogits"], = torch.autograd.grad(loss.total, state["logits"])
    return out


def _own_head(state):
    from tiny_dsv41_b200 import ops

    case = state["case"]
    s = ops.linear_token_statistics(state["hidden"], state["weight"], state["targets"],
                                    temperature=case["temperature"])
    out = {"log_probs": s.log_probs.detach(), "entropy": s.entropy.detach()}
    if case["grad"]:
        out["dhidden"], out["dweight"] = torch.autograd.grad((s.log_probs, s.entropy),
                                                             (state["hidden"], state["weight"]),
                                                             (state["g"], state["h"]))
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"statistics": _own_statistics, "distillation": _own_distillation, "head": _own_head}[op](state)
    with torch.no_grad():
        return {"statistics": _plain_statistics, "distillation": _plain_distillation, "head": _plain_head}[op](state)


# -- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    rows, vocab, size = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    read = rows - case["ignored"]  # rows without a target or a teacher need not be read; their gradient is zeros
    if case["op"] == "head":
        h, passes = case["hidden"], 3 if case["grad"] else 1
        data = (vocab * h * size + read * h * size) + 16 * rows
        if case["grad"]:
            data += vocab * h * size + rows * h * size + 8 * rows
        return {"bytes": data, "flops": 2 * read * vocab * h * passes + 8 * read * vocab}
    data = read * vocab * size + (rows * vocab * size if case["grad"] else 0)
    if case["op"] == "distillation":
        return {"bytes": data + rows * (case["top"] * 12 + 8) + 4, "flops": (8 if case["grad"] else 5) * read * vocab}
    data += rows * (4 + (12 if case["targets"] else 0) + 12 * case["top"] + (8 if case["grad"] else 0))
    return {"bytes": data, "flops": (12 if case["grad"] else 6) * read * vocab}


# -- the definitions in 64 bits -------------------------------------------------------------------
def _blocks(rows, vocab):
    """Row ranges whose 64-bit logits take about 2 GB."""
    step = max(1, (1 << 28) // vocab)
    return [slice(a, min(rows, a + step)) for a in range(0, rows, step)]


def _exact_scores(x, targets, temperature, g=None, h=None):
    """(log_probs, entropy, lp, gradient) of 64-bit logits, by log_softmax."""
    lp = torch.log_softmax(x / temperature, dim=1)
    p = lp.exp()
    entropy = -(p * lp.nan_to_num(neginf=0.0)).sum(dim=1)
    keep = torch.ones(len(x), dtype=torch.bool, device=x.device) if targets is None else targets >= 0
    chosen = None
    if targets is not None:
        one = torch.zeros_like(lp).scatter_(1, targets.clamp(min=0)[:, None], 1.0)
        chosen = lp.masked_fill(one == 0, 0.0).sum(dim=1) * keep
    d = None
    if g is not None:
        # log p of the target and the entropy, each differentiated on its own
        d_chosen = one - p
        d_entropy = -p * (lp.nan_to_num(neginf=0.0) + entropy[:, None])
        d = (d_chosen * g.double()[:, None] + d_entropy * h.double()[:, None]) / temperature * keep[:, None]
    return chosen, entropy * keep, lp, d


def _exact_statistics(case, state):
    parts = []
    for b in _blocks(case["rows"], case["vocab"]):
        x, t = state["logits"].detach()[b].double(), state["targets"][b] if case["targets"] else None
        grads = (state["g"][b], state["h"][b]) if case["grad"] else (None, None)
        chosen, entropy, lp, d = _exact_scores(x, t, case["temperature"], *grads)
        part = {"entropy": entropy}
        if case["targets"]:
            part["log_probs"] = chosen
        if case["top"]:
            values = lp.topk(case["top"], dim=1).values
            part["top_log_probs"] = values if t is None else values.masked_fill((t < 0)[:, None], float("-inf"))
        if case["grad"]:
            part["dlogits"] = d
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["top"]:
        out["top_ids"] = None
    return out


def _exact_distillation(case, state):
    parts = []
    for b in _blocks(case["rows"], case["vocab"]):
        ids, t, w = state["ids"][b], state["teacher"][b].double(), state["weights"][b].double()
        lp = torch.log_softmax(state["logits"].detach()[b].double() / case["temperature"], dim=1)
        # the teacher's and the student's distributions over the vocabulary, zero outside the alternatives
        q = torch.zeros_like(lp)
        q.scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, t.exp(), 0.0))
        inside = torch.zeros_like(lp).scatter_add_(1, ids.clamp(min=0), (ids >= 0).double()) > 0
        have = inside.any(dim=1)
        if case["tail"]:
            rest = (1 - q.sum(dim=1)).clamp(min=0) * have
        else:
            q = q / torch.where(have, q.sum(dim=1), 1.0)[:, None]
            rest = torch.zeros_like(w)
        left = lp.masked_fill(inside, float("-inf")).logsumexp(dim=1)
        rows = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(dim=1)
        rows = (rows + torch.where(rest > 0, rest * (rest.log() - left), 0.0)) * have
        part = {"rows": rows, "weighted": w * rows}
        if case["grad"]:
            mass = torch.where(inside, q, (rest * (lp - left[:, None]).exp().T).T)
            mass = torch.where(rest[:, None] > 0, mass, q)
            d = lp.exp() * (q.sum(dim=1) + rest)[:, None] - mass
            part["dlogits"] = d * (w / case["temperature"] * have)[:, None]
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    out["total"] = out.pop("weighted").sum()
    return out


def _exact_head(case, state):
    weight = state["weight"].detach().double()
    parts, dweight = [], torch.zeros_like(weight) if case["grad"] else None
    for b in _blocks(case["rows"], case["vocab"]):
        hidden = state["hidden"].detach()[b].double()
        grads = (state["g"][b], state["h"][b]) if case["grad"] else (None, None)
        chosen, entropy, _, d = _exact_scores(hidden @ weight.T, state["targets"][b], case["temperature"], *grads)
        part = {"log_probs": chosen, "entropy": entropy}
        if case["grad"]:
            part["dhidden"] = d @ weight
            dweight.addmm_(d.T, hidden)
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case["grad"]:
        out["dweight"] = dweight
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        out = {"statistics": _exact_statistics, "distillation": _exact_distillation, "head": _exact_head}[case["op"]](
            case, state)
    return out
