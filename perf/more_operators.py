"""The workloads on which the operators of a decoding step are measured.

Three operators, in the order in which a step of a language model that serves or samples calls them:

* ``append``: the norms of queries and keys, their position rotation, and the keys and values of the new
  tokens written into a paged cache (``ops.paged_append``);
* ``attend``: attention of the new tokens over that cache, causal or under the mask of a tree of drafted
  tokens (``ops.paged_attention``);
* ``logits``: penalties for repeated tokens, biases and grammar masks on the logits (``ops.process_logits``).

A case is a dict of plain values. The lengths of its sequences follow from it, so that every seed measures
the same work; pages, tokens and values follow from the seed.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_DIM = 128  # of a head
_EPS = 1e-6

# What the largest listed cases cost: drawn ones stay below.
_MOST_TOKENS = 8192
_MOST_CACHE = 8 * 40960 * 4  # cached tokens x key heads
_MOST_SCORES = 3 * 2048 * 8192 * 32  # (query, key) pairs x heads
_MOST_LOGITS = 512 * 151936


def _append(name, seqs, new, longest, heads, kv_heads, page, dtype, shortest=1):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "longest": longest, "shortest": shortest,
            "heads": heads, "kv_heads": kv_heads, "page": page, "dtype": dtype}


def _attend(name, seqs, new, longest, heads, kv_heads, page, dtype, shortest=1, tree=False):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "longest": longest, "shortest": shortest,
            "heads": heads, "kv_heads": kv_heads, "page": page, "dtype": dtype, "tree": tree}


def _logits(name, rows, vocab, dtype, history, penalties, biased, allowed):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "dtype": dtype, "history": history,
            "penalties": penalties, "biased": biased, "allowed": allowed}


def listed():
    return [
        # one step of one request, some thousand tokens in: launch latency
        _append("append, one token", 1, 1, 4001, 32, 4, 64, "bf16"),
        # one step of a rollout group whose members are at different lengths
        _append("append, a group", 64, 1, 2048, 32, 4, 64, "bf16"),
        # the prompts of a group in one packed batch, none of them a multiple of anything
        _append("append, prompts", 5, 2900, 2901, 32, 4, 16, "bf16", shortest=700),
        # one step of one request: the cache is read by as many SMs as there are
        _attend("attend, one request", 1, 1, 4001, 32, 4, 64, "bf16"),
        # one step of a rollout group, from sequences that have just begun to long ones
        _attend("attend, a group", 64, 1, 8192, 32, 4, 64, "bf16"),
        # one step of a few requests near the longest context of the model configurations
        _attend("attend, long contexts", 8, 1, 40960, 32, 4, 128, "bf16", shortest=20000),
        # chunks of prompts, up to 2048 tokens of a sequence, on what is cached of it
        _attend("attend, prompt chunks", 3, 2048, 8192, 32, 4, 64, "bf16", shortest=2048),
        # verifying the drafts of a group: trees of 32 tokens
        _attend("attend, drafted trees", 16, 32, 8192, 32, 4, 16, "bf16", shortest=500, tree=True),
        # verifying the draft of one request, a tree of 60 tokens that is no multiple of anything
        _attend("attend, one drafted tree", 1, 60, 2301, 32, 4, 32, "f16", tree=True),
        # sampling one token under a grammar, with the penalties of a request and its history
        _logits("logits, one row", 1, 151936, "bf16", 2000, True, 40, "few"),
        # a group whose sampler holds 32-bit logits, with long histories
        _logits("logits, a group", 64, 129280, "f32", 8192, True, 0, "all"),
        # the rows of drafted trees, each with its own grammar state, on the tokeniser's odd vocabulary
        _logits("logits, drafted rows", 512, 151669, "bf16", 1024, True, 16, "most"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "logits", "logits"])
    if op == "logits":
        vocab = _spread(rng, 32, 151936)
        rows = _spread(rng, 1, min(512, max(1, _MOST_LOGITS // vocab)))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if dtype == "f32":
            rows = max(1, rows // 2)
        case = _logits("", rows, vocab, dtype, _spread(rng, 1, 8192), rng.random() < 0.8,
                       min(vocab // 2, rng.choice([0, 0, 1, 7, 40, 300])), rng.choice(["few", "most", "all"]))
        return {k: v for k, v in case.items() if k != "name"}
    heads, kv_heads = rng.choice([(32, 4), (32, 4), (4, 2), (8, 8), (16, 1), (12, 4), (6, 2)])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "append":
        new = _spread(rng, 1, 4096)
        seqs = _spread(rng, 1, max(1, min(64, _MOST_TOKENS // new)))
        longest = new + _spread(rng, 1, 1024) - 1
        case = _append("", seqs, new, longest, heads, kv_heads, page, dtype, rng.randint(1, longest))
    else:
        tree = rng.random() < 0.35
        new = _spread(rng, 1, 64) if tree else rng.choice([1, 1, _spread(rng, 1, 2048)])
        longest = new + _spread(rng, 1, 40960 - new)
        most = min(_MOST_CACHE // (longest * kv_heads), _MOST_SCORES // (longest * new * heads))
        seqs = _spread(rng, 1, max(1, min(128, most)))
        case = _attend("", seqs, new, longest, heads, kv_heads, page, dtype, rng.randint(1, longest), tree)
    return {k: v for k, v in case.items() if k != "name"}


# -- the sequences of a case ------------------------------------------------------------------------
def _part(b, k):
    """Spread over (0, 1] by the golden ratio; the first sequence has all."""
    return 1.0 if b == 0 else (b * 0.6180339887498949 + k * 0.37) % 1.0


def _sequences(case):
    """(new tokens, length with them) of each sequence."""
    new, length = [], []
    for b in range(case["seqs"]):
        n = case["new"]
        if n > 1 and not case.get("tree"):
            n = 1 + int((n - 1) * _part(b, 1))
        length.append(max(n, case["shortest"] + int((case["longest"] - case["shortest"]) * _part(b, 0))))
        new.append(n)
    return new, length


def _history_lengths(case):
    return [max(1, int(case["history"] * _part(r, 0))) for r in range(case["rows"])]


def _parents(n, gen):
    """A drafted tree: each token continues one of the eight drafted before it, or the sequence itself (-1)."""
    back = torch.randint(1, 9, (n,), generator=gen).tolist()
    return [max(-1, j - back[j]) for j in range(n)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=g)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "logits":
        return _prepare_logits(case, seed, g, state)
    dtype, page = _TYPES[case["dtype"]], case["page"]
    new, length = _sequences(case)
    state["new"], state["length"] = new, length  # what the program that schedules the batch knows
    pages = [-(-n // page) for n in length]
    total = sum(pages) + 3  # a pool with some pages that nobody has
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    tables = torch.full((len(new), max(pages)), -1, dtype=torch.int32)
    tables = tables.cuda()
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["tables"] = tables
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["lengths"] = torch.tensor(length, dtype=torch.int32, device="cuda")
    tokens, heads, kv_heads = starts[-1], case["heads"], case["kv_heads"]
    for name in ("keys", "values"):
        state[name] = _randn((total, kv_heads, page, _DIM), dtype, g)
    if case["op"] == "append":
        # a projection's output: heads of different scale
        scale = torch.exp(_randn((1, heads + 2 * kv_heads, 1), torch.float32, g))
        qkv = _randn((tokens, heads + 2 * kv_heads, _DIM), torch.float32, g).mul_(scale)
        state["qkv"] = qkv.to(dtype).view(tokens, -1)
        for name in ("wq", "wk"):
            state[name] = (1 + 0.3 * _randn((_DIM,), torch.float32, g)).to(dtype)
        state["positions"] = torch.cat([torch.arange(n - k, n) for k, n in zip(new, length)]).cuda()
        state["freqs"] = (1e6 ** (-torch.arange(0, _DIM, 2, dtype=torch.float32) / _DIM)).cuda()
        return state
    # heads from diffuse to peaked
    spread = torch.exp2(torch.linspace(-1, 2, heads, device="cuda")).view(1, heads, 1)
    state["q"] = _randn((tokens, heads, _DIM), torch.float32, g).mul_(spread).to(dtype)
    if case["tree"]:
        gen = torch.Generator().manual_seed(seed)
        width = -(-case["new"] // 32)
        words = torch.zeros(tokens, width, dtype=torch.int64)
        for b, n in enumerate(new):
            seen = []
            for j, parent in enumerate(_parents(n, gen)):
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << j)
                for w in range(width):
                    words[starts[b] + j, w] = seen[-1] >> 32 * w & 0xFFFFFFFF
        state["tree"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).cuda()
    return state


def _prepare_logits(case, seed, g, state):
    rows, vocab = case["rows"], case["vocab"]
    x = _randn((rows, vocab), torch.float32, g).mul_(2.5)
    # what has been said is likely to be said again: small ids are frequent ones, as in a tokeniser's order
    history = (torch.rand(rows, case["history"], device="cuda", generator=g) ** 4 * vocab).long().clamp_(max=vocab - 1)
    level = 4 + 6 * torch.rand(vocab, device="cuda", generator=g)
    x.scatter_(1, history, level[history])
    state["logits"] = x.to(_TYPES[case["dtype"]])
    lengths = torch.tensor(_history_lengths(case), dtype=torch.int32, device="cuda")
    if case["penalties"]:
        state["history"], state["lengths"] = history, lengths
        state["prompt_lengths"] = lengths // 3
        state["repetition"] = 1 + 0.3 * torch.rand(rows, device="cuda", generator=g)
        state["presence"] = torch.rand(rows, device="cuda", generator=g)
        state["frequency"] = 0.3 * torch.rand(rows, device="cuda", generator=g)
    if case["biased"]:
        count = case["biased"]
        ids = torch.randperm(vocab, device="cuda", generator=g)[:count].expand(rows, -1)
        state["bias_ids"] = (ids + torch.arange(rows, device="cuda")[:, None]) % vocab
        bias = 3 * _randn((rows, count), torch.float32, g)
        bias[:, 0] = -100.0  # the usual way to ban a token
        state["bias"] = bias
    if case["allowed"] != "all":
        words = -(-vocab // 32)
        keep = 0.003 if case["allowed"] == "few" else 0.9
        bits = torch.rand(rows, words * 32, device="cuda", generator=g) < keep
        bits[:, ::max(1, vocab // 3)] = True  # a grammar allows some token in each state
        weight = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        value = torch.empty(rows, words, dtype=torch.int64, device="cuda")
        for r in range(0, rows, 64):
            value[r:r + 64] = (bits[r:r + 64].view(-1, words, 32) * weight).sum(-1)
        state["allowed"] = torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32)
    return state


# -- the plain forms ------------------------------------------------------------------------------
def _slots(state):
    """(page, row in it) of each new token."""
    page = state["case"]["page"]
    starts = state["starts"].long()
    row = torch.arange(sum(state["new"]), device=starts.device)
    seq = torch.searchsorted(starts[1:], row, right=True)
    at = state["lengths"].long()[seq] - starts[seq + 1] + row
    return state["tables"].long()[seq, at // page], at % page


def _plain_append(state):
    case = state["case"]
    heads, kv_heads, half = case["heads"], case["kv_heads"], _DIM // 2
    dtype = state["keys"].dtype
    x = state["qkv"].float().view(-1, heads + 2 * kv_heads, _DIM)
    # 32 bits leave 0.002 of an angle at position 40000
    angle = state["positions"].double()[:, None] * state["freqs"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotated(part, weight):
        y = part * torch.rsqrt((part * part).mean(dim=-1, keepdim=True) + _EPS) * weight.float()
        low, high = y[..., :half], y[..., half:]
        return torch.cat((low * cos - high * sin, high * cos + low * sin), dim=-1).to(dtype)

    page, row = _slots(state)
    state["keys"][page, :, row] = rotated(x[:, heads:heads + kv_heads], state["wk"])
    state["values"][page, :, row] = state["qkv"].view_as(x)[:, heads + kv_heads:]
    return {"q": rotated(x[:, :heads], state["wq"]), "keys": state["keys"], "values": state["values"]}


def _plain_attend(state):
    case, q = state["case"], state["q"]
    heads, kv_heads, page = case["heads"], case["kv_heads"], case["page"]
    seqs, most, longest = case["seqs"], max(state["new"]), max(state["length"])
    starts, lengths = state["starts"].long(), state["lengths"].long()
    new = starts[1:] - starts[:-1]
    # the sequences side by side, each as long as the longest
    pages = state["tables"][:, :-(-longest // page)].clamp(min=0).long()
    k, v = (state[name][pages].transpose(1, 2).reshape(seqs, kv_heads, -1, _DIM)[:, :, :longest].float()
            for name in ("keys", "values"))
    rows = (starts[:-1, None] + torch.arange(most, device=q.device)).clamp(max=len(q) - 1)
    x = q[rows].float().view(seqs, most, kv_heads, heads // kv_heads, _DIM).transpose(1, 2)
    # which of the new tokens a column is: those before them are negative
    j = torch.arange(longest, device=q.device) - (lengths - new)[:, None]
    if case["tree"]:
        word = (j // 32).clamp(0, state["tree"].shape[1] - 1)[:, None].expand(-1, most, -1)
        bit = state["tree"][rows].gather(2, word) >> (j % 32).int()[:, None] & 1
        seen = (j[:, None] < 0) | (bit == 1) & (j < new[:, None])[:, None]
    else:
        seen = j[:, None] <= torch.arange(most, device=q.device)[:, None]
    s = torch.matmul(x.reshape(seqs, kv_heads, -1, _DIM), k.transpose(2, 3)) / math.sqrt(_DIM)
    s = torch.where(seen[:, None, :, None], s.view(seqs, kv_heads, most, -1, longest), float("-inf"))
    e = (s - s.amax(dim=-1, keepdim=True)).exp()
    o = torch.matmul(e.view(seqs, kv_heads, -1, longest), v) / e.sum(dim=-1).view(seqs, kv_heads, -1, 1)
    row = torch.arange(len(q), device=q.device)
    seq = torch.searchsorted(starts[1:], row, right=True)
    o = o.view(seqs, kv_heads, most, -1, _DIM).transpose(1, 2)[seq, row - starts[seq]]
    return o.reshape(q.shape).to(q.dtype)


def _plain_logits(state):
    case = state["case"]
    x = state["logits"].float()
    rows, vocab = x.shape
    if "history" in state:
        column = torch.arange(case["history"], device=x.device)
        known = column < state["lengths"][:, None]
        output = known & (column >= state["prompt_lengths"][:, None])
        counts = torch.zeros(rows, vocab, device=x.device)
        counts.scatter_add_(1, state["history"], output.float())
        said = torch.zeros(rows, vocab, device=x.device)
        said.scatter_add_(1, state["history"], known.float())
        factor = state["repetition"][:, None]
        x = torch.where(said > 0, torch.where(x > 0, x / factor, x * factor), x)
        x = x - state["frequency"][:, None] * counts - state["presence"][:, None] * (counts > 0)
    if "bias" in state:
        x = x.scatter_add(1, state["bias_ids"], state["bias"])
    if "allowed" in state:
        column = torch.arange(vocab, device=x.device)
        bit = (state["allowed"][:, column // 32] >> (column % 32).int()) & 1
        x = torch.where(bit == 1, x, float("-inf"))
    return x.to(state["logits"].dtype)


# -- the framework's operators --------------------------------------------------------------------
def _own_append(state):
    from tiny_dsv41_b200 import ops

    case = state["case"]
    batch = ops.PagedBatch(state["tables"], state["starts"], state["lengths"])
    q = ops.paged_append(state["qkv"], state["wq"], state["wk"], state["positions"], state["freqs"], case["heads"],
                         case["kv_heads"], _EPS, state["keys"], state["values"], batch)
    return {"q": q, "keys": state["keys"], "values": state["values"]}


def _own_attend(state):
    from tiny_dsv41_b200 import ops

    batch = ops.PagedBatch(state["tables"], state["starts"], state["lengths"])
    return ops.paged_attention(state["q"], state["keys"], state["values"], batch, tree=state.get("tree"))


def _own_logits(state):
    from tiny_dsv41_b200 import ops

    more = {}
    if "history" in state:
        more = {name: state[name] for name in ("lengths", "prompt_lengths", "repetition", "presence", "frequency")}
    return ops.process_logits(state["logits"], state.get("history"), bias_ids=state.get("bias_ids"),
                              bias=state.get("bias"), allowed=state.get("allowed"), **more)


def run(state):
    op = state["case"]["op"]
    with torch.no_grad():
        if own:
            return {"append": _own_append, "attend": _own_attend, "logits": _own_logits}[op](state)
        return {"append": _plain_append, "attend": _plain_attend, "logits": _plain_logits}[op](state)


# -- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        data = 2 * rows * vocab * size + rows * case["biased"] * 12
        if case["allowed"] != "all":
            data += rows * -(-vocab // 32) * 4
        said = sum(_history_lengths(case)) if case["penalties"] else 0
        return {"bytes": data + said * 8 + rows * 20, "flops": rows * vocab + 6 * said}
    new, length = _sequences(case)
    tokens, heads, kv_heads = sum(new), case["heads"], case["kv_heads"]
    if case["op"] == "append":
        wide = (heads + 2 * kv_heads) * _DIM
        return {"bytes": tokens * (2 * wide * size + 8) + 8 * case["seqs"], "flops": 10 * tokens * wide}
    data = 2 * sum(length) * kv_heads * _DIM * size + 2 * tokens * heads * _DIM * size
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, length))  # of a tree, the most that it can have
    if case["tree"]:
        data += tokens * -(-case["new"] // 32) * 4
    return {"bytes": data, "flops": 4 * pairs * heads * _DIM}


# -- the definitions in 64 bits -------------------------------------------------------------------
def _exact_append(case, state):
    new, length, page = state["new"], state["length"], case["page"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    x = state["qkv"].double().reshape(sum(new), -1, _DIM)
    scale = torch.cat((state["wq"].double().expand(heads, _DIM), state["wk"].double().expand(kv_heads, _DIM)))
    y = x[:, :heads + kv_heads]
    y = scale * y / torch.sqrt(y.square().sum(-1, keepdim=True) / _DIM + _EPS)
    # dims i and i + 64 are the parts of a complex number that the position turns
    turn = state["positions"].double()[:, None] * state["freqs"].double()
    z = torch.complex(y[..., :_DIM // 2], y[..., _DIM // 2:]) * torch.polar(torch.ones_like(turn), turn)[:, None]
    y = torch.cat((z.real, z.imag), dim=-1)
    out = {"q": y[:, :heads]}
    keys, values = state["keys"].double(), state["values"].double()
    tables = state["tables"].tolist()
    at = [(tables[b][p // page], p % page) for b, (n, m) in enumerate(zip(new, length)) for p in range(m - n, m)]
    flat = torch.tensor([a * page + r for a, r in at], device=x.device)
    for pool, part in ((keys, y[:, heads:]), (values, x[:, heads + kv_heads:])):
        for h in range(kv_heads):
            rows = pool[:, h].reshape(-1, _DIM)
            rows[flat] = part[:, h]
            pool[:, h] = rows.view(-1, page, _DIM)
    out["keys"], out["values"] = keys, values
    return out


def _exact_attend(case, state):
    heads, kv_heads, page = case["heads"], case["kv_heads"], case["page"]
    result, row = [], 0
    tree = state["tree"].cpu().tolist() if case["tree"] else None
    for b, (n, m) in enumerate(zip(state["new"], state["length"])):
        where = torch.arange(m, device="cuda")
        where = state["tables"][b].long()[where // page] * page + where % page
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        if tree is not None:
            block = [[not tree[row + i][j // 32] >> j % 32 & 1 for j in range(n)] for i in range(n)]
            hidden[:, m - n:] = torch.tensor(block, device="cuda")
        parts = []
        for h in range(heads):
            c = h // (heads // kv_heads)
            k = state["keys"][:, c].reshape(-1, _DIM)[where].double()
            v = state["values"][:, c].reshape(-1, _DIM)[where].double()
            s = (state["q"][row:row + n, h].double() @ k.T * _DIM ** -0.5).masked_fill(hidden, float("-inf"))
            parts.append(torch.softmax(s, dim=1) @ v)
        result.append(torch.stack(parts, dim=1))
        row += n
    return torch.cat(result)


def _exact_logits(case, state):
    vocab = case["vocab"]
    rows = []
    for r, length in enumerate(_history_lengths(case)):
        x = state["logits"][r].double()
        if case["penalties"]:
            ids = state["history"][r, :length]
            said = torch.bincount(ids, minlength=vocab)
            output = torch.bincount(ids[length // 3:], minlength=vocab).double()
            factor = state["repetition"][r].double()
            x = torch.where(said == 0, x, x * torch.where(x < 0, factor, 1 / factor))
            x = x - output * state["frequency"][r].double() - output.clamp(max=1) * state["presence"][r].double()
        if case["biased"]:
            x = x.index_add(0, state["bias_ids"][r], state["bias"][r].double())
        if case["allowed"] != "all":
            bits = state["allowed"][r][:, None].bitwise_right_shift(torch.arange(32, device="cuda").int()) & 1
            x = x.masked_fill(bits.flatten()[:vocab] == 0, float("-inf"))
        rows.append(x)
    return torch.stack(rows)


def exact(case, seed):
    # heads x sequences x (query, key) pairs of 64-bit products beyond this take too long
    if case["op"] == "attend" and work(case)["flops"] > 1e13:
        return None
    state = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[case["op"]](case, state)
