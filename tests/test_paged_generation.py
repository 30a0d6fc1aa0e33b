"""Decoding over the paged cache: the append, the attention and the processed logits in the order in which a step of the
model calls them, against the model without a cache."""

import pytest
import torch

from tiny_dsv41_b200 import ops
from tiny_dsv41_b200.models.qwen import Qwen3MoeConfig, Qwen3MoeForCausalLM
from tiny_dsv41_b200.models.qwen.generation import IncrementalLogits, PagedKVCache, generate

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    if torch.cuda.is_available():
        ops.check_status("test")


def _model(device, seed=4):
    torch.manual_seed(seed)
    config = Qwen3MoeConfig.tiny(num_hidden_layers=2, vocab_size=512)
    model = Qwen3MoeForCausalLM(config).eval()
    return model.cuda().to(torch.bfloat16) if device == "cuda" else model


def _same(a, b, device):
    """Logits of the two paths: fp32 on the CPU (sums of some hundred products, a few layers deep); bf16 on the GPU, where
    each path rounds its own activations (as between the dense cache and the full forward)."""
    error = float((a.float() - b.float()).norm() / b.float().norm())
    assert error < (1e-4 if device == "cpu" else 2e-2), error


@torch.no_grad()
def _full(model, ids):
    return model(torch.tensor([ids], device=model.lm_head.weight.device)).logits[0]


class _Rows:
    """Compares the rows of the two paths where both send the token, and all before it, to the same experts.

    The choice of two experts is a step function: where the second and third are close, the rounding of the activations
    decides, and the two paths may differ by an expert. Entering the gate with a relative error of 2e-2 at most (what is
    allowed here), norm 16 (256 normalised values) against rows of norm 0.32 (std 0.02), a router logit is off by 0.1 at
    most and a margin by 0.2: a choice that differs with a larger margin is an error."""

    def __init__(self, model, device):
        self.model, self.device, self.off = model, device, {}

    def __call__(self, sequence, ids, logits, router_logits, at):
        """Rows [at, at + n) of the packed call against the last n of the full forward of `ids`."""
        n = len(logits)
        with torch.no_grad():
            full = self.model(torch.tensor([ids], device=logits.device), output_router_logits=True)
        off = self.off.setdefault(sequence, set())
        for mine, theirs in zip(router_logits, full.router_logits):
            theirs = theirs[len(ids) - n:].float()
            top = theirs.topk(3, dim=-1)
            own = mine[at:at + n].float().topk(3, dim=-1)
            differs = (own.indices[:, :2].sort(-1).values != top.indices[:, :2].sort(-1).values).any(-1)
            # (of two that round to one value, either may be taken)
            differs |= (top.values[:, 1] == top.values[:, 2]) | (own.values[:, 1] == own.values[:, 2])
            assert bool((top.values[:, 1] - top.values[:, 2])[differs].le(0.2).all())
            off |= {len(ids) - n + i for i in differs.nonzero().flatten().tolist()}
        stable = [i for i in range(n) if not any(t <= len(ids) - n + i for t in off)]
        if self.device == "cpu":
            assert len(stable) == n
        for i in stable:
            _same(logits[i], full.logits[0, len(ids) - n + i], self.device)
        return len(stable)


@pytest.mark.parametrize("device", DEVICES)
def test_incremental_logits_over_pages(device):
    model, ids = _model(device), [1, 17, 33, 250, 9, 77, 3]
    inc = IncrementalLogits(model, paged=128)
    for _ in range(5):
        logits = inc(torch.tensor([ids], device=model.lm_head.weight.device))
        want = _full(model, ids)[-1:]
        _same(logits, want, device)
        ids.append(int(want.argmax()))
    assert inc.prefills == 1
    inc(torch.tensor([[5, 6]], device=model.lm_head.weight.device))
    assert inc.prefills == 2
    with pytest.raises(RuntimeError, match="full"):
        inc(torch.tensor([[7] * 129], device=model.lm_head.weight.device))
    _same(inc(torch.tensor([[5, 6]], device=model.lm_head.weight.device)), _full(model, [5, 6])[-1:], device)


@pytest.mark.parametrize("device", DEVICES)
@torch.no_grad()
def test_a_batch_of_sequences_step_by_step(device):
    """Sequences of different lengths, one of them idle for a step, one released and its pages taken by another."""
    model = _model(device)
    where = model.lm_head.weight.device
    cache = PagedKVCache(model.config, 160, page=16, dtype=model.lm_head.weight.dtype, device=where)
    gen = torch.Generator().manual_seed(0)
    ids = {cache.add(): torch.randint(0, 512, (n,), generator=gen).tolist() for n in (1, 40, 17)}

    rows, compared = _Rows(model, device), 0

    def step(new):
        nonlocal compared
        positions = cache.plan([(s, len(t)) for s, t in new.items()])
        tokens = torch.tensor([[t for part in new.values() for t in part]], device=where)
        out = model.model(tokens, None, positions, cache=cache, output_router_logits=True)
        logits, at = model.lm_head(out.last_hidden_state)[0], 0
        for s, t in new.items():
            compared += rows(s, ids[s], logits[at:at + len(t)], out.router_logits, at)
            at += len(t)

    step(dict(ids))
    a, b, c = ids
    for new in ({a: [3], b: [4], c: [5]}, {a: [8, 9, 10], c: [2]}, {b: [1] * 20, a: [7]}):
        for s, t in new.items():
            ids[s] = ids[s] + t
        step(new)
    cache.release(b)
    del ids[b]
    d = cache.add()
    ids[d] = torch.randint(0, 512, (90,), generator=gen).tolist()
    step({d: ids[d]})
    with pytest.raises(RuntimeError, match="full"):
        cache.plan([(a, 100)])
    ids[a] = ids[a] + [11]
    step({a: [11]})  # (the refused plan has changed nothing)
    assert compared >= 20  # (a twentieth of the choices is close: a prefix of some ten rows of each sequence)


@pytest.mark.parametrize("device", DEVICES)
@torch.no_grad()
def test_a_drafted_tree_and_the_path_kept(device):
    """Each drafted token's logits are those after its own path; the kept path goes on as if it had been fed."""
    model = _model(device)
    where = model.lm_head.weight.device
    cache = PagedKVCache(model.config, 256, page=16, dtype=model.lm_head.weight.dtype, device=where)
    gen = torch.Generator().manual_seed(1)
    ids = {cache.add(): torch.randint(0, 512, (n,), generator=gen).tolist() for n in (30, 9)}
    positions = cache.plan([(s, len(t)) for s, t in ids.items()])
    out = model.model(torch.tensor([sum(ids.values(), [])], device=where), None, positions, cache=cache,
                      output_router_logits=True)
    rows, compared, at = _Rows(model, device), 0, 0
    logits = model.lm_head(out.last_hidden_state)[0]
    for s, t in ids.items():
        compared += rows(s, t, logits[at:at + len(t)], out.router_logits, at)
        at += len(t)
    parents = [[-1, 0, 0, 1, 2, 4, -1, 6, 3], [-1, -1, 0, 2, 3]]
    drafts = [torch.randint(0, 512, (len(p),), generator=gen).tolist() for p in parents]
    positions = cache.plan([(s, len(p)) for s, p in zip(ids, parents)], parents)
    out = model.model(torch.tensor([sum(drafts, [])], device=where), None, positions, cache=cache, output_router_logits=True)
    logits, at = model.lm_head(out.last_hidden_state)[0], 0
    for s, tree, tokens in zip(ids, parents, drafts):
        before = set(rows.off[s])
        off = [set() for _ in tree]  # along each token's path
        for j in range(len(tree)):
            path, k = [], j
            while k >= 0:
                path.insert(0, tokens[k])
                k = tree[k]
            rows.off[s] = before | (off[tree[j]] if tree[j] >= 0 else set())
            compared += rows(s, ids[s] + path, logits[at + j:at + j + 1], out.router_logits, at + j)
            off[j] = rows.off[s] - before
        rows.off[s] = before | (off[5] if len(tree) == 9 else set())
        at += len(tree)
    a, b = ids
    cache.keep(a, 9, [0, 2, 4, 5])
    ids[a] = ids[a] + [drafts[0][j] for j in (0, 2, 4, 5)]
    cache.keep(b, 5, [])
    assert cache.lengths == {a: 34, b: 9} and len(cache.pages[b]) == 1
    for s in ids:
        ids[s] = ids[s] + [77, 78]
    positions = cache.plan([(a, 2), (b, 2)])
    out = model.model(torch.tensor([[77, 78, 77, 78]], device=where), None, positions, cache=cache, output_router_logits=True)
    logits = model.lm_head(out.last_hidden_state)[0]
    compared += rows(a, ids[a], logits[:2], out.router_logits, 0) + rows(b, ids[b], logits[2:], out.router_logits, 2)
    assert compared >= 20


def test_cache_refusals():
    config = Qwen3MoeConfig.tiny()
    cache = PagedKVCache(config, 64, page=16, dtype=torch.float32)
    s = cache.add()
    cache.plan([(s, 20)])
    for bad in ((s, 21, [0]), (s, 3, [2, 1]), (s, 3, [1, 1]), (s, 3, [3]), (s, 3, [-1])):
        with pytest.raises(ValueError):
            cache.keep(*bad)
    with pytest.raises(ValueError):
        cache.plan([(s, 1), (s, 1)])
    with pytest.raises(ValueError):
        cache.plan([(s, 2)], [[-1]])
    with pytest.raises(ValueError, match="before its child"):
        cache.plan([(s, 2)], [[-1, 1]])
    with pytest.raises(KeyError):
        cache.plan([(99, 1)])
    assert cache.lengths == {s: 20}
    with pytest.raises(ValueError):
        PagedKVCache(config, 0)
    cache.release(s)
    assert sorted(cache.free) == [0, 1, 2, 3] and not cache.pages


def _definition(x, prompt, answer, repetition, presence, frequency, bias, keep):
    """One row of processed logits, token by token."""
    x = x.double().clone()
    for t in set(prompt + answer):
        x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
    for t in set(answer):
        x[t] -= frequency * answer.count(t) + presence
    for t, v in bias.items():
        x[t] += v
    return x if keep is None else x.masked_fill(~keep, float("-inf"))


def test_generation_takes_the_most_likely_tokens():
    """Greedy answers with penalties, biases and a grammar are those of the full forward, token by token."""
    model = _model("cpu")
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 512, (n,), generator=gen).tolist() for n in (3, 25, 1)]
    bias = {7: 0.05, 500: -100.0}
    grammar = torch.rand(3, 512, generator=gen) < 0.5

    def allowed(i, answer):
        bits = grammar[(i + len(answer)) % 3].view(16, 32).long() << torch.arange(32)
        words = bits.sum(-1)
        return torch.where(words >= 1 << 31, words - (1 << 32), words).int()

    got = generate(model, prompts, 6, temperature=0, repetition=1.3, presence=0.02, frequency=0.01, bias=bias, allowed=allowed,
                   chunk=10)
    for i, prompt in enumerate(prompts):
        answer = []
        for step in range(6):
            x = _definition(_full(model, prompt + answer)[-1], prompt, answer, 1.3, 0.02, 0.01, bias, grammar[(i + step) % 3])
            answer.append(int(x.argmax()))
            assert got.log_probs[i][step] == pytest.approx(float(torch.log_softmax(x, 0)[answer[-1]]), abs=1e-4)
        assert got.tokens[i] == answer


@pytest.mark.parametrize("device", DEVICES)
def test_generation_ends_and_repeats(device):
    """The same draws twice, answers that end at the end token, its log-probability included."""
    model = _model(device)
    prompts = [[1, 2, 3], [4], list(range(40))]
    runs = [generate(model, prompts, 12, temperature=0.8, eos=range(0, 512, 9), generator=torch.Generator().manual_seed(2))
            for _ in range(2)]
    assert runs[0] == runs[1]
    for tokens, scores in zip(*runs[0]):
        assert 1 <= len(tokens) == len(scores) <= 12
        assert all(t % 9 for t in tokens[:-1]) and (tokens[-1] % 9 == 0 or len(tokens) == 12)
        assert all(s <= 0 for s in scores)
    for bad in ((model, [], 3), (model, [[]], 3), (model, prompts, 0), (model, prompts, 5000), (model, [[512]], 3),
                (model, [[-1]], 3)):
        with pytest.raises(ValueError):
            generate(*bad)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(bias={512: 1.0})):
        with pytest.raises(ValueError):
            generate(model, prompts, 3, **kw)
