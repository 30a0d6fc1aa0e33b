"""Incremental decoding for Qwen3-MoE: a per-request KV cache
(the native request cache of ``rollout_manager/backends/qwen_kv_cache.py:22-193``), and a paged one for many sequences.

``KVCache`` stores each layer's post-RoPE keys and values and their positions; the attention
module appends the new tokens' entries and attends over everything cached so far (a position-based
causal mask). ``IncrementalLogits`` keeps one request's cache: called with a token sequence that
extends the cached prefix it runs only the new tokens; any other sequence restarts with a prefill.

``PagedKVCache`` holds the sequences of a batch in pages of one pool and runs the decoding operators
(``ops.paged_append``, ``ops.paged_attention``) where the dense cache concatenates and masks; :func:`generate` samples
a batch of prompts over it, with the penalties, biases and masks of ``ops.process_logits``.
"""

from __future__ import annotations

import math
from typing import Callable, NamedTuple, Sequence

import torch

from ... import ops


class KVCache:
    def __init__(self) -> None:
        self.keys: dict[int, torch.Tensor] = {}
        self.values: dict[int, torch.Tensor] = {}
        self.positions: dict[int, torch.Tensor] = {}

    def append(self, layer: int, k, v, positions):
        if layer in self.keys:
            self.keys[layer] = torch.cat((self.keys[layer], k), dim=1)
            self.values[layer] = torch.cat((self.values[layer], v), dim=1)
            self.positions[layer] = torch.cat((self.positions[layer], positions), dim=1)
        else:
            self.keys[layer], self.values[layer], self.positions[layer] = k, v, positions
        return self.keys[layer], self.values[layer], self.positions[layer]


class PagedKVCache:
    """Keys and values of many sequences in pages of one pool, for all layers; pass it as the model's ``cache``.

    :meth:`plan` says which sequences the next forward serves and how many new tokens each brings; the forward takes
    their ids packed as [1, T] with the positions that it returns. bf16 or fp16 on a GPU (any type on the CPU); the whole
    model is on the pool's device."""

    def __init__(self, config, tokens: int, *, page: int = 64, dtype=torch.bfloat16, device=None) -> None:
        pages = -(-tokens // page)
        if tokens < 1:
            raise ValueError("a cache holds at least one token")
        self.pool = torch.empty(config.num_hidden_layers, 2, pages, config.num_key_value_heads, page, config.head_dim,
                                dtype=dtype, device=device)
        self.page = page
        self.free = list(range(pages - 1, -1, -1))
        self.pages: dict[int, list[int]] = {}
        self.lengths: dict[int, int] = {}
        self.batch: ops.PagedBatch | None = None
        self.tree: torch.Tensor | None = None
        self._next = 0

    def add(self) -> int:
        """A new, empty sequence."""
        self._next += 1
        self.pages[self._next], self.lengths[self._next] = [], 0
        return self._next

    def release(self, sequence: int) -> None:
        self.free += reversed(self.pages.pop(sequence))
        del self.lengths[sequence]

    def plan(self, new: Sequence[tuple[int, int]], parents: Sequence[Sequence[int]] | None = None) -> torch.Tensor:
        """The next forward: (sequence, new tokens) of each sequence that it serves. Returns the positions [1, T]. With
        ``parents`` the new tokens of each sequence are a drafted tree (see ``ops.tree_mask``): a token's position is
        its depth behind the sequence, and :meth:`keep` has to follow. Raises, changing nothing, where the pool has
        not enough free pages."""
        if len({s for s, _ in new}) != len(new) or any(n < 0 for _, n in new):
            raise ValueError("a sequence is planned once, with a number of new tokens")
        if parents is not None and [len(p) for p in parents] != [n for _, n in new]:
            raise ValueError("a tree has a parent for each new token")
        if parents is not None and any(not -1 <= parent < j for tree in parents for j, parent in enumerate(tree)):
            raise ValueError("a parent is drafted before its child")
        need = [max(0, -(-(self.lengths[s] + n) // self.page) - len(self.pages[s])) for s, n in new]
        if sum(need) > len(self.free):
            raise RuntimeError(f"the cache is full: {sum(need)} pages are needed and {len(self.free)} free")
        device, positions, starts = self.pool.device, [], [0]
        for i, (s, n) in enumerate(new):
            length = self.lengths[s]
            self.pages[s] += [self.free.pop() for _ in range(need[i])]
            if parents is None:
                positions += range(length, length + n)
            else:
                depth: list[int] = []
                for parent in parents[i]:
                    depth.append(length if parent < 0 else depth[parent] + 1)
                positions += depth
            self.lengths[s] = length + n
            starts.append(starts[-1] + n)
        width = max((len(self.pages[s]) for s, _ in new), default=0)
        tables = [self.pages[s] + [-1] * (width - len(self.pages[s])) for s, _ in new]
        as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.batch = ops.PagedBatch(as_int(tables).view(len(new), width), as_int(starts),
                                    as_int([self.lengths[s] for s, _ in new]))
        self.tree = None
        if parents is not None:
            flat = torch.tensor([p for tree in parents for p in tree], dtype=torch.int64)
            self.tree = ops.tree_mask(flat, torch.tensor(starts)).to(device)
        return torch.tensor(positions, dtype=torch.int64, device=device).unsqueeze(0)

    def attend(self, layer: int, qkv, wq, wk, positions, freqs, hq: int, hkv: int, eps: float) -> torch.Tensor:
        """Attention [T, hq, 128] of a layer's packed projection; its keys and values are appended."""
        keys, values = self.pool[layer, 0], self.pool[layer, 1]
        q = ops.paged_append(qkv, wq, wk, positions, freqs, hq, hkv, eps, keys, values, self.batch)
        return ops.paged_attention(q, keys, values, self.batch, tree=self.tree)

    def _places(self, sequence: int, tokens: Sequence[int]):
        table = self.pages[sequence]
        at = lambda v: torch.tensor(v, dtype=torch.int64, device=self.pool.device)  # noqa: E731
        return at([table[t // self.page] for t in tokens]), at([t % self.page for t in tokens])

    def keep(self, sequence: int, drafted: int, path: Sequence[int]) -> None:
        """Of the last ``drafted`` tokens of a sequence, keeps those of ``path`` (ascending numbers among them, from one
        root to a leaf), in its order, and drops the others."""
        path = list(path)
        if not 0 <= drafted <= self.lengths[sequence]:
            raise ValueError("a sequence keeps tokens that it has")
        if path != sorted(set(path)) or (path and not 0 <= path[0] <= path[-1] < drafted):
            raise ValueError("a path is ascending numbers of drafted tokens")
        first = self.lengths[sequence] - drafted
        moved = [(first + t, first + i) for i, t in enumerate(path) if t != i]
        if moved:  # (read as a whole before any is written)
            page, row = self._places(sequence, [a for a, _ in moved])
            rows = self.pool[:, :, page, :, row]
            page, row = self._places(sequence, [b for _, b in moved])
            self.pool[:, :, page, :, row] = rows
        self.lengths[sequence] = first + len(path)
        used = -(-self.lengths[sequence] // self.page)
        self.free += reversed(self.pages[sequence][used:])
        del self.pages[sequence][used:]


class Generation(NamedTuple):
    """``tokens``: what each prompt was answered with, the end token included; ``log_probs``: of each of them under the
    distribution that it was drawn from."""

    tokens: list[list[int]]
    log_probs: list[list[float]]


@torch.no_grad()
def generate(model, prompts: Sequence[Sequence[int]], max_new_tokens: int, *, temperature: float = 1.0,
             repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0, bias: dict[int, float] | None = None,
             allowed: Callable[[int, list[int]], torch.Tensor] | None = None, eos: Sequence[int] = (),
             generator: torch.Generator | None = None, page: int = 64, chunk: int = 8192) -> Generation:
    """Samples one answer to each prompt, all of them a token a step, over one paged cache.

    Penalties and ``bias`` (token: value) are those of ``ops.process_logits``; ``allowed(i, answer)`` gives the int32
    words of the tokens that may follow answer ``i`` (a grammar). ``temperature`` 0 takes the most likely token. Prompts
    are read ``chunk`` tokens at a time. Draws come from a CPU ``generator``, one per sequence and step, in order."""
    config, weight = model.config, model.lm_head.weight
    if not prompts or any(not p for p in prompts):
        raise ValueError("generate needs prompts of at least one token")
    if max_new_tokens < 1 or chunk < 1:
        raise ValueError("max_new_tokens and chunk must be positive")
    if not (math.isfinite(temperature) and temperature >= 0):
        raise ValueError("temperature must be finite and not negative")
    if any(not 0 <= t < config.vocab_size for part in (*prompts, bias or ()) for t in part):
        raise ValueError("prompts and biases hold tokens of the vocabulary")
    if any(len(p) + max_new_tokens > config.max_position_embeddings for p in prompts):
        raise ValueError("a prompt and its answer are longer than max_position_embeddings")
    device, chunk = weight.device, min(chunk, config.max_position_embeddings)
    most = [len(p) + max_new_tokens for p in prompts]
    cache = PagedKVCache(config, sum(-(-n // page) * page for n in most), page=page, dtype=weight.dtype, device=device)
    sequences = [cache.add() for _ in prompts]
    history = torch.full((len(prompts), max(most)), -1, dtype=torch.int64)
    for i, p in enumerate(prompts):
        history[i, :len(p)] = torch.tensor(p)
    history = history.to(device)
    prompt_lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)
    answers: list[list[int]] = [[] for _ in prompts]
    log_probs: list[list[float]] = [[] for _ in prompts]

    def forward(part: list[tuple[int, Sequence[int]]]) -> torch.Tensor:
        """The last hidden state of each (prompt, new tokens)."""
        positions = cache.plan([(sequences[i], len(t)) for i, t in part])
        ids = torch.tensor([[x for _, t in part for x in t]], dtype=torch.int64, device=device)
        hidden = model.model(ids, None, positions, cache=cache).last_hidden_state[0]
        return hidden[cache.batch.starts[1:].long() - 1]

    last: dict[int, torch.Tensor] = {}
    pieces = [(i, p[a:a + chunk]) for i, p in enumerate(prompts) for a in range(0, len(p), chunk)]
    while pieces:
        part, room = [], chunk
        while pieces and len(pieces[0][1]) <= room and pieces[0][0] not in [i for i, _ in part]:
            room -= len(pieces[0][1])
            part.append(pieces.pop(0))
        for (i, _), h in zip(part, forward(part)):
            last[i] = h
    running = list(range(len(prompts)))
    hidden = torch.stack([last[i] for i in running])
    for step in range(max_new_tokens):
        rows = torch.tensor(running, device=device)
        more = {}
        if bias:
            more["bias_ids"] = torch.tensor(list(bias), dtype=torch.int64, device=device)
            more["bias"] = torch.tensor(list(bias.values()), dtype=torch.float32, device=device)
        if allowed is not None:
            more["allowed"] = torch.stack([allowed(i, answers[i]) for i in running]).to(device)
        logits = ops.process_logits(model.lm_head(hidden), history[rows], lengths=prompt_lengths[rows] + step,
                                    prompt_lengths=prompt_lengths[rows], repetition=repetition, presence=presence,
                                    frequency=frequency, **more)
        if temperature == 0:
            tokens = logits.float().argmax(-1)
        else:
            p = torch.softmax(logits.float() / temperature, dim=-1).cpu()
            tokens = torch.multinomial(p, 1, generator=generator).squeeze(1).to(device)
        scores = ops.token_statistics(logits, tokens, temperature=temperature or 1.0).log_probs
        history[rows, prompt_lengths[rows].long() + step] = tokens
        going = []
        for i, token, score in zip(running, tokens.tolist(), scores.tolist()):
            answers[i].append(token)
            log_probs[i].append(score)
            if token in eos:
                cache.release(sequences[i])
            else:
                going.append(i)
        running = going
        if not running or step + 1 == max_new_tokens:
            break
        hidden = forward([(i, answers[i][-1:]) for i in running])
    return Generation(answers, log_probs)


class IncrementalLogits:
    """Next-token logits for a growing single sequence, reusing the cache across calls.

    ``paged`` (tokens) keeps it in a ``PagedKVCache`` of that size, whose attention runs the decoding kernels, in place
    of the dense cache and cuDNN's masked attention."""

    def __init__(self, model, *, paged: int = 0) -> None:
        self.model = model  # Qwen3MoeForCausalLM
        self.paged = paged
        self.ids: list[int] = []
        self.cache: KVCache | None = None
        self.prefills = 0

    def _empty(self, device):
        if not self.paged:
            return KVCache()
        cache = PagedKVCache(self.model.config, self.paged, dtype=self.model.lm_head.weight.dtype, device=device)
        cache.add()
        return cache

    @torch.no_grad()
    def __call__(self, input_ids: torch.Tensor) -> torch.Tensor:
        if input_ids.ndim != 2 or input_ids.shape[0] != 1:
            raise ValueError("incremental decoding serves one sequence")
        ids = input_ids[0].tolist()
        if self.cache is None or len(ids) <= len(self.ids) or ids[:len(self.ids)] != self.ids:
            self.cache, self.ids, new = self._empty(input_ids.device), [], ids
            self.prefills += 1
        else:
            new = ids[len(self.ids):]
        start, cache = len(self.ids), self.cache
        self.cache = None  # (a forward that fails leaves a cache of no use)
        tokens = torch.tensor([new], dtype=torch.long, device=input_ids.device)
        if self.paged:
            positions = cache.plan([(1, len(new))])
        else:
            positions = torch.arange(start, start + len(new), device=input_ids.device).unsqueeze(0)
        inner = self.model.model
        hidden = inner(tokens, None, positions, cache=cache).last_hidden_state
        self.ids, self.cache = ids, cache
        return self.model.lm_head(hidden[:, -1:])[:, -1]


__all__ = ["Generation", "IncrementalLogits", "KVCache", "PagedKVCache", "generate"]
