"""The operators of a decoding step over a paged cache of keys and values.

* :func:`paged_append` - norms and position rotation of the new tokens' queries and keys, keys and values written
  to their pages (``qk_norm_rope`` with a cache to write to);
* :func:`paged_attention` - attention of the new tokens over the cache, causal or under the mask of a tree of
  drafted tokens (:func:`tree_mask` makes one from the tree's parents);
* :func:`process_logits` - penalties for repeated tokens, biases and a grammar's mask on the logits.

A :class:`PagedBatch` says which sequences a call serves and where their tokens lie. It holds tensors on the GPU that
no call reads back to the host, so a step may be captured into a CUDA graph and replayed after the tensors were filled
anew. The operators serve and sample: they have no gradients, and refuse inputs that want one.

The reference keeps one dense cache a request (``rollout_manager/backends/qwen_kv_cache.py:22-193``) and samples from
unprocessed logits (``dsv41_train/rl/rollout.py``).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from ._ext import ext

HEAD_DIM = 128
MIN_PAGE = 16
_TYPES = (torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class PagedBatch:
    """The sequences of a call.

    ``tables`` int32 [sequences, pages]: the page of the cache that holds each stretch of a sequence (entries behind its
    length are not read); ``starts`` int32 [sequences + 1]: sequence ``b`` brings the rows ``starts[b]`` to
    ``starts[b + 1]`` of the call (none, one or many; rows from the last start on belong to no sequence);
    ``lengths`` int32 [sequences]: its tokens in the cache, the new ones included, so that row ``i`` of ``n`` lies at
    place ``length - n + i``."""

    tables: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor

    def __post_init__(self) -> None:
        for name in ("tables", "starts", "lengths"):
            value = getattr(self, name)
            if value.dtype != torch.int32:
                raise TypeError(f"{name} must be int32")
            if value.device != self.tables.device:
                raise ValueError("tables, starts and lengths must be on one device")
        if self.tables.ndim != 2 or self.lengths.shape != self.tables.shape[:1] or self.starts.shape != (
                self.tables.shape[0] + 1,):
            raise ValueError("a batch is tables [sequences, pages], starts [sequences + 1] and lengths [sequences]")


def _check_cache(keys: torch.Tensor, values: torch.Tensor, batch: PagedBatch) -> None:
    if keys.ndim != 4 or keys.shape[-1] != HEAD_DIM or keys.shape != values.shape:
        raise ValueError(f"keys and values must both be [pages, heads, page, {HEAD_DIM}]")
    page = keys.shape[2]
    if page < MIN_PAGE or page & (page - 1):
        raise ValueError(f"a page holds a power of two of tokens, {MIN_PAGE} or more")
    if keys.shape[0] < 1 or keys.shape[1] < 1:
        raise ValueError("a cache has at least one page and one head")
    if keys.dtype != values.dtype or values.device != keys.device:
        raise ValueError("keys and values must be of one type and on one device")
    if keys.is_cuda and keys.dtype not in _TYPES:
        raise TypeError("a cache on a GPU is bf16 or fp16")
    if not keys.dtype.is_floating_point:
        raise TypeError("a cache holds floating-point values")
    if batch.tables.device != keys.device:
        raise ValueError("the batch must be on the cache's device")


def _refuse_gradients(what: str, *tensors: torch.Tensor | None) -> None:
    # (forward-mode tangents exist inside a level alone; asking each tensor for one costs a microsecond)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) or (
            getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                                   for t in tensors)):
        raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad() or with detached tensors")


def _dense(x: torch.Tensor, bytes_: int) -> torch.Tensor:
    """``x``, or a copy where it is strided or starts inside a unit of that many bytes."""
    x = x.contiguous()
    return x if x.data_ptr() % bytes_ == 0 else x.clone()


# -- the plain restatement (CPU) --------------------------------------------------------------------
def _sequences(batch: PagedBatch, rows: int, page: int, pages: int):
    """(first row, new tokens, pool row of each cached token) of each sequence."""
    starts, lengths, tables = batch.starts.tolist(), batch.lengths.tolist(), batch.tables.long()
    for b, length in enumerate(lengths):
        first, n = starts[b], starts[b + 1] - starts[b]
        if first < 0 or n < 0 or starts[b + 1] > rows or not n <= length <= tables.shape[1] * page:
            raise ValueError(f"sequence {b} of the batch does not fit: {n} new tokens, length {length}")
        used = tables[b, :-(-length // page)]
        if bool(((used < 0) | (used >= pages)).any()):
            raise ValueError(f"sequence {b} of the batch has a page outside the cache")
        at = torch.arange(length)
        yield first, n, tables[b][at // page] * page + at % page


def _append_reference(qkv, wq, wk, positions, freqs, hq, hkv, eps, keys, values, batch):
    wide = torch.promote_types(qkv.dtype, torch.float32)
    x = qkv.to(wide).view(-1, hq + 2 * hkv, HEAD_DIM)
    angles = positions.double().unsqueeze(-1) * freqs.double()
    cos, sin = (f(angles).to(wide).unsqueeze(1) for f in (torch.cos, torch.sin))

    def rotated(part, weight):
        part = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + eps) * weight.to(wide)
        low, high = part.chunk(2, dim=-1)
        return torch.cat((low * cos - high * sin, high * cos + low * sin), dim=-1).to(qkv.dtype)

    q, k, v = rotated(x[:, :hq], wq), rotated(x[:, hq:hq + hkv], wk), qkv.view(x.shape)[:, hq + hkv:]
    page = keys.shape[2]
    for first, n, at in _sequences(batch, len(x), page, keys.shape[0]):
        at = at[len(at) - n:]
        keys[at // page, :, at % page] = k[first:first + n]
        values[at // page, :, at % page] = v[first:first + n]
    return q


def _attention_reference(q, keys, values, batch, scale, tree):
    wide = torch.promote_types(q.dtype, torch.float32)
    out = torch.zeros_like(q)
    group, page = q.shape[1] // keys.shape[1], keys.shape[2]
    for first, n, at in _sequences(batch, len(q), page, keys.shape[0]):
        if n == 0:
            continue
        # [heads, tokens, dim]
        k, v = (pool[at // page, :, at % page].to(wide).transpose(0, 1).repeat_interleave(group, 0)
                for pool in (keys, values))
        x = torch.arange(len(at)) - (len(at) - n)
        if tree is None:
            seen = x <= torch.arange(n).unsqueeze(1)
        else:
            words = torch.nn.functional.pad(tree[first:first + n], (0, 1))  # (what lies behind the words is not seen)
            word = (x // 32).clamp(0, tree.shape[1])
            seen = (x < 0) | ((words[:, word] >> (x % 32).int()) & 1 == 1)
        s = q[first:first + n].to(wide).transpose(0, 1) @ k.transpose(1, 2) * scale
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
        total = p.sum(-1, keepdim=True)
        o = torch.where(total == 0, torch.zeros_like(total), 1 / total) * (p @ v)
        out[first:first + n] = o.transpose(0, 1).to(q.dtype)
    return out


def _process_reference(x, history, lengths, prompt_lengths, repetition, presence, frequency, bias_ids, bias, allowed):
    rows, vocab = x.shape
    dtype, x = x.dtype, x.to(torch.promote_types(x.dtype, torch.float32), copy=True)
    column = lambda v: v.to(x.dtype).unsqueeze(1)  # noqa: E731
    if history is not None:
        place = torch.arange(history.shape[1]).expand(rows, -1)
        known = history >= 0
        if lengths is not None:
            if bool(((lengths < 0) | (lengths > history.shape[1])).any()):
                raise ValueError("a length beyond the history")
            known = known & (place < lengths.unsqueeze(1))
        if bool((known & (history >= vocab)).any()):
            raise ValueError("history id outside the vocabulary")
        output = known if prompt_lengths is None else known & (place >= prompt_lengths.unsqueeze(1))
        at = torch.where(known, history, 0).long()
        said = torch.zeros(rows, vocab, dtype=torch.int64).scatter_add_(1, at, known.long()) > 0
        times = torch.zeros(rows, vocab, dtype=torch.int64).scatter_add_(1, at, output.long())
        r = column(repetition)
        x = torch.where(said, torch.where(x > 0, x / r, x * r), x)
        x = torch.where(times > 0, x - column(frequency) * times - column(presence), x)
    if bias_ids is not None:
        if bool((bias_ids >= vocab).any()):
            raise ValueError("bias id outside the vocabulary")
        there = bias_ids >= 0
        x = x + torch.zeros_like(x).scatter_add_(1, torch.where(there, bias_ids, 0),
                                                 torch.where(there, bias, 0.0).to(x.dtype))
    if allowed is not None:
        token = torch.arange(vocab)
        x = x.masked_fill((allowed[:, token // 32] >> (token % 32).int()) & 1 == 0, float("-inf"))
    return x.to(dtype)


# -- the operators ----------------------------------------------------------------------------------
def paged_append(qkv: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
                 hq: int, hkv: int, eps: float, keys: torch.Tensor, values: torch.Tensor,
                 batch: PagedBatch) -> torch.Tensor:
    """Queries [T, hq, 128] of the packed projection ``qkv`` [..., (hq + 2 hkv) 128] with T rows, normalised for each head
    with ``wq`` and rotated to ``positions`` (int64, one per row; ``freqs`` fp32 [64]); the keys, normalised with ``wk``
    and rotated, and the values are written to their places in the cache ``keys`` / ``values``
    [pages, hkv, page, 128].

    The cache may be strided between pages, heads and rows (a slice of a pool for all layers). Everything is computed
    in fp32 from an angle reduced in 64 bits, and rounded once. A row's place in the cache is its sequence's, whatever
    its position is (the tokens of a drafted tree share positions). Rows behind the last sequence are not stored; their
    queries are computed like the others'. bf16 or fp16 on a GPU. There, a sequence of the batch that does not fit its
    table, or a page outside the cache, sets the device status (``ops.check_status``) and is not stored; on the CPU it
    raises. Two rows with the same place leave either."""
    _check_cache(keys, values, batch)
    if hq < 1 or hkv != keys.shape[1] or qkv.ndim < 1 or qkv.shape[-1] != (hq + 2 * hkv) * HEAD_DIM:
        raise ValueError("qkv must be [..., (hq + 2 hkv) 128] with the cache's hkv heads")
    if wq.shape != (HEAD_DIM,) or wk.shape != (HEAD_DIM,) or freqs.shape != (HEAD_DIM // 2,):
        raise ValueError("wq and wk must hold 128 values, freqs 64")
    if not (qkv.dtype == wq.dtype == wk.dtype == keys.dtype):
        raise TypeError("qkv, norm weights and cache must be of one type")
    if positions.dtype != torch.int64 or freqs.dtype != torch.float32:
        raise TypeError("positions must be int64 and freqs fp32")
    flat = qkv.reshape(-1, qkv.shape[-1])
    if positions.numel() != len(flat):
        raise ValueError("positions must hold one value per row")
    if any(t.device != keys.device for t in (qkv, wq, wk, positions, freqs)):
        raise ValueError("all tensors must be on the cache's device")
    _refuse_gradients("paged_append", qkv, wq, wk, freqs, keys, values)
    positions = positions.reshape(-1)
    if not keys.is_cuda:
        return _append_reference(flat, wq, wk, positions, freqs, hq, hkv, eps, keys, values, batch)
    if flat.stride(1) != 1 or flat.stride(0) % 8 or flat.data_ptr() % 16:
        flat = _dense(flat, 16)
    return ext().paged_append(flat, wq.contiguous(), wk.contiguous(), positions.contiguous(), freqs.contiguous(), hq,
                              float(eps), keys, values, *_batch_tensors(batch))


def _batch_tensors(batch: PagedBatch):
    tables = batch.tables
    if tables.shape[1] > 1 and tables.stride(1) != 1:
        tables = tables.contiguous()
    return tables, batch.starts.contiguous(), batch.lengths.contiguous()


def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, batch: PagedBatch, *,
                    scale: float | None = None, tree: torch.Tensor | None = None) -> torch.Tensor:
    """Attention [T, hq, 128] of the queries ``q`` [T, hq, 128] of the batch's new tokens over the cache ``keys`` /
    ``values`` [pages, hkv, page, 128], in which their own keys and values are already (:func:`paged_append`);
    hq is a multiple of hkv, whose heads are shared by consecutive queries. ``scale`` is 1 / sqrt(128) by default.

    A token sees the tokens of its sequence up to itself. With ``tree`` (int32 [T, words], see :func:`tree_mask`) it sees
    those before the new tokens, and of the new ones those whose bit is set in its row: bit ``j % 32`` of word ``j // 32``
    for the sequence's new token ``j`` (tokens behind the words are not seen). A row that sees nothing, and a row behind
    the last sequence, is zero. What the cache holds behind a sequence's length is of no effect, whatever it is; the
    sequence's own keys and values have to be finite.

    bf16 or fp16 on a GPU, sums in fp32. The same call on the same inputs gives the same bits. There, a sequence that
    does not fit its table gives zeros, a page outside the cache a result without meaning, and either sets the device
    status (``ops.check_status``); on the CPU it raises."""
    _check_cache(keys, values, batch)
    if q.ndim != 3 or q.shape[2] != HEAD_DIM or q.shape[1] < 1 or q.shape[1] % keys.shape[1]:
        raise ValueError("q must be [rows, heads, 128] with a multiple of the cache's heads")
    if q.dtype != keys.dtype:
        raise TypeError("q and the cache must be of one type")
    if q.device != keys.device or (tree is not None and tree.device != q.device):
        raise ValueError("all tensors must be on the cache's device")
    if tree is not None and tree.dtype != torch.int32:
        raise TypeError("tree must be int32")
    if tree is not None and (tree.ndim != 2 or len(tree) != len(q)):
        raise ValueError("tree must be [rows, words]")
    scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale)
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError("scale must be finite and positive")
    _refuse_gradients("paged_attention", q, keys, values)
    if not keys.is_cuda:
        return _attention_reference(q, keys, values, batch, scale, tree)
    return ext().paged_attention(_dense(q, 16), keys, values, *_batch_tensors(batch), scale,
                                 None if tree is None else tree.contiguous())


def tree_mask(parents: torch.Tensor, starts: torch.Tensor, words: int | None = None) -> torch.Tensor:
    """The ``tree`` of :func:`paged_attention` from each drafted token's parent: ``parents`` int64 [T] counts within the
    sequence and is less than the token's own number there, -1 for one that continues the sequence itself; ``starts`` is
    the batch's. A token sees its ancestors and itself. ``words`` (by default as many as the largest tree needs) is
    the width of the result; rows behind the last sequence are zero. Reads both tensors on the host."""
    if parents.ndim != 1 or parents.dtype != torch.int64:
        raise TypeError("parents must be int64, one per row")
    first = starts.tolist()
    if len(first) < 1 or any(b < a for a, b in zip(first, first[1:])) or first[0] < 0 or first[-1] > len(parents):
        raise ValueError("starts must rise from 0 to at most the rows")
    most = max((b - a for a, b in zip(first, first[1:])), default=0)
    words = max(1, -(-most // 32)) if words is None else words
    if words * 32 < most:
        raise ValueError("a tree has more tokens than the words have bits")
    given = parents.tolist()
    rows = [[0] * words for _ in given]
    for a, b in zip(first, first[1:]):
        for j in range(b - a):
            parent = given[a + j]
            if not -1 <= parent < j:
                raise ValueError("a parent is drafted before its child")
            if parent >= 0:
                rows[a + j] = list(rows[a + parent])
            rows[a + j][j // 32] |= 1 << j % 32
    signed = [[w - (1 << 32) if w >> 31 else w for w in row] for row in rows]
    return torch.tensor(signed, dtype=torch.int32, device=parents.device).view(len(given), words)


def _per_row(value, name: str, logits: torch.Tensor, default: float) -> tuple[torch.Tensor | None, float]:
    """A penalty as fp32 values, one per row, or as a number for all rows."""
    if value is None:
        return None, default
    if isinstance(value, torch.Tensor):
        if value.shape != logits.shape[:-1] or value.device != logits.device or not value.is_floating_point():
            raise ValueError(f"{name} must be a number, or hold one per row on the logits' device")
        if value.dtype != torch.float32 or value.ndim != 1 or not value.is_contiguous():
            value = value.detach().float().reshape(-1).contiguous()
        return value, default
    value = float(value)
    if not math.isfinite(value) or (name == "repetition" and value <= 0):
        raise ValueError(f"{name} must be finite" + (" and positive" if name == "repetition" else ""))
    return None, value


def _rows_of(value: torch.Tensor, name: str, types, logits: torch.Tensor) -> torch.Tensor:
    """[rows, size] of a table whose leading dimensions are the logits', or one or none for all rows."""
    if value.dtype not in types:
        raise TypeError(f"{name} must be {' or '.join(str(t).removeprefix('torch.') for t in types)}")
    if value.device != logits.device:
        raise ValueError(f"{name} must be on the logits' device")
    lead = logits.shape[:-1]
    if len(lead) == 1 and value.ndim == 2 and value.shape[0] == lead[0] and value.is_contiguous():
        return value
    try:
        value = value.expand(*lead, value.shape[-1])
    except (RuntimeError, IndexError):
        raise ValueError(f"{name} must be [..., size] over the logits' rows") from None
    value = value.reshape(lead.numel(), value.shape[-1])
    return value if value.shape[1] <= 1 or value.stride(1) == 1 else value.contiguous()


def process_logits(logits: torch.Tensor, history: torch.Tensor | None = None, *, lengths: torch.Tensor | None = None,
                   prompt_lengths: torch.Tensor | None = None, repetition=None, presence=None, frequency=None,
                   bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   allowed: torch.Tensor | None = None) -> torch.Tensor:
    """``logits`` [..., V] (bf16, fp16 or fp32) as a sampler draws from them, in their type. For each row, in this order:

    * tokens of ``history`` [..., L] (int64 or int32; a negative id is none; ``lengths`` int32 of its places hold one, all by
      default): a logit above 0 is divided by ``repetition``, any other multiplied by it;
    * tokens of its places from ``prompt_lengths`` (int32, 0 by default) on, c times each: less ``frequency`` c and
      ``presence``;
    * ``bias`` (fp32 [..., K]) is added to the tokens ``bias_ids`` (int64 [..., K]; a negative id is none, repeated
      ids add up in their order);
    * tokens whose bit is clear in ``allowed`` (int32 [..., ceil(V / 32)], token v in bit v % 32 of word v // 32) become
      -inf, whatever they were.

    Penalties are numbers or one fp32 per row; ``repetition`` is positive. Tables with fewer leading dimensions, or ones,
    serve several rows. Computed in fp32 and rounded once. On a GPU an id beyond the vocabulary or a length beyond the
    history sets the device status (``ops.check_status``) and is passed over; on the CPU it raises."""
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32) and not (
            logits.dtype == torch.float64 and not logits.is_cuda):
        raise TypeError("logits must be bf16, fp16 or fp32")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., vocabulary]")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if history is None and not (lengths is None and prompt_lengths is None and repetition is None and presence is None
                                and frequency is None):
        raise ValueError("lengths and penalties need a history")
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias and bias_ids go together")
    _refuse_gradients("process_logits", logits, bias, *(v for v in (repetition, presence, frequency)
                                                        if isinstance(v, torch.Tensor)))
    if history is not None:
        history = _rows_of(history, "history", (torch.int64, torch.int32), logits)
        for name, value in (("lengths", lengths), ("prompt_lengths", prompt_lengths)):
            if value is not None and value.dtype != torch.int32:
                raise TypeError(f"{name} must be int32")
            if value is not None and (value.shape != lead or value.device != logits.device):
                raise ValueError(f"{name} must hold one value per row on the logits' device")
        lengths, prompt_lengths = (v if v is None or v.ndim == 1 and v.is_contiguous() else v.reshape(-1).contiguous()
                                   for v in (lengths, prompt_lengths))
    repetition, all_repetition = _per_row(repetition, "repetition", logits, 1.0)
    presence, all_presence = _per_row(presence, "presence", logits, 0.0)
    frequency, all_frequency = _per_row(frequency, "frequency", logits, 0.0)
    if bias is not None:
        bias_ids = _rows_of(bias_ids, "bias_ids", (torch.int64,), logits)
        bias = _rows_of(bias, "bias", (torch.float32,), logits)
        if bias.shape != bias_ids.shape:
            raise ValueError("bias and bias_ids must be alike")
        if bias.stride() != bias_ids.stride():
            bias, bias_ids = bias.contiguous(), bias_ids.contiguous()
    if allowed is not None:
        if allowed.ndim < 1 or allowed.shape[-1] < -(-vocab // 32):
            raise ValueError("allowed must hold a bit per token")
        allowed = _rows_of(allowed, "allowed", (torch.int32,), logits)
    if not logits.is_cuda:
        full = lambda v, number: torch.full((lead.numel(),), number, dtype=torch.float64) if v is None else v  # noqa: E731
        return _process_reference(logits.reshape(-1, vocab), history, lengths, prompt_lengths,
                                  full(repetition, all_repetition), full(presence, all_presence),
                                  full(frequency, all_frequency), bias_ids, bias, allowed).view(logits.shape)
    return ext().process_logits(logits, history, lengths, prompt_lengths, repetition, presence, frequency, all_repetition,
                                all_presence, all_frequency, bias_ids, bias, allowed)


__all__ = ["PagedBatch", "paged_append", "paged_attention", "process_logits", "tree_mask"]
