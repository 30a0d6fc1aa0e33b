"""Statistics of rows of logits for scoring tokens, and distillation from a teacher's top alternatives.

* :func:`token_statistics` - one pass over each row of logits gives the log-probability of a given
  token, the entropy of the distribution and its most likely alternatives, all differentiable.
* :func:`linear_token_statistics` - log-probability and entropy straight from hidden states and the LM
  head's weight: without a backward the logits exist only in the tensor cores' accumulators.
* :func:`distillation_loss` - KL divergence from a teacher's recorded top alternatives (what
  ``token_statistics(..., top=k)`` returns) to a student's logits, the gradient written with the loss.

They extend the selected-token log-probabilities of ``dsv41_train/models/dsv4/model.py:679-684``; the
reference has no entropy, alternatives or distillation.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from ._ext import ext, on_gpu
from .loss import IGNORE_INDEX

MAX_TOP = 128  # alternatives of one row
GRADIENT_BYTES = 4 * 2 ** 30  # of the logits' gradient that linear_token_statistics holds at a time
KEPT_BYTES = 4 * 2 ** 30  # of fp32 logits that it keeps for its backward; larger ones are recomputed
_LOGIT_TYPES = (torch.bfloat16, torch.float16, torch.float32)


class TokenStatistics(NamedTuple):
    """fp32 results in the shape of the logits' leading dimensions (alternatives have one more);
    ``log_probs`` is None without targets and ``top_*`` are None where ``top`` is 0."""

    log_probs: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor | None = None
    top_log_probs: torch.Tensor | None = None


class DistillationLoss(NamedTuple):
    """``total``: the weighted sum, differentiable in the logits; ``rows``: the unweighted fp32 divergence
    of each row, for reporting (not differentiable)."""

    total: torch.Tensor
    rows: torch.Tensor


def _check_temperature(temperature: float) -> float:
    temperature = float(temperature)
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError("temperature must be finite and positive")
    return temperature


def _check_targets(targets: torch.Tensor, shape, device) -> None:
    if targets.dtype != torch.int64:
        raise TypeError("targets must be int64")
    if targets.shape != shape or targets.device != device:
        raise ValueError("targets must hold one token id per row, on the logits' device")


def _differentiates(*tensors: torch.Tensor) -> bool:
    """Whether a call has to go through its autograd function: a gradient is wanted, or a tensor carries a forward-mode
    tangent, which the function refuses and a direct call would drop in silence."""
    return (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)
            or any(forward_ad.unpack_dual(t).tangent is not None for t in tensors))


def _check_logits(logits: torch.Tensor) -> None:
    if logits.dtype not in _LOGIT_TYPES and not (logits.dtype == torch.float64 and not logits.is_cuda):
        raise TypeError("logits must be bf16, fp16 or fp32")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., vocabulary]")


# -- the plain restatement (CPU): in 64 bits, since the CPU's fp32 sums over a vocabulary are off by 2e-5 ----
def _scores_reference(logits: torch.Tensor, targets, temperature: float, top: int) -> TokenStatistics:
    x = logits.double()
    masked = x == float("-inf")
    empty = masked.all(-1, keepdim=True)
    skip = torch.zeros_like(empty) if targets is None else (targets == IGNORE_INDEX).unsqueeze(-1)
    # rows that are ignored or masked throughout take no part: any finite row stands in for them
    lp = torch.log_softmax(torch.where(empty | skip, torch.zeros_like(x), x) / temperature, dim=-1)
    finite = torch.where(masked & ~empty, torch.zeros_like(lp), lp)
    entropy = -(finite.exp() * finite).masked_fill(masked, 0.0).sum(-1)
    entropy = entropy.masked_fill((empty | skip).squeeze(-1), 0.0)
    log_probs = ids = values = None
    if targets is not None:
        if bool(((targets < 0) & ~skip.squeeze(-1) | (targets >= x.shape[-1])).any()):
            raise ValueError("target outside the vocabulary")
        log_probs = lp.gather(-1, targets.clamp(min=0).unsqueeze(-1))
        log_probs = log_probs.masked_fill(empty, float("-inf")).masked_fill(skip, 0.0).squeeze(-1)
    if top:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
        absent = skip | masked.gather(-1, order)
        ids = order.masked_fill(absent, -1)
        values = lp.gather(-1, order).masked_fill(absent, float("-inf"))
    as_float = lambda v: v if v is None or logits.dtype == torch.float64 else v.float()  # noqa: E731
    return TokenStatistics(as_float(log_probs), as_float(entropy), ids, as_float(values))


def _distillation_reference(logits, ids, teacher, weights, temperature, tail) -> DistillationLoss:
    x = logits.double()
    if bool((ids >= x.shape[-1]).any()):
        raise ValueError("teacher id outside the vocabulary")
    off = torch.zeros(x.shape[:-1], dtype=torch.bool) if weights is None else weights == 0
    x = torch.where(off.unsqueeze(-1), x.detach(), x)  # no gradient, whatever such a row holds
    there, at = ids >= 0, ids.clamp(min=0).long()
    t = teacher.to(x.dtype).masked_fill(~there, float("-inf"))
    used = there.any(-1) if tail else (t > float("-inf")).any(-1) | t.isnan().any(-1)
    empty = (x == float("-inf")).all(-1)
    lp = torch.log_softmax(torch.where((used & ~empty).unsqueeze(-1), x, torch.zeros_like(x)) / temperature, dim=-1)
    t = torch.where(used.unsqueeze(-1), t, torch.zeros_like(t))
    q, log_q = t.exp(), t
    if not tail:
        log_q = torch.log_softmax(t, dim=-1)
        q = log_q.exp()
    chosen = lp.gather(-1, at)
    # the mass of a token recorded more than once is the sum of its places'
    mass = torch.zeros_like(x).scatter_add_(-1, at, q).gather(-1, at)
    log_q = torch.where(mass == q, log_q, mass.log())
    rows = torch.where(q > 0, q * (log_q.masked_fill(q == 0, 0.0) - chosen), torch.zeros_like(q)).sum(-1)
    if tail:
        inside = torch.zeros_like(x).scatter_add_(-1, at, there.to(x.dtype)) > 0
        left = ~(inside | (lp == float("-inf"))).all(-1)
        rest = (1 - q.sum(-1)).clamp(min=0)
        apart = torch.where(left.unsqueeze(-1), lp, torch.zeros_like(lp)).masked_fill(
            inside & left.unsqueeze(-1), float("-inf"))
        # (logsumexp's gradient exp(lp - result) is 1 for each of many tokens masked by a lowest value: at -1e38 their
        # number is below 64 bits)
        largest = apart.amax(-1, keepdim=True).detach()
        outside = largest.squeeze(-1) + (apart - largest).exp().sum(-1).log()
        keep = left & (rest > 0)
        rows = rows + torch.where(keep, rest * (torch.where(keep, rest, torch.ones_like(rest)).log() - outside),
                                  torch.zeros_like(rest))
    rows = rows.masked_fill(~used, 0.0).masked_fill(used & empty, float("inf"))
    w = torch.ones_like(rows) if weights is None else weights.to(rows.dtype)
    total, rows = (w * rows).masked_fill(off, 0.0).sum(), rows.detach()
    return DistillationLoss(total, rows) if logits.dtype == torch.float64 else DistillationLoss(total.float(), rows.float())


# -- token statistics -------------------------------------------------------------------------------
class _TokenStatistics(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, top):
        lp, entropy, ids, values, saved = ext().token_stats_fwd(logits, targets, temperature, top, IGNORE_INDEX, True)
        ctx.save_for_backward(logits, targets, ids, saved)
        ctx.temperature = temperature
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return lp, entropy, ids, values

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_entropy, _g_ids, g_values):
        logits, targets, ids, saved = ctx.saved_tensors
        plain = lambda g: None if g is None else g.contiguous()  # noqa: E731
        return ext().token_stats_bwd(logits, targets, ids, saved, ctx.temperature, plain(g_lp), plain(g_entropy),
                                     plain(g_values)), None, None, None


def token_statistics(logits: torch.Tensor, targets: torch.Tensor | None = None, *, temperature: float = 1.0,
                     top: int = 0) -> TokenStatistics:
    """Log-probability of ``targets``, entropy, and the ``top`` most likely tokens of
    ``softmax(logits / temperature)`` for each row of ``logits`` [..., V] (bf16, fp16 or fp32).

    Rows may be strided (``logits[:, :-1]``, a padded vocabulary cut to size); they are read in place.
    A target of -100 leaves its row out: log-probability and entropy 0, alternatives -1 / -inf, zero
    gradient, and the row is not read. Masked logits (-inf) are never alternatives: a row with fewer than
    ``top`` others is filled with id -1 and log-probability -inf. Ties go to the lowest id. A row masked
    throughout has log-probability -inf, entropy 0 and no gradient. On a GPU a target outside the
    vocabulary gives NaN and sets the device status (``ops.check_status``); on the CPU it raises."""
    _check_logits(logits)
    temperature = _check_temperature(temperature)
    shape, vocab = logits.shape[:-1], logits.shape[-1]
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be a whole number in [0, min({MAX_TOP}, vocabulary)]")
    if targets is not None:
        _check_targets(targets, shape, logits.device)
    if not logits.is_cuda:
        return _scores_reference(logits, targets, temperature, top)
    if targets is not None:
        targets = targets.contiguous()
    if _differentiates(logits):
        return TokenStatistics(*_TokenStatistics.apply(logits, targets, temperature, top))
    lp, entropy, ids, values, _ = ext().token_stats_fwd(logits, targets, temperature, top, IGNORE_INDEX, False)
    return TokenStatistics(lp, entropy, ids, values)


# -- statistics of the LM head's product ------------------------------------------------------------
def _aligned(x: torch.Tensor) -> torch.Tensor:
    """``x``, or a copy where it starts inside a 16-byte unit (a view at an odd offset), which TMA cannot read."""
    return x if x.data_ptr() % 16 == 0 else x.clone()


class _LinearTokenStatistics(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, temperature):
        ctx.keep = hidden.shape[0] * weight.shape[0] * 4 <= KEPT_BYTES
        lp, entropy, saved, logits = ext().lm_head_stats_fwd(hidden, weight, targets, temperature, IGNORE_INDEX, True,
                                                             ctx.keep)
        ctx.save_for_backward(hidden, weight, targets, saved, logits)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return lp, entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_entropy):
        C = ext()
        hidden, weight, targets, saved, logits = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        if g_lp is None and g_entropy is None:
            return None, None, None, None
        g_lp, g_entropy = (None if g is None else g.contiguous() for g in (g_lp, g_entropy))
        rows, vocab = hidden.shape[0], weight.shape[0]
        if rows == 0:
            return hidden.new_zeros(hidden.shape), weight.new_zeros(weight.shape), None, None
        chunk = max(128, GRADIENT_BYTES // (vocab * 2) // 128 * 128)
        dx = torch.empty_like(hidden) if need_dx else None
        dw = None
        if need_dw:
            dw = torch.empty_like(weight) if chunk >= rows else torch.zeros(weight.shape, dtype=torch.float32,
                                                                            device=weight.device)
        for start in range(0, rows, chunk):
            part = slice(start, min(rows, start + chunk))
            pick = lambda x: None if x is None else x[part]  # noqa: E731
            dlogits = C.lm_head_stats_bwd(hidden[part], weight, targets[part], saved[part], pick(logits),
                                          ctx.temperature, IGNORE_INDEX, pick(g_lp), pick(g_entropy))
            if need_dx:
                C.gemm_split_k(dlogits, weight, dx[part])
            if need_dw:
                C.gemm(dlogits, hidden[part], dw, True, True, chunk < rows)
            del dlogits
        return dx, None if dw is None else dw.to(weight.dtype), None, None


def linear_token_statistics(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                            temperature: float = 1.0) -> TokenStatistics:
    """:func:`token_statistics` of ``hidden @ weight.T``: log-probability of ``targets`` and entropy of each
    row of ``hidden`` [..., H] under the LM head ``weight`` [V, H].

    The reduction runs in the epilogue of the tensor-core product on its fp32 accumulators, so no
    logit is rounded to bf16. Without a backward no logit is written, and rows with target -100, whose
    results are 0, take no part in the product. Where a backward may follow, each call keeps its fp32 logits
    until then while they take at most ``KEPT_BYTES`` (4 GiB; twice what bf16 logits take), else the product
    is repeated; the logits' gradient, rounded to bf16 and in row blocks of at most ``GRADIENT_BYTES``
    (4 GiB), is multiplied into ``hidden`` and ``weight``. bf16 operands with H a multiple of 8 (a view that
    starts off a 16-byte boundary is copied); on a GPU other types go through the product and
    :func:`token_statistics`, where the logits exist in ``hidden``'s type."""
    temperature = _check_temperature(temperature)
    if hidden.ndim < 1 or weight.ndim != 2 or hidden.shape[-1] != weight.shape[1] or weight.shape[0] < 1:
        raise ValueError("hidden must be [..., H] and weight [V, H]")
    shape = hidden.shape[:-1]
    _check_targets(targets, shape, hidden.device)
    if weight.device != hidden.device:
        raise ValueError("hidden and weight must be on one device")
    if not (on_gpu(hidden) and hidden.dtype == weight.dtype == torch.bfloat16 and hidden.shape[-1] % 8 == 0):
        logits = F.linear(hidden, weight.to(hidden.dtype))
        return token_statistics(logits, targets, temperature=temperature)
    flat = _aligned(hidden.reshape(-1, hidden.shape[-1]).contiguous())
    weight, targets = _aligned(weight.contiguous()), targets.reshape(-1).contiguous()
    if _differentiates(hidden, weight):
        lp, entropy = _LinearTokenStatistics.apply(flat, weight, targets, temperature)
    else:
        lp, entropy, _, _ = ext().lm_head_stats_fwd(flat, weight, targets, temperature, IGNORE_INDEX, False, False)
    return TokenStatistics(lp.view(shape), entropy.view(shape))


# -- distillation -----------------------------------------------------------------------------------
class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, weights, temperature, tail):
        total, rows, dlogits, saved = ext().distill_fwd(logits, ids, teacher, weights, temperature, tail, True)
        ctx.save_for_backward(logits, ids, dlogits, saved)
        ctx.temperature, ctx.handed_out = temperature, False
        ctx.mark_non_differentiable(rows)
        return total, rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_total, _g_rows):
        if ctx.handed_out:
            raise RuntimeError("distillation_loss: the gradient was handed out by an earlier backward; call the "
                               "operator again")
        logits, ids, dlogits, saved = ctx.saved_tensors
        ctx.handed_out = True
        ext().distill_again(dlogits, logits, ids, saved, g_total.contiguous(), ctx.temperature)
        return dlogits, None, None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_log_probs: torch.Tensor,
                      weights: torch.Tensor | None = None, *, temperature: float = 1.0,
                      tail: bool = False) -> DistillationLoss:
    """``sum_r weights_r KL(teacher_r || softmax(logits_r / temperature))`` over a teacher's recorded
    alternatives: ``teacher_ids`` (int32 or int64) and fp32 ``teacher_log_probs``, both [..., K], K <= 128.

    ``tail=False`` renormalises the K alternatives (any constant added to a row of
    ``teacher_log_probs`` cancels, so temperature-scaled logits do as well); ``tail=True`` takes them as
    they are and compares the rest of the mass with the student's mass outside the K tokens. A negative
    id is no alternative, and a row without any has loss 0 and zero gradient and is not read. Repeated
    ids count as one token. ``weights`` (fp32, one per row; 1 by default) carry masks and the
    normalisation, e.g. 1 / tokens: a weight of 0 leaves its row out of the total and gives it a gradient of
    zeros, even where its divergence is infinite or its logits are NaN (``rows`` reports it all the same).
    The gradient is written in the same pass over the logits as the loss, for an upstream gradient of one;
    for any other (a factor applied to ``total``, a loss scale) ``backward`` writes it once more from the
    logits, which costs another pass; either way it is rounded once. Because it is handed over on ``backward``, the
    operator is called again for a second one. Teacher, ids and weights take no gradient. On a GPU an id beyond the
    vocabulary gives NaN and sets the device status."""
    _check_logits(logits)
    temperature = _check_temperature(temperature)
    shape = logits.shape[:-1]
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("teacher_ids must be int32 or int64")
    if teacher_ids.ndim != logits.ndim or teacher_ids.shape[:-1] != shape or teacher_ids.shape != teacher_log_probs.shape:
        raise ValueError("teacher_ids and teacher_log_probs must both be [..., K] over the logits' rows")
    k = teacher_ids.shape[-1]
    if not 1 <= k <= MAX_TOP:
        raise ValueError(f"a teacher records 1 to {MAX_TOP} alternatives")
    if weights is not None and weights.shape != shape:
        raise ValueError("weights must hold one value per row")
    device = logits.device
    if teacher_ids.device != device or teacher_log_probs.device != device or (
            weights is not None and weights.device != device):
        raise ValueError("teacher and weights must be on the logits' device")
    if not logits.is_cuda:
        return _distillation_reference(logits, teacher_ids, teacher_log_probs.detach(),
                                       None if weights is None else weights.detach(), temperature, tail)
    ids, teacher = teacher_ids.contiguous(), teacher_log_probs.detach().float().contiguous()
    weights = None if weights is None else weights.detach().float().contiguous()
    if _differentiates(logits):
        total, rows = _Distillation.apply(logits, ids, teacher, weights, temperature, tail)
    else:
        total, rows, _, _ = ext().distill_fwd(logits, ids, teacher, weights, temperature, tail, False)
    return DistillationLoss(total, rows)


__all__ = ["DistillationLoss", "TokenStatistics", "distillation_loss", "linear_token_statistics",
           "token_statistics"]
