"""Token statistics and distillation: results, gradients and refusals against 64-bit definitions.

Tolerances. The kernels sum in fp32: an exponential is off by 2^-22 of itself and a sum of n rounded
terms by at most n 2^-24, in practice by about sqrt(n) 2^-24; a thread sums up to V / 256 = 600 terms, so
1e-5 bounds the relative error of a sum and the absolute error of its logarithm. A log-probability adds
one fp32 rounding of a value up to some hundred (1e-6 of itself). The entropy multiplies the error of
its two sums by values up to ln V = 12: 1e-4. A gradient is one product of such factors, off by 2e-5 of
the row's largest value, plus one rounding to its type (2^-9 for bf16, 2^-11 for fp16 of itself, and
fp16's smallest step of 6e-8).
"""

import importlib.util
import math
from pathlib import Path

import pytest
import torch

from tiny_dsv41_b200 import ops
from tiny_dsv41_b200.ops import statistics as S

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
ROUND = {torch.float64: 0.0, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    if torch.cuda.is_available():
        ops.check_status("test")


def _generator(seed):
    return torch.Generator().manual_seed(seed)


def _logits(rows, vocab, dtype, seed=0, device="cpu"):
    x = torch.randn(rows, vocab, generator=_generator(seed)) * 3
    return x.to(dtype).to(device)


# -- the definitions, row by row in 64 bits ---------------------------------------------------------
def _row(x, temperature):
    """(lp, p) of one row, or None where nothing is unmasked."""
    y = x.double().cpu() / temperature
    if bool((y == -INF).all()):
        return None
    lp = torch.log_softmax(y, 0)
    return lp, lp.exp()


def _statistics(logits, targets, temperature, top):
    rows, vocab = logits.shape
    out = {"log_probs": torch.zeros(rows, dtype=torch.float64), "entropy": torch.zeros(rows, dtype=torch.float64),
           "top_ids": torch.full((rows, top), -1), "top_log_probs": torch.full((rows, top), -INF, dtype=torch.float64)}
    for r in range(rows):
        if targets is not None and int(targets[r]) == -100:
            continue
        scored = _row(logits[r], temperature)
        if scored is None:
            out["log_probs"][r] = -INF
            continue
        lp, p = scored
        if targets is not None:
            out["log_probs"][r] = lp[int(targets[r])]
        out["entropy"][r] = -(p * lp)[p > 0].sum()
        values = logits[r].double().cpu()
        order = sorted(range(vocab), key=lambda i: (-float(values[i]), i)) if vocab <= 5000 else torch.sort(
            values, descending=True, stable=True).indices[:top].tolist()
        for j in range(top):
            if float(values[order[j]]) != -INF:
                out["top_ids"][r, j], out["top_log_probs"][r, j] = order[j], lp[order[j]]
    return out


def _statistics_gradient(logits, targets, temperature, g, h, ids=None, u=None):
    out = torch.zeros(logits.shape, dtype=torch.float64)
    for r in range(len(logits)):
        scored = None if targets is not None and int(targets[r]) == -100 else _row(logits[r], temperature)
        if scored is None:
            continue
        lp, p = scored
        logs = lp.masked_fill(p == 0, 0.0)
        d = -float(h[r]) * p * (logs - (p * logs).sum())
        if targets is not None:
            d -= float(g[r]) * p
            d[int(targets[r])] += float(g[r])
        for j in range(0 if ids is None else ids.shape[1]):
            if int(ids[r, j]) >= 0:
                d -= float(u[r, j]) * p
                d[int(ids[r, j])] += float(u[r, j])
        out[r] = d / temperature
    return out


def _distillation(logits, ids, teacher, weights, temperature, tail):
    """(row divergences, gradient) by summing over the outcomes: the alternatives, and the rest as one."""
    rows, vocab = logits.shape
    loss, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, vocab, dtype=torch.float64)
    for r in range(rows):
        q = {}
        for i, t in zip(ids[r].tolist(), teacher[r].double().tolist()):
            if i >= 0:
                q[i] = q.get(i, 0.0) + math.exp(t)
        whole = sum(q.values())
        if not q or (not tail and whole == 0):
            continue
        if not tail:
            q = {i: v / whole for i, v in q.items()}
        scored = _row(logits[r], temperature)
        if scored is None:
            loss[r] = INF
            continue
        lp, p = scored
        outside = torch.ones(vocab, dtype=torch.bool)
        outside[list(q)] = False
        left = lp[outside].logsumexp(0) if bool(outside.any()) else torch.tensor(-INF)
        rest = max(0.0, 1.0 - whole) if tail and float(left) > -INF else 0.0
        # repeated ids: each recorded value keeps its own term, against one probability
        for i, t in zip(ids[r].tolist(), teacher[r].double().tolist()):
            one = math.exp(t) / (1.0 if tail else whole) if i >= 0 else 0.0
            if one:
                loss[r] += one * (math.log(one) - float(lp[i]))
        if rest:
            loss[r] += rest * (math.log(rest) - float(left))
        d = (sum(q.values()) + rest) * p
        for i, v in q.items():
            d[i] -= v
        if rest:
            d[outside] -= rest * (lp[outside] - left).exp()
        grad[r] = d * float(weights[r]) / temperature
    return loss, grad


def _close_rows(got, want, absolute, relative=1e-6):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine], want[~fine])
    assert bool(((got - want).abs()[fine] <= absolute + relative * want.abs()[fine]).all()), (got - want)[fine].abs().max()


def _close_gradient(got, want):
    dtype, got = got.dtype, got.double().cpu()
    assert bool(torch.isfinite(got).all())
    bound = 2e-5 * want.abs().amax(-1, keepdim=True) + ROUND[dtype] * want.abs()
    if dtype == torch.float16:
        bound = bound + 6e-8
    assert bool(((got - want).abs() <= bound + 1e-30).all()), ((got - want).abs() / (bound + 1e-30)).max()


def _check_statistics(logits, targets, temperature, top, got):
    want = _statistics(logits, targets, temperature, top)
    if targets is not None:
        _close_rows(got.log_probs, want["log_probs"], 1e-5)
    _close_rows(got.entropy, want["entropy"], 1e-4)
    if top:
        assert torch.equal(got.top_ids.cpu(), want["top_ids"])
        _close_rows(got.top_log_probs, want["top_log_probs"], 1e-5)


# -- token statistics -------------------------------------------------------------------------------
SIZES = [(1, 1), (1, 2), (3, 7), (5, 33), (130, 515), (2, 1000), (9, 4099), (3, 16385), (40, 32003), (2, 151936)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_statistics_sizes(device, dtype, rows, vocab):
    logits = _logits(rows, vocab, dtype, vocab, device)
    targets = torch.randint(0, vocab, (rows,), generator=_generator(1)).to(device)
    if rows > 2:
        targets[1] = -100
    for top in {0, 1, min(20, vocab), min(128, vocab)}:
        got = ops.token_statistics(logits, targets, temperature=0.7, top=top)
        _check_statistics(logits, targets, 0.7, top, got)
    assert ops.token_statistics(logits).log_probs is None


def _special(vocab):
    """Rows at which a running maximum, a threshold or a mask can go wrong."""
    x = torch.randn(16, vocab, generator=_generator(3)) * 3
    x[0] = -INF                                  # masked throughout
    x[1, 1:] = -INF                              # one token left
    x[2] = 0.0                                   # all equal
    x[3] = torch.arange(vocab).float() * 0.01    # every value is a new maximum
    x[4] = -torch.arange(vocab).float() * 0.01
    x[5] = x[5].round()                          # many ties
    x[6] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0)  # zeros of both signs are equal
    x[7] += 1.0e4                                # a common offset
    x[8, ::2] = -INF
    x[9, 5:] = -1.0e4                            # masked by a large value
    x[10] = torch.finfo(torch.bfloat16).min      # the type's lowest value everywhere
    x[11, : vocab // 2] = torch.finfo(torch.bfloat16).min
    x[11, vocab // 2:] = -INF
    x[12, -1] = 80.0                             # all of the mass on one token, the last one
    x[13, 0] = 80.0
    x[14] = -300.0 * torch.arange(vocab).float().flip(0) / vocab
    x[15, : max(1, vocab - 3)] = -INF
    return x


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,temperature", [(40, 1.0), (2051, 0.05), (20000, 1.0), (20000, 50.0)])
def test_statistics_special_rows(device, dtype, vocab, temperature):
    logits = _special(vocab).to(dtype).to(device)
    targets = torch.randint(0, vocab, (16,), generator=_generator(4)).to(device)
    got = ops.token_statistics(logits, targets, temperature=temperature, top=33)
    want = _statistics(logits, targets, temperature, 33)
    # log-probabilities reach 1e6 here, and lowest values / T pass fp32's range: those are -inf
    want["log_probs"][want["log_probs"] < -3.4e38] = -INF
    want["top_log_probs"][want["top_log_probs"] < -3.4e38] = -INF
    _close_rows(got.log_probs, want["log_probs"], 1e-5)
    _close_rows(got.entropy, want["entropy"], 1e-4)
    assert torch.equal(got.top_ids.cpu(), want["top_ids"])
    _close_rows(got.top_log_probs, want["top_log_probs"], 1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_statistics_ignored_and_nan_rows(device):
    logits = _logits(4, 300, torch.float32, 5, device)
    logits[0], logits[2, 17], logits[3, 5] = float("nan"), float("nan"), INF
    targets = torch.tensor([-100, 3, 4, 6], device=device)
    logits.requires_grad_()
    got = ops.token_statistics(logits, targets, top=3)
    assert got.log_probs[0] == 0 and got.entropy[0] == 0 and bool((got.top_ids[0] == -1).all())
    assert bool((got.top_log_probs[0] == -INF).all())
    _check_statistics(logits.detach()[1:2], targets[1:2], 1.0, 3, S.TokenStatistics(*(t.detach()[1:2] for t in got)))
    assert bool(got.log_probs[2].isnan()) and bool(got.entropy[2:].isnan().all())
    got.log_probs[:2].sum().backward()
    assert bool((logits.grad[0] == 0).all()) and bool(logits.grad[1].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_statistics_strides(device, dtype):
    base = _logits(6 * 9, 1031, dtype, 6, device).view(6, 9, 1031)
    targets = torch.randint(0, 900, (6, 9), generator=_generator(7)).to(device)
    for view, t in ((base[:, :-1, :1003], targets[:, 1:]),         # shifted rows, a vocabulary cut to size
                    (base[:, :, 3:1000], targets.clamp(max=900)),   # rows that start anywhere
                    (base[::2, 1], targets[::2, 1]),
                    (base.transpose(0, 1), targets.t()),
                    (base.transpose(1, 2)[..., :5], None),          # no row is contiguous: copied
                    (base[2, 4], targets[2, 4]),                    # one row, no leading dimension
                    (base[:, :0], targets[:, :0])):                 # no rows
        t = None if t is None else t.clamp(max=view.shape[-1] - 1)
        leaf = view.detach()
        leaf.requires_grad_()
        got = ops.token_statistics(leaf, t, top=4)
        assert got.entropy.shape == view.shape[:-1] and got.top_ids.shape == (*view.shape[:-1], 4)
        flat = view.reshape(-1, view.shape[-1])
        if len(flat):
            _check_statistics(flat, None if t is None else t.reshape(-1), 1.0, 4,
                              S.TokenStatistics(*(None if x is None else x.detach().reshape(len(flat), *x.shape[view.ndim - 1:])
                                                  for x in got)))
        got.entropy.sum().backward()
        want = _statistics_gradient(flat, None, 1.0, None, torch.ones(len(flat)))
        assert leaf.grad.shape == view.shape
        if len(flat):
            _close_gradient(leaf.grad.reshape(flat.shape), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (130, 515), (7, 4099), (2, 151936), (3, 151936)])
def test_statistics_gradient(device, dtype, rows, vocab):
    logits = _logits(rows, vocab, dtype, vocab + 1, device).requires_grad_()
    targets = torch.randint(0, vocab, (rows,), generator=_generator(8)).to(device)
    if rows > 2:
        targets[1] = -100
    top = min(5, vocab)
    g, h = torch.randn(rows, generator=_generator(9)), torch.randn(rows, generator=_generator(10))
    u = torch.randn(rows, top, generator=_generator(11))
    got = ops.token_statistics(logits, targets, temperature=0.7, top=top)
    total = (got.log_probs * g.to(device)).sum() + (got.entropy * h.to(device)).sum()
    present = got.top_ids >= 0
    total = total + (got.top_log_probs.masked_fill(~present, 0.0) * u.to(device)).sum()
    total.backward()
    _close_gradient(logits.grad, _statistics_gradient(logits.detach(), targets, 0.7, g, h, got.top_ids.cpu(), u))
    # each output on its own
    for pick, gg, hh in ((0, g, torch.zeros(rows)), (1, torch.zeros(rows), h)):
        leaf = logits.detach().clone().requires_grad_()
        out = ops.token_statistics(leaf, targets, temperature=0.7)
        (out[pick] * (g if pick == 0 else h).to(device)).sum().backward()
        _close_gradient(leaf.grad, _statistics_gradient(leaf.detach(), targets, 0.7, gg, hh))


@pytest.mark.parametrize("device", DEVICES)
def test_entropy_gradient_of_special_rows(device):
    """-p (ln p + H): where all logits are equal the two terms cancel to zero, so the error is bounded by
    the terms (2e-5 of the largest p |ln p| + p H of the row) and not by the result."""
    logits = _special(600).to(device).requires_grad_()
    ops.token_statistics(logits, torch.tensor([0] * 16, device=device)).entropy.sum().backward()
    assert bool(logits.grad.isfinite().all()) and bool((logits.grad[0] == 0).all())
    want = _statistics_gradient(logits.detach(), None, 1.0, None, torch.ones(16))
    for r in range(1, 16):
        lp, p = _row(logits.detach()[r], 1.0)
        logs = lp.masked_fill(p == 0, 0.0)
        terms = float((p * logs.abs() - p * (p * logs).sum()).max())
        off = (logits.grad[r].double().cpu() - want[r]).abs().max()
        assert off <= 2e-5 * terms + 1e-20, (r, off, terms)


@pytest.mark.parametrize("device", DEVICES)
def test_statistics_gradient_against_differences(device):
    logits = _logits(3, 37, torch.float32, 12, device)
    targets, step = torch.tensor([4, -100, 30], device=device), 1e-2

    def value(x):
        s = ops.token_statistics(x, targets, temperature=1.3, top=2)
        return (s.log_probs * 0.7 + s.entropy * 0.4).sum() + s.top_log_probs[[0, 2]].sum()

    leaf = logits.clone().requires_grad_()
    value(leaf).backward()
    for r, i in ((0, 4), (0, 11), (1, 3), (2, 30), (2, 0)):
        up, down = logits.clone(), logits.clone()
        up[r, i] += step
        down[r, i] -= step
        slope = (float(value(up)) - float(value(down))) / (2 * step)
        # a third derivative of at most 1 leaves step^2, and 1e-5 of rounding is divided by the step
        assert abs(slope - float(leaf.grad[r, i])) < step ** 2 + 2e-5 / step


def test_statistics_refusals():
    x, t = torch.randn(3, 8), torch.zeros(3, dtype=torch.int64)
    for temperature in (0.0, -1.0, INF, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_statistics(x, t, temperature=temperature)
    for top in (-1, 9, 1.0, True):
        with pytest.raises(ValueError, match="top"):
            ops.token_statistics(x, t, top=top)
    with pytest.raises(ValueError, match="top"):
        ops.token_statistics(torch.randn(1, 500), top=129)
    with pytest.raises(TypeError, match="int64"):
        ops.token_statistics(x, t.int())
    with pytest.raises(ValueError, match="one token id per row"):
        ops.token_statistics(x, t[:2])
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.token_statistics(x.long(), t)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.token_statistics(x[:, :0], t)
    with pytest.raises(ValueError, match="outside the vocabulary"):
        ops.token_statistics(x, t + 8)


@pytest.mark.gpu
def test_targets_beyond_the_vocabulary_set_the_status():
    x = _logits(3, 64, torch.float32, 13, "cuda")
    got = ops.token_statistics(x, torch.tensor([1, 64, -3], device="cuda"))
    assert got.log_probs.isnan().tolist() == [False, True, True] and bool(got.entropy.isfinite().all())
    with pytest.raises(ops.DeviceStatusError, match="out of bounds"):
        ops.check_status("statistics")
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.token_statistics(x.double())
    with pytest.raises(ValueError, match="on the logits' device"):
        ops.token_statistics(x, torch.zeros(3, dtype=torch.int64))


@pytest.mark.gpu
def test_statistics_repeat_and_streams():
    logits = _logits(50, 20011, torch.bfloat16, 14, "cuda").requires_grad_()
    targets = torch.randint(0, 20011, (50,), device="cuda")
    torch.cuda.synchronize()

    def once():
        s = ops.token_statistics(logits, targets, top=9)
        grad, = torch.autograd.grad(s.log_probs.sum() + s.entropy.sum(), logits)
        return (*s, grad)

    first = once()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        second = once()
    stream.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    rows, vocab = 17000, 151936
    logits = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    logits[-3:] = _logits(3, vocab, torch.bfloat16, 15, "cuda")
    targets = torch.full((rows,), -100, device="cuda")
    targets[-3:] = torch.tensor([5, 1000, vocab - 1], device="cuda")
    logits.requires_grad_()
    got = ops.token_statistics(logits, targets, top=4)
    grad, = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), logits)
    tail = logits.detach()[-3:].clone().requires_grad_()
    alone = ops.token_statistics(tail, targets[-3:], top=4)
    want, = torch.autograd.grad(alone.log_probs.sum() + alone.entropy.sum(), tail)
    # few rows may be split over more thread blocks than many: the sums agree to their rounding
    _close_rows(got.log_probs.detach()[-3:], alone.log_probs.detach().double().cpu(), 1e-5)
    assert torch.equal(got.top_ids[-3:], alone.top_ids)
    _close_gradient(grad[-3:], want.double().cpu())
    assert int(grad[:-3].count_nonzero()) == 0
    del grad
    ids = torch.full((rows, 2), -1, device="cuda")
    ids[-3:] = torch.tensor([[1, 2], [3, -1], [vocab - 1, 0]], device="cuda")
    teacher = torch.full((rows, 2), -1.0, device="cuda")
    loss = ops.distillation_loss(logits, ids, teacher, tail=True)
    grad, = torch.autograd.grad(loss.total, logits)
    rows_want, grad_want = _distillation(tail.detach(), ids[-3:].cpu(), teacher[-3:].cpu(), torch.ones(3), 1.0, True)
    _close_rows(loss.rows[-3:], rows_want, 1e-4)
    _close_gradient(grad[-3:], grad_want)


# -- the LM head ------------------------------------------------------------------------------------
def _head(rows, hidden, vocab, device, dtype, seed=20):
    h = torch.randn(rows, hidden, generator=_generator(seed)).to(dtype).to(device)
    w = (torch.randn(vocab, hidden, generator=_generator(seed + 1)) * 3 / hidden ** 0.5).to(dtype).to(device)
    t = torch.randint(0, vocab, (rows,), generator=_generator(seed + 2)).to(device)
    if rows > 2:
        t[1] = -100
    return h, w, t


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,hidden,vocab", [(1, 8, 1), (1, 64, 32), (3, 72, 257), (130, 256, 515), (300, 128, 4099),
                                               (129, 2048, 1000), (1, 128, 30001)])
def test_linear_statistics(device, rows, hidden, vocab):
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    h, w, t = _head(rows, hidden, vocab, device, dtype)
    h.requires_grad_(), w.requires_grad_()
    got = ops.linear_token_statistics(h, w, t, temperature=0.7)
    assert got.top_ids is None
    logits = (h.detach().double() @ w.detach().double().t()).cpu()
    want = _statistics(logits, t.cpu(), 0.7, 0)
    # a logit is a sum of `hidden` products of size up to 10 in fp32: 1e-5 at most
    _close_rows(got.log_probs.detach(), want["log_probs"], 3e-5, 1e-5)
    _close_rows(got.entropy.detach(), want["entropy"], 3e-4)
    g, e = torch.randn(rows, generator=_generator(23)), torch.randn(rows, generator=_generator(24))
    torch.autograd.backward((got.log_probs, got.entropy), (g.to(device), e.to(device)))
    d = _statistics_gradient(logits, t.cpu(), 0.7, g, e)
    for got_grad, want_grad in ((h.grad, d @ w.detach().double().cpu()), (w.grad, d.t() @ h.detach().double().cpu())):
        # a product of gradients rounded to bf16 once, rounded once more
        off = (got_grad.double().cpu() - want_grad).norm() / want_grad.norm().clamp_min(1e-9)
        assert off < (1e-4 if dtype == torch.float32 else 2 * 2.0 ** -8), off
        assert got_grad.dtype == dtype
    if rows > 2:
        assert bool((h.grad[1] == 0).all())


@pytest.mark.gpu
def test_linear_statistics_in_row_blocks(monkeypatch):
    h, w, t = _head(300, 64, 1003, "cuda", torch.bfloat16, 30)
    g, e = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    grads = []
    for limit in (None, 1):
        if limit:
            monkeypatch.setattr(S, "GRADIENT_BYTES", limit)  # 128 rows at a time
        hh, ww = h.clone().requires_grad_(), w.clone().requires_grad_()
        got = ops.linear_token_statistics(hh, ww, t)
        torch.autograd.backward((got.log_probs, got.entropy), (g, e))
        grads.append((hh.grad, ww.grad))
    assert torch.equal(grads[0][0], grads[1][0])
    # the blocks' sum is rounded to bf16 once in both
    assert ((grads[0][1].float() - grads[1][1].float()).norm() / grads[0][1].float().norm()) < 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab", [(5, 64, 300), (260, 512, 20011), (129, 1024, 9000)])
def test_linear_statistics_recomputed(monkeypatch, rows, hidden, vocab):
    """The backward without kept logits: the same fp32 values, so the same gradients to their bf16 rounding."""
    h, w, t = _head(rows, hidden, vocab, "cuda", torch.bfloat16, 50)
    g, e = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    grads = []
    for kept in (S.KEPT_BYTES, 0):
        monkeypatch.setattr(S, "KEPT_BYTES", kept)
        hh, ww = h.clone().requires_grad_(), w.clone().requires_grad_()
        got = ops.linear_token_statistics(hh, ww, t)
        torch.autograd.backward((got.log_probs, got.entropy), (g, e))
        grads.append((hh.grad.float(), ww.grad.float()))
    for a, b in zip(*grads):
        assert (a - b).norm() <= 2.0 ** -8 * a.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 256, 2048), (300, 512, 40000), (129, 264, 20011), (128, 2048, 5000)])
def test_gemm_split_k(m, n, k):
    gen = _generator(60)
    pitch = (k + 7) // 8 * 8
    a = torch.randn(m, pitch, generator=gen).bfloat16().cuda()[:, :k]
    b = torch.randn(k, n, generator=gen).bfloat16().cuda()
    out = torch.full((m, n), float("nan"), device="cuda", dtype=torch.bfloat16)
    ops.ext().gemm_split_k(a, b, out)
    want = a.double() @ b.double()
    # one rounding to bf16 of each value, and fp32 sums that are off by 1e-5 of the products' size
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * k).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,ignored", [(300, 0), (300, 1), (300, 299), (300, 300), (2500, 1100)])
def test_linear_statistics_leaves_ignored_rows_out(rows, ignored):
    h, w, t = _head(rows, 128, 2003, "cuda", torch.bfloat16, 70)
    t[1] = 7
    t[torch.randperm(rows, generator=_generator(71))[:ignored].cuda()] = -100
    h[t == -100] = float("nan")
    got = ops.linear_token_statistics(h, w, t)
    kept = t != -100
    want = _statistics((h[kept].double() @ w.double().t()).cpu(), t[kept].cpu(), 1.0, 0)
    _close_rows(got.log_probs[kept], want["log_probs"], 3e-5, 1e-5)
    _close_rows(got.entropy[kept], want["entropy"], 3e-4)
    assert bool((got.log_probs[~kept] == 0).all()) and bool((got.entropy[~kept] == 0).all())
    again = ops.linear_token_statistics(h, w, t)
    assert torch.equal(got.log_probs, again.log_probs) and torch.equal(got.entropy, again.entropy)


@pytest.mark.gpu
def test_linear_statistics_other_types_and_views():
    h, w, t = _head(12, 60, 333, "cuda", torch.bfloat16, 40)  # H is no multiple of 8: the product is written
    want = _statistics((h @ w.t()).cpu(), t.cpu(), 1.0, 0)
    got = ops.linear_token_statistics(h, w, t)
    _close_rows(got.log_probs, want["log_probs"], 0.1)  # its logits are rounded to bf16
    h, w, t = _head(24, 64, 333, "cuda", torch.bfloat16, 41)
    a = ops.linear_token_statistics(h.view(4, 6, 64)[:, 1:], w, t.view(4, 6)[:, 1:])
    b = ops.linear_token_statistics(h, w, t)
    assert torch.equal(a.log_probs, b.log_probs.view(4, 6)[:, 1:])
    one = h.clone().requires_grad_()
    ops.linear_token_statistics(one, w, t).log_probs.sum().backward()
    assert one.grad is not None
    empty = ops.linear_token_statistics(h[:0].clone().requires_grad_(), w, t[:0])
    assert empty.log_probs.shape == (0,)
    empty.log_probs.sum().backward()


def test_linear_statistics_refusals():
    h, w, t = _head(4, 8, 10, "cpu", torch.float32)
    with pytest.raises(ValueError, match="weight"):
        ops.linear_token_statistics(h, w[:, :4], t)
    with pytest.raises(ValueError, match="one token id per row"):
        ops.linear_token_statistics(h, w, t[:3])
    with pytest.raises(ValueError, match="temperature"):
        ops.linear_token_statistics(h, w, t, temperature=0)


# -- distillation -----------------------------------------------------------------------------------
def _teacher(logits, k, seed):
    rows, vocab = logits.shape
    t = torch.log_softmax(logits.float().cpu() + torch.randn(rows, vocab, generator=_generator(seed)), -1)
    values, ids = t.topk(k, dim=-1)
    if rows > 3:
        ids[1] = -1                 # no teacher
        ids[2, k // 2:] = -1        # fewer alternatives
        values[1], values[2, k // 2:] = -INF, -INF
        if k == 1:
            ids[2], values[2] = 0, 0.0
    return ids, values


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,k", [(1, 2, 1), (6, 33, 4), (1, 515, 128), (40, 4099, 20), (5, 32003, 64),
                                          (2, 151936, 64)])
def test_distillation(device, dtype, tail, rows, vocab, k):
    logits = _logits(rows, vocab, dtype, vocab + 2, device).requires_grad_()
    ids, teacher = _teacher(logits.detach(), k, 50)
    weights = torch.rand(rows, generator=_generator(51))
    want_rows, want_grad = _distillation(logits.detach(), ids, teacher, weights, 1.3, tail)
    args = (teacher.to(device), weights.to(device))
    for i in (ids, ids.int()):
        logits.grad = None
        loss = ops.distillation_loss(logits, i.to(device), *args, temperature=1.3, tail=tail)
        loss.total.backward()
        _close_rows(loss.rows, want_rows, 1e-4)
        _close_rows(loss.total.detach(), (want_rows * weights.double()).sum(), 1e-4 * float(weights.sum()), 1e-5)
        _close_gradient(logits.grad, want_grad)
    with torch.no_grad():
        alone = ops.distillation_loss(logits, ids.to(device), *args, temperature=1.3, tail=tail)
    _close_rows(alone.rows, want_rows, 1e-4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_special_rows(device, tail):
    vocab = 2051
    logits = _special(vocab).to(device)
    logits[10:12] = 0.0  # (fp32 holds these rows' lowest values, but not their divergence)
    ids = torch.stack([torch.randperm(vocab, generator=_generator(60 + r))[:6] for r in range(16)])
    teacher = torch.log_softmax(torch.randn(16, 6, generator=_generator(80)), -1) - 0.2
    ids[1, 0], ids[12, 0], ids[13, 0] = 0, vocab - 1, 0
    ids[2] = torch.tensor([7, 7, 9, -1, 9, 7])   # repeated
    teacher[4, 2:] = -INF                         # recorded with no mass
    teacher[5] -= 60.0                            # a teacher with nearly all mass in the tail
    teacher[6] = math.log(0.5)                    # more than one in all
    ids[14] = torch.arange(vocab - 6, vocab)      # a student whose mass is all on the alternatives
    logits[14, :-6] -= 200.0
    leaf = logits.clone().requires_grad_()
    weights = torch.linspace(0.1, 1.0, 16)
    loss = ops.distillation_loss(leaf, ids.to(device), teacher.to(device), weights.to(device), tail=tail)
    want_rows, want_grad = _distillation(logits, ids, teacher, weights, 1.0, tail)
    _close_rows(loss.rows, want_rows, 1e-4, 1e-5)
    grad, = torch.autograd.grad(loss.total, leaf)
    _close_gradient(grad, want_grad)


@pytest.mark.parametrize("device", DEVICES)
def test_distillation_where_the_alternatives_are_the_vocabulary(device):
    logits = _logits(3, 16, torch.float32, 52, device).requires_grad_()
    ids = torch.arange(16).expand(3, 16).contiguous().to(device)
    teacher = torch.log_softmax(_logits(3, 16, torch.float32, 53), -1).to(device)
    for tail in (False, True):
        loss = ops.distillation_loss(logits, ids, teacher, tail=tail)
        grad, = torch.autograd.grad(loss.total, logits)
        want = torch.log_softmax(logits.detach().double(), -1)
        q = teacher.double().exp()
        _close_rows(loss.rows, (q * (teacher.double() - want)).sum(-1).cpu(), 1e-4)
        _close_gradient(grad, (want.exp() - q).cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_distillation_ignored_rows_are_not_read(device):
    logits = _logits(3, 100, torch.float32, 54, device)
    logits[1] = float("nan")
    logits.requires_grad_()
    ids = torch.tensor([[1, 2], [-1, -1], [5, -100]], device=device)
    teacher = torch.tensor([[-0.5, -1.5], [0.0, 0.0], [-0.1, -INF]], device=device)
    loss = ops.distillation_loss(logits, ids, teacher)
    grad, = torch.autograd.grad(loss.total, logits)
    assert bool(loss.rows.isfinite().all()) and loss.rows[1] == 0 and bool((grad[1] == 0).all())
    assert bool(grad.isfinite().all()) and bool(loss.total.isfinite())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_upstream_gradient(device, dtype):
    logits = _logits(5, 777, dtype, 55, device).requires_grad_()
    ids, teacher = _teacher(logits.detach(), 8, 56)
    loss = ops.distillation_loss(logits, ids.to(device), teacher.to(device), tail=True)
    (loss.total * 0.25).backward()  # a power of two: the scaled gradient is the rounded one's
    _, want = _distillation(logits.detach(), ids, teacher, torch.full((5,), 0.25), 1.0, True)
    _close_gradient(logits.grad, want)
    assert not loss.rows.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 262144), (torch.float16, 262147), (torch.float32, 500003)])
def test_large_vocabularies(dtype, vocab):
    """Rows that a cluster of 16 blocks, or long stretches, hold."""
    logits = _logits(3, vocab, dtype, 90, "cuda").requires_grad_()
    ids, teacher = _teacher(logits.detach(), 64, 91)
    weights = torch.tensor([0.3, 1.0, 0.7])
    loss = ops.distillation_loss(logits, ids.cuda(), teacher.cuda(), weights.cuda(), tail=True)
    grad, = torch.autograd.grad(loss.total, logits)
    want_rows, want_grad = _distillation(logits.detach(), ids, teacher, weights, 1.0, True)
    _close_rows(loss.rows, want_rows, 1e-4)
    _close_gradient(grad, want_grad)
    targets = torch.tensor([0, vocab - 1, 77], device="cuda")
    got = ops.token_statistics(logits, targets, top=128)
    _check_statistics(logits.detach(), targets, 1.0, 128, S.TokenStatistics(*(x.detach() for x in got)))
    grad, = torch.autograd.grad(got.log_probs.sum() + got.entropy.sum(), logits)
    _close_gradient(grad, _statistics_gradient(logits.detach(), targets, 1.0, torch.ones(3), torch.ones(3)))


@pytest.mark.gpu
def test_operators_in_a_cuda_graph():
    logits = _logits(5, 30011, torch.bfloat16, 92, "cuda")
    ids, teacher = (x.cuda() for x in _teacher(logits, 8, 93))
    targets = torch.randint(0, 30011, (5,), device="cuda")
    hidden, weight, _ = _head(300, 64, 515, "cuda", torch.bfloat16, 94)
    aims = torch.randint(0, 515, (300,), device="cuda")

    def run():
        with torch.no_grad():
            s = ops.token_statistics(logits, targets, top=7)
            d = ops.distillation_loss(logits, ids, teacher, tail=True)
            h = ops.linear_token_statistics(hidden, weight, aims)
        return [*s, *d, h.log_probs, h.entropy]

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    logits.copy_(_logits(5, 30011, torch.bfloat16, 95, "cuda"))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, run()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_distillation_second_backward_is_refused():
    logits = _logits(2, 64, torch.float32, 57, "cuda").requires_grad_()
    loss = ops.distillation_loss(logits, torch.tensor([[1], [2]], device="cuda"), torch.zeros(2, 1, device="cuda"))
    loss.total.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="earlier backward"):
        loss.total.backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_gradient_against_differences(device, tail):
    logits = _logits(3, 41, torch.float32, 58, device)
    ids, teacher = _teacher(logits, 5, 59)
    weights, step = torch.tensor([0.5, 1.0, 0.8]), 1e-2

    def value(x):
        return ops.distillation_loss(x, ids.to(device), teacher.to(device), weights.to(device), temperature=1.5,
                                     tail=tail).total

    leaf = logits.clone().requires_grad_()
    value(leaf).backward()
    for r, i in ((0, int(ids[0, 0])), (0, 11), (1, 3), (2, int(ids[2, 0])), (2, 0)):
        up, down = logits.clone(), logits.clone()
        up[r, i] += step
        down[r, i] -= step
        slope = (float(value(up)) - float(value(down))) / (2 * step)
        assert abs(slope - float(leaf.grad[r, i])) < step ** 2 + 2e-5 / step


@pytest.mark.parametrize("device", DEVICES)
def test_statistics_feed_distillation(device):
    """A teacher's records (ignored rows and masked tokens among them) distil a student equal to it to zero."""
    logits = _logits(6, 200, torch.float32, 61, device)
    logits[:, 150:] = -INF
    targets = torch.tensor([3, -100, 7, 9, -100, 1], device=device)
    records = ops.token_statistics(logits, targets, temperature=2.0, top=10)
    student = logits.clone().requires_grad_()
    loss = ops.distillation_loss(student, records.top_ids, records.top_log_probs, temperature=2.0, tail=True)
    grad, = torch.autograd.grad(loss.total, student)
    assert bool((loss.rows.abs() < 1e-5).all()) and bool((grad.abs() < 1e-6).all())


def test_distillation_refusals():
    x = torch.randn(3, 8)
    ids, t = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    for bad_ids, bad_t, match in ((ids[:2], t[:2], "over the logits' rows"), (ids, t[:, :1], "over the logits' rows"),
                                  (ids[:, :0], t[:, :0], "1 to 128"),
                                  (torch.zeros(3, 129, dtype=torch.int64), torch.zeros(3, 129), "1 to 128"),
                                  (ids + 8, t, "outside the vocabulary")):
        with pytest.raises(ValueError, match=match):
            ops.distillation_loss(x, bad_ids, bad_t)
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.distillation_loss(x, ids.float(), t)
    with pytest.raises(ValueError, match="one value per row"):
        ops.distillation_loss(x, ids, t, torch.ones(2))
    with pytest.raises(ValueError, match="temperature"):
        ops.distillation_loss(x, ids, t, temperature=-2.0)


@pytest.mark.gpu
def test_distillation_ids_beyond_the_vocabulary_set_the_status():
    x = _logits(2, 64, torch.float32, 62, "cuda").requires_grad_()
    ids = torch.tensor([[1, 64], [2, 3]], device="cuda")
    loss = ops.distillation_loss(x, ids, torch.full((2, 2), -1.0, device="cuda"), tail=True)
    grad, = torch.autograd.grad(loss.total, x)
    assert loss.rows.isnan().tolist() == [True, False] and bool(grad[1].isfinite().all())
    with pytest.raises(ops.DeviceStatusError, match="out of bounds"):
        ops.check_status("distillation")


# -- together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
def test_distillation_example(device):
    path = Path(__file__).resolve().parents[1] / "examples" / "distill" / "distill_top_logits.py"
    spec = importlib.util.spec_from_file_location(path.stem, path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    rows = example.main(["--steps", "12", "--top", "8", "--device", device, "--seq-len", "16"])
    losses = [r["loss"] for r in rows if r["event"] == "train"]
    assert len(losses) == 12 and all(map(math.isfinite, losses)) and losses[-1] < 0.8 * losses[0]
    assert rows[0]["event"] == rows[-1]["event"] == "evaluate"
    assert 0 < rows[-1]["entropy"] < rows[0]["entropy"] <= math.log(256) + 1e-3  # the student took on opinions


@pytest.mark.parametrize("device", DEVICES)
def test_lm_head_statistics_mode(device):
    from tiny_dsv41_b200.models.common import LMHead

    torch.manual_seed(0)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    head = LMHead(64, 300).to(device, dtype)
    hidden = torch.randn(2, 5, 64, device=device, dtype=dtype)
    targets = torch.randint(0, 300, (2, 5), device=device)
    got = head(hidden, targets, mode="statistics", temperature=0.7)
    want = _statistics((hidden.double() @ head.weight.detach().double().t()).reshape(10, 300).cpu(), targets.reshape(-1).cpu(), 0.7, 0)
    _close_rows(got.log_probs.detach().reshape(-1), want["log_probs"], 3e-5, 1e-5)
    _close_rows(got.entropy.detach().reshape(-1), want["entropy"], 3e-4)
