"""Token scoring and distillation at inputs where they can go wrong: operands at odd addresses, candidates that
arrive while they are selected, repeated alternatives, weights of zero, upstream gradients, masks of a type's lowest value.

The definitions are restated here in 64 bits. Tolerances are those of the kernels' arithmetic: fp32 sums over a row are
off by 1e-5 of themselves, the entropy by 1e-4, a gradient by 2e-5 of its row's largest value and one rounding to its
type (half a unit in the last place: 2^-9 to 2^-8 of a bf16 value, 2^-12 to 2^-11 of a normal fp16 value, and fp16's
smallest step of 6e-8).
"""

import pytest
import torch

from tiny_dsv41_b200 import ops

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    if torch.cuda.is_available():
        ops.check_status("test")


def _generator(seed):
    return torch.Generator().manual_seed(seed)


def _scores(logits, targets, temperature=1.0):
    """(log-probabilities, entropy) of rows of 64-bit logits; an ignored row has zeros."""
    lp = torch.log_softmax(logits.double().cpu() / temperature, -1)
    targets = targets.cpu()
    keep = targets != -100
    chosen = lp.gather(-1, targets.clamp(min=0)[:, None])[:, 0]
    entropy = -(lp.exp() * lp).nan_to_num(0.0).sum(-1)
    return torch.where(keep, chosen, 0.0), torch.where(keep, entropy, 0.0)


# -- operands at odd addresses ----------------------------------------------------------------------
def _at_offset(x, offset):
    """A contiguous copy of ``x`` that starts ``offset`` elements into an allocation."""
    flat = torch.empty(x.numel() + offset, dtype=x.dtype, device=x.device)
    out = flat[offset:].view(x.shape)
    out.copy_(x)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [20, 256, 257, 600])
def test_head_operands_at_odd_addresses(rows):
    """TMA and the gather of the kept rows read 16 bytes at a time: the operator copies, the extension refuses."""
    g = _generator(1)
    hidden, weight = torch.randn(rows, 64, generator=g).bfloat16().cuda(), torch.randn(515, 64, generator=g).bfloat16().cuda()
    targets = torch.randint(0, 515, (rows,), generator=g).cuda()
    targets[1] = -100
    want = ops.linear_token_statistics(hidden, weight, targets)
    for offset in (1, 4):
        h, w = _at_offset(hidden, offset), _at_offset(weight, offset)
        assert h.is_contiguous() and h.data_ptr() % 16 != 0
        for a, b in ((h, weight), (hidden, w)):
            with pytest.raises(RuntimeError, match="16-byte"):
                ops.ext().lm_head_stats_fwd(a, b, targets, 1.0, -100, False, False)
            got = ops.linear_token_statistics(a, b, targets)
            assert torch.equal(got.log_probs, want.log_probs) and torch.equal(got.entropy, want.entropy)
        h.requires_grad_(), w.requires_grad_()
        trained = ops.linear_token_statistics(h, w, targets)
        trained.log_probs.sum().backward()
        assert h.grad.shape == h.shape and w.grad.shape == w.shape and bool(h.grad.isfinite().all())


# -- alternatives -----------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,rows,vocab", [(torch.bfloat16, 640, 70001), (torch.float32, 600, 33003),
                                              (torch.float16, 700, 40000), (torch.bfloat16, 3, 151936)])
@pytest.mark.parametrize("top", [1, 20, 128])
def test_alternatives_while_candidates_arrive(device, dtype, rows, vocab, top):
    """Rows that keep adding candidates while a threshold is raised over them: rising in part, in steps, everywhere."""
    if device == "cpu":
        rows = min(rows, 8)
    x = torch.randn(rows, vocab, generator=_generator(vocab))
    ramp = torch.arange(vocab) / vocab
    x[0::4] += 12.0 * ramp                                    # each batch holds larger values than the one before
    x[1::4] = (x[1::4] + 8.0 * ramp).round()                  # ... with many equal ones
    x[2::8] = 40.0 * ramp                                     # rising throughout: the candidates do not fit
    x[2::8, ::97] = -INF
    x = x.to(dtype).to(device)
    got = ops.token_statistics(x, top=top)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids, order)
    want = torch.log_softmax(x.double(), -1).gather(-1, order)
    assert bool(((got.top_log_probs - want).abs() <= 1e-5 + 1e-6 * want.abs()).all())
