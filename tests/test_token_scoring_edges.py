"""Token scoring and distillation at inputs where they can go wrong: operands at odd addresses, candidates that
arrive while they are selected, repeated alternatives, weights of zero, upstream gradients, masks of a type's lowest value.

The definitions are restated here in 64 bits. Tolerances are those of the kernels' arithmetic: fp32 sums over a row are
off by 1e-5 of themselves, the entropy by 1e-4, a gradient by 2e-5 of its row's largest value and one rounding to its
type (half a unit in the last place: 2^-9 to 2^-8 of a bf16 value, 2^-12 to 2^-11 of a normal fp16 value, and fp16's
smallest step of 6e-8).
"""

import pytest
import torch
from torch.autograd import forward_ad

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


# -- distillation -----------------------------------------------------------------------------------
def _distillation(logits, ids, teacher, weights, temperature, tail):
    """(rows' divergences, gradient) over the vocabulary: a token's mass is the sum of its places'."""
    x, ids, t = logits.detach().double().cpu(), ids.cpu().long(), teacher.double().cpu()
    there, at = ids >= 0, ids.cpu().clamp(min=0)
    q = torch.zeros_like(x).scatter_add_(-1, at, t.exp().masked_fill(~there, 0.0))
    inside = torch.zeros_like(x).scatter_add_(-1, at, there.double()) > 0
    read = inside.any(-1) if tail else q.sum(-1) > 0
    lp = torch.log_softmax(x / temperature, -1)
    p, left = lp.exp(), lp.masked_fill(inside, -INF).logsumexp(-1)
    rest = torch.zeros(len(x), dtype=torch.float64)
    if tail:
        rest = torch.where(left > -INF, (1 - q.sum(-1)).clamp(min=0), rest)
    else:
        q = q / torch.where(read, q.sum(-1), 1.0)[:, None]
    rows = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(-1)
    rows = (rows + torch.where(rest > 0, rest * (rest.log() - left), 0.0)).masked_fill(~read, 0.0)
    # (the rest's own distribution, not exp(lp - left): at -5e38 a difference of logarithms is below 64 bits)
    share = torch.softmax((x / temperature).masked_fill(inside, -INF), -1)
    outside = torch.where((rest > 0)[:, None] & ~inside, share * rest[:, None], 0.0)
    grad = (q.sum(-1) + rest)[:, None] * p - q - outside
    return rows, grad.masked_fill(~read[:, None], 0.0) * (weights.double().cpu() / temperature)[:, None]


def _close_gradient(got, want, relative=2e-5):
    """Within `relative` of the row's largest value, and half a unit in the last place of the type."""
    dtype, got = got.dtype, got.double().cpu()
    half_unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 0.0}[dtype]
    bound = relative * want.abs().amax(-1, keepdim=True) + half_unit * want.abs()
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert bool(((got - want).abs() <= bound + 1e-30).all()), ((got - want).abs() / (bound + 1e-30)).max()


def _close_loss(got, want):
    got = got.detach().double().cpu()
    assert bool(((got - want).abs() <= 1e-4 + 1e-5 * want.abs()).all()), (got - want).abs().max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab,k", [(9, 7), (2051, 6), (2051, 128), (151936, 64)])
def test_repeated_alternatives_are_one_token(device, dtype, tail, vocab, k):
    g = _generator(vocab + k)
    rows = 6
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).to(device)
    logits[2] = 0.0
    teacher = torch.log_softmax(torch.randn(rows, k, generator=g), -1) - 0.2
    ids = torch.randint(0, max(2, k // 2), (rows, k), generator=g) * (vocab // k)
    ids[1] = vocab - 1                        # one token throughout
    ids[2, : min(k, 6)] = torch.tensor([7, 7, 8, -1, 8, 7])[:k]
    ids[3, 1:] = -1                           # nothing repeated but the absent
    teacher[4, ::2] = -INF                    # places without mass
    weights = torch.rand(rows, generator=g)
    leaf = logits.clone().requires_grad_()
    loss = ops.distillation_loss(leaf, ids.to(device), teacher.to(device), weights.to(device), temperature=1.3, tail=tail)
    want, want_grad = _distillation(logits, ids, teacher, weights, 1.3, tail)
    _close_loss(loss.rows, want)
    assert bool((loss.rows >= -1e-6).all())   # a divergence
    grad, = torch.autograd.grad(loss.total, leaf)
    _close_gradient(grad, want_grad)


@pytest.mark.parametrize("device", DEVICES)
def test_repeated_alternatives_of_an_equal_student(device):
    """A teacher equal to the student with a token recorded as two halves is at distance zero."""
    logits = torch.zeros(2, 8, device=device)
    ids = torch.tensor([[3, 3, 5], [3, 5, -1]], device=device)
    share = torch.tensor([[1 / 16, 1 / 16, 1 / 8], [1 / 8, 1 / 8, 0.0]], device=device)
    rows = ops.distillation_loss(logits, ids, share.log(), tail=True).rows
    assert bool((rows.abs() < 1e-6).all())
    one = ops.distillation_loss(torch.tensor([[-INF, 2.0]], device=device), torch.tensor([[1, 1]], device=device),
                                torch.full((1, 2), 0.5, device=device).log())
    assert abs(float(one.rows)) < 1e-6


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_of_special_rows(device, tail):
    """Rows at which a maximum, a mask or a mass can go wrong, repeated ids among them."""
    vocab, g = 2051, _generator(60)
    x = torch.randn(12, vocab, generator=g) * 3
    x[1, 1:] = -INF                             # one token left
    x[2] = 0.0
    x[3] = torch.arange(vocab) * 0.01
    x[4] += 1.0e4
    x[5, ::2] = -INF
    x[6, 5:] = -1.0e4
    x[7, -1] = 80.0
    x[8, :-6] -= 200.0                          # the student's mass is all on the alternatives
    ids = torch.stack([torch.randperm(vocab, generator=g)[:6] for _ in range(12)])
    teacher = torch.log_softmax(torch.randn(12, 6, generator=g), -1) - 0.2
    ids[1, 0], ids[7, 0], ids[8] = 0, vocab - 1, torch.arange(vocab - 6, vocab)
    ids[1, 1:], ids[5] = -1, torch.arange(1, 13, 2)
    ids[2] = torch.tensor([7, 7, 9, -1, 9, 7])
    teacher[3, 2:] = -INF
    teacher[9] -= 60.0                          # nearly all of the teacher's mass in the tail
    teacher[10] = -0.7                          # more than one in all
    weights = torch.linspace(0.1, 1.0, 12)
    leaf = x.to(device).requires_grad_()
    loss = ops.distillation_loss(leaf, ids.to(device), teacher.to(device), weights.to(device), tail=tail)
    want, want_grad = _distillation(x, ids, teacher, weights, 1.0, tail)
    _close_loss(loss.rows, want)
    grad, = torch.autograd.grad(loss.total, leaf)
    _close_gradient(grad, want_grad)


def _pair(rows, vocab, k, seed, dtype=torch.float32):
    g = _generator(seed)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    values, ids = torch.log_softmax(logits.float() + torch.randn(rows, vocab, generator=g), -1).topk(k, dim=-1)
    return logits, ids, values


@pytest.mark.parametrize("device", DEVICES)
def test_distillation_total_is_updated_in_place(device):
    """A total is a tensor of its own: `total += other` and `total *= factor` are what they are elsewhere."""
    logits, ids, teacher = _pair(5, 300, 8, 70)
    _, want = _distillation(logits, ids, teacher, torch.full((5,), 0.5), 1.0, True)
    leaf = logits.to(device).requires_grad_()
    total = ops.distillation_loss(leaf, ids.to(device), teacher.to(device), tail=True).total
    assert total.shape == () and not total._is_view()
    total += 1.0
    total *= 0.5
    total.backward()
    _close_gradient(leaf.grad, want)
    other = ops.token_statistics(leaf, ids[:, 0].to(device), top=2)
    for x in (other.log_probs, other.entropy, other.top_log_probs):
        x *= 2.0
    other.entropy.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab", [300, 40003])
def test_a_weight_of_zero_masks_its_row(device, dtype, tail, vocab):
    logits, ids, teacher = _pair(8, vocab, 8, 71, dtype)
    weights = torch.tensor([0.5, 0.0, 0.0, 0.0, 0.25, 0.0, -0.0, 1.0])
    want, want_grad = _distillation(logits, ids, teacher, weights, 1.0, tail)
    logits[1] = -INF                       # no distribution
    logits[2] = float("nan")
    logits[3, ids[3, 0]] = -INF            # the teacher's first alternative is impossible: infinite
    logits[5, 17] = INF
    leaf = logits.to(device).requires_grad_()
    loss = ops.distillation_loss(leaf, ids.to(device), teacher.to(device), weights.to(device), tail=tail)
    loss.total.backward()
    off = weights == 0
    _close_loss(loss.total, (want * weights.double()).sum())
    _close_gradient(leaf.grad, want_grad)
    assert bool((leaf.grad[off.to(device)] == 0).all())
    _close_loss(loss.rows[[0, 4, 6, 7]], want[[0, 4, 6, 7]])   # a masked row's divergence is reported
    assert loss.rows[1] == INF and loss.rows[3] == INF and bool(loss.rows[2].isnan()) and bool(loss.rows[5].isnan())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("factor,share", [(65536.0, 1 / 4096), (0.3, 1.0), (0.0, 1.0), (-1.7, 0.5)])
@pytest.mark.parametrize("vocab", [777, 70001])
def test_distillation_gradient_is_rounded_after_the_upstream_factor(device, dtype, tail, factor, share, vocab):
    """One rounding to the logits' type, whatever multiplies the total: a loss scale reaches fp16's small values."""
    logits, ids, teacher = _pair(7, vocab, 16, 72, dtype)
    ids[1], ids[2, 8:], ids[3, 1] = -1, -1, ids[3, 0]
    weights = torch.full((7,), share)
    weights[4] = 0.0
    _, want = _distillation(logits, ids, teacher, weights * factor, 1.3, tail)
    for view in (False, True):
        leaf = torch.cat((logits, logits[:, :3]), 1).to(device)[:, :vocab] if view else logits.to(device)
        leaf = leaf.detach().requires_grad_()
        for i in (ids, ids.int()):
            loss = ops.distillation_loss(leaf, i.to(device), teacher.to(device), weights.to(device), temperature=1.3, tail=tail)
            grad, = torch.autograd.grad(loss.total * factor, leaf)
            _close_gradient(grad, want)


@pytest.mark.parametrize("device", DEVICES)
def test_distillation_under_saved_tensor_hooks(device):
    """What the backward needs is saved where hooks (offloading, checkpointing) see it."""
    from torch.utils.checkpoint import checkpoint

    logits, ids, teacher = _pair(4, 500, 8, 73)
    args = (ids.to(device), teacher.to(device))
    _, want = _distillation(logits, ids, teacher, torch.ones(4), 1.0, True)
    seen = []

    def pack(x):
        seen.append(tuple(x.shape))
        return x.cpu()

    leaf = logits.to(device).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x.to(device)):
        total = ops.distillation_loss(leaf, *args, tail=True).total
    assert (4, 500) in seen
    total.backward()
    _close_gradient(leaf.grad, want)
    leaf.grad = None
    checkpoint(lambda x: ops.distillation_loss(x, *args, tail=True).total, leaf, use_reentrant=False).backward()
    _close_gradient(leaf.grad, want)


# -- masks of the type's lowest value ---------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [40, 3001])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
def test_masks_of_the_lowest_value(device, dtype, vocab, temperature):
    """A masked token's log-probability is (lowest - m) / T - ln S wherever fp32 holds that, and -inf beyond."""
    x = torch.randn(5, vocab, generator=_generator(74)) * 3
    x[:, 6:] = torch.finfo(dtype).min
    x[2] = torch.finfo(dtype).min
    x[3, 1:] = torch.finfo(dtype).min
    x[4, 20:] = -INF
    x = x.to(dtype).to(device)
    targets = torch.tensor([vocab - 1, 2, 7, 0, 9], device=device)
    got = ops.token_statistics(x, targets, temperature=temperature, top=10)
    lp = torch.log_softmax(x.double() / temperature, -1).float()   # (beyond fp32: -inf)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :10]
    assert torch.equal(got.top_ids, order)
    chosen, entropy = _scores(x, targets, temperature)
    for a, b in ((got.log_probs, chosen.float()), (got.top_log_probs, lp.gather(-1, order).cpu())):
        a = a.cpu()
        assert torch.equal(a == -INF, b == -INF), (a, b)
        fine = b > -INF
        assert bool(((a - b).abs()[fine] <= 1e-5 + 1e-6 * b.abs()[fine]).all()), (a, b)
    assert bool(((got.entropy.cpu() - entropy).abs() <= 1e-4).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_of_tokens_masked_by_the_lowest_value(device, dtype, tail):
    """A teacher whose alternatives the student masks: a divergence of 1e38 and a gradient of -q, not infinities."""
    x = torch.randn(3, 600, generator=_generator(75)) * 3
    x[0, :8] = x[1, 3:8] = torch.finfo(dtype).min
    x = x.to(dtype)
    ids, teacher = torch.arange(8).expand(3, 8).contiguous(), torch.full((3, 8), -2.5)
    want, want_grad = _distillation(x, ids, teacher, torch.ones(3), 1.0, tail)
    leaf = x.to(device).requires_grad_()
    loss = ops.distillation_loss(leaf, ids.to(device), teacher.to(device), tail=tail)
    assert bool(loss.rows.isfinite().all())
    _close_loss(loss.rows, want)
    grad, = torch.autograd.grad(loss.total, leaf)
    _close_gradient(grad, want_grad)


# -- autograd ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_tangents_are_refused(grad):
    """The kernels have no forward-mode derivative: a tangent is refused, with gradients on or off, not dropped."""
    x = torch.randn(3, 64, device="cuda")
    hidden, weight = torch.randn(3, 64, device="cuda").bfloat16(), torch.randn(100, 64, device="cuda").bfloat16()
    targets, ids = torch.tensor([1, 2, 3], device="cuda"), torch.tensor([[1], [2], [3]], device="cuda")
    teacher = torch.zeros(3, 1, device="cuda")
    calls = ((x, lambda d: ops.token_statistics(d, targets, top=3)),
             (x, lambda d: ops.distillation_loss(d, ids, teacher)),
             (hidden, lambda d: ops.linear_token_statistics(d, weight, targets)),
             (weight, lambda d: ops.linear_token_statistics(hidden, d, targets)))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for primal, call in calls:
            with pytest.raises((RuntimeError, NotImplementedError), match="forward mode|jvp"):
                call(forward_ad.make_dual(primal, torch.ones_like(primal)))
        ops.token_statistics(x, targets)


@pytest.mark.gpu
def test_gradients_in_a_cuda_graph():
    """Forward and backward of the three operators captured once and replayed on other inputs."""
    g = _generator(76)
    logits, ids, teacher = _pair(6, 20011, 8, 77, torch.bfloat16)
    logits, ids, teacher = logits.cuda(), ids.cuda(), teacher.cuda()
    targets = torch.randint(0, 515, (6,), generator=g).cuda()
    hidden, weight = torch.randn(6, 64, generator=g).bfloat16().cuda(), torch.randn(515, 64, generator=g).bfloat16().cuda()
    for x in (logits, hidden, weight):
        x.requires_grad_()
    factor = torch.tensor(0.3, device="cuda")

    def run():
        s = ops.token_statistics(logits, targets, top=7)
        d = ops.distillation_loss(logits, ids, teacher, tail=True)
        h = ops.linear_token_statistics(hidden, weight, targets)
        grads = torch.autograd.grad(s.log_probs.sum() + s.top_log_probs.sum() + d.total * factor, logits)
        grads += torch.autograd.grad(h.log_probs.sum() + h.entropy.sum(), (hidden, weight))
        return [x.detach() for x in (*s, *d, h.log_probs, h.entropy, *grads)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    with torch.no_grad():
        logits.copy_(torch.randn(6, 20011, generator=g) * 3)
        hidden.copy_(torch.randn(6, 64, generator=g))
        factor.fill_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, run()):
        assert torch.equal(a, b)


# -- the LM head ------------------------------------------------------------------------------------
def _head(rows, hidden, vocab, seed):
    g = _generator(seed)
    h = torch.randn(rows, hidden, generator=g).bfloat16()
    w = (torch.randn(vocab, hidden, generator=g) * 3 / hidden ** 0.5).bfloat16()
    t = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 2:
        t[1] = -100
    return h.cuda(), w.cuda(), t.cuda()


def _close_scores(got, logits, targets, temperature):
    # a logit is a sum of up to 2048 products in fp32: 1e-5 at most (of values up to 15)
    lp, entropy = _scores(logits, targets, temperature)
    assert bool(((got.log_probs.detach().cpu() - lp).abs() <= 3e-5 + 1e-5 * lp.abs()).all())
    assert bool(((got.entropy.detach().cpu() - entropy).abs() <= 3e-4).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 31, 32, 33, 128, 129])
@pytest.mark.parametrize("hidden", [72, 2048])
@pytest.mark.parametrize("vocab", [1003, 40007, 151669])
def test_head_of_few_rows(rows, hidden, vocab):
    """Several tiles to a block, a ring that wraps, narrow and partial tiles, a partial block of the hidden dimension."""
    h, w, t = _head(rows, hidden, vocab, rows + vocab)
    t[0] = vocab - 1
    got = ops.linear_token_statistics(h, w, t, temperature=0.8)
    _close_scores(got, h.double() @ w.double().t(), t, 0.8)
    again = ops.linear_token_statistics(h, w, t, temperature=0.8)
    assert torch.equal(got.log_probs, again.log_probs) and torch.equal(got.entropy, again.entropy)


@pytest.mark.gpu
@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("rows,hidden,vocab", [(5, 72, 257), (130, 256, 515), (300, 128, 4099), (129, 2048, 1000),
                                               (40, 512, 20011)])
def test_head_gradients_value_by_value(monkeypatch, kept, rows, hidden, vocab):
    """The logits' gradient is rounded to bf16 once (2^-8 of each value, beside 3e-5 of its row's largest from the
    statistics and the fp32 logits) before the products, whose results are rounded once more: each value of a
    gradient is within what its own terms allow."""
    if not kept:
        monkeypatch.setattr(ops.statistics, "KEPT_BYTES", 0)
    h, w, t = _head(rows, hidden, vocab, 78)
    g = _generator(79)
    up, down = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    h.requires_grad_(), w.requires_grad_()
    got = ops.linear_token_statistics(h, w, t, temperature=0.7)
    logits = h.detach().double() @ w.detach().double().t()
    _close_scores(got, logits, t, 0.7)
    torch.autograd.backward((got.log_probs, got.entropy), (up.cuda(), down.cuda()))
    lp = torch.log_softmax(logits / 0.7, -1)
    p = lp.exp()
    entropy = -(p * lp).sum(-1, keepdim=True)
    one = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    d = (up.cuda().double()[:, None] * (one - p) - down.cuda().double()[:, None] * p * (lp + entropy)) / 0.7
    d = d * (t != -100)[:, None]
    off = 2.0 ** -8 * d.abs() + 3e-5 * d.abs().amax(-1, keepdim=True)
    hd, wd = h.detach().double(), w.detach().double()
    for grad, want, bound in ((h.grad, d @ wd, off @ wd.abs()), (w.grad, d.t() @ hd, off.t() @ hd.abs())):
        bound = bound + 2.0 ** -8 * want.abs() + 1e-30
        assert bool(((grad.double() - want).abs() <= bound).all()), ((grad.double() - want).abs() / bound).max()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 40, 300])
@pytest.mark.parametrize("grad", [False, True])
def test_head_bad_targets_and_nan_rows(rows, grad):
    h, w, t = _head(rows, 64, 1003, 80)
    h[2], h[3, 5] = float("nan"), INF
    t[0] = 7
    h.requires_grad_(grad)
    got = ops.linear_token_statistics(h, w, t)
    assert bool(got.log_probs[2:4].isnan().all()) and bool(got.entropy[2:4].isnan().all())
    fine = [0] + list(range(4, rows))
    picked = type(got)(got.log_probs[fine], got.entropy[fine])
    _close_scores(picked, h.detach()[fine].double() @ w.double().t(), t[fine], 1.0)
    assert got.log_probs[1] == 0 and got.entropy[1] == 0
    ops.check_status("head")
    t[0] = 1003
    bad = ops.linear_token_statistics(h, w, t)
    assert bool(bad.log_probs[0].isnan()) and bool(bad.entropy[0].isfinite())
    with pytest.raises(ops.DeviceStatusError, match="out of bounds"):
        ops.check_status("head")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_gradient_of_a_rest_masked_by_the_lowest_value(device, dtype, temperature):
    """Every token outside the alternatives has the same share of the teacher's rest, however unlikely all of them are."""
    x = torch.randn(2, 600, generator=_generator(82)) * 3
    x[0, 2:] = torch.finfo(dtype).min
    x[1, 5:] = -1.0e30
    x = x.to(dtype)
    ids, share = torch.tensor([[0, 1], [0, 3]]), torch.tensor([[0.45, 0.45], [0.3, 0.2]])
    _, want_grad = _distillation(x, ids, share.log(), torch.ones(2), temperature, True)
    leaf = x.to(device).requires_grad_()
    total = ops.distillation_loss(leaf, ids.to(device), share.log().to(device), temperature=temperature, tail=True).total
    grad, = torch.autograd.grad(total, leaf)
    _close_gradient(grad, want_grad)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.6, 2.0])
def test_divergences_of_tokens_masked_by_the_lowest_value_below_fp32s_edge(device, dtype, temperature):
    """q (lowest - m) / T fits fp32 although (lowest - m) / T does not: 1e37 and 2e38, not infinities."""
    x = torch.randn(4, 600, generator=_generator(81)) * 3
    x[0, :2] = x[1, :2] = torch.finfo(dtype).min
    x[2, 2:] = torch.finfo(dtype).min            # the rest of the vocabulary is masked
    x = x.to(dtype)
    ids = torch.tensor([[0, 1]] * 4)
    share = torch.tensor([[0.01, 0.01], [0.2, 0.15], [0.45, 0.45], [0.3, 0.2]])
    want, want_grad = _distillation(x, ids, share.log(), torch.ones(4), temperature, True)
    assert bool((want < 3e38).all()) and bool((want[:3] > 1e36).all())
    leaf = x.to(device).requires_grad_()
    loss = ops.distillation_loss(leaf, ids.to(device), share.log().to(device), temperature=temperature, tail=True)
    _close_loss(loss.rows, want)
    grad, = torch.autograd.grad(loss.total, leaf)
    _close_gradient(grad, want_grad)
