"""The operators of a decoding step against definitions in 64 bits, and their refusals.

Tolerances, with u half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24; nothing for the 64-bit inputs of the CPU) and
values rounded once at the end:

* append: the mean of 128 squares, its root, two products and the rotation are some ten fp32 roundings of the parts
  a cos and b sin: 1e-6 (|a| + |b|), and u of the result. The sine and cosine are off by 2^-21 beside 1: 1e-6 more.
* attention: a score is a sum of 128 products in fp32, which a tensor core may cut instead of rounding: off by
  2^-20 of S = scale sum |q_i k_i| at most, and so is a weight relative to itself, beside 2^-20 of the exponential and of
  the joins. A weight is rounded to the type for its product with v (u). With A = sum p |v| / sum p the result is off by
  (u + 2^-19 (S + 2)) A, and by u of itself.
* logits: five fp32 roundings of values up to M = |x| (r or 1 / r) + f c + p + sum |b|: 2^-21 M, and u of the result.

The smallest step of fp16 (2^-24) is added to all.
"""

import math

import pytest
import torch

from tiny_dsv41_b200 import ops
from tiny_dsv41_b200.ops import PagedBatch

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF_STEP = {torch.float64: 0.0, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = 2.0 ** -24
DIM = 128
FREQS = 1e6 ** (-torch.arange(0, DIM, 2, dtype=torch.float32) / DIM)


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    if torch.cuda.is_available():
        ops.check_status("test")


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _close(got, want, room):
    """`got` within `room` (values or a number) of the 64-bit `want`."""
    got = got.double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    assert bool((off <= room).all()), f"off by {float((off - room).max())} more than allowed"


def _batch(new, lengths, page, *, device="cpu", seed=0, spare=2, extra=0, width=None):
    """A batch over shuffled pages of a pool; tables hold -1 behind a sequence's pages."""
    count = [-(-n // page) for n in lengths]
    width = max([1, *count]) if width is None else width
    order = torch.randperm(sum(count) + spare, generator=_gen(seed)).int()
    tables, at = torch.full((len(new), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(count):
        tables[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()] if new else [0], dtype=torch.int32)
    batch = PagedBatch(tables.to(device), starts.to(device), torch.tensor(lengths, dtype=torch.int32, device=device))
    return batch, sum(count) + spare, int(starts[-1]) + extra


def _place(batch, b, j, page):
    return int(batch.tables[b, j // page]), j % page


def _pool(pages, heads, page, dtype, device, layout="plain", seed=1, fill=None):
    """A cache, and its layout: dense, both sides in one tensor, or tokens before heads."""
    shape = (pages, heads, page, DIM)
    values = [torch.randn(shape, generator=_gen(seed + i)) for i in range(2)]
    if fill is not None:
        values = [torch.full(shape, fill) for _ in range(2)]
    if layout == "together":
        both = torch.stack(values, dim=1).to(dtype).to(device)
        return both[:, 0], both[:, 1]
    if layout == "tokens":
        return tuple(v.transpose(1, 2).contiguous().to(dtype).to(device).transpose(1, 2) for v in values)
    return tuple(v.to(dtype).to(device) for v in values)


# -- the definitions in 64 bits -----------------------------------------------------------------------
def _append_definition(qkv, wq, wk, positions, hq, hkv, eps):
    """(q, k, room of each) in 64 bits."""
    x = qkv.double().cpu().view(len(qkv), -1, DIM)[:, :hq + hkv]
    w = torch.cat((wq.double().cpu().expand(hq, DIM), wk.double().cpu().expand(hkv, DIM)))
    y = x / (x.square().sum(-1, keepdim=True) / DIM + eps).sqrt() * w
    a, b = y[..., :DIM // 2], y[..., DIM // 2:]
    angle = (positions.double().cpu()[:, None] * FREQS.double())[:, None]
    out = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), dim=-1)
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    return out, 2e-6 * size


def _attention_definition(q, keys, values, batch, scale, tree=None):
    """(out, room) in 64 bits, head by head."""
    rows, hq, _ = q.shape
    page, hkv = keys.shape[2], keys.shape[1]
    group = hq // hkv
    q, keys, values = q.double().cpu(), keys.cpu(), values.cpu()
    cpu = PagedBatch(batch.tables.cpu(), batch.starts.cpu(), batch.lengths.cpu())
    out, room = torch.zeros(rows, hq, DIM, dtype=torch.float64), torch.zeros(rows, hq, DIM, dtype=torch.float64)
    u = HALF_STEP[keys.dtype]
    for b, length in enumerate(cpu.lengths.tolist()):
        first, end = int(cpu.starts[b]), int(cpu.starts[b + 1])
        at = torch.arange(length)
        pages = cpu.tables[b].long()[at // page]
        k, v = keys[pages, :, at % page].double(), values[pages, :, at % page].double()  # [length, heads, dim]
        n = end - first
        if n == 0:
            continue
        j = at - (length - n)
        if tree is None:
            seen = j <= torch.arange(n)[:, None]
        else:
            words = torch.nn.functional.pad(tree[first:end], (0, 1))
            seen = (j < 0) | (words[:, (j // 32).clamp(0, tree.shape[1])] >> (j % 32).int() & 1 == 1)
        for h in range(hq):
            x, kk, vv = q[first:end, h], k[:, h // group], v[:, h // group]
            s = (x @ kk.T * scale).masked_fill(~seen, -INF)
            p = torch.softmax(s, 1).nan_to_num(nan=0.0)  # (a row that sees nothing)
            out[first:end, h] = p @ vv
            size = (x.abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
            room[first:end, h] = (u + 2.0 ** -19 * (size + 2)) * (p @ vv.abs())
    return out, room + u * out.abs() + SMALLEST


def _logits_definition(x, history, lengths, prompts, repetition, presence, frequency, bias_ids, bias, allowed):
    """(out, room without the rounding of the result) in 64 bits, token by token."""
    out = x.double().cpu().clone()
    room = out.abs().nan_to_num(posinf=0.0)
    for r in range(len(out)):
        if history is not None:
            ids = history[r].tolist()[:int(lengths[r]) if lengths is not None else None]
            prompt = int(prompts[r]) if prompts is not None else 0
            r_, p_, f_ = (float(v[r]) if v is not None else d for v, d in ((repetition, 1.0), (presence, 0.0),
                                                                           (frequency, 0.0)))
            for t in set(i for i in ids if i >= 0):
                out[r, t] = out[r, t] / r_ if out[r, t] > 0 else out[r, t] * r_
                times = sum(i == t for i in ids[prompt:])
                room[r, t] = out[r, t].abs() + abs(f_) * times + abs(p_)
                if times:
                    out[r, t] -= f_ * times + p_
        if bias is not None:
            for t, v in zip(bias_ids[r].tolist(), bias[r].tolist()):
                if t >= 0:
                    out[r, t] += v
                    room[r, t] += abs(v)
        if allowed is not None:
            for t in range(out.shape[1]):
                if not int(allowed[r, t // 32]) >> t % 32 & 1:
                    out[r, t] = -INF
    return out, 2.0 ** -21 * room + SMALLEST


# -- append -----------------------------------------------------------------------------------------
SEQUENCES = {
    "one": ([1], [1]),
    "one far on": ([1], [300]),
    "decode": ([1, 1, 1, 1, 1], [1, 16, 17, 33, 64]),
    "prompts": ([3, 40, 17], [3, 40, 17]),
    "mixed": ([0, 5, 1, 0, 20, 1], [9, 21, 100, 0, 20, 1]),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", SEQUENCES)
@pytest.mark.parametrize("heads, page, layout", [((4, 2), 16, "plain"), ((5, 1), 32, "together"), ((3, 3), 64, "tokens")])
def test_append(device, dtype, which, heads, page, layout):
    hq, hkv = heads
    new, lengths = SEQUENCES[which]
    batch, pages, rows = _batch(new, lengths, page, device=device, extra=2)
    keys, values = _pool(pages, hkv, page, dtype, device, layout)
    before = keys.clone(), values.clone()
    qkv = (torch.randn(rows, (hq + 2 * hkv) * DIM, generator=_gen(3)) * 2).to(dtype).to(device)
    wq, wk = ((1 + 0.2 * torch.randn(DIM, generator=_gen(s))).to(dtype).to(device) for s in (4, 5))
    positions = torch.randint(0, 40960, (rows,), generator=_gen(6)).to(device)
    q = ops.paged_append(qkv, wq, wk, positions, FREQS.to(device), hq, hkv, 1e-6, keys, values, batch)
    want, room = _append_definition(qkv, wq, wk, positions, hq, hkv, 1e-6)
    room = room + HALF_STEP[dtype] * want.abs() + SMALLEST
    assert q.dtype == dtype
    _close(q, want[:, :hq], room[:, :hq])
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for b, (n, length) in enumerate(zip(new, lengths)):
        for i in range(n):
            at, row = _place(batch, b, length - n + i, page)
            t = int(batch.starts[b]) + i
            touched[at, row] = True
            _close(keys[at, :, row], want[t, hq:], room[t, hq:])
            assert torch.equal(values[at, :, row], qkv.view(rows, -1, DIM)[t, hq + hkv:])
    for now, was in zip((keys, values), before):  # nothing else has changed
        assert torch.equal(now.transpose(1, 2)[~touched], was.transpose(1, 2)[~touched])


@pytest.mark.parametrize("device", DEVICES)
def test_append_many_rows(device):
    """More rows than one block a row takes, from rows of a wider tensor."""
    hq, hkv, page, new = 2, 1, 128, [700, 1, 555]
    batch, pages, rows = _batch(new, [701, 900, 555], page, device=device)
    keys, values = _pool(pages, hkv, page, torch.bfloat16, device)
    wide = torch.randn(rows, (hq + 2 * hkv) * DIM + 12, generator=_gen(3)).bfloat16().to(device)
    qkv = wide[:, 4:-8]
    w = torch.ones(DIM, dtype=torch.bfloat16, device=device)
    positions = torch.arange(rows, device=device) * 31
    q = ops.paged_append(qkv, w, w, positions, FREQS.to(device), hq, hkv, 1e-5, keys, values, batch)
    want, room = _append_definition(qkv.contiguous(), w, w, positions, hq, hkv, 1e-5)
    room = room + HALF_STEP[torch.bfloat16] * want.abs()
    _close(q, want[:, :hq], room[:, :hq])
    for b in range(3):
        n, length = new[b], int(batch.lengths[b])
        at = torch.arange(length - n, length)
        where = batch.tables[b].cpu().long()[at // page]
        first = int(batch.starts[b])
        _close(keys.cpu()[where, :, at % page], want[first:first + n, hq:], room[first:first + n, hq:])
        assert torch.equal(values.cpu()[where, :, at % page], qkv.cpu()[first:first + n, -DIM:].unsqueeze(1))


@pytest.mark.parametrize("device", DEVICES)
def test_append_odd_layouts(device):
    """qkv and weights that start off 8 bytes, positions of a batch [1, T], far positions, an empty call."""
    batch, pages, rows = _batch([3], [3], 16, device=device)
    keys, values = _pool(pages, 1, 16, torch.float16, device)
    flat = torch.randn(1 + rows * 3 * DIM, generator=_gen(2)).half().to(device)
    qkv = flat[1:].view(1, rows, 3 * DIM)
    w = torch.randn(DIM + 1, generator=_gen(9)).half().to(device)[1:]
    positions = torch.tensor([[0, 2 ** 20 + 1, 10 ** 9]], device=device)
    q = ops.paged_append(qkv, w, w, positions, FREQS.to(device), 1, 1, 1e-6, keys, values, batch)
    want, room = _append_definition(qkv[0], w, w, positions[0], 1, 1, 1e-6)
    _close(q, want[:, :1], room[:, :1] + HALF_STEP[torch.float16] * want[:, :1].abs() + SMALLEST)
    none = PagedBatch(batch.tables[:0], batch.starts[:1], batch.lengths[:0])
    q = ops.paged_append(qkv[0, :0], w, w, positions[0, :0], FREQS.to(device), 1, 1, 1e-6, keys, values, none)
    assert q.shape == (0, 1, DIM)


# -- attention --------------------------------------------------------------------------------------
def _attend(new, lengths, heads, page, dtype, device, *, layout="plain", tree=None, extra=0, scale=None, seed=0, sharp=1.0):
    hq, hkv = heads
    batch, pages, rows = _batch(new, lengths, page, device=device, seed=seed, extra=extra)
    keys, values = _pool(pages, hkv, page, dtype, device, layout, seed=seed + 1)
    # behind a sequence's length, and in pages that nobody has, stands what was there before
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, length in enumerate(lengths):
        for j in range(length):
            used[_place(batch, b, j, page)] = True
    for pool in (keys, values):
        pool.transpose(1, 2)[~used] = float("nan")
    q = (torch.randn(rows, hq, DIM, generator=_gen(seed + 9)) * sharp).to(dtype).to(device)
    if tree is not None:
        tree = tree.to(device)
    out = ops.paged_attention(q, keys, values, batch, scale=scale, tree=tree)
    assert out.shape == q.shape and out.dtype == dtype
    want, room = _attention_definition(q, keys, values, batch, DIM ** -0.5 if scale is None else scale,
                                       None if tree is None else tree.cpu())
    _close(out, want, room)
    return out


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 255, 257, 300]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, page, layout", [((8, 2), 16, "plain"), ((4, 4), 32, "together"), ((5, 1), 64, "tokens"),
                                                 ((16, 1), 128, "plain"), ((20, 1), 256, "plain")])
def test_attention_single_tokens(device, dtype, heads, page, layout):
    _attend([1] * len(LENGTHS), LENGTHS, heads, page, dtype, device, layout=layout, extra=3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new, lengths", [([1], [1]), ([1], [1000]), ([7], [7]), ([33], [33]), ([129], [129]), ([40], [171]),
                                          ([0, 3, 0, 0, 20, 1, 0], [5, 3, 0, 17, 150, 64, 1]), ([2, 65, 9], [130, 65, 140])])
@pytest.mark.parametrize("heads, page", [((4, 2), 16), ((6, 2), 64), ((8, 1), 32)])
def test_attention_several_tokens(device, new, lengths, heads, page):
    _attend(new, lengths, heads, page, torch.bfloat16, device, extra=1, sharp=3.0)


@pytest.mark.gpu
def test_attention_long_and_many():
    """One sequence of many blocks beside short ones, and more sequences than threads."""
    _attend([1, 2, 1], [9001, 5, 4000], (8, 2), 64, torch.bfloat16, "cuda")
    new = [(b * 7) % 3 for b in range(300)]
    _attend(new, [n + (b * 37) % 90 for b, n in enumerate(new)], (2, 1), 16, torch.float16, "cuda", seed=5)


@pytest.mark.gpu
def test_attention_of_wide_groups():
    """More heads of one key head than a tile has rows, and as many."""
    _attend([1, 3], [40, 200], (260, 1), 16, torch.bfloat16, "cuda")
    _attend([1, 3], [40, 200], (256, 1), 16, torch.bfloat16, "cuda")
    _attend([2, 1], [300, 7], (200, 1), 64, torch.float16, "cuda", tree=_random_tree([2, 1], 1, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("heads, page, dtype", [((8, 1), 16, torch.bfloat16), ((5, 1), 64, torch.float16),
                                                ((6, 2), 128, torch.bfloat16), ((48, 1), 32, torch.bfloat16)])
def test_attention_of_prompts(heads, page, dtype):
    """Tiles of many rows: ragged ends, cached prefixes, tiles that several blocks share, sequences without new tokens."""
    _attend([700, 0, 3, 1, 257], [1900, 40, 5, 1, 257], heads, page, dtype, "cuda", extra=2, sharp=3.0)
    _attend([1100], [1100], heads, page, dtype, "cuda")
    _attend([100, 64, 31] * 9, [6000, 64, 900] * 9, heads, page, dtype, "cuda", sharp=2.0)


def _random_tree(new, words, seed, device="cpu"):
    parents, gen = [], _gen(seed)
    for n in new:
        parents += [int(torch.randint(-1, j, (1,), generator=gen)) if j else -1 for j in range(n)]
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()])
    return ops.tree_mask(torch.tensor(parents), starts, words)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("new, lengths", [([1], [1]), ([7], [7]), ([32], [40]), ([33, 0, 5], [200, 4, 130]),
                                          ([70, 64], [200, 64]), ([128], [300]), ([60] * 5, [1000, 60, 61, 127, 129])])
@pytest.mark.parametrize("heads, page, dtype", [((4, 2), 16, torch.bfloat16), ((8, 1), 64, torch.float16)])
def test_attention_of_trees(device, new, lengths, heads, page, dtype):
    _attend(new, lengths, heads, page, dtype, device, tree=_random_tree(new, -(-max(new) // 32), 3))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads", [(4, 2), (8, 1)])
def test_attention_rows_that_see_nothing(device, heads):
    """No bit, and no token before the new ones; bits of tokens that are not there; fewer words than tokens."""
    new = [40, 3, 50]
    tree = torch.zeros(93, 1, dtype=torch.int32)
    tree[5] = -1        # all of the first 32, ahead of itself too
    tree[6] = 1 << 30
    tree[40:43] = -8    # bits of tokens 3 to 31 of a sequence with 3
    tree[44] = 3
    out = _attend(new, [40, 10, 50], heads, 16, torch.bfloat16, device, tree=tree)
    assert not bool(out[0].any()) and bool(out[5].any()) and bool(out[41].any()) and not bool(out[43].any())
    none = torch.zeros(93, 0, dtype=torch.int32)
    out = _attend(new, [40, 10, 50], heads, 16, torch.bfloat16, device, tree=none)
    assert not bool(out[5].any()) and bool(out[41].any())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_scales_and_sizes(device):
    """Scores far apart, a scale, weights that one key takes, values at the end of fp16."""
    _attend([1, 20], [200, 150], (4, 2), 32, torch.bfloat16, device, scale=2.0, sharp=4.0)
    _attend([1, 20], [200, 150], (4, 2), 32, torch.float16, device, scale=1e-3)
    batch, pages, _ = _batch([1], [100], 16, device=device)
    keys, values = _pool(pages, 1, 16, torch.float16, device)
    values.fill_(60000.0)
    out = ops.paged_attention(torch.ones(1, 2, DIM, dtype=torch.float16, device=device), keys, values, batch)
    assert bool((out == 60000.0).all())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_of_nothing(device):
    keys, values = _pool(2, 1, 16, torch.bfloat16, device)
    empty = PagedBatch(*(torch.zeros(s, dtype=torch.int32, device=device) for s in ((0, 3), (1,), (0,))))
    assert ops.paged_attention(torch.zeros(0, 2, DIM, dtype=torch.bfloat16, device=device), keys, values, empty).shape == (0, 2, DIM)
    out = ops.paged_attention(torch.ones(3, 2, DIM, dtype=torch.bfloat16, device=device), keys, values, empty)
    assert out.shape == (3, 2, DIM) and not bool(out.any())


def test_attention_in_wider_types_on_the_cpu():
    for dtype in (torch.float32, torch.float64):
        batch, pages, rows = _batch([2, 3], [20, 3], 16)
        keys, values = _pool(pages, 2, 16, dtype, "cpu")
        q = torch.randn(rows, 4, DIM, generator=_gen(1)).to(dtype)
        want, room = _attention_definition(q, keys, values, batch, 0.1)
        _close(ops.paged_attention(q, keys, values, batch, scale=0.1), want, room)


# -- the mask of a tree -----------------------------------------------------------------------------
def test_tree_mask():
    parents = torch.tensor([-1, 0, 0, 1, -1, -1, -1] + [-1] + list(range(39)) + [5])
    starts = torch.tensor([0, 5, 7, 47])
    tree = ops.tree_mask(parents, starts)
    assert tree.shape == (48, 2) and tree.dtype == torch.int32
    bits = lambda r: {j for j in range(64) if int(tree[r, j // 32]) >> j % 32 & 1}  # noqa: E731
    assert [bits(r) for r in range(7)] == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {4}, {0}, {1}]
    assert bits(46) == set(range(40)) and bits(47) == set()
    for bad in (torch.tensor([0]), torch.tensor([-2]), torch.tensor([-1, 1])):
        with pytest.raises(ValueError, match="before its child"):
            ops.tree_mask(bad, torch.tensor([0, len(bad)]))
    with pytest.raises(ValueError, match="bits"):
        ops.tree_mask(torch.full((33,), -1), torch.tensor([0, 33]), 1)
    with pytest.raises(ValueError, match="starts"):
        ops.tree_mask(torch.full((3,), -1), torch.tensor([0, 4]))
    with pytest.raises(TypeError, match="int64"):
        ops.tree_mask(torch.full((3,), -1.0), torch.tensor([0, 3]))


# -- logits -----------------------------------------------------------------------------------------
def _words(keep):
    """int32 words of a truth table [rows, V]."""
    rows, vocab = keep.shape
    padded = torch.zeros(rows, -(-vocab // 32) * 32, dtype=torch.int64)
    padded[:, :vocab] = keep
    value = (padded.view(rows, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(value >= 1 << 31, value - (1 << 32), value).int()


def _check_logits(x, device, history=None, lengths=None, prompts=None, repetition=None, presence=None, frequency=None,
                  bias_ids=None, bias=None, allowed=None):
    there = lambda v: None if v is None else v.to(device)  # noqa: E731
    got = ops.process_logits(there(x), there(history), lengths=there(lengths), prompt_lengths=there(prompts),
                             repetition=there(repetition), presence=there(presence), frequency=there(frequency),
                             bias_ids=there(bias_ids), bias=there(bias), allowed=there(allowed))
    assert got.dtype == x.dtype and got.is_contiguous()
    want, room = _logits_definition(x, history, lengths, prompts, repetition, presence, frequency, bias_ids, bias, allowed)
    got, want = got.double().cpu(), torch.where(want.to(x.dtype).isinf(), want.to(x.dtype).double(), want)  # (beyond the type's range)
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    fine = want.isfinite()
    _close(got[fine], want[fine], (room + HALF_STEP[x.dtype] * want.abs())[fine])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 7), (2, 31), (2, 32), (3, 33), (2, 513), (3, 4099), (2, 20011)])
def test_logits(device, dtype, rows, vocab):
    x = (torch.randn(rows, vocab, generator=_gen(vocab)) * 4).to(dtype)
    history = (torch.rand(rows, 50, generator=_gen(1)) ** 3 * vocab).long().clamp(max=vocab - 1)
    history[:, 7] = -1
    lengths = torch.tensor([50, 0, 31][:rows], dtype=torch.int32)
    prompts = torch.tensor([20, 0, 40][:rows], dtype=torch.int32)
    repetition, presence, frequency = (torch.rand(rows, generator=_gen(s)) + a for s, a in ((2, 0.8), (3, -0.5), (4, -0.5)))
    count = min(vocab, 9)
    bias_ids = torch.stack([torch.randperm(vocab, generator=_gen(5 + r))[:count] for r in range(rows)])
    bias = torch.randn(rows, count, generator=_gen(6)) * 5
    keep = torch.rand(rows, vocab, generator=_gen(7)) < 0.5
    allowed = _words(keep)
    penalties = dict(history=history, lengths=lengths, prompts=prompts, repetition=repetition, presence=presence,
                     frequency=frequency)
    _check_logits(x, device, **penalties)
    _check_logits(x, device, bias_ids=bias_ids, bias=bias)
    _check_logits(x, device, allowed=allowed)
    _check_logits(x, device, **penalties, bias_ids=bias_ids, bias=bias, allowed=allowed)
    _check_logits(x, device, history=history.int(), repetition=repetition)
    same = ops.process_logits(x.to(device))
    assert torch.equal(same.cpu(), x) and same.data_ptr() != x.data_ptr()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_special_values(device, dtype):
    """Masked, infinite and NaN logits, with and without a penalty, a bias and the mask."""
    x = torch.tensor([[-INF, INF, float("nan"), 0.0, -0.0, 1.0, torch.finfo(dtype).min, torch.finfo(dtype).max] * 5]).to(dtype)
    ones = torch.ones(1)
    _check_logits(x, device, history=torch.arange(8)[None], repetition=ones * 1.5, presence=ones, frequency=ones)
    _check_logits(x, device, bias_ids=torch.tensor([[0, 1, 2, 3]]), bias=torch.tensor([[1.0, -1.0, 2.0, -INF]]))
    keep = torch.zeros(1, 40, dtype=torch.bool)
    _check_logits(x, device, history=torch.arange(8)[None], presence=ones, allowed=_words(keep))
    keep[0, 3] = keep[0, 13] = True
    _check_logits(x, device, history=torch.arange(8)[None], presence=ones, allowed=_words(keep))


@pytest.mark.parametrize("device", DEVICES)
def test_logits_repeated_ids(device):
    """One token a thousand times, the same bias id again and again, ids that are none."""
    vocab = 300
    x = torch.randn(2, vocab, generator=_gen(1))
    history = torch.full((2, 1000), 17)
    history[1, ::2] = 299
    _check_logits(x, device, history=history, prompts=torch.tensor([400, 1000], dtype=torch.int32),
                  repetition=torch.tensor([1.2, 0.7]), presence=torch.tensor([0.3, 0.4]), frequency=torch.tensor([0.01, 0.02]))
    ids = torch.tensor([[5, 5, -1, 5, 299, 0, 299], [-1, -1, -1, -1, -1, -1, -1]])
    bias = torch.randn(2, 7, generator=_gen(2))
    _check_logits(x, device, bias_ids=ids, bias=bias)
    first = ops.process_logits(x.to(device), bias_ids=ids.to(device), bias=bias.to(device))
    assert torch.equal(first, ops.process_logits(x.to(device), bias_ids=ids.to(device), bias=bias.to(device)))


@pytest.mark.parametrize("device", DEVICES)
def test_logits_of_long_lists(device):
    """A history beyond 16-bit counts, and more biases than a block lists, some of them repeated."""
    vocab = 700
    x = torch.randn(2, vocab, generator=_gen(1)).bfloat16()
    history = (torch.rand(2, 40000, generator=_gen(2)) ** 3 * vocab).long()
    history[0, 20000:] = 3
    ones = torch.ones(2)
    _check_logits(x, device, history=history, lengths=torch.tensor([40000, 17000], dtype=torch.int32),
                  prompts=torch.tensor([100, 0], dtype=torch.int32), repetition=ones * 1.1, presence=ones, frequency=ones * 1e-3)
    ids = torch.randint(-1, vocab, (2, 1300), generator=_gen(3))
    _check_logits(x.float(), device, bias_ids=ids, bias=torch.randn(2, 1300, generator=_gen(4)))
    _check_logits(x, device, history=history[:, :16384], frequency=ones * 1e-3, bias_ids=ids[:, :300],
                  bias=torch.randn(2, 300, generator=_gen(4)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_layouts(device, dtype):
    """Rows of a wider tensor, several leading dimensions, tables for all rows, numbers for penalties."""
    wide = torch.randn(2, 3, 77, generator=_gen(1)).to(dtype).to(device)
    history = torch.randint(0, 70, (12,), generator=_gen(2)).to(device)
    allowed = _words(torch.rand(1, 70, generator=_gen(3)) < 0.7).to(device)
    ids, bias = torch.tensor([3, 9], device=device), torch.tensor([1.0, -2.0], device=device)
    for x in (wide[..., 3:73], wide[:, :, :70], wide[:, ::2, 5:75], wide.transpose(0, 1)[..., :70]):
        got = ops.process_logits(x, history, repetition=1.25, presence=0.5, frequency=0.125, bias_ids=ids, bias=bias,
                                 allowed=allowed)
        flat = x.reshape(-1, 70).cpu()
        rows = len(flat)
        full = lambda v: torch.full((rows,), v)  # noqa: E731
        want, room = _logits_definition(flat, history.cpu().expand(rows, -1), None, None, full(1.25), full(0.5),
                                        full(0.125), ids.cpu().expand(rows, -1), bias.cpu().expand(rows, -1),
                                        allowed.cpu().expand(rows, -1))
        assert got.shape == x.shape
        fine = want.isfinite()
        got = got.reshape(rows, 70).double().cpu()
        assert torch.equal(got.isfinite(), fine)
        _close(got[fine], want[fine], (room + HALF_STEP[dtype] * want.abs())[fine])
    assert ops.process_logits(wide[:0]).shape == (0, 3, 77)
    one = ops.process_logits(wide[0, 0], history, presence=1.0)
    assert one.shape == (77,)
    assert ops.process_logits(wide, history[:0], presence=1.0).equal(wide.contiguous())


# -- refusals ---------------------------------------------------------------------------------------
def _call(device="cpu"):
    batch, pages, rows = _batch([2], [5], 16, device=device)
    keys, values = _pool(pages, 1, 16, torch.bfloat16, device)
    qkv = torch.randn(rows, 4 * DIM, generator=_gen(1)).bfloat16().to(device)
    w = torch.ones(DIM, dtype=torch.bfloat16, device=device)
    return dict(qkv=qkv, wq=w, wk=w, positions=torch.arange(2, device=device), freqs=FREQS.to(device), hq=2, hkv=1, eps=1e-6,
                keys=keys, values=values, batch=batch)


@pytest.mark.parametrize("device", DEVICES)
def test_append_refusals(device):
    good = _call(device)
    ops.paged_append(**good)
    wrong = [("wq", good["wq"].float(), TypeError), ("positions", good["positions"].int(), TypeError),
             ("positions", good["positions"][:1], ValueError), ("freqs", good["freqs"][:63], ValueError),
             ("freqs", good["freqs"].double(), TypeError), ("hq", 3, ValueError), ("hkv", 2, ValueError),
             ("wk", good["wk"][:64], ValueError), ("keys", good["keys"][..., :64], ValueError),
             ("keys", good["keys"][:, :, :15], ValueError), ("keys", good["keys"].float(), (TypeError, ValueError)),
             ("values", good["values"][:1], ValueError)]
    for name, value, error in wrong:
        with pytest.raises(error):
            ops.paged_append(**{**good, name: value})
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.paged_append(**{**good, "qkv": good["qkv"].clone().requires_grad_()})
    with torch.no_grad():
        ops.paged_append(**{**good, "qkv": good["qkv"].clone().requires_grad_()})


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refusals(device):
    c = _call(device)
    q = torch.randn(2, 2, DIM, generator=_gen(1)).bfloat16().to(device)
    good = dict(q=q, keys=c["keys"], values=c["values"], batch=c["batch"])
    ops.paged_attention(**good)
    tree = torch.zeros(2, 1, dtype=torch.int32, device=device)
    wrong = [("q", q.float(), TypeError), ("q", q[0], ValueError), ("q", q[..., :64], ValueError), ("scale", 0.0, ValueError),
             ("scale", -1.0, ValueError), ("scale", INF, ValueError), ("tree", tree.long(), TypeError),
             ("tree", tree[:1], ValueError), ("tree", tree[:, 0], ValueError), ("values", c["values"].half(), ValueError)]
    for name, value, error in wrong:
        with pytest.raises(error):
            ops.paged_attention(**{**good, name: value})
    three = torch.cat((c["keys"],) * 3, dim=1)
    with pytest.raises(ValueError, match="heads"):
        ops.paged_attention(q, three, three, c["batch"])
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.paged_attention(**{**good, "q": q.clone().requires_grad_()})


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    x = torch.randn(1, 10)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.process_logits(forward_ad.make_dual(x, torch.ones_like(x)))
        ops.process_logits(x)


def test_batch_refusals():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    PagedBatch(i(2, 3), i(3), i(2))
    for bad in ((i(2, 3), i(2), i(2)), (i(2, 3), i(3), i(3)), (i(2), i(3), i(2))):
        with pytest.raises(ValueError):
            PagedBatch(*bad)
    with pytest.raises(TypeError):
        PagedBatch(i(2, 3).long(), i(3), i(2))


BAD_BATCHES = {  # of 3 + 2 rows over a pool of 6 pages of 16: (tables, starts, lengths), and the rows that stay good
    "a page outside the cache": ([[0, 6], [1, 2]], [0, 3, 5], [20, 18], [3, 4]),
    "a negative page": ([[-1, 3], [1, 2]], [0, 3, 5], [20, 18], [3, 4]),
    "a length beyond the table": ([[0, 3], [1, 2]], [0, 3, 5], [33, 18], [3, 4]),
    "a negative length": ([[0, 3], [1, 2]], [0, 3, 5], [-5, 18], [3, 4]),
    "more new tokens than length": ([[0, 3], [1, 2]], [0, 3, 5], [2, 18], [3, 4]),
    "starts beyond the rows": ([[0, 3], [1, 2]], [0, 3, 6], [20, 18], [0, 1, 2]),
    "falling starts": ([[0, 3], [1, 2]], [0, 3, 1], [20, 18], []),
    "a negative start": ([[0, 3], [1, 2]], [-1, 3, 5], [20, 18], [3, 4]),
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", BAD_BATCHES)
def test_bad_batches(device, which):
    tables, starts, lengths, good = BAD_BATCHES[which]
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    batch = PagedBatch(i(tables), i(starts), i(lengths))
    keys, values = _pool(6, 1, 16, torch.bfloat16, device)
    before = keys.clone(), values.clone()
    q = torch.randn(5, 2, DIM, generator=_gen(1)).bfloat16().to(device)
    qkv = torch.randn(5, 4 * DIM, generator=_gen(1)).bfloat16().to(device)
    w = torch.ones(DIM, dtype=torch.bfloat16, device=device)
    append = lambda: ops.paged_append(qkv, w, w, torch.arange(5, device=device), FREQS.to(device), 2, 1, 1e-6, keys,  # noqa: E731
                                      values, batch)
    if device == "cpu":
        with pytest.raises(ValueError):
            ops.paged_attention(q, keys, values, batch)
        with pytest.raises(ValueError):
            append()
        return
    out = ops.paged_attention(q, keys, values, batch)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status("attention")
    fine = PagedBatch(i([[0, 3], [1, 2]]), i([0, 3, 5]), i([20, 18]))
    if good:
        assert torch.equal(out[good], ops.paged_attention(q, keys, values, fine)[good])
    ops.check_status("the same without the fault")
    append()
    if which == "a negative page":  # (the new tokens lie in the other one)
        ops.check_status("append")
        return
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status("append")
    for now, was in zip((keys, values), before):
        assert torch.equal(now[[0, 4, 5]], was[[0, 4, 5]])


@pytest.mark.parametrize("device", DEVICES)
def test_logits_refusals(device):
    x = torch.randn(2, 40, generator=_gen(1)).to(device)
    h = torch.zeros(2, 3, dtype=torch.long, device=device)
    i = torch.zeros(2, dtype=torch.int32, device=device)
    b = torch.zeros(2, 2, device=device)
    for kw, error in [(dict(repetition=1.1), ValueError), (dict(lengths=i), ValueError), (dict(bias=b), ValueError),
                      (dict(history=h.float()), TypeError), (dict(history=h, lengths=i.long()), TypeError),
                      (dict(history=h, lengths=i[:1]), ValueError), (dict(history=h, repetition=0.0), ValueError),
                      (dict(history=h, repetition=INF), ValueError), (dict(history=h, presence=b), ValueError),
                      (dict(history=h[0, 0]), ValueError), (dict(history=torch.zeros(3, 3, dtype=torch.long, device=device)), ValueError),
                      (dict(bias_ids=h, bias=b), ValueError), (dict(bias_ids=h[:, :2].int(), bias=b), TypeError),
                      (dict(bias_ids=h[:, :2], bias=b.double()), TypeError),
                      (dict(allowed=torch.zeros(2, 1, dtype=torch.int32, device=device)), ValueError),
                      (dict(allowed=torch.zeros(2, 2, dtype=torch.int64, device=device)), TypeError)]:
        with pytest.raises(error):
            ops.process_logits(x, **kw)
    with pytest.raises(TypeError):
        ops.process_logits(x.int())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.process_logits(x.clone().requires_grad_())
    beyond = torch.tensor([[1, 40, 2], [0, 0, 0]], device=device)
    calls = (lambda: ops.process_logits(x, beyond, presence=1.0),
             lambda: ops.process_logits(x, bias_ids=beyond, bias=torch.ones(2, 3, device=device)),
             lambda: ops.process_logits(x, h, lengths=torch.tensor([3, 4], dtype=torch.int32, device=device), presence=1.0))
    for call in calls:
        if device == "cpu":
            with pytest.raises(ValueError):
                call()
        else:
            call()
            with pytest.raises(ops.DeviceStatusError):
                ops.check_status("logits")


# -- streams, graphs, large caches ------------------------------------------------------------------
@pytest.mark.gpu
def test_captured_step_follows_its_batch():
    """One graph serves batches of other lengths, with another graph's replays between."""
    hq, hkv, page = 8, 2, 16
    batch, pages, rows = _batch([1, 1, 2], [100, 40, 7], page, device="cuda", extra=1, width=20)
    big = torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20)
    batch = PagedBatch(big, batch.starts, batch.lengths)
    keys, values = _pool(60, hkv, page, torch.bfloat16, "cuda")
    q = torch.randn(rows, hq, DIM, generator=_gen(1)).bfloat16().cuda()
    x = torch.randn(rows, 5000, generator=_gen(2)).bfloat16().cuda()
    history = torch.randint(0, 5000, (rows, 64), generator=_gen(3)).cuda()
    known = torch.full((rows,), 64, dtype=torch.int32, device="cuda")

    def step():
        return (ops.paged_attention(q, keys, values, batch),
                ops.process_logits(x, history, lengths=known, presence=0.5, repetition=1.1))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for starts, lengths, n in (([0, 1, 2, 4], [100, 40, 7], 64), ([0, 0, 5, 5], [320, 5, 3], 9), ([0, 1, 2, 3], [1, 1, 1], 0),
                               ([0, 3, 3, 4], [319, 200, 1], 33)):
        batch.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        known.fill_(n)
        q.add_(0.25)
        for graph, _ in graphs:
            graph.replay()
        want = step()
        for _, out in graphs:
            for got, expected in zip(out, want):
                assert torch.equal(got, expected)
        definition, room = _attention_definition(q, keys, values, batch, DIM ** -0.5)
        _close(want[0], definition, room)


@pytest.mark.gpu
def test_two_streams_at_once():
    other = torch.cuda.Stream()
    batch, pages, rows = _batch([1] * 9, [700] * 9, 32, device="cuda")
    keys, values = _pool(pages, 2, 32, torch.bfloat16, "cuda")
    q = torch.randn(rows, 8, DIM, generator=_gen(1)).bfloat16().cuda()
    want = ops.paged_attention(q, keys, values, batch)
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        results.append(ops.paged_attention(q, keys, values, batch))
        with torch.cuda.stream(other):
            results.append(ops.paged_attention(q, keys, values, batch))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pages whose elements lie past 2^31 and 2^32 of the pool."""
    heads, page = 4, 64
    each = heads * page * DIM
    pages = 2 ** 32 // each + 3
    pools = [torch.empty(pages, heads, page, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    chosen = [pages - 1, 0, 2 ** 31 // each, pages - 2]
    small = [torch.randn(4, heads, page, DIM, generator=_gen(i)).bfloat16().cuda() for i in range(2)]
    for pool, part in zip(pools, small):
        pool[chosen] = part
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = PagedBatch(i([chosen[:2], chosen[2:]]), i([0, 1, 4]), i([100, 128]))
    near = PagedBatch(i([[0, 1], [2, 3]]), i([0, 1, 4]), i([100, 128]))
    qkv = torch.randn(4, (8 + 2 * heads) * DIM, generator=_gen(5)).bfloat16().cuda()
    w = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
    args = (qkv, w, w, torch.arange(4, device="cuda"), FREQS.cuda(), 8, heads, 1e-6)
    q = ops.paged_append(*args, *pools, batch)
    assert torch.equal(q, ops.paged_append(*args, *small, near))
    for pool, part in zip(pools, small):
        assert torch.equal(pool[chosen], part)
    assert torch.equal(ops.paged_attention(q, *pools, batch), ops.paged_attention(q, *small, near))
