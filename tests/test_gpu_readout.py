"""GPU suite: the readout operators against their formulas in 64 bits, at the sizes, orders and masks where they can go wrong.

Tolerances count roundings.  `half(t)` is half a step of a type relative to the value; sums of n terms in 32 bits are off by at most
n * 2^-23 of the sum of magnitudes (tensor cores may cut off instead of rounding)."""

import math

import numpy as np
import pytest
import torch

from graphtsetlinmachine_b200 import readout
from graphtsetlinmachine_b200.tm import MultiClassGraphTsetlinMachine
from util import random_graphs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
STEP = 2.0 ** -23


@pytest.fixture(autouse=True)
def _library(engine_lib):
    yield
    import ctypes as C
    failed = C.c_int(-1)
    assert engine_lib.gtm_softmax_failed(0, C.byref(failed)) == 0 and failed.value == 0      # no wait ran out


def half(kind):
    return torch.finfo(kind).eps / 2


def least(kind):
    """Half a step of the smallest values."""
    return torch.finfo(kind).smallest_normal * torch.finfo(kind).eps / 2


def normal(gen, *shape, kind=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(kind)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def near(got, want, bound):
    assert got.shape == want.shape
    got, want = got.double(), want.double()
    off = (got - want).abs() - bound
    assert not torch.isnan(got).any() and off.max().item() <= 0 if got.numel() else True, "off by %g more than the bound" % off.max().item()


# ------------------------------------------------------------------------------------------------------- embed
def bags_of(gen, count, ids, wide=torch.int64):
    inner = torch.randint(ids + 1, (count - 1,), generator=gen, device="cuda").sort().values
    return torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), inner, torch.tensor([ids], device="cuda")]).to(wide)


def plain_bags(ids, offsets, rows):
    """Matrix of how often each row is in each bag, 64 bits."""
    offsets = offsets.long().cpu().tolist()
    m = torch.zeros(len(offsets) - 1, rows, dtype=torch.float64)
    ids = ids.long().cpu()
    for b in range(len(offsets) - 1):
        mine = ids[offsets[b]:offsets[b + 1]]
        mine = mine[mine >= 0]
        m[b].index_add_(0, mine, torch.ones(len(mine), dtype=torch.float64))
    return m.cuda()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("columns", [1, 2, 7, 64, 250, 256, 1001])
def test_embed_rows(kind, columns):
    gen = generator(columns)
    table = normal(gen, 83, columns, kind=kind)
    ids = torch.randint(-1, 83, (5, 61), generator=gen, device="cuda")
    out = readout.embed(table, ids, scale=3.0)
    want = table.double()[ids.clamp_min(0)] * 3.0 * (ids >= 0)[..., None]
    near(out, want, half(kind) * want.abs() + 2.0 ** -24 * want.abs() + least(kind))
    assert torch.equal(readout.embed(table, ids.int(), scale=3.0), out)
    assert readout.embed(table, ids[:0]).shape == (0, 61, columns)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("count,ids,columns", [(1, 0, 8), (1, 1, 64), (1, 128, 64), (1, 129, 8), (1, 5000, 24), (7, 1000, 256), (300, 900, 33), (40, 20000, 130), (3, 257, 1032)])
def test_embed_bags_and_their_gradient(kind, count, ids, columns):
    gen = generator(ids + columns)
    rows = 97
    table = normal(gen, rows, columns, kind=kind)
    which = torch.randint(-1, rows, (ids,), generator=gen, device="cuda", dtype=torch.int32)
    offsets = bags_of(gen, count, ids)
    m = plain_bags(which, offsets, rows)
    out = readout.embed(table, which, offsets, scale=0.5)
    want, size = 0.5 * m @ table.double(), 0.5 * m @ table.double().abs()
    near(out, want, half(kind) * want.abs() + (ids + 2) * STEP * size + least(kind))
    gradient = normal(gen, count, columns, kind=kind)
    got = readout.embed_gradient(gradient, which, rows, offsets, scale=0.5)
    want, size = 0.5 * m.t() @ gradient.double(), 0.5 * m.t() @ gradient.double().abs()
    near(got, want, half(kind) * want.abs() + (ids + 2) * STEP * size + least(kind))
    assert torch.equal(readout.embed_gradient(gradient, which.long(), rows, offsets.int(), scale=0.5), got)
    # the same pair of sums from either side: <embed(T), G> = <T, gradient(G)>
    left, right = (out.double() * gradient.double()).sum(), (table.double() * got.double()).sum()
    slack = (half(kind) + (ids + 2) * STEP) * 2 * (m @ table.double().abs() * gradient.double().abs()).sum() + 1e-6
    assert abs(left - right) <= slack


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 65535, 65536, 70001])
def test_embed_gradient_sorts_any_table(rows):
    gen = generator(rows)
    ids = torch.randint(rows, (9001,), generator=gen, device="cuda")
    ids[::3] = rows - 1                                          # a third of all ids are one row
    ids[5::7] = -1
    gradient = torch.randint(-4, 5, (9001, 12), generator=gen, device="cuda").float()      # sums without roundings
    want = torch.zeros(rows + 1, 12, dtype=torch.float64, device="cuda").index_add_(0, torch.where(ids < 0, rows, ids), gradient.double())[:rows]
    assert torch.equal(readout.embed_gradient(gradient, ids, rows).double(), want)


def test_embed_gradient_without_bags_to_take_from():
    got = readout.embed_gradient(torch.empty(0, 4, device="cuda"), torch.zeros(300, dtype=torch.int64, device="cuda"), 6, torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert torch.equal(got, torch.zeros(6, 4, device="cuda"))
    assert readout.embed(got, torch.zeros(300, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")).shape == (0, 4)


def test_embed_gradient_is_the_same_every_time():
    gen = generator(1)
    ids = torch.randint(50, (30000,), generator=gen, device="cuda")
    gradient = normal(gen, 30000, 64)
    first = readout.embed_gradient(gradient, ids, 50)
    for _ in range(3):
        assert torch.equal(readout.embed_gradient(gradient, ids, 50), first)


def test_embed_outside_of_the_table_and_of_bags():
    table = torch.arange(12, device="cuda", dtype=F32).reshape(4, 3)
    out = readout.embed(table, torch.tensor([0, 4, -5, 2 ** 40, 3], device="cuda"))
    assert torch.isnan(out[[1, 3]]).all() and torch.equal(out[2], torch.zeros(3, device="cuda")) and torch.equal(out[4], table[3])
    ids = torch.tensor([3, 1, 2, 9, 1], device="cuda")
    # offsets that begin late, and that leave the list: kept within it
    out = readout.embed(table, ids, torch.tensor([1, 3, 3, 4, 99], device="cuda"))
    assert torch.equal(out[0], table[1] + table[2]) and torch.equal(out[1], torch.zeros(3, device="cuda"))
    assert torch.isnan(out[2]).all() and torch.equal(out[3], table[1])
    got = readout.embed_gradient(torch.ones(4, 3, device="cuda"), ids, 4, torch.tensor([1, 3, 3, 4, 99], device="cuda"))
    assert torch.equal(got[:, 0], torch.tensor([0., 2., 1., 0.], device="cuda"))
    # a padded row and a row that is not asked for may hold anything
    table[0] = math.nan
    assert torch.equal(readout.embed(table, torch.tensor([1, -1], device="cuda"))[1], torch.zeros(3, device="cuda"))


@pytest.mark.parametrize("kind", TYPES)
def test_embed_strides(kind):
    gen = generator(3)
    wide = normal(gen, 50, 200, kind=kind)
    for table in (wide[:, 1:65], wide[::2, 3:67], wide[:1].expand(50, 200), wide[:, 8:136]):
        ids = torch.randint(table.shape[0], (333,), generator=gen, device="cuda")
        assert torch.equal(readout.embed(table, ids), readout.embed(table.contiguous(), ids))
        offsets = bags_of(gen, 5, 333)
        assert torch.equal(readout.embed(table, ids, offsets), readout.embed(table.contiguous(), ids, offsets))
        gradient = normal(gen, 333, 200, kind=kind)[:, 5:5 + 32]
        assert torch.equal(readout.embed_gradient(gradient, ids, 50), readout.embed_gradient(gradient.contiguous(), ids, 50))


# ------------------------------------------------------------------------------------------------- softmax loss
def plain_softmax(x, w, scale):
    """(logits, how far those in 32 bits may be off, log normalisers), 64 bits."""
    x, w = x.double(), w.double()
    logits = scale * x @ w.t()
    off = (x.shape[1] + 16) * STEP * scale * x.abs() @ w.abs().t()
    return logits, off, torch.logsumexp(logits, 1)


def softmax_case(kind, n, d, v, seed=0, margin=3.0):
    gen = generator(seed + n + d + v)
    w = normal(gen, v, d) / math.sqrt(d)
    labels = torch.randint(v, (n,), generator=gen, device="cuda")
    return (normal(gen, n, d) + margin * w[labels]).to(kind), w.to(kind), labels


def check_loss(x, w, labels, scale, ignored=-1):
    logits, off, normaliser = plain_softmax(x, w, scale)
    kept = labels != ignored
    at = labels.clamp_min(0).long()
    want = torch.where(kept, normaliser - logits[torch.arange(len(at)), at], 0.0)
    bound = off.amax(1) + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs()      # the exponentials' 2^-21, the logarithm's and the sums' roundings
    losses, normalisers = readout.softmax_loss(x, w, labels, scale=scale, ignore_label=ignored)
    near(normalisers, normaliser, bound)
    near(losses, want, 2 * bound)
    return normalisers


def check_gradient(x, w, labels, normalisers, gradients, scale, ignored=-1):
    kind = x.dtype
    logits, off, normaliser = plain_softmax(x, w, scale)
    kept = (labels != ignored).double()
    p = torch.softmax(logits, 1)
    at = labels.clamp_min(0).long()
    y = torch.zeros_like(p)
    y[torch.arange(len(at)), at] = 1.0
    g = (gradients.double() * kept * scale)[:, None]
    q, size = (p - y) * g, g.abs().amax()
    # of q: the logits' and normalisers' errors, the exponential's; its rounding to the operands' type (three parts of bf16 reach 2^-24)
    wrong = p * g.abs() * (2 * off.amax(1, keepdim=True) + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs()[:, None])
    wrong += (2.0 ** -22 if kind == F32 else half(kind)) * (q.abs() + wrong) + 2.0 ** -23 * y * g.abs()
    if kind == F16:
        wrong += size * 2.0 ** -38                                # half a step of the smallest fp16, after the scaling by 2^14
    # values below 2^-126 become zero: an exponential (times g), and of the three parts of q the two smaller ones; products of them likewise
    wrong += 2.0 ** -126 * (g.abs() + 2)
    dx, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, gradients, scale=scale, ignore_label=ignored)
    assert dx.dtype == kind and dw.dtype == kind
    xs, ws = x.double() * kept[:, None], w.double()
    for got, want, bound, terms in ((dx, q @ ws, (wrong + (len(w) + 16) * STEP * q.abs()) @ ws.abs(), len(w)),
                                    (dw, q.t() @ xs, (wrong + (len(x) + 16) * STEP * q.abs()).t() @ xs.abs(), len(x))):
        bound = bound + terms * 2.0 ** -126
        near(got, want, bound + half(kind) * (want.abs() + bound) + least(kind))
    return dx, dw


SIZES = [(1, 1, 1), (1, 64, 10), (2, 7, 2), (60, 64, 10), (129, 65, 129), (256, 128, 256), (257, 200, 257), (300, 520, 1000), (33, 1024, 5001), (1000, 72, 300), (2100, 16, 40), (5000, 33, 7), (700, 300, 32), (3, 64, 33), (5, 1000, 513), (8, 40, 4000), (64, 130, 700), (65, 130, 700), (17, 2000, 333), (40, 8, 20000)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_softmax_loss_and_gradient(kind, n, d, v):
    x, w, labels = softmax_case(kind, n, d, v)
    normalisers = check_loss(x, w, labels, 1.25)
    gen = generator(n)
    check_gradient(x, w, labels, normalisers, normal(gen, n).abs() + 0.1, 1.25)


@pytest.mark.parametrize("kind", TYPES)
def test_softmax_in_pieces_of_the_labels(kind):
    """More labels times examples than the workspace holds of P at a time, the last piece smaller."""
    n = 4500 if kind == F32 else 9000
    x, w, labels = softmax_case(kind, n, 24, 9001)
    normalisers = check_loss(x, w, labels, 1.0)
    check_gradient(x, w, labels, normalisers, torch.full((n,), 1.0 / n, device="cuda"), 1.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n, d, v", [(1, 1024, 279), (2, 1000, 279), (8, 1024, 1000), (9, 512, 300), (1, 160, 279), (1, 700, 20), (8, 700, 20)])
def test_gradient_where_the_label_is_nearly_certain(kind, n, d, v):
    """P - 1 of the label: its logit's error is in the normaliser too, so that what is left of it is times 1 - P.  The gradients of the weights are
    P - 1 times the features."""
    gen = generator(n + d + v)
    w = normal(gen, v, d) / math.sqrt(d)
    labels = torch.randperm(v, generator=gen, device="cuda")[:n]            # every label once: a row of dw is one example's
    x = 14.0 * w[labels] / (w[labels] ** 2).sum(1, keepdim=True) + 0.1 * normal(gen, n, d)
    x, w = x.to(kind), w.to(kind)
    logits, off, normaliser = plain_softmax(x, w, 1.0)
    at = torch.arange(n)
    others = logits.clone()
    others[at, labels] = -math.inf
    q = -(torch.logsumexp(others, 1) - normaliser).exp()
    _, normalisers = readout.softmax_loss(x, w, labels)
    _, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(n, device="cuda"))
    xs = x.double()
    rows = dw[labels].double()
    others = torch.softmax(logits, 1)
    others[at, labels] = 0.0
    mixed = others[:, labels].t()                                           # what other examples add to a label's row
    rows = rows - (mixed - torch.diag(torch.diag(mixed))) @ xs
    got = (rows * xs).sum(1) / (xs * xs).sum(1)
    # the normaliser's rounding and those of the sum and the logarithm in it, near one; the exponentials' 2^-21; the logits' errors, times 1 - P
    bound = 2.0 ** -23 * normaliser.abs() + 2.0 ** -22 + q.abs() * (2 * off.amax(1) + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs())
    # q as an operand and the result are rounded, each by half a step; products of up to n terms; examples mixed in are off as their P are
    bound = bound + q.abs() * (2 * max(half(kind), 2.0 ** -22) + (n + 16) * STEP)
    length = xs.norm(dim=1)
    amount = (mixed - torch.diag(torch.diag(mixed))) @ length / length      # of the others' P, at the most, in units of the example's features
    bound = bound + amount * (2 * max(half(kind), 2.0 ** -22) + 2 * off.amax() + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs().amax())
    if kind == F16:
        bound = bound + 2.0 ** -24 * math.sqrt(d) / length                  # results below fp16's normal ones
    near(got, q, bound)


@pytest.mark.parametrize("kind", TYPES)
def test_softmax_of_few_examples_in_pieces_of_the_labels(kind):
    x, w, labels = softmax_case(kind, 20, 8, (1 << 20) + 5000)
    normalisers = check_loss(x, w, labels, 1.0)
    check_gradient(x, w, labels, normalisers, torch.full((20,), 0.05, device="cuda"), 1.0)


@pytest.mark.parametrize("kind", TYPES)
def test_softmax_gradient_against_differences(kind):
    """Central differences of the formula in 64 bits, in random directions."""
    n, d, v = 50, 40, 70
    x, w, labels = softmax_case(kind, n, d, v)
    _, normalisers = readout.softmax_loss(x, w, labels)
    dx, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(1, device="cuda"))

    def loss(x, w):
        logits = x @ w.t()
        return (torch.logsumexp(logits, 1) - logits[torch.arange(n), labels]).sum()

    gen = generator(5)
    for got, at in ((dx, 0), (dw, 1)):
        base = [x.double(), w.double()]
        way = normal(gen, *base[at].shape).double()
        h = 1e-5
        ends = []
        for sign in (1, -1):
            moved = list(base)
            moved[at] = base[at] + sign * h * way
            ends.append(loss(*moved))
        want = (ends[0] - ends[1]) / (2 * h)
        slack = (3 * half(kind) * (got.double().abs() * way.abs()).sum() + 2 * half(kind) * (n * way.abs().amax() * base[1 - at].abs().sum(1).amax()) + 1e-4)
        assert abs((got.double() * way).sum() - want) <= slack


@pytest.mark.parametrize("kind", TYPES)
def test_softmax_ignored_examples_hold_anything(kind):
    x, w, labels = softmax_case(kind, 70, 33, 50)
    labels[::4] = -7
    gradients = torch.rand(70, device="cuda") + 0.5
    normalisers = check_loss(x, w, labels, 1.0, ignored=-7)
    dx, dw = check_gradient(x, w, labels, normalisers, gradients, 1.0, ignored=-7)
    for value in (math.nan, math.inf, -math.inf, torch.finfo(kind).min):
        y = x.clone()
        y[::4] = value
        losses, n2 = readout.softmax_loss(y, w, labels, ignore_label=-7)
        assert (losses[::4] == 0).all() and torch.equal(n2[labels != -7], normalisers[labels != -7])
        got = readout.softmax_loss_gradient(y, w, labels, n2, gradients, ignore_label=-7)
        want = readout.softmax_loss_gradient(x, w, labels, n2.where(labels != -7, 0.0), gradients, ignore_label=-7)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (got[0][::4] == 0).all()
    labels[:] = -7                                               # nothing is left
    losses, normalisers = readout.softmax_loss(x, w, labels, ignore_label=-7)
    got = readout.softmax_loss_gradient(x, w, labels, normalisers, gradients, ignore_label=-7)
    assert (losses == 0).all() and (got[0] == 0).all() and (got[1] == 0).all()


def test_softmax_labels_that_there_are_not():
    x, w, labels = softmax_case(BF16, 20, 16, 8)
    labels[3], labels[4] = 8, -2
    losses, _ = readout.softmax_loss(x, w, labels)
    assert torch.isnan(losses[[3, 4]]).all() and torch.isnan(losses).sum() == 2


def test_softmax_values_that_are_no_numbers():
    x, w, labels = softmax_case(F32, 9, 16, 300)
    x[2, 3] = math.nan
    x[5, 1] = math.inf
    losses, normalisers = readout.softmax_loss(x, w, labels)
    fine = torch.tensor([i not in (2, 5) for i in range(9)], device="cuda")
    assert torch.isnan(losses[~fine]).all() and not torch.isnan(losses[fine]).any()
    label, log_probability = readout.softmax_predict(x, w)
    assert (label[~fine] == -1).all() and torch.isnan(log_probability[~fine]).all() and (label[fine] >= 0).all()


@pytest.mark.parametrize("kind", TYPES)
def test_softmax_large_logits(kind):
    x, w, labels = softmax_case(kind, 64, 32, 200)
    x = (x.float() * 100).to(kind)
    normalisers = check_loss(x, w, labels, 3.0)
    check_gradient(x, w, labels, normalisers, torch.full((64,), 1e-4, device="cuda"), 3.0)


@pytest.mark.parametrize("kind", TYPES)
def test_softmax_strides(kind):
    gen = generator(8)
    wide_x, wide_w = normal(gen, 90, 120, kind=kind), normal(gen, 400, 120, kind=kind)
    labels = torch.randint(150, (90,), generator=gen, device="cuda")
    gradients = torch.rand(90, device="cuda")
    for x, w in ((wide_x[:, 3:67], wide_w[:150, 5:69]), (wide_x[:, 8:72], wide_w[:300:2, 16:80]), (wide_x[:1, :64].expand(90, 64), wide_w[:150, :64]), (wide_x[:, :33], wide_w[:150, :33])):
        ours, theirs = [], []
        for a, b, to in ((x, w, ours), (x.contiguous(), w.contiguous(), theirs)):
            losses, normalisers = readout.softmax_loss(a, b, labels.int())
            to += [losses, normalisers, *readout.softmax_loss_gradient(a, b, labels.int(), normalisers, gradients), *readout.softmax_predict(a, b)]
        assert all(torch.equal(p, q) for p, q in zip(ours, theirs))


def test_softmax_no_examples():
    w = torch.randn(5, 8, device="cuda")
    x, labels = torch.empty(0, 8, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    losses, normalisers = readout.softmax_loss(x, w, labels)
    dx, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(1, device="cuda"))
    assert losses.shape == (0,) and dx.shape == (0, 8) and torch.equal(dw, torch.zeros_like(w))
    assert readout.softmax_predict(x, w)[0].shape == (0,)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_softmax_predict(kind, n, d, v):
    """Whole-numbered features and weights: logits are exact, equal ones are common, the lowest label wins."""
    gen = generator(n + d + v)
    x = torch.randint(-2, 3, (n, d), generator=gen, device="cuda")
    w = torch.randint(-2, 3, (v, d), generator=gen, device="cuda")
    logits = (x.double() @ w.double().t()) * 0.25
    label, log_probability = readout.softmax_predict(x.to(kind), w.to(kind), scale=0.25)
    top = logits.amax(1, keepdim=True)
    want = torch.where(logits == top, torch.arange(v, device="cuda"), v).amin(1)
    assert torch.equal(label, want)
    chosen = (logits - torch.logsumexp(logits, 1, keepdim=True)).amax(1)
    # the scale of products by the tensor cores is raised by 1.5e-8 for every 16 columns, to make up for what they cut off: whole-numbered sums
    # lose nothing, so it moves log probabilities by that share of the distance to the mean logit under the softmax
    mean = (torch.softmax(logits, 1) * (top - logits)).sum(1)
    near(log_probability, chosen, 2.0 ** -20 * (1 + chosen.abs()) + 1.5e-8 * (d / 16 + 8) * mean)


# -------------------------------------------------------------------------------------------------------- adamw
def plain_adamw(p, g, m, v, t, lr, betas, eps, decay, scale):
    b1, b2 = betas
    g = g * scale
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * decay) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


def flat_parts(state, name, sizes):
    at, out = 0, []
    for n in sizes:
        out.append(state[name][at:at + n])
        at += -(-n // 256) * 256
    return out


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("gradient_kind", TYPES)
@pytest.mark.parametrize("sizes", [[1], [255], [256, 0, 257], [5000, 3, 70001], [17] * 600])
def test_adamw_32(kind, gradient_kind, sizes):
    gen = generator(len(sizes))
    storage = normal(gen, sum(sizes) + 3 * len(sizes), kind=kind)
    params, at = [], 0
    for i, n in enumerate(sizes):                 # tensors at any boundary of their elements
        at += i % 4
        params.append(storage[at:at + n])
        at += n
    outside = storage.clone()
    state = readout.adamw_state(params)
    m = [torch.zeros(n, dtype=torch.float64, device="cuda") for n in sizes]
    v = [torch.zeros(n, dtype=torch.float64, device="cuda") for n in sizes]
    copies = [torch.full((n,), 7.0, dtype=BF16, device="cuda") for n in sizes]
    kw = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    for t in range(1, 4):
        gradients = [normal(gen, n, kind=gradient_kind) for n in sizes]
        before = [p.double() for p in params]
        readout.adamw_step(params, gradients, state, gradient_scale=0.5, copies=copies, **kw)
        for i, (p, m2, v2) in enumerate(zip(params, flat_parts(state, "first", sizes), flat_parts(state, "second", sizes))):
            want, m[i], v[i] = plain_adamw(before[i], gradients[i].double(), m[i], v[i], t, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"], 0.5)
            if not sizes[i]:
                continue
            # a handful of roundings each: of the moments relative to their terms, of the step relative to lr (its ratio is below 10)
            near(m2, m[i], 8 * STEP * (m[i].abs() + gradients[i].double().abs()))
            near(v2, v[i], 8 * STEP * (v[i].abs() + gradients[i].double() ** 2))
            near(p, want, half(kind) * (want.abs() + 1e-6) + 4 * STEP * before[i].abs() + 64 * STEP * kw["lr"] * 10 + least(kind))
            assert torch.equal(copies[i], p.to(BF16))
            m[i], v[i] = m2.double(), v2.double()
    assert int(state["steps"]) == 3
    touched = torch.zeros_like(storage, dtype=torch.bool)
    at = 0
    for i, n in enumerate(sizes):
        at += i % 4
        touched[at:at + n] = True
        at += n
    assert torch.equal(storage[~touched], outside[~touched])


def e4m3_around(x):
    """The e4m3 values below and above magnitudes up to 448."""
    x = x.double().abs().clamp_max(448.0)
    step = torch.where(x >= 2.0 ** -6, torch.exp2(torch.floor(torch.log2(x.clamp_min(2.0 ** -6))) - 3), torch.full_like(x, 2.0 ** -9))
    low = torch.floor(x / step) * step
    return low, torch.where(low == x, low, low + step), step


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("sizes", [[1], [256, 0, 257], [5000, 3, 70001]])
def test_adamw_8(kind, sizes):
    gen = generator(11)
    params = [normal(gen, n, kind=kind) for n in sizes]
    state = readout.adamw_state(params, state_bits=8)
    kw = dict(lr=0.01, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    for t in range(1, 4):
        gradients = [normal(gen, n, kind=kind) * torch.exp(normal(gen, n)).to(kind) for n in sizes]
        held = {k: v.clone() for k, v in state.items()}
        before = [p.double() for p in params]
        again = [p.clone() for p in params]
        readout.adamw_step(params, gradients, state, seed=5, **kw)
        readout.adamw_step(again, gradients, held_again := {k: v.clone() for k, v in held.items()}, seed=5, **kw)
        assert all(torch.equal(a, b) for a, b in zip(again, params)) and all(torch.equal(held_again[k].view(torch.uint8), state[k].view(torch.uint8)) for k in state)
        values = {}
        for name in ("first", "second"):
            values[name] = held[name].double() * held[name + "_scales"].double().repeat_interleave(256)
        at = 0
        for i, n in enumerate(sizes):
            m, v = values["first"][at:at + n], values["second"][at:at + n] ** 2
            want, m, v = plain_adamw(before[i], gradients[i].double(), m, v, t, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"], 1.0)
            if n:
                near(params[i], want, half(kind) * (want.abs() + 1e-6) + 4 * STEP * before[i].abs() + 64 * STEP * kw["lr"] * 10 + least(kind))
            for name, x in (("first", m), ("second", v.sqrt())):
                if not n:
                    continue
                blocks = -(-n // 256)
                scales = state[name + "_scales"][at // 256:at // 256 + blocks].double()
                tops = torch.nn.functional.pad(x, (0, blocks * 256 - n)).reshape(-1, 256).abs().amax(1)
                near(scales, tops / 448, 16 * STEP * tops / 448 + 2.0 ** -125)
                code = state[name][at:at + n].double()
                r = (x / scales.repeat_interleave(256)[:n]).abs()
                low, high, step = e4m3_around(r)
                slack = 32 * STEP * (r + 1)              # where the 32-bit value is on the other side of a code
                assert (code.abs() >= low - step * (r - low <= slack)).all() and (code.abs() <= high + step * (high - r <= slack)).all()
                assert ((code.sign() == x.sign()) | (code == 0)).all()
                if name == "second":
                    assert (code[x > 0] > 0).all()
                elif n > 60000:                          # the rounding favours neither side: n values, each off by a step at most
                    off = (code.abs() - r) / step
                    assert abs(off.mean().item()) <= 5 / math.sqrt(n)
            at += -(-n // 256) * 256


def test_adamw_8_decays():
    """A moment that gets no gradients decays on the average, although a step is less than half the distance of two codes."""
    n = 1 << 16
    p = [torch.zeros(n, device="cuda")]
    state = readout.adamw_state(p, state_bits=8)
    readout.adamw_step(p, [torch.ones(n, device="cuda")], state, lr=0.0, betas=(0.9, 0.99), weight_decay=0.0)
    # one element of every block keeps its gradient, so that the scale stays
    gradient = torch.zeros(n, device="cuda")
    gradient[::256] = 1.0
    for _ in range(50):
        readout.adamw_step(p, [gradient], state, lr=0.0, betas=(0.9, 0.99), weight_decay=0.0)
    root = state["second"].float().reshape(-1, 256) * state["second_scales"][:, None]
    rest = root[:, 1:].double()
    want = 0.1 * 0.99 ** 25                             # root of 0.01 * 0.99^50
    # without a gradient the root is multiplied by sqrt(0.99) and rounded without bias, 50 times, each time with a spread of at most half
    # the distance of two codes, 1/16 of it: the mean of 65,280 is within 5 * sqrt(50) / 16 / sqrt(65,280) = 0.9 % of the product
    assert abs(rest.mean().item() / want - 1) <= 0.01


def test_adamw_holds_what_is_not_finite():
    for bits in (32, 8):
        p = [torch.ones(600, device="cuda")]
        g = torch.ones(600, device="cuda")
        g[3], g[300] = math.nan, math.inf
        state = readout.adamw_state(p, state_bits=bits)
        readout.adamw_step(p, [g], state, lr=0.1)
        bad = torch.isnan(p[0])
        assert bad[[3, 300]].all() and bad.sum() == 2
        readout.adamw_step(p, [torch.ones(600, device="cuda")], state, lr=0.1)
        assert torch.isnan(p[0]).sum() == 2


# ------------------------------------------------------------------------------------- streams, graphs, all together
def step_of(batch):
    """One training step over a batch: everything that it writes."""
    table, weights, ids, offsets, labels, params, state = batch
    features = readout.embed(table, ids, offsets, scale=0.1)
    losses, normalisers = readout.softmax_loss(features, weights, labels)
    dx, dw = readout.softmax_loss_gradient(features, weights, labels, normalisers, torch.full((1,), 0.01, device="cuda"))
    dt = readout.embed_gradient(dx, ids, table.shape[0], offsets, scale=0.1)
    readout.adamw_step(params, [dt, dw], state, lr=0.01, copies=[table, weights])
    return losses, dx, dw, dt, readout.softmax_predict(features, weights)[0]


def batch_of(seed, bits):
    gen = generator(seed)
    params = [normal(gen, 90, 48), normal(gen, 130, 48)]
    ids = torch.randint(90, (2000,), generator=gen, device="cuda", dtype=torch.int32)
    return [params[0].to(BF16), params[1].to(BF16), ids, bags_of(gen, 70, 2000), torch.randint(130, (70,), generator=gen, device="cuda"), params, readout.adamw_state(params, bits)]


def flat(out, batch):
    return [t.clone().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.clone() for t in (*out, *batch[5], batch[0], batch[1], *batch[6].values())]


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_on_another_stream_and_captured(bits):
    want = []
    batch = batch_of(2, bits)
    for _ in range(3):
        want.append(flat(step_of(batch), batch))
    # on a stream of its own, next to other work on the default stream
    batch, stream = batch_of(2, bits), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    noise = batch_of(9, bits)
    for k in range(3):
        with torch.cuda.stream(stream):
            out = step_of(batch)
            got = flat(out, batch)
        step_of(noise)
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))
    # two graphs, replayed in turn: one step each of two batches
    torch.cuda.synchronize()
    batches, graphs, outs = [batch_of(2, bits), batch_of(2, bits)], [], []
    for b in batches:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step_of(b)
        graphs.append(g)
        outs.append(out)
    for k in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, b in zip(outs, batches):
            assert all(torch.equal(p, q) for p, q in zip(flat(out, b), want[k]))


def test_long_rows_and_many_examples():
    """Offsets that pass 32 bits: a table of more than 2^31 elements, its last rows used."""
    rows, columns = (1 << 21) + 5, 1032
    table = torch.zeros(rows, columns, dtype=BF16, device="cuda")
    table[-3:] = torch.arange(3 * columns, device="cuda").reshape(3, columns).to(BF16) / 64
    ids = torch.tensor([rows - 1, 0, rows - 3, rows - 2], device="cuda")
    assert torch.equal(readout.embed(table, ids), table[ids])
    got = readout.embed_gradient(table[ids].contiguous(), ids, rows)
    assert torch.equal(got[ids], table[ids]) and not got[:-3].any()
    del got
    x = table[-3:].clone()
    label, _ = readout.softmax_predict(x, table, scale=1e-3)
    assert (label >= rows - 3).all()
    losses, normalisers = readout.softmax_loss(x, table, torch.tensor([rows - 1, 0, -1], device="cuda"), scale=1e-3)
    logits = x.double() @ table[-3:].double().t() * 1e-3
    want = torch.logsumexp(torch.cat([logits, torch.full((3, 1), math.log(rows - 3), device="cuda", dtype=torch.float64)], 1), 1)
    near(normalisers, want, 2.0 ** -18 * (1 + want.abs()))


@pytest.mark.parametrize("bits", [32, 8])
def test_readout_learns_from_clauses(bits):
    np.random.seed(4)
    rng = np.random.default_rng(4)
    graphs = random_graphs(60, rng, max_nodes=5)
    labels = rng.integers(0, 3, size=60)
    tm = MultiClassGraphTsetlinMachine(40, 100, 2.0, depth=1, seed=1)
    tm.fit(graphs, labels, epochs=2)
    head = readout.ClauseReadout(tm, embedding_size=24, state_bits=bits)
    history = head.fit(graphs, labels, epochs=3, batch_size=25)
    assert len(history) == 3 and all(math.isfinite(v) for v in history)
    predicted, log_probability = head.score(graphs)
    assert predicted.shape == (60,) and (log_probability <= 0).all() and np.array_equal(head.predict(graphs), predicted)
    assert np.array_equal(predicted, head.predict(graphs))
    # gradients of a batch against the formula, from the same weights
    ids, offsets = head.active_clauses(graphs)
    outputs, _ = tm.transform(graphs)
    m = torch.from_numpy(outputs).double().cuda()
    assert torch.equal(m, plain_bags(ids, offsets, 40))
    y = torch.from_numpy(labels).cuda()
    table, weights = (c.double().requires_grad_() for c in head.copies)
    loss = torch.nn.functional.cross_entropy((m @ table) * 24 ** -0.5 @ weights.t(), y, reduction="none")
    loss.mean().backward()
    losses, (dt, dw) = head.gradients(ids, offsets, y)
    # features and their gradients are rounded to bf16 between the operators: each rounding is half(bf16) of the values that it meets
    features = (m @ table.detach()).abs() * 24 ** -0.5
    logits_off = 2 * half(BF16) * (features @ weights.detach().abs().t()).amax(1)
    near(losses, loss.detach(), 2 * logits_off + 1e-5)
    size = (2 * logits_off.amax() + 3 * half(BF16)) * 2
    near(dt, table.grad, size * (m.t() @ torch.ones(60, 1, device="cuda", dtype=torch.float64) / 60 * weights.detach().abs().sum(0)) * 24 ** -0.5 + 1e-7)
    near(dw, weights.grad, size * features.sum(0) / 60 + 1e-7)
    # learning goes on from what is there, and the machine is as it was
    sums = tm.score(graphs)
    head.fit(graphs, labels, epochs=1, incremental=True)
    assert np.array_equal(tm.score(graphs), sums)
    with pytest.raises(ValueError):
        head.fit(graphs, labels + 1, epochs=1, incremental=True)


def test_saved_parameters_are_known_to_have_changed():
    p = torch.ones(3, device="cuda", requires_grad=True)
    saved = (p * p).sum()
    with torch.no_grad():
        readout.adamw_step([p], [torch.ones(3, device="cuda")], readout.adamw_state([p]), lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    assert not readout.softmax_failed()


def test_other_shapes_and_devices_are_refused():
    x, w, labels = softmax_case(F32, 20, 16, 40)
    _, n = readout.softmax_loss(x, w, labels)
    one = torch.ones(1, device="cuda")
    for call in (lambda: readout.softmax_loss(x.t(), w, labels), lambda: readout.softmax_loss(x, w[:, :8], labels), lambda: readout.softmax_loss(x, w, labels[:5]),
                 lambda: readout.softmax_loss(x, w, labels, scale=-1.0), lambda: readout.softmax_loss(x, w, labels.cpu()), lambda: readout.softmax_loss(x, w[:0], labels),
                 lambda: readout.softmax_loss_gradient(x, w, labels, n[:3], one), lambda: readout.softmax_loss_gradient(x, w, labels, n, torch.ones(2, device="cuda")),
                 lambda: readout.embed(x, labels[::2]), lambda: readout.embed(x[0], labels), lambda: readout.embed(x, labels, labels[:0]),
                 lambda: readout.embed_gradient(x, labels[:3], 5), lambda: readout.embed_gradient(x, labels, 0), lambda: readout.adamw_step([x], [w], readout.adamw_state([x]), 0.1),
                 lambda: readout.adamw_step([x], [x.clone()], readout.adamw_state([w]), 0.1), lambda: readout.adamw_step([x], [x.clone()], readout.adamw_state([x]), 0.1, seed=-1)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: readout.softmax_loss(x, w.half(), labels), lambda: readout.softmax_loss(x.double(), w.double(), labels), lambda: readout.softmax_loss(x, w, labels.float()),
                 lambda: readout.adamw_step([x], [x.clone()], readout.adamw_state([x]), 0.1, copies=[x.clone()])):
        with pytest.raises(TypeError):
            call()
