"""GPU suite: readout operators at their edges - an example unlike the others, one more example than a kernel takes, sums of thousands of
terms of one sign - and in calls that the usual sizes do not make.

Tolerances count roundings, as in test_gpu_readout."""

import math
import threading

import numpy as np
import pytest
import torch

from graphtsetlinmachine_b200 import _lib, readout
from graphtsetlinmachine_b200.tm import MultiClassGraphTsetlinMachine
from test_gpu_readout import F16, F32, STEP, TYPES, _library, batch_of, check_gradient, check_loss, flat, generator, half, least, near, normal, plain_softmax, softmax_case, step_of  # noqa: F401  (_library: no wait ran out)
from util import random_graphs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(40, 16, 8), (50, 40, 70), (300, 24, 700)])
@pytest.mark.parametrize("bad", ["label", math.inf, math.nan])
def test_an_example_without_a_gradient_leaves_the_others_alone(kind, n, d, v, bad):
    """A label that there is not, or an incoming gradient that is not finite: the example's own gradient and that of the weights, nothing else."""
    x, w, labels = softmax_case(kind, n, d, v)
    labels[::5] = -7
    gradients = torch.rand(n, generator=generator(n), device="cuda") + 0.5
    _, normalisers = readout.softmax_loss(x, w, labels, ignore_label=-7)
    without = labels.clone()
    without[3] = -7
    want, _ = readout.softmax_loss_gradient(x, w, without, normalisers, gradients, ignore_label=-7)
    if bad == "label":
        labels[3] = v
    else:
        gradients[3] = bad
    dx, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, gradients, ignore_label=-7)
    others = torch.arange(n, device="cuda") != 3
    assert torch.equal(dx[others], want[others]) and (dx[labels == -7] == 0).all()
    assert not torch.isfinite(dx[3]).any() and not torch.isfinite(dw).any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [65536, 65537, 70001])
def test_few_labels_and_many_examples_take_the_same_logits(kind, n):
    """Logits with a large part that all labels share: P of the label, nearly certain, less one is right only where the normaliser has the same error
    as the logit.  The weights' first columns are c times the unit matrix, so that features' gradients show P - 1 by itself."""
    v, d, c = 10, 2048, 4.0
    gen = generator(n)
    labels, at = torch.randint(v, (n,), generator=gen, device="cuda"), torch.arange(n, device="cuda")
    w = torch.full((v, d), 1 / 16, device="cuda")
    w[:, :v] = c * torch.eye(v, device="cuda")
    x = normal(gen, n, d).abs()
    x[:, :v] *= 0.1
    x[at, labels] = 12 / c
    x, w = x.to(kind), w.to(kind)
    logits = x.double() @ w.double().t()
    off = (d + 16) * STEP * logits.amax(1)
    normaliser = torch.logsumexp(logits, 1)
    logits[at, labels] = -math.inf
    q = -(torch.logsumexp(logits, 1) - normaliser).exp()
    _, normalisers = readout.softmax_loss(x, w, labels)
    dx, _ = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(1, device="cuda"))
    # the normaliser's rounding and those of the sum and the logarithm in it; the logits' errors and the exponential's, times 1 - P; P's rounding and dx'
    bound = 2.0 ** -23 * normaliser + 2.0 ** -22 + q.abs() * (2 * off + 2.0 ** -20 + 2.0 ** -22 * normaliser + 2 * max(half(kind), 2.0 ** -22)) + least(kind)
    near(dx[at, labels].double() / c, q, bound)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(70001, 33, 7), (200003, 8, 32), (66000, 300, 2)])
def test_few_labels_and_many_examples(kind, n, d, v):
    x, w, labels = softmax_case(kind, n, d, v)
    labels[::9] = -1
    normalisers = check_loss(x, w, labels, 1.25)
    check_gradient(x, w, labels, normalisers, normal(generator(n), n).abs() + 0.1, 1.25)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(3, 4096, 300), (16, 4096, 300), (16, 32768, 300), (300, 2048, 1000), (9, 700, 40)])
def test_softmax_of_whole_numbers_of_one_sign(kind, n, d, v):
    """Logits without a rounding: what is left is the exponentials' and the sums', however many columns there are and whichever kernel multiplies."""
    gen = generator(n + d)
    x, w = torch.randint(0, 3, (n, d), generator=gen, device="cuda"), torch.randint(0, 3, (v, d), generator=gen, device="cuda")
    scale = 2.0 ** -6
    logits = (x.double() @ w.double().t()) * scale
    normaliser, top = torch.logsumexp(logits, 1), logits.amax(1)
    x, w = x.to(kind), w.to(kind)
    _, log_probability = readout.softmax_predict(x, w, scale=scale)
    losses, normalisers = readout.softmax_loss(x, w, logits.argmax(1), scale=scale)
    # an exponential's argument is rounded twice: 2^-22 of the distance to the largest logit, on the average under the softmax
    mean = (torch.softmax(logits, 1) * (top[:, None] - logits)).sum(1)
    bound = 2.0 ** -20 * (1 + (top - normaliser).abs()) + 2.0 ** -22 * mean
    near(log_probability, top - normaliser, bound)
    near(losses, normaliser - top, bound)
    near(normalisers, normaliser, bound + 2.0 ** -22 * normaliser)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(16, 1024, 300), (16, 32768, 300), (16, 131072, 300), (5, 20000, 40)])
def test_softmax_of_long_sums_of_one_sign(kind, n, d, v):
    """What tensor cores cut off a sum of one sign adds up: steps of 16 lose less than 2^-22 of the sum so far each, and 20 of a chunk (320 elements; fewer large
    ones of 32-bit inputs) meet half of its sum on the average, so that 16 times 2^-22 is beyond them; chunks are added with rounding, 2^-24 each.  The scale leaves one label, so that the normaliser is its logit."""
    gen = generator(n + d)
    x, w = normal(gen, n, d).abs().to(kind), (normal(gen, v, d).abs() / 1024).to(kind)
    logits = x.double() @ w.double().t() * 1024.0
    _, normalisers = readout.softmax_loss(x, w, logits.argmax(1), scale=1024.0)
    want = torch.logsumexp(logits, 1)
    near(normalisers, want, (16 * 2.0 ** -22 + (d / (128 if kind == F32 else 256) + 4) * 2.0 ** -24) * want)


# ------------------------------------------------------------------------------------------- waits that run out
def lose(launches):
    """The next product kernels wait 50 ms for copies that do not come."""
    _lib.check(_lib.load().gtm_debug_softmax_lose(launches))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(300, 200, 700), (70, 40, 33)])
def test_a_wait_that_runs_out_leaves_no_numbers(kind, n, d, v):
    x, w, labels = softmax_case(kind, n, d, v)
    labels[::5] = -1
    one = torch.ones(1, device="cuda")
    fine = [*readout.softmax_loss(x, w, labels), *readout.softmax_predict(x, w)]
    fine += readout.softmax_loss_gradient(x, w, labels, fine[1], one)
    assert not readout.softmax_failed()
    lose(1)
    losses, normalisers = readout.softmax_loss(x, w, labels)
    assert torch.isnan(losses[labels != -1]).all() and torch.isnan(normalisers).all() and readout.softmax_failed() and not readout.softmax_failed()
    lose(1)
    label, log_probability = readout.softmax_predict(x, w)
    assert (label == -1).all() and torch.isnan(log_probability).all() and readout.softmax_failed()
    for launches, rows in ((1, labels != -1), (2, labels == labels)):               # P, or what is made of it too
        lose(launches)
        dx, dw = readout.softmax_loss_gradient(x, w, labels, fine[1], one)
        assert torch.isnan(dx[rows]).all() and torch.isnan(dw).all() and readout.softmax_failed()
    # and nothing is left of it
    again = [*readout.softmax_loss(x, w, labels), *readout.softmax_predict(x, w)]
    again += readout.softmax_loss_gradient(x, w, labels, again[1], one)
    assert all(torch.equal(a, b) for a, b in zip(again, fine)) and not readout.softmax_failed()


def test_a_question_hides_no_failure_from_another_thread():
    x, w, labels = softmax_case(F32, 20, 16, 40)
    assert not readout.softmax_failed()
    told = []
    thread = threading.Thread(target=lambda: told.append(readout.softmax_failed()))      # what came before is not its matter
    thread.start()
    thread.join()
    lose(1)
    readout.softmax_loss(x, w, labels)
    thread = threading.Thread(target=lambda: told.append(readout.softmax_failed()))
    thread.start()
    thread.join()
    assert told[1] and readout.softmax_failed() and not readout.softmax_failed()


def test_a_classifier_tells_of_a_wait_that_ran_out():
    rng = np.random.default_rng(7)
    graphs, labels = random_graphs(60, rng, max_nodes=5), rng.permutation(60) % 40
    np.random.seed(4)
    tm = MultiClassGraphTsetlinMachine(40, 100, 2.0, depth=1, seed=1)
    tm.fit(graphs, labels % 3, epochs=1)
    head = readout.ClauseReadout(tm, embedding_size=24)
    head.fit(graphs, labels, epochs=1)
    before = head.score(graphs)
    lose(1)
    with pytest.raises(RuntimeError, match="ran out"):
        head.score(graphs)
    after = head.score(graphs)
    assert all(np.array_equal(a, b) for a, b in zip(before, after))
    for launches in (1, 2, 3):
        lose(launches)
        with pytest.raises(RuntimeError, match="ran out"):
            head.fit(graphs, labels, epochs=1)
    lose(1)
    readout.softmax_loss(*softmax_case(F32, 20, 16, 40))                     # not the classifier's matter
    assert all(math.isfinite(v) for v in head.fit(graphs, labels, epochs=1))


def test_a_classifier_of_more_graphs_than_are_scored_at_a_time(monkeypatch):
    rng = np.random.default_rng(5)
    graphs, labels = random_graphs(60, rng, max_nodes=5), rng.integers(0, 3, size=60)
    np.random.seed(4)
    tm = MultiClassGraphTsetlinMachine(40, 100, 2.0, depth=1, seed=1)
    tm.fit(graphs, labels, epochs=1)
    head = readout.ClauseReadout(tm, embedding_size=24)
    head.fit(graphs, labels, epochs=1)
    whole, bags = head.score(graphs), head.active_clauses(graphs)
    monkeypatch.setattr(readout, "OUTPUTS", 40 * 17 + 3)                          # 17 graphs, the last piece 9
    pieces = head.score(graphs)
    assert all(torch.equal(a, b) for a, b in zip(head.active_clauses(graphs), bags))
    # sums of up to 40 rows in another order, rounded to bfloat16: logits below 8 in magnitude are off by 2^-8 of that
    assert pieces[0].shape == (60,) and np.abs(pieces[1] - whole[1]).max() <= 2 ** -4
    # a fit that fails leaves what was learned
    monkeypatch.setattr(tm, "transform", lambda graphs: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        head.fit(graphs, labels + 1, epochs=1)
    monkeypatch.undo()
    again = head.score(graphs)
    assert all(np.array_equal(a, b) for a, b in zip(again, whole))


# ------------------------------------------------------------------------------------------------------- adamw
def test_adamw_of_the_same_tensor_twice_is_refused():
    p = torch.ones(600, device="cuda")
    for params in ([p, p], [p[:400], p[300:500]]):
        with pytest.raises(_lib.GtmError, match="overlap"):
            readout.adamw_step(params, [torch.ones_like(q) for q in params], readout.adamw_state(params), 0.1)
    with pytest.raises(_lib.GtmError, match="overlap"):
        readout.adamw_step([p], [p], readout.adamw_state([p]), 0.1)
    assert (p == 1).all()
    # one gradient for two parameters, and neighbours in one memory, are fine
    params, g = [p[:300], p[300:]], torch.ones(300, device="cuda")
    readout.adamw_step(params, [g, g], readout.adamw_state(params), 0.1)
    assert torch.equal(params[0], params[1]) and (p < 1).all()


# ------------------------------------------------------------------------- pieces, slices, streams, threads
@pytest.mark.parametrize("kind", TYPES)
def test_softmax_in_pieces_of_the_examples(kind):
    """More parts of statistics than the workspace holds at a time: the second piece of examples begins behind row 35,000."""
    n, d, v = 40000, 8, 30000
    x, w, labels = softmax_case(kind, n, d, v)
    labels[::7] = -1
    losses, normalisers = readout.softmax_loss(x, w, labels)
    label, log_probability = readout.softmax_predict(x, w)
    rows = torch.cat([torch.arange(0, n, 97, device="cuda"), torch.arange(35200, 35500, device="cuda"), torch.tensor([n - 1], device="cuda")])
    logits, off, normaliser = plain_softmax(x[rows], w, 1.0)
    bound = off.amax(1) + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs()
    near(normalisers[rows], normaliser, bound)
    at = labels[rows]
    near(losses[rows], torch.where(at >= 0, normaliser - logits[torch.arange(len(rows)), at.clamp_min(0)], 0.0), 2 * bound)
    top = logits.amax(1)
    near(log_probability[rows], top - normaliser, 2 * bound)
    # the label is one of those that cannot be told from the best
    assert (logits[torch.arange(len(rows)), label[rows]] >= top - 2 * off.amax(1)).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(9000, 300, 520), (4300, 1100, 260), (300, 5000, 40)])
def test_softmax_gradient_of_many_tiles(kind, n, d, v):
    """More than 64 tiles of the features' gradient, whose slices are counted by a bound."""
    x, w, labels = softmax_case(kind, n, d, v)
    normalisers = check_loss(x, w, labels, 1.0)
    check_gradient(x, w, labels, normalisers, torch.full((n,), 1.0 / n, device="cuda"), 1.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(50, 40, 70), (40, 30, 9)])
def test_softmax_gradient_against_differences_along_itself(kind, n, d, v):
    """Central differences of the formula in 64 bits in the gradient's own direction, where they are its square: what the roundings may be off is
    a small part of that, so that no gradient would not pass."""
    x, w, labels = softmax_case(kind, n, d, v)
    _, normalisers = readout.softmax_loss(x, w, labels)
    got = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(1, device="cuda"))
    base, at = [x.double(), w.double()], torch.arange(n)
    logits, off, normaliser = plain_softmax(x, w, 1.0)
    p = torch.softmax(logits, 1)
    q = p.clone()
    q[at, labels] -= 1.0
    # of q: the logits' and normalisers' errors, the exponential's 2^-21, the rounding to the operands' type
    wrong = p * (2 * off.amax(1, keepdim=True) + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs()[:, None]) + max(half(kind), 2.0 ** -22) * q.abs() + 2.0 ** -23
    bounds = [(wrong + (v + 16) * STEP * q.abs()) @ base[1].abs(), (wrong + (n + 16) * STEP * q.abs()).t() @ base[0].abs()]

    def loss(x, w):
        logits = x @ w.t()
        return (torch.logsumexp(logits, 1) - logits[at, labels]).sum()

    for i in (0, 1):
        way = got[i].double()
        way = way / way.norm()
        ends, h = [], 1e-5
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * h * way
            ends.append(loss(*moved))
        want = (ends[0] - ends[1]) / (2 * h)
        # differences: the third derivative's part h^2, and the losses' 2^-52 over h
        slack = ((bounds[i] + half(kind) * (got[i].double().abs() + bounds[i])) * way.abs()).sum() + 1e-6 * (1 + want.abs())
        assert slack <= 0.25 * want and abs((got[i].double() * way).sum() - want) <= slack


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_on_two_streams_at_once(bits):
    """Two batches in turn on one stream, and at the same time on two: each is what it is alone."""
    alone = []
    for seed in (2, 9):
        batch = batch_of(seed, bits)
        for _ in range(4):
            out = step_of(batch)
        alone.append(flat(out, batch))
    batches, streams, outs = [batch_of(2, bits), batch_of(9, bits)], [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    torch.cuda.synchronize()
    for _ in range(4):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                outs[k] = step_of(batches[k])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(flat(outs[k], batches[k]), alone[k]))


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_two_threads_at_once(bits):
    alone, batches, got, failed = [], [batch_of(s, bits) for s in (2, 9)], [None, None], []
    for seed in (2, 9):
        batch = batch_of(seed, bits)
        for _ in range(8):
            out = step_of(batch)
        alone.append(flat(out, batch))
    torch.cuda.synchronize()
    begin = threading.Barrier(2)

    def steps(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                begin.wait(timeout=60)
                for _ in range(8):
                    out = step_of(batches[k])
                got[k] = flat(out, batches[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                    # noqa: BLE001  told by the test
            failed.append(e)

    threads = [threading.Thread(target=steps, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(got[k], alone[k]))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,d,v", [(40, 24, 70), (9, 24, 300), (3, 24, 300), (30, 24, 10)])
def test_labels_masked_by_the_lowest_value(kind, n, d, v):
    """A column of ones, and the type's lowest value in it for labels that are not to be: logits of about that, probability zero, no NaN."""
    x, w, labels = softmax_case(kind, n, d, v)
    masked = torch.arange(v, device="cuda") % 3 == 1
    labels = torch.where(masked[labels], labels - 1, labels)
    x[:, 5], w[:, 5] = 1.0, 0.0
    kept = (~masked).nonzero()[:, 0]
    position = torch.zeros(v, dtype=torch.int64, device="cuda")
    position[kept] = torch.arange(len(kept), device="cuda")
    w[masked, 5] = torch.finfo(kind).min
    # as if there were only the other labels
    logits, off, normaliser = plain_softmax(x, w[kept], 1.0)
    bound = off.amax(1) + 2.0 ** -20 + 2.0 ** -22 * normaliser.abs()
    losses, normalisers = readout.softmax_loss(x, w, labels)
    near(normalisers, normaliser, bound)
    near(losses, normaliser - logits[torch.arange(n), position[labels]], 2 * bound)
    label, log_probability = readout.softmax_predict(x, w)
    near(log_probability, logits.amax(1) - normaliser, 2 * bound)
    assert not masked[label].any()
    dx, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(1, device="cuda"))
    want, _ = readout.softmax_loss_gradient(x, w[kept].contiguous(), position[labels], normalisers, torch.ones(1, device="cuda"))
    assert torch.isfinite(dx).all() and (dw[masked] == 0).all() and torch.isfinite(dw).all()
    size = torch.softmax(logits, 1) @ w[kept].double().abs() + w[labels].double().abs()
    near(dx, want, 4 * max(half(kind), (v + 16) * STEP) * size + least(kind))


def test_gradients_of_very_long_sums():
    """Sums of hundreds of thousands of terms of one sign, where neither product is cut into splits for want of tiles.  What tensor cores cut off is on the
    average of all results below 2^-23 for each of at most 2,048 steps of 16 terms; results' roundings have no sign."""
    bound = 2048 * 2.0 ** -23
    n, d, v = 1 << 18, 38 * 256, 33                              # dw: 38 tiles of 262,144 terms
    gen = generator(1)
    x, w = torch.rand(n, d, generator=gen, device="cuda", dtype=F16), torch.zeros(v, d, device="cuda", dtype=F16)
    labels = torch.arange(n, device="cuda") % 32
    _, normalisers = readout.softmax_loss(x, w, labels)
    _, dw = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.full((1,), 1 / 64, device="cuda"))
    want = torch.stack([x[i::16].double().sum(0) for i in range(16)]).sum(0) / 64 / v      # of the label that no example has
    assert abs((dw[32].double() / want - 1).mean().item()) <= bound
    del x, dw
    n, d, v = 64, 19 * 256, 1 << 20                              # dx: 19 tiles of 1,048,576 terms
    x, w = torch.zeros(n, d, device="cuda", dtype=F16), torch.rand(v, d, generator=gen, device="cuda", dtype=F16)
    w[0] = 0.0
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    _, normalisers = readout.softmax_loss(x, w, labels)
    dx, _ = readout.softmax_loss_gradient(x, w, labels, normalisers, torch.ones(1, device="cuda"))
    want = torch.stack([w[i::64].double().sum(0) for i in range(64)]).sum(0) / v
    assert abs((dx.double() / want - 1).mean().item()) <= bound


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,v", [(20, 300), (2, 300), (20, 10)])
def test_softmax_of_the_largest_scale(kind, n, v):
    """Any scale above zero and finite: logits that are equal stay so, however far it would take others."""
    x, w = torch.zeros(n, 16, device="cuda", dtype=kind), torch.ones(v, 16, device="cuda", dtype=kind)
    for scale in (1e-38, 1.0, 3.4e38):
        losses, normalisers = readout.softmax_loss(x, w, torch.zeros(n, dtype=torch.int64, device="cuda"), scale=scale)
        label, log_probability = readout.softmax_predict(x, w, scale=scale)
        want = torch.full((n,), math.log(v), device="cuda", dtype=torch.float64)
        near(losses, want, 2.0 ** -20 * want)
        near(normalisers, want, 2.0 ** -20 * want)
        near(log_probability, -want, 2.0 ** -20 * want)
        assert (label == 0).all()
