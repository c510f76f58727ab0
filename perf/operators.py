"""Performance cases of the readout operators: a softmax classifier trained on what clauses answer.

A machine's clauses answer for a graph; the rows of an embedding table that belong to the active clauses (or to the symbols of
a node) are added up; a softmax over labels is learned from the sums; AdamW moves the weights.  Three operators, each with
its gradient or update, are measured:

``op``  "embed"           rows of a table by id: one row for each id, or the sum of a bag of ids
        "embed_gradient"  the table's gradient
        "embed_train"     both, one after the other
        "loss_train"      softmax cross entropy and the gradients of features and label weights
        "predict"         most probable label and its log probability
        "adamw"           one step over all tensors, states in 32 or in 8 bits

Where ``own`` is false, ``run`` computes them from elementary torch operations in 32 bits.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -1
BLOCK = 256                 # elements of a tensor that share the scale of an 8-bit state
BETAS, EPS, LR, DECAY, SEED = (0.9, 0.999), 1e-8, 1e-3, 0.01, 1234
E4M3_LARGEST, SCALE_LEAST = 448.0, 2.0 ** -126


def listed():
    return [
        # online inference: the active clauses of one graph of a machine with 2,000 clauses
        dict(name="embed_one_graph", op="embed", ids=37, bags=1, rows=2000, dim=64, type="fp32", index="int32", spread="even", padding=0.0),
        # node symbols of a batch of padded sequences, wide rows of a length that fits no vector
        dict(name="embed_symbols", op="embed", ids=24001, bags=0, rows=49999, dim=1001, type="bf16", index="int64", spread="zipf", padding=0.05),
        # the same kind of batch in training, a few symbols being most of it
        dict(name="embed_symbols_gradient", op="embed_gradient", ids=65539, bags=0, rows=30011, dim=512, type="fp16", index="int64", spread="zipf", padding=0.05),
        # a training step of 4,096 graphs over the 20,000 clauses of the largest machine, one clause in a hundred active
        dict(name="embed_clauses_train", op="embed_train", ids=819200, bags=4096, rows=20000, dim=256, type="bf16", index="int32", spread="even", padding=0.0),
        # ten labels, a batch that fills no tile
        dict(name="loss_small", op="loss_train", examples=60, dim=64, labels=10, type="fp32", margin=2.0, ignored=0.0),
        # a batch of ragged sizes, padded examples among it
        dict(name="loss_ragged", op="loss_train", examples=1003, dim=520, labels=20011, type="fp16", margin=4.0, ignored=0.2),
        # training with a large label set
        dict(name="loss_large", op="loss_train", examples=8192, dim=1024, labels=65536, type="bf16", margin=4.0, ignored=0.02),
        # online inference: one example, a large label set
        dict(name="predict_one", op="predict", examples=1, dim=1024, labels=131072, type="bf16", margin=9.0),
        # evaluation of a set of images in 32 bits
        dict(name="predict_images", op="predict", examples=2000, dim=333, labels=1000, type="fp32", margin=9.0),
        # the two tensors of a small readout
        dict(name="adamw_small", op="adamw", tensors=2, least=640, most=128000, total=128640, type="fp32", gradients="fp32", bits=32),
        # a model of many tensors, from biases to matrices
        dict(name="adamw_many", op="adamw", tensors=150, least=17, most=4000000, total=60000000, type="fp32", gradients="bf16", bits=32),
        # large tables with states in 8 bits
        dict(name="adamw_tables_8bit", op="adamw", tensors=5, least=20000, most=120000000, total=200000000, type="bf16", gradients="bf16", bits=8),
    ]


def _log_between(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    op = rng.choice(["embed", "embed_gradient", "embed_train", "loss_train", "loss_train", "predict", "adamw", "adamw"])
    if op.startswith("embed"):
        ids = _log_between(rng, 1, 800000)
        dim = _log_between(rng, 8, min(2048, max(8, 200000000 // ids)))
        return dict(op=op, ids=ids, bags=rng.choice([0, _log_between(rng, 1, min(ids, 8192))]) if ids * dim < 100000000 else _log_between(rng, 1, 8192),
                    rows=_log_between(rng, 2, 60000), dim=dim, type=rng.choice(sorted(TYPES)), index=rng.choice(["int32", "int64"]),
                    spread=rng.choice(["even", "zipf"]), padding=rng.choice([0.0, 0.1]))
    if op == "adamw":
        bits = rng.choice([32, 8])
        total = _log_between(rng, 5000, 50000000)
        kind = rng.choice(["fp32", "bf16"])
        return dict(op=op, tensors=_log_between(rng, 1, 200), least=rng.randrange(1, 500), most=max(1000, total // 2), total=total, type=kind,
                    gradients=kind if bits == 8 else rng.choice(["fp32", "bf16"]), bits=bits)
    kind = rng.choice(sorted(TYPES))
    examples = _log_between(rng, 1, 8192)
    dim = _log_between(rng, 16, 2048)
    most = 5.0e11 if op == "loss_train" else 1.0e12
    labels = _log_between(rng, 2, max(2, min(130000, int(most / (1 if kind != "fp32" else 6) / examples / dim))))
    if op == "predict":
        return dict(op=op, examples=examples, dim=dim, labels=labels, type=kind, margin=9.0)
    return dict(op=op, examples=examples, dim=dim, labels=labels, type=kind, margin=rng.choice([0.0, 4.0, 8.0]), ignored=rng.choice([0.0, 0.1]))


# ------------------------------------------------------------------------------------------------- inputs
def _ids(case, gen):
    n, rows = case["ids"], case["rows"]
    if case["spread"] == "zipf":     # the k-th most frequent id with a probability near 1 / k
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        ids = torch.exp(u * math.log(rows + 1)).long() - 1
        ids = (ids.clamp(0, rows - 1) * 7919 + 13) % rows        # frequent ids are spread over the table
    else:
        ids = torch.randint(rows, (n,), generator=gen, device="cuda")
    if case["padding"]:
        ids[torch.rand(n, generator=gen, device="cuda") < case["padding"]] = -1
    return ids.to(getattr(torch, case["index"]))


def _offsets(case, gen):
    """Bags of uneven sizes, empty ones among them."""
    inner = torch.randint(case["ids"] + 1, (case["bags"] - 1,), generator=gen, device="cuda").sort().values
    ends = torch.tensor([0, case["ids"]], device="cuda")
    return torch.cat([ends[:1], inner, ends[1:]]).to(getattr(torch, case["index"]))


def sizes_of(case):
    """Sizes of the tensors of an "adamw" case: spread over their logarithm, then scaled to the total."""
    rng = np.random.RandomState(case["tensors"])
    raw = np.exp(rng.uniform(math.log(case["least"]), math.log(case["most"] + 1), case["tensors"]))
    raw[0] = case["most"]
    raw[-1] = case["least"]
    return [max(1, int(v)) for v in raw * (case["total"] / raw.sum())]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, kind = case["op"], TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    state = dict(case=case)
    if op.startswith("embed"):
        state["ids"] = _ids(case, gen)
        state["offsets"] = _offsets(case, gen) if case["bags"] else None
        if op != "embed_gradient":
            state["table"] = normal(case["rows"], case["dim"]).to(kind)
        if op != "embed":
            state["gradient"] = (normal(case["bags"] or case["ids"], case["dim"]) * 0.1).to(kind)
        state["scale"] = math.sqrt(case["dim"])
    elif op == "adamw":
        sizes = sizes_of(case)
        starts = np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])])
        total = int(starts[-1])
        real = torch.zeros(total, dtype=torch.bool, device="cuda")
        for n, at in zip(sizes, starts):
            real[at:at + n] = True
        flat = torch.where(real, normal(total) * 0.05, 0.0).to(kind)
        gradient = torch.where(real, normal(total) * torch.exp(normal(total) - 6), 0.0).to(TYPES[case["gradients"]])
        # states some way into training, of the size that such gradients leave
        first = torch.where(real, normal(total) * 1e-3, 0.0)
        second = torch.where(real, torch.exp(2 * normal(total) - 13), 0.0)
        state.update(flat=flat, flat_gradient=gradient, steps=torch.full((1,), 100, dtype=torch.int64, device="cuda"),
                     params=[flat[at:at + n] for n, at in zip(sizes, starts)],
                     gradients=[gradient[at:at + n] for n, at in zip(sizes, starts)])
        if case["bits"] == 32:
            state.update(first=first, second=second)
        else:
            root = second.sqrt()
            for name, x in (("first", first), ("second", root)):
                scales = (x.reshape(-1, BLOCK).abs().amax(1) / E4M3_LARGEST).clamp_min(SCALE_LEAST)
                state[name + "_scales"] = scales
                state[name] = (x.reshape(-1, BLOCK) / scales[:, None]).clamp(-E4M3_LARGEST, E4M3_LARGEST).to(torch.float8_e4m3fn).reshape(-1)
    else:
        n, d, v = case["examples"], case["dim"], case["labels"]
        weights = normal(v, d) / math.sqrt(d)
        labels = torch.randint(v, (n,), generator=gen, device="cuda")
        # an example has a part in the direction of its label's weights: some way into training, or (to predict) at its end
        features = normal(n, d) + case["margin"] * weights[labels] / weights[labels].norm(dim=1, keepdim=True)
        state.update(features=features.to(kind), weights=weights.to(kind), scale=1.0)
        if op == "loss_train":
            labels[torch.rand(n, generator=gen, device="cuda") < case["ignored"]] = IGNORE
            state["labels"] = labels
            state["gradients"] = torch.full((n,), 1.0 / n, device="cuda")
    return state


# --------------------------------------------------------------------------------------------- plain forms
def _plain_bag_of(state, count):
    """Bag of each id."""
    at = torch.arange(count, device="cuda")
    if state["offsets"] is None:
        return at
    return torch.searchsorted(state["offsets"].long()[1:].contiguous(), at, right=True)


def _plain_embed(state):
    ids, table = state["ids"].long(), state["table"]
    rows = table[ids.clamp_min(0)].float() * (ids >= 0)[:, None]
    if state["offsets"] is not None:
        rows = torch.zeros(state["offsets"].numel() - 1, table.shape[1], device="cuda").index_add_(0, _plain_bag_of(state, ids.numel()), rows)
    return (rows * state["scale"]).to(table.dtype)


def _plain_embed_gradient(state):
    ids, gradient = state["ids"].long(), state["gradient"]
    rows = gradient.float()[_plain_bag_of(state, ids.numel())] * (ids >= 0)[:, None]
    out = torch.zeros(state["case"]["rows"], gradient.shape[1], device="cuda").index_add_(0, ids.clamp_min(0), rows)
    return (out * state["scale"]).to(gradient.dtype)


def _plain_loss_train(state):
    x, w, labels = state["features"].float(), state["weights"].float(), state["labels"]
    kept = labels != IGNORE
    at = labels.clamp_min(0)[:, None]
    logits = (x @ w.t()) * state["scale"]
    top = logits.amax(1, keepdim=True)
    normaliser = (logits - top).exp().sum(1, keepdim=True).log() + top
    losses = ((normaliser - logits.gather(1, at))[:, 0]) * kept
    p = (logits - normaliser).exp()
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    p *= (state["gradients"] * kept * state["scale"])[:, None]
    return losses, normaliser[:, 0], (p @ w).to(state["features"].dtype), (p.t() @ x).to(state["weights"].dtype)


def _plain_predict(state):
    logits = (state["features"].float() @ state["weights"].float().t()) * state["scale"]
    top, label = logits.max(1)
    rest = (logits - top[:, None]).exp().scatter_(1, label[:, None], 0.0).sum(1)      # all but the label: 1 + rest would drop a small rest's bits
    return label, -torch.log1p(rest)


def _hash(x):
    """32 bits of int64 tensors: the mixing steps of MurmurHash3's finaliser."""
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _round_to_e4m3(x, scales, random, least):
    """|x| / scale to a neighbouring e4m3 value, the upper one with the probability of its nearness; `random`: 16 bits."""
    r = x.abs().reshape(-1, BLOCK) * (1.0 / scales)[:, None]
    r = r.reshape(-1)
    normal = ((r.view(torch.int32) + (random << 4).int()) & ~0xFFFFF).view(torch.float32)
    small = torch.floor(r * 512 + random.float() * 2.0 ** -16) * 2.0 ** -9
    q = torch.where(r >= 2.0 ** -6, normal, small).clamp_max(E4M3_LARGEST)
    if least:
        q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
    return torch.where(x < 0, -q, q).to(torch.float8_e4m3fn)


def _plain_adamw(state):
    s = state
    f = lambda v: float(np.float32(v))                 # noqa: E731  constants are rounded once, like the tensors they meet
    b1, b2 = BETAS
    s["steps"] += 1
    t = s["steps"].double()
    step_size = (LR / (1 - b1 ** t)).float()
    root_correction = (1 / (1 - b2 ** t).sqrt()).float()
    g = s["flat_gradient"].float()
    p = s["flat"].float()
    if s["case"]["bits"] == 32:
        first, second = s["first"], s["second"]
    else:
        first = (s["first"].float().reshape(-1, BLOCK) * s["first_scales"][:, None]).reshape(-1)
        root = (s["second"].float().reshape(-1, BLOCK) * s["second_scales"][:, None]).reshape(-1)
        second = root * root
    first = first * f(b1) + g * f(1 - b1)
    second = second * f(b2) + (g * g) * f(1 - b2)
    root = second.sqrt()
    s["flat"].copy_(p * f(1 - LR * DECAY) - step_size * (first / (root * root_correction + f(EPS))))
    if s["case"]["bits"] == 32:
        s["first"].copy_(first)
        s["second"].copy_(second)
        return s["flat"], s["first"], s["second"]
    key = _hash(_hash(torch.full_like(s["steps"], SEED)) + s["steps"])
    random = _hash(torch.arange(g.numel(), device="cuda") * 0x9E3779B1 + key)
    for name, x, bits, least in (("first", first, random >> 16, False), ("second", root, random & 0xFFFF, True)):
        scales = (x.reshape(-1, BLOCK).abs().amax(1) * f(1 / E4M3_LARGEST)).clamp_min(SCALE_LEAST)
        s[name + "_scales"].copy_(scales)
        s[name].copy_(_round_to_e4m3(x, scales, bits, least))
    return s["flat"], s["first"], s["first_scales"], s["second"], s["second_scales"]


def run(state):
    op = state["case"]["op"]
    if own:
        from graphtsetlinmachine_b200 import readout

        if op == "embed":
            return readout.embed(state["table"], state["ids"], offsets=state["offsets"], scale=state["scale"])
        if op == "embed_gradient":
            return readout.embed_gradient(state["gradient"], state["ids"], state["case"]["rows"], offsets=state["offsets"], scale=state["scale"])
        if op == "embed_train":
            return (readout.embed(state["table"], state["ids"], offsets=state["offsets"], scale=state["scale"]),
                    readout.embed_gradient(state["gradient"], state["ids"], state["case"]["rows"], offsets=state["offsets"], scale=state["scale"]))
        if op == "loss_train":
            losses, normalisers = readout.softmax_loss(state["features"], state["weights"], state["labels"], scale=state["scale"], ignore_label=IGNORE)
            return (losses, normalisers) + tuple(readout.softmax_loss_gradient(
                state["features"], state["weights"], state["labels"], normalisers, state["gradients"], scale=state["scale"], ignore_label=IGNORE))
        if op == "predict":
            return tuple(readout.softmax_predict(state["features"], state["weights"], scale=state["scale"]))
        names = ("first", "second") if state["case"]["bits"] == 32 else ("first", "first_scales", "second", "second_scales")
        readout.adamw_step(state["params"], state["gradients"], {n: state[n] for n in names + ("steps",)}, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=SEED)
        return (state["flat"],) + tuple(state[n] for n in names)
    if op == "embed":
        return _plain_embed(state)
    if op == "embed_gradient":
        return _plain_embed_gradient(state)
    if op == "embed_train":
        return _plain_embed(state), _plain_embed_gradient(state)
    if op == "loss_train":
        return _plain_loss_train(state)
    if op == "predict":
        return _plain_predict(state)
    return _plain_adamw(state)


# ------------------------------------------------------------------------------------------------- floors
def work(case):
    op, size = case["op"], TYPES[case["type"]].itemsize
    if op.startswith("embed"):
        index = 4 if case["index"] == "int32" else 8
        outs = case["bags"] or case["ids"]
        read = min(case["rows"], case["ids"])
        ahead = case["ids"] * index + (case["bags"] + 1) * index * bool(case["bags"]) + (read + outs) * case["dim"] * size
        back = case["ids"] * index + (case["rows"] + outs) * case["dim"] * size
        passes = {"embed": (ahead,), "embed_gradient": (back,), "embed_train": (ahead, back)}[op]
        return {"bytes": sum(passes), "flops": len(passes) * case["ids"] * case["dim"]}
    if op == "adamw":
        n = sum(sizes_of(case))
        states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": int(n * (2 * size + TYPES[case["gradients"]].itemsize + states)), "flops": 15 * n}
    n, d, v = case["examples"], case["dim"], case["labels"]
    if op == "predict":
        return {"bytes": (n + v) * d * size + n * 12, "flops": 2 * n * v * d}
    return {"bytes": 2 * (n + v) * d * size + n * 20, "flops": 6 * n * v * d}


# -------------------------------------------------------------------------------------- values in 64 bits
def _exact_embed(state):
    """Bags by differences of running sums in 64 bits."""
    ids, table = state["ids"].long(), state["table"].double()
    padded = torch.cat([table, torch.zeros(1, table.shape[1], dtype=torch.float64, device="cuda")])
    rows = padded[torch.where(ids < 0, table.shape[0], ids)]
    if state["offsets"] is not None:
        sums = torch.cat([torch.zeros(1, table.shape[1], dtype=torch.float64, device="cuda"), rows.cumsum(0)])
        rows = sums[state["offsets"].long()[1:]] - sums[state["offsets"].long()[:-1]]
    return rows * state["scale"]


def _exact_embed_gradient(state):
    """Column by column a histogram of ids, weighted by the gradient."""
    ids = state["ids"].long()
    rows, offsets = state["case"]["rows"], state["offsets"]
    gradient = state["gradient"].double()
    if offsets is not None:
        gradient = gradient.repeat_interleave(offsets.long().diff(), dim=0)
    columns = [torch.bincount(ids + 1, weights=gradient[:, c], minlength=rows + 1)[1:] for c in range(gradient.shape[1])]
    return torch.stack(columns, 1) * state["scale"]


def _exact_loss_train(state):
    x, w, labels = state["features"].double(), state["weights"].double(), state["labels"]
    logits = (x @ w.t()) * state["scale"]
    normalisers = torch.logsumexp(logits, 1)
    kept = labels >= 0
    at = torch.where(kept, labels, 0)
    losses = torch.where(kept, normalisers - logits[torch.arange(len(at), device="cuda"), at], 0.0)
    logits.sub_(normalisers[:, None]).exp_()
    logits[torch.arange(len(at), device="cuda"), at] -= 1
    logits.mul_(torch.where(kept, state["gradients"].double() * state["scale"], 0.0)[:, None])
    return losses, normalisers, logits @ w, logits.t() @ x


def _exact_predict(state):
    logits = (state["features"].double() @ state["weights"].double().t()) * state["scale"]
    return logits.argmax(1), logits.amax(1) - torch.logsumexp(logits, 1)


def _exact_adamw(state):
    s, (b1, b2) = state, BETAS
    t = int(s["steps"]) + 1
    g = s["flat_gradient"].double()
    m, v = s["first"].double(), s["second"].double()
    if s["case"]["bits"] == 8:
        m = m * s["first_scales"].double().repeat_interleave(BLOCK)
        v = (v * s["second_scales"].double().repeat_interleave(BLOCK)).square()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g.square()
    moved = s["flat"].double() * (1 - LR * DECAY) - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    if s["case"]["bits"] == 32:
        return moved, m, v
    # which of two codes a value goes to may hang on its last bit in 32: the codes have no value in 64
    scales = [x.reshape(-1, BLOCK).abs().amax(1).div(E4M3_LARGEST).clamp_min(SCALE_LEAST) for x in (m, v.sqrt())]
    return moved, None, scales[0], None, scales[1]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        return _exact_embed(state)
    if op == "embed_gradient":
        return _exact_embed_gradient(state)
    if op == "embed_train":
        return _exact_embed(state), _exact_embed_gradient(state)
    if op == "loss_train":
        return _exact_loss_train(state)
    if op == "predict":
        return _exact_predict(state)
    return _exact_adamw(state)
