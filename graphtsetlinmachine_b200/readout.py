"""A softmax readout on what clauses answer: its operators, and a classifier that learns with them.

The clauses of a trained machine answer for a graph (``transform``); the rows of an embedding table that belong to the active
clauses are added up (``embed``), a softmax over labels is learned from the sums (``softmax_loss``), and AdamW moves the weights
(``adamw_step``).  NOT IN THE REFERENCE, whose ``transform`` (tm.py:814-851) leaves that to other libraries.

The operators take torch tensors on one CUDA device and call the kernels of ``libgtm_b200.so`` through the C ABI; there is no
other path.  Gradients are functions of their own (``embed_gradient``, ``softmax_loss_gradient``), not part of autograd.  Work goes to the
current stream of the tensors' device, whichever device is current, and no call synchronises.  Results, and workspaces, come from
torch's allocator on that stream, so that calls can be captured into a CUDA graph (after one call outside it has loaded the kernels).
Matrices are float32, bfloat16 or float16 with any row stride and elements next to each other within a row; a tensor in
another order is refused, not copied.  The softmax operators multiply float32 matrices in parts on the tensor cores: an infinite
element gives NaN logits there (mask with the lowest value instead).
"""

import array
import ctypes as C

import numpy as np
import torch

from . import _lib

__all__ = ["embed", "embed_gradient", "softmax_loss", "softmax_loss_gradient", "softmax_predict", "softmax_failed", "adamw_state", "adamw_step",
           "ClauseReadout"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INDEX = {torch.int32: 0, torch.int64: 1}
# the current stream's handle, without the object around it where torch has that
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
BLOCK = 256      # elements; every tensor starts at a multiple of it in the flat states of `adamw_step`
OUTPUTS = 1 << 28      # clause outputs, of four bytes each, that `ClauseReadout` has on the host at a time


def _cuda(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s is a torch tensor, not %s" % (name, type(t).__name__))
    if not t.is_cuda:
        raise ValueError("%s lies on %s: readout operators work on CUDA tensors" % (name, t.device))
    return t


def _device_of(name, t, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s is a torch tensor, not %s" % (name, type(t).__name__))
    if t.device != device:
        raise ValueError("%s lies on %s, the first argument on %s" % (name, t.device, device))


def _matrix(name, t, dtype=None):
    """Checks a matrix; returns its rows, its columns and its row stride in elements."""
    if t.dim() != 2:
        raise ValueError("%s has %d dimensions instead of two" % (name, t.dim()))
    if t.dtype not in _TYPES or (dtype is not None and t.dtype != dtype):
        raise TypeError("%s is of %s: %s" % (name, t.dtype, dtype or "float32, bfloat16 and float16 are taken"))
    rows, columns = t.shape
    if columns == 0:
        raise ValueError("%s has no columns" % name)
    stride, step = t.stride()
    if step != 1 and columns > 1:
        raise ValueError("the elements of a row of %s lie %d apart: give it as %s.contiguous()" % (name, step, name))
    return rows, columns, stride if rows > 1 else columns


def _index(name, t, device, dim=1):
    _device_of(name, t, device)
    wide = _INDEX.get(t.dtype)
    if wide is None:
        raise TypeError("%s is of %s: int32 and int64 are taken" % (name, t.dtype))
    if (dim is not None and t.dim() != dim) or not t.is_contiguous():
        raise ValueError("%s is not a contiguous tensor%s" % (name, "" if dim is None else " of %d dimension(s)" % dim))
    return wide


def _vector(name, t, size, device):
    _device_of(name, t, device)
    if t.dtype != torch.float32 or t.shape != (size,) or not t.is_contiguous():
        raise ValueError("%s is not a contiguous float32 tensor of %d elements" % (name, size))


def _stream(device):
    return _current_stream(device.index)


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device)


def _bags(ids, offsets, device):
    """Checks ids and offsets: (wide ids, wide offsets, number of results, their leading shape)."""
    if offsets is None:
        return _index("ids", ids, device, None), 0, ids.numel(), tuple(ids.shape)
    wide, wide_offsets, bags = _index("ids", ids, device), _index("offsets", offsets, device), offsets.shape[0] - 1
    if bags < 0:
        raise ValueError("offsets has an element more than there are bags, so at least one")
    return wide, wide_offsets, bags, (bags,)


def embed(table, ids, offsets=None, scale=1.0):
    """``scale`` times the rows ``ids`` of ``table``: ``[*ids.shape, columns]``; with ``offsets`` (bag ``b`` is
    ``ids[offsets[b]:offsets[b + 1]]``) the sums of the bags' rows: ``[bags, columns]``, of the table's type, summed in 32 bits.

    A negative id is padding: a row of zeros, nothing in a bag.  An id beyond the table gives NaN.  ``offsets`` must not decrease;
    ids outside every bag are not used."""
    device = _cuda("table", table).device
    rows, columns, stride = _matrix("table", table)
    wide, wide_offsets, count, shape = _bags(ids, offsets, device)
    number = ids.numel()
    if rows == 0:
        raise ValueError("table has no rows")
    lib = _lib.load()
    out = torch.empty(shape + (columns,), dtype=table.dtype, device=device)
    workspace, size = None, 0
    if offsets is not None and number > 128:
        need = C.c_uint64()
        _lib.check(lib.gtm_embed_workspace(number, columns, 1, C.byref(need)))
        size = need.value
        workspace = _workspace(size, device)
    _lib.check(lib.gtm_embed(device.index, _stream(device), _TYPES[table.dtype], table.data_ptr(), rows, columns, stride, ids.data_ptr(), wide, number,
                             None if offsets is None else offsets.data_ptr(), wide_offsets, count, scale, out.data_ptr(),
                             None if workspace is None else workspace.data_ptr(), size))
    return out


def embed_gradient(gradient, ids, rows, offsets=None, scale=1.0):
    """Gradient ``[rows, columns]`` of the table of ``embed(table, ids, offsets, scale)`` from the ``gradient`` of its result.

    Each row is summed in 32 bits in the order of ``ids``: results do not change from run to run."""
    device = _cuda("gradient", gradient).device
    wide, wide_offsets, count, shape = _bags(ids, offsets, device)
    if gradient.dim() < 1 or tuple(gradient.shape[:-1]) != shape:
        raise ValueError("gradient has shape %s, the result of embed has %s rows" % (tuple(gradient.shape), shape))
    if gradient.dim() != 2:
        if not gradient.is_contiguous():
            raise ValueError("gradient is not contiguous: only one of two dimensions may have a row stride")
        gradient = gradient.view(count, gradient.shape[-1])
    _, columns, stride = _matrix("gradient", gradient)
    rows = int(rows)
    if rows < 1:
        raise ValueError("a table of %d rows" % rows)
    lib = _lib.load()
    out = torch.empty((rows, columns), dtype=gradient.dtype, device=device)
    need = C.c_uint64()
    _lib.check(lib.gtm_embed_gradient_workspace(ids.numel(), rows, columns, C.byref(need)))
    workspace = _workspace(need.value, device)
    _lib.check(lib.gtm_embed_gradient(device.index, _stream(device), _TYPES[gradient.dtype], gradient.data_ptr(), columns, stride, ids.data_ptr(), wide, ids.numel(),
                                      None if offsets is None else offsets.data_ptr(), wide_offsets, count, scale, out.data_ptr(), rows,
                                      workspace.data_ptr(), need.value))
    return out


def _softmax_arguments(features, weights, scale, call):
    """Checks features and weights: (library, device, the arguments that describe them, workspace or None, its address, its size).
    Of a call: 0 for the loss, 1 for its gradient, 2 for the prediction."""
    device = _cuda("features", features).device
    _device_of("weights", weights, device)
    n, d, x_stride = _matrix("features", features)
    v, columns, w_stride = _matrix("weights", weights, features.dtype)
    if d != columns:
        raise ValueError("features have %d columns, weights %d" % (d, columns))
    if v == 0:
        raise ValueError("weights has no rows: there is no label")
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale %r is not above zero and finite" % scale)
    lib = _lib.load()
    kind, x, w = _TYPES[features.dtype], features.data_ptr(), weights.data_ptr()
    workspace, address, size = None, None, 0
    if call == 1 or v > 32 or v * d > 24576 or n > 65536:
        need = C.c_uint64()
        _lib.check(lib.gtm_softmax_workspace(kind, x, n, x_stride, w, v, w_stride, d, call, C.byref(need)))
        size = need.value
        workspace = _workspace(max(size, 1), device)
        address = workspace.data_ptr()
    return lib, device, (device.index, _stream(device), kind, x, n, x_stride, w, v, w_stride, d), workspace, address, size


def _wanted(labels, n, device):
    wide = _index("labels", labels, device)
    if labels.shape[0] != n:
        raise ValueError("%d labels for %d examples" % (labels.shape[0], n))
    return wide


def softmax_loss(features, weights, labels, scale=1.0, ignore_label=-1):
    """Softmax cross entropy of ``labels`` (one per example) where the logits are ``scale * features @ weights.T``, which are never
    kept: (losses, normalisers), float32 of one element per example; a normaliser is the logarithm of the sum of an example's
    exponentials.  ``scale`` is above zero.

    An example whose label is ``ignore_label`` has loss zero; the loss of a label that there is not is NaN."""
    lib, device, what, workspace, address, size = _softmax_arguments(features, weights, scale, 0)
    n = what[4]
    wide = _wanted(labels, n, device)
    losses = torch.empty(n, dtype=torch.float32, device=device)
    normalisers = torch.empty(n, dtype=torch.float32, device=device)
    _lib.check(lib.gtm_softmax_loss(*what, labels.data_ptr(), wide, ignore_label, scale, losses.data_ptr(), normalisers.data_ptr(), address, size))
    return losses, normalisers


def softmax_loss_gradient(features, weights, labels, normalisers, gradients, scale=1.0, ignore_label=-1):
    """Gradients (of features, of weights; each of the inputs' type) of ``softmax_loss`` with the same arguments.  ``normalisers``: what
    that call gave; ``gradients``: dL/dlosses, float32 of one element per example or of one element for all (1 / n for the mean).

    An ignored example's gradient is zero, and it adds nothing to the weights' gradient, whatever its features hold.  An example whose label
    there is not, or whose element of ``gradients`` is not finite, spoils its own gradient and the weights', not that of other examples."""
    lib, device, what, workspace, address, size = _softmax_arguments(features, weights, scale, 1)
    n = what[4]
    wide = _wanted(labels, n, device)
    _vector("normalisers", normalisers, n, device)
    _device_of("gradients", gradients, device)
    if gradients.dtype != torch.float32 or gradients.dim() > 1 or gradients.numel() not in (1, n) or not gradients.is_contiguous():
        raise ValueError("gradients is not a contiguous float32 tensor of one element, or of one for each of %d examples" % n)
    features_gradient = torch.empty(features.shape, dtype=features.dtype, device=device)
    weights_gradient = torch.empty(weights.shape, dtype=weights.dtype, device=device)
    _lib.check(lib.gtm_softmax_loss_gradient(*what, labels.data_ptr(), wide, ignore_label, scale, normalisers.data_ptr(), gradients.data_ptr(),
                                             1 if gradients.numel() == n else 0, features_gradient.data_ptr(), weights_gradient.data_ptr(),
                                             address, size))
    return features_gradient, weights_gradient


def softmax_predict(features, weights, scale=1.0):
    """(labels int64, log probabilities float32): each example's most probable label under logits ``scale * features @ weights.T``,
    the lowest of equal ones.  -1 and NaN where an example's logits are not numbers."""
    lib, device, what, workspace, address, size = _softmax_arguments(features, weights, scale, 2)
    labels = torch.empty(what[4], dtype=torch.int64, device=device)
    log_probabilities = torch.empty(what[4], dtype=torch.float32, device=device)
    _lib.check(lib.gtm_softmax_predict(*what, scale, labels.data_ptr(), log_probabilities.data_ptr(), address, size))
    return labels, log_probabilities


def softmax_failed(device=0):
    """Whether a wait inside a softmax kernel (ten seconds at most) ran out on the device since the calling thread asked last.  What could not be
    computed then is NaN (a label -1) in the call's results.  Waits for the device."""
    failed = C.c_int()
    _lib.check(_lib.load().gtm_softmax_failed(int(device), C.byref(failed)))
    return bool(failed.value)


def _padded(sizes):
    return sum([-(-n // BLOCK) for n in sizes]) * BLOCK


def adamw_state(params, state_bits=32):
    """States of ``adamw_step`` for a list of CUDA tensors, all zero: a dict of ``steps`` (int64, one element) and the flat moments of all
    tensors, each tensor at a multiple of 256 elements.  32 bits: ``first`` and ``second``, float32.  8 bits: ``first`` and ``second``
    (of the second moment's root), float8_e4m3fn, in units of ``first_scales`` and ``second_scales``, one float32 per 256 elements."""
    params = list(params)
    if not params:
        raise ValueError("no tensors")
    if state_bits not in (8, 32):
        raise ValueError("states of %r bits: 8 or 32" % (state_bits,))
    device, total = _cuda("params[0]", params[0]).device, _padded([p.numel() for p in params])
    kind = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
    state = {"steps": torch.zeros(1, dtype=torch.int64, device=device)}
    for name in ("first", "second"):
        state[name] = torch.zeros(total, dtype=torch.uint8 if state_bits == 8 else kind, device=device).view(kind)
        if state_bits == 8:
            state[name + "_scales"] = torch.zeros(total // BLOCK, dtype=torch.float32, device=device)
    return state


def _pointers(name, tensors, shapes, device):
    """Data pointers of a list of contiguous tensors of one type on one device, of the given shapes (an array of integers), and that type."""
    count, index = len(tensors), device.index
    try:
        kind = tensors[0].dtype
        # lists are compared as a whole; which tensor it is matters when they differ
        same = ([t.dtype for t in tensors] == [kind] * count and [t.get_device() for t in tensors] == [index] * count
                and all([t.is_contiguous() for t in tensors]) and [t.shape for t in tensors] == shapes)
    except AttributeError:
        raise TypeError("%s is a list of torch tensors" % name) from None
    if kind not in _TYPES:
        raise TypeError("%s[0] is of %s: float32, bfloat16 and float16 are taken" % (name, kind))
    if not same:
        for i, t in enumerate(tensors):
            if t.dtype != kind or t.device != device or not t.is_contiguous() or t.shape != shapes[i]:
                raise ValueError("%s[%d] is not a contiguous %s tensor on %s of the parameter's shape" % (name, i, kind, device))
    return array.array("Q", [t.data_ptr() for t in tensors]), kind


def _address(a):
    return None if a is None else a.buffer_info()[0]


def adamw_step(params, gradients, state, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, gradient_scale=1.0, copies=None, seed=0):
    """One AdamW step over a list of tensors, in place, in one launch for up to 512 of them.  ``state`` (see ``adamw_state``) decides
    between states of 32 and of 8 bits, and counts the steps on the device.  All parameters have one type, all gradients have one; ``copies`` (optional,
    bfloat16 or float16) receive the parameters once more; nothing that is written may share memory with anything else.  States of 8 bits are rounded by a hash of ``seed`` (0 to 2^32 - 1), the step and the
    element: the same call gives the same result.  The numbers, ``lr`` among them, are those of the call: a captured step keeps them."""
    params, gradients = list(params), list(gradients)
    if not params:
        raise ValueError("no tensors")
    if len(gradients) != len(params) or (copies is not None and len(copies) != len(params)):
        raise ValueError("%d parameters, %d gradients%s" % (len(params), len(gradients), "" if copies is None else ", %d copies" % len(copies)))
    device = _cuda("params[0]", params[0]).device
    shapes = [p.shape for p in params]
    sizes = [p.numel() for p in params]
    param_ptrs, param_kind = _pointers("params", params, shapes, device)
    gradient_ptrs, gradient_kind = _pointers("gradients", gradients, shapes, device)
    copy_ptrs, copy_kind = (None, torch.bfloat16) if copies is None else _pointers("copies", list(copies), shapes, device)
    if copy_kind == torch.float32:
        raise TypeError("copies are bfloat16 or float16")
    counts = array.array("q", sizes)
    total = _padded(sizes)
    first, second, steps = state["first"], state["second"], state["steps"]
    narrow = first.dtype == torch.float8_e4m3fn
    if not narrow and first.dtype != torch.float32:
        raise TypeError("state is of %s: float32 or float8_e4m3fn" % first.dtype)
    scales = (state["first_scales"], state["second_scales"]) if narrow else (None, None)
    for name, t, size, kind in (("first", first, total, first.dtype), ("second", second, total, first.dtype), ("steps", steps, 1, torch.int64),
                                ("first_scales", scales[0], total // BLOCK, torch.float32), ("second_scales", scales[1], total // BLOCK, torch.float32)):
        if t is not None and (t.dtype != kind or t.numel() != size or t.device != device or not t.is_contiguous()):
            raise ValueError("state[%r] is not a contiguous %s tensor of %d elements on %s" % (name, kind, size, device))
    if not 0 <= seed < 1 << 32:
        raise ValueError("seed %r is not within 0 to 2^32 - 1" % (seed,))
    _lib.check(_lib.load().gtm_adamw_step(
        device.index, _stream(device), len(params), _address(counts), _TYPES[param_kind], _address(param_ptrs), _TYPES[gradient_kind], _address(gradient_ptrs),
        _TYPES[copy_kind], _address(copy_ptrs),
        8 if narrow else 32, first.data_ptr(), second.data_ptr(), scales[0].data_ptr() if narrow else None, scales[1].data_ptr() if narrow else None,
        steps.data_ptr(), lr, betas[0], betas[1], eps, weight_decay, gradient_scale, seed))
    # whoever has saved one of them for a backward pass learns that it is another now
    torch.autograd.graph.increment_version(params if copies is None else params + list(copies))


class ClauseReadout:
    """Softmax classifier on the clause outputs of a trained machine.

    Each clause has an embedding row; the rows of a graph's active clauses are added up, and labels are scored by their product with
    the sum.  ``fit``, ``score`` and ``predict`` take graphs as the machine's do.  The machine itself is not changed.

    ``tm``: a fitted machine (any class).  ``embedding_size``: columns of the two weight matrices.  They are held in 32 bits and
    multiplied in bfloat16; ``state_bits`` (32 or 8) are those of AdamW's states."""

    def __init__(self, tm, embedding_size=64, learning_rate=1e-2, weight_decay=0.01, state_bits=32, seed=0):
        if embedding_size < 1:
            raise ValueError("embedding_size %r" % (embedding_size,))
        if state_bits not in (8, 32):
            raise ValueError("state_bits %r: 8 or 32" % (state_bits,))
        self.tm = tm
        self.embedding_size = int(embedding_size)
        self.learning_rate = learning_rate
        self.weight_decay = weight_decay
        self.state_bits = state_bits
        self.seed = int(seed)
        self.number_of_outputs = None
        self.device = torch.device("cuda", tm.device)

    def _pieces(self, graphs):
        """The graphs, or as many of them at a time as have ``OUTPUTS`` clause outputs."""
        number, most = graphs.number_of_graphs, max(1, OUTPUTS // self.tm.number_of_clauses)
        if number == 0:
            raise ValueError("there are no graphs")
        for first in range(0, number, most):
            yield graphs if most >= number else graphs[first:min(first + most, number)]

    def active_clauses(self, graphs):
        """(ids int32, offsets int64) of the clauses that are active for each graph, on the device: bags for ``embed``."""
        clauses, counts = [], []
        for piece in self._pieces(graphs):
            outputs, _ = self.tm.transform(piece)
            clauses.append(np.nonzero(outputs)[1].astype(np.int32))
            counts.append(np.count_nonzero(outputs, axis=1))
        offsets = np.zeros(graphs.number_of_graphs + 1, dtype=np.int64)
        np.cumsum(np.concatenate(counts), out=offsets[1:])
        return torch.from_numpy(np.concatenate(clauses)).to(self.device), torch.from_numpy(offsets).to(self.device)

    def _init(self, outputs):
        self.number_of_outputs = outputs
        generator = torch.Generator(device=self.device).manual_seed(self.seed)
        clauses, columns = self.tm.number_of_clauses, self.embedding_size
        # sums of some tens of rows of unit length have logits of the order of one
        self.weights = [torch.randn(rows, columns, generator=generator, device=self.device) / columns ** 0.5 for rows in (clauses, outputs)]
        self.copies = [w.to(torch.bfloat16) for w in self.weights]
        self.state = adamw_state(self.weights, self.state_bits)

    def _scale(self):
        return 1.0 / self.embedding_size ** 0.5

    def fit(self, graphs, Y, epochs=10, batch_size=256, incremental=False):
        """``epochs`` ordered passes over the graphs in batches; mean loss of every pass, a list."""
        Y = np.asarray(Y)
        if Y.shape != (graphs.number_of_graphs,) or (Y.size and Y.min() < 0):
            raise ValueError("Y holds one label, zero or more, for each of %d graphs" % graphs.number_of_graphs)
        if batch_size < 1:
            raise ValueError("batch_size %r" % (batch_size,))
        again = self.number_of_outputs is None or not incremental
        if not again and Y.size and int(np.max(Y)) >= self.number_of_outputs:
            raise ValueError("label %d of a readout of %d labels" % (int(np.max(Y)), self.number_of_outputs))
        ids, offsets = self.active_clauses(graphs)
        if again:
            self._init(int(np.max(Y) + 1))
        ends = offsets.cpu().numpy()
        labels = torch.from_numpy(Y.astype(np.int64)).to(self.device)
        history = []
        softmax_failed(self.device.index)                            # of others before
        for _ in range(epochs):
            total = torch.zeros((), device=self.device)
            for first in range(0, len(Y), batch_size):
                last = min(len(Y), first + batch_size)
                bags = (offsets[first:last + 1] - offsets[first]).contiguous()
                total += self._step(ids[int(ends[first]):int(ends[last])], bags, labels[first:last]).sum()
            history.append(total / len(Y))
        history = [float(v) for v in history]
        self._complete()
        return history

    def _complete(self):
        if softmax_failed(self.device.index):
            raise RuntimeError("a wait inside a softmax kernel ran out: what it was to compute is missing")

    def gradients(self, ids, offsets, labels):
        """(losses, gradients of the two weight matrices for their mean) of a batch of bags."""
        scale = self._scale()
        table, outputs = self.copies
        features = embed(table, ids, offsets, scale=scale)
        losses, normalisers = softmax_loss(features, outputs, labels)
        mean = torch.full((1,), 1.0 / max(1, labels.numel()), device=self.device)
        features_gradient, outputs_gradient = softmax_loss_gradient(features, outputs, labels, normalisers, mean)
        return losses, [embed_gradient(features_gradient, ids, table.shape[0], offsets, scale=scale), outputs_gradient]

    def _step(self, ids, offsets, labels):
        losses, gradients = self.gradients(ids, offsets, labels)
        adamw_step(self.weights, gradients, self.state, self.learning_rate, weight_decay=self.weight_decay, copies=self.copies, seed=self.seed & 0xFFFFFFFF)
        return losses

    def score(self, graphs):
        """(labels int64, log probabilities float32) of the most probable label of every graph, numpy arrays."""
        if self.number_of_outputs is None:
            raise RuntimeError("the readout is not fitted")
        scored = []
        for piece in self._pieces(graphs):
            features = embed(self.copies[0], *self.active_clauses(piece), scale=self._scale())
            scored.append([t.cpu().numpy() for t in softmax_predict(features, self.copies[1])])
        labels, log_probabilities = (np.concatenate(parts) for parts in zip(*scored))
        if np.isnan(log_probabilities).any():
            self._complete()
        return labels, log_probabilities

    def predict(self, graphs):
        return self.score(graphs)[0]
