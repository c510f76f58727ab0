"""GPU suite: readout operators at their edges - an example unlike the others, one more example than a kernel takes, sums of thousands of
terms of one sign - and in calls that the usual sizes do not make.

Tolerances count roundings, as in test_gpu_readout."""

import math

import pytest
import torch

from graphtsetlinmachine_b200 import readout
from test_gpu_readout import TYPES, _library, generator, softmax_case  # noqa: F401  (_library: no wait ran out)

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
