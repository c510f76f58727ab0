"""CPU suite: what the readout kernels' sources must not hold, and what their entry points refuse."""

import ctypes as C
import glob
import os
import re
from types import SimpleNamespace

import pytest

from graphtsetlinmachine_b200 import _lib, readout

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_kernels_that_begin_early_load_nothing_by_the_read_only_path():
    """Data loaded that way must not change while a kernel lives, and these kernels are set up while the one before them still writes."""
    sources = glob.glob(os.path.join(ROOT, "graphtsetlinmachine_b200", "csrc", "gtm_readout*"))
    assert len(sources) >= 7
    for path in sources:
        code = re.sub(r"//[^\n]*", "", open(path).read())
        assert not re.search(r"__ldg|__restrict__|ld\.global\.nc|ld\.global\.[a-z.]*nc", code), path
        # and every kernel waits for the one before it
        kernels = re.findall(r"__global__ void[^{;]*\)\s*\n\{(.*?)\n\}", code, flags=re.S)
        assert all("wait_for_previous();" in k for k in kernels), path


def _pointers(*addresses):
    return (C.c_void_p * len(addresses))(*addresses)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("change", [
    dict(params=(0x10000, 0x10000)), dict(params=(0x10000, 0x10000 + 299 * 4)), dict(params=(0x10000, 0x10000 - 699 * 4)), dict(copies=(0x10000, 0x60000)),
    dict(copies=(0x50000, 0x50000)), dict(gradients=(0x10000, 0x40000)), dict(gradients=(0x30000, 0x10000 + 1196)), dict(first=0x20000), dict(second=0x70000),
    dict(steps=0x70000), dict(steps=0x10000 + 1192), dict(first=0x50000 + 592),
])
def test_steps_over_memory_that_is_written_twice_are_refused(bits, change):
    """Addresses that nothing follows: two tensors of 300 and 700 floats, their copies and states, of which one begins inside another."""
    a = dict(params=(0x10000, 0x20000), gradients=(0x30000, 0x40000), copies=(0x50000, 0x60000), first=0x70000, second=0x80000, steps=0x90000)
    a.update(change)
    lib = _lib.load()
    assert lib.gtm_adamw_step(0, None, 2, (C.c_int64 * 2)(300, 700), 0, _pointers(*a["params"]), 0, _pointers(*a["gradients"]), 1, _pointers(*a["copies"]), bits, a["first"],
                              a["second"], 0xa0000, 0xb0000, a["steps"], 0.1, 0.9, 0.99, 1e-8, 0.0, 1.0, 0) == 1
    assert b"overlap" in lib.gtm_last_error()


def test_a_classifier_of_no_graphs_is_refused():
    none, head = SimpleNamespace(number_of_graphs=0), readout.ClauseReadout(SimpleNamespace(device=0, number_of_clauses=10))
    for incremental in (False, True):
        with pytest.raises(ValueError, match="no graphs"):
            head.fit(none, [], incremental=incremental)
    with pytest.raises(ValueError, match="no graphs"):
        head.active_clauses(none)
    head.number_of_outputs = 3                                   # as after a fit
    for call in (lambda: head.fit(none, [], incremental=True), lambda: head.score(none), lambda: head.predict(none)):
        with pytest.raises(ValueError, match="no graphs"):
            call()
