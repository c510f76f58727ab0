"""CPU suite: what the readout operators refuse before anything reaches a device, through Python and through the C ABI."""

import ctypes as C

import pytest
import torch

from graphtsetlinmachine_b200 import _lib, readout


def test_tensors_on_the_host_are_refused():
    x, ids = torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: readout.embed(x, ids), lambda: readout.embed_gradient(x, ids, 5), lambda: readout.softmax_loss(x, x, ids),
                 lambda: readout.softmax_predict(x, x), lambda: readout.adamw_state([x]), lambda: readout.adamw_step([x], [x], {}, 0.1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        readout.embed(x.numpy(), ids)
    with pytest.raises(ValueError):
        readout.adamw_step([], [], {}, 0.1)


POINTER = C.c_void_p(4096)      # never followed: the calls below are refused first


def _embed(lib, **kw):
    a = dict(device=0, stream=None, type=0, table=POINTER, rows=4, columns=8, stride=8, ids=POINTER, wide=1, n=3, offsets=None, wide_offsets=0, bags=0, scale=1.0,
             out=POINTER, workspace=None, bytes=0)
    a.update(kw)
    return lib.gtm_embed(*a.values())


def _embed_gradient(lib, **kw):
    a = dict(device=0, stream=None, type=0, gradient=POINTER, columns=8, stride=8, ids=POINTER, wide=1, n=3, offsets=None, wide_offsets=0, bags=0, scale=1.0,
             out=POINTER, rows=4, workspace=POINTER, bytes=1 << 40)
    a.update(kw)
    return lib.gtm_embed_gradient(*a.values())


def _loss(lib, **kw):
    a = dict(device=0, stream=None, type=1, x=POINTER, n=3, x_stride=8, w=POINTER, v=50, w_stride=8, columns=8, labels=POINTER, wide=1, ignored=-1, scale=1.0,
             losses=POINTER, normalisers=POINTER, workspace=POINTER, bytes=1 << 40)
    a.update(kw)
    return lib.gtm_softmax_loss(*a.values())


def _predict(lib, **kw):
    a = dict(device=0, stream=None, type=1, x=POINTER, n=3, x_stride=8, w=POINTER, v=50, w_stride=8, columns=8, scale=1.0, labels=POINTER, out=POINTER,
             workspace=POINTER, bytes=1 << 40)
    a.update(kw)
    return lib.gtm_softmax_predict(*a.values())


@pytest.mark.parametrize("call,bad", [
    (_embed, dict(type=3)), (_embed, dict(rows=0)), (_embed, dict(columns=0)), (_embed, dict(n=-1)), (_embed, dict(n=1 << 31)), (_embed, dict(table=None)),
    (_embed, dict(ids=None)), (_embed, dict(out=None)), (_embed, dict(stride=-8)), (_embed, dict(out=C.c_void_p(4100))), (_embed, dict(offsets=POINTER, bags=-1)),
    (_embed, dict(offsets=POINTER, bags=2, n=1000)), (_embed_gradient, dict(rows=0)), (_embed_gradient, dict(rows=1 << 31)), (_embed_gradient, dict(bytes=16)),
    (_embed_gradient, dict(workspace=None)), (_embed_gradient, dict(workspace=C.c_void_p(4097))), (_embed_gradient, dict(gradient=None)), (_embed_gradient, dict(out=None)),
    (_loss, dict(type=-1)), (_loss, dict(n=-1)), (_loss, dict(n=1 << 23)), (_loss, dict(v=0)), (_loss, dict(v=1 << 29)), (_loss, dict(columns=0)), (_loss, dict(scale=0.0)),
    (_loss, dict(scale=-1.0)), (_loss, dict(scale=float("nan"))), (_loss, dict(scale=float("inf"))), (_loss, dict(x=None)), (_loss, dict(w=None)), (_loss, dict(labels=None)),
    (_loss, dict(losses=None)), (_loss, dict(workspace=C.c_void_p(4097))), (_loss, dict(bytes=8)), (_loss, dict(x_stride=-8)), (_loss, dict(x=C.c_void_p(4097))), (_embed, dict(table=C.c_void_p(4098))), (_embed, dict(ids=C.c_void_p(4100))), (_predict, dict(labels=None)),
    (_predict, dict(bytes=8)), (_predict, dict(scale=0.0)),
])
def test_bad_arguments_are_refused(call, bad):
    lib = _lib.load()
    assert call(lib, **bad) == 1
    assert lib.gtm_last_error().startswith(b"gtm_")


def _adamw(lib, **kw):
    one = (C.c_void_p * 1)(4096)
    a = dict(device=0, stream=None, n=1, counts=(C.c_int64 * 1)(5), type=0, params=one, gradient_type=0, gradients=one, copy_type=1, copies=None, bits=32, first=POINTER,
             second=POINTER, first_scales=None, second_scales=None, steps=POINTER, lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, decay=0.0, scale=1.0, seed=0)
    a.update(kw)
    return lib.gtm_adamw_step(*a.values())


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(counts=None), dict(params=None), dict(counts=(C.c_int64 * 1)(-5)), dict(type=3), dict(gradient_type=9), dict(copies=(C.c_void_p * 1)(4096), copy_type=0),
    dict(bits=16), dict(bits=8), dict(first=None), dict(first=C.c_void_p(4100)), dict(steps=None), dict(steps=C.c_void_p(4100)), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0),
    dict(lr=-0.1), dict(lr=float("nan")), dict(decay=-1.0), dict(params=(C.c_void_p * 1)(4097)), dict(params=(C.c_void_p * 1)(0)),
])
def test_bad_steps_are_refused(bad):
    lib = _lib.load()
    assert _adamw(lib, **bad) == 1
    assert lib.gtm_last_error().startswith(b"gtm_adamw_step")


def test_workspaces_grow_with_what_they_hold():
    lib, out = _lib.load(), C.c_uint64()

    def size(call, *args):
        assert call(*args, C.byref(out)) == 0
        return out.value

    assert size(lib.gtm_embed_workspace, 1000, 64, 0) == 0 and size(lib.gtm_embed_workspace, 128, 64, 1) == 0
    assert size(lib.gtm_embed_workspace, 1000, 64, 1) >= 2 * 8 * 64 * 4
    assert size(lib.gtm_embed_gradient_workspace, 1000, 50, 64) >= 2 * 8000 + 51 * 4 + 2 * 8 * 64 * 4
    # of 8192 x 65536 logits in 16 bits (1 GB) an eighth at most is held
    forward = size(lib.gtm_softmax_workspace, 1, POINTER, 8192, 1024, POINTER, 65536, 1024, 1024, 0)
    backward = size(lib.gtm_softmax_workspace, 1, POINTER, 8192, 1024, POINTER, 65536, 1024, 1024, 1)
    assert forward < 8192 * 65536 * 2 // 8 and backward < 8192 * 65536 * 2 // 4
    assert size(lib.gtm_softmax_workspace, 1, POINTER, 0, 8, POINTER, 5, 8, 8, 0) == 0
    assert lib.gtm_softmax_workspace(1, POINTER, 3, 8, POINTER, 5, 8, 8, 0, None) == 1


def test_softmax_workspaces_are_those_of_a_call():
    lib, out = _lib.load(), C.c_uint64()
    sizes = []
    for what in (0, 1, 2):
        assert lib.gtm_softmax_workspace(0, POINTER, 1, 1024, POINTER, 65536, 1024, 1024, what, C.byref(out)) == 0
        sizes.append(out.value)
    # in 32 bits a prediction for one example reads the weights as they are; loss and gradient have them in three parts of 16 bits
    assert sizes[2] < 65536 * 1024 * 4 < 65536 * 1024 * 6 <= min(sizes[:2])
    for what in (-1, 3):
        assert lib.gtm_softmax_workspace(0, POINTER, 1, 1024, POINTER, 65536, 1024, 1024, what, C.byref(out)) == 1
