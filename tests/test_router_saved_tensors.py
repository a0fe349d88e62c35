"""The router's gradients read what autograd hands back, at the address where it hands it back.

Saved tensors need not return at the address that they had: hooks unpack them elsewhere, and non-reentrant checkpointing
computes them again.  Here, without a GPU, the native calls are replaced by a recorder of the addresses they are given."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from asap_b200 import _native as N
from asap_b200 import router


class Recorder:
    """Stands in for the library: each call's structure and addresses, as they were at the time."""

    def __init__(self):
        self.calls = []

    def __call__(self, name, desc, *args):
        d = desc._obj
        self.calls.append((name, {f: getattr(d, f) for f, _ in d._fields_}, args))

    def last(self, name):
        return next((d, a) for n, d, a in reversed(self.calls) if n == name)


class Here:
    def __init__(self, index):
        pass

    def __enter__(self):
        return 0

    def __exit__(self, *exc):
        return False


@pytest.fixture
def native(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(router.N, "run", rec)
    monkeypatch.setattr(router, "_OnDevice", Here)
    return rec


def route(logits, k=2):
    """router.route's autograd function, past the checks that want a GPU."""
    return router._Route.apply(logits, (k, 1, None, 1, 1, 1, 1.0, None))


def balance(logits, ids, cu):
    return router._BalanceLoss.apply(logits, ids, 1, 1.0, cu, 1 if cu is None else cu.numel() - 1)


class Moved:
    """Saved-tensor hooks that hand back copies, and keep both."""

    def __init__(self, change=lambda t: t):
        self.kept, self.change = [], change

    def pack(self, t):
        return t.clone()

    def unpack(self, t):
        t = self.change(t.clone())
        self.kept.append(t)
        return t

    def hooks(self):
        return torch.autograd.graph.saved_tensors_hooks(self.pack, self.unpack)


def strided(t):
    """The same values, columns apart."""
    wide = t.new_zeros((*t.shape[:-1], 2 * t.shape[-1]))
    wide[..., ::2] = t
    return wide[..., ::2]


@pytest.mark.parametrize("change", [lambda t: t, strided], ids=["moved", "strided"])
def test_route_gradient_reads_the_unpacked_tensors(native, change):
    x, moved = torch.randn(4, 8, requires_grad=True), Moved(change)
    with moved.hooks():
        weights, ids = route(x)
    weights.sum().backward()
    desc, (ids_ptr, *_) = native.last("asap_route_backward")
    rows, choice = moved.kept
    if change is strided:  # read through contiguous copies of them, not at the forward's addresses
        assert desc["logits"] not in (x.data_ptr(), rows.data_ptr()) and ids_ptr not in (ids.data_ptr(), choice.data_ptr())
    else:
        assert (desc["logits"], ids_ptr) == (rows.data_ptr(), choice.data_ptr())
    assert desc["ld"] == 8


@pytest.mark.parametrize("seqs", [None, 2])
def test_balance_gradient_reads_the_unpacked_tensors(native, seqs):
    x, moved = torch.randn(4, 8, requires_grad=True), Moved()
    ids = torch.zeros(4, 2, dtype=torch.int32)
    cu = None if seqs is None else torch.tensor([0, 3, 4], dtype=torch.int32)
    with moved.hooks():
        loss, counts = balance(x, ids, cu)
    first, (ws0, nbytes0, *_) = native.last("asap_balance_loss")
    loss.backward()
    desc, (ws, nbytes, *_) = native.last("asap_balance_backward")
    rows, buf = moved.kept  # ids and offsets are not read again
    assert desc["logits"] == rows.data_ptr()
    lo, hi = buf.data_ptr(), buf.data_ptr() + 4 * buf.numel()
    assert lo <= desc["counts"] < desc["counts"] + 4 * counts.numel() == ws and ws + nbytes <= hi and nbytes == nbytes0
    # the same layout as the forward's
    assert ws - desc["counts"] == ws0 - first["counts"] and ws % 8 == 0


def test_gradients_under_checkpointing_read_the_recomputed_tensors(native):
    made = []

    def f(x):
        y = x * 2.0
        made.append(y)
        weights, ids = route(y)
        made.append(ids)
        loss, _ = balance(y, torch.zeros(4, 2, dtype=torch.int32), None)
        return weights.sum() + loss

    x = torch.randn(4, 8, requires_grad=True)
    checkpoint(f, x, use_reentrant=False).backward()
    first, _, again, ids = made
    desc, (ids_ptr, *_) = native.last("asap_route_backward")
    assert desc["logits"] == again.data_ptr() != first.data_ptr()
    assert ids_ptr == ids.data_ptr()
    desc, (ws, *_) = native.last("asap_balance_backward")
    assert desc["logits"] == again.data_ptr()
    again_desc, (again_ws, *_) = native.last("asap_balance_loss")  # the second forward's
    assert (desc["counts"], ws) == (again_desc["counts"], again_ws)


@pytest.mark.parametrize("change,which", [(lambda t: t.double() if t.is_floating_point() else t, "logits"),
                                          (lambda t: t[:-1], "shape"), (lambda t: t.to("meta"), "device")])
def test_gradients_refuse_what_comes_back_as_something_else(native, change, which):
    for op in (lambda x: route(x)[0].sum(), lambda x: balance(x, torch.zeros(4, 2, dtype=torch.int32), None)[0]):
        moved = Moved(change)
        with moved.hooks():
            out = op(torch.randn(4, 8, requires_grad=True))
        with pytest.raises(RuntimeError, match="saved for the gradient came back"):
            out.backward()


def test_two_gradients_of_one_forward(native):
    x = torch.randn(4, 8, requires_grad=True)
    weights, ids = route(x)
    for _ in range(2):
        weights.sum().backward(retain_graph=True)
        desc, (ids_ptr, *_) = native.last("asap_route_backward")
        assert (desc["logits"], ids_ptr) == (x.data_ptr(), ids.data_ptr())
    assert N.lib().asap_balance_ws_bytes(4, 1) > 0
