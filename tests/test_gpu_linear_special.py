"""What the FP8 linear and shared expert promise beside their values: special rows, streams, reloading, refusals."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from asap_b200 import linear as lin
from asap_b200.linear import Fp8Linear, Fp8SharedExpert
from asap_b200.router import balance_loss, route
from test_gpu_linear import hidden, weight
from test_gpu_moe_layer import layer  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m", [6, 200, 9000])  # the few-rows kernels (16 and 64 columns wide), the 128 x 256 tiles
@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
@pytest.mark.parametrize("limit", [0.0, 0.75])
def test_shared_expert_special_rows_with_and_without_a_limit(cuda_ok, m, scales, limit):
    gen = torch.Generator(device=DEV).manual_seed(m)
    w13, s13 = weight(gen, 512, 384, scales)
    w2, s2 = weight(gen, 384, 256, scales)
    layer = Fp8SharedExpert(w13, s13, w2, s2, swiglu_limit=limit)
    x = hidden(gen, m, 384, torch.bfloat16)
    clean = layer(x)
    assert clean.isfinite().all()
    x[0, 1], x[1, 2], x[2, 380], x[3] = float("nan"), float("inf"), float("-inf"), 0.0
    y = layer(x)
    lin.check()
    assert y[:3].isnan().all() and (y[3] == 0).all()
    assert torch.equal(y[4:], clean[4:])


def test_layer_after_its_shared_expert_refused(layer):
    """The message that was out is taken back: the layer's next calls, on every slot, are as before."""
    lb, moe_layer, gate, _ = layer
    x = torch.randn(40, moe_layer.hidden_size, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)).bfloat16()
    with torch.no_grad():
        topk = route(gate(x)[:, :16], 4)
        want = moe_layer(x, topk)
    for _ in range(3):
        with pytest.raises(RuntimeError, match="no gradient"):
            moe_layer(x.clone().requires_grad_(True), topk)
    with torch.no_grad():
        for _ in range(3):
            assert torch.equal(moe_layer(x, topk), want)
    torch.cuda.synchronize()
    lb.check()


def test_forward_mode_tangents_are_refused(cuda_ok):
    gen = torch.Generator(device=DEV).manual_seed(1)
    linear = Fp8Linear(*weight(gen, 128, 256, "fp32"))
    shared = Fp8SharedExpert(*weight(gen, 256, 256, "fp32"), *weight(gen, 256, 128, "fp32"))
    x, t = hidden(gen, 4, 256, torch.bfloat16), hidden(gen, 4, 256, torch.bfloat16)
    l, ids = torch.randn(4, 8, device=DEV, generator=gen), torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    with fwAD.dual_level():
        dual, dual_l = fwAD.make_dual(x, t), fwAD.make_dual(l, torch.ones_like(l))
        for call in (lambda: linear(dual), lambda: shared(dual), lambda: route(dual_l, 2), lambda: balance_loss(dual_l, ids),
                     lambda: linear(dual[1:]), lambda: route(dual_l.clone().requires_grad_(True), 2)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(linear(dual.detach()), linear(x)) and torch.equal(linear(x), linear(x))
        assert torch.equal(route(dual_l.detach(), 2).topk_ids, route(l, 2).topk_ids)


@pytest.mark.parametrize("m", [3, 2000])
@pytest.mark.parametrize("made", ["e8m0", "strided", "from_float"])
def test_layer_made_on_a_busy_stream_serves_another(cuda_ok, made, m):
    """What a layer lays out of its scales is there when it has been made, whatever stream calls it first."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    dense = 0.02 * torch.randn(512, 1024, device=DEV, generator=gen)
    w, s = weight(gen, 512, 1024, "fp32" if made == "strided" else "e8m0")
    wide = s.float().repeat_interleave(2, 1)  # the scales as every other column

    def make():
        if made == "from_float":
            return Fp8Linear.from_float(dense)
        return Fp8Linear(w, wide[:, ::2] if made == "strided" else s)

    x = hidden(gen, m, 1024, torch.bfloat16)
    want = make()(x)
    torch.cuda.synchronize()
    for n in (8 * 4 * 512, 4 * 8 * 4, 512 * 1024):  # what the layer's own tensors will be made of
        torch.full((n,), 90, dtype=torch.uint8, device=DEV)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)  # some 60 ms of the current stream
    layer = make()
    with torch.cuda.stream(other):
        y = layer(x)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [3, 40, 2500])
@pytest.mark.parametrize("scales", ["fp32", "strided", "e8m0"])
def test_reload_after_new_values_in_place(cuda_ok, scales, m):
    gen = torch.Generator(device=DEV).manual_seed(m)
    kind = "e8m0" if scales == "e8m0" else "fp32"
    old, new = [[weight(gen, 512, 256, kind), weight(gen, 256, 256, kind)] for _ in range(2)]
    if scales == "strided":
        old = [(w, s.t().contiguous().t().requires_grad_(True)) for w, s in old]  # as a parameter may
    (w13, s13), (w2, s2) = old
    layer, shared = Fp8Linear(w13, s13), Fp8SharedExpert(w13, s13, w2, s2)
    x = hidden(gen, m, 256, torch.bfloat16)
    first = layer(x), shared(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer(x), shared(x)
    with torch.no_grad():
        for (w, s), (v, t) in zip(old, new):
            w.view(torch.uint8).copy_(v.view(torch.uint8))
            s.copy_(t)
    layer.reload()
    shared.reload()
    want = Fp8Linear(*new[0])(x), Fp8SharedExpert(*new[0], *new[1])(x)
    graph.replay()
    for a, b, c, d in zip((layer(x), shared(x)), want, captured, first):
        assert torch.equal(a, b) and torch.equal(c, b) and not torch.equal(a, d)
    assert not layer._w.scale.requires_grad and layer._w.scale.grad_fn is None  # no history grows with every reload
    lin.check()
