"""What the router and the balance loss promise beside their values: gradients of saved tensors that come back elsewhere,
special rows, tangents."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from asap_b200.router import balance_loss, route
from test_gpu_router import make_logits

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMS = [("softmax", True, False), ("softmax", False, False), ("softmax", True, True), ("sigmoid", True, True),
         ("sigmoid", False, False)]  # scoring, renormalised, biased


# ----------------------------------------------------------------------------- saved tensors that come back elsewhere
def step(logits, cu, bias):
    """One layer's worth of what has a gradient, on logits that only this call holds."""
    y = logits * 2.0
    top = route(y, 6, scoring="sigmoid", bias=bias, num_groups=8, top_groups=4)
    loss, _ = balance_loss(y, top.topk_ids, scoring="sigmoid", coef=0.3, cu_seqlens=cu)
    return (top.topk_weights.square().sum(1) * torch.arange(logits.shape[0], device=DEV)).sum() + 100.0 * loss


def gradient(logits, how, cu, bias):
    x = logits.clone().requires_grad_(True)
    if how == "checkpoint":
        out = checkpoint(step, x, cu, bias, use_reentrant=False)
    elif how == "cpu":
        with torch.autograd.graph.save_on_cpu(pin_memory=False):
            out = step(x, cu, bias)
    elif how == "hooks":
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
            out = step(x, cu, bias)
    else:
        out = step(x, cu, bias)
    # what the forward let go of is handed on
    junk = [torch.full((logits.numel(),), 3.0e4, device=DEV, dtype=logits.dtype) for _ in range(8)]
    junk += [torch.full((n,), -1, device=DEV, dtype=torch.int32) for n in (logits.shape[0] * 6, 4096, 64) for _ in range(4)]
    (grad,) = torch.autograd.grad(out, x)
    del junk
    return grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["checkpoint", "cpu", "hooks"])
@pytest.mark.parametrize("T", [8, 300, 1500])  # the balance loss in one launch and in three
def test_gradients_of_saved_tensors_that_come_back_elsewhere(cuda_ok, T, how, dtype):
    logits = make_logits(T, 64, dtype, T)
    cu = torch.tensor([0, T // 3, T - 2], dtype=torch.int32, device=DEV)
    bias = 0.1 * torch.randn(64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T))
    want = gradient(logits, None, cu, bias)
    assert want.isfinite().all() and (want != 0).any()
    for _ in range(2):
        assert torch.equal(gradient(logits, how, cu, bias), want)
