"""What the router and the balance loss promise beside their values: gradients of saved tensors that come back elsewhere,
special rows, tangents."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from asap_b200.router import balance_loss, route
from test_gpu_router import check_balance, check_route, make_logits

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


# ---------------------------------------------------------------------------------------------------- special rows
def weights_and_gradient(logits, scoring, renorm, biased, **kw):
    T, E = logits.shape
    x = logits.clone().requires_grad_(True)
    bias = 0.01 * torch.arange(E, device=DEV, dtype=torch.float32) if biased else None
    top = route(x, 6, scoring=scoring, renormalize=renorm, bias=bias, **kw)
    grad = torch.randn(T, 6, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T))
    return top, torch.autograd.grad(top.topk_weights, x, grad)[0]


@pytest.mark.parametrize("scoring,renorm,biased", FORMS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min])
@pytest.mark.parametrize("E", [64, 72, 1000])
def test_route_gradient_of_padding_rows(cuda_ok, E, value, scoring, renorm, biased):
    """Rows behind the valid tokens have gradient 0 whatever they hold, and so has a row with no expert left."""
    n = 30
    clean = make_logits(40, E, torch.float32, E)
    clean[4] = float("-inf")
    logits = clean.clone()
    logits[n:, 5], logits[33], logits[35, 40:] = value, value, value
    top, dl = weights_and_gradient(logits, scoring, renorm, biased,
                                   num_tokens=torch.tensor([n], dtype=torch.int32, device=DEV))
    assert (top.topk_ids[n:] == -1).all() and (top.topk_weights[n:] == 0).all()
    assert (dl[n:] == 0).all() and (dl[4] == 0).all()
    assert dl[:n].isfinite().all() and (dl[:4] != 0).any(1).all()


@pytest.mark.parametrize("scoring,renorm,biased", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E", [16, 72, 1000])
def test_route_gradient_of_a_nan_row_is_nan(cuda_ok, E, dtype, scoring, renorm, biased):
    """As its weights are, in every form; a row of NaN alone chose nothing and has gradient 0."""
    clean = make_logits(41, E, dtype, E)
    want_top, want = weights_and_gradient(clean, scoring, renorm, biased)
    logits = clean.clone()
    logits[7, E - 1] = logits[20, 0] = float("nan")
    logits[12] = float("nan")
    top, dl = weights_and_gradient(logits, scoring, renorm, biased)
    assert top.topk_weights[[7, 12, 20]].isnan().all() and (top.topk_ids[12] == -1).all()
    assert dl[[7, 20]].isnan().all() and (dl[12] == 0).all()
    rest = [r for r in range(41) if r not in (7, 12, 20)]
    assert torch.equal(dl[rest], want[rest]) and torch.equal(top.topk_ids[rest], want_top.topk_ids[rest])


# ------------------------------------------------------------------------------------------------------- the choice
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,big", [(200, 64, 16.0), (1000, 256, 16.0), (1000, 256, 1024.0), (300, 512, 1024.0),
                                     (300, 256, 2.0 ** 20), (100, 256, 3.0e38)])
def test_route_groups_whose_two_best_cancel(cuda_ok, T, E, big, scoring):
    """One expert of a group far up and the rest far down: the group's sum is small, the rounding of its addends is not."""
    logits = make_logits(T, E, torch.float32, E)
    bias = torch.full((E,), -big, device=DEV)
    bias[::E // 8] = big
    for k in (4, 7):
        check_route(logits, k, scoring=scoring, bias=bias, num_groups=8, top_groups=4)
    bias[::E // 4] = 0.5  # every other group without such an expert: sums of two sizes
    bias[1::E // 4] = 0.5
    check_route(logits, 6, scoring=scoring, bias=bias, num_groups=8, top_groups=4)


@pytest.mark.parametrize("low", [-1e4, -1e9, torch.finfo(torch.float32).min, float("-inf")])
def test_route_groups_of_experts_biased_away(cuda_ok, low):
    """A rank's experts switched off by a very negative bias: whole groups, and all but one of a group."""
    E = 256
    logits = make_logits(200, E, torch.float32, 9)
    bias = 0.1 * torch.randn(E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    bias[32:96] = low
    bias[129:160] = low
    for scoring in ("sigmoid", "softmax"):
        check_route(logits, 8, scoring=scoring, bias=bias, num_groups=8, top_groups=4)


# ----------------------------------------------------------------------------------------------------- balance loss
@pytest.mark.parametrize("T,E,k", [(511, 16, 2), (512, 16, 2), (256, 64, 6), (257, 64, 6), (128, 128, 6), (129, 128, 6),
                                   (64, 256, 8), (32, 512, 8), (33, 512, 8), (16, 1000, 8), (17, 1000, 8)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_balance_around_the_single_launch(cuda_ok, T, E, k, scoring):
    """The last sizes of the single launch and the first of the three."""
    logits = make_logits(T, E, torch.float32, T + E)
    ids = route(logits, k, scoring=scoring).topk_ids
    check_balance(logits, ids, scoring)
    check_balance(logits, ids, scoring, cu=torch.tensor([0, 5, 5, T - 3], dtype=torch.int32, device=DEV))
