"""Router, balance loss and counts against the definition in 64 bits on the CPU.

Ids have to be equal: the choice ranks as unrounded scores rank, ties to the lowest expert.  Tolerances of computed
values, in units of 2^-24 (half a unit in the last place of fp32): a score takes an exponential (2 ulp, 4 units), a sum
of at most 32 terms per lane and 5 across the warp (37), and two divisions and products (4); a weight adds the sum of the
selected (5) and its division and scale (3): 64 units of the value.  A gradient adds a sum of products (10) and
differences whose terms are named where they are used; it is rounded to its type, eps / 2."""

import numpy as np
import pytest
import torch

from asap_b200.router import balance_loss, expert_counts, route

pytestmark = pytest.mark.gpu
U = 64 * 2.0 ** -24
DEV = "cuda"
NINF = float("-inf")


# ------------------------------------------------------------------------------------------------- the definition
def scores64(logits, scoring):
    l = logits.double().cpu()
    if scoring == "sigmoid":
        return torch.sigmoid(l)
    top = l.masked_fill(l.isnan(), NINF).amax(1, keepdim=True)
    e = torch.where(torch.isneginf(l), torch.zeros_like(l), torch.exp(l - torch.where(torch.isneginf(top), 0.0, top)))
    return e / e.sum(1, keepdim=True)


def choose64(logits, k, scoring, bias=None, groups=1, top_groups=1, valid=None):
    """-> ids int32 [T, k] by plain loops."""
    s = scores64(logits, scoring).numpy()
    l = logits.double().cpu().numpy()
    rank = l if bias is None else s + bias.double().cpu().numpy()
    T, E = l.shape
    ids = np.full((T, k), -1, np.int32)
    size = E // groups
    for t in range(T if valid is None else valid):
        open_ = [e for e in range(E) if l[t, e] > -np.inf and rank[t, e] > -np.inf]
        if groups > 1 and top_groups < groups:
            value = {}
            for g in range(groups):
                best = sorted((rank[t, e] for e in open_ if e // size == g), reverse=True)
                if best:
                    value[g] = best[0] if bias is None else sum(best[:2])
            kept = sorted(value, key=lambda g: (-value[g], g))[:top_groups]
            open_ = [e for e in open_ if e // size in kept]
        best = sorted(open_, key=lambda e: (-rank[t, e], e))[:k]
        ids[t, :len(best)] = best
    return ids


def weights64(logits, ids, scoring, renorm, scale):
    s = scores64(logits, scoring)
    i = torch.as_tensor(ids).long()
    sel = s.gather(1, i.clamp_min(0)).masked_fill(i < 0, 0.0)
    return scale * (sel / (sel.sum(1, keepdim=True) + 1e-20) if renorm else sel)


def make_logits(T, E, dtype, seed, masked=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    l = 2.0 * torch.randn(T, E, device=DEV, generator=gen)
    if masked:
        l[:, torch.randperm(E, device=DEV, generator=gen)[:masked]] = NINF
        l[::5] = NINF
    return l.to(dtype)


def check_route(logits, k, **kw):
    top = route(logits, k, **kw)
    a = dict(scoring=kw.get("scoring", "softmax"), bias=kw.get("bias"), groups=kw.get("num_groups", 1),
             top_groups=kw.get("top_groups", 1))
    valid = None if kw.get("num_tokens") is None else max(0, min(int(kw["num_tokens"]), logits.shape[0]))
    ids = choose64(logits, k, valid=valid, **a)
    np.testing.assert_array_equal(top.topk_ids.cpu().numpy(), ids)
    w = weights64(logits, ids, a["scoring"], kw.get("renormalize", True), kw.get("routed_scaling_factor", 1.0))
    got = top.topk_weights.double().cpu()
    assert ((got - w).abs() <= U * w.abs() + 1e-44).all(), ((got - w).abs() / w.abs().clamp_min(1e-300)).max()
    return top


# ---------------------------------------------------------------------------------------------------------- route
SHAPES = [(1, 1, 1, 1, 1), (3, 2, 2, 1, 1), (7, 8, 3, 8, 4), (33, 16, 2, 1, 1), (40, 16, 16, 4, 2), (64, 62, 3, 1, 1),
          (100, 64, 6, 8, 3), (31, 72, 5, 8, 4), (20, 96, 4, 3, 2), (50, 130, 8, 1, 1), (257, 256, 8, 8, 4),
          (30, 209, 32, 1, 1), (25, 512, 8, 16, 4), (9, 1000, 9, 8, 5), (9, 1024, 32, 32, 7), (600, 256, 8, 1, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,kept", SHAPES)
def test_route_against_the_definition(cuda_ok, T, E, k, groups, kept, scoring, dtype):
    bias = 0.1 * torch.randn(E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(E))
    for i, (b, renorm, masked) in enumerate([(None, True, 0), (bias, True, 0), (bias, False, E // 3), (None, False, E // 3)]):
        logits = make_logits(T, E, dtype, 31 * T + E + i, masked)
        check_route(logits, k, scoring=scoring, bias=b, num_groups=groups, top_groups=kept, renormalize=renorm,
                    routed_scaling_factor=2.5)


@pytest.mark.parametrize("n", [0, 1, 17, 40, 99, -3])
def test_route_padding_rows(cuda_ok, n):
    logits = make_logits(40, 64, torch.float32, n + 5)
    top = check_route(logits, 6, scoring="sigmoid", num_tokens=torch.tensor([n], dtype=torch.int32, device=DEV))
    lo = max(0, min(n, 40))
    assert (top.topk_ids[lo:] == -1).all() and (top.topk_weights[lo:] == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(64, 8), (256, 8), (72, 8), (16, 1), (512, 1)])
def test_route_ties_and_near_ties(cuda_ok, E, groups, scoring):
    """Equal logits with and without a bias; pairs whose score + bias agree to the last bits of fp32; all equal."""
    T, k = 200, 5
    kept = max(1, groups // 2)
    gen = torch.Generator(device=DEV).manual_seed(E)
    coarse = torch.randint(-3, 4, (T, E), device=DEV, generator=gen).float()
    zero = torch.zeros(E, device=DEV)
    bias = 0.05 * torch.randn(E, device=DEV, generator=gen)
    for l in (coarse, coarse.bfloat16(), torch.zeros(T, E, device=DEV), coarse * 0.0 - 0.0):
        for b in (None, zero, bias):
            check_route(l, k, scoring=scoring, bias=b, num_groups=groups, top_groups=kept)
    # per token, partners whose logit is solved for the same score + bias, then rounded to fp32
    l = 0.5 * torch.randn(T, E, device=DEV, generator=gen, dtype=torch.float64)
    if scoring == "sigmoid":
        for _ in range(E // 2):
            i, j = torch.randint(0, E, (2, T), device=DEV, generator=gen)
            r = torch.arange(T, device=DEV)
            want = (torch.sigmoid(l[r, i]) + bias[i].double() - bias[j].double()).clamp(1e-3, 1 - 1e-3)
            l[r, j] = torch.log(want / (1 - want))
    else:
        l[:, 1::2] = l[:, ::2] * (1 + 1e-9)
    check_route(l.float(), k, scoring=scoring, bias=bias, num_groups=groups, top_groups=kept)
    check_route(l.float(), k, scoring=scoring, num_groups=groups, top_groups=kept)
    step = torch.nextafter(torch.ones(1, device=DEV), torch.full((1,), 2.0, device=DEV))
    l = torch.where(torch.rand(T, E, device=DEV, generator=gen) < 0.5, step, torch.ones(1, device=DEV))
    check_route(l, k, scoring=scoring, num_groups=groups, top_groups=kept)


def test_route_special_values(cuda_ok):
    E, k = 64, 6
    low = torch.finfo(torch.float32).min
    l = make_logits(12, E, torch.float32, 3)
    l[0] = NINF                  # nothing left: ids -1, weights 0
    l[1, 4:] = NINF              # fewer than k left
    l[2] = low                   # the type's lowest value is not a mask
    l[3, 10:] = low
    l[4] = 0.0
    l[4, ::2] = -0.0             # +0 and -0 tie
    for scoring in ("softmax", "sigmoid"):
        top = check_route(l, k, scoring=scoring)
        assert (top.topk_ids[0] == -1).all() and (top.topk_weights[0] == 0).all()
        assert (top.topk_ids[1, 4:] == -1).all() and (top.topk_ids[1, :4] >= 0).all()
        assert (top.topk_ids[2].cpu() == torch.arange(k)).all() and (top.topk_ids[4].cpu() == torch.arange(k)).all()
    # a NaN logit is not chosen and shows in its row's weights, no other row's
    n = make_logits(6, E, torch.float32, 4)
    clean = route(n, k, scoring="sigmoid")
    n[2, 7] = float("nan")
    n[3] = float("nan")
    for bias in (None, torch.zeros(E, device=DEV)):
        top = route(n, k, scoring="sigmoid", bias=bias)
        assert top.topk_weights[2:4].isnan().all() and (top.topk_ids[3] == -1).all()
        assert (top.topk_ids[2] != 7).all() and (top.topk_ids[2] >= 0).all()
        for r in (0, 1, 4, 5):
            assert torch.equal(top.topk_ids[r], clean.topk_ids[r])
    # a bias of -inf or NaN switches an expert off, +inf puts it first
    b = torch.zeros(E, device=DEV)
    b[5], b[6], b[40], b[9] = NINF, float("nan"), float("inf"), float("inf")
    top = route(make_logits(50, E, torch.float32, 5), k, scoring="sigmoid", bias=b)
    assert not ((top.topk_ids == 5) | (top.topk_ids == 6)).any()
    assert (top.topk_ids[:, 0] == 9).all() and (top.topk_ids[:, 1] == 40).all()


def test_route_strides_streams_and_graph(cuda_ok):
    wide = make_logits(90, 200, torch.bfloat16, 8)
    for l in (wide[:, :64], wide[:, 3:67], wide[:, :128:2], wide[::2, 8:72], wide[:64, :90].t()[:, :64]):
        check_route(l, 6, scoring="sigmoid")
    l = make_logits(300, 256, torch.float32, 9)
    bias = 0.1 * torch.randn(256, device=DEV)
    n = torch.tensor([300], dtype=torch.int32, device=DEV)
    kw = dict(scoring="sigmoid", bias=bias, num_groups=8, top_groups=4, num_tokens=n)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        side = route(l, 8, **kw)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        top = route(l, 8, **kw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(side.topk_ids, top.topk_ids) and torch.equal(side.topk_weights, top.topk_weights)
    l.copy_(make_logits(300, 256, torch.float32, 10))
    n.fill_(123)
    g.replay()
    torch.cuda.synchronize()
    want = route(l, 8, **kw)
    assert torch.equal(top.topk_ids, want.topk_ids) and torch.equal(top.topk_weights, want.topk_weights)
    assert route(l[:0], 8).topk_ids.shape == (0, 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring,renorm,biased", [("softmax", True, False), ("softmax", False, False),
                                                   ("softmax", True, True), ("sigmoid", True, True),
                                                   ("sigmoid", False, False)])
@pytest.mark.parametrize("T,E,k", [(1, 8, 1), (5, 16, 16), (37, 64, 6), (20, 209, 8), (70, 256, 8), (6, 1024, 32)])
def test_route_gradient(cuda_ok, T, E, k, scoring, renorm, biased, dtype):
    gen = torch.Generator(device=DEV).manual_seed(T + E)
    bias = 0.1 * torch.randn(E, device=DEV, generator=gen) if biased else None
    logits = make_logits(T, E, dtype, T * E, masked=E // 4 if k <= E // 2 else 0).requires_grad_(True)
    top = route(logits, k, scoring=scoring, bias=bias, renormalize=renorm, routed_scaling_factor=2.5)
    grad = torch.randn(T, k, device=DEV, generator=gen)
    (dl,) = torch.autograd.grad(top.topk_weights, logits, grad)
    assert dl.dtype == dtype and not top.topk_ids.requires_grad
    ids = top.topk_ids.long().cpu()
    x = logits.detach().double().cpu()
    dead = torch.isneginf(x)
    x = x.masked_fill(dead, -1e4).requires_grad_(True)  # exp underflows to 0, and so does its slope
    s = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, 1)
    s = s * ~dead
    sel = s.gather(1, ids.clamp_min(0)).masked_fill(ids < 0, 0.0)
    n = sel.sum(1, keepdim=True) + 1e-20 if renorm else torch.ones(T, 1, dtype=torch.float64)
    w = 2.5 * sel / n
    g64 = grad.double().cpu()
    (want,) = torch.autograd.grad(w, x, g64)
    want = want.masked_fill(dead, 0.0)
    # dl = s_e (ds_e - sum ds s), ds = c / N (g - sum g s / N): the terms before they cancel
    ds = (2.5 / n * (g64.abs() + ((g64 * sel).abs().sum(1, keepdim=True) / n if renorm else 0))).masked_fill(ids < 0, 0.0)
    mag = torch.zeros_like(x).scatter_add(1, ids.clamp_min(0), ds).detach()
    mag = s.detach() * (mag + ((ds * sel).sum(1, keepdim=True).detach() if scoring == "softmax" else 0))
    tol = 2 * U * mag + torch.finfo(dtype).eps / 2 * want.abs() + 1e-38
    diff = (dl.double().cpu() - want).abs()
    assert (diff <= tol).all(), (diff / tol).max()
    with pytest.raises(RuntimeError, match="differentiated again"):
        (d2,) = torch.autograd.grad(route(logits, k, scoring=scoring).topk_weights, logits,
                                    grad.requires_grad_(True), create_graph=True)


def test_route_gradient_against_differences(cuda_ok):
    """The kernel's own weights at shifted logits: fp32 leaves (w(x + h) - w(x - h)) / 2h good to about 1e-4."""
    logits = make_logits(3, 16, torch.float32, 2)
    grad = torch.randn(3, 4, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    for kw in (dict(scoring="softmax"), dict(scoring="sigmoid"), dict(scoring="softmax", renormalize=False)):
        x = logits.clone().requires_grad_(True)
        top = route(x, 4, **kw)
        (dl,) = torch.autograd.grad(top.topk_weights, x, grad)
        h = 2.0 ** -8
        for t in range(3):
            for e in range(16):
                d = []
                for sign in (1, -1):
                    y = logits.clone()
                    y[t, e] += sign * h
                    moved = route(y, 4, **kw)
                    # the same experts, in whatever order
                    order = [(moved.topk_ids[t] == i).nonzero() for i in top.topk_ids[t]]
                    if any(o.numel() == 0 for o in order):
                        break
                    d.append((moved.topk_weights[t, torch.cat(order).flatten()].double() * grad[t].double()).sum())
                if len(d) == 2:
                    # error h^2 / 6 times a third derivative of at most 4, and 2 weights' rounding over 2 h
                    assert abs((d[0] - d[1]).item() / (2 * h) - dl[t, e].item()) < 4 * h * h + 64 * 2.0 ** -24 / h


def test_route_broadcast_and_strided_gradients(cuda_ok):
    logits = make_logits(9, 64, torch.float32, 6).requires_grad_(True)
    top = route(logits, 6, scoring="sigmoid")
    (a,) = torch.autograd.grad(top.topk_weights.sum(), logits, retain_graph=True)  # an expanded gradient
    (b,) = torch.autograd.grad(top.topk_weights, logits, torch.ones(6, 9, device=DEV).t(), retain_graph=True)
    (c,) = torch.autograd.grad(top.topk_weights, logits, torch.ones(9, 6, device=DEV))
    assert torch.equal(a, c) and torch.equal(b, c)
    base = make_logits(1, 64, torch.float32, 6).requires_grad_(True)
    g = torch.rand(9, 6, device=DEV)
    (shared,) = torch.autograd.grad(route(base.expand(9, 64), 6).topk_weights, base, g)  # one row for all tokens
    (rows,) = torch.autograd.grad(route(base.expand(9, 64).contiguous(), 6).topk_weights, base, g)
    assert torch.allclose(shared, rows, rtol=1e-6, atol=1e-8)


# --------------------------------------------------------------------------------------------------- balance loss
def balance64(logits, ids, scoring, coef, cu):
    T, E = logits.shape
    k = ids.shape[1]
    x = logits.detach().double().cpu()
    dead = torch.isneginf(x)
    x = x.masked_fill(dead, -1e4).requires_grad_(True)
    i = ids.long().cpu()
    ok = (i >= 0) & (i < E)
    cu = [0, T] if cu is None else cu.tolist()
    counts = torch.zeros(len(cu) - 1, E, dtype=torch.int32)
    loss, filled = x.new_zeros(()), 0
    a = torch.zeros(T, E, dtype=torch.float64)
    for s, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        rows = [t for t in range(lo, hi) if ok[t].any()]
        if not rows:
            continue
        filled += 1
        for t in rows:
            for e in i[t][ok[t]].tolist():
                counts[s, e] += 1
        f = E / (k * len(rows)) * counts[s].double()
        if scoring == "softmax":
            p = torch.softmax(x[rows], 1)
        else:
            sg = torch.sigmoid(x[rows]) * ~dead[rows]
            p = sg / sg.sum(1, keepdim=True)
        loss = loss + (f * p.mean(0)).sum()
        a[rows] = f / len(rows)
    loss = coef * loss / max(filled, 1)
    (dl,) = torch.autograd.grad(loss, x) if filled else (torch.zeros_like(x),)
    p = torch.softmax(x.detach(), 1)
    if scoring == "sigmoid":
        sg = torch.sigmoid(x.detach()) * ~dead
        p = sg / sg.sum(1, keepdim=True).clamp_min(1e-300)
    a = abs(coef) / max(filled, 1) * a
    # dl = p (a - sum a p) [(1 - sigmoid)]: the terms before they cancel
    mag = p * (a + (a * p).sum(1, keepdim=True))
    if scoring == "sigmoid":
        mag = mag * torch.sigmoid(-x.detach())
    return loss.detach(), counts, dl.masked_fill(dead, 0.0), mag


def check_balance(logits, ids, scoring, coef=0.3, cu=None, grad=None):
    x = logits.detach().requires_grad_(True)
    loss, counts = balance_loss(x, ids, scoring=scoring, coef=coef, cu_seqlens=cu)
    (dl,) = torch.autograd.grad(loss if grad is None else loss * grad, x)
    ref, c64, d64, mag = balance64(logits, ids, scoring, coef, cu)
    assert torch.equal(counts.cpu(), c64) and counts.dtype == torch.int32
    assert abs(loss.item() - ref.item()) <= 2 * U * abs(ref.item()) + 1e-44
    g = 1.0 if grad is None else grad
    tol = 2 * U * abs(g) * mag + torch.finfo(logits.dtype).eps / 2 * abs(g) * d64.abs() + \
        (2.0 ** -25 if logits.dtype == torch.float16 else 1e-38)
    diff = (dl.double().cpu() - g * d64).abs()
    assert (diff <= tol).all(), (diff / tol).max()
    x2 = logits.detach().requires_grad_(True)
    again, _ = balance_loss(x2, ids, scoring=scoring, coef=coef, cu_seqlens=cu)
    assert torch.equal(again, loss), "the same bits every time"
    return loss, counts, dl


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,cuts,tail", [
    (1, 8, 1, None, 0), (7, 16, 2, None, 0), (7, 16, 2, [0, 0, 3, 3, 4], 2), (64, 64, 6, [10], 0), (257, 64, 6, None, 0),
    (64, 256, 8, [1, 2, 3, 40], 5), (65, 256, 8, [1, 2, 3, 40], 5), (300, 256, 8, [100, 100, 164, 292], 8),
    (600, 72, 5, [5, 599], 0), (33, 1024, 32, [16], 1), (400, 500, 3, None, 7), (513, 16, 2, None, 0)])
def test_balance_against_the_definition(cuda_ok, T, E, k, cuts, tail, scoring, dtype):
    logits = make_logits(T, E, dtype, T + E, masked=E // 4 if k < E // 2 else 0)
    ids = route(logits, k, scoring=scoring).topk_ids
    cu = None
    if cuts is not None or tail:
        cu = torch.tensor([0] + (cuts or []) + [T - tail], dtype=torch.int32, device=DEV)
    _, _, dl = check_balance(logits, ids, scoring, cu=cu)
    assert (dl[T - tail:] == 0).all()


def test_balance_many_sequences_and_odd_ids(cuda_ok):
    gen = torch.Generator(device=DEV).manual_seed(1)
    T, E = 3000, 32
    logits = make_logits(T, E, torch.float32, 1)
    ids = torch.randint(-3, E + 3, (T, 4), device=DEV, generator=gen, dtype=torch.int32)  # unrouted, repeated, out of range
    ids[100:140] = -1
    cu = torch.sort(torch.randint(0, T, (1500,), device=DEV, generator=gen, dtype=torch.int32)).values
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), cu, torch.tensor([T - 3], dtype=torch.int32, device=DEV)])
    check_balance(logits, ids, "softmax", cu=cu)
    check_balance(logits, ids, "sigmoid", cu=cu[::40].contiguous())
    for n in (20, 600):
        none = torch.full((n, 4), -1, dtype=torch.int32, device=DEV)
        loss, counts, dl = check_balance(logits[:n], none, "softmax")
        assert loss.item() == 0 and (counts == 0).all() and (dl == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [20, 700])
def test_balance_values(cuda_ok, T, scoring):
    """Even choice gives coef; very negative rows, upstream gradients, strides."""
    E, k = 16, 2
    even = torch.arange(T * k, device=DEV, dtype=torch.int32).remainder(E).view(T, k)
    if T * k % E == 0:
        loss, _ = balance_loss(torch.zeros(T, E, device=DEV), even, scoring=scoring, coef=0.25)
        assert abs(loss.item() - 0.25) < 0.25 * 2 * U
    logits = make_logits(T, E, torch.float32, T)
    logits[::3] -= 200.0  # sigmoids that underflow before they are normalised
    check_balance(logits, even, scoring, grad=-3.0)
    wide = make_logits(T, 3 * E, torch.bfloat16, T)
    for l in (wide[:, :E], wide[:, 5:5 + E], wide[:, ::3]):
        check_balance(l, even, scoring)
    x = logits.clone().requires_grad_(True)
    loss, _ = balance_loss(x, even.t().contiguous().t(), scoring=scoring, coef=0.3)
    assert torch.equal(loss, balance_loss(logits, even, scoring=scoring, coef=0.3)[0])


def test_balance_gradient_against_differences(cuda_ok):
    T, E = 12, 8
    logits = make_logits(T, E, torch.float32, 4)
    ids = route(logits, 2).topk_ids
    cu = torch.tensor([0, 5, 12], dtype=torch.int32, device=DEV)
    for scoring in ("softmax", "sigmoid"):
        _, _, dl = check_balance(logits, ids, scoring, coef=10.0, cu=cu)
        h = 2.0 ** -6
        for t in range(T):
            for e in range(E):
                v = []
                for sign in (1, -1):
                    y = logits.clone()
                    y[t, e] += sign * h
                    v.append(balance_loss(y, ids, scoring=scoring, coef=10.0, cu_seqlens=cu)[0].double().item())
                # third derivatives of at most 6 a, a <= 10 E; the loss (of size 10) is good to 2 U
                assert abs((v[0] - v[1]) / (2 * h) - dl[t, e].item()) < 10 * E * h * h + 2 * U * 20 / h


def test_balance_streams_graph_and_saved_tensors(cuda_ok):
    logits = make_logits(700, 64, torch.float32, 3)
    ids = route(logits, 6).topk_ids
    want, counts = balance_loss(logits, ids)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = logits.clone().requires_grad_(True)
        loss, _ = balance_loss(x, ids)
        (dl,) = torch.autograd.grad(loss, x)
    s.synchronize()
    assert torch.equal(loss, want)
    g = torch.cuda.CUDAGraph()
    y = logits.clone().requires_grad_(True)
    with torch.cuda.graph(g):  # forward and backward of a leaf that no eager graph holds
        loss_g, counts_g = balance_loss(y, ids)
        (dl_g,) = torch.autograd.grad(loss_g, y)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss_g, want) and torch.equal(dl_g, dl) and torch.equal(counts_g, counts)
    z = logits.clone().requires_grad_(True)
    loss, counts = balance_loss(z, ids)
    counts += 1  # the gradient needs them
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (5, 8, 64), (1000, 8, 256), (4097, 32, 1024), (129, 3, 7)])
def test_expert_counts(cuda_ok, T, k, E):
    ids = torch.randint(-2, E + 2, (T, k), dtype=torch.int32, device=DEV)
    want = torch.bincount(ids[(ids >= 0) & (ids < E)].long(), minlength=E)
    assert torch.equal(expert_counts(ids, E).long(), want)
    assert torch.equal(expert_counts(ids.t().contiguous().t(), E).long(), want)
    assert (expert_counts(ids[:0], E) == 0).all()


def test_router_refusals(cuda_ok):
    l = make_logits(4, 16, torch.float32, 0)
    ids = route(l, 2).topk_ids
    for kw, match in ((dict(top_k=0), "top_k"), (dict(top_k=17), "top_k"), (dict(scoring="relu"), "scoring"),
                      (dict(num_groups=3), "groups"), (dict(num_groups=4, top_groups=5), "groups"),
                      (dict(bias=torch.zeros(15, device=DEV)), "bias"), (dict(bias=torch.zeros(16)), "bias"),
                      (dict(bias=torch.zeros(16, device=DEV).half()), "bias"),
                      (dict(num_tokens=torch.tensor([4], device=DEV)), "num_tokens"),
                      (dict(num_tokens=torch.tensor([4, 4], dtype=torch.int32, device=DEV)), "num_tokens")):
        kw = dict(dict(top_k=2), **kw)
        with pytest.raises(ValueError, match=match):
            route(l, **kw)
    with pytest.raises(ValueError, match="logits must be"):
        route(l.double(), 2)
    with pytest.raises(ValueError, match="experts"):
        route(torch.zeros(2, 1025, device=DEV), 2)
    for args, kw, match in (((l, ids.long()), {}, "topk_ids"), ((l, ids[:3]), {}, "topk_ids"), ((l[:0], ids[:0]), {}, "tokens"),
                            ((l, ids), dict(cu_seqlens=torch.zeros(1, dtype=torch.int32, device=DEV)), "cu_seqlens"),
                            ((l, ids), dict(cu_seqlens=torch.zeros(3, device=DEV)), "cu_seqlens")):
        with pytest.raises(ValueError, match=match):
            balance_loss(*args, **kw)
    with pytest.raises(ValueError, match="int32"):
        expert_counts(ids.long(), 16)
    with pytest.raises(ValueError, match="experts"):
        expert_counts(ids, 0)
